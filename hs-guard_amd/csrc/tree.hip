// Drafted trees over live sessions: the maps of a packed batch of trees, and the causal conv + SiLU along their paths.
//
// A row is one session's tree of at most 64 nodes, packed in an order in which every parent comes first. A node's mask has
// bit j for node j itself and for each ancestor, so it is all that the other operators need: the depth is its bit count,
// the parent the highest bit below the node's own, the ancestors in order its bits in order.
#include "hsg_common.h"

namespace hsg {
namespace {

constexpr int MOST = HSG_TREE_MAX_NODES;   // a wave's lanes, a mask's bits
constexpr int ROWS_PER_WG = 4;

// ---------------------------------------------------------------------------------------------------------
// Maps: size_n = clamp(lens[n], 0, tokens + 1), offset_n = sum of the sizes before, mask = {self} u mask(parent),
// pos = start + depth.
//
// A wave takes a row, a lane a node. Masks by pointer doubling: after step s a lane holds the last 2^s nodes of its path
// and jumps to the next one up, so six exchanges settle 64 nodes whatever the tree's depth. Offsets: every workgroup sums
// the sizes of the rows before its own (n / 256 reads a thread), so the rows need no second launch. A launch's latency
// bounds it: 4 rows of 24 nodes 2.8 us, 512 of 64 4.0.
// ---------------------------------------------------------------------------------------------------------
__global__ __launch_bounds__(64 * ROWS_PER_WG) void tree_maps_kernel(const int64_t* parents, int64_t tokens,
                                                                     const int64_t* lens, const int64_t* starts,
                                                                     const int64_t* commits, int n_rows, int max_nodes,
                                                                     int64_t* offsets, int64_t* lens_out,
                                                                     int64_t* commits_out, int64_t* pos, int64_t* masks) {
  __shared__ int64_t part[ROWS_PER_WG];
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int row0 = blockIdx.x * ROWS_PER_WG;
  const auto size_of = [&](int r) {
    const int64_t len = lens[r];
    return len < 0 ? (int64_t)0 : len > tokens ? tokens + 1 : len;   // the sum of any number of rows fits 63 bits
  };
  int64_t before = 0;
  for (int r = threadIdx.x; r < row0; r += 64 * ROWS_PER_WG) before += size_of(r);
  for (int o = 1; o < 64; o <<= 1) before += __shfl_xor(before, o, 64);
  if (lane == 0) part[wave] = before;
  __syncthreads();
  int64_t off = 0;
  for (int w = 0; w < ROWS_PER_WG; ++w) off += part[w];
  for (int w = 0; w < wave; ++w)
    if (row0 + w < n_rows) off += size_of(row0 + w);
  const int r = row0 + wave;
  if (r < n_rows) {
    const int64_t len = lens[r], size = size_of(r);
    const int64_t done = commits ? commits[r] : 0;
    const int64_t start = starts[r];
    const bool fits = (len >= 0) & (size <= max_nodes) & (off + size <= tokens) & (start >= 0) & (done >= 0) & (done <= size);
    const bool inside = fits && lane < size;
    const int64_t p = inside ? parents[off + lane] : lane - 1;
    const bool good = (p >= -1) & (p < lane) & ((p == lane - 1) | (lane >= done));
    const bool valid = fits && __all(good);
    uint64_t mask = 1ull << lane;
    int up = valid ? (int)p : -1;
#pragma unroll
    for (int s = 0; s < 6; ++s) {
      const int at = up < 0 ? lane : up;   // a lane at the root adds its own bits again
      mask |= (uint64_t)__shfl((long long)mask, at, 64);
      const int next = __shfl(up, at, 64);
      up = up < 0 ? -1 : next;
    }
    // a rejected row's tokens (there may be more than 64 of them) are nobody's: zeros
    for (int64_t i = lane; i < size && off + i < tokens; i += 64) {
      pos[off + i] = valid ? start + (int64_t)__popcll(mask) - 1 : 0;
      masks[off + i] = valid ? (int64_t)mask : 0;
    }
    if (lane == 0) {
      offsets[r] = off;
      lens_out[r] = valid ? size : 0;
      if (commits_out) commits_out[r] = valid ? done : 0;
    }
  }
  // the tokens behind the last row (of a buffer rounded up to a bucket)
  if (row0 + ROWS_PER_WG >= n_rows) {
    int64_t end = 0;
    for (int w = 0; w < ROWS_PER_WG; ++w) end += part[w];
    for (int w = 0; w < ROWS_PER_WG; ++w)
      if (row0 + w < n_rows) end += size_of(row0 + w);
    for (int64_t i = end + threadIdx.x; i < tokens; i += 64 * ROWS_PER_WG) {
      pos[i] = 0;
      masks[i] = 0;
    }
  }
}

// ---------------------------------------------------------------------------------------------------------
// Conv + SiLU: out = silu(sum_t w[3 - t] x(t nodes up)), past the root from the slot's history (oldest first), summed in
// fp32 and rounded once. A workgroup holds one row's nodes and the history of a block of channels in LDS, NODES x CH of
// them (16 KB), so each input is read once whatever the tree; a thread's four 16-byte loads, the history and the weights are all
// in flight before the first is waited for (352 rows of 21 nodes, 6,144 channels, with commits: 45 us without that, 34.5 with it,
// 4.2 TB/s against the 5.2 of a copy). The committed chain moves the history after every read of it: no other workgroup reads
// these channels of the slot.
// ---------------------------------------------------------------------------------------------------------
constexpr int TAPS = 4;
constexpr int TILE = 8192;    // values of a workgroup's tile (352 x 21 nodes: half as many 43 us, twice 35.5)

template <int NODES>
__global__ __launch_bounds__(256) void tree_conv_kernel(const uint16_t* x, int64_t x_stride, uint16_t* pool,
                                                        int64_t pool_rows, const uint16_t* weight, const int64_t* slots,
                                                        const int64_t* lens, const int64_t* offsets,
                                                        const int64_t* commits, const int64_t* masks, int max_nodes,
                                                        int channels, uint16_t* out, int64_t out_stride) {
  constexpr int CH = TILE / NODES;            // channels of the workgroup
  constexpr int COLS = CH / 8;                // 16-byte pieces of them
  constexpr int STEP = 256 / COLS;            // nodes apart of a thread's pieces
  constexpr int EACH = NODES / STEP;          // pieces of a thread
  __shared__ __align__(16) uint16_t tile[(NODES + TAPS - 1) * CH];   // nodes, then the history
  const int n = blockIdx.y;
  const int64_t slot = slots[n], len64 = lens[n], off = offsets[n];
  const int64_t done64 = commits ? commits[n] : 0;
  if ((slot < 0) | (slot >= pool_rows) | (len64 <= 0) | (len64 > max_nodes)) return;
  const int len = (int)len64;
  const int col = threadIdx.x % COLS, first = threadIdx.x / COLS;
  const int c = blockIdx.x * CH + 8 * col;
  const bool mine = c < channels;
  uint16_t* const hist = pool + slot * (TAPS - 1) * channels + c;
  // every load is in flight before the first is waited for
  constexpr int OLD = (TAPS - 1 + STEP - 1) / STEP;   // history rows of a thread
  u32x4 piece[EACH], old[OLD], wt[TAPS] = {};
  uint64_t mask[EACH];
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int i = first + STEP * e;
    if (i >= len || !mine) break;
    piece[e] = *reinterpret_cast<const u32x4*>(x + (off + i) * x_stride + c);
    mask[e] = (uint64_t)masks[off + i];
  }
#pragma unroll
  for (int h = 0; h < OLD; ++h)
    if (mine && first + STEP * h < TAPS - 1)
      old[h] = *reinterpret_cast<const u32x4*>(hist + (int64_t)(first + STEP * h) * channels);
  if (mine && first < len) {
#pragma unroll
    for (int t = 0; t < TAPS; ++t) wt[t] = *reinterpret_cast<const u32x4*>(weight + (int64_t)c * TAPS + 8 * t);
  }
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int i = first + STEP * e;
    if (i >= len || !mine) break;
    *reinterpret_cast<u32x4*>(&tile[i * CH + 8 * col]) = piece[e];
  }
#pragma unroll
  for (int h = 0; h < OLD; ++h)
    if (mine && first + STEP * h < TAPS - 1)
      *reinterpret_cast<u32x4*>(&tile[(NODES + first + STEP * h) * CH + 8 * col]) = old[h];
  __syncthreads();
  if (!mine) return;
  // weight[channel][tap]: piece t holds channels 2 t and 2 t + 1
  float w[8][TAPS];
#pragma unroll
  for (int t = 0; t < TAPS; ++t) {
    unpack2(wt[t][0], w[2 * t][0], w[2 * t][1]);
    unpack2(wt[t][1], w[2 * t][2], w[2 * t][3]);
    unpack2(wt[t][2], w[2 * t + 1][0], w[2 * t + 1][1]);
    unpack2(wt[t][3], w[2 * t + 1][2], w[2 * t + 1][3]);
  }
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int i = first + STEP * e;
    if (i >= len) break;
    uint64_t up = mask[e] & ((1ull << i) - 1);                    // the ancestors not yet taken
    int row[TAPS];
    row[0] = i;
    int h = TAPS - 1;                                             // the next history row up, plus one
#pragma unroll
    for (int t = 1; t < TAPS; ++t) {
      const int top = 63 - __clzll((long long)(up | 1ull));
      row[t] = up ? top : NODES + --h;
      up &= ~(1ull << top);
    }
    float acc[8] = {};
#pragma unroll
    for (int t = TAPS - 1; t >= 0; --t) {
      float v[8];
      load8_bf16(&tile[row[t] * CH + 8 * col], v);
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] = __builtin_fmaf(w[j][TAPS - 1 - t], v[j], acc[j]);
    }
    u32x4 y;
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = pack_bf16x2(siluf_(acc[2 * j]), siluf_(acc[2 * j + 1]));
    *reinterpret_cast<u32x4*>(out + (off + i) * out_stride + c) = y;
  }
  const int done = (int)(done64 < 0 ? 0 : done64 > len ? len : done64);
  if (done > 0) {
    // history row h becomes entry done + h of (history, chain)
    for (int h = first; h < TAPS - 1; h += STEP) {
      const int e = done + h;
      const int from = e < TAPS - 1 ? NODES + e : e - (TAPS - 1);
      *reinterpret_cast<u32x4*>(hist + (int64_t)h * channels) = *reinterpret_cast<const u32x4*>(&tile[from * CH + 8 * col]);
    }
  }
}

}  // namespace
}  // namespace hsg

extern "C" int hsg_tree_maps(const int64_t* parents, int64_t tokens, const int64_t* lens, const int64_t* starts,
                             const int64_t* commits, int32_t n_rows, int32_t max_nodes, int64_t* offsets,
                             int64_t* lens_out, int64_t* commits_out, int64_t* pos, int64_t* masks, void* stream) {
  using namespace hsg;
  if (n_rows < 0 || tokens < 0 || tokens > ((int64_t)1 << 40)) return HSG_ERR_ARG;
  if (max_nodes <= 0 || max_nodes > MOST || n_rows > 65535) return HSG_ERR_SHAPE;   // (the sums before a row grow as rows^2)
  if (n_rows == 0 && tokens == 0) return HSG_OK;
  if (n_rows && (!lens || !starts || !offsets || !lens_out || (commits && !commits_out))) return HSG_ERR_ARG;
  if (tokens && (!parents || !pos || !masks)) return HSG_ERR_ARG;
  // every workgroup reads lens while others write
  if (n_rows && (lens_out == lens || offsets == lens || (commits && commits_out == lens))) return HSG_ERR_ARG;
  const unsigned blocks = n_rows ? ((unsigned)n_rows + ROWS_PER_WG - 1) / ROWS_PER_WG : 1;
  hipLaunchKernelGGL(tree_maps_kernel, dim3(blocks), dim3(64 * ROWS_PER_WG), 0, reinterpret_cast<hipStream_t>(stream),
                     parents, tokens, lens, starts, commits, n_rows, max_nodes, offsets, lens_out,
                     commits ? commits_out : nullptr, pos, masks);
  return launch_status();
}

extern "C" int hsg_tree_conv_silu(const void* x, int64_t x_stride, void* pool, int64_t pool_rows, const void* weight,
                                  int32_t kernel_size, const int64_t* slots, const int64_t* lens, const int64_t* offsets,
                                  const int64_t* commits, const int64_t* masks, int32_t n_rows, int32_t max_nodes,
                                  int32_t channels, void* out, int64_t out_stride, void* stream) {
  using namespace hsg;
  if (n_rows < 0 || channels <= 0 || pool_rows <= 0) return HSG_ERR_ARG;
  if (kernel_size != TAPS || max_nodes <= 0 || max_nodes > MOST) return HSG_ERR_SHAPE;
  if (n_rows == 0) return HSG_OK;
  if (!x || !pool || !weight || !slots || !lens || !offsets || !masks || !out) return HSG_ERR_ARG;
  if (x_stride < channels || out_stride < channels || (out == x && out_stride != x_stride)) return HSG_ERR_ARG;
  if (channels % 8 || x_stride % 8 || out_stride % 8 || !aligned(x, 16) || !aligned(pool, 16) || !aligned(weight, 16) ||
      !aligned(out, 16))
    return HSG_ERR_ALIGN;
  if (n_rows > 65535) return HSG_ERR_SHAPE;
  const auto launch = [&](auto kernel, int nodes) {
    const int ch = TILE / nodes;
    hipLaunchKernelGGL(kernel, dim3((channels + ch - 1) / ch, n_rows), dim3(256), 0, reinterpret_cast<hipStream_t>(stream),
                       static_cast<const uint16_t*>(x), x_stride, static_cast<uint16_t*>(pool), pool_rows,
                       static_cast<const uint16_t*>(weight), slots, lens, offsets, commits, masks, max_nodes, channels,
                       static_cast<uint16_t*>(out), out_stride);
  };
  // Few rows take the narrowest blocks of channels, of which there are the most (of 6,144 channels: 1 x 12 nodes 3.3 against 4.4
  // us, 8 x 12 3.7 and 4.6, 20 x 12 4.6 and 5.0, 40 x 12 6.2 and 6.3); many rows blocks of their nodes (352 x 21 34.9 and 43 us,
  // 352 x 12 21.5 and 24; of 8 nodes at most, 16 x 512 values were as fast as 8 x 1024).
  if (n_rows > 32 && max_nodes <= 16) launch(tree_conv_kernel<16>, 16);
  else if (n_rows > 32 && max_nodes <= 32) launch(tree_conv_kernel<32>, 32);
  else launch(tree_conv_kernel<64>, 64);
  return launch_status();
}
