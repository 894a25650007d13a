// Window attention of a drafted tree's nodes over the slot's ring and each node's own ancestors, gated, for gfx950 on MFMA.
//
// Node i of a row stands at start + depth_i. It sees the ring's keys at 0 <= p < start, p > start + depth_i - W, and of the
// tree's keys those of its ancestors and its own that lie within W of it. Nothing of the ring moves but the columns of the
// committed chain, after all reads: at its workgroup's end where a (row, kv head) has one, else in a launch of its own.
//
// Query rows r = node * G + (query head of the kv head) form tiles of 16, one or two to a wave. Per block of 32 keys, on
// v_mfma_f32_16x16x32_bf16:
//   S^T[key, query] = K . Q^T      a lane's column is one query: maxima, sums and rescales are per-lane scalars
//   O^T[d, query] += V^T . P^T     B = P straight from the S^T accumulators (the product's key order is the lane's own)
// The running maximum is moved only when a block's exceeds it by 2^8, so the accumulators are seldom rescaled; sums are fp32
// and P is rounded to bf16 for its product (2^-8 of each weight at most, as the output's own rounding; over a row's keys they
// average out), the weights' sum taking it as rounded.
//
// Up to 16 query rows a (row, kv head), bound by reading the ring: the four waves split its KEYS, a wave's keys and values
// going straight from memory to its operand registers (of a value 8 dims of a lane's 8 keys, whose 16-bit halves it swaps),
// and meet in LDS at the end, weighted by their maxima; no barrier and no LDS write in the loop. 352 rows of one node over
// full rings, 16 q / 4 kv heads: 118 us, 5.6 TB/s (nontemporal loads; with ordinary ones 122, while keys through LDS, which
// other workgroups read too, take 117 us with nontemporal and 105 with ordinary loads at 128 x 64).
// More query rows: every wave has one or two tiles of its own and needs every key, so blocks pass through LDS once for the
// four waves (two stages of 32 KB, direct-to-LDS loads, one barrier a block; two workgroups on a CU). Keys are read as they
// lie, values by transpose reads, both ahead of their products, and waves at their products go before waves at their softmax.
// 128 rows of 64 nodes with commits: 109 us, where the bytes alone take 78; a block of a workgroup takes 2.1 us, of which its
// 64 products a wave are 0.9 for the two workgroups that share a SIMD, the rest softmax, LDS reads and the issue of the next
// block's loads; 5.5 us before the loop (ring positions, queries, first block) and 6 after it (gates, outputs) are not
// hidden. Operands by byte permutes instead of transpose reads and reads right before their products made it 131 us; four
// tiles a wave spilled: 1,040 us.
// Where few rows leave the chip short of workgroups, workgroups split a row's key blocks further and a second launch joins
// their partial sums: a lone row of 12 nodes 9.4 + 3.7 us, both a chain of dependent loads.
//
// A masked pair has P = 0, which would carry a NaN or an infinity of a value to queries that do not see it: columns that no
// query of the row sees are not read (another key's are, in their place), and a query row with a result that is not finite is
// computed again from the keys that it sees alone (walk_keys).
#include <math.h>
#include <stddef.h>

#include "hsg_common.h"

namespace hsg {
namespace {

constexpr int D = 256;
constexpr int NW = 4;
constexpr int KB = 32;                 // keys of a block
constexpr int W_MAX = 512;
constexpr int MOST = HSG_TREE_MAX_NODES;
constexpr int BLOCKS = W_MAX / KB + MOST / KB;
constexpr int KP_NONE = -(1 << 30);    // an empty ring column
constexpr int KP_FAR = 1 << 29;        // clamp of a position relative to the row's start
constexpr float LOG2E = 1.4426950408889634f;
constexpr int SPLITS_MAX = 8;          // workgroups that split a row's key blocks
constexpr float SLACK = 8.f;           // log2 of how far a score may exceed the running maximum before it is moved

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(4))) int i32x4;

struct TreeAttnParams {
  const uint16_t* q; int64_t q_sl, q_sh, q_sg;
  uint16_t* ring_k; uint16_t* ring_v; int64_t ring_rows; int W;
  const uint16_t* new_k; int64_t nk_sl, nk_sh;
  const uint16_t* new_v; int64_t nv_sl, nv_sh;
  const uint16_t* gate; int64_t g_sl, g_sh, g_sg, g_off;
  const int64_t* ring_pos; const int64_t* slots; const int64_t* starts; const int64_t* lens; const int64_t* offsets;
  const int64_t* commits; const int64_t* masks;
  int max_nodes, hkv, G;
  float scale;
  int pairs;        // rows x kv heads
  int qblocks;      // workgroups of query rows a pair
  int splits;       // workgroups of key blocks
  bool write_here;  // rows commit, and a pair has one workgroup
  float* part_o;    // [pair][split][query row][D]: partial sums
  float* part_ml;   // [pair][split][query row][2]: their maxima and weights' sums
  uint16_t* out; int64_t o_sl, o_sh, o_sg;
};

// A (row, kv head): element pointers of its first node
struct TreeKeys {
  const uint16_t* q; const uint16_t* k; const uint16_t* v; const uint16_t* gate; uint16_t* out;
  const uint16_t* ring_k; const uint16_t* ring_v;   // column 0
  const int64_t* ring_pos; const int64_t* masks;
  int64_t start;
  int len;
};

__device__ __forceinline__ bool tree_keys(const TreeAttnParams& p, int n, int h, TreeKeys& ro) {
  const int64_t slot = p.slots[n], len = p.lens[n], off = p.offsets[n];
  ro.start = p.starts[n];
  if ((slot < 0) | (slot >= p.ring_rows) | (len <= 0) | (len > p.max_nodes)) return false;
  ro.len = (int)len;
  ro.q = p.q + off * p.q_sl + h * p.q_sh;
  ro.k = p.new_k + off * p.nk_sl + h * p.nk_sh;
  ro.v = p.new_v + off * p.nv_sl + h * p.nv_sh;
  ro.gate = p.gate ? p.gate + off * p.g_sl + h * p.g_sh + p.g_off : nullptr;
  ro.out = p.out + off * p.o_sl + h * p.o_sh;
  const int64_t ring = ((slot * p.hkv + h) * (int64_t)(p.W + 1)) * D;
  ro.ring_k = p.ring_k + ring;
  ro.ring_v = p.ring_v + ring;
  ro.ring_pos = p.ring_pos + slot * (int64_t)(p.W + 1);
  ro.masks = p.masks + off;
  return true;
}

__device__ __forceinline__ bf16x8 as_bf16x8(u32x4 w) { return __builtin_bit_cast(bf16x8, w); }
__device__ __forceinline__ u32x4 load16(const uint16_t* p) { return *reinterpret_cast<const u32x4*>(p); }
// 16 bytes at byte `off` of a base that is the same for all lanes: its address takes one register of a lane
__device__ __forceinline__ u32x4 load16_at(const uint16_t* base, uint32_t off) {
  return __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(base) + off));
}
// the largest of three, a NaN aside, in one instruction (fmaxf quiets its operands first, an instruction each)
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
// sigmoid to a few fp32 steps (its product is rounded to bf16), 4 instructions against the exact one's 16: an epilogue of 2
// tiles holds 64 a lane
__device__ __forceinline__ float gate_of(float x) { return __builtin_amdgcn_rcpf(1.0f + exp2_fast(-LOG2E * x)); }

// node i's ancestors and itself
__device__ __forceinline__ uint64_t mask_of(const int64_t* masks, int i) {
  const uint64_t self = 1ull << i;
  return ((uint64_t)masks[i] & (self - 1)) | self;
}

// node i's depth
__device__ __forceinline__ int depth_of(const int64_t* masks, int i) { return (int)__popcll(mask_of(masks, i)) - 1; }

// position of a ring column's key before the row's start, or KP_NONE
__device__ __forceinline__ int key_place(int64_t kpos, int64_t start) {
  const int64_t d = kpos - start;
  return kpos < 0 || d >= 0 ? KP_NONE : (int)(d < -KP_FAR ? -KP_FAR : d);
}

// ND values (dims d0 ..) of query `row` by definition, over the keys it sees alone: in one pass with a running maximum. A query
// has D / ND lanes (with 8 dims a wave has two queries), which share each key's product; all of the wave's lanes come here. A
// lane asks for one of 32 keys whether its query sees it, and of those that any of the wave's does, 8 are in flight at a time.
// One session whose ring holds a NaN comes here in every layer and call, and all others of the call wait for it: 128 x 64 nodes
// with one such ring 52.6 ms where each lane walked each key's 256 dims alone, 1.9 now.
template <int ND>
__device__ __forceinline__ void walk_keys(const TreeAttnParams& p, const TreeKeys& ro, int row, int d0, float (&y)[ND]) {
  constexpr int EACH = 8;
  const int lane = threadIdx.x & 63;
  const int l = row / p.G;
  const uint64_t mask = mask_of(ro.masks, l);
  const int depth = (int)__popcll(mask) - 1;
  const auto load = [](const uint16_t* from, float (&x)[ND]) {
    if constexpr (ND == 8) load8_bf16(from, x);
    else load4_bf16(from, x);
  };
  float q[ND];
  load(ro.q + l * p.q_sl + (row - l * p.G) * p.q_sg + d0, q);
  float m = -INFINITY, sum = 0.f;
#pragma unroll
  for (int e = 0; e < ND; ++e) y[e] = 0.f;
  const int ring_blocks = p.W / KB;
#pragma unroll 1
  for (int b = 0; b < ring_blocks + (ro.len + KB - 1) / KB; ++b) {
    const bool ring = b < ring_blocks;
    const int first = ring ? b * KB : (b - ring_blocks) * KB;
    const int at = first + (lane & 31);
    const bool sees = ring ? key_place(ro.ring_pos[at], ro.start) > depth - p.W
                           : at < ro.len && (mask >> at & 1) && depth_of(ro.masks, at) > depth - p.W;
    const uint64_t ballot = __ballot(sees);
    const uint32_t mine = (uint32_t)(ballot >> (lane & 32));
    uint32_t any = (uint32_t)ballot | (uint32_t)(ballot >> 32);
    const uint16_t* const kb = (ring ? ro.ring_k : ro.k) + d0;
    const uint16_t* const vb = (ring ? ro.ring_v : ro.v) + d0;
    const int64_t k_st = ring ? D : p.nk_sl, v_st = ring ? D : p.nv_sl;
#pragma unroll 1
    while (any) {
      float k[EACH][ND], v[EACH][ND], s[EACH];
      bool on[EACH];
#pragma unroll
      for (int e = 0; e < EACH; ++e) {
        const int r = any ? __builtin_ctz(any) : -1;   // none left: the block's first key, not used
        any &= any - 1;
        on[e] = r >= 0 && (mine >> (r & 31) & 1u);
        const int64_t key = first + max(r, 0);
        load(kb + key * k_st, k[e]);
        load(vb + key * v_st, v[e]);
      }
      float top = m;
#pragma unroll
      for (int e = 0; e < EACH; ++e) {
        s[e] = 0.f;
#pragma unroll
        for (int i = 0; i < ND; ++i) s[e] = __builtin_fmaf(q[i], k[e][i], s[e]);
        s[e] = (ND == 8 ? sum32_dpp(s[e]) : wave_sum(s[e])) * p.scale;
        if (on[e]) top = fmaxf(top, s[e]);
      }
      const float base = top == -INFINITY ? 0.f : top;
      const float alpha = expf(m - base);
      m = top;
      sum *= alpha;
#pragma unroll
      for (int i = 0; i < ND; ++i) y[i] *= alpha;
#pragma unroll
      for (int e = 0; e < EACH; ++e) {
        const float w = expf(s[e] - base);
        if (on[e]) {
          sum += w;
#pragma unroll
          for (int i = 0; i < ND; ++i) y[i] = __builtin_fmaf(w, v[e][i], y[i]);
        }
      }
    }
  }
#pragma unroll
  for (int e = 0; e < ND; ++e) y[e] /= sum;
}

template <int ND>
__device__ __forceinline__ bool all_finite(const float (&y)[ND]) {
  float odd = 0.f;
#pragma unroll
  for (int e = 0; e < ND; ++e) odd += y[e] * 0.f;
  return odd == 0.f;
}

// The gate of ND values (dims d0 ..) of query `row`
template <int N8>
__device__ __forceinline__ void load_gate(const TreeAttnParams& p, const TreeKeys& ro, int row, int d0, u32x4 (&gw)[N8]) {
  if (!ro.gate) return;
  const int l = row / p.G, g = row - l * p.G;
  const uint16_t* src = ro.gate + l * p.g_sl + g * p.g_sg + d0;
#pragma unroll
  for (int e = 0; e < N8; ++e) gw[e] = load16(src + 8 * e);
}

// ND normalised values of query `row`, gated and stored (dims d0 ..)
template <int ND>
__device__ __forceinline__ void store_gated(const TreeAttnParams& p, const TreeKeys& ro, int row, int d0, float (&y)[ND],
                                            const u32x4 (&gw)[ND / 8]) {
  const int l = row / p.G, g = row - l * p.G;
  uint16_t* dst = ro.out + l * p.o_sl + g * p.o_sg + d0;
  if (ro.gate) {
#pragma unroll
    for (int e = 0; e < ND / 8; ++e) {
      float gt[8];
      unpack8(gw[e], gt);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[8 * e + i] *= gate_of(gt[i]);
    }
  }
#pragma unroll
  for (int e = 0; e < ND; e += 8) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = pack_bf16x2(y[e + 2 * i], y[e + 2 * i + 1]);
    *reinterpret_cast<u32x4*>(dst + e) = w;
  }
}

// The committed chain's keys and values into the ring (of a chain longer than the window its last W), 16 nodes at a time of
// which the caller takes every `step`-th: a thread's 16-byte pieces are loaded before any of them is stored
__device__ __forceinline__ void write_chain(const TreeAttnParams& p, int n, int h, int block, int step) {
  const int64_t slot = p.slots[n], len = p.lens[n], off = p.offsets[n], start = p.starts[n], done64 = p.commits[n];
  if ((slot < 0) | (slot >= p.ring_rows) | (len <= 0) | (len > p.max_nodes) | (done64 <= 0)) return;
  const int done = (int)(done64 > len ? len : done64);
  const int64_t ring = ((slot * p.hkv + h) * (int64_t)(p.W + 1)) * D;
  const int64_t start_col = ((start % p.W) + p.W) % p.W;
  constexpr int EACH = 2;   // nodes of a thread: 8 nodes of 32 pieces at a time
  const int d = 8 * (threadIdx.x & 31);
  for (int first = max(0, done - p.W) + block * (8 * EACH); first < done; first += step * (8 * EACH)) {
    u32x4 k[EACH], v[EACH];
    int node[EACH];
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      node[e] = first + 8 * e + (int)(threadIdx.x >> 5);
      const int64_t t = off + min(node[e], done - 1);
      k[e] = load16(p.new_k + t * p.nk_sl + h * p.nk_sh + d);
      v[e] = load16(p.new_v + t * p.nv_sl + h * p.nv_sh + d);
    }
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      if (node[e] >= done) continue;
      const int64_t at = ring + ((start_col + node[e]) % p.W) * D + d;
      *reinterpret_cast<u32x4*>(p.ring_k + at) = k[e];
      *reinterpret_cast<u32x4*>(p.ring_v + at) = v[e];
    }
  }
}

// byte offset of an LDS pointer
__device__ __forceinline__ uint32_t lds_offset(const void* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}

__device__ __forceinline__ const uint16_t* lds_pointer(uint32_t byte) {
  return (const uint16_t*)(const __attribute__((address_space(3))) uint16_t*)(uintptr_t)byte;
}

// 1 KB from memory into LDS without a register between: lane l's 16 bytes at byte `off` of `base` go to byte `to` + 16 l.
// Counted by vmcnt in the order of issue.
__device__ __forceinline__ void load_lds16(const void* base, uint32_t off, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(off), "s"(base) : "memory", "m0");
}

// LDS transpose read: within each group of 16 lanes, lane 4 q + e receives element e of the 4-value vectors that lanes q, q + 4,
// q + 8 and q + 12 of its group address
typedef __attribute__((ext_vector_type(4))) short s16x4;
__device__ __forceinline__ u32x2 ld_tr4(const uint16_t* p) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p)));
}

// Rows of 512 bytes, each loaded whole. The 16-byte pieces of a row are permuted by its number (piece pc of row r at pc ^ r %
// 16), so that the scores' operand, one piece of 16 rows, and the values' transpose reads, 4 pieces of 16 rows, spread over
// the banks.
struct KeyStage {
  uint16_t k[KB][D];
  uint16_t v[KB][D];
};

// T: tiles of a wave; STAGED: keys pass through LDS, else the waves split them
template <int T, bool STAGED>
struct TreeAttnLds {
  static constexpr int QW = STAGED ? NW : 1;    // waves with queries of their own
  union {
    u32x4 q[STAGED ? 1 : D / 32][64];           // the queries' operands, in the order of the lanes
    KeyStage stage[STAGED ? 2 : 1];
    f32x4 o[STAGED ? 1 : NW][16][64];           // every wave's partial sums
  };
  int kp[W_MAX + MOST];       // places of the ring's keys before the start; then the nodes' depths
  uint64_t mask[MOST];        // the nodes' ancestors and themselves
  uint32_t live[BLOCKS];      // per block: the keys that some query of the row sees; a block's other columns hold anything
  uint32_t whole[BLOCKS];     // every query sees every key
  float ml[NW][T][16][2];
  uint32_t odd[QW * T];       // query rows with a result that is not finite
  __device__ TreeAttnLds() {}
};

template <int T, bool STAGED>
__global__ __launch_bounds__(64 * NW, 2) void tree_attn_kernel(const TreeAttnParams p) {
  static_assert(STAGED || T == 1, "the split of the keys takes one tile");
  constexpr int QW = STAGED ? NW : 1, KW = NW / QW;   // waves of queries, of keys
  constexpr int ROWS = 16 * T * QW;     // query rows of the workgroup
  __shared__ __align__(16) TreeAttnLds<T, STAGED> lds;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wk = wave % KW, wq = wave / KW;
  const int g4 = lane >> 4, c = lane & 15;
  // Workgroups are dealt round-robin over the 8 XCDs: the ones of a pair follow one another on one XCD, whose L2 then serves
  // its keys to all but the first.
  const int per = p.qblocks * p.splits;
  const int seq = blockIdx.x >> 3;
  const int pair = seq / per * 8 + (blockIdx.x & 7);
  if (pair >= p.pairs) return;
  const int part = seq % per;
  const int qb = part / p.splits, split = part - qb * p.splits;
  const int n = pair / p.hkv, h = pair - n * p.hkv;
  TreeKeys ro;
  if (!tree_keys(p, n, h, ro)) return;
  const int W = p.W, G = p.G, len = ro.len;
  const int M = G * len;
  const int r_wg = qb * ROWS;
  if (r_wg >= M) return;
  const int r_lo = r_wg + 16 * T * wq;
  const int tiles = min(T, max(0, (M - r_lo + 15) >> 4));   // of this wave
  const int l_hi = (min(r_wg + ROWS, M) - 1) / G;           // last node of the workgroup
  const int RB = W / KB;
  const int n_blocks = RB + l_hi / KB + 1;
  const int step = KW * p.splits;
  const int b_first = wk + KW * split;                      // the first of the wave's blocks

  // ---- queries, and places of the keys ----
  int64_t ring_pos[W_MAX / (64 * NW)];
#pragma unroll
  for (int e = 0; e < W_MAX / (64 * NW); ++e) ring_pos[e] = ro.ring_pos[min((int)threadIdx.x + 64 * NW * e, W - 1)];
  const uint64_t mask = threadIdx.x < MOST ? mask_of(ro.masks, min((int)threadIdx.x, len - 1)) : 0ull;
  bf16x8 qr[STAGED ? T : 1][D / 32];
  int node[T];
  const uint32_t sign = p.scale < 0.f ? 0x80008000u : 0u;    // a scale's sign goes to the queries
#pragma unroll
  for (int t = 0; t < T; ++t) {
    const int row = min(r_lo + 16 * t + c, M - 1);           // past the valid rows: the last one again, not stored
    const int l = row / G;
    const uint16_t* src = ro.q + l * p.q_sl + (row - l * G) * p.q_sg + 8 * g4;
    node[t] = l;
    if constexpr (STAGED) {
#pragma unroll
      for (int ks = 0; ks < D / 32; ++ks) qr[t][ks] = as_bf16x8(load16(src + 32 * ks) ^ sign);
    } else {
#pragma unroll
      for (int ks = wk; ks < D / 32; ks += KW) lds.q[ks][lane] = load16(src + 32 * ks) ^ sign;
    }
  }
  const auto live_nodes = [&](int b) {   // of the tree's block b
    const int n = len - (b - RB) * KB;
    return n >= KB ? ~0u : (1u << n) - 1u;
  };
  // a key that no query sees is read as one that is
  const auto live_of = [&](int b) { return b < RB ? __builtin_amdgcn_readfirstlane(lds.live[b]) : live_nodes(b); };
  const auto seen_row = [](uint32_t live, int r) { return (uint32_t)(live >> r & 1u ? r : __builtin_ctz(live)); };
  // (STAGED) block b's keys and values on their way into a stage
  constexpr int EACH = 2 * KB * D * 2 / 1024 / NW;      // a wave's loads of a block
  const auto fetch = [&](int b, int stage, bool all) __attribute__((always_inline)) {
    const bool ring = b < RB;
    const uint16_t* kb = ring ? ro.ring_k + b * (KB * D) : ro.k + (int64_t)(b - RB) * KB * p.nk_sl;
    const uint16_t* vb = ring ? ro.ring_v + b * (KB * D) : ro.v + (int64_t)(b - RB) * KB * p.nv_sl;
    const uint32_t to = lds_offset(&lds.stage[stage]) + 1024 * (EACH / 2) * wave;
    // load e of the wave brings rows 2 o and 2 o + 1 of keys and values, o = wave * (EACH / 2) + e
    const int l = lane_per_site(lane);
    const int row = wave * EACH + (l >> 5);
    const uint32_t piece = 16 * ((l & 31) ^ (row & 15));   // (the rows of a wave share all but bits 1 and 2, which 2 e sets)
    if (all) {
      const uint32_t off = row * (2 * D) + piece;
#pragma unroll
      for (int e = 0; e < EACH / 2; ++e) {
        load_lds16(kb + 2 * e * D, off ^ (32 * e), to + 1024 * e);
        load_lds16(vb + 2 * e * D, off ^ (32 * e), to + (uint32_t)offsetof(KeyStage, v) + 1024 * e);
      }
    } else {
      const uint32_t live = live_of(b);
      const uint32_t k_st = ring ? 2 * D : (uint32_t)(2 * p.nk_sl), v_st = ring ? 2 * D : (uint32_t)(2 * p.nv_sl);
#pragma unroll
      for (int e = 0; e < EACH / 2; ++e) {
        const uint32_t at = seen_row(live, row + 2 * e);
        load_lds16(kb, at * k_st + (piece ^ (32 * e)), to + 1024 * e);
        load_lds16(vb, at * v_st + (piece ^ (32 * e)), to + (uint32_t)offsetof(KeyStage, v) + 1024 * e);
      }
    }
  };
  // the tree's first block, which needs nothing of the maps, is on its way first
  const bool tree_first = STAGED && (RB - b_first) % step == 0;
  if constexpr (STAGED) {
    if (tree_first) fetch(RB, 0, false);
  }
#pragma unroll
  for (int e = 0; e < W_MAX / (64 * NW); ++e) {
    const int col = threadIdx.x + 64 * NW * e;
    const int place = col < W ? key_place(ring_pos[e], ro.start) : KP_NONE;
    lds.kp[col] = place;
    const uint64_t live = __ballot(place > -W), whole = __ballot(place > len - 1 - W);
    if (lane == 0) {
      lds.live[col / KB] = (uint32_t)live;
      lds.live[col / KB + 1] = (uint32_t)(live >> 32);
      lds.whole[col / KB] = (uint32_t)whole == ~0u;
      lds.whole[col / KB + 1] = (uint32_t)(whole >> 32) == ~0u;
    }
  }
  if (threadIdx.x < MOST) {
    lds.mask[threadIdx.x] = mask;
    lds.kp[W_MAX + threadIdx.x] = (int)__popcll(mask) - 1;
  }
  if (threadIdx.x < QW * T) lds.odd[threadIdx.x] = 0u;
  if constexpr (STAGED) lds_barrier();   // (the block's loads stay in flight)
  else __syncthreads();

  // ---- the wave's key blocks ----
  const float sl2 = fmaxf(fabsf(p.scale) * LOG2E, 1e-37f);   // (not 0: a masked score is -inf)
  float m[T], sum[T];   // (sum: of the lane's own keys)
  f32x4 O[T][2][8];
#pragma unroll
  for (int t = 0; t < T; ++t) {
    m[t] = -INFINITY;
    sum[t] = 0.f;
#pragma unroll
    for (int hh = 0; hh < 2; ++hh)
#pragma unroll
      for (int i = 0; i < 8; ++i) O[t][hh][i] = (f32x4){0.f, 0.f, 0.f, 0.f};
  }
  // bit b: the wave takes block b, which some query may see; and of these the ones that all see whole
  uint32_t rest = 0u, whole;
  {
    const uint32_t some = (uint32_t)__ballot(lane < RB && lds.live[min(lane, BLOCKS - 1)] != 0u) | (~0u << RB);
    whole = (uint32_t)__ballot(lane < RB && lds.whole[min(lane, BLOCKS - 1)] != 0u);
    for (int b = b_first; b < n_blocks; b += step) rest |= some & (1u << b);
  }
  // probabilities of block b for the scores S, rounded; the accumulators follow a maximum that has moved
  const auto softmax = [&](int b, f32x4 (&S)[T][2], bf16x8 (&pb)[T]) __attribute__((always_inline)) {
    const bool ring = b < RB;
    float top[T];
    bool move = false;
    if (!(whole >> b & 1u)) {
      const int at = (ring ? b * KB : W_MAX + (b - RB) * KB) + 4 * g4;
      i32x4 place[2];
      place[0] = *reinterpret_cast<const i32x4*>(&lds.kp[at]);
      place[1] = *reinterpret_cast<const i32x4*>(&lds.kp[at + 16]);
#pragma unroll
      for (int t = 0; t < T; ++t) {
        const int floor = lds.kp[W_MAX + node[t]] - W;
        const uint32_t bits = ring ? ~0u : (uint32_t)(lds.mask[node[t]] >> ((b - RB) * KB)) >> (4 * g4);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const bool ok = place[e >> 2][e & 3] > floor && (bits >> (16 * (e >> 2) + (e & 3)) & 1u);
          S[t][e >> 2][e & 3] = ok ? S[t][e >> 2][e & 3] : -INFINITY;
        }
      }
    }
#pragma unroll
    for (int t = 0; t < T; ++t) {   // the lane's own keys tell whether the maximum moves
      top[t] = max3(max3(S[t][0][0], S[t][0][1], S[t][0][2]), max3(S[t][0][3], S[t][1][0], S[t][1][1]),
                    max3(S[t][1][2], S[t][1][3], -INFINITY)) * sl2;
      move |= top[t] > m[t] + SLACK;
    }
    if (__any(move)) {
#pragma unroll
      for (int t = 0; t < T; ++t) {
        const float high = max_pair32(max_pair16(top[t]));
        const float to = high > m[t] + SLACK ? high : m[t];
        const float alpha = to == -INFINITY ? 1.f : exp2_fast(m[t] - to);
        m[t] = to;
        sum[t] *= alpha;
#pragma unroll
        for (int hh = 0; hh < 2; ++hh)
#pragma unroll
          for (int i = 0; i < 8; ++i) O[t][hh][i] *= alpha;
      }
    }
#pragma unroll
    for (int t = 0; t < T; ++t) {
      const float base = m[t] == -INFINITY ? 0.f : m[t];
      u32x4 w;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float p0 = exp2_fast(__builtin_fmaf(S[t][i >> 1][2 * (i & 1)], sl2, -base));
        const float p1 = exp2_fast(__builtin_fmaf(S[t][i >> 1][2 * (i & 1) + 1], sl2, -base));
        w[i] = pack_bf16x2(p0, p1);
        float q0, q1;
        unpack2(w[i], q0, q1);   // the weights as rounded: what dominates a row keeps no rounding
        sum[t] += q0 + q1;
      }
      pb[t] = as_bf16x8(w);
    }
  };
  // O^T += V^T . P^T for dims 128 hh + 8 c .. + 7 of the lane's keys 16 (s / 4) + 4 g4 + s % 4
  const auto add_values = [&](int hh, const u32x4 (&v)[8], const bf16x8 (&pb)[T]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      u32x4 w;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        w[e] = __builtin_amdgcn_perm(v[2 * e + 1][i >> 1], v[2 * e][i >> 1], i & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
      for (int t = 0; t < T; ++t)
        O[t][hh][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(w), pb[t], O[t][hh][i], 0, 0, 0);
    }
  };

  if constexpr (!STAGED) {
    // keys and values straight from memory to the operand registers: a block's values are loaded before its scores, the next
    // block's keys after them
    u32x4 kr[2][D / 32], vr[2][8];
    const auto load_keys = [&](int b) __attribute__((always_inline)) {
      const bool ring = b < RB;
      const uint16_t* base = ring ? ro.ring_k + b * (KB * D) : ro.k + (int64_t)(b - RB) * KB * p.nk_sl;
      const uint32_t st = ring ? D : (uint32_t)p.nk_sl, live = live_of(b);
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        const uint32_t off = 2 * (seen_row(live, 16 * kt + c) * st + 8 * g4);
#pragma unroll
        for (int ks = 0; ks < D / 32; ++ks) kr[kt][ks] = load16_at(base + 32 * ks, off);
      }
    };
    if (rest) load_keys(__builtin_ctz(rest));
    while (rest) {
      const int b = __builtin_ctz(rest);
      const bool ring = b < RB;
      {
        const uint16_t* base = ring ? ro.ring_v + b * (KB * D) : ro.v + (int64_t)(b - RB) * KB * p.nv_sl;
        const uint32_t st = ring ? D : (uint32_t)p.nv_sl, live = live_of(b);
#pragma unroll
        for (int s = 0; s < 8; ++s) {
          const uint32_t off = 2 * (seen_row(live, 16 * (s >> 2) + 4 * g4 + (s & 3)) * st + 8 * c);
          vr[0][s] = load16_at(base, off);
          vr[1][s] = load16_at(base + 128, off);
        }
      }
      __builtin_amdgcn_sched_barrier(0);   // the loads are issued here, before the scores wait for the keys
      f32x4 S[T][2];
#pragma unroll
      for (int t = 0; t < T; ++t) S[t][0] = S[t][1] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < D / 32; ++ks)
#pragma unroll
        for (int t = 0; t < T; ++t) {
          const bf16x8 qf = as_bf16x8(lds.q[ks][lane]);
          S[t][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(kr[0][ks]), qf, S[t][0], 0, 0, 0);
          S[t][1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(kr[1][ks]), qf, S[t][1], 0, 0, 0);
        }
      rest &= rest - 1;
      if (rest) load_keys(__builtin_ctz(rest));
      __builtin_amdgcn_sched_barrier(0);
      bf16x8 pb[T];
      softmax(b, S, pb);
      add_values(0, vr[0], pb);
      add_values(1, vr[1], pb);
    }
  } else {
    // every wave needs every block: blocks pass through LDS, the next one on its way while one is at work
    constexpr int K_AHEAD = T == 1 ? 4 : 2, V_AHEAD = 5;   // pairs of reads
    int stage = 0, b = -1;
    if (tree_first) b = RB, rest &= ~(1u << RB);
    else if (rest) b = __builtin_ctz(rest), rest &= rest - 1, fetch(b, 0, whole >> b & 1u);
    while (b >= 0) {
      asm volatile("" ::: "memory");                      // the block before has been read
      __builtin_amdgcn_s_waitcnt(0x0f70);                 // vmcnt(0): the block has landed
      __builtin_amdgcn_s_barrier();                       // for every wave; and the block before is read no more
      asm volatile("" ::: "memory");
      const int next = rest ? __builtin_ctz(rest) : -1;
      rest &= rest - 1;
      if (next >= 0) fetch(next, stage ^ 1, whole >> next & 1u);
      if (tiles > 0) {
        const KeyStage& ks_ = lds.stage[stage];
        const int c_here = lane_per_site(c);   // the addresses are made here rather than kept over the loop
        // of two workgroups on a SIMD, the one at its products goes first (128 x 64 nodes 114 -> 109 us)
        __builtin_amdgcn_s_setprio(1);
        f32x4 S[T][2];
#pragma unroll
        for (int t = 0; t < T; ++t) S[t][0] = S[t][1] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < D / 32; ++ks) {
          // pieces 4 ks + g4 and 16 more share an address: the permutation takes the low 4 bits
          const uint16_t* const at = &ks_.k[c][8 * ((4 * (ks & 3) + g4) ^ c_here) + 128 * (ks >> 2)];
          const bf16x8 k0 = as_bf16x8(load16(at)), k1 = as_bf16x8(load16(at + 16 * D));
#pragma unroll
          for (int t = 0; t < T; ++t) {
            S[t][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k0, qr[t][ks], S[t][0], 0, 0, 0);
            S[t][1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k1, qr[t][ks], S[t][1], 0, 0, 0);
          }
        }
        // reads of the operands run ahead of the products
        __builtin_amdgcn_sched_group_barrier(0x100, 2 * K_AHEAD, 0);
#pragma unroll
        for (int i = 0; i < D / 32 - K_AHEAD; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x008, 2 * T, 0);
          __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, 2 * K_AHEAD * T, 0);
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_setprio(0);
        bf16x8 pb[T];
        softmax(b, S, pb);
        __builtin_amdgcn_s_setprio(1);
        // value operands by transpose reads: lane (g4, c) addresses key 4 g4 + c / 4, and of product i's dims 4 at 128 hh +
        // 8 (4 q + i / 2) + 4 (i + q) % 2, q = c % 4; the products of two neighbours i read both halves of a piece
        const int lane_here = lane_per_site(lane);
        const int row = lane_here >> 2, q = lane_here & 3;
        const uint16_t* const v_at = &ks_.v[row][8 * ((4 * q) ^ (row & 15)) + 4 * (q & 1)];
        const uint32_t v_lds = lds_offset(v_at);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint16_t* const at = lds_pointer(v_lds ^ (8 * i));
#pragma unroll
          for (int hh = 0; hh < 2; ++hh) {
            const u32x2 lo = ld_tr4(at + 128 * hh), hi = ld_tr4(at + 128 * hh + 16 * D);
            const bf16x8 vf = as_bf16x8((u32x4){lo[0], lo[1], hi[0], hi[1]});
#pragma unroll
            for (int t = 0; t < T; ++t)
              O[t][hh][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pb[t], O[t][hh][i], 0, 0, 0);
          }
        }
        __builtin_amdgcn_sched_group_barrier(0x100, 2 * V_AHEAD, 1);
#pragma unroll
        for (int i = 0; i < 16 - V_AHEAD; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x008, T, 1);
          __builtin_amdgcn_sched_group_barrier(0x100, 2, 1);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, V_AHEAD * T, 1);
      }
      __builtin_amdgcn_s_setprio(0);
      b = next;
      stage ^= 1;
    }
  }

  // ---- the waves' partial sums meet; outputs ----
  // (rows and addresses are made again here rather than kept over the loop)
  const int lane_end = lane_per_site(lane);
  const int ge = lane_end >> 4, ce = lane_end & 15;
  // lane (ge, ce) of product (hh, i), register r: query ce, dim 128 hh + 32 ge + 8 r + i, or (STAGED) + 8 (i / 2) + 4 ((i +
  // ge) % 2) + r; a lane stores 8 R dims at a time
  constexpr int R = STAGED ? 4 : 8 / KW, TIMES = STAGED ? 2 : 1;
  const auto half_of = [&](int x) { return STAGED ? x : wk * R / 4; };
  const int r0 = STAGED ? 0 : wk * R % 4;
  u32x4 gw[T][TIMES][R];
  const auto load_gates = [&](int t) __attribute__((always_inline)) {
#pragma unroll
    for (int x = 0; x < TIMES; ++x)
      load_gate(p, ro, min(r_lo + 16 * t + ce, M - 1), 128 * half_of(x) + 32 * ge + 8 * r0, gw[t][x]);
  };
  if (p.splits == 1) {
#pragma unroll
    for (int t = 0; t < T; ++t) load_gates(t);
  }
#pragma unroll
  for (int t = 0; t < T; ++t) sum[t] = add_xor32(add_xor16(sum[t]));
  if constexpr (!STAGED) {
#pragma unroll
    for (int t = 0; t < T; ++t)
      if (ge == 0) {
        lds.ml[wave][t][ce][0] = m[t];
        lds.ml[wave][t][ce][1] = sum[t];
      }
    __syncthreads();   // (the queries in LDS are read no more, either)
  }
#pragma unroll
  for (int t = 0; t < T; ++t) {
    const int row = r_lo + 16 * t + ce;
    float top = m[t], total = sum[t];
    if constexpr (!STAGED) {
      top = -INFINITY;
      total = 0.f;
#pragma unroll
      for (int w = 0; w < KW; ++w) top = fmaxf(top, lds.ml[w][t][ce][0]);
      const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int w = 0; w < KW; ++w) total += exp2_fast(lds.ml[w][t][ce][0] - base) * lds.ml[w][t][ce][1];
      const float mine = exp2_fast(m[t] - base);
#pragma unroll
      for (int hh = 0; hh < 2; ++hh)
#pragma unroll
        for (int i = 0; i < 8; ++i) lds.o[wave][8 * hh + i][lane_end] = O[t][hh][i] * mine;
      __syncthreads();
    }
#pragma unroll
    for (int x = 0; x < TIMES; ++x) {
      const int hh = half_of(x);
      float y[8 * R];
      if constexpr (!STAGED) {
#pragma unroll
        for (int e = 0; e < 8 * R; ++e) y[e] = 0.f;
#pragma unroll
        for (int w = 0; w < KW; ++w)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float* src = reinterpret_cast<const float*>(&lds.o[w][8 * hh + i][lane_end]) + r0;
#pragma unroll
            for (int r = 0; r < R; ++r) y[8 * r + i] += src[r];
          }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) y[4 * i + r] = ge & 1 ? O[t][x][i ^ 1][r] : O[t][x][i][r];
      }
      const int d0 = 128 * hh + 32 * ge + 8 * r0;
      if (row >= M) continue;
      if (p.splits == 1) {
        const float inv = 1.0f / total;
#pragma unroll
        for (int e = 0; e < 8 * R; ++e) y[e] *= inv;
        if (all_finite(y)) store_gated(p, ro, row, d0, y, gw[t][x]);
        else atomicOr(&lds.odd[wq * T + t], 1u << ce);
      } else {
        const int64_t at = ((int64_t)pair * p.splits + split) * ((int64_t)G * p.max_nodes) + row;
        float* dst = p.part_o + at * D + d0;
#pragma unroll
        for (int e = 0; e < 8 * R; e += 4) *reinterpret_cast<f32x4*>(dst + e) = (f32x4){y[e], y[e + 1], y[e + 2], y[e + 3]};
        if (hh == 0 && ge == 0 && r0 == 0) {
          p.part_ml[2 * at] = top;
          p.part_ml[2 * at + 1] = total;
        }
      }
    }
  }
  if (p.splits > 1) return;
  // ---- query rows with a result that is not finite: again, over the keys that they see alone ----
  __syncthreads();
  for (int i0 = 2 * wave; i0 < ROWS; i0 += 2 * NW) {   // two rows a wave, of which one may be finite
    const uint32_t odd = __builtin_amdgcn_readfirstlane(lds.odd[i0 >> 4]) >> (i0 & 15) & 3u;
    if (!odd) continue;
    const int row = min(r_wg + i0 + (lane >> 5), M - 1), d0 = 8 * (lane & 31);
    float y[8];
    u32x4 one[1];
    load_gate(p, ro, row, d0, one);
    walk_keys(p, ro, row, d0, y);
    if (odd >> (lane >> 5) & 1u) store_gated(p, ro, row, d0, y, one);
  }
  // ---- the pair's only workgroup writes its committed chain after its reads: 64 x 12 nodes 35.6 us, with a launch for it 34.2 +
  // 4.1; 352 x 1 125.8 and 122.4 + 4.8. (The arguments are loaded again: kept over the loop, they took the scalar registers that
  // its schedule needs.) ----
  const auto* args = (const __attribute__((address_space(4))) TreeAttnParams*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(args));
  const TreeAttnParams& late = *(const TreeAttnParams*)args;
  if (late.write_here) {
    __syncthreads();
    write_chain(late, (int)blockIdx.x / late.hkv, (int)blockIdx.x % late.hkv, 0, 1);
  }
}

// Joins the splits' partial sums: a wave a query row, 4 dims a lane; every split's loads are in flight at once
__global__ __launch_bounds__(256) void tree_attn_join_kernel(const TreeAttnParams p) {
  const int pair = blockIdx.x;
  const int n = pair / p.hkv, h = pair - n * p.hkv;
  const int row = blockIdx.y * 4 + (threadIdx.x >> 6), d0 = 4 * (threadIdx.x & 63);
  const int64_t stride = (int64_t)p.G * p.max_nodes;
  const int64_t first = (int64_t)pair * p.splits * stride + row;
  f32x4 v[SPLITS_MAX];
  float m[SPLITS_MAX], l[SPLITS_MAX];
  if (row >= stride) return;
#pragma unroll
  for (int s = 0; s < SPLITS_MAX; ++s) {
    const int64_t at = first + min(s, p.splits - 1) * stride;   // (a row of no tree: whatever the workspace holds, not used)
    v[s] = *reinterpret_cast<const f32x4*>(p.part_o + at * D + d0);
    m[s] = p.part_ml[2 * at];
    l[s] = p.part_ml[2 * at + 1];
  }
  TreeKeys ro;
  if (!tree_keys(p, n, h, ro) || row >= p.G * ro.len) return;
  const int node = row / p.G, g = row - node * p.G;
  u32x2 gate = {0u, 0u};
  if (ro.gate) gate = *reinterpret_cast<const u32x2*>(ro.gate + node * p.g_sl + g * p.g_sg + d0);
  float top = -INFINITY, total = 0.f;
#pragma unroll
  for (int s = 0; s < SPLITS_MAX; ++s)
    if (s < p.splits) top = fmaxf(top, m[s]);
  const float base = top == -INFINITY ? 0.f : top;
  float y[4] = {};
#pragma unroll
  for (int s = 0; s < SPLITS_MAX; ++s) {
    if (s >= p.splits) continue;
    const float w = exp2_fast(m[s] - base);
    total = __builtin_fmaf(w, l[s], total);
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = __builtin_fmaf(w, v[s][i], y[i]);
  }
  const float inv = 1.0f / total;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] *= inv;
  if (__any(!all_finite(y))) walk_keys(p, ro, row, d0, y);
  if (ro.gate) {
    float gt[4];
    unpack2(gate[0], gt[0], gt[1]);
    unpack2(gate[1], gt[2], gt[3]);
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] *= gate_of(gt[e]);
  }
  store4_bf16(ro.out + node * p.o_sl + g * p.o_sg + d0, y);
}

__global__ __launch_bounds__(256) void tree_ring_write_kernel(const TreeAttnParams p) {
  write_chain(p, blockIdx.x / p.hkv, blockIdx.x % p.hkv, blockIdx.y, gridDim.y);
}

// Query rows of a workgroup. Up to 16 the waves split their keys (352 x 1 node 119 us, against 127 through LDS); beyond, keys
// pass through LDS for 4 waves of one tile, or of two where that fills the chip (256 CUs) and wastes little. 64 x 64 nodes, 16 q
// / 4 kv heads: 55 us with 128 rows, 68 with 64; 20 x 64 36 and 30; 100 x 33 (129 to 192 rows are three workgroups of 64) 84 and
// 67.
inline int rows_of(int64_t pairs, int64_t rows) {
  if (rows <= 64) return rows <= 16 ? 16 : 64;
  return (rows + 63) / 64 == 3 || pairs * ((rows + 127) / 128) < 256 ? 64 : 128;
}

// Workgroups of a row's key blocks: few rows leave the chip short of workgroups, and one CU moves only a few tens of GB/s. 16 x 4
// nodes (64 units): 14.0, 12.5 and 13.4 us with 2, 4 and 8, and a join of 3.9; 30 x 14 (120): 24.7 with 1, as long as 18.0 with 2
// and a join of 6.6; 60 x 14 32.4 with 1, 28.9 and 11.7 with 2.
inline int splits_of(int64_t pairs, int64_t rows) {
  const int per = rows_of(pairs, rows);
  const int64_t units = pairs * ((rows + per - 1) / per);
  return units <= 32 ? SPLITS_MAX : units <= 64 ? 4 : 1;
}

inline size_t part_bytes(int64_t pairs, int64_t rows, int splits) {
  return splits == 1 ? 0 : (size_t)(pairs * splits * rows) * (D + 2) * sizeof(float);
}

}  // namespace
}  // namespace hsg

extern "C" size_t hsg_tree_attention_workspace_bytes(int32_t n_rows, int32_t hkv, int32_t groups, int32_t max_nodes) {
  using namespace hsg;
  if (n_rows <= 0 || hkv <= 0 || groups <= 0 || max_nodes <= 0 || max_nodes > MOST) return 0;
  const int64_t rows = (int64_t)groups * max_nodes;
  const int64_t pairs = (int64_t)n_rows * hkv;
  return part_bytes(pairs, rows, splits_of(pairs, rows));
}

extern "C" int hsg_tree_attention(const void* q, int64_t q_sl, int64_t q_sh, int64_t q_sg, void* ring_k, void* ring_v,
                                  int64_t ring_rows, int32_t window, const void* new_k, int64_t nk_sl, int64_t nk_sh,
                                  const void* new_v, int64_t nv_sl, int64_t nv_sh, const void* gate, int64_t g_sl,
                                  int64_t g_sh, int64_t g_sg, int64_t g_off, const int64_t* ring_pos,
                                  const int64_t* slots, const int64_t* starts, const int64_t* lens,
                                  const int64_t* offsets, const int64_t* commits, const int64_t* masks, int32_t n_rows,
                                  int32_t max_nodes, int32_t hkv, int32_t groups, int32_t head_dim, float scale, void* out,
                                  int64_t o_sl, int64_t o_sh, int64_t o_sg, void* workspace, size_t workspace_bytes,
                                  void* stream) {
  using namespace hsg;
  if (n_rows < 0 || hkv <= 0 || groups <= 0 || ring_rows <= 0) return HSG_ERR_ARG;
  if (head_dim != D || window <= 0 || window > W_MAX || window % KB != 0 || max_nodes <= 0 || max_nodes > MOST)
    return HSG_ERR_SHAPE;
  if (!isfinite(scale)) return HSG_ERR_ARG;
  if (n_rows == 0) return HSG_OK;
  if (!q || !ring_k || !ring_v || !new_k || !new_v || !ring_pos || !slots || !starts || !lens || !offsets || !masks || !out)
    return HSG_ERR_ARG;
  // a row's keys are addressed by 32-bit byte offsets
  if (nk_sl < 0 || nv_sl < 0 || nk_sl >= (1 << 24) || nv_sl >= (1 << 24)) return HSG_ERR_SHAPE;
  const int64_t strides[] = {q_sl, q_sh, q_sg, nk_sl, nk_sh, nv_sl, nv_sh, o_sl, o_sh, o_sg};
  for (int64_t st : strides)
    if (st % 8) return HSG_ERR_ALIGN;
  if (gate && (g_sl % 8 || g_sh % 8 || g_sg % 8 || g_off % 8 || !aligned(gate, 16))) return HSG_ERR_ALIGN;
  if (!aligned(q, 16) || !aligned(ring_k, 16) || !aligned(ring_v, 16) || !aligned(new_k, 16) || !aligned(new_v, 16) ||
      !aligned(out, 16) || !aligned(workspace, 16))
    return HSG_ERR_ALIGN;
  const int64_t rows = (int64_t)groups * max_nodes;
  const int64_t pairs = (int64_t)n_rows * hkv;
  const int per_wg = rows_of(pairs, rows);
  TreeAttnParams p{};
  p.q = static_cast<const uint16_t*>(q); p.q_sl = q_sl; p.q_sh = q_sh; p.q_sg = q_sg;
  p.ring_k = static_cast<uint16_t*>(ring_k); p.ring_v = static_cast<uint16_t*>(ring_v);
  p.ring_rows = ring_rows; p.W = window;
  p.new_k = static_cast<const uint16_t*>(new_k); p.nk_sl = nk_sl; p.nk_sh = nk_sh;
  p.new_v = static_cast<const uint16_t*>(new_v); p.nv_sl = nv_sl; p.nv_sh = nv_sh;
  p.gate = static_cast<const uint16_t*>(gate); p.g_sl = g_sl; p.g_sh = g_sh; p.g_sg = g_sg; p.g_off = g_off;
  p.ring_pos = ring_pos; p.slots = slots; p.starts = starts; p.lens = lens; p.offsets = offsets;
  p.commits = commits; p.masks = masks;
  p.max_nodes = max_nodes; p.hkv = hkv; p.G = groups; p.scale = scale;
  if (pairs >= (1 << 24) || rows >= (1 << 20)) return HSG_ERR_SHAPE;
  p.pairs = (int)pairs;
  p.qblocks = (int)((rows + per_wg - 1) / per_wg);
  p.splits = splits_of(pairs, rows);
  if (!workspace || workspace_bytes < part_bytes(pairs, rows, p.splits)) p.splits = 1;
  p.write_here = commits && p.qblocks == 1 && p.splits == 1;
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = p.splits > 1 ? p.part_o + pairs * p.splits * rows * D : nullptr;
  p.out = static_cast<uint16_t*>(out); p.o_sl = o_sl; p.o_sh = o_sh; p.o_sg = o_sg;
  const int64_t blocks = (pairs + 7) / 8 * 8 * p.qblocks * p.splits;
  if (blocks >= (1 << 24)) return HSG_ERR_SHAPE;   // a launch holds less than 2^32 threads
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(64 * NW), 0, st, p); };
  if (per_wg == 16) launch(tree_attn_kernel<1, false>);
  else if (per_wg == 64) launch(tree_attn_kernel<1, true>);
  else launch(tree_attn_kernel<2, true>);
  if (p.splits > 1)
    hipLaunchKernelGGL(tree_attn_join_kernel, dim3((unsigned)pairs, (unsigned)((rows + 3) / 4)), dim3(256), 0, st, p);
  if (commits && !p.write_here)
    hipLaunchKernelGGL(tree_ring_write_kernel, dim3((unsigned)pairs, (unsigned)((max_nodes + 15) / 16)), dim3(256), 0, st, p);
  return launch_status();
}
