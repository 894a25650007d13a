// The gated-delta rule along every path of a drafted tree, from the slot's recurrent state, which does not move but for the
// committed chain; with the layer's gated RMSNorm.
//
// Along a path S <- e^g S + k u^T with u = beta (v - e^g S^T k), o = S^T q (q, k of unit length, q times scale). Unrolled over
// a tree, with G_i the sum of g down the path to node i, only the state before the tree, S0, is needed:
//   R_i = beta_i (v_i - e^G_i S0^T k_i),       A_ij = beta_i e^(G_i - G_j) (k_i . k_j)   j a proper ancestor of i
//   (I + A) U = R                               (unit lower triangular: parents come first)
//   o_i = e^G_i S0^T q_i + sum_j P_ij u_j,     P_ij = e^(G_i - G_j) (q_i . k_j)           j an ancestor of i, or i
//   S1  = e^G_c S0 + sum over the chain of e^(G_c - G_j) k_j u_j^T                         c the last committed node
// A tree is a chunk of the delta rule's chunk form whose causal mask is the ancestors' mask: the state is read once for all
// branches, and no branch needs a state of its own.
//
// A workgroup of 4 waves takes one (row, value head): wave w columns 32 w .. 32 w + 31 of V, lane (g, c) = (lane / 16,
// lane % 16) the pairs 32 w + 2 c, + 1, so that its accumulators' columns are neighbours. S0 (64 KB in fp32) goes straight
// from memory to registers, a lane holding rows 32 s + 8 g + i: the B operand of the products with k and q as it lies.
// k and q are exact in bf16 and their lengths divide the products afterwards; a state value is split into three bf16 parts
// (two from fp16) that hold all its digits, so S0^T k is as exact as fp32 products. k.k and q.k are bf16 products, exact up
// to fp32 sums. U and the accumulators share the MFMA layout (a lane's 4 registers are 4 consecutive nodes of one column),
// so U never leaves the registers; A, P and the inverses of A's diagonal blocks go through LDS as fp32.
// G is summed and its differences taken in fp64: a steep decay early on a path must not cost the digits of the later ones.
//
// A masked pair has a coefficient of 0, which would carry a NaN or an infinity of one branch to all others: where a result
// is not finite, the workgroup computes its row again by walking each node's own ancestors (walk_row).
#include <math.h>

#include <type_traits>

#include "hsg_common.h"

namespace hsg {
namespace {

constexpr int KD = 128;
constexpr int NW = 4;

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(2))) float f32x2;

struct TreeStepParams {
  const uint16_t* qkv; int64_t qkv_stride; int q_off, k_off, v_off;
  const uint16_t* a; const uint16_t* b; int64_t ab_stride;
  const uint16_t* A_log; const uint16_t* dt_bias;
  void* state; int64_t state_rows;
  const int64_t* slots; const int64_t* lens; const int64_t* offsets; const int64_t* commits; const int64_t* masks;
  int max_nodes, H, HV;
  float scale;
  const uint16_t* z; int64_t z_stride; const uint16_t* norm_w; float eps;
  uint16_t* out;
};

template <int NT>
struct TreeStepLds {
  static constexpr int N = 16 * NT;
  static constexpr int PITCH = N + 4;
  union {
    struct {
      float A[N][PITCH];   // -A_ij
      float P[N][PITCH];
    };
    float U[N][KD];        // walk_row
  };
  float T[NT][16][20];     // (I + A_bb)^-1 of the diagonal blocks
  double G[N];
  uint64_t mask[N];        // ancestors and itself, within the row
  float g[N], beta[N], kinv[N], qinv[N];
  float part[N][NW];
  int odd[NW];             // a wave saw a value that is not finite
  __device__ TreeStepLds() {}
};

// One (row, value head)
struct TreeRow {
  const uint16_t* q; const uint16_t* k; const uint16_t* v;   // of the first node
  const uint16_t* z; uint16_t* out;
  int64_t state_at;                                          // element offset of S0
  int len, done;
};

__device__ __forceinline__ bf16x8 load_bf16x8(const uint16_t* p) {
  return __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(p));
}

// the upper halves of two fp32 words as a bf16 pair (a in the low half)
__device__ __forceinline__ uint32_t upper_pair(float a, float b) {
  return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}
__device__ __forceinline__ float upper(float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); }

// Eight fp32 values as PARTS bf16 operands whose sum they are: 8 digits each, cut off rather than rounded
template <int PARTS>
__device__ __forceinline__ void split8(const float (&x)[8], bf16x8 (&out)[PARTS]) {
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = x[i];
#pragma unroll
  for (int p = 0; p < PARTS; ++p) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = upper_pair(r[2 * i], r[2 * i + 1]);
    out[p] = __builtin_bit_cast(bf16x8, w);
    if (p + 1 < PARTS) {
#pragma unroll
      for (int i = 0; i < 8; ++i) r[i] -= upper(r[i]);
    }
  }
}

__device__ __forceinline__ float state_at(const void* state, bool half, int64_t at) {
  return half ? h2f(static_cast<const uint16_t*>(state)[at]) : static_cast<const float*>(state)[at];
}

__device__ __forceinline__ float log_decay(float a, float a_log, float dt_bias) {
  const float x = a + dt_bias;
  return -expf(a_log) * (x > 20.0f ? x : log1pf(expf(x)));
}

// The row by its definition, node by node over each one's own ancestors: nothing is multiplied by a masked 0, and decays
// are sums over the nodes between rather than differences. Thread t < 128 takes column t.
template <int NT, bool HALF, bool GATED>
__device__ __forceinline__ void walk_row(const TreeStepParams& p, const TreeRow& ro, TreeStepLds<NT>& lds) {
  const int col = threadIdx.x & (KD - 1);
  const bool mine = threadIdx.x < KD;
  const auto dot = [](const uint16_t* x, const uint16_t* y) {
    float s = 0.f;
#pragma unroll 4
    for (int k = 0; k < KD; ++k) s = __builtin_fmaf(bf2f(x[k]), bf2f(y[k]), s);
    return s;
  };
  const auto between = [&](uint64_t nodes) {
    float s = 0.f;
    for (; nodes; nodes &= nodes - 1) s += lds.g[__builtin_ctzll(nodes)];
    return expf(s);
  };
  __syncthreads();   // P, which U lies over, is read no more
  for (int i = 0; i < ro.len; ++i) {
    const uint64_t path = lds.mask[i];
    const uint16_t* ki = ro.k + i * p.qkv_stride;
    const uint16_t* qi = ro.q + i * p.qkv_stride;
    float o = 0.f;
    if (mine) {
      float ks = 0.f, qs = 0.f;
#pragma unroll 4
      for (int k = 0; k < KD; ++k) {
        const float s = state_at(p.state, HALF, ro.state_at + (int64_t)k * KD + col);
        ks = __builtin_fmaf(bf2f(ki[k]), s, ks);
        qs = __builtin_fmaf(bf2f(qi[k]), s, qs);
      }
      const float e = between(path);
      float read = e * lds.kinv[i] * ks;
      o = e * lds.qinv[i] * qs;
      for (uint64_t up = path & ~(1ull << i); up; up &= up - 1) {
        const int j = __builtin_ctzll(up);
        const uint16_t* kj = ro.k + j * p.qkv_stride;
        const float d = between(path & ~lds.mask[j]) * lds.kinv[j];
        read += d * lds.kinv[i] * dot(ki, kj) * lds.U[j][col];
        o += d * lds.qinv[i] * dot(qi, kj) * lds.U[j][col];
      }
      const float u = lds.beta[i] * (bf2f(ro.v[i * p.qkv_stride + col]) - read);
      lds.U[i][col] = u;
      o += lds.qinv[i] * lds.kinv[i] * dot(qi, ki) * u;
    }
    if constexpr (GATED) {
      const float ss = wave_sum(o * o);
      if (mine && (threadIdx.x & 63) == 0) lds.part[i][threadIdx.x >> 6] = ss;
      __syncthreads();
      if (mine) {
        const float r = rsqrtf((lds.part[i][0] + lds.part[i][1]) * (1.0f / KD) + p.eps);
        o *= r * bf2f(p.norm_w[col]) * siluf_(bf2f(ro.z[i * p.z_stride + col]));
      }
    }
    if (mine) ro.out[(int64_t)i * p.HV * KD + col] = f2bf(o);
  }
  if (ro.done > 0) {
    const int c = ro.done - 1;
    __syncthreads();   // the sums of squares are read no more
    for (int j = threadIdx.x; j < ro.done; j += 64 * NW)
      lds.part[j][0] = between(lds.mask[c] & ~lds.mask[j]) * lds.kinv[j];
    __syncthreads();
    if (mine) {
      const float e = between(lds.mask[c]);
      for (int k = 0; k < KD; ++k) {
        const int64_t at = ro.state_at + (int64_t)k * KD + col;
        float s = e * state_at(p.state, HALF, at);
        for (int j = 0; j < ro.done; ++j)
          s = __builtin_fmaf(lds.part[j][0] * bf2f(ro.k[j * p.qkv_stride + k]), lds.U[j][col], s);
        if constexpr (HALF) static_cast<uint16_t*>(p.state)[at] = f2h(s);
        else static_cast<float*>(p.state)[at] = s;
      }
    }
  }
}

template <int NT, bool HALF, bool GATED>
__global__ __launch_bounds__(64 * NW) void gdn_tree_kernel(const TreeStepParams p) {
  constexpr int PARTS = HALF ? 2 : 3;
  __shared__ TreeStepLds<NT> lds;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g4 = lane >> 4, c = lane & 15;
  const int n = blockIdx.x / p.HV, hv = blockIdx.x - n * p.HV;
  const int64_t slot = p.slots[n], len64 = p.lens[n], off = p.offsets[n];
  const int64_t done64 = p.commits ? p.commits[n] : 0;
  if ((slot < 0) | (slot >= p.state_rows) | (len64 <= 0) | (len64 > p.max_nodes)) return;
  const int len = (int)len64;
  const int tiles = (len + 15) >> 4;
  const int h = hv / (p.HV / p.H);
  TreeRow ro;
  ro.q = p.qkv + off * p.qkv_stride + p.q_off + h * KD;
  ro.k = p.qkv + off * p.qkv_stride + p.k_off + h * KD;
  ro.v = p.qkv + off * p.qkv_stride + p.v_off + hv * KD;
  ro.z = GATED ? p.z + off * p.z_stride + hv * KD : nullptr;
  ro.out = p.out + off * ((int64_t)p.HV * KD) + hv * KD;
  ro.state_at = (slot * p.HV + hv) * (int64_t)(KD * KD);
  ro.len = len;
  ro.done = (int)(done64 < 0 ? 0 : done64 > len ? len : done64);
  const int col = 32 * wave + 2 * c;   // the lane's columns col, col + 1

  // ---- S0: rows 32 s + 8 g4 + i ----
  float s0[4][2][8];
#pragma unroll
  for (int s = 0; s < 4; ++s)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t at = ro.state_at + (32 * s + 8 * g4 + i) * KD + col;
      if constexpr (HALF) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(p.state) + at);
        s0[s][0][i] = h2f((uint16_t)w);
        s0[s][1][i] = h2f((uint16_t)(w >> 16));
      } else {
        const f32x2 w = *reinterpret_cast<const f32x2*>(static_cast<const float*>(p.state) + at);
        s0[s][0][i] = w[0];
        s0[s][1][i] = w[1];
      }
    }

  // ---- a node's scalars: lane = node ----
  if (wave == 0) {
    const int i = min(lane, len - 1);
    const bool valid = lane < len;
    const uint64_t self = 1ull << lane;
    uint64_t mask = (uint64_t)p.masks[off + i];
    mask = valid ? (mask & (self - 1)) | self : self;
    const float a = bf2f(p.a[(off + i) * p.ab_stride + hv]), b = bf2f(p.b[(off + i) * p.ab_stride + hv]);
    const float g = valid ? log_decay(a, bf2f(p.A_log[hv]), bf2f(p.dt_bias[hv])) : 0.f;
    // the sum down the path, by pointer doubling
    double sum = g;
    const uint64_t above = mask & ~self;
    int up = above ? 63 - __clzll((long long)above) : -1;
#pragma unroll
    for (int s = 0; s < 6; ++s) {
      const int at = up < 0 ? lane : up;
      const double more = __shfl(sum, at, 64);
      const int next = __shfl(up, at, 64);
      sum += up < 0 ? 0.0 : more;
      up = up < 0 ? -1 : next;
    }
    if (lane < 16 * NT) {
      lds.mask[lane] = mask;
      lds.g[lane] = g;
      lds.G[lane] = sum;
      lds.beta[lane] = valid ? sigmoid_f32(b) : 0.f;
    }
  }
  // ---- the lengths of k and q: wave = tile ----
  const auto row_of = [&](int t) { return (int64_t)min(16 * t + c, len - 1) * p.qkv_stride; };   // an operand's row
  if (wave < NT) {
    float kk = 0.f, qq = 0.f;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      float x[8];
      load8_bf16(ro.k + row_of(wave) + 32 * s + 8 * g4, x);
#pragma unroll
      for (int i = 0; i < 8; ++i) kk = __builtin_fmaf(x[i], x[i], kk);
      load8_bf16(ro.q + row_of(wave) + 32 * s + 8 * g4, x);
#pragma unroll
      for (int i = 0; i < 8; ++i) qq = __builtin_fmaf(x[i], x[i], qq);
    }
    kk = add_xor32(add_xor16(kk));
    qq = add_xor32(add_xor16(qq));
    if (g4 == 0) {
      lds.kinv[16 * wave + c] = 1.0f / sqrtf(kk + 1e-6f);
      lds.qinv[16 * wave + c] = p.scale / sqrtf(qq + 1e-6f);
    }
  }
  lds_barrier();

  // ---- -A and P: (block pair, which of the two) dealt over the waves ----
  for (int it = wave; it < NT * (NT + 1); it += NW) {
    const int pair = it >> 1;
    const bool is_q = it & 1;
    const int bi = pair < 1 ? 0 : pair < 3 ? 1 : pair < 6 ? 2 : 3;
    const int bj = pair - bi * (bi + 1) / 2;
    if (bi >= tiles) break;
    const uint16_t* x = (is_q ? ro.q : ro.k) + row_of(bi) + 8 * g4;
    const uint16_t* y = ro.k + row_of(bj) + 8 * g4;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < 4; ++s)
      acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(load_bf16x8(x + 32 * s), load_bf16x8(y + 32 * s), acc, 0, 0, 0);
    const int j = 16 * bj + c;
    const double Gj = lds.G[j];
    const float kj = lds.kinv[j];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = 16 * bi + 4 * g4 + r;
      const bool on = (lds.mask[i] >> j & 1) && i < len && (is_q || i != j);
      const float d = expf((float)(lds.G[i] - Gj)) * kj * acc[r];
      if (is_q) lds.P[i][j] = on ? lds.qinv[i] * d : 0.f;
      else lds.A[i][j] = on ? -lds.beta[i] * lds.kinv[i] * d : 0.f;
    }
  }
  lds_barrier();

  // ---- the inverses of the diagonal blocks: wave = block, lane c = column ----
  if (wave < tiles) {
    float t[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float acc = i == c ? 1.f : 0.f;
#pragma unroll
      for (int m = 0; m < i; ++m) acc = __builtin_fmaf(lds.A[16 * wave + i][16 * wave + m], t[m], acc);
      t[i] = acc;
    }
    if (g4 == 0) {
#pragma unroll
      for (int i = 0; i < 16; ++i) lds.T[wave][i][c] = t[i];
    }
  }

  // ---- S0^T k and S0^T q of every node, the wave's columns ----
  f32x4 u[NT][2], o[NT][2];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int j = 0; j < 2; ++j) u[t][j] = o[t][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    bf16x8 part[2][PARTS];
#pragma unroll
    for (int j = 0; j < 2; ++j) split8<PARTS>(s0[s][j], part[j]);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if (t >= tiles) break;
      const bf16x8 kf = load_bf16x8(ro.k + row_of(t) + 32 * s + 8 * g4);
      const bf16x8 qf = load_bf16x8(ro.q + row_of(t) + 32 * s + 8 * g4);
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int w = PARTS - 1; w >= 0; --w) {
          u[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, part[j][w], u[t][j], 0, 0, 0);
          o[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(qf, part[j][w], o[t][j], 0, 0, 0);
        }
    }
  }
  // ---- R, and the state's part of the outputs ----
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    if (t >= tiles) break;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = 16 * t + 4 * g4 + r;
      const uint32_t vw = *reinterpret_cast<const uint32_t*>(ro.v + (int64_t)min(i, len - 1) * p.qkv_stride + col);
      float v[2];
      unpack2(vw, v[0], v[1]);
      const float e = expf((float)lds.G[i]);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        u[t][j][r] = i < len ? lds.beta[i] * (v[j] - e * lds.kinv[i] * u[t][j][r]) : 0.f;
        o[t][j][r] *= e * lds.qinv[i];
      }
    }
  }
  lds_barrier();

  // ---- U, block by block, and the outputs ----
#pragma unroll
  for (int b = 0; b < NT; ++b) {
    if (b >= tiles) break;
#pragma unroll
    for (int t = 0; t < b; ++t) {
      const f32x4 a = *reinterpret_cast<const f32x4*>(&lds.A[16 * b + c][16 * t + 4 * g4]);
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int j = 0; j < 2; ++j) u[b][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[r], u[t][j][r], u[b][j], 0, 0, 0);
    }
    const f32x4 a = *reinterpret_cast<const f32x4*>(&lds.T[b][c][4 * g4]);
    f32x4 x[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int j = 0; j < 2; ++j) x[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[r], u[b][j][r], x[j], 0, 0, 0);
    u[b][0] = x[0];
    u[b][1] = x[1];
#pragma unroll
    for (int t = 0; t <= b; ++t) {
      const f32x4 q = *reinterpret_cast<const f32x4*>(&lds.P[16 * b + c][16 * t + 4 * g4]);
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int j = 0; j < 2; ++j) o[b][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(q[r], u[t][j][r], o[b][j], 0, 0, 0);
    }
  }

  // ---- sums of squares of the outputs; is every value finite ----
  float odd = 0.f;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    if (t >= tiles) break;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = 16 * t + 4 * g4 + r;
      const float o0 = o[t][0][r], o1 = o[t][1][r];
      if (i < len) odd += (u[t][0][r] + u[t][1][r]) * 0.f + (o0 + o1) * 0.f;
      if constexpr (GATED) {
        const float ss = sum16_dpp(o0 * o0 + o1 * o1);
        if (c == 0) lds.part[i][wave] = ss;
      }
    }
  }
  const uint64_t bad = __ballot(!(odd == 0.f));
  if (lane == 0) lds.odd[wave] = bad != 0;
  __syncthreads();
  if (lds.odd[0] | lds.odd[1] | lds.odd[2] | lds.odd[3]) {
    walk_row<NT, HALF, GATED>(p, ro, lds);
    return;
  }

  // ---- gated norm, outputs ----
  float nw[2] = {0.f, 0.f};
  if constexpr (GATED) unpack2(*reinterpret_cast<const uint32_t*>(p.norm_w + col), nw[0], nw[1]);
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    if (t >= tiles) break;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = 16 * t + 4 * g4 + r;
      float y[2] = {o[t][0][r], o[t][1][r]};
      if constexpr (GATED) {
        const f32x4 ss = *reinterpret_cast<const f32x4*>(lds.part[i]);
        const float rs = rsqrtf(((ss[0] + ss[1]) + (ss[2] + ss[3])) * (1.0f / KD) + p.eps);
        float z[2];
        unpack2(*reinterpret_cast<const uint32_t*>(ro.z + (int64_t)min(i, len - 1) * p.z_stride + col), z[0], z[1]);
#pragma unroll
        for (int j = 0; j < 2; ++j) y[j] *= rs * nw[j] * siluf_(z[j]);
      }
      if (i < len) *reinterpret_cast<uint32_t*>(ro.out + (int64_t)i * p.HV * KD + col) = pack_bf16x2(y[0], y[1]);
    }
  }

  // ---- the committed chain moves the state ----
  if (ro.done > 0) {
    const double Gc = lds.G[ro.done - 1];
    const float ec = expf((float)Gc);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = 16 * t + 4 * g4 + r;
        const float d = i < ro.done ? expf((float)(Gc - lds.G[i])) * lds.kinv[i] : 0.f;
#pragma unroll
        for (int j = 0; j < 2; ++j) u[t][j][r] *= d;
      }
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        // accumulator row 4 g4 + r is state row 32 s + 8 g4 + 4 hh + r
        f32x4 acc[2];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[j][r] = ec * s0[s][j][4 * hh + r];
        const uint16_t* kcol = ro.k + 32 * s + 8 * (c >> 2) + 4 * hh + (c & 3);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          if (16 * t >= ro.done) break;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float kv = bf2f(kcol[(int64_t)min(16 * t + 4 * g4 + r, ro.done - 1) * p.qkv_stride]);
#pragma unroll
            for (int j = 0; j < 2; ++j) acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(kv, u[t][j][r], acc[j], 0, 0, 0);
          }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int64_t at = ro.state_at + (32 * s + 8 * g4 + 4 * hh + r) * KD + col;
          if constexpr (HALF)
            *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p.state) + at) =
                (uint32_t)f2h(acc[0][r]) | ((uint32_t)f2h(acc[1][r]) << 16);
          else
            *reinterpret_cast<f32x2*>(static_cast<float*>(p.state) + at) = (f32x2){acc[0][r], acc[1][r]};
        }
      }
  }
}

}  // namespace
}  // namespace hsg

extern "C" int hsg_gdn_tree_step(const void* qkv, int64_t qkv_stride, int32_t q_off, int32_t k_off, int32_t v_off,
                                 const void* a, const void* b, int64_t ab_stride, const void* A_log, const void* dt_bias,
                                 void* state, int32_t state_dtype, int64_t state_rows, const int64_t* slots,
                                 const int64_t* lens, const int64_t* offsets, const int64_t* commits,
                                 const int64_t* masks, int32_t n_rows, int32_t max_nodes, int32_t H, int32_t HV, int32_t K,
                                 int32_t V, float scale, const void* z, int64_t z_stride, const void* norm_w, float eps,
                                 void* out, void* stream) {
  using namespace hsg;
  if (n_rows < 0 || state_rows <= 0 || H <= 0 || HV <= 0 || HV % H) return HSG_ERR_ARG;
  if (state_dtype != HSG_STATE_F32 && state_dtype != HSG_STATE_F16) return HSG_ERR_ARG;
  if (K != KD || V != KD || max_nodes <= 0 || max_nodes > HSG_TREE_MAX_NODES) return HSG_ERR_SHAPE;
  if (n_rows == 0) return HSG_OK;
  if (!qkv || !a || !b || !A_log || !dt_bias || !state || !slots || !lens || !offsets || !masks || !out ||
      (z && !norm_w))
    return HSG_ERR_ARG;
  if (q_off < 0 || k_off < 0 || v_off < 0 || ab_stride < HV || (z && z_stride < (int64_t)HV * KD)) return HSG_ERR_ARG;
  if (qkv_stride % 8 || q_off % 8 || k_off % 8 || v_off % 8 || !aligned(qkv, 16) || !aligned(state, 16) ||
      !aligned(out, 4) || (z && (z_stride % 2 || !aligned(z, 4) || !aligned(norm_w, 4))))
    return HSG_ERR_ALIGN;
  const int64_t blocks = (int64_t)n_rows * HV;
  if (blocks >= (1 << 24)) return HSG_ERR_SHAPE;   // a launch holds less than 2^32 threads
  TreeStepParams p{};
  p.qkv = static_cast<const uint16_t*>(qkv); p.qkv_stride = qkv_stride; p.q_off = q_off; p.k_off = k_off; p.v_off = v_off;
  p.a = static_cast<const uint16_t*>(a); p.b = static_cast<const uint16_t*>(b); p.ab_stride = ab_stride;
  p.A_log = static_cast<const uint16_t*>(A_log); p.dt_bias = static_cast<const uint16_t*>(dt_bias);
  p.state = state; p.state_rows = state_rows;
  p.slots = slots; p.lens = lens; p.offsets = offsets; p.commits = commits; p.masks = masks;
  p.max_nodes = max_nodes; p.H = H; p.HV = HV; p.scale = scale;
  p.z = static_cast<const uint16_t*>(z); p.z_stride = z_stride; p.norm_w = static_cast<const uint16_t*>(norm_w); p.eps = eps;
  p.out = static_cast<uint16_t*>(out);
  const auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(64 * NW), 0, reinterpret_cast<hipStream_t>(stream), p);
  };
  const auto by_type = [&](auto nt) {
    constexpr int NT = decltype(nt)::value;
    if (state_dtype == HSG_STATE_F16) z ? launch(gdn_tree_kernel<NT, true, true>) : launch(gdn_tree_kernel<NT, true, false>);
    else z ? launch(gdn_tree_kernel<NT, false, true>) : launch(gdn_tree_kernel<NT, false, false>);
  };
  if (max_nodes <= 16) by_type(std::integral_constant<int, 1>{});
  else if (max_nodes <= 32) by_type(std::integral_constant<int, 2>{});
  else by_type(std::integral_constant<int, 4>{});
  return launch_status();
}
