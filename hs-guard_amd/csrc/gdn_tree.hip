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
// so U never leaves the registers; A, P and the inverses of A's diagonal blocks go through LDS as fp32. A committed state is
// as exact as the step-by-step fp32 recurrence leaves it, also where a path's keys resemble one another (substitute below).
// G is summed and its differences taken in fp64: a steep decay early on a path must not cost the digits of the later ones.
//
// Bound by reading the state where trees are small (352 x 1 node, 16 value heads, fp32: 59 us, 6.4 TB/s; 67 without
// nontemporal loads), by the issue of a CU's two workgroups where they are large: 128 x 64 nodes with commits 91 us for 380
// MB. A workgroup then lives 20 us, 6 of them until its loads are there, 2 in the coefficients, 2.7 in the state's products,
// 1.9 in U, 2.2 in the commit; its products alone are 4.7. LDS reads ahead of the products and priorities of the waves
// changed nothing; 8 waves of 16 columns spilled (a third slower). Over an fp16 state a wave's 32 columns are half a line,
// which nontemporal accesses move twice: 96 x 33 nodes, 32 value heads, 69 us for 331 MB moved where 263 are needed.
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
      f32x4 T[NT][64];     // (I + A_bb)^-1 of the diagonal blocks, as the A operand of a lane
    };
    float U[N][KD];        // walk_row
  };
  uint16_t k[N * KD], q[N * KD];   // row by row, 16-byte pieces at kq_at
  double G[N];                     // the decay down to the node, as a power of 2
  uint64_t mask[N];                // ancestors and itself, within the row
  float g[N], beta[N], eG[N], kinv[N], qinv[N];
  float left[N];                   // e^(G_c - G_i) on the committed chain, else 0
  float part[N][NW];
  int odd[NW];                     // a wave saw a value that is not finite
  __device__ TreeStepLds() {}
};

// Element offset of 16-byte piece pc of row i: the pieces of a row are permuted by its number, so that reads of one piece of
// 16 rows, and transpose reads of 4, spread over the banks
__device__ __forceinline__ int kq_at(int i, int pc) { return i * KD + 8 * (pc ^ (i & 15)); }

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

// LDS transpose read: within each group of 16 lanes, lane 4 q + e receives element e of the 4-value vectors that lanes q, q + 4,
// q + 8 and q + 12 of its group address
typedef __attribute__((ext_vector_type(4))) short s16x4;
__device__ __forceinline__ u32x2 ld_tr4(const uint16_t* p) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p)));
}

// the upper halves of two fp32 words as a bf16 pair (a in the low half)
__device__ __forceinline__ uint32_t upper_pair(float a, float b) {
  return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}
__device__ __forceinline__ float upper(float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); }

// silu to a few fp32 steps (its product is rounded to bf16): 5 instructions against siluf_'s 14, and a lane has up to 32
__device__ __forceinline__ float silu_fast(float x) {
  return x * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * x));
}

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

// Rows of T = (I + A_bb)^-1 from x = -A_bb: row i of T is e_i plus the sum of x_ik (row k of T) over k < i. Lane (g, c) holds
// x's row c and columns 4 g .. 4 g + 3 of T's row c; step K gives row K, settled by then, to the rows below it (x_cK is 0 for
// c <= K), as a broadcast within 16 lanes that the product takes as a modifier. Each row is a sum of what the solve itself
// is a sum of, so nothing grows that has to cancel: chains of 16 to 64 nodes whose keys resemble one another leave their
// state as exact as the step-by-step recurrence does (2e-7 to 7e-7). The product (I + x)(I + x^2)(I + x^4)(I + x^8) does not:
// the powers' entries there are binomials up to 3,400 that cancel to order 1, and the state was off by 1e-5 to 3.5e-4. (15
// dependent steps are also shorter than its three rounds of fp32 products: 128 x 64 nodes 93.5 -> 91.9 us, 96 x 33 71.3 -> 68.4.)
template <int K = 0>
__device__ __forceinline__ void substitute(const f32x4 (&x)[4], f32x4& t, int rows) {
  if constexpr (K < 15) {
    if (K % 4 == 0 && K + 1 >= rows) return;   // rows past the tree's end are 0 in x
#pragma unroll
    for (int r = 0; r < 4; ++r) t[r] = __builtin_fmaf(x[K / 4][K % 4], dpp_<0x150 + K>(t[r]), t[r]);   // row_newbcast:K
    substitute<K + 1>(x, t, rows);
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
// are sums over the nodes between rather than differences. Of each node, four threads an ancestor make its two products, and
// thread t < 128 takes column t. One session whose state holds a NaN comes here in every layer and call, and all others of the
// call wait for it: a row of 64 nodes 15.0 ms where every thread made all products by itself, from memory, 0.5 now.
template <int NT, bool HALF, bool GATED>
__device__ __forceinline__ void walk_row(const TreeStepParams& p, const TreeRow& ro, TreeStepLds<NT>& lds, int tid) {
  const int col = tid & (KD - 1);
  const bool mine = tid < KD;
  const auto between = [&](uint64_t nodes) {
    float s = 0.f;
#pragma unroll 1
    for (; nodes; nodes &= nodes - 1) s += lds.g[__builtin_ctzll(nodes)];
    return s;
  };
#pragma unroll 1
  for (int i = 0; i < ro.len; ++i) {
    const uint64_t path = lds.mask[i];
    // the ancestors' products: thread 4 j + e has dims 32 e .. of node j's, and the decays of nodes 16 e .. between
    __syncthreads();   // P, which U lies over, and the coefficients of the node before are read no more
    {
      const int j = tid >> 2, e = tid & 3;
      const bool on = j <= i && (path >> j & 1u);
      float kk = 0.f, qk = 0.f, g = 0.f;
      if (on) {
#pragma unroll 1
        for (int pc = 4 * e; pc < 4 * e + 4; ++pc) {
          float x[8], y[8], z[8];
          load8_bf16(&lds.k[kq_at(j, pc)], x);
          load8_bf16(&lds.k[kq_at(i, pc)], y);
          load8_bf16(&lds.q[kq_at(i, pc)], z);
#pragma unroll
          for (int d = 0; d < 8; ++d) {
            kk = __builtin_fmaf(x[d], y[d], kk);
            qk = __builtin_fmaf(x[d], z[d], qk);
          }
        }
        g = between(path & ~lds.mask[j] & (0xffffull << (16 * e)));
      }
      kk = add_xor2(add_xor1(kk));
      qk = add_xor2(add_xor1(qk));
      g = add_xor2(add_xor1(g));
      if (on && e == 0) {
        const float d = expf(g) * lds.kinv[j];
        lds.part[j][2] = d * lds.kinv[i] * kk;
        lds.part[j][3] = d * lds.qinv[i] * qk;
      }
    }
    __syncthreads();
    float o = 0.f;
    if (mine) {
      float ks = 0.f, qs = 0.f;
#pragma unroll 1
      for (int pc = 0; pc < KD / 8; ++pc) {
        float x[8], y[8];
        load8_bf16(&lds.k[kq_at(i, pc)], x);
        load8_bf16(&lds.q[kq_at(i, pc)], y);
#pragma unroll
        for (int d = 0; d < 8; ++d) {
          const float s = state_at(p.state, HALF, ro.state_at + (int64_t)(8 * pc + d) * KD + col);
          ks = __builtin_fmaf(x[d], s, ks);
          qs = __builtin_fmaf(y[d], s, qs);
        }
      }
      const float e = expf(between(path));
      float read = e * lds.kinv[i] * ks;
      o = e * lds.qinv[i] * qs;
#pragma unroll 1
      for (uint64_t up = path & ~(1ull << i); up; up &= up - 1) {
        const int j = __builtin_ctzll(up);
        const float u = lds.U[j][col];
        read = __builtin_fmaf(lds.part[j][2], u, read);
        o = __builtin_fmaf(lds.part[j][3], u, o);
      }
      const float u = lds.beta[i] * (bf2f(ro.v[i * p.qkv_stride + col]) - read);
      lds.U[i][col] = u;
      o = __builtin_fmaf(lds.part[i][3], u, o);
    }
    if constexpr (GATED) {
      const float ss = wave_sum(o * o);
      if (mine && (tid & 63) == 0) lds.part[i][tid >> 6] = ss;
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
    for (int j = tid; j < ro.done; j += 64 * NW)
      lds.part[j][0] = expf(between(lds.mask[c] & ~lds.mask[j])) * lds.kinv[j];
    __syncthreads();
    if (mine) {
      const float e = expf(between(lds.mask[c]));
#pragma unroll 1
      for (int pc = 0; pc < KD / 8; ++pc) {
        const int64_t at = ro.state_at + (int64_t)(8 * pc) * KD + col;
        float s[8];
#pragma unroll
        for (int d = 0; d < 8; ++d) s[d] = e * state_at(p.state, HALF, at + d * KD);
#pragma unroll 1
        for (int j = 0; j < ro.done; ++j) {
          const float w = lds.part[j][0], u = lds.U[j][col];
          float x[8];
          load8_bf16(&lds.k[kq_at(j, pc)], x);
#pragma unroll
          for (int d = 0; d < 8; ++d) s[d] = __builtin_fmaf(w * x[d], u, s[d]);
        }
#pragma unroll
        for (int d = 0; d < 8; ++d) {
          if constexpr (HALF) static_cast<uint16_t*>(p.state)[at + d * KD] = f2h(s[d]);
          else static_cast<float*>(p.state)[at + d * KD] = s[d];
        }
      }
    }
  }
}

// Workgroups on a CU that the registers are held to
constexpr int occupancy(int nt, bool half) {
  return nt == 1 ? 4 : nt == 2 ? (half ? 4 : 3) : nt == 3 && half ? 3 : 2;
}

// NT: tiles of 16 nodes. One tile over an fp32 state does not move it: S0's registers are free as it is split, and four
// workgroups on a CU instead of three (352 x 1 node 59 against 67 us; with commits two tiles were as fast, and at 12 nodes
// 2 % faster).
template <int NT, bool HALF, bool GATED>
__global__ __launch_bounds__(64 * NW, occupancy(NT, HALF)) void gdn_tree_kernel(const TreeStepParams p) {
  constexpr bool MOVES = HALF || NT > 1;
  constexpr int PARTS = HALF ? 2 : 3;
  __shared__ TreeStepLds<NT> lds;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g4 = lane >> 4, c = lane & 15;
  const int n = blockIdx.x / p.HV, hv = blockIdx.x - n * p.HV;
  const int64_t slot = p.slots[n], len64 = p.lens[n], off = p.offsets[n];
  const int64_t done64 = MOVES && p.commits ? p.commits[n] : 0;
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

  // Loads are waited for in the order of their issue: what the first phases need is loaded before S0, what the last ones need
  // after it.
  // ---- the tiles of k, then of q, dealt over the waves but the first, which has the nodes' scalars ----
  constexpr int EACH = (2 * NT + NW - 2) / (NW - 1);
  const int first_job = wave ? wave - 1 : 2 * NT;
  // (lane offsets are 32 bits on a uniform base: 64-bit addresses per lane cost the registers of a workgroup on the CU)
  const uint32_t stride = (uint32_t)p.qkv_stride;
  u32x4 kq[EACH][4];
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int job = first_job + (NW - 1) * e;
    if (job >= 2 * NT) break;
    const uint16_t* const src = job >= NT ? ro.q : ro.k;
    const uint32_t row = (uint32_t)min(16 * (job % NT) + c, len - 1) * stride + 8 * g4;
#pragma unroll
    for (int s = 0; s < 4; ++s) kq[e][s] = *reinterpret_cast<const u32x4*>(src + 32 * s + row);
  }
  const int64_t node = off + min(lane, len - 1);
  uint64_t mask = 0;
  float a = 0.f, b = 0.f, a_log = 0.f, dt = 0.f;
  if (wave == 0) {
    mask = (uint64_t)p.masks[node];
    a = bf2f(p.a[node * p.ab_stride + hv]);
    b = bf2f(p.b[node * p.ab_stride + hv]);
    a_log = bf2f(p.A_log[hv]);
    dt = bf2f(p.dt_bias[hv]);
  }
  // ---- S0: rows 32 s + 8 g4 + i ----
  typedef std::conditional_t<HALF, uint32_t, f32x2> StatePair;
  typedef std::conditional_t<HALF, uint16_t, float> StateValue;
  StateValue* const state = static_cast<StateValue*>(p.state) + ro.state_at;
  const uint32_t state_lane = 8 * g4 * KD + col;
  StatePair raw[4][8];
#pragma unroll
  for (int s = 0; s < 4; ++s)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      raw[s][i] = __builtin_nontemporal_load(reinterpret_cast<const StatePair*>(state + (32 * s + i) * KD + state_lane));
  const auto s0 = [&](int s, int j, int i) {
    if constexpr (HALF) return h2f((uint16_t)(raw[s][i] >> (16 * j)));
    else return raw[s][i][j];
  };
  // ---- v and z ----
  // A wave has at most 63 loads on their way: with more than a tile it would stand here until the first are back, so that
  // there v is loaded after the first barrier and z after the state's products (96 x 33 nodes 4 % faster, 128 x 64 2 %).
  constexpr bool LATE = NT > 1;
  uint32_t vw[NT][4], zw[GATED ? NT : 1][4], nw = 0;
  const auto load_v = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = min(16 * t + 4 * g4 + r, len - 1);
        vw[t][r] = *reinterpret_cast<const uint32_t*>(ro.v + ((uint32_t)i * stride + col));
      }
  };
  const auto load_z = [&]() __attribute__((always_inline)) {
    if constexpr (GATED) {
      nw = *reinterpret_cast<const uint32_t*>(p.norm_w + col);
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = min(16 * t + 4 * g4 + r, len - 1);
          zw[t][r] = *reinterpret_cast<const uint32_t*>(ro.z + ((uint32_t)i * (uint32_t)p.z_stride + col));
        }
    }
  };
  if constexpr (!LATE) {
    load_v();
    load_z();
  }
  __builtin_amdgcn_sched_barrier(0);   // the loads stay where they stand

  // ---- k and q to LDS, and their lengths ----
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int job = first_job + (NW - 1) * e;
    if (job >= 2 * NT) break;
    const bool is_q = job >= NT;
    const int row = 16 * (job % NT) + c;
    uint16_t* const to = is_q ? lds.q : lds.k;
    float ss = 0.f;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      float y[8];
      unpack8(kq[e][s], y);
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(y[i], y[i], ss);
      *reinterpret_cast<u32x4*>(to + kq_at(row, 4 * s + g4)) = kq[e][s];
    }
    ss = add_xor32(add_xor16(ss));
    if (g4 == 0) (is_q ? lds.qinv : lds.kinv)[row] = (is_q ? p.scale : 1.0f) / sqrtf(ss + 1e-6f);
  }
  // ---- a node's scalars: lane = node ----
  if (wave == 0) {
    const bool valid = lane < len;
    const uint64_t self = 1ull << lane;
    mask = valid ? (mask & (self - 1)) | self : 0ull;
    const float g = valid ? log_decay(a, a_log, dt) : 0.f;
    // the sum down the path, by pointer doubling
    double sum = (double)g * 1.4426950408889634;   // of 2
    const uint64_t above = mask & ~self;
    int up = above ? 63 - __clzll((long long)above) : -1;
    for (int far = 1; far < len; far <<= 1) {
      const int at = up < 0 ? lane : up;
      const double more = __shfl(sum, at, 64);
      const int next = __shfl(up, at, 64);
      sum += up < 0 ? 0.0 : more;
      up = up < 0 ? -1 : next;
    }
    const double Gc = __shfl(sum, max(ro.done - 1, 0), 64);
    if (lane < 16 * NT) {
      lds.mask[lane] = mask;
      lds.g[lane] = g;
      lds.G[lane] = sum;
      lds.eG[lane] = __builtin_amdgcn_exp2f((float)sum);
      lds.left[lane] = lane < ro.done ? __builtin_amdgcn_exp2f((float)(Gc - sum)) : 0.f;
      lds.beta[lane] = valid ? sigmoid_f32(b) : 0.f;
    }
  }
  lds_barrier();
  if constexpr (LATE) {
    load_v();
    __builtin_amdgcn_sched_barrier(0);
  }

  const auto k_part = [&](int t, int s) { return load_bf16x8(&lds.k[kq_at(16 * t + c, 4 * s + g4)]); };
  const auto q_part = [&](int t, int s) { return load_bf16x8(&lds.q[kq_at(16 * t + c, 4 * s + g4)]); };
  // ---- -A and P, block pairs dealt over the waves: every pair's products are issued before the first is used ----
  constexpr int PAIRS = (NT * (NT + 1) / 2 + NW - 1) / NW;
  const auto row_block = [](int pair) { return pair < 1 ? 0 : pair < 3 ? 1 : pair < 6 ? 2 : pair < 10 ? 3 : NT; };
  f32x4 kk[PAIRS], qk[PAIRS];
#pragma unroll
  for (int e = 0; e < PAIRS; ++e) {
    const int pair = wave + NW * e, bi = row_block(pair), bj = pair - bi * (bi + 1) / 2;
    if (bi >= tiles) break;
    kk[e] = qk[e] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const bf16x8 y = k_part(bj, s);
      kk[e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k_part(bi, s), y, kk[e], 0, 0, 0);
      qk[e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(q_part(bi, s), y, qk[e], 0, 0, 0);
    }
  }
#pragma unroll
  for (int e = 0; e < PAIRS; ++e) {
    const int pair = wave + NW * e, bi = row_block(pair), bj = pair - bi * (bi + 1) / 2;
    if (bi >= tiles) break;
    const int j = 16 * bj + c, i0 = 16 * bi + 4 * g4;
    const double Gj = lds.G[j];
    const float kj = lds.kinv[j];
    const f32x4 be = *reinterpret_cast<const f32x4*>(&lds.beta[i0]), ki = *reinterpret_cast<const f32x4*>(&lds.kinv[i0]);
    const f32x4 qi = *reinterpret_cast<const f32x4*>(&lds.qinv[i0]);
    float pv[4], av[4];
    bool on[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      on[r] = lds.mask[i0 + r] >> j & 1;
      const float d = __builtin_amdgcn_exp2f((float)(lds.G[i0 + r] - Gj)) * kj;
      pv[r] = qi[r] * d * qk[e][r];
      av[r] = -be[r] * ki[r] * d * kk[e][r];
      // made for every pair: a branch around each waits for its own reads (one tile: registers)
      if constexpr (NT > 1) asm("" : "+v"(pv[r]), "+v"(av[r]));
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      lds.P[i0 + r][j] = on[r] ? pv[r] : 0.f;
      lds.A[i0 + r][j] = on[r] && i0 + r != j ? av[r] : 0.f;
    }
  }
  lds_barrier();

  // ---- the inverses of the diagonal blocks, by forward substitution: every lane has 4 columns of its row c of T ----
  const auto inverse = [&](int blk) {
    f32x4 t, x[4];
#pragma unroll
    for (int m = 0; m < 4; ++m) x[m] = *reinterpret_cast<const f32x4*>(&lds.A[16 * blk + c][16 * blk + 4 * m]);
#pragma unroll
    for (int r = 0; r < 4; ++r) t[r] = 4 * g4 + r == c ? 1.f : 0.f;
    substitute(x, t, len - 16 * blk);
    return t;
  };
  f32x4 t0 = {0.f, 0.f, 0.f, 0.f};
  if constexpr (NT == 1) t0 = inverse(0);
  else if (wave < tiles) lds.T[wave][lane] = inverse(wave);

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
    for (int j = 0; j < 2; ++j) {
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = s0(s, j, i);
      split8<PARTS>(x, part[j]);
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if (t >= tiles) break;
      const bf16x8 kf = k_part(t, s), qf = q_part(t, s);
#pragma unroll
      for (int w = PARTS - 1; w >= 0; --w)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          u[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, part[j][w], u[t][j], 0, 0, 0);
          o[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(qf, part[j][w], o[t][j], 0, 0, 0);
        }
    }
    __builtin_amdgcn_sched_barrier(0);   // the parts of one step at a time in registers
  }
  if constexpr (LATE) {
    load_z();
    __builtin_amdgcn_sched_barrier(0);
  }
  // ---- R, and the state's part of the outputs ----
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    if (t >= tiles) break;
    const int i0 = 16 * t + 4 * g4;
    const f32x4 e = *reinterpret_cast<const f32x4*>(&lds.eG[i0]), be = *reinterpret_cast<const f32x4*>(&lds.beta[i0]);
    const f32x4 ki = *reinterpret_cast<const f32x4*>(&lds.kinv[i0]), qi = *reinterpret_cast<const f32x4*>(&lds.qinv[i0]);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float v[2];
      unpack2(vw[t][r], v[0], v[1]);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        u[t][j][r] = i0 + r < len ? be[r] * (v[j] - e[r] * ki[r] * u[t][j][r]) : 0.f;
        o[t][j][r] *= e[r] * qi[r];
      }
    }
  }
  if constexpr (NT > 1) lds_barrier();

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
    const f32x4 a = NT == 1 ? t0 : lds.T[b][lane];
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
      odd += (u[t][0][r] + u[t][1][r]) * 0.f + (o0 + o1) * 0.f;   // (rows past the end: u is 0, o of the last row's q)
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
    // (the arguments are read again: kept until here, with all that this takes, they cost a register spill)
    const auto* args = (const __attribute__((address_space(4))) TreeStepParams*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(args));
    walk_row<NT, HALF, GATED>(*(const TreeStepParams*)args, ro, lds, 64 * wave + lane_per_site(lane));
    return;
  }

  // ---- gated norm, outputs ----
  float w2[2];
  unpack2(nw, w2[0], w2[1]);
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    if (t >= tiles) break;
    uint32_t w[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float y[2] = {o[t][0][r], o[t][1][r]};
      if constexpr (GATED) {
        const f32x4 ss = *reinterpret_cast<const f32x4*>(lds.part[16 * t + 4 * g4 + r]);
        const float rs = rsqrtf(((ss[0] + ss[1]) + (ss[2] + ss[3])) * (1.0f / KD) + p.eps);
        float z[2];
        unpack2(zw[t][r], z[0], z[1]);
#pragma unroll
        for (int j = 0; j < 2; ++j) y[j] *= rs * w2[j] * silu_fast(z[j]);
      }
      w[r] = pack_bf16x2(y[0], y[1]);
      if constexpr (NT > 1) asm("" : "+v"(w[r]));   // made for every row: a branch around each waits for its own reads
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = 16 * t + 4 * g4 + r;
      if (i < len) *reinterpret_cast<uint32_t*>(ro.out + ((uint32_t)i * (uint32_t)(p.HV * KD) + col)) = w[r];
    }
  }

  // ---- the committed chain moves the state: u scaled, split as the state was, times k^T read from LDS transposed ----
  if (MOVES && ro.done > 0) {
    const float ec = lds.eG[ro.done - 1];
    constexpr int NP = (NT + 1) / 2;     // pairs of tiles: a product takes 32 nodes, the lane's own 4 of either tile
    // (an fp16 state takes u with all its digits too: the 16 of two parts, cut off, made every update smaller and moved values
    // by up to 1.2e-4 of their row beyond fp16's own rounding, where 7.6e-6 is the bar now; 96 x 33 nodes 68.4 -> 70.4 us)
    constexpr int U_PARTS = 3;
    bf16x8 up[NP][2][U_PARTS];
#pragma unroll
    for (int t2 = 0; t2 < NP; ++t2) {
      float x[2][8] = {};
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const int t = 2 * t2 + hh;
        if (t >= NT) break;
        const int i0 = 16 * t + 4 * g4;
        const f32x4 le = *reinterpret_cast<const f32x4*>(&lds.left[i0]), ki = *reinterpret_cast<const f32x4*>(&lds.kinv[i0]);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int j = 0; j < 2; ++j) x[j][4 * hh + r] = i0 + r < ro.done ? u[t][j][r] * (le[r] * ki[r]) : 0.f;
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) split8<U_PARTS>(x[j], up[t2][j]);
    }
    // state rows 32 s ..: accumulator row 4 g4 + r is state row 32 s + 8 g4 + 4 hh + r, operand row m = c is k's dim 32 s +
    // 8 (c / 4) + 4 hh + c % 4, which transpose reads of 4-value vectors 8 dims apart give
    const auto move = [&](int s, const auto& was) __attribute__((always_inline)) {
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        f32x4 acc[2];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[j][r] = ec * was(j, 4 * hh + r);
#pragma unroll
        for (int t2 = 0; t2 < NP; ++t2) {
          if (32 * t2 >= ro.done) break;
          const auto four = [&](int t) {
            const int i = 16 * t + 4 * g4 + (c >> 2);   // this lane's address: node row, vector c % 4
            return ld_tr4(&lds.k[kq_at(i, 4 * s + (c & 3)) + 4 * hh]);
          };
          const u32x2 lo = four(2 * t2);
          u32x2 hi = {0u, 0u};
          if (2 * t2 + 1 < NT) hi = four(2 * t2 + 1 < NT ? 2 * t2 + 1 : 0);
          const bf16x8 kf = __builtin_bit_cast(bf16x8, (u32x4){lo[0], lo[1], hi[0], hi[1]});
#pragma unroll
          for (int w = U_PARTS - 1; w >= 0; --w)
#pragma unroll
            for (int j = 0; j < 2; ++j)
              acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, up[t2][j][w], acc[j], 0, 0, 0);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          StateValue* const at = state + (32 * s + 4 * hh + r) * KD + state_lane;
          if constexpr (HALF)
            __builtin_nontemporal_store((uint32_t)f2h(acc[0][r]) | ((uint32_t)f2h(acc[1][r]) << 16),
                                        reinterpret_cast<uint32_t*>(at));
          else __builtin_nontemporal_store((f32x2){acc[0][r], acc[1][r]}, reinterpret_cast<f32x2*>(at));
        }
      }
    };
    // (through an empty asm: the values as converted and split for the products would be kept for this)
#pragma unroll
    for (int s = 0; s < 4; ++s) {
#pragma unroll
      for (int i = 0; i < 8; ++i) asm volatile("" : "+v"(raw[s][i]));
      move(s, [&](int j, int i) { return s0(s, j, i); });
      __builtin_amdgcn_sched_barrier(0);
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
  if ((state_dtype != HSG_STATE_F32 && state_dtype != HSG_STATE_F16) || !isfinite(scale)) return HSG_ERR_ARG;
  if (K != KD || V != KD || max_nodes <= 0 || max_nodes > HSG_TREE_MAX_NODES) return HSG_ERR_SHAPE;
  if (n_rows == 0) return HSG_OK;
  if (!qkv || !a || !b || !A_log || !dt_bias || !state || !slots || !lens || !offsets || !masks || !out ||
      (z && !norm_w))
    return HSG_ERR_ARG;
  // a row's values are addressed by 32-bit byte offsets
  if (qkv_stride < 0 || qkv_stride >= (1 << 24) || z_stride >= (1 << 24) || HV >= (1 << 16)) return HSG_ERR_SHAPE;
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
  // Tiles by the bound on a row's nodes: registers and LDS decide how many workgroups a CU holds. 352 x 1, fp16 state: 46 us
  // with one tile, 49 with two, 55 with three; 200 x 24 with commits 82.6 with two, 85.2 with three; 96 x 33, fp16, 32 value
  // heads, 68.6 with three, 79.7 with four (fp32, 16 heads 49.7 and 51.8).
  if (max_nodes <= 16 && (state_dtype == HSG_STATE_F16 || !commits)) by_type(std::integral_constant<int, 1>{});
  else if (max_nodes <= 32) by_type(std::integral_constant<int, 2>{});
  else if (max_nodes <= 48) by_type(std::integral_constant<int, 3>{});
  else by_type(std::integral_constant<int, 4>{});
  return launch_status();
}
