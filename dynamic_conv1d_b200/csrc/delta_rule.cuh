// delta_rule.cuh -- what the kernels of the gated delta rule share.
//
//     S_t = a_t S_{t-1} + k_t u_t^T,   u_t = beta_t (v_t - a_t S_{t-1}^T k_t),   o_t = scale S_t^T q_t
// with a_t = exp(log_decay_t), S dk x dv.  Over a chunk of C tokens with the state S0 before it, with
// b the running sum of log_decay and G_ij = exp(b_i - b_j):
//     L_ij = G_ij (k_i . k_j)  (j < i),   r = (I + L beta)^-1 (V - e^b K S0),   U = beta r
//     O = scale e^b Q S0 + P U,  P_ij = scale G_ij (q_i . k_j)  (j <= i)
//     S1 = e^(b_C) S0 + K^T (e^(b_C - b) U)
// (r_t = v_t - a_t S_{t-1}^T k_t) and for the gradients dO of O and dS1 of S1:
//     dU = (I + beta L)^-T (P^T dO + e^(b_C - b) K dS1)
//     dS0 = e^(b_C) dS1 + Q^T (scale e^b dO) - K^T (beta e^b dU)
//     dV = beta dU,  dbeta_i = dU_i . r_i
//     W_ij = scale G_ij beta_j (dO_i . r_j)  (j <= i),   N_ij = -beta_i beta_j G_ij (dU_i . r_j)  (j < i)
//     dQ = W K + scale e^b dO S0^T
//     dK = W^T Q + (N + N^T) K + e^(b_C - b) beta r dS1^T - beta e^b dU S0^T
//     dlog_decay_t = sum_{i >= t > j} (W_ij (q_i . k_j) + N_ij (k_i . k_j)) + e^(b_C) <dS1, S0>
//                    + sum_{i >= t} e^b_i (scale q_i S0 dO_i - beta_i k_i S0 dU_i) + sum_{j < t} e^(b_C - b_j) beta_j k_j dS1 r_j
//
// T = (I + A)^-1, P and the gates of all chunks come from one launch over the chunks (delta_prep.cu); then chains
// walk the chunks of each (batch row, head) (delta_rule_fwd.cu, delta_rule_bwd.cu), and the gradients of q, k
// and the gates come from another launch over the chunks.
//
// The chains run on the warps' own matrix instructions (m16n8k16), not on tensor memory: a chunk is
// three small products that depend on one another, and between them their results only change from the
// layout of the instruction's accumulators to that of its first operand, which is the same registers.  The state
// is held transposed, 16 columns of v as the rows of the instruction's tile; a team of warps
// shares those columns, each holding some of dk and working out some of the tokens.
//
// Operands are bf16; a number that must keep its digits is the sum of two or three bf16 parts
// (16 or 24 digits), and a product of two such is the sum of its parts' products above the last
// digit kept.  fp32 tensors are three parts throughout.
#pragma once

#include <type_traits>

#include "common.cuh"

namespace dynconv {
namespace dr {

constexpr int kMaxKey = 128;    // dk
constexpr int kMaxValue = 256;  // dv

// A [B, T, H, d] tensor: element strides of batch, time and head; d is dense (1 for the gates).
struct View {
  const void* p;
  int64_t sb, st, sh;
};

// What the launch over the chunks leaves for the chains, in the caller's workspace: T and P as the blocks (i, j),
// j <= i, of 16 x 16, [B*H][chunks][blocks][parts][512 bytes] in the order in which a warp reads them as second
// operands; the gates; and copies of k, q and v where the chains cannot have them from tensor maps: k and q as
// tiles of their parts as they lie in shared memory [B*H][chunks][parts][halves][C][64], v as
// [B*H][chunks * C][dv16] (dv16: dv up to a multiple of 16).
struct Prepared {
  uint4 *t, *p;
  void* gates;
  __nv_bfloat16 *k, *q;  // null: read in place
  void* v;               // (backward: dO)
};

struct Forward {
  View q, k, v, g, beta, o;   // g: log_decay
  int gates32;                // g and beta are float32 (else of the tensors' type; kernels take their type, GT: a branch on
                              // it cost the preparation 5 us of 61, each load waited for before the next)
  const float* s_in;          // [B*H][dk][dv] or null (zero)
  float* s_out;               // or null (not wanted)
  // for the backward (null: not wanted), transposed and as 8 x 8 matrices of 128 bytes: the states before the
  // chunks [1 or 3 parts][B*H][chunks][dv16 / 16][dk16 / 16][4] and the remainders r
  // [2 or 3 parts][B*H][chunks][dv16 / 16][C / 16][4]
  __nv_bfloat16 *states, *rest;
  Prepared pre;
  int B, H, dk, dv;
  int64_t T;
  float scale;
};

// One token: q, k, v, g, beta without a time stride.
struct Step {
  View q, k, v, g, beta;
  int gates32;
  void* o;
  float* state;
  const void* slots;
  int slot_bytes;
  int64_t B, n_rows;
  int H, dk, dv;
  float scale;
};

struct Backward {
  View q, k, g, beta, d_o;
  View dq, dk_, dv_, dg, dbeta;         // written
  int gates32;                          // so g, beta, dg and dbeta
  const __nv_bfloat16 *states, *rest;   // of the forward
  __nv_bfloat16 *dstates, *du;          // dS1 of the chunks and dU, laid out like them
  const float* ds_out;                  // gradient of the state after the last token, or null
  float* ds_in;                         // or null (not wanted)
  Prepared pre;
  int B, H, dk, dv;
  int64_t T;
  float scale;
};

int step_launch(const Step& p, int dtype, cudaStream_t st);
int forward_launch(const Forward& p, int dtype, cudaStream_t st);
int backward_launch(const Backward& p, int dtype, cudaStream_t st);
int grad_launch(const Backward& p, int dtype, cudaStream_t st);  // the last of its launches

constexpr int chunk_of(int dtype) { return dtype == DYNCONV_DTYPE_F32 ? 32 : 64; }
inline int64_t chunks_of(int64_t T, int dtype) { return (T + chunk_of(dtype) - 1) / chunk_of(dtype); }
inline bool packs_keys(int64_t dk, int dtype) { return dtype == DYNCONV_DTYPE_F32 || dk % 8 != 0; }
inline bool packs_values(int64_t dv, int dtype) { return dv % (dtype == DYNCONV_DTYPE_F32 ? 4 : 8) != 0; }

// Bytes of what the forward keeps, which the backward has once more for its own: states, remainders.
struct Kept {
  size_t states, rest;
};
inline Kept kept_bytes(int64_t B, int64_t T, int64_t H, int64_t dk, int64_t dv, int dtype) {
  const bool f32 = dtype == DYNCONV_DTYPE_F32;
  const int64_t n = B * H * chunks_of(T, dtype), dk16 = (dk + 15) / 16 * 16, dv16 = (dv + 15) / 16 * 16;
  return Kept{(size_t)(2 * (f32 ? 3 : 1) * n * dv16 * dk16), (size_t)(2 * (f32 ? 3 : 2) * n * chunk_of(dtype) * dv16)};
}
// Carves the workspace of `Prepared` (at `base`, which may be null); its bytes.
size_t prepared_bytes(Prepared* p, void* base, int64_t B, int64_t T, int64_t H, int64_t dk, int64_t dv, int dtype, bool back);
// Chains whose state goes back to the caller hold their numbers as three parts (`exact`), as fp32 ones do.
int prep_launch(const Prepared& to, const View& k, const View& q, const View& v, const View& g, const View& beta, int gates32, int B, int H,
                int64_t T, int dk, int dv, float scale, int dtype, bool exact, bool back, cudaStream_t st);

// ---------------------------------------------------------------- matrix instructions

__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void stsm_t(uint32_t addr, uint32_t r0, uint32_t r1, uint32_t r2, uint32_t r3) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(r0), "r"(r1),
               "r"(r2), "r"(r3)
               : "memory");
}

// Offsets (in elements) of a lane's row for the four 8 x 8 matrices of one ldmatrix.  `rows_first`: the
// second matrix is 8 rows further down and the third 8 columns to the right; else the other way about.
__device__ __forceinline__ int lane_offset(int pitch, bool rows_first) {
  const int l = threadIdx.x & 31, a = (l >> 3) & 1, b = l >> 4, r = l & 7;
  return rows_first ? (r + 8 * a) * pitch + 8 * b : (r + 8 * b) * pitch + 8 * a;
}

__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float low(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float high(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

// x and y as N bf16 parts each, packed in pairs.
template <int N>
__device__ __forceinline__ void split(float x, float y, uint32_t (&p)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    p[i] = pack(x, y);
    if (i + 1 < N) x -= low(p[i]), y -= high(p[i]);
  }
}

// The parts of a 16 x 16 first operand from two neighbouring 16 x 8 accumulators.
template <int N>
__device__ __forceinline__ void operand(const float (&c0)[4], const float (&c1)[4], uint32_t (&a)[N][4]) {
  uint32_t p[N];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float(&c)[4] = i < 2 ? c0 : c1;
    split<N>(c[2 * (i & 1)], c[2 * (i & 1) + 1], p);
#pragma unroll
    for (int j = 0; j < N; ++j) a[j][i] = p[j];
  }
}

// X += first operand parts x second operand parts, the pairs above the last digit kept.
template <int NA, int NB, int KEEP>
__device__ __forceinline__ void mma_parts(float (&c0)[4], float (&c1)[4], const uint32_t (&a)[NA][4],
                                          const uint32_t (&b)[NB][4]) {
#pragma unroll
  for (int s = KEEP - 1; s >= 0; --s)  // (small products first)
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      const int j = s - i;
      if (j < 0 || j >= NB) continue;
      mma(c0, a[i], b[j][0], b[j][1]);
      mma(c1, a[i], b[j][2], b[j][3]);
    }
}

// The same with the products of each level (the parts' indexes added up) in accumulators of their own, of which
// there are L: a chain of dependent instructions is what few warps wait for.
template <int NA, int NB, int KEEP, int L>
__device__ __forceinline__ void mma_levels(float (&c)[L][2][4], const uint32_t (&a)[NA][4], const uint32_t (&b)[NB][4]) {
#pragma unroll
  for (int s = KEEP - 1; s >= 0; --s)
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      const int j = s - i;
      if (j < 0 || j >= NB) continue;
      mma(c[s < L ? s : L - 1][0], a[i], b[j][0], b[j][1]);
      mma(c[s < L ? s : L - 1][1], a[i], b[j][2], b[j][3]);
    }
}
template <int L>
__device__ __forceinline__ void sum_levels(float (&out)[2][4], const float (&c)[L][2][4]) {
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float x = c[L - 1][m][e];
#pragma unroll
      for (int s = L - 2; s >= 0; --s) x += c[s][m][e];
      out[m][e] = x;
    }
}

// The warp's index, known to be the same in all its lanes: branches on it leave matrix instructions
// without the reconvergence that the compiler otherwise puts before each.
__device__ __forceinline__ int warp_index() { return __shfl_sync(0xffffffffu, (int)threadIdx.x / 32, 0); }

__device__ __forceinline__ void zero(float (&c)[4]) { c[0] = c[1] = c[2] = c[3] = 0.f; }

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// ------------------------------------------------------------------ a chunk's tiles

// A tile of one part of K or Q is [2 halves][C tokens][64 columns] with the 16-byte pieces of a row of 128
// bytes exchanged as by a tensor map's 128-byte swizzle (one half where dk <= 64): no bank conflicts for ldmatrix.
__device__ __forceinline__ uint32_t key_swizzle(int r, int piece) { return r * 128 + ((piece ^ (r & 7)) << 4); }
// A lane's row addresses in it for 16 tokens x 16 columns at a time (rows_first: as for lane_offset).
struct KeyLane {
  uint32_t off[4];
  __device__ __forceinline__ explicit KeyLane(bool rows_first) {
    const int l = threadIdx.x & 31, a = (l >> 3) & 1, b = l >> 4, r = (l & 7) + 8 * (rows_first ? a : b);
#pragma unroll
    for (int i = 0; i < 4; ++i) off[i] = key_swizzle(r, 2 * i + (rows_first ? b : a));
  }
  // columns 16 kk .. of the tokens from 16 block on
  template <int C>
  __device__ __forceinline__ uint32_t at(int block, int kk) const {
    return off[kk & 3] + (kk >> 2) * (C * 128) + block * 2048;
  }
};

// PX: parts of the input tensors; NP: parts of the chain's own numbers; PP: parts of P; C: tokens.
template <int PX_, int NP_, int PP_, int C_>
struct Cfg {
  static constexpr int PX = PX_, NP = NP_, PP = PP_, C = C_;
  using T = typename std::conditional<PX_ == 1, __nv_bfloat16, float>::type;
  static constexpr int kBlocks = C / 16, kLower = kBlocks * (kBlocks + 1) / 2;  // blocks of 16 tokens; pairs j <= i
  static constexpr int kSquare = C + 8;   // pitch of a C x C matrix
  static constexpr int kTile = C * kMaxKey;  // elements of one part of K or Q
};
// P has two parts in bf16 too: with one, the outputs were 2.5e-3 off in the root mean square, where their own rounding is 1.65e-3.
template <bool EXACT, bool BACK>
using CfgBf16 = Cfg<1, EXACT ? 3 : 2, 2, 64>;
using CfgF32 = Cfg<3, 3, 3, 32>;
__host__ __device__ constexpr int lower(int i, int j) { return i * (i + 1) / 2 + j; }

// Gates of a chunk, as the chains read them.
template <int C>
struct alignas(16) Gates {
  float beta[C], e[C], out[C];  // beta, e^b, e^(b_C - b)
  float hi[C], lo[C];           // b log2(e) as a sum of two floats
  float total;                  // e^(b_C)
  int bad;                      // forward: the first token whose key or gates are not finite (C: none)
};

// A number as a sum of two floats.
struct Two {
  float hi, lo;
};
__device__ __forceinline__ Two quick_two(float a, float b) {  // |a| >= |b|
  const float s = __fadd_rn(a, b);
  return Two{s, __fsub_rn(b, __fsub_rn(s, a))};
}
__device__ __forceinline__ Two add(Two a, Two b) {
  const float s = __fadd_rn(a.hi, b.hi), t = __fsub_rn(s, a.hi);
  const float e = __fadd_rn(__fsub_rn(a.hi, __fsub_rn(s, t)), __fsub_rn(b.hi, t));
  return quick_two(s, __fadd_rn(e, __fadd_rn(a.lo, b.lo)));
}
// 2^x by the special-function unit (2 ulp, 0 below 2^-126)
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float exp2_two(Two x) { return exp2_fast(x.hi) * fmaf(x.lo, 0.69314718f, 1.f); }

// Whether a tensor map can read v (its rows at positive multiples of 16 bytes).
inline bool mappable(const View& v, int64_t B, int64_t T, int64_t H, int elem) {
  if (reinterpret_cast<uintptr_t>(v.p) & 15) return false;
  const int64_t s[3] = {v.sb, v.st, v.sh}, n[3] = {B, T, H};
  for (int i = 0; i < 3; ++i)
    if (n[i] > 1 && (s[i] <= 0 || s[i] * elem % 16 != 0 || s[i] * elem >= ((int64_t)1 << 40))) return false;
  return true;
}
// A tile of rows of 32, 64 or 128 bytes as a tensor map with the swizzle of that width leaves it: where the 16-byte piece of a
// row lies.  (32: no swizzle.)
__device__ __forceinline__ uint32_t row_swizzle(int row_bytes, int r, int piece) {
  const int turn = row_bytes == 128 ? r & 7 : row_bytes == 64 ? (r >> 1) & 3 : 0;
  return r * row_bytes + ((piece ^ turn) << 4);
}
// Tiles of `rows` tokens and `cols` columns (32, 64 or 128 bytes) of a [B, T, H, width] tensor, swizzled as above; fp32
// as pairs of 16-bit numbers.
inline int view_map(CUtensorMap* map, const View& v, int64_t B, int64_t T, int64_t H, int width, int elem, int cols, int rows) {
  const int per = elem / 2;
  const cuuint64_t dims[4] = {(cuuint64_t)(width * per), (cuuint64_t)H, (cuuint64_t)T, (cuuint64_t)B};
  const cuuint64_t strides[3] = {(cuuint64_t)(H > 1 ? v.sh * elem : 16), (cuuint64_t)(T > 1 ? v.st * elem : 16),
                                 (cuuint64_t)(B > 1 ? v.sb * elem : 16)};
  const cuuint32_t box[4] = {(cuuint32_t)(cols * per), 1, (cuuint32_t)rows, 1};
  const int bytes = cols * elem;
  return encode_tensor_map_bf16(map, v.p, 4, dims, strides, box,
                                bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B
                                : bytes == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                                              : CU_TENSOR_MAP_SWIZZLE_NONE);
}
// The same of v or dO, from the tensor or from its copy.
inline int value_map(CUtensorMap* map, const Prepared& pre, const View& v, int64_t B, int64_t T, int64_t H, int dv, int elem, int cols, int C) {
  if (!pre.v) return view_map(map, v, B, T, H, dv, elem, cols, C);
  const int64_t dv16 = (dv + 15) / 16 * 16, all = (T + C - 1) / C * C;
  return view_map(map, View{pre.v, H * all * dv16, dv16, all * dv16}, B, all, H, (int)dv16, elem, cols, C);
}
struct Maps {
  CUtensorMap k, q, v;  // (v: or dO)
};

inline bool vectors_of(const View& v, int width, int elem) {
  const int per = 16 / elem;
  return width % per == 0 && v.sb % per == 0 && v.st % per == 0 && v.sh % per == 0 && (reinterpret_cast<uintptr_t>(v.p) & 15) == 0;
}

}  // namespace dr
}  // namespace dynconv
