// vocab_loss.cuh -- what the vocabulary-loss kernels share.
//
// Softmax cross entropy of hidden [N, D] against a vocabulary weight [V, D] without the
// logits [N, V] in memory.  With l = hidden weight^T:
//     lse_n = log sum_v exp(l_nv),  loss_n = lse_n - l_{n,t_n}
//     dl_nv = (exp(l_nv - lse_n) - [v = t_n]) * g_n, for the target itself expm1(-loss_n) * g_n
//     dhidden = dl weight,  dweight = dl^T hidden
// The factors g_n are dloss (sum) or dloss / count (mean) of every row that counts: they multiply
// the finished products in fp32, and the operand dl is exp(l - lse) - [v = t] alone, so that
// its largest entry, near -1, is not rounded together with a factor that is the same for every
// row (one bf16 rounding of the factor moved both gradients by up to 2^-8).  With one dloss
// per row (no reduction) the factors differ and are part of dl.
// Forward: one matrix product whose epilogue keeps, of each tile, every row's maximum and sum of
// exponentials (fp32) over all words but the target; a second kernel merges the tiles.  With lse' over
// the others, loss = log(1 + exp(lse' - l_t)) and lse = l_t + loss: a row that its target dominates keeps
// the digits of a small loss, which a sum with the target's own 1 in it, or a difference of lse and
// l_t, would lose.  For the same reason the backward gets lse and the rows' losses.  Backward, piece of the
// vocabulary by piece: the product again, with dl in bf16 (three parts of it for fp32
// tensors) into a piece buffer, then its two products.  dhidden accumulates in fp32 over the pieces.
#pragma once

#include "common.cuh"

namespace dynconv {
namespace vl {

constexpr float kLog2e = 1.4426950408889634f;

enum Reduction { kNone = 0, kSum = 1, kMean = 2 };
constexpr int kKeepRows = 4;  // added to the reduction by callers whose lse has [2][N] numbers

struct Problem {
  const void* hidden;       // [N, D]
  const void* weight;       // [V, D]
  const int64_t* target;    // [N]
  int64_t N, D, V;
  int64_t ignore;
  int reduction;
  // forward
  float* lse;               // [N]
  float* row_loss;          // [N], or null: not kept
  float* loss;              // [N] (kNone) or [1]
  float* stats;             // [2]: sum of the rows' losses, number of rows that count
  float2* part;             // [tiles][rows at once]: of a tile's row, without the target's word,
                            // m = max * log2(e) rounded, and sum of 2^(l * log2(e) - m)
  float* tgt;               // [N]: the target's logit
  // backward
  const float* dloss;       // [N] (kNone) or [1]
  void* dhidden;            // [N, D] or null
  void* dweight;            // [V, D] or null
  void* piece;              // [parts][N][pitch]: dl of one piece of the vocabulary
  float* acc_h;             // [z_h][N][D] fp32; rows of copy_pitch(D) where operands are copies
  float* acc_w;             // [z_w][piece rows][D] fp32 likewise, where dweight is not written at once
  // either way, where operands are copies
  __nv_bfloat16* hidden_copy;  // [parts][N or rows at once][copy_pitch]; for dweight always
  __nv_bfloat16* weight_copy;  // [parts][words at once][copy_pitch]
  cudaStream_t st;
};

// How the backward is cut: columns of a piece, its row pitch, and over how many CTAs a
// tile's inner dimension is spread where there are few tiles.
struct Plan {
  int64_t piece, pitch;
  int z_h, z_w;
};

// The larger of two numbers; NaN if either is (fmaxf would drop it, and with it a row's NaN logits).
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// A row's factor within dl: 0 where the target is ignored or outside the vocabulary.
__device__ __forceinline__ float row_factor(const Problem& p, int64_t n, int64_t t) {
  if (t == p.ignore || t < 0 || t >= p.V) return 0.f;
  return p.reduction == kNone ? p.dloss[n] : 1.f;
}

// The factor of both finished gradients.  (No row that counts: dl is zero, and so are they.)
__device__ __forceinline__ float result_factor(const Problem& p) {
  if (p.reduction == kNone) return 1.f;
  if (p.reduction == kSum) return p.dloss[0];
  return p.stats[1] > 0.f ? p.dloss[0] / p.stats[1] : 0.f;
}

// The forward takes this many rows at a time: it bounds the tiles' partial sums in the workspace
// (8 bytes for each row and tile), and the weight is read again once per 32768 rows only.
constexpr int64_t kRowsAtOnce = 32768;
constexpr int kTileColumns = 128;  // of the vocabulary: the forward keeps a (maximum, sum) for each

// The products run on bf16 operands that TMA can address.  fp32 tensors are copied as three bf16
// parts: x = x0 + x1 + x2, each part the rest rounded to bf16 (8 digits each: the three hold all
// 24), and a product of two such numbers is the six products of parts whose indices add up to at
// most two; the three left out are below 2^-23 of it.  bf16 tensors whose rows are no multiple of
// 16 bytes are copied as they are, with padded rows ("one part").
inline bool copied(int64_t D, int dtype) { return dtype == DYNCONV_DTYPE_F32 || D % 8 != 0; }
inline int parts_of(int dtype) { return dtype == DYNCONV_DTYPE_F32 ? 3 : 1; }
__host__ __device__ constexpr int products_of(int parts) { return parts == 3 ? 6 : 1; }
// The tensor core's accumulation truncates (vocab_loss_tc.cu): of copied operands, 4 blocks of 64
// inner elements are summed there, and these sums in fp32 registers.
constexpr int kCopyChain = 4;
inline int64_t copy_pitch(int64_t D) { return (D + 7) / 8 * 8; }
inline size_t copy_bytes(int64_t rows, int64_t D, int dtype) { return (size_t)parts_of(dtype) * 2 * rows * copy_pitch(D); }
// Words of the vocabulary that are copied at once: at most 512 MB of copies.
inline int64_t words_at_once(int64_t D, int64_t V, int dtype) {
  const int64_t most = ((int64_t)512 << 20) / (int64_t)copy_bytes(1, D, dtype) / 256 * 256;
  return most < 1024 ? (V < 1024 ? V : 1024) : most < V ? most : V;
}

Plan plan(int64_t N, int64_t D, int64_t V, int dtype);
int merge_launch(const Problem& rows, int64_t tiles);  // the rows' losses from their tiles
int total_launch(const Problem& p);                    // their sum and number
// The part of a forward problem that begins at row r0.
inline Problem rows_from(const Problem& p, int64_t r0, int64_t elem) {
  Problem r = p;
  r.N = p.N - r0 < kRowsAtOnce ? p.N - r0 : kRowsAtOnce;
  r.hidden = (const char*)p.hidden + r0 * p.D * elem;
  r.target += r0, r.lse += r0, r.tgt += r0;
  if (p.row_loss) r.row_loss += r0;
  if (p.reduction == kNone) r.loss += r0;
  return r;
}
// out [rows][D] = result_factor * the sum of n_parts [rows][ld], in their order, rounded to dtype
int finish_launch(const Problem& p, const float* parts, int n_parts, int64_t rows, int64_t ld, void* out, int dtype);

int forward(const Problem& p, int dtype);
int backward(const Problem& p, const Plan& pl, int dtype);

}  // namespace vl
}  // namespace dynconv
