// linear_attention.cuh -- what the linear-attention kernels share.
//
// Linear attention with one decay factor g = exp(log_decay) for each head:
//     S_t = g S_{t-1} + k_t v_t^T          (dk x dv, fp32)
//     o_t = scale * q_t S_t
// Written over a chunk of tokens with the state S before it, i and j counting from its start:
//     o_i = scale * ( sum_{j<=i} g^(i-j) (q_i . k_j) v_j  +  g^(i+1) q_i S )
// The gradients are the same computation with the tensors' parts exchanged:
//     dq_i = scale * ( sum_{j<=i} g^(i-j) (do_i . v_j) k_j + g^(i+1) do_i S^T )
//     dk_j = sum_{i>=j} g^(i-j) (v_j . scale do_i) q_i + g^(j') v_j R^T
//     dv_j = sum_{i>=j} g^(i-j) (k_j . scale q_i) do_i + g^(j') k_j R
// where R, the gradient of the state from all later tokens, obeys the same recurrence from
// the last token to the first, and j' counts tokens from the chunk's end.  So every
// kernel here computes one "role"
//     out_r = a_scale * sum_c g^|r-c| (x_r . y_c) w_c + i_scale * g^(a+e) x_r S
//     S    <- g^L S + sum_c w_scale * g^(L-e-a(c)) y_c w_c^T
// over chunks in scan order, which is time order (e = 1) or reversed time (e = 0); a
// counts a chunk's tokens in scan order and L is their number.
//
// One chain is a (role, batch row, head, slice of w's columns).  A chain can be cut into
// segments that run at the same time: a first pass computes each segment's own state
// from zero, a scan turns these into the states at the segments' starts, and the main
// pass starts from them.
#pragma once

#include "common.cuh"

namespace dynconv {
namespace la {

constexpr int kMaxRoles = 3;
constexpr int kMaxDim = 256;  // dk, dv

// A [B, T, H, d] tensor: element strides of batch, time and head; d is dense.
struct View {
  const void* p;
  int64_t sb, st, sh;
};

struct Role {
  View x, y, w, out;
  const float* s_in;  // [B*H][dk*dv] or null (zero)
  float* s_out;       // [B*H][dk*dv] or null (not wanted)
  int si, sj;         // element strides of a state's x-dimension and w-dimension in s_in / s_out
  int dx, dw;         // width of x and y, width of w and out
  int reverse;
  float a_scale, i_scale, w_scale;
};

struct Params {
  Role role[kMaxRoles];
  int n_roles;
  int B, H;
  int64_t T;
  const float* log_decay;  // [H]
  int n_seg;               // segments of a chain
  int chunks_per_seg;
  float* seg;              // n_seg > 1: [role][n_seg][B*H][dx*dw] (dx*dw is the same for every role)
  int scan_final;          // the state pass covers the last segment too, and the scan writes s_out
};

// log2 of the decay factor.  A factor of zero is kept finite, so that 0 * log stays 0.
__device__ __forceinline__ double log2_decay(const float* log_decay, int h) {
  const double l2 = (double)log_decay[h] * 1.4426950408889634;
  return l2 < -16384.0 ? -16384.0 : l2;  // (a NaN stays one)
}

// A state's factor over n tokens as a sum of two floats.  The same factor multiplies the
// state chunk after chunk, so its rounding would add up: a head that remembers 4096 tokens
// keeps 128 chunks of 32, and one float's 2^-24 became 2e-6 of the state.
struct Factor {
  float hi, lo;
};
__device__ __forceinline__ Factor decay_factor(double l2, double n) {
  const double f = exp2(l2 * n);
  const float hi = (float)f;
  return Factor{hi, isinf(hi) ? 0.f : (float)(f - (double)hi)};
}
// f * S + a
__device__ __forceinline__ float decay_add(Factor f, float S, float a) { return fmaf(f.hi, S, fmaf(f.lo, S, a)); }

inline bool wants_states(const Params& p) {
  for (int r = 0; r < p.n_roles; ++r)
    if (p.role[r].s_out) return true;
  return false;
}

__device__ __forceinline__ float* seg_state(const Params& p, int role, int seg, int64_t bh, int64_t n) {
  return p.seg + ((int64_t)(role * p.n_seg + seg) * p.B * p.H + bh) * n;
}

// Cuts chains into the number of segments with the lowest estimated time, counted in chunks of one
// CTA: both passes run in rounds of `slots` CTAs; an uncut chain costs `whole` and the state pass
// `state_pass` of a chunk's time per chunk, a round's start `start` and the scan `scan` chunks.
// Sets n_seg and chunks_per_seg; p->scan_final says what the state pass covers.
void plan_segments(Params* p, int chunk, int slice, int slots, double whole, double state_pass, double start,
                   double scan);

// Launches the scan over segment states (role.s_in -> p.seg in place; chunk = tokens per chunk).
int scan_launch(const Params& p, int chunk, cudaStream_t st);
// CUDA-core kernels: any type, strides and widths up to kMaxDim.
void simple_plan(Params* p);  // chooses n_seg and chunks_per_seg
int simple_launch(const Params& p, int dtype, cudaStream_t st);
// tcgen05 kernels: see tc_supported for their envelope.
bool tc_supported(const Params& p, int dtype);
void tc_plan(Params* p, bool states);  // states: the state after the last token is wanted
int tc_launch(const Params& p, cudaStream_t st);

int step_launch(const View& q, const View& k, const View& v, float* state, const float* log_decay, void* o,
                const void* slots, int slot_bytes, int64_t B, int64_t n_rows, int H, int dk, int dv, float scale,
                int dtype, cudaStream_t st);

}  // namespace la
}  // namespace dynconv
