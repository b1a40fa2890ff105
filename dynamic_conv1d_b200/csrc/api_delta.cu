// api_delta.cu -- extern "C" entry points of the gated delta rule and of the norms around it (declared in
// include/dynconv.h).  Like api.cu it validates, carves the caller's workspace and dispatches; it
// allocates nothing and never synchronises.
#include <algorithm>

#include "common.cuh"
#include "delta_rule.cuh"
#include "norm.cuh"

namespace dynconv {
namespace {

constexpr int64_t kMaxRows = 65535;  // grid limits: batch rows and heads of a step, their product in a sequence

// Takes DYNCONV_GATES_F32 or DYNCONV_WEIGHTS_F32, the same number, out of `dtype`.
static_assert(DYNCONV_GATES_F32 == DYNCONV_WEIGHTS_F32, "one flag");
bool take_f32(int& dtype) {
  const bool there = dtype >= 0 && (dtype & DYNCONV_GATES_F32);
  if (there) dtype -= DYNCONV_GATES_F32;
  return there;
}

int check_widths(int64_t dk, int64_t dv) {
  if (dk < 1 || dk > dr::kMaxKey || dv < 1 || dv > dr::kMaxValue)
    return set_error(DYNCONV_ERR_UNSUPPORTED, "gated delta rule: dk=%lld (1..%d), dv=%lld (1..%d)", (long long)dk, dr::kMaxKey,
                     (long long)dv, dr::kMaxValue);
  return DYNCONV_OK;
}

int check_rule(int64_t B, int64_t T, int64_t H, int64_t dk, int64_t dv, int dtype) {
  int s;
  if ((s = check_dtype(dtype))) return s;
  if (B < 0 || B > kMaxRows || T < 0 || H <= 0 || H > kMaxRows || B * H > kMaxRows || T > (1 << 30))
    return set_error(DYNCONV_ERR_SHAPE, "gated delta rule: bad sizes B=%lld T=%lld H=%lld", (long long)B, (long long)T,
                     (long long)H);
  return check_widths(dk, dv);
}

dr::View view(const void* p, const int64_t* strides, int i) {
  return dr::View{p, strides[3 * i], strides[3 * i + 1], strides[3 * i + 2]};
}

int pass_state(const float* in, float* out, int64_t n, cudaStream_t st) {
  if (!out || n == 0) return DYNCONV_OK;
  const cudaError_t e = in ? cudaMemcpyAsync(out, in, n * sizeof(float), cudaMemcpyDeviceToDevice, st)
                           : cudaMemsetAsync(out, 0, n * sizeof(float), st);
  return cuda_status(e, "gated delta rule state");
}

// Rows that tensor maps read have to lie at positive multiples of 16 bytes.
int check_rows(const char* name, const dr::View& v, int64_t B, int64_t T, int64_t H, int64_t width, int dtype) {
  const int elem = dtype == DYNCONV_DTYPE_F32 ? 4 : 2;
  if (width % (16 / elem) != 0 || dr::mappable(v, B, T, H, elem)) return DYNCONV_OK;
  return set_error(DYNCONV_ERR_ALIGN, "%s: rows of %lld numbers that do not lie at positive multiples of 16 bytes", name, (long long)width);
}

bool misaligned(const void* p) { return reinterpret_cast<uintptr_t>(p) & 15; }

int check_norm(int64_t rows, int64_t D, int dtype) {
  int s;
  if ((s = check_dtype(dtype))) return s;
  if (rows < 0 || rows > ((int64_t)1 << 40) || D < 1)
    return set_error(DYNCONV_ERR_SHAPE, "norm: bad sizes rows=%lld D=%lld", (long long)rows, (long long)D);
  if (D > norm::kMaxWidth) return set_error(DYNCONV_ERR_UNSUPPORTED, "norm: D=%lld (1..%d)", (long long)D, norm::kMaxWidth);
  return DYNCONV_OK;
}

// The gradient of a weight that no row contributes to.
int zero_sum(void* p, int64_t D, int dtype, bool w32, cudaStream_t st) {
  if (!p) return DYNCONV_OK;
  return cuda_status(cudaMemsetAsync(p, 0, D * (dtype == DYNCONV_DTYPE_BF16 && !w32 ? 2 : 4), st), "norm: gradient of no rows");
}

}  // namespace
}  // namespace dynconv

using namespace dynconv;

extern "C" {

int dynconv_delta_step(const void* q, const void* k, const void* v, const void* log_decay, const void* beta, float* state,
                       void* o, const void* slots, int slot_bytes, const int64_t* strides, int64_t B, int64_t n_rows,
                       int64_t H, int64_t dk, int64_t dv, float scale, int dtype, void* stream) {
  int s;
  const bool gates32 = take_f32(dtype);
  if ((s = op_entry((cudaStream_t)stream))) return s;
  if ((s = check_dtype(dtype))) return s;
  if (B < 0 || B > kMaxRows || H <= 0 || H > kMaxRows)
    return set_error(DYNCONV_ERR_SHAPE, "delta_step: bad sizes B=%lld H=%lld", (long long)B, (long long)H);
  if ((s = check_widths(dk, dv))) return s;
  if (slots && slot_bytes != 4 && slot_bytes != 8)
    return set_error(DYNCONV_ERR_ARGUMENT, "delta_step: slots of %d bytes (expected 4 or 8)", slot_bytes);
  if (n_rows < 0 || (!slots && n_rows < B))
    return set_error(DYNCONV_ERR_SHAPE, "delta_step: %lld rows of state for %lld rows of input", (long long)n_rows, (long long)B);
  if (B == 0) return DYNCONV_OK;
  if (!q || !k || !v || !log_decay || !beta || !o || !strides || (!state && n_rows > 0))
    return set_error(DYNCONV_ERR_ARGUMENT, "delta_step: null tensor");
  dr::Step p{};
  dr::View* views[5] = {&p.q, &p.k, &p.v, &p.g, &p.beta};
  const void* at[5] = {q, k, v, log_decay, beta};
  for (int i = 0; i < 5; ++i) *views[i] = dr::View{at[i], strides[2 * i], 0, strides[2 * i + 1]};
  p.gates32 = gates32, p.o = o, p.state = state, p.slots = slots, p.slot_bytes = slot_bytes;
  p.B = B, p.n_rows = n_rows, p.H = (int)H, p.dk = (int)dk, p.dv = (int)dv, p.scale = scale;
  return dr::step_launch(p, dtype, (cudaStream_t)stream);
}

size_t dynconv_delta_kept_bytes(int64_t B, int64_t T, int64_t H, int64_t dk, int64_t dv, int dtype) {
  take_f32(dtype);
  if (check_rule(B, T, H, dk, dv, dtype) || B * T == 0) return 0;
  const dr::Kept n = dr::kept_bytes(B, T, H, dk, dv, dtype);
  return n.states + n.rest;  // (both are multiples of 512)
}

size_t dynconv_delta_workspace_bytes(int64_t B, int64_t T, int64_t H, int64_t dk, int64_t dv, int dtype, int backward) {
  take_f32(dtype);
  if (check_rule(B, T, H, dk, dv, dtype) || B * T == 0) return 0;
  return dr::prepared_bytes(nullptr, nullptr, B, T, H, dk, dv, dtype, backward != 0) +
         (backward ? dynconv_delta_kept_bytes(B, T, H, dk, dv, dtype) : 0);
}

int dynconv_delta_fwd(const void* q, const void* k, const void* v, const void* log_decay, const void* beta,
                      const float* initial_state, void* o, float* final_state, void* kept, size_t kept_bytes,
                      const int64_t* strides, void* workspace, size_t workspace_bytes, int64_t B, int64_t T, int64_t H, int64_t dk,
                      int64_t dv, float scale, int dtype, void* stream) {
  int s;
  cudaStream_t st = (cudaStream_t)stream;
  const bool gates32 = take_f32(dtype);
  if ((s = op_entry(st))) return s;
  if ((s = check_rule(B, T, H, dk, dv, dtype))) return s;
  if (B * T == 0) return pass_state(initial_state, final_state, B * H * dk * dv, st);
  if (!q || !k || !v || !log_decay || !beta || !o || !strides) return set_error(DYNCONV_ERR_ARGUMENT, "delta_fwd: null tensor");
  const dr::Kept n = dr::kept_bytes(B, T, H, dk, dv, dtype);
  if (kept && kept_bytes < n.states + n.rest)
    return set_error(DYNCONV_ERR_WORKSPACE, "delta_fwd: kept %zu < %zu bytes", kept_bytes, n.states + n.rest);
  const size_t need = dr::prepared_bytes(nullptr, nullptr, B, T, H, dk, dv, dtype, false);
  if (!workspace || workspace_bytes < need)
    return set_error(DYNCONV_ERR_WORKSPACE, "delta_fwd: workspace %zu < %zu bytes", workspace_bytes, need);
  if (misaligned(kept) || misaligned(workspace))
    return set_error(DYNCONV_ERR_ALIGN, "delta_fwd: kept or the workspace is not 16-byte aligned");
  dr::Forward p{};
  p.q = view(q, strides, 0), p.k = view(k, strides, 1), p.v = view(v, strides, 2);
  p.g = view(log_decay, strides, 3), p.beta = view(beta, strides, 4), p.o = view(o, strides, 5);
  if ((s = check_rows("delta_fwd", p.q, B, T, H, dk, dtype)) || (s = check_rows("delta_fwd", p.k, B, T, H, dk, dtype)) ||
      (s = check_rows("delta_fwd", p.v, B, T, H, dv, dtype)))
    return s;
  dr::prepared_bytes(&p.pre, workspace, B, T, H, dk, dv, dtype, false);
  p.gates32 = gates32, p.s_in = initial_state, p.s_out = final_state;
  if (kept) p.states = (__nv_bfloat16*)kept, p.rest = (__nv_bfloat16*)((char*)kept + n.states);
  p.B = (int)B, p.H = (int)H, p.dk = (int)dk, p.dv = (int)dv, p.T = T, p.scale = scale;
  return dr::forward_launch(p, dtype, st);
}

int dynconv_delta_bwd(const void* q, const void* k, const void* log_decay, const void* beta, const void* kept,
                      size_t kept_bytes, const void* d_o, const float* d_final_state, void* dq, void* d_k, void* d_v,
                      void* d_log_decay, void* d_beta, float* d_initial_state, const int64_t* strides, void* workspace,
                      size_t workspace_bytes, int64_t B, int64_t T, int64_t H, int64_t dk, int64_t dv, float scale, int dtype,
                      void* stream) {
  int s;
  cudaStream_t st = (cudaStream_t)stream;
  const bool gates32 = take_f32(dtype);
  if ((s = op_entry(st))) return s;
  if ((s = check_rule(B, T, H, dk, dv, dtype))) return s;
  if (B * T == 0) return pass_state(d_final_state, d_initial_state, B * H * dk * dv, st);
  if (!q || !k || !log_decay || !beta || !kept || !d_o || !dq || !d_k || !d_v || !d_log_decay || !d_beta || !strides)
    return set_error(DYNCONV_ERR_ARGUMENT, "delta_bwd: null tensor");
  const dr::Kept n = dr::kept_bytes(B, T, H, dk, dv, dtype);
  const size_t kept_need = n.states + n.rest, pre = dr::prepared_bytes(nullptr, nullptr, B, T, H, dk, dv, dtype, true), need = pre + kept_need;
  if (kept_bytes < kept_need) return set_error(DYNCONV_ERR_WORKSPACE, "delta_bwd: kept %zu < %zu bytes", kept_bytes, kept_need);
  if (!workspace || workspace_bytes < need)
    return set_error(DYNCONV_ERR_WORKSPACE, "delta_bwd: workspace %zu < %zu bytes", workspace_bytes, need);
  if (misaligned(kept) || misaligned(workspace))
    return set_error(DYNCONV_ERR_ALIGN, "delta_bwd: kept or the workspace is not 16-byte aligned");
  dr::Backward p{};
  dr::View* views[10] = {&p.q, &p.k, &p.g, &p.beta, &p.d_o, &p.dq, &p.dk_, &p.dv_, &p.dg, &p.dbeta};
  const void* at[10] = {q, k, log_decay, beta, d_o, dq, d_k, d_v, d_log_decay, d_beta};
  for (int i = 0; i < 10; ++i) *views[i] = view(at[i], strides, i);
  p.states = (const __nv_bfloat16*)kept, p.rest = (const __nv_bfloat16*)((const char*)kept + n.states);
  if ((s = check_rows("delta_bwd", p.q, B, T, H, dk, dtype)) || (s = check_rows("delta_bwd", p.k, B, T, H, dk, dtype)) ||
      (s = check_rows("delta_bwd", p.d_o, B, T, H, dv, dtype)))
    return s;
  dr::prepared_bytes(&p.pre, workspace, B, T, H, dk, dv, dtype, true);
  p.dstates = (__nv_bfloat16*)((char*)workspace + pre), p.du = (__nv_bfloat16*)((char*)workspace + pre + n.states);
  p.gates32 = gates32, p.ds_out = d_final_state, p.ds_in = d_initial_state;
  p.B = (int)B, p.H = (int)H, p.dk = (int)dk, p.dv = (int)dv, p.T = T, p.scale = scale;
  return dr::backward_launch(p, dtype, st);
}

size_t dynconv_norm_workspace_bytes(int64_t D) {
  return D < 1 || D > norm::kMaxWidth ? 0 : (size_t)norm::partial_rows() * D * sizeof(float);
}

int dynconv_gated_norm_fwd(const void* x, const void* weight, const void* gate, void* y, const int64_t* strides, int64_t N,
                           int64_t G, int64_t D, float eps, float scale, int dtype, void* stream) {
  int s;
  const bool w32 = take_f32(dtype);
  if ((s = op_entry((cudaStream_t)stream))) return s;
  if (N < 0 || G < 0 || (G > 0 && N > ((int64_t)1 << 40) / G)) return set_error(DYNCONV_ERR_SHAPE, "gated_norm: bad sizes N=%lld G=%lld", (long long)N, (long long)G);
  if ((s = check_norm(N * G, D, dtype))) return s;
  if (N * G == 0) return DYNCONV_OK;
  if (!x || !y || !strides) return set_error(DYNCONV_ERR_ARGUMENT, "gated_norm: null tensor");
  norm::Gated p{};
  p.x = x, p.weight = weight, p.gate = gate, p.y = y;
  p.x_outer = strides[0], p.x_inner = strides[1], p.gate_outer = strides[2], p.gate_inner = strides[3];
  p.N = N, p.G = G, p.D = (int)D, p.eps = eps, p.scale = scale;
  return norm::gated_launch(p, dtype, w32, false, (cudaStream_t)stream);
}

int dynconv_gated_norm_bwd(const void* x, const void* weight, const void* gate, const void* dy, void* dx, void* dweight,
                           void* dgate, const int64_t* strides, void* workspace, size_t workspace_bytes, int64_t N, int64_t G,
                           int64_t D, float eps, float scale, int dtype, void* stream) {
  int s;
  cudaStream_t st = (cudaStream_t)stream;
  const bool w32 = take_f32(dtype);
  if ((s = op_entry(st))) return s;
  if (N < 0 || G < 0 || (G > 0 && N > ((int64_t)1 << 40) / G)) return set_error(DYNCONV_ERR_SHAPE, "gated_norm: bad sizes N=%lld G=%lld", (long long)N, (long long)G);
  if ((s = check_norm(N * G, D, dtype))) return s;
  if (N * G == 0) return zero_sum(dweight, D, dtype, w32, st);
  if (!x || !dy || !strides || (dweight && !weight) || (dgate && !gate)) return set_error(DYNCONV_ERR_ARGUMENT, "gated_norm: null tensor");
  if (dweight && (!workspace || workspace_bytes < dynconv_norm_workspace_bytes(D)))
    return set_error(DYNCONV_ERR_WORKSPACE, "gated_norm: workspace %zu < %zu bytes", workspace_bytes, dynconv_norm_workspace_bytes(D));
  norm::Gated p{};
  p.x = x, p.weight = weight, p.gate = gate, p.dy = dy, p.dx = dx, p.dgate = dgate, p.dweight = dweight;
  p.part = dweight ? (float*)workspace : nullptr;
  p.x_outer = strides[0], p.x_inner = strides[1], p.gate_outer = strides[2], p.gate_inner = strides[3];
  p.N = N, p.G = G, p.D = (int)D, p.eps = eps, p.scale = scale;
  return norm::gated_launch(p, dtype, w32, true, st);
}

int dynconv_residual_norm_fwd(const void* x, const void* residual, const void* weight, const void* scale, float factor, void* y,
                              void* h, int64_t N, int64_t D, float eps, int dtype, void* stream) {
  int s;
  const bool w32 = take_f32(dtype);
  if ((s = op_entry((cudaStream_t)stream))) return s;
  if ((s = check_norm(N, D, dtype))) return s;
  if (N == 0) return DYNCONV_OK;
  if (!x || !residual || !weight || !y || !h) return set_error(DYNCONV_ERR_ARGUMENT, "residual_norm: null tensor");
  norm::Residual p{};
  p.x = x, p.residual = residual, p.weight = weight, p.scale = scale, p.factor = factor, p.y = y, p.h = h;
  p.N = N, p.D = (int)D, p.eps = eps;
  return norm::residual_launch(p, dtype, w32, false, (cudaStream_t)stream);
}

int dynconv_residual_norm_bwd(const void* h, const void* x, const void* weight, const void* scale, float factor, const void* dy,
                              const void* dh, void* dx, void* dresidual, void* dweight, void* dscale, void* workspace,
                              size_t workspace_bytes, int64_t N, int64_t D, float eps, int dtype, void* stream) {
  int s;
  cudaStream_t st = (cudaStream_t)stream;
  const bool w32 = take_f32(dtype);
  if ((s = op_entry(st))) return s;
  if ((s = check_norm(N, D, dtype))) return s;
  if (N == 0) {
    if ((s = zero_sum(dweight, D, dtype, w32, st))) return s;
    return zero_sum(dscale, D, dtype, w32, st);
  }
  if (!h || !weight || (dscale && (!x || !scale))) return set_error(DYNCONV_ERR_ARGUMENT, "residual_norm: null tensor");
  const size_t one = dynconv_norm_workspace_bytes(D), need = one * ((dweight != nullptr) + (dscale != nullptr));
  if (need && (!workspace || workspace_bytes < need))
    return set_error(DYNCONV_ERR_WORKSPACE, "residual_norm: workspace %zu < %zu bytes", workspace_bytes, need);
  norm::Residual p{};
  p.h = (void*)h, p.x = x, p.weight = weight, p.scale = scale, p.factor = factor, p.dy = dy, p.dh = dh;
  p.dx = dx, p.dresidual = dresidual, p.dweight = dweight, p.dscale = dscale;
  p.part_w = dweight ? (float*)workspace : nullptr;
  p.part_s = dscale ? (float*)((char*)workspace + (dweight ? one : 0)) : nullptr;
  p.N = N, p.D = (int)D, p.eps = eps;
  return norm::residual_launch(p, dtype, w32, true, st);
}

}  // extern "C"
