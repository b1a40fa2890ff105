// api_lm.cu -- extern "C" entry points of the operators around the convolutions: steps of
// one token, linear attention with decay, and the vocabulary loss (declared in
// include/dynconv.h).  Like api.cu it validates, carves the caller's workspace and
// dispatches; it allocates nothing and never synchronises.
#include <algorithm>

#include "common.cuh"
#include "linear_attention.cuh"
#include "vocab_loss.cuh"

namespace dynconv {

int lr_step_launch(const void* x, const void* z, const void* U, const void* sw, void* cache, void* y,
                   const void* slots, int slot_bytes, int64_t B, int64_t n_rows, int64_t D, int R, int W, int G,
                   int dtype, int residual, cudaStream_t st);
int hw_step_launch(const void* x, const void* weight, const void* sw, void* cache, void* y, const void* slots,
                   int slot_bytes, int64_t B, int64_t n_rows, int64_t D, int64_t H, int W, int dtype, int residual,
                   cudaStream_t st);

namespace {

constexpr int64_t kMaxRows = 65535;  // batch rows of a step call, and B*H of an attention call (grid limits)

size_t align_up(size_t v) { return (v + 255) / 256 * 256; }

int check_step(int64_t B, int64_t n_rows, int64_t D, int64_t W, const void* slots, int slot_bytes, int dtype) {
  int s;
  if ((s = check_dtype(dtype))) return s;
  if (B < 0 || B > kMaxRows || D <= 0 || D > INT32_MAX / 16)
    return set_error(DYNCONV_ERR_SHAPE, "step: bad sizes B=%lld D=%lld", (long long)B, (long long)D);
  if (W < 1 || W > 8) return set_error(DYNCONV_ERR_UNSUPPORTED, "W=%lld not supported (1..8)", (long long)W);
  if (slots && slot_bytes != 4 && slot_bytes != 8)
    return set_error(DYNCONV_ERR_ARGUMENT, "step: slots of %d bytes (expected 4 or 8)", slot_bytes);
  if (n_rows < 0 || (!slots && n_rows < B))
    return set_error(DYNCONV_ERR_SHAPE, "step: %lld rows of cache for %lld rows of input", (long long)n_rows,
                     (long long)B);
  return DYNCONV_OK;
}

int check_attention(int64_t B, int64_t T, int64_t H, int64_t dk, int64_t dv, int dtype) {
  int s;
  if ((s = check_dtype(dtype))) return s;
  if (B < 0 || T < 0 || H <= 0 || B * H > kMaxRows || T > (1 << 30))
    return set_error(DYNCONV_ERR_SHAPE, "linear attention: bad sizes B=%lld T=%lld H=%lld", (long long)B, (long long)T,
                     (long long)H);
  if (dk < 1 || dk > la::kMaxDim || dv < 1 || dv > la::kMaxDim)
    return set_error(DYNCONV_ERR_UNSUPPORTED, "linear attention: dk=%lld dv=%lld (1..%d)", (long long)dk, (long long)dv,
                     la::kMaxDim);
  return DYNCONV_OK;
}

la::View view(const void* p, const int64_t* strides, int i) {
  return la::View{p, strides[3 * i], strides[3 * i + 1], strides[3 * i + 2]};
}

// Contiguous states of an empty sequence: the state passes through.
int pass_state(const float* in, float* out, int64_t n, cudaStream_t st) {
  if (!out || n == 0) return DYNCONV_OK;
  const cudaError_t e = in ? cudaMemcpyAsync(out, in, n * sizeof(float), cudaMemcpyDeviceToDevice, st)
                           : cudaMemsetAsync(out, 0, n * sizeof(float), st);
  return cuda_status(e, "linear attention state");
}

la::Params la_forward_params(int64_t B, int64_t T, int64_t H, int64_t dk, int64_t dv, float scale) {
  la::Params p{};
  p.n_roles = 1;
  p.B = (int)B, p.H = (int)H, p.T = T;
  la::Role& r = p.role[0];
  r.dx = (int)dk, r.dw = (int)dv, r.si = (int)dv, r.sj = 1;
  r.reverse = 0, r.a_scale = r.i_scale = scale, r.w_scale = 1.f;
  return p;
}

// Roles 0, 1, 2: dq, dk, dv (see linear_attention.cuh).
la::Params la_backward_params(int64_t B, int64_t T, int64_t H, int64_t dk, int64_t dv, float scale) {
  la::Params p{};
  p.n_roles = 3;
  p.B = (int)B, p.H = (int)H, p.T = T;
  la::Role &q = p.role[0], &k = p.role[1], &v = p.role[2];
  q.dx = (int)dv, q.dw = (int)dk, q.si = 1, q.sj = (int)dv;
  q.reverse = 0, q.a_scale = q.i_scale = scale, q.w_scale = 1.f;
  k.dx = (int)dv, k.dw = (int)dk, k.si = 1, k.sj = (int)dv;
  k.reverse = 1, k.a_scale = scale, k.i_scale = 1.f, k.w_scale = scale;
  v.dx = (int)dk, v.dw = (int)dv, v.si = (int)dv, v.sj = 1;
  v.reverse = 1, v.a_scale = scale, v.i_scale = 1.f, v.w_scale = scale;
  return p;
}

size_t la_seg_bytes(const la::Params& p) {
  if (p.n_seg <= 1) return 0;
  return align_up((size_t)p.n_roles * p.n_seg * p.B * p.H * p.role[0].dx * p.role[0].dw * sizeof(float));
}

int la_run(la::Params& p, int dtype, void* ws, size_t ws_bytes, cudaStream_t st) {
  const bool tc = la::tc_supported(p, dtype);
  tc ? la::tc_plan(&p, la::wants_states(p)) : la::simple_plan(&p);
  const size_t need = la_seg_bytes(p);
  if (need && (!ws || ws_bytes < need))
    return set_error(DYNCONV_ERR_WORKSPACE, "linear attention: workspace %zu < %zu bytes", ws_bytes, need);
  p.seg = (float*)ws;
  return tc ? la::tc_launch(p, st) : la::simple_launch(p, dtype, st);
}

int check_loss(int64_t N, int64_t D, int64_t V, int reduction, int dtype) {
  int s;
  reduction &= ~vl::kKeepRows;
  if ((s = check_dtype(dtype))) return s;
  if (N < 0 || D < 1 || V < 1 || N > (1 << 30) || D > INT32_MAX / 16 || V > (int64_t)1 << 22)
    return set_error(DYNCONV_ERR_SHAPE, "vocabulary loss: bad sizes N=%lld D=%lld V=%lld", (long long)N, (long long)D,
                     (long long)V);
  if (reduction < vl::kNone || reduction > vl::kMean)
    return set_error(DYNCONV_ERR_ARGUMENT, "vocabulary loss: reduction %d (none=0, sum=1, mean=2; +4: lse and the rows' losses)", reduction);
  return DYNCONV_OK;
}

bool misaligned(const void* p) { return reinterpret_cast<uintptr_t>(p) & 15; }

struct LossBackwardBytes {
  size_t piece, acc_h, acc_w, hidden_copy, weight_copy;
  size_t total() const { return piece + acc_h + acc_w + hidden_copy + weight_copy; }
};

LossBackwardBytes loss_backward_bytes(const vl::Plan& pl, int64_t N, int64_t D, int dtype, int want_hidden,
                                      int want_weight) {
  const bool copy = vl::copied(D, dtype);
  const size_t elem = 2 * vl::parts_of(dtype);
  const int64_t ld = copy ? vl::copy_pitch(D) : D;
  LossBackwardBytes b;
  b.hidden_copy = copy || want_weight ? align_up(vl::copy_bytes(N, D, dtype)) : 0;
  b.weight_copy = copy ? align_up(vl::copy_bytes(pl.piece, D, dtype)) : 0;
  b.piece = align_up((size_t)N * pl.pitch * elem);
  b.acc_h = want_hidden ? align_up((size_t)pl.z_h * N * ld * sizeof(float)) : 0;
  b.acc_w = want_weight && (pl.z_w > 1 || (copy && dtype == DYNCONV_DTYPE_BF16)) ? align_up((size_t)pl.z_w * pl.piece * ld * sizeof(float)) : 0;
  return b;
}

}  // namespace
}  // namespace dynconv

using namespace dynconv;

extern "C" {

int dynconv_lr_step(const void* x, const void* z, const void* U, const void* static_w, void* cache, void* y,
                    const void* slots, int slot_bytes, int64_t B, int64_t n_rows, int64_t D, int64_t R, int64_t W,
                    int64_t G, int dtype, int residual, void* stream) {
  int s;
  if ((s = op_entry((cudaStream_t)stream))) return s;
  if ((s = check_step(B, n_rows, D, W, slots, slot_bytes, dtype))) return s;
  if (R < 1 || R > 64) return set_error(DYNCONV_ERR_UNSUPPORTED, "lr_step: R=%lld (1..64)", (long long)R);
  if (G < 1 || G > 16) return set_error(DYNCONV_ERR_SHAPE, "lr_step: G=%lld (1..16)", (long long)G);
  if (B == 0) return DYNCONV_OK;
  if (!x || !z || !U || !y || (!cache && W > 1)) return set_error(DYNCONV_ERR_ARGUMENT, "lr_step: null tensor");
  return lr_step_launch(x, z, U, static_w, cache, y, slots, slot_bytes, B, n_rows, D, (int)R, (int)W, (int)G, dtype,
                        residual, (cudaStream_t)stream);
}

int dynconv_hw_step(const void* x, const void* weight, const void* static_w, void* cache, void* y, const void* slots,
                    int slot_bytes, int64_t B, int64_t n_rows, int64_t D, int64_t H, int64_t W, int dtype,
                    int residual, void* stream) {
  int s;
  if ((s = op_entry((cudaStream_t)stream))) return s;
  if ((s = check_step(B, n_rows, D, W, slots, slot_bytes, dtype))) return s;
  if (H <= 0 || D % H != 0)
    return set_error(DYNCONV_ERR_SHAPE, "D=%lld must be divisible by H=%lld", (long long)D, (long long)H);
  if (B == 0) return DYNCONV_OK;
  if (!x || !weight || !y || (!cache && W > 1)) return set_error(DYNCONV_ERR_ARGUMENT, "hw_step: null tensor");
  return hw_step_launch(x, weight, static_w, cache, y, slots, slot_bytes, B, n_rows, D, H, (int)W, dtype, residual,
                        (cudaStream_t)stream);
}

size_t dynconv_la_workspace_bytes(int64_t B, int64_t T, int64_t H, int64_t dk, int64_t dv, int dtype, int backward) {
  if (check_attention(B, T, H, dk, dv, dtype) || B * T == 0) return 0;
  la::Params p = backward ? la_backward_params(B, T, H, dk, dv, 1.f) : la_forward_params(B, T, H, dk, dv, 1.f);
  // strides, alignment and the states wanted decide the path and the cut at the call: enough for each
  la::simple_plan(&p);
  const size_t simple = la_seg_bytes(p);
  la::tc_plan(&p, false);
  const size_t tc = la_seg_bytes(p);
  la::tc_plan(&p, true);
  const size_t tc_states = la_seg_bytes(p);
  return std::max(simple, std::max(tc, tc_states));
}

int dynconv_la_fwd(const void* q, const void* k, const void* v, const float* log_decay, const float* initial_state,
                   void* o, float* final_state, const int64_t* strides, void* workspace, size_t workspace_bytes,
                   int64_t B, int64_t T, int64_t H, int64_t dk, int64_t dv, float scale, int dtype, void* stream) {
  int s;
  cudaStream_t st = (cudaStream_t)stream;
  if ((s = op_entry(st))) return s;
  if ((s = check_attention(B, T, H, dk, dv, dtype))) return s;
  if (B * T == 0) return pass_state(initial_state, final_state, B * H * dk * dv, st);
  if (!q || !k || !v || !log_decay || !o || !strides) return set_error(DYNCONV_ERR_ARGUMENT, "la_fwd: null tensor");
  la::Params p = la_forward_params(B, T, H, dk, dv, scale);
  p.log_decay = log_decay;
  la::Role& r = p.role[0];
  r.x = view(q, strides, 0), r.y = view(k, strides, 1), r.w = view(v, strides, 2), r.out = view(o, strides, 3);
  r.s_in = initial_state, r.s_out = final_state;
  return la_run(p, dtype, workspace, workspace_bytes, st);
}

int dynconv_la_bwd(const void* q, const void* k, const void* v, const float* log_decay, const float* initial_state,
                   const void* d_o, const float* d_final_state, void* dq, void* dk_, void* dv_, float* d_initial_state,
                   const int64_t* strides, void* workspace, size_t workspace_bytes, int64_t B, int64_t T, int64_t H,
                   int64_t dk, int64_t dv, float scale, int dtype, void* stream) {
  int s;
  cudaStream_t st = (cudaStream_t)stream;
  if ((s = op_entry(st))) return s;
  if ((s = check_attention(B, T, H, dk, dv, dtype))) return s;
  if (B * T == 0) return pass_state(d_final_state, d_initial_state, B * H * dk * dv, st);
  if (!q || !k || !v || !log_decay || !d_o || !dq || !dk_ || !dv_ || !strides)
    return set_error(DYNCONV_ERR_ARGUMENT, "la_bwd: null tensor");
  la::Params p = la_backward_params(B, T, H, dk, dv, scale);
  p.log_decay = log_decay;
  const la::View vq = view(q, strides, 0), vk = view(k, strides, 1), vv = view(v, strides, 2),
                 vo = view(d_o, strides, 3);
  la::Role &rq = p.role[0], &rk = p.role[1], &rv = p.role[2];
  rq.x = vo, rq.y = vv, rq.w = vk, rq.out = view(dq, strides, 4), rq.s_in = initial_state;
  rk.x = vv, rk.y = vo, rk.w = vq, rk.out = view(dk_, strides, 5), rk.s_in = d_final_state;
  rv.x = vk, rv.y = vq, rv.w = vo, rv.out = view(dv_, strides, 6), rv.s_in = d_final_state;
  rv.s_out = d_initial_state;
  return la_run(p, dtype, workspace, workspace_bytes, st);
}

int dynconv_la_step(const void* q, const void* k, const void* v, float* state, const float* log_decay, void* o,
                    const void* slots, int slot_bytes, const int64_t* strides, int64_t B, int64_t n_rows, int64_t H,
                    int64_t dk, int64_t dv, float scale, int dtype, void* stream) {
  int s;
  if ((s = op_entry((cudaStream_t)stream))) return s;
  if ((s = check_step(B, n_rows, 1, 1, slots, slot_bytes, dtype))) return s;
  if ((s = check_attention(0, 1, H, dk, dv, dtype))) return s;
  if (H > kMaxRows) return set_error(DYNCONV_ERR_SHAPE, "la_step: H=%lld", (long long)H);
  if (B == 0) return DYNCONV_OK;
  if (!q || !k || !v || !state || !log_decay || !o || !strides)
    return set_error(DYNCONV_ERR_ARGUMENT, "la_step: null tensor");
  const la::View vq{q, strides[0], 0, strides[1]}, vk{k, strides[2], 0, strides[3]}, vv{v, strides[4], 0, strides[5]};
  return la::step_launch(vq, vk, vv, state, log_decay, o, slots, slot_bytes, B, n_rows, (int)H, (int)dk, (int)dv,
                         scale, dtype, (cudaStream_t)stream);
}

size_t dynconv_vocab_loss_fwd_workspace_bytes(int64_t N, int64_t D, int64_t V, int dtype) {
  if (check_loss(N, D, V, 0, dtype)) return 0;
  const int64_t tiles = (V + vl::kTileColumns - 1) / vl::kTileColumns + 1;  // (an even number is written)
  const int64_t rows = std::min(N, vl::kRowsAtOnce);
  size_t n = align_up((size_t)tiles * rows * sizeof(float2)) + align_up((size_t)N * sizeof(float));
  if (vl::copied(D, dtype))
    n += align_up(vl::copy_bytes(rows, D, dtype)) + align_up(vl::copy_bytes(vl::words_at_once(D, V, dtype), D, dtype));
  return n;
}

int dynconv_vocab_loss_fwd(const void* hidden, const void* weight, const int64_t* target, float* loss, float* lse,
                           float* stats, void* workspace, size_t workspace_bytes, int64_t N, int64_t D, int64_t V,
                           int64_t ignore_index, int reduction, int dtype, void* stream) {
  int s;
  cudaStream_t st = (cudaStream_t)stream;
  if ((s = op_entry(st))) return s;
  if ((s = check_loss(N, D, V, reduction, dtype))) return s;
  const bool keep = reduction & vl::kKeepRows;
  reduction &= ~vl::kKeepRows;
  if (!stats || (!loss && (N > 0 || reduction != vl::kNone)))
    return set_error(DYNCONV_ERR_ARGUMENT, "vocab_loss_fwd: null loss or stats");
  vl::Problem p{};
  p.hidden = hidden, p.weight = weight, p.target = target;
  p.N = N, p.D = D, p.V = V, p.ignore = ignore_index, p.reduction = reduction;
  p.lse = lse, p.row_loss = keep && lse ? lse + N : nullptr, p.loss = loss, p.stats = stats, p.st = st;
  if (N == 0) return vl::total_launch(p);
  if (!hidden || !weight || !target || !lse) return set_error(DYNCONV_ERR_ARGUMENT, "vocab_loss_fwd: null tensor");
  const size_t need = dynconv_vocab_loss_fwd_workspace_bytes(N, D, V, dtype);
  if (!workspace || workspace_bytes < need)
    return set_error(DYNCONV_ERR_WORKSPACE, "vocab_loss_fwd: workspace %zu < %zu bytes", workspace_bytes, need);
  if (misaligned(workspace) ||
      (!vl::copied(D, dtype) && (misaligned(hidden) || misaligned(weight))))
    return set_error(DYNCONV_ERR_ALIGN, "vocab_loss_fwd: workspace or bf16 tensor not 16-byte aligned");
  p.tgt = (float*)workspace;
  p.part = (float2*)((char*)workspace + align_up((size_t)N * sizeof(float)));
  if (vl::copied(D, dtype)) {  // (the copies end the workspace)
    const size_t words = align_up(vl::copy_bytes(vl::words_at_once(D, V, dtype), D, dtype));
    const size_t rows = align_up(vl::copy_bytes(std::min(N, vl::kRowsAtOnce), D, dtype));
    p.weight_copy = (__nv_bfloat16*)((char*)workspace + need - words);
    p.hidden_copy = (__nv_bfloat16*)((char*)workspace + need - words - rows);
  }
  return vl::forward(p, dtype);
}

size_t dynconv_vocab_loss_bwd_workspace_bytes(int64_t N, int64_t D, int64_t V, int dtype, int want_dhidden,
                                              int want_dweight) {
  if (check_loss(N, D, V, 0, dtype) || N == 0) return 0;
  return loss_backward_bytes(vl::plan(N, D, V, dtype), N, D, dtype, want_dhidden, want_dweight).total();
}

int dynconv_vocab_loss_bwd(const void* hidden, const void* weight, const int64_t* target, const float* lse,
                           const float* stats, const float* dloss, void* dhidden, void* dweight, void* workspace,
                           size_t workspace_bytes, int64_t N, int64_t D, int64_t V, int64_t ignore_index,
                           int reduction, int dtype, void* stream) {
  int s;
  cudaStream_t st = (cudaStream_t)stream;
  if ((s = op_entry(st))) return s;
  if ((s = check_loss(N, D, V, reduction, dtype))) return s;
  if (!dhidden && !dweight) return DYNCONV_OK;
  if (N == 0) {
    if (!dweight) return DYNCONV_OK;
    return cuda_status(cudaMemsetAsync(dweight, 0, (size_t)V * D * (dtype == DYNCONV_DTYPE_BF16 ? 2 : 4), st),
                       "vocab_loss_bwd memset");
  }
  if (!hidden || !weight || !target || !lse || !stats || !dloss)
    return set_error(DYNCONV_ERR_ARGUMENT, "vocab_loss_bwd: null tensor");
  vl::Problem p{};
  p.hidden = hidden, p.weight = weight, p.target = target;
  p.N = N, p.D = D, p.V = V, p.ignore = ignore_index, p.reduction = reduction & ~vl::kKeepRows;
  p.row_loss = reduction & vl::kKeepRows ? const_cast<float*>(lse) + N : nullptr;
  p.lse = const_cast<float*>(lse), p.stats = const_cast<float*>(stats), p.dloss = dloss;
  p.dhidden = dhidden, p.dweight = dweight, p.st = st;
  p.piece = workspace;
  const vl::Plan pl = vl::plan(N, D, V, dtype);
  const LossBackwardBytes b = loss_backward_bytes(pl, N, D, dtype, dhidden != nullptr, dweight != nullptr);
  if (!workspace || workspace_bytes < b.total())
    return set_error(DYNCONV_ERR_WORKSPACE, "vocab_loss_bwd: workspace %zu < %zu bytes", workspace_bytes, b.total());
  if (misaligned(workspace) ||
      (!vl::copied(D, dtype) && (misaligned(hidden) || misaligned(weight) || misaligned(dhidden) || misaligned(dweight))))
    return set_error(DYNCONV_ERR_ALIGN, "vocab_loss_bwd: workspace or bf16 tensor not 16-byte aligned");
  p.acc_h = (float*)((char*)workspace + b.piece);
  p.acc_w = (float*)((char*)workspace + b.piece + b.acc_h);
  p.hidden_copy = (__nv_bfloat16*)((char*)workspace + b.piece + b.acc_h + b.acc_w);
  p.weight_copy = (__nv_bfloat16*)((char*)p.hidden_copy + b.hidden_copy);
  return vl::backward(p, pl, dtype);
}

}  // extern "C"
