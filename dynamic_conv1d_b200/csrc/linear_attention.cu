// linear_attention.cu -- linear attention with a decay for each head on the CUDA cores:
// the chunked kernels for fp32 and for shapes outside the tensor-core envelope, the scan
// over segment states, and the step for single tokens.  The formulas stand in
// linear_attention.cuh.
#include "linear_attention.cuh"

namespace dynconv {
namespace la {

namespace {

// ------------------------------------------------------------------ chunked, simple

constexpr int kC = 32;        // tokens of a chunk
constexpr int kSlice = 32;    // columns of w per CTA
constexpr int kThreads = 256;

__host__ __device__ constexpr size_t simple_smem_floats(int dx) {
  return (size_t)2 * kC * (dx + 1) + 2 * kC * (kC + 1) + (size_t)dx * (kSlice + 1) + kC + 1;
}

// One CTA runs one segment of one chain, chunk after chunk, with the state in shared
// memory.  state_only: the segment's own state from zero, into p.seg.
// Everything is fp32; each output is rounded once.
template <typename T>
__global__ void __launch_bounds__(kThreads) la_simple_kernel(const __grid_constant__ Params p, int n_slices,
                                                             int state_only) {
  extern __shared__ float sm[];
  int64_t id = blockIdx.x;
  const int slice = (int)(id % n_slices);
  id /= n_slices;
  const int64_t bh = id % ((int64_t)p.B * p.H);
  id /= (int64_t)p.B * p.H;
  const int seg = (int)(id % p.n_seg);
  const int ri = (int)(id / p.n_seg);
  const Role& ro = p.role[ri];
  const int dx = ro.dx, dw = ro.dw;
  const int c0 = slice * kSlice;
  if (c0 >= dw || (state_only && seg == p.n_seg - 1)) return;
  const int nc = min(kSlice, dw - c0);
  const int b = (int)(bh / p.H), h = (int)(bh % p.H);
  const int tid = threadIdx.x;

  float* xs = sm;                    // [kC][dx+1]
  float* ys = xs + kC * (dx + 1);    // [kC][dx+1]
  float* ws = ys + kC * (dx + 1);    // [kC][kC+1]
  float* as = ws + kC * (kC + 1);    // [kC][kC+1]
  float* S = as + kC * (kC + 1);     // [dx][kSlice+1]
  float* pw = S + dx * (kSlice + 1); // decay^0 .. decay^kC

  const double l2 = log2_decay(p.log_decay, h);
  if (tid <= kC) pw[tid] = (float)exp2(l2 * tid);
  const Factor f_full = decay_factor(l2, kC);
  const int64_t n_state = (int64_t)dx * dw;
  for (int i = tid; i < dx * kSlice; i += kThreads) {
    const int r = i / kSlice, c = i % kSlice;
    float v = 0.f;
    if (c < nc && !state_only) {
      if (p.n_seg > 1)
        v = seg_state(p, ri, seg, bh, n_state)[(int64_t)r * dw + c0 + c];
      else if (ro.s_in)
        v = ro.s_in[bh * n_state + (int64_t)r * ro.si + (int64_t)(c0 + c) * ro.sj];
    }
    S[r * (kSlice + 1) + c] = v;
  }

  const T* xp = (const T*)ro.x.p + b * ro.x.sb + h * ro.x.sh;
  const T* yp = (const T*)ro.y.p + b * ro.y.sb + h * ro.y.sh;
  const T* wp = (const T*)ro.w.p + b * ro.w.sb + h * ro.w.sh;
  T* op = (T*)ro.out.p + b * ro.out.sb + h * ro.out.sh;
  const int64_t n_chunks = (p.T + kC - 1) / kC;
  const int64_t first = (int64_t)seg * p.chunks_per_seg;
  const int64_t last = min(n_chunks, first + p.chunks_per_seg);
  const int e = ro.reverse ? 0 : 1;
  for (int64_t ch = first; ch < last; ++ch) {
    const int64_t a0 = ch * kC;  // scan position of the chunk's first token
    const int L = (int)min((int64_t)kC, p.T - a0);
    __syncthreads();
    for (int i = tid; i < kC * dx; i += kThreads) {
      const int r = i / dx, d = i - r * dx;
      const int64_t t = ro.reverse ? p.T - 1 - (a0 + r) : a0 + r;
      xs[r * (dx + 1) + d] = (r < L && !state_only) ? Elem<T>::to_f(xp[t * ro.x.st + d]) : 0.f;
      ys[r * (dx + 1) + d] = r < L ? Elem<T>::to_f(yp[t * ro.y.st + d]) : 0.f;
    }
    for (int i = tid; i < kC * kSlice; i += kThreads) {
      const int r = i / kSlice, c = i % kSlice;
      const int64_t t = ro.reverse ? p.T - 1 - (a0 + r) : a0 + r;
      ws[r * (kC + 1) + c] = (r < L && c < nc) ? Elem<T>::to_f(wp[t * ro.w.st + c0 + c]) : 0.f;
    }
    __syncthreads();
    if (!state_only) {
      // scores: thread (ty, tx) owns rows ty, ty+16 and columns tx, tx+16
      const int ty = tid >> 4, tx = tid & 15;
      float acc[2][2] = {};
      for (int d = 0; d < dx; ++d) {
        const float x0 = xs[ty * (dx + 1) + d], x1 = xs[(ty + 16) * (dx + 1) + d];
        const float y0 = ys[tx * (dx + 1) + d], y1 = ys[(tx + 16) * (dx + 1) + d];
        acc[0][0] = fmaf(x0, y0, acc[0][0]);
        acc[0][1] = fmaf(x0, y1, acc[0][1]);
        acc[1][0] = fmaf(x1, y0, acc[1][0]);
        acc[1][1] = fmaf(x1, y1, acc[1][1]);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int r = ty + 16 * i, c = tx + 16 * j;
          as[r * (kC + 1) + c] = c <= r ? acc[i][j] * pw[r - c] * ro.a_scale : 0.f;
        }
      __syncthreads();
      float o1[2][2] = {}, o2[2][2] = {};
      for (int j = 0; j < kC; ++j) {
        const float a_0 = as[ty * (kC + 1) + j], a_1 = as[(ty + 16) * (kC + 1) + j];
        const float w_0 = ws[j * (kC + 1) + tx], w_1 = ws[j * (kC + 1) + tx + 16];
        if (j <= ty) {  // a later token's w may be inf or NaN: not even times zero
          o1[0][0] = fmaf(a_0, w_0, o1[0][0]);
          o1[0][1] = fmaf(a_0, w_1, o1[0][1]);
        }
        if (j <= ty + 16) {
          o1[1][0] = fmaf(a_1, w_0, o1[1][0]);
          o1[1][1] = fmaf(a_1, w_1, o1[1][1]);
        }
      }
      for (int d = 0; d < dx; ++d) {
        const float x0 = xs[ty * (dx + 1) + d], x1 = xs[(ty + 16) * (dx + 1) + d];
        const float s0 = S[d * (kSlice + 1) + tx], s1 = S[d * (kSlice + 1) + tx + 16];
        o2[0][0] = fmaf(x0, s0, o2[0][0]);
        o2[0][1] = fmaf(x0, s1, o2[0][1]);
        o2[1][0] = fmaf(x1, s0, o2[1][0]);
        o2[1][1] = fmaf(x1, s1, o2[1][1]);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = ty + 16 * i;
        if (r >= L) continue;
        const int64_t t = ro.reverse ? p.T - 1 - (a0 + r) : a0 + r;
        const float f = ro.i_scale * pw[r + e];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int c = tx + 16 * j;
          if (c < nc) op[t * ro.out.st + c0 + c] = Elem<T>::from_f(fmaf(f, o2[i][j], o1[i][j]));
        }
      }
      __syncthreads();  // the state's readers are done
    }
    const int c = tid & 31;
    const Factor f = L == kC ? f_full : decay_factor(l2, L);
    for (int r = tid >> 5; r < dx; r += kThreads / 32) {
      float acc = 0.f;
      for (int j = 0; j < L; ++j)
        acc = fmaf(ys[j * (dx + 1) + r], ws[j * (kC + 1) + c] * pw[L - e - j], acc);
      S[r * (kSlice + 1) + c] = decay_add(f, S[r * (kSlice + 1) + c], ro.w_scale * acc);
    }
  }
  __syncthreads();
  const bool to_user = !state_only && seg == p.n_seg - 1 && ro.s_out;
  if (!state_only && !to_user) return;
  for (int i = tid; i < dx * kSlice; i += kThreads) {
    const int r = i / kSlice, c = i % kSlice;
    if (c >= nc) continue;
    const float v = S[r * (kSlice + 1) + c];
    if (state_only)
      seg_state(p, ri, seg, bh, n_state)[(int64_t)r * dw + c0 + c] = v;
    else
      ro.s_out[bh * n_state + (int64_t)r * ro.si + (int64_t)(c0 + c) * ro.sj] = v;
  }
}

// ----------------------------------------------------------------------------- scan

// In place over the segments of each (role, batch row, head): what segment s added to a
// state of zero becomes the state at its start.  One thread per state element; the next
// segment's value is loaded before the current one is used.
__global__ void __launch_bounds__(256) la_scan_kernel(const __grid_constant__ Params p, int chunk) {
  const Role& ro = p.role[blockIdx.z];
  const int64_t n_state = (int64_t)ro.dx * ro.dw;
  const int64_t bh = blockIdx.y;
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n_state) return;
  const int r = (int)(i / ro.dw), c = (int)(i % ro.dw);
  const Factor f = decay_factor(log2_decay(p.log_decay, (int)(bh % p.H)), (double)chunk * p.chunks_per_seg);
  float S = ro.s_in ? ro.s_in[bh * n_state + (int64_t)r * ro.si + (int64_t)c * ro.sj] : 0.f;
  float* s0 = seg_state(p, blockIdx.z, 0, bh, n_state) + i;
  const int64_t step = (int64_t)p.B * p.H * n_state;
  float own = *s0;
  for (int s = 0; s < p.n_seg; ++s) {
    const float next = s + 2 < p.n_seg ? s0[step] : 0.f;
    *s0 = S;
    S = decay_add(f, S, own);
    own = next;
    s0 += step;
  }
}

// ----------------------------------------------------------------------------- step

// One token: S <- g S + k v^T and o = scale * q S for SLICE columns of one row's and
// head's state.  Lanes own four neighbouring columns, the threads above them rows; all of
// the state's loads are issued before the first is used.
template <typename T, int SLICE, int VEC>
__global__ void __launch_bounds__(256) la_step_kernel(View q, View k, View v, float* state,
                                                      const float* __restrict__ log_decay, T* __restrict__ o,
                                                      const void* __restrict__ slots, int slot_bytes, int64_t n_rows,
                                                      int H, int dk, int dv, float scale) {
  constexpr int kLanes = SLICE / VEC;         // threads across a row
  constexpr int kRowGroups = 256 / kLanes;    // rows per pass
  __shared__ float ks[kMaxDim], qs[kMaxDim];
  __shared__ float part[kRowGroups][SLICE];
  const int h = blockIdx.y;
  const int64_t b = blockIdx.z;
  const int tid = threadIdx.x;
  const int64_t row = !slots ? b : slot_bytes == 8 ? static_cast<const int64_t*>(slots)[b] : static_cast<const int32_t*>(slots)[b];
  const bool live = row >= 0 && row < n_rows;
  const T* qp = (const T*)q.p + b * q.sb + h * q.sh;
  const T* kp = (const T*)k.p + b * k.sb + h * k.sh;
  const T* vp = (const T*)v.p + b * v.sb + h * v.sh;
  const int c = blockIdx.x * SLICE + (tid % kLanes) * VEC;
  const int rg = tid / kLanes;
  const bool in = live && c < dv;
  float* S = state + ((live ? row : 0) * H + h) * (int64_t)dk * dv + c;
  constexpr int kAhead = 4;  // state vectors in flight per thread
  float s[kAhead][VEC];
  auto load = [&](int r0) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int r = r0 + u * kRowGroups;
      if (in && r < dk) {
        if constexpr (VEC == 4) {
          const float4 f = *reinterpret_cast<const float4*>(S + (int64_t)r * dv);
          s[u][0] = f.x, s[u][1] = f.y, s[u][2] = f.z, s[u][3] = f.w;
        } else {
          s[u][0] = S[(int64_t)r * dv];
        }
      }
    }
  };
  load(rg);
  for (int i = tid; i < dk; i += 256) {
    ks[i] = Elem<T>::to_f(kp[i]);
    qs[i] = Elem<T>::to_f(qp[i]) * scale;
  }
  float vv[VEC], acc[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    vv[e] = c + e < dv ? Elem<T>::to_f(vp[c + e]) : 0.f;
    acc[e] = 0.f;
  }
  const float g = (float)exp2(log2_decay(log_decay, h));
  __syncthreads();
  for (int r0 = rg; r0 < dk; r0 += kAhead * kRowGroups) {
    if (r0 != rg) load(r0);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int r = r0 + u * kRowGroups;
      if (!in || r >= dk) continue;
      const float kr = ks[r], qr = qs[r];
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        s[u][e] = fmaf(g, s[u][e], kr * vv[e]);
        acc[e] = fmaf(qr, s[u][e], acc[e]);
      }
      if constexpr (VEC == 4)
        *reinterpret_cast<float4*>(S + (int64_t)r * dv) = make_float4(s[u][0], s[u][1], s[u][2], s[u][3]);
      else
        S[(int64_t)r * dv] = s[u][0];
    }
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e) part[rg][(tid % kLanes) * VEC + e] = acc[e];
  __syncthreads();
  for (int i = tid; i < SLICE; i += 256) {
    const int col = blockIdx.x * SLICE + i;
    if (col >= dv) continue;
    float sum = 0.f;
#pragma unroll 8
    for (int r = 0; r < kRowGroups; ++r) sum += part[r][i];
    o[(b * H + h) * dv + col] = Elem<T>::from_f(live ? sum : 0.f);
  }
}

template <typename T, int SLICE, int VEC>
int step_go(const View& q, const View& k, const View& v, float* state, const float* log_decay, void* o,
            const void* slots, int slot_bytes, int64_t B, int64_t n_rows, int H, int dk, int dv, float scale,
            cudaStream_t st) {
  const dim3 grid((unsigned)((dv + SLICE - 1) / SLICE), (unsigned)H, (unsigned)B);
  la_step_kernel<T, SLICE, VEC><<<grid, 256, 0, st>>>(q, k, v, state, log_decay, (T*)o, slots, slot_bytes, n_rows, H,
                                                      dk, dv, scale);
  DYNCONV_CHECK_LAUNCH("la_step_kernel");
  return DYNCONV_OK;
}

template <typename T>
int step_pick(const View& q, const View& k, const View& v, float* state, const float* log_decay, void* o,
              const void* slots, int slot_bytes, int64_t B, int64_t n_rows, int H, int dk, int dv, float scale,
              cudaStream_t st) {
  const bool vec = dv % 4 == 0 && (reinterpret_cast<uintptr_t>(state) & 15) == 0;
  if (!vec) return step_go<T, 32, 1>(q, k, v, state, log_decay, o, slots, slot_bytes, B, n_rows, H, dk, dv, scale, st);
  return step_go<T, 32, 4>(q, k, v, state, log_decay, o, slots, slot_bytes, B, n_rows, H, dk, dv, scale, st);
}

}  // namespace

int step_launch(const View& q, const View& k, const View& v, float* state, const float* log_decay, void* o,
                const void* slots, int slot_bytes, int64_t B, int64_t n_rows, int H, int dk, int dv, float scale,
                int dtype, cudaStream_t st) {
  if (dtype == DYNCONV_DTYPE_BF16)
    return step_pick<__nv_bfloat16>(q, k, v, state, log_decay, o, slots, slot_bytes, B, n_rows, H, dk, dv, scale, st);
  return step_pick<float>(q, k, v, state, log_decay, o, slots, slot_bytes, B, n_rows, H, dk, dv, scale, st);
}

int scan_launch(const Params& p, int chunk, cudaStream_t st) {
  const int64_t n = (int64_t)p.role[0].dx * p.role[0].dw;
  const dim3 grid((unsigned)((n + 255) / 256), (unsigned)(p.B * p.H), (unsigned)p.n_roles);
  la_scan_kernel<<<grid, 256, 0, st>>>(p, chunk);
  DYNCONV_CHECK_LAUNCH("la_scan_kernel");
  return DYNCONV_OK;
}

// Cuts chains until there are about four CTAs for each SM, with eight chunks at least in a segment.
void simple_plan(Params* p) {
  const int64_t chunks = (p->T + kC - 1) / kC;
  int64_t chains = 0;
  for (int r = 0; r < p->n_roles; ++r) chains += (int64_t)p->B * p->H * ((p->role[r].dw + kSlice - 1) / kSlice);
  int64_t seg = (4 * (int64_t)sm_count() + chains - 1) / chains;
  seg = seg < chunks / 8 ? seg : chunks / 8;
  if (seg < 1) seg = 1;
  p->chunks_per_seg = (int)((chunks + seg - 1) / seg);
  p->n_seg = (int)((chunks + p->chunks_per_seg - 1) / p->chunks_per_seg);
}

namespace {
template <typename T>
int simple_go(const Params& p, cudaStream_t st) {
  int dx = 0, dw = 0;
  for (int r = 0; r < p.n_roles; ++r) {
    dx = p.role[r].dx > dx ? p.role[r].dx : dx;
    dw = p.role[r].dw > dw ? p.role[r].dw : dw;
  }
  const size_t smem = simple_smem_floats(dx) * sizeof(float);
  cudaError_t e = cudaFuncSetAttribute(la_simple_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return cuda_status(e, "cudaFuncSetAttribute(la_simple)");
  }
  const int n_slices = (dw + kSlice - 1) / kSlice;
  const int64_t blocks = (int64_t)p.n_roles * p.n_seg * p.B * p.H * n_slices;
  if (blocks > INT32_MAX) return set_error(DYNCONV_ERR_SHAPE, "linear attention: B*H too large");
  if (p.n_seg > 1) {
    la_simple_kernel<T><<<(unsigned)blocks, kThreads, smem, st>>>(p, n_slices, 1);
    DYNCONV_CHECK_LAUNCH("la_simple_kernel (states)");
    int s = scan_launch(p, kC, st);
    if (s) return s;
  }
  la_simple_kernel<T><<<(unsigned)blocks, kThreads, smem, st>>>(p, n_slices, 0);
  DYNCONV_CHECK_LAUNCH("la_simple_kernel");
  return DYNCONV_OK;
}
}  // namespace

int simple_launch(const Params& p, int dtype, cudaStream_t st) {
  return dtype == DYNCONV_DTYPE_BF16 ? simple_go<__nv_bfloat16>(p, st) : simple_go<float>(p, st);
}

}  // namespace la
}  // namespace dynconv
