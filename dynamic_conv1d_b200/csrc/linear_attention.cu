// linear_attention.cu -- linear attention with a decay for each head on the CUDA cores:
// the chunked kernels for fp32 and for shapes outside the tensor-core envelope, the scan
// over segment states, and the step for single tokens.  The formulas stand in
// linear_attention.cuh.
#include "linear_attention.cuh"

namespace dynconv {
namespace la {

namespace {

// ------------------------------------------------------------------ chunked, CUDA cores

constexpr int kC = 32;        // tokens of a chunk
constexpr int kSlice = 32;    // columns of w per CTA
constexpr int kThreads = 256;
constexpr int kLd = kC + 4;   // pitch of the chunk x chunk and slice x chunk tiles

__host__ __device__ constexpr int row_pitch(int dx) { return (dx + 3) / 4 * 4 + 4; }  // of x, y and the state

__host__ __device__ constexpr size_t simple_smem_floats(int dx) {
  return (size_t)(2 * kC + kSlice) * row_pitch(dx) + 3 * kC * kLd + kC + 4;
}

__device__ __forceinline__ float4 f4(const float* p) { return *reinterpret_cast<const float4*>(p); }

__device__ __forceinline__ void dot4(float& acc, const float4& a, const float4& b) {
  acc = fmaf(a.x, b.x, acc);
  acc = fmaf(a.y, b.y, acc);
  acc = fmaf(a.z, b.z, acc);
  acc = fmaf(a.w, b.w, acc);
}

// One CTA runs one segment of one chain, chunk after chunk, with the state in shared
// memory.  state_only: the segment's own state from zero, into p.seg.
// Everything is fp32; each output is rounded once.  Every product runs along a dense dimension of
// both operands (w and the state are kept transposed), four elements per shared-memory read, and
// a thread owns 2 x 2 scores and outputs or 2 x 4 elements of the state.  Bound by the latency of a
// chunk's four phases: 2 x 512 tokens, 4 heads of 64 in fp32 take 24 us forward and 57 us backward
// (B200), cut into segments of one to two chunks.  Longer ones are far from the bytes' time: 4 x 4096
// tokens, 16 heads of 128 in fp32 2.4 and 6.4 ms (82 and 144 us), 8 heads of 256 in bf16 3.9 and 10.2 ms (41
// and 72 us).
template <typename T>
__global__ void __launch_bounds__(kThreads) la_simple_kernel(const __grid_constant__ Params p, int n_slices,
                                                             int state_only) {
  extern __shared__ __align__(16) float sm[];
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
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int ld = row_pitch(dx), d4 = (ld - 4) / 4;

  float* xs = sm;                // [kC][ld]
  float* ys = xs + kC * ld;      // [kC][ld]
  float* St = ys + kC * ld;      // [kSlice][ld]: the state, transposed
  float* wt = St + kSlice * ld;  // [kSlice][kLd]: w, transposed
  float* ht = wt + kC * kLd;     // [kSlice][kLd]: w weighted by the decays to the chunk's end
  float* as = ht + kC * kLd;     // [kC][kLd]: scores under the decay mask
  float* pw = as + kC * kLd;     // decay^0 .. decay^kC

  const double l2 = log2_decay(p.log_decay, h);
  if (tid <= kC) pw[tid] = (float)exp2(l2 * tid);
  const Factor f_full = decay_factor(l2, kC);
  const int64_t n_state = (int64_t)dx * dw;
  for (int r = warp; r < ld; r += kThreads / 32) {  // (columns beyond dx stay zero, here and in x and y)
    float v = 0.f;
    if (r < dx && lane < nc && !state_only) {
      if (p.n_seg > 1)
        v = seg_state(p, ri, seg, bh, n_state)[(int64_t)r * dw + c0 + lane];
      else if (ro.s_in)
        v = ro.s_in[bh * n_state + (int64_t)r * ro.si + (int64_t)(c0 + lane) * ro.sj];
    }
    St[lane * ld + r] = v;
  }
  for (int i = tid; i < 2 * kC * 4; i += kThreads) {  // (x and y are adjacent)
    const int r = i >> 2, c = (dx & ~3) + (i & 3);
    if (c < ld) xs[r * ld + c] = 0.f;
  }

  const T* xp = (const T*)ro.x.p + b * ro.x.sb + h * ro.x.sh;
  const T* yp = (const T*)ro.y.p + b * ro.y.sb + h * ro.y.sh;
  const T* wp = (const T*)ro.w.p + b * ro.w.sb + h * ro.w.sh + c0;
  T* op = (T*)ro.out.p + b * ro.out.sb + h * ro.out.sh + c0;
  const int64_t n_chunks = (p.T + kC - 1) / kC;
  const int64_t first = (int64_t)seg * p.chunks_per_seg;
  const int64_t last = min(n_chunks, first + p.chunks_per_seg);
  const int e = ro.reverse ? 0 : 1;
  const int ty = tid >> 4, tx = tid & 15;
  for (int64_t ch = first; ch < last; ++ch) {
    const int64_t a0 = ch * kC;  // scan position of the chunk's first token
    const int L = (int)min((int64_t)kC, p.T - a0);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kC / 8; ++i) {
      const int r = warp + i * 8;
      const int64_t t = ro.reverse ? p.T - 1 - (a0 + r) : a0 + r;
      for (int d = lane; d < dx; d += 32) {
        if (!state_only) xs[r * ld + d] = r < L ? Elem<T>::to_f(xp[t * ro.x.st + d]) : 0.f;
        ys[r * ld + d] = r < L ? Elem<T>::to_f(yp[t * ro.y.st + d]) : 0.f;
      }
      const float w = (r < L && lane < nc) ? Elem<T>::to_f(wp[t * ro.w.st + lane]) : 0.f;
      wt[lane * kLd + r] = w;
      ht[lane * kLd + r] = r < L ? w * pw[L - e - r] : 0.f;
    }
    __syncthreads();
    if (!state_only) {
      // scores, and the product with the state: thread (ty, tx) owns rows ty, ty+16, columns tx, tx+16
      float sc[2][2] = {}, o2[2][2] = {};
#pragma unroll 2
      for (int d = 0; d < d4; ++d) {
        const float4 x0 = f4(xs + ty * ld + 4 * d), x1 = f4(xs + (ty + 16) * ld + 4 * d);
        const float4 y0 = f4(ys + tx * ld + 4 * d), y1 = f4(ys + (tx + 16) * ld + 4 * d);
        const float4 s0 = f4(St + tx * ld + 4 * d), s1 = f4(St + (tx + 16) * ld + 4 * d);
        dot4(sc[0][0], x0, y0);
        dot4(sc[0][1], x0, y1);
        dot4(sc[1][0], x1, y0);
        dot4(sc[1][1], x1, y1);
        dot4(o2[0][0], x0, s0);
        dot4(o2[0][1], x0, s1);
        dot4(o2[1][0], x1, s0);
        dot4(o2[1][1], x1, s1);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int r = ty + 16 * i, c = tx + 16 * j;
          as[r * kLd + c] = c <= r ? sc[i][j] * pw[r - c] * ro.a_scale : 0.f;
        }
      __syncthreads();
      float o1[2][2] = {};
      for (int j = 0; j < kC; j += 4) {
        if (j > ty + 16) break;
        float4 w[2] = {f4(wt + tx * kLd + j), f4(wt + (tx + 16) * kLd + j)};
#pragma unroll
        for (int i = 1; i >= 0; --i) {
          const int r = ty + 16 * i;
          // a later token's w may be inf or NaN: not even times zero (row ty+16 first: it sees more)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            if (j + 0 > r) w[c].x = 0.f;
            if (j + 1 > r) w[c].y = 0.f;
            if (j + 2 > r) w[c].z = 0.f;
            if (j + 3 > r) w[c].w = 0.f;
          }
          const float4 a = f4(as + r * kLd + j);
          dot4(o1[i][0], a, w[0]);
          dot4(o1[i][1], a, w[1]);
        }
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
          if (c < nc) op[t * ro.out.st + c] = Elem<T>::from_f(fmaf(f, o2[i][j], o1[i][j]));
        }
      }
      // (the state's readers were done before the barrier above)
    }
    const Factor f = L == kC ? f_full : decay_factor(l2, L);
    for (int i = tid; i < d4 * 16; i += kThreads) {
      const int c = i & 15, d = (i >> 4) * 4;
      float4 acc[2] = {};
#pragma unroll 2
      for (int j = 0; j < kC; j += 4) {
        const float4 h0 = f4(ht + c * kLd + j), h1 = f4(ht + (c + 16) * kLd + j);
        const float hv[2][4] = {{h0.x, h0.y, h0.z, h0.w}, {h1.x, h1.y, h1.z, h1.w}};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float4 y = f4(ys + (j + k) * ld + d);
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            acc[m].x = fmaf(hv[m][k], y.x, acc[m].x);
            acc[m].y = fmaf(hv[m][k], y.y, acc[m].y);
            acc[m].z = fmaf(hv[m][k], y.z, acc[m].z);
            acc[m].w = fmaf(hv[m][k], y.w, acc[m].w);
          }
        }
      }
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        float* S = St + (c + 16 * m) * ld + d;
        float4 v = f4(S);
        v.x = decay_add(f, v.x, ro.w_scale * acc[m].x);
        v.y = decay_add(f, v.y, ro.w_scale * acc[m].y);
        v.z = decay_add(f, v.z, ro.w_scale * acc[m].z);
        v.w = decay_add(f, v.w, ro.w_scale * acc[m].w);
        *reinterpret_cast<float4*>(S) = v;
      }
    }
  }
  __syncthreads();
  const bool to_user = !state_only && seg == p.n_seg - 1 && ro.s_out;
  if ((!state_only && !to_user) || lane >= nc) return;
  for (int r = warp; r < dx; r += kThreads / 32) {
    const float v = St[lane * ld + r];
    if (state_only)
      seg_state(p, ri, seg, bh, n_state)[(int64_t)r * dw + c0 + lane] = v;
    else
      ro.s_out[bh * n_state + (int64_t)r * ro.si + (int64_t)(c0 + lane) * ro.sj] = v;
  }
}

// ----------------------------------------------------------------------------- scan

// In place over the segments of each (role, batch row, head): what segment s added to a
// state of zero becomes the state at its start.  One thread per state element; eight
// segments' values are under way before the first is used.
__global__ void __launch_bounds__(256) la_scan_kernel(const __grid_constant__ Params p, int chunk) {
  __shared__ Factor factor[2];  // over a whole segment, over the last
  const Role& ro = p.role[blockIdx.z];
  const int64_t n_state = (int64_t)ro.dx * ro.dw;
  const int64_t bh = blockIdx.y;
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (threadIdx.x < 2) {
    const double span = (double)chunk * p.chunks_per_seg;
    factor[threadIdx.x] = decay_factor(log2_decay(p.log_decay, (int)(bh % p.H)),
                                       threadIdx.x == 0 ? span : (double)p.T - span * (p.n_seg - 1));
  }
  __syncthreads();
  if (i >= n_state) return;
  const Factor f = factor[0];
  const int r = (int)(i / ro.dw), c = (int)(i % ro.dw);
  const int64_t at = bh * n_state + (int64_t)r * ro.si + (int64_t)c * ro.sj;
  const int own_segs = p.n_seg - (p.scan_final ? 0 : 1);  // segments that have left their own state
  float S = ro.s_in ? ro.s_in[at] : 0.f;
  float* s0 = seg_state(p, blockIdx.z, 0, bh, n_state) + i;
  const int64_t step = (int64_t)p.B * p.H * n_state;
  constexpr int kFly = 8;
  for (int s = 0; s < p.n_seg; s += kFly) {
    float own[kFly];
#pragma unroll
    for (int k = 0; k < kFly; ++k) own[k] = s + k < own_segs ? s0[(s + k) * step] : 0.f;
#pragma unroll
    for (int k = 0; k < kFly; ++k) {
      if (s + k >= p.n_seg) break;
      s0[(s + k) * step] = S;
      if (s + k + 1 < p.n_seg)
        S = decay_add(f, S, own[k]);
      else if (p.scan_final && ro.s_out)
        ro.s_out[at] = decay_add(factor[1], S, own[k]);
    }
  }
}

// ----------------------------------------------------------------------------- step

// One token: S <- g S + k v^T and o = scale * q S for SLICE columns of one row's and
// head's state.  Lanes own four neighbouring columns, the threads above them rows; all of
// the state's loads are issued before the first is used.  Bound by HBM: the state is read and
// written once (8 dk dv bytes per row and head).  128 rows x 32 heads x 128 x 128: 88 us, 6.1 TB/s
// (94% of the copy rate); one row of 16 heads 2.4 us, a launch's time.  Slices of 32 columns: four
// CTAs for each state of 128 x 128, so that one row already fills 64 SMs.
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

void plan_segments(Params* p, int chunk, int slice, int slots, double whole, double state_pass, double start,
                   double scan) {
  const int64_t chunks = (p->T + chunk - 1) / chunk;
  int64_t chains = 0;
  for (int r = 0; r < p->n_roles; ++r) chains += (int64_t)p->B * p->H * ((p->role[r].dw + slice - 1) / slice);
  double best = 1e300;
  p->n_seg = 1, p->chunks_per_seg = (int)chunks;
  for (int64_t want = 1; want <= 64 && want <= chunks; ++want) {
    const int64_t per = (chunks + want - 1) / want, seg = (chunks + per - 1) / per;
    double cost = (double)((chains * seg + slots - 1) / slots) * ((double)per * (seg > 1 ? 1.0 : whole) + start);
    const int64_t first = seg - (p->scan_final ? 0 : 1);  // segments of the state pass
    if (seg > 1) cost += (double)((chains * first + slots - 1) / slots) * ((double)per * state_pass + start) + scan;
    if (cost < best) {
      best = cost;
      p->n_seg = (int)seg, p->chunks_per_seg = (int)per;
    }
  }
}

// Measured at 64 x 64: a chunk 4 us, of the state pass 2.5 us, 4 us to start, 4 us for the scan; four CTAs per SM.
void simple_plan(Params* p) { plan_segments(p, kC, kSlice, 4 * sm_count(), 1.0, 0.6, 1.0, 1.0); }

namespace {
template <typename T>
int simple_go(const Params& p, cudaStream_t st) {
  int dx = 0, dw = 0;
  for (int r = 0; r < p.n_roles; ++r) {
    dx = p.role[r].dx > dx ? p.role[r].dx : dx;
    dw = p.role[r].dw > dw ? p.role[r].dw : dw;
  }
  const size_t smem = simple_smem_floats(dx) * sizeof(float);
  constexpr int kMost = (int)(simple_smem_floats(kMaxDim) * sizeof(float));
  if (int s = allow_shared(la_simple_kernel<T>, kMost, "cudaFuncSetAttribute(la_simple)")) return s;
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
