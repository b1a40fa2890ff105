// delta_step.cu -- one token of the gated delta rule for each of B sequences:
//     S <- a S + k u^T,  u = beta (v - a S^T k),  o = scale S^T q
// The output needs no second look at the state: S^T q = a S_old^T q + (k . q) u, so one pass over the
// old state gives both S_old^T k and S_old^T q, one exchange through shared memory adds them up, and
// the state is written from registers.
//
// Bound by HBM: 8 dk dv bytes per row and head.  Slices of 16 columns, so that one row of 16 heads of
// 128 x 128 already fills 128 SMs, and many small CTAs, whose loads, exchanges and stores overlap; a thread
// holds up to 16 numbers of the state, all loaded before the first is used.
#include "delta_rule.cuh"

namespace dynconv {
namespace dr {
namespace {

constexpr int kThreads = 128, kSlice = 16;

template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads, 10) delta_step_kernel(Step p) {
  constexpr int kLanes = kSlice / VEC;           // threads across a row
  constexpr int kGroups = kThreads / kLanes;     // rows at a time
  constexpr int kRows = kMaxKey / kGroups;       // rows per thread
  __shared__ float ks[kMaxKey], qs[kMaxKey];
  __shared__ float part_k[kThreads / 32][kSlice], part_q[kThreads / 32][kSlice], dot[kThreads / 32];
  const int h = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t b = blockIdx.z;
  const int64_t row = !p.slots ? b : p.slot_bytes == 8 ? static_cast<const int64_t*>(p.slots)[b] : static_cast<const int32_t*>(p.slots)[b];
  const bool live = row >= 0 && row < p.n_rows;
  const int at = (tid % kLanes) * VEC, c = blockIdx.x * kSlice + at, group = tid / kLanes;
  const bool in = live && c < p.dv;
  float* S = p.state + ((live ? row : 0) * p.H + h) * (int64_t)p.dk * p.dv + c;
  float s[kRows][VEC];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int r = group + i * kGroups;
#pragma unroll
    for (int e = 0; e < VEC; ++e) s[i][e] = 0.f;
    if (in && r < p.dk) {
      if constexpr (VEC == 4) {
        const float4 f = *reinterpret_cast<const float4*>(S + (int64_t)r * p.dv);
        s[i][0] = f.x, s[i][1] = f.y, s[i][2] = f.z, s[i][3] = f.w;
      } else {
        s[i][0] = S[(int64_t)r * p.dv];
      }
    }
  }
  const T* q = (const T*)p.q.p + b * p.q.sb + h * p.q.sh;
  const T* k = (const T*)p.k.p + b * p.k.sb + h * p.k.sh;
  const T* v = (const T*)p.v.p + b * p.v.sb + h * p.v.sh;
  const float g = Elem<T>::to_f(((const T*)p.g.p)[b * p.g.sb + h * p.g.sh]);
  const float beta = Elem<T>::to_f(((const T*)p.beta.p)[b * p.beta.sb + h * p.beta.sh]);
  float vv[VEC], kq = 0.f;
#pragma unroll
  for (int e = 0; e < VEC; ++e) vv[e] = c + e < p.dv ? Elem<T>::to_f(v[c + e]) : 0.f;
  if (tid < kMaxKey) {  // (four whole warps)
    const float x = tid < p.dk ? Elem<T>::to_f(k[tid]) : 0.f, y = tid < p.dk ? Elem<T>::to_f(q[tid]) : 0.f;
    ks[tid] = x, qs[tid] = y;
    kq = x * y;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) kq += __shfl_xor_sync(0xffffffffu, kq, d);
    if (lane == 0) dot[warp] = kq;
  }
  __syncthreads();
  float sk[VEC], sq[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) sk[e] = sq[e] = 0.f;
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const float kr = ks[group + i * kGroups], qr = qs[group + i * kGroups];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      sk[e] = fmaf(kr, s[i][e], sk[e]);
      sq[e] = fmaf(qr, s[i][e], sq[e]);
    }
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
#pragma unroll
    for (int d = kLanes; d < 32; d <<= 1) {
      sk[e] += __shfl_xor_sync(0xffffffffu, sk[e], d);
      sq[e] += __shfl_xor_sync(0xffffffffu, sq[e], d);
    }
    if (lane < kLanes) part_k[warp][at + e] = sk[e], part_q[warp][at + e] = sq[e];
  }
  __syncthreads();
  const float a = expf(g);
  kq = dot[0] + dot[1] + dot[2] + dot[3];
  float u[VEC], o[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    float x = 0.f, y = 0.f;
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) x += part_k[i][at + e], y += part_q[i][at + e];
    u[e] = beta * fmaf(-a, x, vv[e]);
    o[e] = p.scale * fmaf(a, y, kq * u[e]);
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int r = group + i * kGroups;
    if (!in || r >= p.dk) continue;
    const float kr = ks[r];
#pragma unroll
    for (int e = 0; e < VEC; ++e) s[i][e] = fmaf(a, s[i][e], kr * u[e]);
    if constexpr (VEC == 4)
      *reinterpret_cast<float4*>(S + (int64_t)r * p.dv) = make_float4(s[i][0], s[i][1], s[i][2], s[i][3]);
    else
      S[(int64_t)r * p.dv] = s[i][0];
  }
  if (group == 0) {
    T* to = (T*)p.o + (b * p.H + h) * p.dv + c;
#pragma unroll
    for (int e = 0; e < VEC; ++e)
      if (c + e < p.dv) to[e] = Elem<T>::from_f(live ? o[e] : 0.f);
  }
}

template <typename T>
int go(const Step& p, cudaStream_t st) {
  const dim3 grid((unsigned)((p.dv + kSlice - 1) / kSlice), (unsigned)p.H, (unsigned)p.B);
  if (p.dv % 4 == 0 && (reinterpret_cast<uintptr_t>(p.state) & 15) == 0)
    delta_step_kernel<T, 4><<<grid, kThreads, 0, st>>>(p);
  else
    delta_step_kernel<T, 1><<<grid, kThreads, 0, st>>>(p);
  DYNCONV_CHECK_LAUNCH("delta_step_kernel");
  return DYNCONV_OK;
}

}  // namespace

int step_launch(const Step& p, int dtype, cudaStream_t st) {
  return dtype == DYNCONV_DTYPE_BF16 ? go<__nv_bfloat16>(p, st) : go<float>(p, st);
}

}  // namespace dr
}  // namespace dynconv
