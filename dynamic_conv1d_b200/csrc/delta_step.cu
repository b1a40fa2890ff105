// delta_step.cu -- one token of the gated delta rule for each of B sequences:
//     S <- a S + k u^T,  u = beta (v - a S^T k),  o = scale S^T q
// The output needs no second look at the state: S^T q = a S_old^T q + (k . q) u, so one pass over the
// old state gives both S_old^T k and S_old^T q, one exchange through shared memory adds them up, and
// the state is written from registers.
//
// Bound by HBM: 8 dk dv bytes per row and head.  CTAs of 128 threads take 16 columns (32 of up to 64 rows), so
// that one row of 16 heads of 128 x 128 already fills 128 SMs, and loads, exchanges and stores of many CTAs
// overlap; a thread holds up to 16 numbers of the state, all loaded before the first is used.
// 256 rows of 16 heads of 128 x 128: 91 us, 5.87 TB/s (98 us with the sums exchanged whole: 24 shuffles for 16
// numbers took a third of the shared memory's time); 512 rows of 64 x 64: 46 us, 5.8 TB/s (76 us in the CTAs of
// the larger states, half of whose rows are empty); 127 columns, 4 bytes at a time: 100 us; one row: 2.1 us.
#include "delta_rule.cuh"

namespace dynconv {
namespace dr {
namespace {

constexpr int kThreads = 128;

// Columns of a CTA.
__host__ __device__ constexpr int slice(int keys) { return 16 * kMaxKey / keys; }
// CTAs per SM, with a few registers spilled (9 and 8 without: 97 and 113 us in the first and third case above)
__host__ __device__ constexpr int ctas(int vec) { return vec == 4 ? 10 : 9; }

template <typename T, typename GT, int VEC, int KEYS>
__global__ void __launch_bounds__(kThreads, ctas(VEC)) delta_step_kernel(Step p) {
  constexpr int kSlice = slice(KEYS);
  constexpr int kLanes = kSlice / VEC;           // threads across a row
  constexpr int kGroups = kThreads / kLanes;     // rows at a time
  constexpr int kRows = KEYS / kGroups;          // rows per thread
  __shared__ float2 keys[KEYS];                                     // k, q
  __shared__ __align__(16) float part[kThreads / 32][2][kSlice];  // a warp's sums of S^T k, S^T q
  __shared__ float dot[KEYS / 32];
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
  const float g = Elem<GT>::to_f(((const GT*)p.g.p)[b * p.g.sb + h * p.g.sh]);
  const float beta = Elem<GT>::to_f(((const GT*)p.beta.p)[b * p.beta.sb + h * p.beta.sh]);
  float vv[VEC], kq = 0.f;
#pragma unroll
  for (int e = 0; e < VEC; ++e) vv[e] = c + e < p.dv ? Elem<T>::to_f(v[c + e]) : 0.f;
  if (tid < KEYS) {  // (whole warps)
    const float x = tid < p.dk ? Elem<T>::to_f(k[tid]) : 0.f, y = tid < p.dk ? Elem<T>::to_f(q[tid]) : 0.f;
    keys[tid] = make_float2(x, y);
    kq = x * y;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) kq += __shfl_xor_sync(0xffffffffu, kq, d);
    if (lane == 0) dot[warp] = kq;
  }
  __syncthreads();
  float sum[2 * VEC];
#pragma unroll
  for (int e = 0; e < 2 * VEC; ++e) sum[e] = 0.f;
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const float2 x = keys[group + i * kGroups];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      sum[e] = fmaf(x.x, s[i][e], sum[e]);
      sum[VEC + e] = fmaf(x.y, s[i][e], sum[VEC + e]);
    }
  }
  // over the warp's rows, half of the sums going to either lane of a pair: 7 exchanges, not 24, and each lane ends with
  // its own (6, and two)
#pragma unroll
  for (int d = 16, n = VEC; d >= kLanes; d >>= 1, n >>= 1) {
    const bool upper = lane & d;
#pragma unroll
    for (int e = 0; e < n; ++e) {
      const float mine = upper ? sum[n + e] : sum[e], other = upper ? sum[e] : sum[n + e];
      sum[e] = mine + __shfl_xor_sync(0xffffffffu, other, d);
    }
  }
  if constexpr (kSlice == 16)
    part[warp][lane >> 4][at + (VEC == 4 ? lane >> 2 & 3 : 0)] = sum[0];
  else if constexpr (VEC == 4)
    *reinterpret_cast<float2*>(&part[warp][lane >> 4][at + (lane >> 2 & 2)]) = make_float2(sum[0], sum[1]);
  else
    part[warp][0][at] = sum[0], part[warp][1][at] = sum[1];
  __syncthreads();
  const float a = expf(g);
  kq = KEYS == 64 ? dot[0] + dot[1] : dot[0] + dot[1] + dot[KEYS / 32 - 2] + dot[KEYS / 32 - 1];
  float u[VEC], o[VEC], x[VEC], y[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) x[e] = y[e] = 0.f;
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i)
    if constexpr (VEC == 4) {
      const float4 m = *reinterpret_cast<const float4*>(&part[i][0][at]), n = *reinterpret_cast<const float4*>(&part[i][1][at]);
      x[0] += m.x, x[1] += m.y, x[2] += m.z, x[3] += m.w;
      y[0] += n.x, y[1] += n.y, y[2] += n.z, y[3] += n.w;
    } else {
      x[0] += part[i][0][at], y[0] += part[i][1][at];
    }
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    u[e] = beta * fmaf(-a, x[e], vv[e]);
    o[e] = p.scale * fmaf(a, y[e], kq * u[e]);
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int r = group + i * kGroups;
    if (!in || r >= p.dk) continue;
    const float kr = keys[r].x;
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

template <typename T, typename GT, int VEC, int KEYS>
void launch(const Step& p, cudaStream_t st) {
  const dim3 grid((unsigned)((p.dv + slice(KEYS) - 1) / slice(KEYS)), (unsigned)p.H, (unsigned)p.B);
  delta_step_kernel<T, GT, VEC, KEYS><<<grid, kThreads, 0, st>>>(p);
}

template <typename T, typename GT>
int go(const Step& p, cudaStream_t st) {
  if (p.dv % 4 == 0 && (reinterpret_cast<uintptr_t>(p.state) & 15) == 0)
    p.dk <= 64 ? launch<T, GT, 4, 64>(p, st) : launch<T, GT, 4, kMaxKey>(p, st);
  else
    p.dk <= 64 ? launch<T, GT, 1, 64>(p, st) : launch<T, GT, 1, kMaxKey>(p, st);
  DYNCONV_CHECK_LAUNCH("delta_step_kernel");
  return DYNCONV_OK;
}

}  // namespace

int step_launch(const Step& p, int dtype, cudaStream_t st) {
  if (dtype != DYNCONV_DTYPE_BF16) return go<float, float>(p, st);
  return p.gates32 ? go<__nv_bfloat16, float>(p, st) : go<__nv_bfloat16, __nv_bfloat16>(p, st);
}

}  // namespace dr
}  // namespace dynconv
