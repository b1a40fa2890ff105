// conv_step.cu -- one token of the dynamic short convolutions, on a cache of each
// sequence's last W-1 inputs (the single-token form of headwise.cu / lowrank_tc.cu).
//
//   lowrank : y[b,c] = sum_w (sum_r z[b,g,r] U[g,r,w,d] + static_w[g,w,d]) * past[w]
//   headwise: y[b,c] = sum_w (weight[b,d/hs,w] + static_w[w,d]) * past[w]
//
// with c = g*D + d, past[0] = x[b,c] and past[w] = cache[row, W-1-w, c] (the cache is in
// time order, oldest input first), then cache[row] drops its oldest input and takes x.
// `row` is b, or slots[b] when the rows' caches lie in a pool; a slot outside the pool
// leaves every cache alone and its output row is zero.
//
// A thread owns VEC neighbouring channels of RB batch rows: it alone reads and rewrites
// their cache, so the update in place needs no barrier.  Everything accumulates in
// fp32 and each output is rounded once.
#include "common.cuh"

namespace dynconv {

namespace {

constexpr int kThreads = 128;

__device__ __forceinline__ int64_t slot_of(const void* slots, int slot_bytes, int b) {
  if (!slots) return b;
  return slot_bytes == 8 ? static_cast<const int64_t*>(slots)[b] : static_cast<const int32_t*>(slots)[b];
}

template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T* p, float (&v)[VEC]) {
  if constexpr (VEC == 2 && sizeof(T) == 2) {
    const uint32_t u = *reinterpret_cast<const uint32_t*>(p);
    v[0] = __uint_as_float(u << 16);
    v[1] = __uint_as_float(u & 0xFFFF0000u);
  } else if constexpr (VEC == 2) {
    const float2 u = *reinterpret_cast<const float2*>(p);
    v[0] = u.x;
    v[1] = u.y;
  } else {
    v[0] = Elem<T>::to_f(*p);
  }
}

template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[VEC]) {
  if constexpr (VEC == 2 && sizeof(T) == 2) {
    *reinterpret_cast<uint32_t*>(p) = pack_bf16x2(v[0], v[1]);
  } else if constexpr (VEC == 2) {
    *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
  } else {
    *p = Elem<T>::from_f(v[0]);
  }
}

// Finishes one batch row of a thread's channels: taps -> y, and the cache moved on by one
// token.  C = channels of a row.
template <typename T, int W, int VEC>
__device__ __forceinline__ void finish_row(const T* x, T* cache, T* y, int64_t b, int64_t row, int64_t n_rows, int64_t C,
                                           int64_t c, const float (&taps)[W][VEC], int residual) {
  float out[VEC];
  if (row < 0 || row >= n_rows) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) out[e] = 0.f;
    store_vec<T, VEC>(y + b * C + c, out);
    return;
  }
  float past[W][VEC];
  load_vec<T, VEC>(x + b * C + c, past[0]);
  T* cr = cache + row * (int64_t)(W - 1) * C + c;
#pragma unroll
  for (int w = 1; w < W; ++w) load_vec<T, VEC>(cr + (int64_t)(W - 1 - w) * C, past[w]);
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    out[e] = residual ? past[0][e] : 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) out[e] = fmaf(taps[w][e], past[w][e], out[e]);
  }
  store_vec<T, VEC>(y + b * C + c, out);
#pragma unroll
  for (int w = 1; w < W; ++w) store_vec<T, VEC>(cr + (int64_t)(W - 1 - w) * C, past[w - 1]);
}

// Grid: (channel blocks, blocks of RB batch rows).  The thread keeps the W taps of its
// channels for RB rows in registers and walks the ranks once, so each U element is loaded
// once per RB rows; the rows' z sit in shared memory as fp32 (broadcast reads).
template <typename T, int W, int VEC, int RB>
__global__ void __launch_bounds__(kThreads) lr_step_kernel(const T* __restrict__ x, const T* __restrict__ z,
                                                           const T* __restrict__ U, const T* __restrict__ sw, T* cache,
                                                           T* __restrict__ y, const void* __restrict__ slots,
                                                           int slot_bytes, int64_t B, int64_t n_rows, int64_t D, int R,
                                                           int G, int residual) {
  extern __shared__ float zs[];  // [G*R][RB]
  const int64_t C = (int64_t)G * D;
  const int64_t b0 = (int64_t)blockIdx.y * RB;
  for (int i = threadIdx.x; i < G * R * RB; i += kThreads) {
    const int r = i / RB, j = i - r * RB;
    zs[i] = b0 + j < B ? Elem<T>::to_f(z[(b0 + j) * G * R + r]) : 0.f;
  }
  __syncthreads();
  const int64_t c = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * VEC;
  if (c >= C) return;
  const int64_t g = c / D, d = c - g * D;  // VEC divides D: a thread's channels share a group
  float taps[RB][W][VEC];
#pragma unroll
  for (int w = 0; w < W; ++w) {
    float s[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) s[e] = 0.f;
    if (sw) load_vec<T, VEC>(sw + (g * W + w) * D + d, s);
#pragma unroll
    for (int j = 0; j < RB; ++j)
#pragma unroll
      for (int e = 0; e < VEC; ++e) taps[j][w][e] = s[e];
  }
  const T* Ug = U + g * R * (int64_t)W * D + d;
  const float* zg = zs + g * R * RB;
#pragma unroll 4
  for (int r = 0; r < R; ++r) {
    float u[W][VEC];
#pragma unroll
    for (int w = 0; w < W; ++w) load_vec<T, VEC>(Ug + ((int64_t)r * W + w) * D, u[w]);
#pragma unroll
    for (int j = 0; j < RB; ++j) {
      const float zv = zg[r * RB + j];
#pragma unroll
      for (int w = 0; w < W; ++w)
#pragma unroll
        for (int e = 0; e < VEC; ++e) taps[j][w][e] = fmaf(zv, u[w][e], taps[j][w][e]);
    }
  }
#pragma unroll
  for (int j = 0; j < RB; ++j)
    if (b0 + j < B)
      finish_row<T, W, VEC>(x, cache, y, b0 + j, slot_of(slots, slot_bytes, (int)(b0 + j)), n_rows, C, c, taps[j],
                            residual);
}

// One batch row per blockIdx.y; the head's W weights are read by all its channels' threads
// (the same few cache lines).
template <typename T, int W, int VEC>
__global__ void __launch_bounds__(kThreads) hw_step_kernel(const T* __restrict__ x, const T* __restrict__ weight,
                                                           const T* __restrict__ sw, T* cache, T* __restrict__ y,
                                                           const void* __restrict__ slots, int slot_bytes,
                                                           int64_t n_rows, int64_t D, int64_t H, int residual) {
  const int64_t b = blockIdx.y;
  const int64_t c = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * VEC;
  if (c >= D) return;
  const int64_t hs = D / H;
  float taps[W][VEC];
#pragma unroll
  for (int w = 0; w < W; ++w) {
    float s[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) s[e] = 0.f;
    if (sw) load_vec<T, VEC>(sw + (int64_t)w * D + c, s);
#pragma unroll
    for (int e = 0; e < VEC; ++e) taps[w][e] = s[e] + Elem<T>::to_f(weight[(b * H + (c + e) / hs) * W + w]);
  }
  finish_row<T, W, VEC>(x, cache, y, b, slot_of(slots, slot_bytes, (int)b), n_rows, D, c, taps, residual);
}

struct StepArgs {
  const void *x, *z, *U, *sw;
  void *cache, *y;
  const void* slots;
  int slot_bytes;
  int64_t B, n_rows, D;
  int R, G, W, residual;
  cudaStream_t st;
};

template <typename T, int W, int VEC, int RB>
int lr_launch(const StepArgs& a) {
  const int64_t C = a.G * a.D;
  const dim3 grid((unsigned)((C / VEC + kThreads - 1) / kThreads), (unsigned)((a.B + RB - 1) / RB));
  const size_t smem = (size_t)a.G * a.R * RB * sizeof(float);
  lr_step_kernel<T, W, VEC, RB><<<grid, kThreads, smem, a.st>>>(
      (const T*)a.x, (const T*)a.z, (const T*)a.U, (const T*)a.sw, (T*)a.cache, (T*)a.y, a.slots, a.slot_bytes, a.B,
      a.n_rows, a.D, a.R, a.G, a.residual);
  DYNCONV_CHECK_LAUNCH("lr_step_kernel");
  return DYNCONV_OK;
}

template <typename T, int W>
int lr_pick(const StepArgs& a, bool pairs) {
  const bool many = a.B >= 4;
  if (pairs) return many ? lr_launch<T, W, 2, 8>(a) : lr_launch<T, W, 2, 1>(a);
  return many ? lr_launch<T, W, 1, 8>(a) : lr_launch<T, W, 1, 1>(a);
}

template <typename T, int W>
int hw_pick(const StepArgs& a, bool pairs) {
  const int vec = pairs ? 2 : 1;
  const dim3 grid((unsigned)((a.D / vec + kThreads - 1) / kThreads), (unsigned)a.B);
  if (pairs)
    hw_step_kernel<T, W, 2><<<grid, kThreads, 0, a.st>>>((const T*)a.x, (const T*)a.z, (const T*)a.sw, (T*)a.cache,
                                                         (T*)a.y, a.slots, a.slot_bytes, a.n_rows, a.D, a.R, a.residual);
  else
    hw_step_kernel<T, W, 1><<<grid, kThreads, 0, a.st>>>((const T*)a.x, (const T*)a.z, (const T*)a.sw, (T*)a.cache,
                                                         (T*)a.y, a.slots, a.slot_bytes, a.n_rows, a.D, a.R, a.residual);
  DYNCONV_CHECK_LAUNCH("hw_step_kernel");
  return DYNCONV_OK;
}

template <typename T>
int lr_width(const StepArgs& a, bool pairs) {
  switch (a.W) {
    case 1: return lr_pick<T, 1>(a, pairs);
    case 2: return lr_pick<T, 2>(a, pairs);
    case 3: return lr_pick<T, 3>(a, pairs);
    case 4: return lr_pick<T, 4>(a, pairs);
    case 5: return lr_pick<T, 5>(a, pairs);
    case 6: return lr_pick<T, 6>(a, pairs);
    case 7: return lr_pick<T, 7>(a, pairs);
    default: return lr_pick<T, 8>(a, pairs);
  }
}

template <typename T>
int hw_width(const StepArgs& a, bool pairs) {
  switch (a.W) {
    case 1: return hw_pick<T, 1>(a, pairs);
    case 2: return hw_pick<T, 2>(a, pairs);
    case 3: return hw_pick<T, 3>(a, pairs);
    case 4: return hw_pick<T, 4>(a, pairs);
    case 5: return hw_pick<T, 5>(a, pairs);
    case 6: return hw_pick<T, 6>(a, pairs);
    case 7: return hw_pick<T, 7>(a, pairs);
    default: return hw_pick<T, 8>(a, pairs);
  }
}

// Whether channel pairs can be read as one word: an even channel count and word-aligned tensors.
bool word_pairs(int64_t D, int dtype, const void* const* ptrs, int n) {
  const uintptr_t mask = dtype == DYNCONV_DTYPE_BF16 ? 3 : 7;
  if (D % 2 != 0) return false;
  for (int i = 0; i < n; ++i)
    if (reinterpret_cast<uintptr_t>(ptrs[i]) & mask) return false;
  return true;
}

}  // namespace

int lr_step_launch(const void* x, const void* z, const void* U, const void* sw, void* cache, void* y,
                   const void* slots, int slot_bytes, int64_t B, int64_t n_rows, int64_t D, int R, int W, int G,
                   int dtype, int residual, cudaStream_t st) {
  const StepArgs a{x, z, U, sw, cache, y, slots, slot_bytes, B, n_rows, D, R, G, W, residual, st};
  const void* ptrs[] = {x, U, sw, cache, y};
  const bool pairs = word_pairs(D, dtype, ptrs, 5);
  return dtype == DYNCONV_DTYPE_BF16 ? lr_width<__nv_bfloat16>(a, pairs) : lr_width<float>(a, pairs);
}

int hw_step_launch(const void* x, const void* weight, const void* sw, void* cache, void* y, const void* slots,
                   int slot_bytes, int64_t B, int64_t n_rows, int64_t D, int64_t H, int W, int dtype, int residual,
                   cudaStream_t st) {
  const StepArgs a{x, weight, nullptr, sw, cache, y, slots, slot_bytes, B, n_rows, D, (int)H, 1, W, residual, st};
  const void* ptrs[] = {x, sw, cache, y};
  const bool pairs = word_pairs(D, dtype, ptrs, 4);
  return dtype == DYNCONV_DTYPE_BF16 ? hw_width<__nv_bfloat16>(a, pairs) : hw_width<float>(a, pairs);
}

}  // namespace dynconv
