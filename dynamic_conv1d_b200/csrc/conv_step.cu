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
// A thread owns neighbouring channels of its batch rows: it alone reads and rewrites their
// cache, so the update in place needs no barrier (the few-rows kernel reads all of it before
// one).  Everything accumulates in fp32 and each output is rounded once.
//
// Measured (B200, graph replay): one row of 3 x 2048 channels at rank 15 2.3 us, a launch's time; 512
// such rows 9.2 us; 256 rows of 3 x 4096 at rank 31 13.4 us with the tensors in L2 and 18.5 us
// from HBM, where their 53 MB take 8.2 us.  What holds it there is the schedule: 1536 blocks at five per SM are
// 2.08 rounds, the third for 56 of them, and a block goes through its phases (slots, then
// caches; U's tile; products; stores) one after the other with only four others to fill the gaps.  W = 8: 256 rows of 3 x 2048 at rank 15 9.6 us,
// 512 rows of 3 x 4096 at rank 31 51 us (30 and 191 on the CUDA cores, which keep the widest filters
// with more than 47 ranks).  fp32 stays on the CUDA cores: 256 rows of 3 x 4096 at rank 31 52 us, W = 8 and 512
// rows 195 us (floors 16 and 64).  Headwise, 64 rows of 2048: 2.4 us; 512 rows of 8192 channels from HBM 20 us in
// bf16 (10.3 at the copy rate), 24.5 us in fp32 (20.8).
#include "common.cuh"

namespace dynconv {

namespace {

constexpr int kThreads = 128;
// The CUDA-core path runs a block per row with its taps in parallel up to this many rows, as long as
// the rows' loads of U (G D / VEC x R W for each) stay below this number; blocks of eight rows read U
// an eighth as often but take longer to start.  Measured per row / in eights, fp32 (us): 3 x 2048 at rank
// 15, W = 4: 1 row 2.5 / 6.0, 16 5.2 / 7.8, 32 8.1 / 7.9, 64 14.0 / 8.5; 3 x 4096 at rank 31, W = 8: 1 row 3.7 /
// 10.1, 4 7.7 / 11.1, 8 13.2 / 13.0, 20 29 / 13.6; 512 at rank 7: 64 rows 2.8 / 5.8.
constexpr int kFewRows = 64;
constexpr int64_t kFewLoads = 6 << 20;

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

// Few rows outside the tensor-core form: the time is the latency of the loads, so each warp takes one
// tap and all its ranks' loads are in flight at once; the taps' products meet in shared memory.  Block: W warps of 32
// channel vectors, one batch row.
template <typename T, int W, int VEC>
__global__ void __launch_bounds__(32 * W) lr_step_few_kernel(const T* __restrict__ x, const T* __restrict__ z,
                                                             const T* __restrict__ U, const T* __restrict__ sw, T* cache,
                                                             T* __restrict__ y, const void* __restrict__ slots,
                                                             int slot_bytes, int64_t n_rows, int64_t D, int R, int G,
                                                             int residual) {
  __shared__ float part[W][32 * VEC];
  __shared__ float zs[64];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t C = (int64_t)G * D, b = blockIdx.y;
  const int64_t per = (D / VEC + 31) / 32;  // blocks of a group
  const int64_t g = blockIdx.x / per;
  const int64_t d = ((blockIdx.x - g * per) * 32 + lane) * VEC, c = g * D + d;
  const int64_t row = slot_of(slots, slot_bytes, (int)b);
  const bool in = d < D, live = row >= 0 && row < n_rows;
  const T* Ug = U + (g * R * W + w) * D + d;
  constexpr int kFly = 16;
  float u[kFly][VEC];
  auto fetch = [&](int r0) {
#pragma unroll
    for (int i = 0; i < kFly; ++i)
      if (in && r0 + i < R) load_vec<T, VEC>(Ug + (int64_t)(r0 + i) * W * D, u[i]);
  };
  fetch(0);
  float past[VEC], next[VEC], tap[VEC];  // this tap's input, and the one that takes its place
  T* cr = cache + (live ? row : 0) * (int64_t)(W - 1) * C + c;
#pragma unroll
  for (int e = 0; e < VEC; ++e) past[e] = next[e] = tap[e] = 0.f;
  if (in && live) {
    const T* xr = x + b * C + c;
    load_vec<T, VEC>(w == 0 ? xr : cr + (int64_t)(W - 1 - w) * C, past);
    if (w > 0) load_vec<T, VEC>(w == 1 ? xr : cr + (int64_t)(W - w) * C, next);
  }
  if (in && sw) load_vec<T, VEC>(sw + (g * W + w) * D + d, tap);
  for (int r = threadIdx.x; r < R; r += 32 * W) zs[r] = Elem<T>::to_f(z[(b * G + g) * R + r]);
  __syncthreads();  // (also: every cache row has been read before one is written)
  for (int r0 = 0; r0 < R; r0 += kFly) {
    if (r0 > 0) fetch(r0);
#pragma unroll
    for (int i = 0; i < kFly; ++i)
      if (in && r0 + i < R) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) tap[e] = fmaf(zs[r0 + i], u[i][e], tap[e]);
      }
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e) part[w][lane * VEC + e] = live ? tap[e] * past[e] : 0.f;  // (z of a padding row may be anything)
  if (in && live && w > 0) store_vec<T, VEC>(cr + (int64_t)(W - 1 - w) * C, next);
  __syncthreads();
  if (w != 0 || !in) return;
  float out[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    out[e] = residual ? past[e] : 0.f;
#pragma unroll
    for (int k = 0; k < W; ++k) out[e] += part[k][lane * VEC + e];
  }
  store_vec<T, VEC>(y + b * C + c, out);
}

// bf16, whole 16-byte groups of channels: the taps are a small matrix product (rows x ranks
// by ranks x channels), 2 R operations for each byte of the batch: on the CUDA cores 53 us for
// 256 rows of 3 x 4096 channels at R = 31, so it goes to the tensor cores.  mma.sync is the
// fitting form here: a warp's 16 x 32 outputs are consumed in registers by the convolution
// itself, K is R <= 64, and the tensor pipe is 10% busy.  One row takes no longer than in the
// few-rows form (2.3 against 2.5 us), so every batch goes this way.
//
// Block: 32 channels of one group, four warps with 16 rows each, U's tile staged once for 64
// rows, the static filter in it as one more rank whose z is one.  Channels are staged
// permuted, so that a thread's four column pairs are eight neighbouring channels: one
// 16-byte access per row and tensor.  (64 channels and 128 or 256 rows per block measured
// 10 to 25% longer.)
constexpr int kMmaRows = 64, kMmaCh = 32, kMmaThreads = 128;
// us[w][k / 2][position] = channels' (U[k], U[k + 1]) pairs: B fragments are single words.
// Row pitch 40 words: the four k rows that a fragment load touches lie 8 banks apart.
constexpr int kPitch = 40;
// Shared memory of the tiles of U and z: wide filters with many ranks do not fit.
constexpr bool mma_fits(int W, int KS) {
  return (W * KS * 8 * kPitch + (KS == 1 ? 4 : 64) * (KS * 8 + 4)) * 4 <= 48 * 1024;
}

__device__ __forceinline__ void mma_16n8k16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
      "%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void unpack8(const uint4& u, float (&v)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}

template <int W, int KS>
__global__ void __launch_bounds__(kMmaThreads, W > 4 ? 3 : KS == 1 ? 6 : 5) lr_step_mma_kernel(const __nv_bfloat16* __restrict__ x,
                                                          const __nv_bfloat16* __restrict__ z,
                                                          const __nv_bfloat16* __restrict__ U,
                                                          const __nv_bfloat16* __restrict__ sw, __nv_bfloat16* cache,
                                                          __nv_bfloat16* __restrict__ y, const void* __restrict__ slots,
                                                          int slot_bytes, int64_t B, int64_t n_rows, int64_t D, int R,
                                                          int G, int residual) {
  constexpr int K2 = KS * 8;
  __shared__ uint32_t us[W * K2 * kPitch];
  __shared__ uint32_t zs[4][KS == 1 ? 1 : 16][K2 + 4];  // each warp's rows of z (pitch: 8 rows meet no bank twice)
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t C = (int64_t)G * D;
  const int64_t per = (D + kMmaCh - 1) / kMmaCh;
  const int64_t g = blockIdx.x / per, d0 = (blockIdx.x - g * per) * kMmaCh;
  const int r0 = lane >> 2, q = lane & 3;
  const int64_t d = d0 + q * 8, c = g * D + d;
  const int64_t b0 = (int64_t)blockIdx.y * kMmaRows + warp * 16;
  // this thread's inputs and caches, under way while U is staged and multiplied
  uint4 past[2][W];
  int64_t rows[2];
#pragma unroll
  for (int hf = 0; hf < 2; ++hf) {
    const int64_t b = b0 + r0 + hf * 8;
    rows[hf] = -1;
#pragma unroll
    for (int w = 0; w < W; ++w) past[hf][w] = make_uint4(0, 0, 0, 0);
    if (b >= B || d >= D) continue;
    const int64_t row = slot_of(slots, slot_bytes, (int)b);
    if (row < 0 || row >= n_rows) continue;
    rows[hf] = row;
    const __nv_bfloat16* cr = cache + row * (int64_t)(W - 1) * C + c;
    past[hf][0] = *reinterpret_cast<const uint4*>(x + b * C + c);
#pragma unroll
    for (int w = 1; w < W; ++w) past[hf][w] = *reinterpret_cast<const uint4*>(cr + (int64_t)(W - 1 - w) * C);
  }
  // z; rank R is the static filter's, with a z of one.  Up to 16 ranks a thread loads its fragment's
  // elements itself; above, a lane takes a rank of each of the warp's rows (whole lines) and the
  // fragments come out of shared memory (256 rows, 3 x 4096 channels, rank 31: 18.7 against
  // 20.4 us; at rank 15, 3 x 2048 channels, 7.5 against 5.6).
  constexpr bool kDirect = KS == 1;
  constexpr int kHalves = (KS + 1) / 2;
  const uint16_t one = sw ? 0x3F80 : 0;
  uint32_t a[KS][4];
  uint16_t zv[kDirect ? 1 : 16][kHalves];
  if constexpr (kDirect) {
    const uint16_t* zr = reinterpret_cast<const uint16_t*>(z) + ((b0 + r0) * G + g) * R;
    const int64_t eight = (int64_t)8 * G * R;
    const bool there[2] = {b0 + r0 < B, b0 + r0 + 8 < B};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int k = q * 2 + (i >> 1) * 8;
      const uint16_t* at = zr + (i & 1) * eight + k;
      uint32_t lo = k == R ? one : 0, hi = k + 1 == R ? one : 0;
      if (there[i & 1] && k < R) lo = at[0];
      if (there[i & 1] && k + 1 < R) hi = at[1];
      a[0][i] = lo | (hi << 16);
    }
  } else {
#pragma unroll
    for (int r = 0; r < 16; ++r)
#pragma unroll
      for (int h = 0; h < kHalves; ++h) {
        const int k = h * 32 + lane;
        zv[r][h] = k == R ? one : 0;
        if (b0 + r < B && k < R) zv[r][h] = reinterpret_cast<const uint16_t*>(z)[((b0 + r) * G + g) * R + k];
      }
  }
  // stage U: a thread takes 8 channels of a rank pair; position of channel c in the tile:
  // column pair j = (c % 8) / 2 of thread c / 8 is column 2 (c / 8) + c % 2 of product j
#pragma unroll
  for (int n = 0; n < (W * K2 * 4 + kMmaThreads - 1) / kMmaThreads; ++n) {
    const int i = threadIdx.x + n * kMmaThreads;
    if (W * K2 * 4 % kMmaThreads != 0 && i >= W * K2 * 4) break;
    const int oct = i & 3, rest = i >> 2, k2 = rest % K2, w = rest / K2;
    const int64_t du = d0 + oct * 8;
    uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
    const __nv_bfloat16* src = U + ((g * R + 2 * k2) * W + w) * D + du;
    const __nv_bfloat16* st = sw + (g * W + w) * D + du;
    if (du < D && 2 * k2 < R) lo = *reinterpret_cast<const uint4*>(src);
    if (du < D && 2 * k2 + 1 < R) hi = *reinterpret_cast<const uint4*>(src + (int64_t)W * D);
    if (du < D && sw && 2 * k2 == R) lo = *reinterpret_cast<const uint4*>(st);
    if (du < D && sw && 2 * k2 + 1 == R) hi = *reinterpret_cast<const uint4*>(st);
    uint32_t* dst = us + (w * K2 + k2) * kPitch + oct * 2;
    const uint32_t l[4] = {lo.x, lo.y, lo.z, lo.w}, h[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      dst[j * 8] = __byte_perm(l[j], h[j], 0x5410);
      dst[j * 8 + 1] = __byte_perm(l[j], h[j], 0x7632);
    }
  }
  if constexpr (!kDirect) {
#pragma unroll
    for (int r = 0; r < 16; ++r)
#pragma unroll
      for (int h = 0; h < kHalves; ++h)
        if (h * 32 + lane < KS * 16) reinterpret_cast<uint16_t*>(zs[warp][r])[h * 32 + lane] = zv[r][h];
  }
  __syncthreads();
  if (b0 >= B) return;  // (whole warps: all lanes take part in the products, channels there or not)
  if constexpr (!kDirect) {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int i = 0; i < 4; ++i) a[ks][i] = zs[warp][r0 + (i & 1) * 8][ks * 8 + (i >> 1) * 4 + q];
  }
  float out[2][8];
#pragma unroll
  for (int hf = 0; hf < 2; ++hf) {
    float v[8];
    unpack8(past[hf][0], v);
#pragma unroll
    for (int e = 0; e < 8; ++e) out[hf][e] = residual ? v[e] : 0.f;
  }
#pragma unroll
  for (int w = 0; w < W; ++w) {  // tap by tap: its 32 weights, then their part of the outputs
    float acc[4][4] = {};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const uint32_t* f = us + (w * K2 + ks * 8 + q) * kPitch + r0;
#pragma unroll
      for (int j = 0; j < 4; ++j) mma_16n8k16(acc[j], a[ks], f[j * 8], f[4 * kPitch + j * 8]);
    }
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      float v[8];
      unpack8(past[hf][w], v);
#pragma unroll
      for (int e = 0; e < 8; ++e) out[hf][e] = fmaf(acc[e >> 1][hf * 2 + (e & 1)], v[e], out[hf][e]);
    }
  }
#pragma unroll
  for (int hf = 0; hf < 2; ++hf) {
    const int64_t b = b0 + r0 + hf * 8;
    if (b >= B || d >= D) continue;
    uint4* yr = reinterpret_cast<uint4*>(y + b * C + c);
    if (rows[hf] < 0) {
      *yr = make_uint4(0, 0, 0, 0);
      continue;
    }
    const float(&o)[8] = out[hf];
    *yr = make_uint4(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]), pack_bf16x2(o[4], o[5]), pack_bf16x2(o[6], o[7]));
    __nv_bfloat16* cr = cache + rows[hf] * (int64_t)(W - 1) * C + c;
#pragma unroll
    for (int w = 1; w < W; ++w) *reinterpret_cast<uint4*>(cr + (int64_t)(W - 1 - w) * C) = past[hf][w - 1];
  }
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

template <typename T, int W, int VEC>
int lr_many(const StepArgs& a) {
  const int64_t C = a.G * a.D;
  constexpr int RB = 8;
  const dim3 grid((unsigned)((C / VEC + kThreads - 1) / kThreads), (unsigned)((a.B + RB - 1) / RB));
  const size_t smem = (size_t)a.G * a.R * RB * sizeof(float);
  lr_step_kernel<T, W, VEC, RB><<<grid, kThreads, smem, a.st>>>(
      (const T*)a.x, (const T*)a.z, (const T*)a.U, (const T*)a.sw, (T*)a.cache, (T*)a.y, a.slots, a.slot_bytes, a.B,
      a.n_rows, a.D, a.R, a.G, a.residual);
  DYNCONV_CHECK_LAUNCH("lr_step_kernel");
  return DYNCONV_OK;
}

template <typename T, int W, int VEC>
int lr_few(const StepArgs& a) {
  const int64_t blocks = a.G * ((a.D / VEC + 31) / 32);
  lr_step_few_kernel<T, W, VEC><<<dim3((unsigned)blocks, (unsigned)a.B), 32 * W, 0, a.st>>>(
      (const T*)a.x, (const T*)a.z, (const T*)a.U, (const T*)a.sw, (T*)a.cache, (T*)a.y, a.slots, a.slot_bytes,
      a.n_rows, a.D, a.R, a.G, a.residual);
  DYNCONV_CHECK_LAUNCH("lr_step_few_kernel");
  return DYNCONV_OK;
}

template <int W, int KS>
int lr_mma_go(const StepArgs& a) {
  const dim3 grid((unsigned)(a.G * ((a.D + kMmaCh - 1) / kMmaCh)), (unsigned)((a.B + kMmaRows - 1) / kMmaRows));
  using bf = __nv_bfloat16;
  lr_step_mma_kernel<W, KS><<<grid, kMmaThreads, 0, a.st>>>((const bf*)a.x, (const bf*)a.z, (const bf*)a.U, (const bf*)a.sw,
                                                    (bf*)a.cache, (bf*)a.y, a.slots, a.slot_bytes, a.B, a.n_rows, a.D,
                                                    a.R, a.G, a.residual);
  DYNCONV_CHECK_LAUNCH("lr_step_mma_kernel");
  return DYNCONV_OK;
}

int mma_steps(const StepArgs& a) { return (a.R + (a.sw ? 1 : 0) + 15) / 16; }  // ranks, the static filter's among them

template <int W>
int lr_mma(const StepArgs& a) {
  const int ks = mma_steps(a);
  if (ks == 1) return lr_mma_go<W, 1>(a);
  if (ks == 2) return lr_mma_go<W, 2>(a);
  if constexpr (mma_fits(W, 4))
    if (ks == 4) return lr_mma_go<W, 4>(a);
  if constexpr (mma_fits(W, 5))
    if (ks == 5) return lr_mma_go<W, 5>(a);
  return lr_mma_go<W, 3>(a);
}

bool aligned_octets(const StepArgs& a) {
  if (a.D % 8 != 0) return false;
  const void* ptrs[] = {a.x, a.U, a.sw, a.cache, a.y};
  for (const void* q : ptrs)
    if (reinterpret_cast<uintptr_t>(q) & 15) return false;
  return true;
}

template <typename T, int W>
int lr_pick(const StepArgs& a, bool pairs) {
  if constexpr (sizeof(T) == 2)
    if (aligned_octets(a) && mma_fits(W, mma_steps(a))) return lr_mma<W>(a);
  const int64_t loads = a.G * a.D / (pairs ? 2 : 1) * a.R * W;
  if (a.B <= kFewRows && a.B * loads <= kFewLoads) return pairs ? lr_few<T, W, 2>(a) : lr_few<T, W, 1>(a);
  return pairs ? lr_many<T, W, 2>(a) : lr_many<T, W, 1>(a);
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
