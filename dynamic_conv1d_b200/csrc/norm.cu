// norm.cu -- root-mean-square norms fused with what stands next to them in a layer.
//
// Gated norm (after a block, one row per head):
//     r = rsqrt(mean(x^2) + eps),  y = scale * x r * w * silu(g)           (w, g optional)
//     dn = scale * dy w silu(g),   dx = r (dn - x r^2 mean(dn x))
//     dw = sum_rows scale * dy x r silu(g),  dg = scale * dy x r w silu'(g)
// Residual norm (between two blocks):
//     h = residual + s * x,  r = rsqrt(mean(h^2) + eps),  y = h r * w      (s a number or one per channel)
//     dt = dh + r (dy w - h r^2 mean(dy w h)),  dresidual = dt,  dx = s dt
//     dw = sum_rows dy h r,  ds = sum_rows dt x
// Both sums that a backward row needs (of squares and of dn x) are of its inputs, so one pass over
// the row gives them and nothing is kept from the forward but h, which the caller has anyway.  That h is rounded to the
// rows' type, where y came from the sum itself: in bf16 dw is off by 2.3e-3 of its length, of which its own rounding is 1.6e-3;
// dx, dresidual and ds show nothing of it.  (The sum itself would have to be made again, from x and residual: two tensors for one.)
//
// A row is read once into registers (up to 16 numbers per thread) and written once; sums are fp32.  A row belongs to 8..32 lanes of a warp, or to a whole CTA of 128 to 1024 threads above
// 512 channels.  The sums over rows stay in the threads that own their columns; the CTAs'
// partial rows are added up in a fixed order by a second launch, so results do not change from
// run to run.
//
// The residual norm is bound by HBM: 16384 rows of 2048 in bf16 take 49 us forward (5.4 TB/s) and 66 us back (6.1 TB/s), in fp32 86
// and 120 us (6.2 and 6.7 TB/s); 8192 x 4096 in bf16 59 and 73 us (one CTA of 512 threads is all an SM holds of the forward).
// The gated norm by its instructions: 16384 x 16 rows of 128 in bf16 take 40 us forward (issue 77%, DRAM 50%) and 73 us
// back (issue 75%, DRAM 49%), in fp32 74 and 147 us.  Rows of more than 8192 numbers belong to 1024 threads of 64 registers: no
// next row is under way and the backward spills (76 to 736 bytes); 2048 x 16384 in bf16: residual norm 60 and 222 us, gated
// norm 62 and 253 us; 509 x 8190 in fp32: residual norm 20 and 27 us.
#include "common.cuh"
#include "norm.cuh"

namespace dynconv {
namespace norm {
namespace {

constexpr int kPerThread = 16;  // numbers of a row per thread, at most (32 spilled: the backward holds four tensors' and two sums)

// A thread's share of a row, as stored.  (A float32 weight's eight numbers beside a row in bf16 are two pieces of 16 bytes.)
template <typename T, int VEC>
struct alignas(VEC * sizeof(T) < 16 ? VEC * sizeof(T) : 16) Vec {
  T e[VEC];
};

// Sums a and b over the TPR threads of a row, in every one of them.
template <int TPR>
__device__ __forceinline__ float2 row_sum(float2 v, int& flip) {
  constexpr int kIn = TPR < 32 ? TPR : 32;
#pragma unroll
  for (int d = kIn / 2; d > 0; d >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, d);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, d);
  }
  if constexpr (TPR > 32) {
    constexpr int kWarps = TPR / 32;
    __shared__ float2 part[2][kWarps];  // (alternating: one barrier for each row)
    if ((threadIdx.x & 31) == 0) part[flip][threadIdx.x >> 5] = v;
    __syncthreads();
    v = part[flip][0];
#pragma unroll
    for (int i = 1; i < kWarps; ++i) v.x += part[flip][i].x, v.y += part[flip][i].y;
    flip ^= 1;
  }
  return v;
}

// (the quick exponential is off by 2^-21 + 2^-23 |z|; silu of -inf is NaN, as -inf * 0 is)
__device__ __forceinline__ float sigmoid(float z) { return __fdividef(1.f, 1.f + __expf(-z)); }

// Threads of a CTA for a row of TPR threads.
__host__ __device__ constexpr int cta(int tpr) { return tpr <= 32 ? 256 : tpr; }

// The sums over this CTA's rows: thread (row group, lane) holds N_ACC columns; groups are added in
// order through shared memory and the result is the CTA's row of `part`.
template <int TPR, int VEC, int NV>
__device__ __forceinline__ void store_sums(const float (&acc)[NV * VEC], float* part, int D) {
  constexpr int kGroups = cta(TPR) / TPR;
  const int lane = threadIdx.x % TPR, group = threadIdx.x / TPR;
  if constexpr (kGroups == 1) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const int c = (i * TPR + lane) * VEC + e;
        if (c < D) part[c] = acc[i * VEC + e];
      }
  } else {
    __shared__ float sh[kGroups][TPR * 4 + 1];
#pragma unroll
    for (int j = 0; j < NV * VEC; j += 4) {  // four numbers of each thread at a time
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (j + e < NV * VEC) sh[group][lane * 4 + e] = acc[j + e];
      __syncthreads();
      for (int t = threadIdx.x; t < TPR * 4; t += cta(TPR)) {
        const int k = j + t % 4;  // the number's index in its thread
        const int c = (k / VEC * TPR + t / 4) * VEC + k % VEC;
        if (k < NV * VEC && c < D) {
          float s = sh[0][t];
          for (int g = 1; g < kGroups; ++g) s += sh[g][t];
          part[c] = s;
        }
      }
    }
  }
}

// A thread's columns of a weight: held over all rows where its share of a row is small, else read again for each.  A
// weight has the row's type or float32, which keeps the digits of a master weight and of its gradient's sum.  float32
// beside rows in bf16 lies in shared memory, each thread's own columns where it alone reads them, but for the small shares of a
// backward (HOLD).  Residual norm, forward and back: 4096 x 8192 66 and 79 us so, 87 and 147 us read again for each row; 8192 x
// 4096 48 and 86 us so, 59 and 73 us held.
template <typename T, typename W, int VEC, int TPR, int NV, bool HOLD>
struct Columns {
  using V = Vec<W, VEC>;
  static constexpr bool kSmall = VEC * NV <= 8, kStashed = sizeof(W) != sizeof(T) && !(HOLD && kSmall), kHeld = !kStashed && kSmall;
  static constexpr int kPiece = VEC < 4 ? VEC : 4;  // numbers of a float32 vector that are read at once
  static constexpr int kBytes = kStashed ? NV * VEC * (int)sizeof(W) * cta(TPR) : 0;
  using Piece = Vec<W, kPiece>;
  V held[kHeld ? NV : 1];
  const W* at;
  Piece* own;
  __device__ __forceinline__ Columns(const void* p, int lane, int D, uint8_t* room) : at((const W*)p + lane * VEC), own((Piece*)room + threadIdx.x) {
    if constexpr (kHeld || kStashed) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (p && (i * TPR + lane) * VEC < D) {
          if constexpr (kHeld) {
            held[i] = *reinterpret_cast<const V*>(at + i * TPR * VEC);
          } else {
#pragma unroll
            for (int j = 0; j < VEC / kPiece; ++j)
              own[(i * (VEC / kPiece) + j) * cta(TPR)] = *reinterpret_cast<const Piece*>(at + i * TPR * VEC + j * kPiece);
          }
        }
    }
  }
  __device__ __forceinline__ V operator[](int i) const {
    if constexpr (kHeld) {
      return held[i];
    } else if constexpr (kStashed) {
      V v;
#pragma unroll
      for (int j = 0; j < VEC / kPiece; ++j) {
        const Piece x = own[(i * (VEC / kPiece) + j) * cta(TPR)];
#pragma unroll
        for (int e = 0; e < kPiece; ++e) v.e[j * kPiece + e] = x.e[e];
      }
      return v;
    } else {
      return *reinterpret_cast<const V*>(at + i * TPR * VEC);
    }
  }
};

// Whether a thread's share of a row is small enough to have the next row's loads under way meanwhile.
constexpr bool ahead(int vec, int nv) { return vec * nv <= 8; }

// CTAs of a backward that an SM runs at once.  Narrow rows: 512 threads of 100 to 128 registers, the next rows under way
// (gated, 16384 x 16 x 128: 74 us, and 79 at 80 registers and 768 threads).
__host__ __device__ constexpr int backward_ctas(int tpr) {
  const int n = (cta(tpr) > 512 ? 1024 : 512) / cta(tpr);
  return n < 1 ? 1 : n;
}

// Walks this CTA's rows: load(row, buffer) for each, the next one's before the work on the present one.
template <typename Buf, int TPR, bool AHEAD, typename Load, typename Work>
__device__ __forceinline__ void walk(int64_t rows, Load&& load, Work&& work) {
  constexpr int kRows = cta(TPR) / TPR;
  const int64_t step = (int64_t)gridDim.x * kRows;
  int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / TPR, first = (int64_t)blockIdx.x * kRows;
  Buf now;
  if (AHEAD && first < rows) load(row, now);
  for (; first < rows; first += step, row += step) {
    if constexpr (AHEAD) {
      Buf next;
      if (first + step < rows) load(row + step, next);
      work(row, now);
      now = next;
    } else {
      load(row, now);
      work(row, now);
    }
  }
}

// The same with the rows to come in shared memory: each thread copies its own pieces of 16 bytes asynchronously and reads
// them back itself, so nothing but its own copies has to be waited for, and rows under way cost no registers.
// start(row, slot) asks for a row's pieces, work(row, slot) has them.
template <int TPR, int STAGES, typename Start, typename Work>
__device__ __forceinline__ void walk_ring(int64_t rows, Start&& start, Work&& work) {
  constexpr int kRows = cta(TPR) / TPR;
  const int64_t step = (int64_t)gridDim.x * kRows;
  int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / TPR, first = (int64_t)blockIdx.x * kRows;
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) {
    start(row + i * step, i);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  for (int slot = 0; first < rows; first += step, row += step) {
    start(row + (STAGES - 1) * step, slot == 0 ? STAGES - 1 : slot - 1);  // (the slot that the row before this one had)
    asm volatile("cp.async.commit_group;" ::: "memory");
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
    work(row, slot);
    slot = slot == STAGES - 1 ? 0 : slot + 1;
  }
}

// The backward's rows in shared memory: a piece of each of N tensors for each thread, as many rows as the CTAs' shares of an SM's
// shared memory hold beside float32 weights, at most four; none (0) where a piece is not 16 bytes or two rows do not fit.  Of 2-byte
// types alone: residual norm, 16384 x 2048 in bf16, takes 65 us so and 105 us with one row ahead in registers (3 CTAs on an SM instead
// of 2: 74 us); of 4-byte types the registers' row is enough already, 62 us for 8192 x 2048 and 66 us with the ring.
template <typename T, int VEC, int TPR, int NV, int N, int WEIGHTS>
struct Ring {
  static constexpr int kSlot = N * NV * cta(TPR) * 16, kFit = (208 * 1024 / backward_ctas(TPR) - WEIGHTS) / kSlot;
  static constexpr int kStages = sizeof(T) != 2 || VEC != 8 || kFit < 2 ? 0 : kFit < 4 ? kFit : 4;
  static constexpr int kBytes = kStages * kSlot;
  // Where a thread's piece i of a tensor lies, and its copy from n numbers behind `from` (null: none).
  static __device__ __forceinline__ uint8_t* at(uint8_t* ring, int slot, int tensor, int i) {
    return ring + slot * kSlot + ((tensor * NV + i) * cta(TPR) + threadIdx.x) * 16;
  }
  static __device__ __forceinline__ void copy(uint8_t* ring, int slot, int tensor, int i, const void* from, int64_t n) {
    if (from)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(at(ring, slot, tensor, i))), "l"((const T*)from + n) : "memory");
  }
};
// Those of the two norms.  The gated norm's rows lie in the registers of the bf16 kernel anyway; beside a float32 weight the
// compiler waits for the next row too early (16384 x 16 x 128: 91 us, 72 us with the ring and with a bf16 weight).
template <typename T, typename W, int VEC, int TPR, int NV>
struct GatedBack {
  using Cols = Columns<T, W, VEC, TPR, NV, true>;
  using R = Ring<T, VEC, TPR, NV, 3, Cols::kBytes>;
  static constexpr bool kRing = R::kStages > 0 && sizeof(W) != sizeof(T);
  static constexpr int kRingBytes = kRing ? R::kBytes : 0;
};
template <typename T, typename W, int VEC, int TPR, int NV>
struct ResidualBack {
  using Cols = Columns<T, W, VEC, TPR, NV, true>;
  using R = Ring<T, VEC, TPR, NV, 4, 2 * Cols::kBytes>;
};

template <typename T, typename W, int VEC, int TPR, int NV>
__global__ void __launch_bounds__(cta(TPR)) gated_fwd_kernel(Gated p) {
  using V = Vec<T, VEC>;
  struct Buf {
    V x[NV], z[NV];
  };
  const int lane = threadIdx.x % TPR;
  int flip = 0;
  const int64_t rows = p.N * p.G;
  extern __shared__ __align__(16) uint8_t room[];
  const Columns<T, W, VEC, TPR, NV, false> w(p.weight, lane, p.D, room);
  walk<Buf, TPR, ahead(VEC, NV)>(
      rows,
      [&](int64_t row, Buf& a) {
        const int64_t n = p.G == 1 ? row : row / p.G, g = row - n * p.G;
        const T* x = (const T*)p.x + n * p.x_outer + g * p.x_inner;
        const T* z = (const T*)p.gate + n * p.gate_outer + g * p.gate_inner;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int c = (i * TPR + lane) * VEC;
          if (row < rows && c < p.D) {
            a.x[i] = *reinterpret_cast<const V*>(x + c);
            if (p.gate) a.z[i] = *reinterpret_cast<const V*>(z + c);
          }
        }
      },
      [&](int64_t row, const Buf& a) {
        const bool in = row < rows;
        float2 s = make_float2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if (in && (i * TPR + lane) * VEC < p.D)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
              const float v = Elem<T>::to_f(a.x[i].e[e]);
              s.x = fmaf(v, v, s.x);
            }
        const float r = p.scale * rsqrtf(row_sum<TPR>(s, flip).x / p.D + p.eps);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int c = (i * TPR + lane) * VEC;
          if (!in || c >= p.D) continue;
          V y;
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            float v = Elem<T>::to_f(a.x[i].e[e]) * r;
            if (p.weight) v *= Elem<W>::to_f(w[i].e[e]);
            if (p.gate) {
              const float zf = Elem<T>::to_f(a.z[i].e[e]);
              v *= zf * sigmoid(zf);
            }
            y.e[e] = Elem<T>::from_f(v);
          }
          *reinterpret_cast<V*>((T*)p.y + row * p.D + c) = y;
        }
      });
}

template <typename T, typename W, int VEC, int TPR, int NV>
__global__ void __launch_bounds__(cta(TPR), backward_ctas(TPR)) gated_bwd_kernel(Gated p) {
  using V = Vec<T, VEC>;
  struct Buf {
    V x[NV], z[NV], d[NV];
  };
  const int lane = threadIdx.x % TPR;
  int flip = 0;
  const int64_t rows = p.N * p.G;
  float acc[NV * VEC];
  using B = GatedBack<T, W, VEC, TPR, NV>;
  using R = typename B::R;
  extern __shared__ __align__(16) uint8_t room[];
  const typename B::Cols w(p.weight, lane, p.D, room + B::kRingBytes);
#pragma unroll
  for (int i = 0; i < NV * VEC; ++i) acc[i] = 0.f;
  auto work = [&](int64_t row, const Buf& a) {
    const bool in = row < rows;
    // a narrow row's gates stay in registers between the sums and the gradients; a wide one's are made twice
    constexpr bool kKeep = ahead(VEC, NV);
    float sg[kKeep ? NV * VEC : 1];
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (in && (i * TPR + lane) * VEC < p.D)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float v = Elem<T>::to_f(a.x[i].e[e]);
          float dn = Elem<T>::to_f(a.d[i].e[e]);
          if (p.weight) dn *= Elem<W>::to_f(w[i].e[e]);
          if (p.gate) {
            const float zf = Elem<T>::to_f(a.z[i].e[e]), g = sigmoid(zf);
            if constexpr (kKeep) sg[i * VEC + e] = g;
            dn *= zf * g;
          }
          s.x = fmaf(v, v, s.x);
          s.y = fmaf(dn, v, s.y);
        }
    s = row_sum<TPR>(s, flip);
    const float r = rsqrtf(s.x / p.D + p.eps), rs = p.scale * r, m = s.y / p.D * r * r;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * VEC;
      if (!in || c >= p.D) continue;
      V dx, dz;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float v = Elem<T>::to_f(a.x[i].e[e]), d = Elem<T>::to_f(a.d[i].e[e]);
        const float dw = p.weight ? d * Elem<W>::to_f(w[i].e[e]) : d, vr = v * rs;
        if (p.gate) {
          const float zf = Elem<T>::to_f(a.z[i].e[e]);
          float g;
          if constexpr (kKeep)
            g = sg[i * VEC + e];
          else
            g = sigmoid(zf);
          const float silu = zf * g;
          dx.e[e] = Elem<T>::from_f(rs * fmaf(dw, silu, -v * m));
          dz.e[e] = Elem<T>::from_f(dw * vr * (g + silu * (1.f - g)));
          acc[i * VEC + e] = fmaf(d * vr, silu, acc[i * VEC + e]);
        } else {
          dx.e[e] = Elem<T>::from_f(rs * fmaf(-v, m, dw));
          acc[i * VEC + e] = fmaf(d, vr, acc[i * VEC + e]);
        }
      }
      if (p.dx) *reinterpret_cast<V*>((T*)p.dx + row * p.D + c) = dx;
      if (p.dgate) *reinterpret_cast<V*>((T*)p.dgate + row * p.D + c) = dz;
    }
  };
  if constexpr (B::kRing) {
    walk_ring<TPR, R::kStages>(
        rows,
        [&](int64_t row, int slot) {
          const int64_t n = p.G == 1 ? row : row / p.G, g = row - n * p.G;
#pragma unroll
          for (int i = 0; i < NV; ++i) {
            const int c = (i * TPR + lane) * VEC;
            if (row < rows && c < p.D) {
              R::copy(room, slot, 0, i, p.x, n * p.x_outer + g * p.x_inner + c);
              R::copy(room, slot, 1, i, p.dy, row * p.D + c);
              R::copy(room, slot, 2, i, p.gate, n * p.gate_outer + g * p.gate_inner + c);
            }
          }
        },
        [&](int64_t row, int slot) {
          Buf a;
#pragma unroll
          for (int i = 0; i < NV; ++i) {
            a.x[i] = *reinterpret_cast<const V*>(R::at(room, slot, 0, i));
            a.d[i] = *reinterpret_cast<const V*>(R::at(room, slot, 1, i));
            if (p.gate) a.z[i] = *reinterpret_cast<const V*>(R::at(room, slot, 2, i));
          }
          work(row, a);
        });
  } else {
    walk<Buf, TPR, ahead(VEC, NV)>(
        rows,
        [&](int64_t row, Buf& a) {
          const int64_t n = p.G == 1 ? row : row / p.G, g = row - n * p.G;
          const T* x = (const T*)p.x + n * p.x_outer + g * p.x_inner;
          const T* z = (const T*)p.gate + n * p.gate_outer + g * p.gate_inner;
          const T* dy = (const T*)p.dy + row * p.D;
#pragma unroll
          for (int i = 0; i < NV; ++i) {
            const int c = (i * TPR + lane) * VEC;
            if (row < rows && c < p.D) {
              a.x[i] = *reinterpret_cast<const V*>(x + c);
              a.d[i] = *reinterpret_cast<const V*>(dy + c);
              if (p.gate) a.z[i] = *reinterpret_cast<const V*>(z + c);
            }
          }
        },
        work);
  }
  if (p.part) store_sums<TPR, VEC, NV>(acc, p.part + (int64_t)blockIdx.x * p.D, p.D);
}

template <typename T, typename W, int VEC, int TPR, int NV>
__global__ void __launch_bounds__(cta(TPR)) residual_fwd_kernel(Residual p) {
  using V = Vec<T, VEC>;
  struct Buf {
    V x[NV], r[NV];
  };
  const int lane = threadIdx.x % TPR;
  int flip = 0;
  using Cols = Columns<T, W, VEC, TPR, NV, false>;
  extern __shared__ __align__(16) uint8_t room[];
  const Cols w(p.weight, lane, p.D, room), sc(p.scale, lane, p.D, room + Cols::kBytes);
  walk<Buf, TPR, ahead(VEC, NV)>(
      p.N,
      [&](int64_t row, Buf& a) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int c = (i * TPR + lane) * VEC;
          if (row < p.N && c < p.D) {
            a.x[i] = *reinterpret_cast<const V*>((const T*)p.x + row * p.D + c);
            a.r[i] = *reinterpret_cast<const V*>((const T*)p.residual + row * p.D + c);
          }
        }
      },
      [&](int64_t row, const Buf& a) {
        const bool in = row < p.N;
        float h[NV * VEC];  // unrounded: y is the norm of the sum itself
        float2 s = make_float2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int c = (i * TPR + lane) * VEC;
          if (!in || c >= p.D) continue;
          V hv;
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const float f = p.scale ? Elem<W>::to_f(sc[i].e[e]) : p.factor;
            const float v = fmaf(f, Elem<T>::to_f(a.x[i].e[e]), Elem<T>::to_f(a.r[i].e[e]));
            h[i * VEC + e] = v;
            hv.e[e] = Elem<T>::from_f(v);
            s.x = fmaf(v, v, s.x);
          }
          *reinterpret_cast<V*>((T*)p.h + row * p.D + c) = hv;
        }
        const float r = rsqrtf(row_sum<TPR>(s, flip).x / p.D + p.eps);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int c = (i * TPR + lane) * VEC;
          if (!in || c >= p.D) continue;
          V y;
#pragma unroll
          for (int e = 0; e < VEC; ++e) y.e[e] = Elem<T>::from_f(h[i * VEC + e] * r * Elem<W>::to_f(w[i].e[e]));
          *reinterpret_cast<V*>((T*)p.y + row * p.D + c) = y;
        }
      });
}

template <typename T, typename W, int VEC, int TPR, int NV>
__global__ void __launch_bounds__(cta(TPR), backward_ctas(TPR)) residual_bwd_kernel(Residual p) {
  using V = Vec<T, VEC>;
  using R = typename ResidualBack<T, W, VEC, TPR, NV>::R;
  using Cols = typename ResidualBack<T, W, VEC, TPR, NV>::Cols;
  struct Buf {
    V h[NV], d[NV], u[NV], x[NV];
  };
  extern __shared__ __align__(16) uint8_t ring[];
  const int lane = threadIdx.x % TPR;
  int flip = 0;
  float acc_w[NV * VEC], acc_s[NV * VEC];
  const Cols w(p.weight, lane, p.D, ring + R::kBytes), sc(p.scale, lane, p.D, ring + R::kBytes + Cols::kBytes);
#pragma unroll
  for (int i = 0; i < NV * VEC; ++i) acc_w[i] = acc_s[i] = 0.f;
  auto work = [&](int64_t row, const Buf& a) {
    const bool in = row < p.N;
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (in && (i * TPR + lane) * VEC < p.D)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float v = Elem<T>::to_f(a.h[i].e[e]);
          s.x = fmaf(v, v, s.x);
          s.y = fmaf(Elem<T>::to_f(a.d[i].e[e]) * Elem<W>::to_f(w[i].e[e]), v, s.y);
        }
    s = row_sum<TPR>(s, flip);
    const float r = rsqrtf(s.x / p.D + p.eps), m = s.y / p.D * r * r;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * VEC;
      if (!in || c >= p.D) continue;
      V dt, dx;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float v = Elem<T>::to_f(a.h[i].e[e]), d = Elem<T>::to_f(a.d[i].e[e]);
        const float t = fmaf(r, fmaf(d, Elem<W>::to_f(w[i].e[e]), -v * m), Elem<T>::to_f(a.u[i].e[e]));
        dt.e[e] = Elem<T>::from_f(t);
        dx.e[e] = Elem<T>::from_f(t * (p.scale ? Elem<W>::to_f(sc[i].e[e]) : p.factor));
        acc_w[i * VEC + e] = fmaf(d, v * r, acc_w[i * VEC + e]);
        if (p.part_s) acc_s[i * VEC + e] = fmaf(t, Elem<T>::to_f(a.x[i].e[e]), acc_s[i * VEC + e]);
      }
      if (p.dresidual) *reinterpret_cast<V*>((T*)p.dresidual + row * p.D + c) = dt;
      if (p.dx) *reinterpret_cast<V*>((T*)p.dx + row * p.D + c) = dx;
    }
  };
  if constexpr (R::kStages > 0) {
    walk_ring<TPR, R::kStages>(
        p.N,
        [&](int64_t row, int slot) {
#pragma unroll
          for (int i = 0; i < NV; ++i) {
            const int c = (i * TPR + lane) * VEC;
            if (row < p.N && c < p.D) {
              const int64_t n = row * p.D + c;
              R::copy(ring, slot, 0, i, p.h, n), R::copy(ring, slot, 1, i, p.dy, n), R::copy(ring, slot, 2, i, p.dh, n);
              R::copy(ring, slot, 3, i, p.part_s ? p.x : nullptr, n);
            }
          }
        },
        [&](int64_t row, int slot) {
          Buf a;
#pragma unroll
          for (int i = 0; i < NV; ++i) {
            a.h[i] = *reinterpret_cast<const V*>(R::at(ring, slot, 0, i));
            a.d[i] = p.dy ? *reinterpret_cast<const V*>(R::at(ring, slot, 1, i)) : V{};
            a.u[i] = p.dh ? *reinterpret_cast<const V*>(R::at(ring, slot, 2, i)) : V{};
            a.x[i] = *reinterpret_cast<const V*>(R::at(ring, slot, 3, i));
          }
          work(row, a);
        });
  } else {
    walk<Buf, TPR, ahead(VEC, NV)>(
        p.N,
        [&](int64_t row, Buf& a) {
#pragma unroll
          for (int i = 0; i < NV; ++i) {
            const int c = (i * TPR + lane) * VEC;
            if (row < p.N && c < p.D) {
              a.h[i] = *reinterpret_cast<const V*>((const T*)p.h + row * p.D + c);
              a.d[i] = p.dy ? *reinterpret_cast<const V*>((const T*)p.dy + row * p.D + c) : V{};
              a.u[i] = p.dh ? *reinterpret_cast<const V*>((const T*)p.dh + row * p.D + c) : V{};
              if (p.part_s) a.x[i] = *reinterpret_cast<const V*>((const T*)p.x + row * p.D + c);
            }
          }
        },
        work);
  }
  if (p.part_w) store_sums<TPR, VEC, NV>(acc_w, p.part_w + (int64_t)blockIdx.x * p.D, p.D);
  if (p.part_s) store_sums<TPR, VEC, NV>(acc_s, p.part_s + (int64_t)blockIdx.x * p.D, p.D);
}

// out[c] = sum over the CTAs' partial rows.  32 columns per CTA; 32 threads of a column take every
// 32nd row and are added in order.  (One thread per column would read 600 rows one after another.)
template <typename T>
__global__ void __launch_bounds__(1024) column_sum_kernel(const float* __restrict__ part_a, T* __restrict__ out_a,
                                                          const float* __restrict__ part_b, T* __restrict__ out_b,
                                                          int P, int D) {
  __shared__ float sh[32][33];
  const float* part = blockIdx.y ? part_b : part_a;
  T* out = blockIdx.y ? out_b : out_a;
  const int c = blockIdx.x * 32 + threadIdx.x % 32, r = threadIdx.x / 32;
  float s = 0.f;
  if (c < D)
#pragma unroll 4
    for (int i = r; i < P; i += 32) s += part[(int64_t)i * D + c];
  sh[r][threadIdx.x % 32] = s;
  __syncthreads();
  if (r == 0 && c < D) {
    s = sh[0][threadIdx.x];
#pragma unroll
    for (int i = 1; i < 32; ++i) s += sh[i][threadIdx.x];
    out[c] = Elem<T>::from_f(s);
  }
}

// The most numbers that can be read at once: the pointers (or-ed addresses; of the weights, of their own type, apart) and
// strides (or-ed) decide.
int vec_of(uintptr_t addresses, uintptr_t weights, int64_t strides, int dtype, bool w32) {
  const int elem = dtype == DYNCONV_DTYPE_BF16 ? 2 : 4, w_elem = w32 ? 4 : elem;
  for (int n : {16 / elem, 2})
    if (addresses % (n * elem) == 0 && weights % (n * w_elem < 16 ? n * w_elem : 16) == 0 && strides % n == 0) return n;
  return 1;
}
uintptr_t bits(const void* p) { return reinterpret_cast<uintptr_t>(p); }

// CTAs of a launch: per_sm for each SM (a backward's run at once; of a forward's 2048 threads the registers let three
// eighths to a half do so, the others follow), no more than there is work for.
int64_t grid_of(int64_t rows, int tpr, int per_sm) {
  const int64_t want = (rows * tpr + cta(tpr) - 1) / cta(tpr);
  const int64_t most = (int64_t)sm_count() * per_sm;
  return want < most ? want : most;
}

// Threads of a row: the fewest that hold it at VEC x NV numbers each, where narrow rows take one
// vector each (more rows in flight), up to a warp, and wide ones a CTA.  Rows of 513 to 4096 numbers have 8 of them in
// a thread: 32768 rows of 1024 in bf16 take 48 us forward and 71 us back with 128 threads (72 and 89 us with 256, half
// of them idle), 8192 rows of 4096 61 and 74 us with 512 (56 and 93 us with 256 of 16 numbers).
template <typename T, typename W, int VEC, typename F>
int pick(int64_t D, F&& go) {
  constexpr int kNV = kPerThread / VEC;
  constexpr int kOne = VEC >= 4 ? 1 : 4 / VEC;  // vectors per thread of a narrow row
  if (D <= 8 * VEC * kOne) return go.template operator()<T, W, VEC, 8, kOne>();
  if (D <= 16 * VEC * kOne) return go.template operator()<T, W, VEC, 16, kOne>();
  if (D <= 32 * VEC * kOne) return go.template operator()<T, W, VEC, 32, kOne>();
  if (D <= 32 * kPerThread) return go.template operator()<T, W, VEC, 32, kNV>();
  if (D <= 128 * kPerThread / 2) return go.template operator()<T, W, VEC, 128, kNV / 2>();
  if (D <= 256 * kPerThread / 2) return go.template operator()<T, W, VEC, 256, kNV / 2>();
  if (D <= 512 * kPerThread / 2) return go.template operator()<T, W, VEC, 512, kNV / 2>();
  if (D <= 512 * kPerThread) return go.template operator()<T, W, VEC, 512, kNV>();
  return go.template operator()<T, W, VEC, 1024, kNV>();
}

// (static shared memory counts too, so any bytes at all are asked for)
template <typename K>
int room(K* kern, int bytes) {
  return bytes == 0 ? DYNCONV_OK : allow_shared(kern, bytes, "cudaFuncSetAttribute(norm)");
}

struct GatedGo {
  const Gated& p;
  bool backward;
  cudaStream_t st;
  template <typename T, typename W, int VEC, int TPR, int NV>
  int operator()() const {
    Gated q = p;
    constexpr int kRoom = Columns<T, W, VEC, TPR, NV, false>::kBytes;
    using B = GatedBack<T, W, VEC, TPR, NV>;
    const int64_t g = grid_of(q.N * q.G, TPR, backward ? backward_ctas(TPR) : 2048 / cta(TPR));
    if (!backward) {
      if (int s = room(gated_fwd_kernel<T, W, VEC, TPR, NV>, kRoom)) return s;
      gated_fwd_kernel<T, W, VEC, TPR, NV><<<(unsigned)g, cta(TPR), q.weight ? kRoom : 0, st>>>(q);
      DYNCONV_CHECK_LAUNCH("gated_fwd_kernel");
      return DYNCONV_OK;
    }
    if (int s = room(gated_bwd_kernel<T, W, VEC, TPR, NV>, B::kRingBytes + B::Cols::kBytes)) return s;
    gated_bwd_kernel<T, W, VEC, TPR, NV><<<(unsigned)g, cta(TPR), B::kRingBytes + (q.weight ? B::Cols::kBytes : 0), st>>>(q);
    DYNCONV_CHECK_LAUNCH("gated_bwd_kernel");
    if (q.part) {
      column_sum_kernel<W><<<(unsigned)((q.D + 31) / 32), 1024, 0, st>>>(q.part, (W*)q.dweight, nullptr, nullptr, (int)g, q.D);
      DYNCONV_CHECK_LAUNCH("column_sum_kernel");
    }
    return DYNCONV_OK;
  }
};

struct ResidualGo {
  const Residual& p;
  bool backward;
  cudaStream_t st;
  template <typename T, typename W, int VEC, int TPR, int NV>
  int operator()() const {
    Residual q = p;
    using B = ResidualBack<T, W, VEC, TPR, NV>;
    constexpr int kRoom = Columns<T, W, VEC, TPR, NV, false>::kBytes;
    const int weights = q.scale ? 2 : 1;
    const int64_t g = grid_of(q.N, TPR, backward ? backward_ctas(TPR) : 2048 / cta(TPR));
    if (!backward) {
      if (int s = room(residual_fwd_kernel<T, W, VEC, TPR, NV>, 2 * kRoom)) return s;
      residual_fwd_kernel<T, W, VEC, TPR, NV><<<(unsigned)g, cta(TPR), weights * kRoom, st>>>(q);
      DYNCONV_CHECK_LAUNCH("residual_fwd_kernel");
      return DYNCONV_OK;
    }
    if (int s = room(residual_bwd_kernel<T, W, VEC, TPR, NV>, B::R::kBytes + 2 * B::Cols::kBytes)) return s;
    residual_bwd_kernel<T, W, VEC, TPR, NV><<<(unsigned)g, cta(TPR), B::R::kBytes + weights * B::Cols::kBytes, st>>>(q);
    DYNCONV_CHECK_LAUNCH("residual_bwd_kernel");
    if (q.part_w || q.part_s) {
      const float *a = q.part_w, *b = q.part_s;
      W *oa = (W*)q.dweight, *ob = (W*)q.dscale;
      if (!a) a = b, oa = ob;
      const dim3 grid((unsigned)((q.D + 31) / 32), q.part_w && q.part_s ? 2 : 1);
      column_sum_kernel<W><<<grid, 1024, 0, st>>>(a, oa, b, ob, (int)g, q.D);
      DYNCONV_CHECK_LAUNCH("column_sum_kernel");
    }
    return DYNCONV_OK;
  }
};

// vec: numbers that can be read at once, a 16-byte vector of them, two or one.
template <typename T, typename W, typename Go>
int with_vec(int64_t D, int vec, const Go& go) {
  constexpr int kVec = 16 / (int)sizeof(T);
  return vec == kVec ? pick<T, W, kVec>(D, go) : vec == 2 ? pick<T, W, 2>(D, go) : pick<T, W, 1>(D, go);
}
template <typename Go>
int dispatch(int64_t D, int dtype, bool w32, int vec, const Go& go) {
  if (dtype != DYNCONV_DTYPE_BF16) return with_vec<float, float>(D, vec, go);
  return w32 ? with_vec<__nv_bfloat16, float>(D, vec, go) : with_vec<__nv_bfloat16, __nv_bfloat16>(D, vec, go);
}

}  // namespace

// Rows of partial sums that a backward may write.
int64_t partial_rows() { return (int64_t)sm_count() * 4; }

int gated_launch(const Gated& p, int dtype, bool w32, bool backward, cudaStream_t st) {
  const int64_t strides = p.D | p.x_outer | p.x_inner | (p.gate ? p.gate_outer | p.gate_inner : 0);
  const uintptr_t all = bits(p.x) | bits(p.gate) | bits(p.y) | bits(p.dy) | bits(p.dx) | bits(p.dgate);
  return dispatch(p.D, dtype, w32, vec_of(all, bits(p.weight), strides, dtype, w32), GatedGo{p, backward, st});
}

int residual_launch(const Residual& p, int dtype, bool w32, bool backward, cudaStream_t st) {
  const uintptr_t all = bits(p.x) | bits(p.residual) | bits(p.y) | bits(p.h) | bits(p.dy) | bits(p.dh) | bits(p.dx) | bits(p.dresidual);
  return dispatch(p.D, dtype, w32, vec_of(all, bits(p.weight) | bits(p.scale), p.D, dtype, w32), ResidualGo{p, backward, st});
}

}  // namespace norm
}  // namespace dynconv
