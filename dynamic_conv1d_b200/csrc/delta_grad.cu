// delta_grad.cu -- the gradients of the gated delta rule from what the chains left for every chunk: the state before it, r,
// dU and the gradient of the state after it (formulas: delta_rule.cuh).
//
// A CTA of eight warps takes one (batch row, head, chunk) after another.  v's columns come in slabs, the next one by TMA
// while this one is worked on.  A warp has 16 tokens and, of dk, a half (a quarter with chunks of 32): it sums
// dO S0^T, r dS1^T and dU S0^T over the slabs, and the first warps of each 16 tokens the triangles dO r^T and dU r^T.
// These become W and N, which go through shared memory into the products with K and Q; their products with
// Q K^T and K K^T, entry by entry, are what the log decays' gradients are sums of.  Row sums and column sums
// of the same numbers are taken, so what has to cancel does.
#include "delta_rule.cuh"

namespace dynconv {
namespace dr {
namespace {

constexpr int kThreads = 256;

template <int PX_, int C_>
struct Grad {
  static constexpr int PX = PX_, C = C_, NB = C / 16, kGroups = 8 / NB, kCols = kMaxKey / kGroups;  // a warp's columns of dk
  static constexpr int PU = PX == 1 ? 2 : 3, PS = PX == 1 ? 1 : 3;  // parts of r and dU, of the states
  static constexpr int kSlab = PX == 1 ? 4 : 2;                     // slices of 16 columns of v
  static constexpr int kTile = C * kMaxKey, kSquare = C + 8;
  using E = typename std::conditional<PX_ == 1, __nv_bfloat16, float>::type;
  static constexpr int kDo = C * 16 * (int)sizeof(E), kU = NB * 512;  // bytes of a slice: of dO, of one part of r or dU
  static constexpr int kS = 8 * 512;                                  // of one part of a state, at most
  static constexpr int kSlabBytes = kSlab * (kDo + 2 * PU * kU + 2 * PS * kS);
  static constexpr int kKq = 2 * PX * kTile * 2, kWn = 2 * PX * C * kSquare * 2;
  static constexpr int kBytes = 1024 + 2 * kSlabBytes + kKq + kWn;
  struct Slab {
    uint8_t* at;
    __device__ __forceinline__ E* d_o(int slice) const { return (E*)(at + slice * kDo); }
    __device__ __forceinline__ uint8_t* r(int part, int slice) const { return at + kSlab * kDo + (part * kSlab + slice) * kU; }
    __device__ __forceinline__ uint8_t* du(int part, int slice) const { return r(PU, 0) + (part * kSlab + slice) * kU; }
    __device__ __forceinline__ uint8_t* s0(int part, int slice) const { return r(2 * PU, 0) + (part * kSlab + slice) * kS; }
    __device__ __forceinline__ uint8_t* ds(int part, int slice) const { return s0(PS, 0) + (part * kSlab + slice) * kS; }
  };
};

// A 16 x 16 block kept as four matrices of 128 bytes, transposed: as second operand {0,1},{2,3}; as first {0,2,1,3}.
__device__ __forceinline__ void turned(uint32_t (&f)[4], const uint8_t* block) { ldsm_t(f, smem_u32(block) + (threadIdx.x & 31) * 16); }
__device__ __forceinline__ void first(uint32_t (&a)[4], const uint32_t (&f)[4]) { a[0] = f[0], a[1] = f[2], a[2] = f[1], a[3] = f[3]; }

template <typename E>
__device__ __forceinline__ void store2(E* to, float x, float y, int n, bool pairs) {
  if (sizeof(E) == 2 && pairs) {
    if (n > 0) *reinterpret_cast<uint32_t*>(to) = pack(x, y);
  } else {
    if (n > 0) to[0] = Elem<E>::from_f(x);
    if (n > 1) to[1] = Elem<E>::from_f(y);
  }
}

template <typename R>
__global__ void __launch_bounds__(kThreads, 1) delta_grad_kernel(Backward p, const __grid_constant__ Maps maps, int64_t items, int pairs) {
  constexpr int PX = R::PX, C = R::C, NB = R::NB, PU = R::PU, PS = R::PS, kSlab = R::kSlab, kSquare = R::kSquare;
  constexpr int NT = R::kCols / 8, KX = PX > PS ? PX : PS, KS = PU > PS ? PU : PS;
  using E = typename R::E;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t slab_full[2], kq_full;
  __shared__ int abort_flag;
  __shared__ Gates<C> gate;
  __shared__ float row_sum[2][C], col_sum[2][NB][C], from_state[R::kGroups][C], to_state[R::kGroups][C], inner[8];
  uint8_t* const smem = align_smem_1024(smem_raw);
  uint8_t *const k_tile = smem, *const q_tile = smem + R::kKq / 2, *const slabs = smem + R::kKq;
  __nv_bfloat16 *const W = (__nv_bfloat16*)(slabs + 2 * R::kSlabBytes), *const N = W + PX * C * kSquare;
  const int tid = threadIdx.x, l = tid & 31, warp = warp_index(), row = l >> 2, col = 2 * (l & 3);
  const int group = warp / NB, rb = group & 1 ? NB - 1 - warp % NB : warp % NB;  // (the triangle's long rows on different schedulers)
  const int chunks = (int)((p.T + C - 1) / C), n_k16 = (p.dk + 15) / 16, slices = (p.dv + 15) / 16, n_slabs = (slices + kSlab - 1) / kSlab;
  const int halves = p.dk > 64 ? 2 : 1;
  const int64_t all = (int64_t)p.B * p.H * chunks;
  if (tid == 0) {
    mbar_init(&slab_full[0], 1), mbar_init(&slab_full[1], 1), mbar_init(&kq_full, 1);
    abort_flag = 0;
    fence_barrier_init();
  }
  __syncthreads();
  // (one thread)
  auto load_slab = [&](int64_t item, int slab, int at) {
    const int64_t bh = item / chunks;
    const int c = (int)(item % chunks), first = slab * kSlab, n = min(kSlab, slices - first);
    const typename R::Slab s{slabs + at * R::kSlabBytes};
    uint64_t* const bar = &slab_full[at];
    const uint32_t state = n * n_k16 * 512;
    mbar_arrive_expect_tx(bar, n * (R::kDo + 2 * PU * R::kU) + 2 * PS * state);
    for (int i = 0; i < n; ++i) {
      if (p.pre.v)
        bulk_load(s.d_o(i), (const E*)p.pre.v + (item * slices + first + i) * (C * 16), R::kDo, bar);
      else
        tma_load_4d(s.d_o(i), &maps.v, bar, (first + i) * 16 * (int)(sizeof(E) / 2), (int)(bh % p.H), c * C, (int)(bh / p.H), policy_evict_normal());
    }
    for (int i = 0; i < PU; ++i) {
      const int64_t from = ((i * all + item) * slices + first) * (R::kU / 2);
      bulk_load(s.r(i, 0), p.rest + from, n * R::kU, bar);
      bulk_load(s.du(i, 0), p.du + from, n * R::kU, bar);
    }
    for (int i = 0; i < PS; ++i) {
      const int64_t from = ((i * all + item) * slices + first) * n_k16 * 256;
      bulk_load(s.s0(i, 0), p.states + from, state, bar);
      bulk_load(s.ds(i, 0), p.dstates + from, state, bar);
    }
  };
  auto load_kq = [&](int64_t item) {
    const int64_t bh = item / chunks;
    const int c = (int)(item % chunks);
    mbar_arrive_expect_tx(&kq_full, 2 * PX * halves * C * 128);
    if (p.pre.k) {
      for (int i = 0; i < PX; ++i) {
        const int64_t from = (item * PX + i) * halves * (C * 64);
        bulk_load(k_tile + i * R::kTile * 2, p.pre.k + from, halves * C * 128, &kq_full);
        bulk_load(q_tile + i * R::kTile * 2, p.pre.q + from, halves * C * 128, &kq_full);
      }
    } else {
      for (int d = 0; d < halves; ++d) {
        tma_load_4d(k_tile + d * C * 128, &maps.k, &kq_full, 64 * d, (int)(bh % p.H), c * C, (int)(bh / p.H), policy_evict_normal());
        tma_load_4d(q_tile + d * C * 128, &maps.q, &kq_full, 64 * d, (int)(bh % p.H), c * C, (int)(bh / p.H), policy_evict_normal());
      }
    }
  };
  const KeyLane key_across(false), key_down(true);
  const int s_down = lane_offset(kSquare, true), s_across = lane_offset(kSquare, false), o_down = lane_offset(16, true);
  const int kk0 = group * NT / 2;  // its first 16 columns of dk

  int64_t item = blockIdx.x;
  if (item >= items) return;
  int n_loaded = 0;  // slabs so far
  if (tid == 0) load_slab(item, 0, 0);
  for (int done = 0; item < items; item += gridDim.x, ++done) {
    const int64_t bh = item / chunks, b = bh / p.H, h = bh % p.H;
    const int c = (int)(item % chunks);
    const int64_t t0 = (int64_t)c * C;
    const int rows = (int)(p.T - t0 < C ? p.T - t0 : C);
    float dq[NT][4], kr[NT][4], ku[NT][4];  // dO S0^T, r dS1^T, dU S0^T
    float X[NB][2][4];                      // groups 0 and 1: dO r^T, dU r^T, blocks j <= rb
    float dot = 0.f;
#pragma unroll
    for (int n = 0; n < NT; ++n) zero(dq[n]), zero(kr[n]), zero(ku[n]);
#pragma unroll
    for (int j = 0; j < NB; ++j) zero(X[j][0]), zero(X[j][1]);
    for (int slab = 0; slab < n_slabs; ++slab, ++n_loaded) {
      const int at = n_loaded & 1;
      if (!__syncthreads_and(mbar_wait(&slab_full[at], (n_loaded >> 1) & 1, kErrWaitMma, &abort_flag))) {
        if (tid == 0) {  // (what is in flight lands before the shared memory goes)
          mbar_drain(&slab_full[at], (n_loaded >> 1) & 1);
          if (slab > 0) mbar_drain(&kq_full, done & 1);
        }
        return;
      }
      if (tid == 0) {  // (everybody is done with the other slab, and with the keys of the item before)
        if (slab == 0) load_kq(item);
        if (slab + 1 < n_slabs)
          load_slab(item, slab + 1, at ^ 1);
        else if (item + gridDim.x < items)
          load_slab(item + gridDim.x, 0, at ^ 1);
      }
      if (slab == 0) {
        const uint4* g = (const uint4*)p.pre.gates + item * (sizeof(Gates<C>) / 16);
        for (int i = tid; i < (int)sizeof(Gates<C>) / 16; i += kThreads) ((uint4*)&gate)[i] = g[i];
      }
      const typename R::Slab s{slabs + at * R::kSlabBytes};
      const int n = min(kSlab, slices - slab * kSlab);
      for (int v = 0; v < n; ++v) {
        uint32_t dO[PX][4], r[PU][4], u[PU][4];
        if constexpr (PX == 1) {
          ldsm(dO[0], smem_u32(s.d_o(v) + 16 * rb * 16 + o_down));
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 f = *reinterpret_cast<const float2*>(s.d_o(v) + (16 * rb + row + 8 * (e & 1)) * 16 + 8 * (e >> 1) + col);
            uint32_t part[PX];
            split<PX>(f.x, f.y, part);
#pragma unroll
            for (int i = 0; i < PX; ++i) dO[i][e] = part[i];
          }
        }
#pragma unroll
        for (int i = 0; i < PU; ++i) {
          uint32_t f[4];
          turned(f, s.r(i, v) + rb * 512);
          first(r[i], f);
          turned(f, s.du(i, v) + rb * 512);
          first(u[i], f);
        }
#pragma unroll
        for (int m = 0; m < NT / 2; ++m) {
          if (kk0 + m >= n_k16) continue;
          uint32_t f[PS][4], g[PS][4];
#pragma unroll
          for (int i = 0; i < PS; ++i) {
            turned(f[i], s.s0(i, 0) + (v * n_k16 + kk0 + m) * 512);
            turned(g[i], s.ds(i, 0) + (v * n_k16 + kk0 + m) * 512);
          }
          mma_parts<PX, PS, KX>(dq[2 * m], dq[2 * m + 1], dO, f);
          mma_parts<PU, PS, KS>(ku[2 * m], ku[2 * m + 1], u, f);
          mma_parts<PU, PS, KS>(kr[2 * m], kr[2 * m + 1], r, g);
          // <dS1, S0>, each pair of matrices by one of the warps that read it
          if ((v + m) % NB == rb) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float x = 0.f, y = 0.f, x1 = 0.f, y1 = 0.f;
#pragma unroll
              for (int i = PS - 1; i >= 0; --i) x += low(f[i][e]), x1 += high(f[i][e]), y += low(g[i][e]), y1 += high(g[i][e]);
              dot = fmaf(x, y, fmaf(x1, y1, dot));
            }
          }
        }
        if (group < 2) {
#pragma unroll
          for (int j = 0; j < NB; ++j) {
            if (j > rb) continue;
            uint32_t f[PU][4];
#pragma unroll
            for (int i = 0; i < PU; ++i) turned(f[i], s.r(i, v) + j * 512);
            if (group == 0)
              mma_parts<PX, PU, PU>(X[j][0], X[j][1], dO, f);
            else
              mma_parts<PU, PU, PU>(X[j][0], X[j][1], u, f);
          }
        }
        if (group == (R::kGroups == 2 ? 0 : 2) + (v & 1)) {
          // dV = beta dU
          float x[4][2];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            x[e][0] = x[e][1] = 0.f;
#pragma unroll
            for (int i = PU - 1; i >= 0; --i) x[e][0] += low(u[i][e]), x[e][1] += high(u[i][e]);
          }
          const float* beta = ((const Gates<C>*)p.pre.gates)[item].beta;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int t = 16 * rb + row + 8 * (e & 1), d = (slab * kSlab + v) * 16 + 8 * (e >> 1) + col;
            if (t < rows) {
              const float f = beta[t];
              store2((E*)p.dv_.p + b * p.dv_.sb + h * p.dv_.sh + (t0 + t) * p.dv_.st + d, x[e][0] * f, x[e][1] * f, p.dv - d, pairs & 1);
            }
          }
        }
      }
    }
    // Q K^T and K K^T for the same blocks, then W and N and their sums
    if (!__syncthreads_and(mbar_wait(&kq_full, done & 1, kErrWaitMma, &abort_flag))) {
      if (tid == 0) mbar_drain(&kq_full, done & 1), mbar_drain(&slab_full[n_loaded & 1], (n_loaded >> 1) & 1);
      return;
    }
    const uint32_t k_at = smem_u32(k_tile), q_at = smem_u32(q_tile);
    if (group < 2) {
      float Y[NB][2][4];
#pragma unroll
      for (int j = 0; j < NB; ++j) zero(Y[j][0]), zero(Y[j][1]);
      const uint32_t a_at = group == 0 ? q_at : k_at;
#pragma unroll
      for (int kk = 0; kk < 8; ++kk) {
        if (kk >= n_k16) continue;
        uint32_t a[PX][4];
#pragma unroll
        for (int i = 0; i < PX; ++i) ldsm(a[i], a_at + 2 * i * R::kTile + key_down.at<C>(rb, kk));
#pragma unroll
        for (int j = 0; j < NB; ++j) {
          if (j > rb) continue;
          uint32_t f[PX][4];
#pragma unroll
          for (int i = 0; i < PX; ++i) ldsm(f[i], k_at + 2 * i * R::kTile + key_across.at<C>(j, kk));
          mma_parts<PX, PX, PX>(Y[j][0], Y[j][1], a, f);
        }
      }
      __nv_bfloat16* const out = group == 0 ? W : N;
      float sums[2] = {0.f, 0.f};
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        if (j > rb) continue;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const int cc = 16 * j + 8 * n + col;
          const float2 hi = *reinterpret_cast<const float2*>(gate.hi + cc), lo = *reinterpret_cast<const float2*>(gate.lo + cc);
          const float2 beta = *reinterpret_cast<const float2*>(gate.beta + cc);
          float below[2] = {0.f, 0.f};
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int r = 16 * rb + row + 8 * half;
            const float f = group == 0 ? p.scale : -gate.beta[r];
            float x = X[j][n][2 * half], y = X[j][n][2 * half + 1];
            if (group == 1 && (cc == r || cc + 1 == r) && r < rows)
              ((E*)p.dbeta.p)[b * p.dbeta.sb + h * p.dbeta.sh + (t0 + r) * p.dbeta.st] = Elem<E>::from_f(cc == r ? x : y);
            x *= f * beta.x * exp2_fast((gate.hi[r] - hi.x) + (gate.lo[r] - lo.x));
            y *= f * beta.y * exp2_fast((gate.hi[r] - hi.y) + (gate.lo[r] - lo.y));
            const int last = group == 0 ? r : r - 1;
            x = cc <= last ? x : 0.f, y = cc < last ? y : 0.f;
            uint32_t part[PX];
            split<PX>(x, y, part);
#pragma unroll
            for (int i = 0; i < PX; ++i) *reinterpret_cast<uint32_t*>(out + i * C * kSquare + r * kSquare + cc) = part[i];
            // (a token's own term does not depend on the decays)
            const float mx = cc < r ? x * Y[j][n][2 * half] : 0.f, my = cc + 1 < r ? y * Y[j][n][2 * half + 1] : 0.f;
            sums[half] += mx + my;
            below[0] += mx, below[1] += my;
          }
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) {
            below[0] += __shfl_xor_sync(0xffffffffu, below[0], d);
            below[1] += __shfl_xor_sync(0xffffffffu, below[1], d);
          }
          if (row == 0) col_sum[group][rb][cc] = below[0], col_sum[group][rb][cc + 1] = below[1];
        }
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        sums[half] += __shfl_xor_sync(0xffffffffu, sums[half], 1);
        sums[half] += __shfl_xor_sync(0xffffffffu, sums[half], 2);
        if ((l & 3) == 0) row_sum[group][16 * rb + row + 8 * half] = sums[half];
      }
    }
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
    if (l == 0) inner[warp] = dot;
    // the states' parts, scaled, and what the decays get from them
    {
      float from[2] = {0.f, 0.f}, to[2] = {0.f, 0.f};
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int r = 16 * rb + row + 8 * half;
        const float fq = p.scale * gate.e[r], fr = gate.out[r] * gate.beta[r], fu = -gate.beta[r] * gate.e[r];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if (kk0 + n / 2 >= n_k16) continue;
          const int kk = kk0 + n / 2, piece = (2 * kk + (n & 1)) & 7;
          const uint32_t at = (kk >> 2) * (C * 128) + 2048 * rb + key_swizzle(row + 8 * half, piece) + 2 * col;
          float qx = 0.f, qy = 0.f, kx = 0.f, ky = 0.f;
#pragma unroll
          for (int i = PX - 1; i >= 0; --i) {
            const uint32_t uq = *reinterpret_cast<const uint32_t*>(q_tile + 2 * i * R::kTile + at);
            const uint32_t uk = *reinterpret_cast<const uint32_t*>(k_tile + 2 * i * R::kTile + at);
            qx += low(uq), qy += high(uq), kx += low(uk), ky += high(uk);
          }
          float &q0 = dq[n][2 * half], &q1 = dq[n][2 * half + 1], &r0 = kr[n][2 * half], &r1 = kr[n][2 * half + 1];
          const float u0 = ku[n][2 * half] * fu, u1 = ku[n][2 * half + 1] * fu;
          q0 *= fq, q1 *= fq, r0 *= fr, r1 *= fr;
          from[half] += qx * q0 + qy * q1 + kx * u0 + ky * u1;
          to[half] += kx * r0 + ky * r1;
          r0 += u0, r1 += u1;
        }
        from[half] += __shfl_xor_sync(0xffffffffu, from[half], 1);
        from[half] += __shfl_xor_sync(0xffffffffu, from[half], 2);
        to[half] += __shfl_xor_sync(0xffffffffu, to[half], 1);
        to[half] += __shfl_xor_sync(0xffffffffu, to[half], 2);
        if ((l & 3) == 0) from_state[group][r] = from[half], to_state[group][r] = to[half];
      }
    }
    __syncthreads();
    if (warp == 7) {
      // dlog_decay: sums of tokens from t on, and before t
      constexpr int M = C / 32;
      float a[M], e[M];
#pragma unroll
      for (int i = 0; i < M; ++i) {
        const int t = l * M + i;
        a[i] = row_sum[0][t] + row_sum[1][t];
        e[i] = 0.f;
        float below = 0.f;
        for (int j = t / 16; j < NB; ++j) below += col_sum[0][j][t] + col_sum[1][j][t];
        a[i] -= below;
#pragma unroll
        for (int g = 0; g < R::kGroups; ++g) a[i] += from_state[g][t], e[i] += to_state[g][t];
      }
      float total = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) total += inner[i];
      total *= gate.total;
#pragma unroll
      for (int i = M - 2; i >= 0; --i) a[i] += a[i + 1];
      float own = 0.f;
#pragma unroll
      for (int i = 0; i < M; ++i) own += e[i];
      float after = a[0], before = own;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const float x = __shfl_down_sync(0xffffffffu, after, d), y = __shfl_up_sync(0xffffffffu, before, d);
        if (l + d < 32) after += x;
        if (l >= d) before += y;
      }
      const float later = __shfl_down_sync(0xffffffffu, after, 1);
      float earlier = __shfl_up_sync(0xffffffffu, before, 1);
      if (l == 0) earlier = 0.f;
#pragma unroll
      for (int i = 0; i < M; ++i) {
        const int t = l * M + i;
        const float x = total + a[i] + (l < 31 ? later : 0.f) + earlier;
        if (t < rows) ((E*)p.dg.p)[b * p.dg.sb + h * p.dg.sh + (t0 + t) * p.dg.st] = Elem<E>::from_f(x);
        earlier += e[i];
      }
    }
    // dQ += W K, dK += W^T Q + (N + N^T) K
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      uint32_t wa[PX][4], na[PX][4], wt[PX][4], nt[PX][4];
#pragma unroll
      for (int i = 0; i < PX; ++i) {
        const int part = i * C * kSquare;
        if (j <= rb) {
          ldsm(wa[i], smem_u32(W + part + 16 * rb * kSquare + 16 * j + s_down));
          ldsm(na[i], smem_u32(N + part + 16 * rb * kSquare + 16 * j + s_down));
        }
        if (j >= rb) {
          ldsm_t(wt[i], smem_u32(W + part + 16 * j * kSquare + 16 * rb + s_across));
          ldsm_t(nt[i], smem_u32(N + part + 16 * j * kSquare + 16 * rb + s_across));
        }
      }
#pragma unroll
      for (int m = 0; m < NT / 2; ++m) {
        if (kk0 + m >= n_k16) continue;
        uint32_t f[PX][4], g[PX][4];
        const uint32_t at = key_down.at<C>(j, (kk0 + m) & 7);
#pragma unroll
        for (int i = 0; i < PX; ++i) {
          ldsm_t(f[i], k_at + 2 * i * R::kTile + at);
          if (j >= rb) ldsm_t(g[i], q_at + 2 * i * R::kTile + at);
        }
        if (j <= rb) {
          mma_parts<PX, PX, PX>(dq[2 * m], dq[2 * m + 1], wa, f);
          mma_parts<PX, PX, PX>(kr[2 * m], kr[2 * m + 1], na, f);
        }
        if (j >= rb) {
          mma_parts<PX, PX, PX>(kr[2 * m], kr[2 * m + 1], nt, f);
          mma_parts<PX, PX, PX>(kr[2 * m], kr[2 * m + 1], wt, g);
        }
      }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int d = 8 * (group * NT + n) + col;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int t = 16 * rb + row + 8 * half;
        if (t >= rows) continue;
        store2((E*)p.dq.p + b * p.dq.sb + h * p.dq.sh + (t0 + t) * p.dq.st + d, dq[n][2 * half], dq[n][2 * half + 1], p.dk - d, pairs & 2);
        store2((E*)p.dk_.p + b * p.dk_.sb + h * p.dk_.sh + (t0 + t) * p.dk_.st + d, kr[n][2 * half], kr[n][2 * half + 1], p.dk - d, pairs & 2);
      }
    }
  }
}

// Rows whose pairs of bf16 can be written at once.
bool even(const View& v, int width) {
  return width % 2 == 0 && v.sb % 2 == 0 && v.st % 2 == 0 && v.sh % 2 == 0 && (reinterpret_cast<uintptr_t>(v.p) & 3) == 0;
}

template <typename R>
int go(const Backward& p, cudaStream_t st) {
  const cudaError_t e = cudaFuncSetAttribute(delta_grad_kernel<R>, cudaFuncAttributeMaxDynamicSharedMemorySize, R::kBytes);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return cuda_status(e, "cudaFuncSetAttribute(delta_grad)");
  }
  Maps maps{};
  int s;
  if (!p.pre.k && ((s = view_map(&maps.k, p.k, p.B, p.T, p.H, p.dk, 2, 64, R::C)) || (s = view_map(&maps.q, p.q, p.B, p.T, p.H, p.dk, 2, 64, R::C))))
    return s;
  if (!p.pre.v && (s = view_map(&maps.v, p.d_o, p.B, p.T, p.H, p.dv, sizeof(typename R::E), 16, R::C))) return s;
  const int64_t items = (int64_t)p.B * p.H * ((p.T + R::C - 1) / R::C);
  const int pairs = (even(p.dv_, p.dv) ? 1 : 0) | (even(p.dq, p.dk) && even(p.dk_, p.dk) ? 2 : 0);
  const unsigned grid = (unsigned)(items < sm_count() ? items : sm_count());
  delta_grad_kernel<R><<<grid, kThreads, R::kBytes, st>>>(p, maps, items, pairs);
  DYNCONV_CHECK_LAUNCH("delta_grad_kernel");
  return DYNCONV_OK;
}

}  // namespace

int grad_launch(const Backward& p, int dtype, cudaStream_t st) {
  return dtype == DYNCONV_DTYPE_F32 ? go<Grad<3, 32>>(p, st) : go<Grad<1, 64>>(p, st);
}

}  // namespace dr

DYNCONV_DEFINE_ERROR_ACCESSOR(dr_grad_error_word)

}  // namespace dynconv
