// delta_grad.cu -- the gradients of the gated delta rule from what the chains left for every chunk: the state before it, r,
// dU and the gradient of the state after it (formulas: delta_rule.cuh).
//
// A CTA of eight warps takes one (batch row, head, chunk) after another.  v's columns come in slabs, the next one by TMA
// while this one is worked on.  A warp has 16 tokens and, of dk, a half (a quarter with chunks of 32): it sums
// dO S0^T, r dS1^T and dU S0^T over the slabs, and some blocks of the triangles dO r^T and dU r^T.
// These become W and N, which go through shared memory into the products with K and Q; their products with
// Q K^T and K K^T, entry by entry, are what the log decays' gradients are sums of.  Row sums and column sums
// of the same numbers are taken, so what has to cancel does.
//
// 4 x 4096 tokens, 16 heads of 128 x 128: 440 us for 0.9 GB.  No unit is near its limit (issue 32%, matrix units 34%, shared memory
// 41%, DRAM 24%): eight warps of 255 registers, all that an SM holds, wait for their own instructions, and spill 260 bytes (none
// with dk <= 64 or in fp32); sixteen warps of half as much each took 460 us.
// Items go heads first, since the heads of the same tokens share what they read.
#include "delta_rule.cuh"

namespace dynconv {
namespace dr {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;

// KK: 16-column pieces of dk, 4 or 8 (columns behind dk are zeros in the tiles of K and Q, and read as zeros from states)
template <int PX_, int C_, int KK_>
struct Grad {
  static constexpr int PX = PX_, C = C_, NB = C / 16, kGroups = kWarps / NB, KK = KK_, NT = 2 * KK / kGroups;  // a warp's 8-column tiles of dk
  // a group of warps has every kGroups / 2-th block column of one of the triangles
  static constexpr int kStep = kGroups / 2, kBlocks = NB > kStep ? NB / kStep : 1;
  static constexpr int PU = PX == 1 ? 2 : 3, PS = PX == 1 ? 1 : 3;  // parts of r and dU, of the states
  static constexpr int kSlab = PX == 1 ? 4 : 2;                     // slices of 16 columns of v
  static constexpr int kTile = C * kMaxKey, kSquare = C + 8;
  using E = typename std::conditional<PX_ == 1, __nv_bfloat16, float>::type;
  static constexpr int kRow = 16 * (int)sizeof(E), kDo = C * kRow, kU = NB * 512;  // bytes of a slice: of dO (tile: [C][kSlab * 16]), of one
                                                                                   // part of r or dU
  static_assert(kSlab * kRow == 128, "a tile of dO has rows of 128 bytes");
  static constexpr int kS = KK * 512;                                 // of one part of a state, at most
  static constexpr int kSlabBytes = kSlab * (kDo + 2 * PU * kU + 2 * PS * kS);
  static constexpr int kKq = 2 * PX * kTile * 2, kWn = 2 * PX * C * kSquare * 2;
  static constexpr int kBytes = 1024 + 2 * kSlabBytes + kKq + kWn;
  // where a slab's parts begin, the parts of each kSlab slices apart
  static constexpr uint32_t kR = kSlab * kDo, kDu = kR + PU * kSlab * kU, kS0 = kDu + PU * kSlab * kU, kDs = kS0 + PS * kSlab * kS;
};

// A 16 x 16 block kept as four matrices of 128 bytes is read transposed, as second operand, or as first, whose
// middle two matrices are the other way about.
// So are a lane's offsets in it.
__device__ __forceinline__ uint32_t second_lane() { return (threadIdx.x & 31) * 16; }
__device__ __forceinline__ uint32_t first_lane() {
  const int l = threadIdx.x & 31;
  return ((l >> 4 & 1) + (l >> 2 & 2)) * 128 + (l & 7) * 16;
}

// c0, c1 += a b.  fp32: the sum by itself first, since the instruction's own additions are cut off, not rounded, and dk
// is a sum of some fifty of them.
template <int NA, int NB, int KEEP, bool ROUND>
__device__ __forceinline__ void add_parts(float (&c0)[4], float (&c1)[4], const uint32_t (&a)[NA][4], const uint32_t (&b)[NB][4]) {
  if constexpr (ROUND) {
    float x[2][4];
    zero(x[0]), zero(x[1]);
    mma_parts<NA, NB, KEEP>(x[0], x[1], a, b);
#pragma unroll
    for (int e = 0; e < 4; ++e) c0[e] += x[0][e], c1[e] += x[1][e];
  } else {
    mma_parts<NA, NB, KEEP>(c0, c1, a, b);
  }
}
// (out of line: the kernel has to stay in the instruction cache)
template <typename E>
__device__ __noinline__ void store2_slow(E* to, float x, float y, int n) {
  if (n > 0) to[0] = Elem<E>::from_f(x);
  if (n > 1) to[1] = Elem<E>::from_f(y);
}
template <typename E>
__device__ __forceinline__ void store2(E* to, float x, float y, int n, bool pairs) {
  if (pairs) {
    if (n <= 0) return;
    if constexpr (sizeof(E) == 2)
      *reinterpret_cast<uint32_t*>(to) = pack(x, y);
    else
      *reinterpret_cast<float2*>(to) = make_float2(x, y);
  } else {
    store2_slow(to, x, y, n);
  }
}

template <typename R, typename GT>
__global__ void __launch_bounds__(kThreads, 1) delta_grad_kernel(Backward p, const __grid_constant__ Maps maps, int items, int pairs) {
  constexpr int PX = R::PX, C = R::C, NB = R::NB, PU = R::PU, PS = R::PS, kSlab = R::kSlab, kSquare = R::kSquare;
  constexpr bool kRound = PX > 1;
  constexpr int NT = R::NT, KK = R::KK, KX = PX > PS ? PX : PS, KS = PU > PS ? PU : PS;
  using E = typename R::E;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t slab_full[2], kq_full;
  __shared__ int abort_flag;
  __shared__ Gates<C> gate;
  __shared__ float row_sum[R::kGroups][C], col_sum[2][NB][C], from_state[R::kGroups][C], to_state[R::kGroups][C], inner[kWarps];
  uint8_t* const smem = align_smem_1024(smem_raw);
  uint8_t *const k_tile = smem, *const q_tile = smem + R::kKq / 2, *const slabs = smem + R::kKq;
  __nv_bfloat16 *const W = (__nv_bfloat16*)(slabs + 2 * R::kSlabBytes), *const N = W + PX * C * kSquare;
  const int tid = threadIdx.x, l = tid & 31, warp = warp_index(), row = l >> 2, col = 2 * (l & 3);
  const int group = warp / NB, rb = group & 1 ? NB - 1 - warp % NB : warp % NB;  // (the triangle's long rows on different schedulers)
  const int chunks = (int)((p.T + C - 1) / C), n_k16 = (p.dk + 15) / 16, slices = (p.dv + 15) / 16, n_slabs = (slices + kSlab - 1) / kSlab;
  constexpr int halves = KK / 4;
  const int64_t all = (int64_t)p.B * p.H * chunks;
  if (tid == 0) {
    mbar_init(&slab_full[0], 1), mbar_init(&slab_full[1], 1), mbar_init(&kq_full, 1);
    abort_flag = 0;
    fence_barrier_init();
  }
  if (n_k16 < KK) {  // pieces of the states that no load writes
    for (int i = tid; i < 2 * R::kSlabBytes / 16; i += kThreads) ((uint4*)slabs)[i] = make_uint4(0, 0, 0, 0);
    fence_proxy_async_smem();
  }
  __syncthreads();
  // (one thread)
  // Items count heads first, then chunks: neighbouring SMs read neighbouring heads of the same tokens, whole pages of DRAM.
  auto place = [&](int item, int& b, int& h, int& c) {
    h = item % p.H;
    c = item / p.H % chunks, b = item / p.H / chunks;
    return (int64_t)(b * p.H + h) * chunks + c;  // among what the chains left
  };
  auto load_slab = [&](int nth, int slab, int at) {
    int b, h, c;
    const int64_t item = place(nth, b, h, c);
    const int first = slab * kSlab, n = min(kSlab, slices - first);
    uint8_t* const s = slabs + at * R::kSlabBytes;
    uint64_t* const bar = &slab_full[at];
    const uint32_t state = n * n_k16 * 512;
    mbar_arrive_expect_tx(bar, kSlab * R::kDo + n * 2 * PU * R::kU + 2 * PS * state);
    tma_load_4d(s, &maps.v, bar, first * 16 * (int)(sizeof(E) / 2), h, c * C, b, policy_evict_normal());
#pragma unroll 1
    for (int i = 0; i < PU; ++i) {
      const int64_t from = ((i * all + item) * slices + first) * (R::kU / 2);
      bulk_load(s + R::kR + i * kSlab * R::kU, p.rest + from, n * R::kU, bar);
      bulk_load(s + R::kDu + i * kSlab * R::kU, p.du + from, n * R::kU, bar);
    }
#pragma unroll 1
    for (int i = 0; i < PS; ++i) {
      const int64_t from = ((i * all + item) * slices + first) * n_k16 * 256;
#pragma unroll 1
      for (int v = 0; v < (n_k16 == KK ? 1 : n); ++v) {  // (slices lie KK pieces apart)
        const uint32_t one = n_k16 == KK ? state : n_k16 * 512;
        bulk_load(s + R::kS0 + (i * kSlab + v) * R::kS, p.states + from + v * n_k16 * 256, one, bar);
        bulk_load(s + R::kDs + (i * kSlab + v) * R::kS, p.dstates + from + v * n_k16 * 256, one, bar);
      }
    }
  };
  auto load_kq = [&](int nth) {
    int b, h, c;
    const int64_t item = place(nth, b, h, c);
    mbar_arrive_expect_tx(&kq_full, 2 * PX * halves * C * 128);
    if (p.pre.k) {
      for (int i = 0; i < PX; ++i) {
        const int64_t from = (item * PX + i) * halves * (C * 64);
        bulk_load(k_tile + i * R::kTile * 2, p.pre.k + from, halves * C * 128, &kq_full);
        bulk_load(q_tile + i * R::kTile * 2, p.pre.q + from, halves * C * 128, &kq_full);
      }
    } else {
      for (int d = 0; d < halves; ++d) {
        tma_load_4d(k_tile + d * C * 128, &maps.k, &kq_full, 64 * d, h, c * C, b, policy_evict_normal());
        tma_load_4d(q_tile + d * C * 128, &maps.q, &kq_full, 64 * d, h, c * C, b, policy_evict_normal());
      }
    }
  };
  const KeyLane key_across(false), key_down(true);
  const int s_down = lane_offset(kSquare, true), s_across = lane_offset(kSquare, false);
  const int o_row = 16 * rb + (l & 15);  // a lane's row of dO's tile as first operand; its piece is l / 16
  const int kk0 = group * NT / 2;  // its first 16 columns of dk
  uint32_t own_down[NT / 2];
#pragma unroll
  for (int m = 0; m < NT / 2; ++m) {
    const int kk = kk0 + m;
    own_down[m] = key_swizzle((l & 7) + 8 * (l >> 3 & 1), (2 * kk & 7) + (l >> 4)) + (kk >> 2) * (C * 128);
  }

  int n_loaded = -1;  // slabs worked on (-1: before the first one's load)
  for (int nth = blockIdx.x, done = 0; nth < items; nth += gridDim.x, ++done) {
    int b_, h_, c;
    const int64_t item = place(nth, b_, h_, c), b = b_, h = h_;
    const int64_t t0 = (int64_t)c * C;
    const int rows = (int)(p.T - t0 < C ? p.T - t0 : C);
    E* const dv_at = (E*)p.dv_.p + b * p.dv_.sb + h * p.dv_.sh + t0 * p.dv_.st;
    float beta_own[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) beta_own[i] = ((const Gates<C>*)p.pre.gates)[item].beta[16 * rb + row + 8 * i];
    float dq[NT][4], kr[NT][4], ku[NT][4];  // dO S0^T, r dS1^T, dU S0^T
    float X[R::kBlocks][2][4];              // blocks of dO r^T (even groups) or dU r^T
    float dot[2][4];                        // its diagonals add up to <dS1, S0>
#pragma unroll
    for (int n = 0; n < NT; ++n) zero(dq[n]), zero(kr[n]), zero(ku[n]);
#pragma unroll
    for (int j = 0; j < R::kBlocks; ++j) zero(X[j][0]), zero(X[j][1]);
    zero(dot[0]), zero(dot[1]);
    for (int slab = n_loaded < 0 ? -1 : 0; slab < n_slabs; ++slab, ++n_loaded) {
      const int at = n_loaded & 1;
      if (n_loaded >= 0 && !__syncthreads_and(mbar_wait(&slab_full[at], (n_loaded >> 1) & 1, kErrWaitMma, &abort_flag))) {
        if (tid == 0) {  // (what is in flight lands before the shared memory goes)
          mbar_drain(&slab_full[at], (n_loaded >> 1) & 1);
          if (slab > 0) mbar_drain(&kq_full, done & 1);
        }
        return;
      }
      if (tid == 0) {  // (everybody is done with the other slab, and with the keys of the item before)
        if (slab == 0) load_kq(nth);
        const int next = slab + 1 < n_slabs ? nth : nth + (int)gridDim.x;
        if (next < items) load_slab(next, slab + 1 < n_slabs ? slab + 1 : 0, at ^ 1);
      }
      if (slab < 0) continue;
      if (slab == 0) {
        const uint4* g = (const uint4*)p.pre.gates + item * (sizeof(Gates<C>) / 16);
        for (int i = tid; i < (int)sizeof(Gates<C>) / 16; i += kThreads) ((uint4*)&gate)[i] = g[i];
      }
      const int n = min(kSlab, slices - slab * kSlab);
      const uint32_t base = smem_u32(slabs) + at * R::kSlabBytes;
      uint32_t a_r = base + R::kR + rb * 512 + first_lane(), b_r = base + R::kR + (group >> 1) * 512 + second_lane();
      uint32_t b_s = base + R::kS0 + kk0 * 512 + second_lane();
#pragma unroll 1
      for (int v = 0; v < n; ++v, a_r += R::kU, b_r += R::kU, b_s += R::kS) {
        uint32_t dO[PX][4], r[PU][4], u[PU][4], f[NT / 2][PS][4], x[R::kBlocks][PU][4];
        if constexpr (PX == 1) {
          ldsm(dO[0], base + row_swizzle(128, o_row, 2 * v + (l >> 4)));
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 t = *reinterpret_cast<const float2*>(slabs + at * R::kSlabBytes + row_swizzle(128, 16 * rb + row + 8 * (e & 1), 4 * v + 2 * (e >> 1) + (col >> 2)) + 4 * (col & 3));
            uint32_t part[PX];
            split<PX>(t.x, t.y, part);
#pragma unroll
            for (int i = 0; i < PX; ++i) dO[i][e] = part[i];
          }
        }
#pragma unroll
        for (int i = 0; i < PU; ++i) ldsm_t(u[i], a_r + R::kDu - R::kR + i * kSlab * R::kU);
#pragma unroll
        for (int m = 0; m < NT / 2; ++m)
#pragma unroll
          for (int i = 0; i < PS; ++i) ldsm_t(f[m][i], b_s + m * 512 + i * kSlab * R::kS);
#pragma unroll
        for (int i = 0; i < PU; ++i) ldsm_t(r[i], a_r + i * kSlab * R::kU);
#pragma unroll
        for (int m = 0; m < NT / 2; ++m) add_parts<PX, PS, KX, kRound>(dq[2 * m], dq[2 * m + 1], dO, f[m]);
        // (all tiles' products of one pair of parts, then of the next: none waits for the one before)
        if constexpr (kRound) {
#pragma unroll
          for (int m = 0; m < NT / 2; ++m) add_parts<PU, PS, KS, true>(ku[2 * m], ku[2 * m + 1], u, f[m]);
        } else {
#pragma unroll
          for (int t = KS - 1; t >= 0; --t)
#pragma unroll
            for (int i = 0; i < PU; ++i)
#pragma unroll
              for (int m = 0; m < NT / 2; ++m)
                if (t - i >= 0 && t - i < PS) {
                  mma(ku[2 * m], u[i], f[m][t - i][0], f[m][t - i][1]);
                  mma(ku[2 * m + 1], u[i], f[m][t - i][2], f[m][t - i][3]);
                }
        }
        uint32_t g[NT / 2][PS][4];
#pragma unroll
        for (int m = 0; m < NT / 2; ++m)
#pragma unroll
          for (int i = 0; i < PS; ++i) ldsm_t(g[m][i], b_s + R::kDs - R::kS0 + m * 512 + i * kSlab * R::kS);
#pragma unroll
        for (int c = 0; c < R::kBlocks; ++c)
          if ((group >> 1) + c * R::kStep <= rb)
#pragma unroll
            for (int i = 0; i < PU; ++i) ldsm_t(x[c][i], b_r + c * R::kStep * 512 + i * kSlab * R::kU);
        // <dS1, S0>: the trace of a product; each piece by one of the warps that read it
        if ((v & (NB - 1)) == rb) {
#pragma unroll
          for (int m = 0; m < NT / 2; ++m) {
            uint32_t t[PS][4];
#pragma unroll
            for (int i = 0; i < PS; ++i) t[i][0] = f[m][i][0], t[i][1] = f[m][i][2], t[i][2] = f[m][i][1], t[i][3] = f[m][i][3];
            mma_parts<PS, PS, PS>(dot[0], dot[1], t, g[m]);
          }
        }
        if constexpr (kRound) {
#pragma unroll
          for (int m = 0; m < NT / 2; ++m) add_parts<PU, PS, KS, true>(kr[2 * m], kr[2 * m + 1], r, g[m]);
        } else {
#pragma unroll
          for (int t = KS - 1; t >= 0; --t)
#pragma unroll
            for (int i = 0; i < PU; ++i)
#pragma unroll
              for (int m = 0; m < NT / 2; ++m)
                if (t - i >= 0 && t - i < PS) {
                  mma(kr[2 * m], r[i], g[m][t - i][0], g[m][t - i][1]);
                  mma(kr[2 * m + 1], r[i], g[m][t - i][2], g[m][t - i][3]);
                }
        }
#pragma unroll
        for (int c = 0; c < R::kBlocks; ++c) {
          if ((group >> 1) + c * R::kStep > rb) continue;
          if (group & 1)
            add_parts<PU, PU, PU, kRound>(X[c][0], X[c][1], u, x[c]);
          else
            add_parts<PX, PU, PU, kRound>(X[c][0], X[c][1], dO, x[c]);
        }
        if (group == (v & (R::kGroups - 1))) {
          // dV = beta dU
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int t = 16 * rb + row + 8 * (e & 1), d = (slab * kSlab + v) * 16 + 8 * (e >> 1) + col;
            float x0 = low(u[PU - 1][e]), x1 = high(u[PU - 1][e]);
#pragma unroll
            for (int i = PU - 2; i >= 0; --i) x0 += low(u[i][e]), x1 += high(u[i][e]);
            const float beta = e & 1 ? beta_own[1] : beta_own[0];
            if (t < rows) store2(dv_at + (int64_t)t * p.dv_.st + d, x0 * beta, x1 * beta, p.dv - d, pairs & 1);
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
    {
      const bool is_n = group & 1;
      float Y[R::kBlocks][2][4];
#pragma unroll
      for (int n = 0; n < R::kBlocks; ++n) zero(Y[n][0]), zero(Y[n][1]);
      const uint32_t a_at = is_n ? k_at : q_at;
#pragma unroll 1
      for (int hf = 0; hf < halves; ++hf)
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          uint32_t a[PX][4];
#pragma unroll
          for (int i = 0; i < PX; ++i) ldsm(a[i], a_at + hf * (C * 128) + 2 * i * R::kTile + key_down.at<C>(rb, kk));
#pragma unroll
          for (int n = 0; n < R::kBlocks; ++n) {
            const int j = (group >> 1) + n * R::kStep;
            if (j > rb) continue;
            uint32_t f[PX][4];
#pragma unroll
            for (int i = 0; i < PX; ++i) ldsm(f[i], k_at + hf * (C * 128) + 2 * i * R::kTile + key_across.at<C>(j, kk));
            mma_parts<PX, PX, PX>(Y[n][0], Y[n][1], a, f);
          }
        }
      // the gates, for all blocks before the first is written: loads do not pass stores
      float f_r[2], hi_r[2], lo_r[2];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int r = 16 * rb + row + 8 * half;
        f_r[half] = is_n ? -gate.beta[r] : p.scale, hi_r[half] = gate.hi[r], lo_r[half] = gate.lo[r];
      }
      float sums[2] = {0.f, 0.f}, below[R::kBlocks][2][2], own[2] = {0.f, 0.f};
#pragma unroll
      for (int jn = 0; jn < R::kBlocks; ++jn) {
        const int j = (group >> 1) + jn * R::kStep;
        if (j > rb) continue;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const int cc = 16 * j + 8 * n + col;
          const float2 hi = *reinterpret_cast<const float2*>(gate.hi + cc), lo = *reinterpret_cast<const float2*>(gate.lo + cc);
          const float2 beta = *reinterpret_cast<const float2*>(gate.beta + cc);
          below[jn][n][0] = below[jn][n][1] = 0.f;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int r = 16 * rb + row + 8 * half;
            float &x = X[jn][n][2 * half], &y = X[jn][n][2 * half + 1];
            own[half] = cc == r ? x : cc + 1 == r ? y : own[half];
            x *= f_r[half] * beta.x * exp2_fast((hi_r[half] - hi.x) + (lo_r[half] - lo.x));
            y *= f_r[half] * beta.y * exp2_fast((hi_r[half] - hi.y) + (lo_r[half] - lo.y));
            const int last = is_n ? r - 1 : r;
            x = cc <= last ? x : 0.f, y = cc < last ? y : 0.f;
            // (a token's own term does not depend on the decays)
            const float mx = cc < r ? x * Y[jn][n][2 * half] : 0.f, my = cc + 1 < r ? y * Y[jn][n][2 * half + 1] : 0.f;
            sums[half] += mx + my;
            below[jn][n][0] += mx, below[jn][n][1] += my;
          }
        }
      }
#pragma unroll
      for (int d = 4; d < 32; d <<= 1)
#pragma unroll
        for (int jn = 0; jn < R::kBlocks; ++jn)
          if ((group >> 1) + jn * R::kStep <= rb)
#pragma unroll
            for (int n = 0; n < 2; ++n) {
              below[jn][n][0] += __shfl_xor_sync(0xffffffffu, below[jn][n][0], d);
              below[jn][n][1] += __shfl_xor_sync(0xffffffffu, below[jn][n][1], d);
            }
      __nv_bfloat16* const out = (is_n ? N : W) + (16 * rb + row) * kSquare + col;
#pragma unroll
      for (int jn = 0; jn < R::kBlocks; ++jn) {
        const int j = (group >> 1) + jn * R::kStep;
        if (j > rb) continue;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const int cc = 16 * j + 8 * n;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            uint32_t part[PX];
            split<PX>(X[jn][n][2 * half], X[jn][n][2 * half + 1], part);
#pragma unroll
            for (int i = 0; i < PX; ++i) *reinterpret_cast<uint32_t*>(out + i * C * kSquare + 8 * half * kSquare + cc) = part[i];
          }
          if (row == 0) *reinterpret_cast<float2*>(&col_sum[is_n][rb][cc + col]) = make_float2(below[jn][n][0], below[jn][n][1]);
        }
      }
      // dbeta: the diagonal of dU r^T
      if (is_n && (rb - (group >> 1)) % R::kStep == 0 && rb >= (group >> 1)) {
        GT* const db = (GT*)p.dbeta.p + b * p.dbeta.sb + h * p.dbeta.sh + t0 * p.dbeta.st;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int r = 16 * rb + row + 8 * half, c = (row + 8 * half) & 7;  // (the lane that holds column r)
          if ((c >> 1) == (l & 3) && r < rows) db[r * p.dbeta.st] = Elem<GT>::from_f(own[half]);
        }
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        sums[half] += __shfl_xor_sync(0xffffffffu, sums[half], 1);
        sums[half] += __shfl_xor_sync(0xffffffffu, sums[half], 2);
        if ((l & 3) == 0) row_sum[group][16 * rb + row + 8 * half] = sums[half];
      }
    }
    {
      float x = 0.f;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (row + 8 * (e >> 1) == 8 * n + col + (e & 1)) x += dot[n][e];
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
      if (l == 0) inner[warp] = x;
    }
    // the states' parts, scaled, and what the decays get from them
    {
      float from[2] = {0.f, 0.f}, to[2] = {0.f, 0.f};
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int r = 16 * rb + row + 8 * half;
        const float fq = p.scale * gate.e[r], fr = gate.out[r] * gate.beta[r], fu = -gate.beta[r] * gate.e[r];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const int kk = kk0 + n / 2, piece = (2 * kk + (n & 1)) & 7;
          const uint32_t at = (kk >> 2) * (C * 128) + 2048 * rb + key_swizzle(row + 8 * half, piece) + 2 * col;
          float qx, qy, kx, ky;
#pragma unroll
          for (int i = PX - 1; i >= 0; --i) {
            const uint32_t uq = *reinterpret_cast<const uint32_t*>(q_tile + 2 * i * R::kTile + at);
            const uint32_t uk = *reinterpret_cast<const uint32_t*>(k_tile + 2 * i * R::kTile + at);
            if (i == PX - 1)
              qx = low(uq), qy = high(uq), kx = low(uk), ky = high(uk);
            else
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
    if (warp == kWarps - 1) {
      // dlog_decay: sums of tokens from t on, and before t
      constexpr int M = C / 32;
      float a[M], e[M];
#pragma unroll
      for (int i = 0; i < M; ++i) {
        const int t = l * M + i;
        a[i] = e[i] = 0.f;
        float below = 0.f;
#pragma unroll
        for (int j = 0; j < NB; ++j) below += j >= t / 16 ? col_sum[0][j][t] + col_sum[1][j][t] : 0.f;
        a[i] -= below;
#pragma unroll
        for (int g = 0; g < R::kGroups; ++g) a[i] += row_sum[g][t] + from_state[g][t], e[i] += to_state[g][t];
      }
      float total = 0.f;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) total += inner[i];
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
        if (t < rows) ((GT*)p.dg.p)[b * p.dg.sb + h * p.dg.sh + (t0 + t) * p.dg.st] = Elem<GT>::from_f(x);
        earlier += e[i];
      }
    }
    // dQ += W K, dK += W^T Q + (N + N^T) K
#pragma unroll 1
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
        uint32_t f[PX][4], g[PX][4];
        const uint32_t at = own_down[m] + j * 2048;
#pragma unroll
        for (int i = 0; i < PX; ++i) {
          ldsm_t(f[i], k_at + 2 * i * R::kTile + at);
          if (j >= rb) ldsm_t(g[i], q_at + 2 * i * R::kTile + at);
        }
        if (j <= rb) {
          add_parts<PX, PX, PX, kRound>(dq[2 * m], dq[2 * m + 1], wa, f);
          add_parts<PX, PX, PX, kRound>(kr[2 * m], kr[2 * m + 1], na, f);
        }
        if (j >= rb) {
          add_parts<PX, PX, PX, kRound>(kr[2 * m], kr[2 * m + 1], nt, f);
          add_parts<PX, PX, PX, kRound>(kr[2 * m], kr[2 * m + 1], wt, g);
        }
      }
    }
    // bf16: two lanes exchange halves of two tiles, so that each stores four columns of one
    E* const dq_at = (E*)p.dq.p + b * p.dq.sb + h * p.dq.sh + t0 * p.dq.st;
    E* const dk_at = (E*)p.dk_.p + b * p.dk_.sb + h * p.dk_.sh + t0 * p.dk_.st;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int t = 16 * rb + row + 8 * half;
      E *const to_q = dq_at + (int64_t)t * p.dq.st, *const to_k = dk_at + (int64_t)t * p.dk_.st;
      if (sizeof(E) == 2 && (pairs & 4)) {
        const int odd = l & 1;
#pragma unroll
        for (int n = 0; n < NT; n += 2) {
          const int d = 8 * (group * NT + n + odd) + col - 2 * odd;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float(&x)[4] = i ? kr[n] : dq[n];
            const float(&y)[4] = i ? kr[n + 1] : dq[n + 1];
            const uint32_t mine = pack(x[2 * half], x[2 * half + 1]), next = pack(y[2 * half], y[2 * half + 1]);
            const uint32_t got = __shfl_xor_sync(0xffffffffu, odd ? mine : next, 1);
            if (t < rows && d < p.dk)
              *reinterpret_cast<uint2*>((i ? to_k : to_q) + d) = odd ? make_uint2(got, next) : make_uint2(mine, got);
          }
        }
      } else if (t < rows) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const int d = 8 * (group * NT + n) + col;
          store2(to_q + d, dq[n][2 * half], dq[n][2 * half + 1], p.dk - d, pairs & 2);
          store2(to_k + d, kr[n][2 * half], kr[n][2 * half + 1], p.dk - d, pairs & 2);
        }
      }
    }
  }
}

// Rows whose numbers can be written n at a time.
bool whole(const View& v, int width, int n, int elem) {
  return width % n == 0 && v.sb % n == 0 && v.st % n == 0 && v.sh % n == 0 && (reinterpret_cast<uintptr_t>(v.p) & (n * elem - 1)) == 0;
}

template <typename R, typename GT>
int launch(const Backward& p, cudaStream_t st) {
  const cudaError_t e = cudaFuncSetAttribute(delta_grad_kernel<R, GT>, cudaFuncAttributeMaxDynamicSharedMemorySize, R::kBytes);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return cuda_status(e, "cudaFuncSetAttribute(delta_grad)");
  }
  Maps maps{};
  int s;
  if (!p.pre.k && ((s = view_map(&maps.k, p.k, p.B, p.T, p.H, p.dk, 2, 64, R::C)) || (s = view_map(&maps.q, p.q, p.B, p.T, p.H, p.dk, 2, 64, R::C))))
    return s;
  if ((s = value_map(&maps.v, p.pre, p.d_o, p.B, p.T, p.H, p.dv, sizeof(typename R::E), 16 * R::kSlab, R::C))) return s;
  const int64_t items = (int64_t)p.B * p.H * ((p.T + R::C - 1) / R::C);
  if (items > INT32_MAX - 65536) return set_error(DYNCONV_ERR_SHAPE, "gated delta rule: B*H*T too large");
  const int elem = sizeof(typename R::E);
  const int pairs = (whole(p.dv_, p.dv, 2, elem) ? 1 : 0) | (whole(p.dq, p.dk, 2, elem) && whole(p.dk_, p.dk, 2, elem) ? 2 : 0) |
                    (whole(p.dq, p.dk, 4, elem) && whole(p.dk_, p.dk, 4, elem) ? 4 : 0);
  const unsigned grid = (unsigned)(items < sm_count() ? items : sm_count());
  delta_grad_kernel<R, GT><<<grid, kThreads, R::kBytes, st>>>(p, maps, (int)items, pairs);
  DYNCONV_CHECK_LAUNCH("delta_grad_kernel");
  return DYNCONV_OK;
}
template <typename R>
int go(const Backward& p, cudaStream_t st) {
  return p.gates32 ? launch<R, float>(p, st) : launch<R, typename R::E>(p, st);
}

}  // namespace

int grad_launch(const Backward& p, int dtype, cudaStream_t st) {
  if (p.dk <= 64) return dtype == DYNCONV_DTYPE_F32 ? go<Grad<3, 32, 4>>(p, st) : go<Grad<1, 64, 4>>(p, st);
  return dtype == DYNCONV_DTYPE_F32 ? go<Grad<3, 32, 8>>(p, st) : go<Grad<1, 64, 8>>(p, st);
}

}  // namespace dr

DYNCONV_DEFINE_ERROR_ACCESSOR(dr_grad_error_word)

}  // namespace dynconv
