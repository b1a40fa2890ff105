// delta_prep.cu -- what the chunks of the gated delta rule need before their state is known: the gates, and
// from K and Q the triangular matrices T and P (formulas: delta_rule.cuh).  A CTA of four warps per
// chunk and head, heads of the same tokens side by side, since they share the rows of K and Q that a fused projection
// lays out together; five CTAs on an SM, so that one's products fill the other's barriers.  Apart from the chains,
// because T needs nothing of them: as helper warps of a chain's CTA the same work held up the chain (440 against
// 360 us for the forward).
//
// 4 x 4096 tokens, 16 heads of 128: 63 us for 134 MB read and 90 MB written; bound by its barriers and by the
// instructions that split numbers into parts (issue 46%, DRAM 25%), not by memory.  32768 tokens with three parts: 145 us.
#include "delta_rule.cuh"

namespace dynconv {
namespace dr {
namespace {

constexpr int kThreads = 128;

// A token's gates, read ahead by the lanes of one warp.
template <int C>
struct TokenGates {
  float g[C / 32], beta[C / 32];
};

// Log decays below this give a factor of zero in fp32; as minus infinity they would make NaN of a difference.
constexpr float kLeastDecay = -104.f;

// Running sum of the log decays and what follows from it, by one warp.  The sum is held as two floats: a
// difference of two sums is the logarithm of a factor, and fp32 would leave 2^-24 of the sums' size
// in it.  With `check`, `s.bad` becomes the first token whose gates are not finite.
template <int C>
__device__ __noinline__ void make_gates(Gates<C>& s, TokenGates<C> own, bool check) {
  constexpr int N = C / 32;
  const int l = threadIdx.x & 31;
  Two a[N];
  int bad = C;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float g = own.g[i] < kLeastDecay ? kLeastDecay : own.g[i];  // (a NaN stays one)
    if (!(g < INFINITY) || !(fabsf(own.beta[i]) < INFINITY)) bad = min(bad, l * N + i);
    const float p = __fmul_rn(g, 1.44269502f);  // log2(e) in two floats
    a[i] = quick_two(p, fmaf(g, 1.44269502f, -p) + g * 1.92596303e-8f);
    if (i) a[i] = add(a[i - 1], a[i]);
  }
  if (check) {
    bad = __reduce_min_sync(0xffffffffu, bad);
    if (l == 0) s.bad = bad;
  }
  Two sum = a[N - 1];
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const Two t{__shfl_up_sync(0xffffffffu, sum.hi, d), __shfl_up_sync(0xffffffffu, sum.lo, d)};
    if (l >= d) sum = add(t, sum);
  }
  const Two total{__shfl_sync(0xffffffffu, sum.hi, 31), __shfl_sync(0xffffffffu, sum.lo, 31)};
  Two before{__shfl_up_sync(0xffffffffu, sum.hi, 1), __shfl_up_sync(0xffffffffu, sum.lo, 1)};
  if (l == 0) before = Two{0.f, 0.f};
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const Two b = add(before, a[i]);
    const int t = l * N + i;
    s.hi[t] = b.hi, s.lo[t] = b.lo;
    s.beta[t] = own.beta[i];
    s.e[t] = exp2_two(b);
    s.out[t] = exp2_two(add(total, Two{-b.hi, -b.lo}));
  }
  if (l == 31) s.total = exp2_two(total);
}

// K or Q where no tensor map reads it: fp32, which is split into its parts, and bf16 of odd widths.  Two columns per
// thread at a time, zeros behind the rows and columns that are there.
template <int C, int PARTS, typename E>
__device__ __noinline__ void load_slow(uint8_t* dst, const E* src, int64_t step, int rows, int cols, int halves) {
  for (int i = threadIdx.x; i < C * 32 * halves; i += kThreads) {
    const int r = i / (32 * halves), c = 2 * (i % (32 * halves));
    const E* from = src + r * step + c;
    const float x = r < rows && c < cols ? Elem<E>::to_f(from[0]) : 0.f;
    const float y = r < rows && c + 1 < cols ? Elem<E>::to_f(from[1]) : 0.f;
    uint32_t p[PARTS];
    split<PARTS>(x, y, p);
#pragma unroll
    for (int k = 0; k < PARTS; ++k)
      *reinterpret_cast<uint32_t*>(dst + (k * 2 + (c >> 6)) * (C * 128) + key_swizzle(r, (c & 63) >> 3) + 2 * (c & 7)) = p[k];
  }
}

// ------------------------------------------------------------------------- T and P

// T, the inverse of I + A, on four warps, in blocks of 16: diagonal blocks by substitution in fp32
// (a lane per column), then T_ij = -T_ii (sum_k A_ik T_kj) on matrix instructions, transposed, so that
// the inner sum is the next product's first operand as it stands.  Off-diagonal blocks
// A_ij lie in the place of the blocks (j, i) of `t`, which T leaves empty; diagonal ones in `diag`.
template <typename G>
struct Inverse {
  static constexpr int C = G::C, NP = G::NP, kS = G::kSquare, kPart = C * kS;

  static __device__ __forceinline__ void diagonal(__nv_bfloat16* t, const float* diag) {
    const int w = warp_index(), j = threadIdx.x & 15;
    if (w >= G::kBlocks) return;
    const float4* a = (const float4*)(diag + w * 256);
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < i; k += 4) {
        const float4 f = a[i * 4 + k / 4];  // (zero from column i on)
        sum[0] = fmaf(f.x, x[k], sum[0]);
        if (k + 1 < i) sum[1] = fmaf(f.y, x[k + 1], sum[1]);
        if (k + 2 < i) sum[2] = fmaf(f.z, x[k + 2], sum[2]);
        if (k + 3 < i) sum[3] = fmaf(f.w, x[k + 3], sum[3]);
      }
      x[i] = i == j ? 1.f : -((sum[0] + sum[1]) + (sum[2] + sum[3]));
    }
    if ((threadIdx.x & 31) < 16) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float r = x[i];
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          const __nv_bfloat16 h = __float2bfloat16_rn(r);
          t[p * kPart + (16 * w + i) * kS + 16 * w + j] = h;
          r -= __bfloat162float(h);
        }
      }
    }
  }

  // T_ij from A_ab (a0 <= a <= i, j <= b <= b1) and the blocks of T that are done; one warp.
  static __device__ __forceinline__ void block(__nv_bfloat16* t, int i, int j, int a0, int b1) {
    const uint32_t base = smem_u32(t);
    const int across = lane_offset(kS, false);
    auto at = [&](int p, int bi, int bj, int lane) { return base + 2 * (p * kPart + 16 * bi * kS + 16 * bj + lane); };
    float y0[4], y1[4];
    zero(y0), zero(y1);
    for (int a = a0; a <= i; ++a) {
      float x0[4], x1[4];
      zero(x0), zero(x1);
      for (int b = j; b <= b1; ++b) {
        uint32_t l[NP][4], r[NP][4];
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          ldsm_t(l[p], at(p, b, j, across));  // T_bj, transposed
          ldsm(r[p], at(p, b, a, across));    // A_ab
        }
        mma_parts<NP, NP, NP>(x0, x1, l, r);
      }
      uint32_t l[NP][4], r[NP][4];
      operand<NP>(x0, x1, l);
#pragma unroll
      for (int p = 0; p < NP; ++p) ldsm(r[p], at(p, i, a, across));  // T_ia
      mma_parts<NP, NP, NP>(y0, y1, l, r);
    }
    uint32_t l[NP][4];
#pragma unroll
    for (int e = 0; e < 4; ++e) y0[e] = -y0[e], y1[e] = -y1[e];
    operand<NP>(y0, y1, l);
#pragma unroll
    for (int p = 0; p < NP; ++p) stsm_t(at(p, i, j, across), l[p][0], l[p][1], l[p][2], l[p][3]);
  }

  static __device__ __forceinline__ void run(__nv_bfloat16* t, const float* diag) {
    const int w = warp_index();
    diagonal(t, diag);
    __syncthreads();
    for (int level = 0; level < G::kBlocks / 2; ++level) {
      const int i = level ? 2 + (w >> 1) : 2 * w + 1, j = level ? w & 1 : 2 * w;
      if (level || w < G::kBlocks / 2) block(t, i, j, level ? 2 : i, level ? 1 : j);
      __syncthreads();
    }
  }
};

// A = L beta (backward: beta L) and P of a chunk from its K and Q.  Row block i of either has i + 1 blocks of
// 16 x 16.  Of four row blocks, warp 0 takes A's first and last, warp 1 the two between them, warps 2 and 3 the same of P:
// five blocks each, of which the first is of the first row block and the last three of the second.
// (Of two row blocks, warp 0 takes A's and warp 2 P's.)
template <typename G>
struct Scores {
  static constexpr int C = G::C, kS = G::kSquare, kPart = C * kS, PX = G::PX, NB = G::kBlocks, kUnits = NB == 4 ? 5 : 3;
  float X[kUnits][2][4];
  int w, row, col, i0, i1;
  bool is_p;

  __device__ __forceinline__ Scores() {
    const int l = threadIdx.x & 31;
    w = warp_index(), row = l >> 2, col = 2 * (l & 3);
    is_p = w >= 2;
    i0 = NB == 4 ? w & 1 : 0, i1 = NB - 1 - i0;  // the row blocks
  }
  __device__ __forceinline__ bool idle() const { return NB == 2 && (w & 1); }
  __device__ __forceinline__ int block_of(int u) const { return u <= i0 ? u : u - i0 - 1; }

  __device__ __forceinline__ void products(uint32_t k, uint32_t q, int n_k16) {
    if (idle()) return;
#pragma unroll
    for (int u = 0; u < kUnits; ++u) zero(X[u][0]), zero(X[u][1]);
    const KeyLane across(false), down(true);
    const uint32_t a_at = is_p ? q : k;
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) {
      if (kk >= n_k16) continue;
      uint32_t a0[PX][4], a1[PX][4], am[PX][4];
#pragma unroll
      for (int i = 0; i < PX; ++i) {
        ldsm(a0[i], a_at + 2 * i * G::kTile + down.at<C>(i0, kk));
        ldsm(a1[i], a_at + 2 * i * G::kTile + down.at<C>(i1, kk));
#pragma unroll
        for (int e = 0; e < 4; ++e) am[i][e] = i0 ? a0[i][e] : a1[i][e];
      }
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        uint32_t b[PX][4];
#pragma unroll
        for (int i = 0; i < PX; ++i) ldsm(b[i], k + 2 * i * G::kTile + across.at<C>(block_of(u), kk));
        if (u == 0)
          mma_parts<PX, PX, PX>(X[u][0], X[u][1], a0, b);
        else if (u == 1)
          mma_parts<PX, PX, PX>(X[u][0], X[u][1], am, b);
        else
          mma_parts<PX, PX, PX>(X[u][0], X[u][1], a1, b);
      }
    }
  }

  // The first token whose key is not finite: its square shows it.
  __device__ __forceinline__ void find_bad(int* bad) const {
    if (idle() || is_p) return;
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int i = u <= i0 ? i0 : i1;
      if (block_of(u) != i) continue;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (row + 8 * (e >> 1) == 8 * n + col + (e & 1) && !(X[u][n][e] < INFINITY)) atomicMin(bad, 16 * i + row + 8 * (e >> 1));
    }
  }

  // Applies the gates, all blocks before the first is written: loads do not pass stores.
  template <bool BACK>
  __device__ __forceinline__ void scale(const Gates<C>& s, float scale) {
    if (idle()) return;
    float hi_r[2][2], lo_r[2][2], beta_r[2][2];  // of the two row blocks
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int r = 16 * (b ? i1 : i0) + row + 8 * half;
        hi_r[b][half] = s.hi[r], lo_r[b][half] = s.lo[r], beta_r[b][half] = is_p ? scale : s.beta[r];
      }
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int i = u <= i0 ? i0 : i1, j = block_of(u);
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const int c = 16 * j + 8 * n + col;
        const float2 hi = *reinterpret_cast<const float2*>(s.hi + c), lo = *reinterpret_cast<const float2*>(s.lo + c);
        const float2 beta = *reinterpret_cast<const float2*>(s.beta + c);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int r = 16 * i + row + 8 * half, last = is_p ? r : r - 1;  // the last column that counts
          // (block 0 is of the first row block, blocks from 2 on of the second)
          const bool b1 = u >= 2 || (u == 1 && i0 == 0);
          const float h = b1 ? hi_r[1][half] : hi_r[0][half], l = b1 ? lo_r[1][half] : lo_r[0][half];
          const float f = b1 ? beta_r[1][half] : beta_r[0][half];
          float &x = X[u][n][2 * half], &y = X[u][n][2 * half + 1];
          x *= (BACK || is_p ? f : beta.x) * exp2_fast((h - hi.x) + (l - lo.x));
          y *= (BACK || is_p ? f : beta.y) * exp2_fast((h - hi.y) + (l - lo.y));
          x = c <= last ? x : 0.f, y = c < last ? y : 0.f;
        }
      }
    }
  }

  __device__ __forceinline__ void write(__nv_bfloat16* t, float* diag, __nv_bfloat16* p_out) const {
    if (idle()) return;
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int i = u <= i0 ? i0 : i1, j = block_of(u);
      __nv_bfloat16* const to = is_p ? p_out + (16 * i + row) * kS + 16 * j + col : t + (16 * j + row) * kS + 16 * i + col;
      float* const to_diag = diag + i * 256 + row * 16 + col;
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const float x = X[u][n][2 * half], y = X[u][n][2 * half + 1];
          const int at = 8 * half * kS + 8 * n;
          if (is_p) {
            uint32_t p[G::PP];
            split<G::PP>(x, y, p);
#pragma unroll
            for (int e = 0; e < G::PP; ++e) *reinterpret_cast<uint32_t*>(to + e * kPart + at) = p[e];
          } else if (j == i) {
            *reinterpret_cast<float2*>(to_diag + 8 * half * 16 + 8 * n) = make_float2(x, y);
          } else {
            uint32_t p[G::NP];
            split<G::NP>(x, y, p);
#pragma unroll
            for (int e = 0; e < G::NP; ++e) *reinterpret_cast<uint32_t*>(to + e * kPart + at) = p[e];
          }
        }
    }
  }
};

template <typename G>
struct PrepSmem {
  static constexpr int kT = G::NP * G::C * G::kSquare, kP = G::PP * G::C * G::kSquare;  // elements
  static constexpr int kKq = 2 * G::PX * G::kTile, kSpace = kT + kP > kKq ? kT + kP : kKq;  // T and P take K's and Q's place
  static constexpr size_t kBytes = 1024 + 2 * (size_t)kSpace + G::kBlocks * 1024 + sizeof(Gates<G::C>);
};

template <typename G, bool BACK, typename GT>
__global__ void __launch_bounds__(kThreads) delta_prep_kernel(Prepared to, const __grid_constant__ Maps maps, View k, View q, View v, View g,
                                                              View beta, int H, int64_t T, int dk, int dv, float scale) {
  constexpr int C = G::C, PX = G::PX, NB = G::kBlocks;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full;
  __shared__ int abort_flag;
  uint8_t* const smem = align_smem_1024(smem_raw);
  using E = typename G::T;
  uint8_t *const ks = smem, *const qs = ks + 2 * PX * G::kTile;
  __nv_bfloat16 *const t = (__nv_bfloat16*)ks, *const p = t + PrepSmem<G>::kT;
  float* const diag = (float*)(smem + 2 * PrepSmem<G>::kSpace);
  Gates<C>& s = *(Gates<C>*)(diag + NB * 256);
  const int tid = threadIdx.x, lane = tid & 31, w = warp_index(), n_k16 = (dk + 15) / 16, halves = dk > 64 ? 2 : 1;
  // (heads first: CTAs that run together read neighbouring heads of the same tokens, whole pages of DRAM)
  const int64_t h = blockIdx.x % H, chunk = blockIdx.x / H, b = blockIdx.y, bh = b * H + h, t0 = chunk * C;
  const int64_t at = bh * ((T + C - 1) / C) + chunk;
  const int rows = (int)(T - t0 < C ? T - t0 : C);
  if (to.k) {
#pragma unroll 1
    for (int i = 0; i < 2; ++i) {
      const View& x = i ? q : k;
      load_slow<C, PX, E>(i ? qs : ks, (const E*)x.p + b * x.sb + h * x.sh + t0 * x.st, x.st, rows, dk, halves);
    }
  } else if (tid == 0) {
    mbar_init(&full, 1);
    abort_flag = 0;
    fence_barrier_init();
    mbar_arrive_expect_tx(&full, 2 * halves * C * 128);
    for (int d = 0; d < halves; ++d) {
      tma_load_4d(ks + d * C * 128, &maps.k, &full, 64 * d, (int)h, (int)t0, (int)b, policy_evict_normal());
      tma_load_4d(qs + d * C * 128, &maps.q, &full, 64 * d, (int)h, (int)t0, (int)b, policy_evict_normal());
    }
  }
  if (w == 3) {
    TokenGates<C> own;
#pragma unroll
    for (int i = 0; i < C / 32; ++i) {  // (zeros behind the last token)
      const int r = lane * (C / 32) + i;
      own.g[i] = r < rows ? Elem<GT>::to_f(((const GT*)g.p)[b * g.sb + h * g.sh + (t0 + r) * g.st]) : 0.f;
      own.beta[i] = r < rows ? Elem<GT>::to_f(((const GT*)beta.p)[b * beta.sb + h * beta.sh + (t0 + r) * beta.st]) : 0.f;
    }
    make_gates<C>(s, own, !BACK);
  }
  __syncthreads();
  if (!to.k && !__syncthreads_and(mbar_wait(&full, 0, kErrWaitProducer, &abort_flag))) {
    if (tid == 0) mbar_drain(&full, 0);
    return;
  }
  Scores<G> scores;
  scores.products(smem_u32(ks), smem_u32(qs), n_k16);
  if constexpr (!BACK) scores.find_bad(&s.bad);
  __syncthreads();
  if constexpr (!BACK) {
    // Products with a masked zero would carry what is not finite to earlier tokens: keys and gates from the
    // first bad token on are zeroed, and the chains make NaN of what depends on them.  (rare)
    const int bad = s.bad;
    if (bad < C) {
      for (int i = tid; i < PX * halves * C * 32; i += kThreads)
        if (i / 32 % C >= bad) ((uint32_t*)ks)[i / (halves * C * 32) * (G::kTile / 2) + i % (halves * C * 32)] = 0;
      if (tid >= bad && tid < C) {
        s.beta[tid] = 0.f;
        s.hi[tid] = bad > 0 ? s.hi[bad - 1] : 0.f, s.lo[tid] = bad > 0 ? s.lo[bad - 1] : 0.f;
        s.e[tid] = bad > 0 ? s.e[bad - 1] : 1.f;
      }
      if (tid < C) s.out[tid] = 0.f;  // (the state after the chunk is NaN)
      __syncthreads();
      scores.products(smem_u32(ks), smem_u32(qs), n_k16);
      __syncthreads();
    }
  }
  // gates and copies
  for (int i = tid; i < (int)sizeof(Gates<C>) / 16; i += kThreads)
    ((uint4*)to.gates)[at * (sizeof(Gates<C>) / 16) + i] = ((const uint4*)&s)[i];
  if (to.k) {
    for (int i = tid; i < PX * halves * C * 8; i += kThreads) {
      const int from = i / (halves * C * 8) * (G::kTile / 8) + i % (halves * C * 8);
      ((uint4*)to.k)[at * (PX * halves * C * 8) + i] = ((const uint4*)ks)[from];
      ((uint4*)to.q)[at * (PX * halves * C * 8) + i] = ((const uint4*)qs)[from];
    }
    __syncthreads();
  }
  scores.template scale<BACK>(s, scale);
  scores.write(t, diag, p);
  if (to.v) {
    const int dv16 = (dv + 15) / 16 * 16;
    const E* from = (const E*)v.p + b * v.sb + h * v.sh + t0 * v.st;
    for (int i = tid; i < C * dv16; i += kThreads) {
      const int r = i / dv16, c = i % dv16;
      ((E*)to.v)[at * (C * dv16) + i] = r < rows && c < dv ? from[r * v.st + c] : Elem<E>::from_f(0.f);
    }
  }
  __syncthreads();
  Inverse<G>::run(t, diag);
  // blocks (i, j), j <= i, as second operands: of a product with the transpose, or (BACK) with the matrix itself
  const int turn = lane_offset(G::kSquare, BACK);
#pragma unroll
  for (int n = 0; n < (G::kLower + 3) / 4; ++n) {
    const int pair = 4 * n + w;
    if (pair >= G::kLower) continue;
    const int i = pair >= 6 ? 3 : pair >= 3 ? 2 : pair >= 1 ? 1 : 0, from = 16 * i * G::kSquare + 16 * (pair - lower(i, 0)) + turn;
#pragma unroll
    for (int e = 0; e < G::NP + G::PP; ++e) {
      const bool is_p = e >= G::NP;
      const int part = is_p ? e - G::NP : e;
      const uint32_t addr = smem_u32((is_p ? p : t) + part * C * G::kSquare + from);
      uint32_t f[4];
      if constexpr (BACK)
        ldsm_t(f, addr);
      else
        ldsm(f, addr);
      (is_p ? to.p : to.t)[((at * G::kLower + pair) * (is_p ? G::PP : G::NP) + part) * 32 + lane] = make_uint4(f[0], f[1], f[2], f[3]);
    }
  }
}

template <typename G, bool BACK, typename GT>
int launch(const Prepared& to, const View& k, const View& q, const View& v, const View& g, const View& beta, int B, int H, int64_t T, int dk,
           int dv, float scale, cudaStream_t st) {
  const cudaError_t e = cudaFuncSetAttribute(delta_prep_kernel<G, BACK, GT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)PrepSmem<G>::kBytes);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return cuda_status(e, "cudaFuncSetAttribute(delta_prep)");
  }
  Maps maps{};
  if (!to.k) {
    int s;
    if ((s = view_map(&maps.k, k, B, T, H, dk, 2, 64, G::C)) || (s = view_map(&maps.q, q, B, T, H, dk, 2, 64, G::C))) return s;
  }
  const int64_t blocks = (T + G::C - 1) / G::C * H;
  if (blocks > INT32_MAX) return set_error(DYNCONV_ERR_SHAPE, "gated delta rule: H*T too large");
  const dim3 grid((unsigned)blocks, (unsigned)B);
  delta_prep_kernel<G, BACK, GT><<<grid, kThreads, PrepSmem<G>::kBytes, st>>>(to, maps, k, q, v, g, beta, H, T, dk, dv, scale);
  DYNCONV_CHECK_LAUNCH("delta_prep_kernel");
  return DYNCONV_OK;
}

template <typename G, bool BACK>
int go(const Prepared& to, const View& k, const View& q, const View& v, const View& g, const View& beta, int gates32, int B, int H, int64_t T,
       int dk, int dv, float scale, cudaStream_t st) {
  return gates32 ? launch<G, BACK, float>(to, k, q, v, g, beta, B, H, T, dk, dv, scale, st)
                 : launch<G, BACK, typename G::T>(to, k, q, v, g, beta, B, H, T, dk, dv, scale, st);
}

}  // namespace

size_t prepared_bytes(Prepared* p, void* base, int64_t B, int64_t T, int64_t H, int64_t dk, int64_t dv, int dtype, bool back) {
  const bool f32 = dtype == DYNCONV_DTYPE_F32;
  const int64_t C = chunk_of(dtype), n = B * H * chunks_of(T, dtype), pairs = f32 ? CfgF32::kLower : CfgBf16<true, true>::kLower;
  const int64_t dk64 = dk > 64 ? 128 : 64, dv16 = (dv + 15) / 16 * 16;
  char* at = (char*)base;
  auto take = [&](int64_t bytes) {  // (all multiples of 16)
    char* r = at;
    at += bytes;
    return r;
  };
  Prepared out{};
  out.t = (uint4*)take(n * pairs * 3 * 512);  // (two parts or three: three fit either)
  out.p = (uint4*)take(n * pairs * (f32 ? 3 : 2) * 512);
  out.gates = take(n * (f32 ? sizeof(Gates<32>) : sizeof(Gates<64>)));
  if (packs_keys(dk, dtype)) {
    out.k = (__nv_bfloat16*)take(n * (f32 ? 3 : 1) * C * dk64 * 2);
    out.q = (__nv_bfloat16*)take(n * (f32 ? 3 : 1) * C * dk64 * 2);
  }
  if (packs_values(dv, dtype)) out.v = take(n * C * dv16 * (f32 ? 4 : 2));
  if (p) *p = out;
  return at - (char*)base;
}

int prep_launch(const Prepared& to, const View& k, const View& q, const View& v, const View& g, const View& beta, int gates32, int B, int H, int64_t T,
                int dk, int dv, float scale, int dtype, bool exact, bool back, cudaStream_t st) {
  auto call = [&](auto run) { return run(to, k, q, v, g, beta, gates32, B, H, T, dk, dv, scale, st); };
  if (dtype == DYNCONV_DTYPE_F32) return back ? call(go<CfgF32, true>) : call(go<CfgF32, false>);
  if (exact) return back ? call(go<CfgBf16<true, true>, true>) : call(go<CfgBf16<true, false>, false>);
  return back ? call(go<CfgBf16<false, true>, true>) : call(go<CfgBf16<false, false>, false>);
}

}  // namespace dr

DYNCONV_DEFINE_ERROR_ACCESSOR(dr_prep_error_word)

}  // namespace dynconv
