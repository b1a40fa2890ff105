// linear_attention_tc.cu -- linear attention with a decay for each head on the tensor cores
// (bf16, widths up to 128).  The formulas stand in linear_attention.cuh.
//
// A CTA runs one segment of one chain: a role, a batch row and head, and 64 columns of w.
// Chunks have 128 tokens.  Per chunk four products (tcgen05, fp32 accumulators in TMEM):
//     Sc = X Y^T            128 x 128   both operands as TMA laid them down (K-major)
//     O1 = A W              A = Sc under the decay mask, bf16, written back to TMEM
//     O2 = X S              S = the state before the chunk, bf16 in shared memory
//     KV = Y^T W'           W' = W weighted by the decays to the chunk's end
// and out = a_scale O1 + (row factor) O2.  The state itself stays in registers in fp32 (lane
// = row of S, 64 columns): S <- g^L S + KV.  W' is a product of a bf16 value and a weight, so
// its rounding to bf16 would cost the state its precision: it is split into NS bf16 parts
// (two: 2^-17 of each term, three: 2^-25, when the state goes back to the caller).
//
// Warps: a producer (TMA rings two deep), an MMA issuer, and four groups of four whose warps own 32
// TMEM lanes each: two for the scores (Sc -> A, and the outputs), one for the state (KV -> S), one
// for the weights (W -> W').  The issuer runs
//     A(i-1) ready: O1(i-1);  Sc(i);  W'(i) ready: KV(i);  S(i) ready: O2(i)
// so that while the scores groups mask chunk i and write the outputs of chunk i-1, the pipe has
// KV and O2 of chunk i and O1 and Sc of the next.
//
// What bounds it: no unit by itself.  A chunk takes 3000 to 3700 cycles at 128 x 128, of which the tensor
// pipe is active 46%, issue slots 50% and, by ncu's L1 / shared counter, shared memory 54%; warps
// wait mostly for TMEM and for one another's barriers: the phases of a chunk hang on each other and
// one CTA per SM has no other chain to fill the gaps.  (Counted at the port, with the products' operand
// reads and TMA's writes, about 400 KB pass per chunk and CTA: 80 KB brought in, 224 KB of operands, W' 48, S 16,
// outputs 32, 3100 cycles at 128 bytes.  The counter does not show that much; whether it sees operand
// reads is not documented.)  Slices of 64 columns read x and y once each for the two halves of w, and compute the
// scores twice; 128 columns in one CTA would not fit two chunks of tiles into shared memory.  A CTA pair
// over 128 columns (cta_group::2, as the vocabulary loss has) has not been built.
// Measured (B200, 16 heads of 128, bf16): forward of 4 x 4096 tokens 64 us, 4.2 TB/s of its 268 MB
// (41 us at the copy rate); its backward, three roles in one launch, 188 us (384 chains on 148
// SMs are three rounds of one per SM where 2.6 would do); 65536 tokens with a state in and out
// 389 us.
//
// A masked score is zero whatever its value was, but 0 * inf in O1 is NaN: a value of w that is
// not finite is taken out of the tile and marks the rows that may see it (the slow path
// of the weights group), so rows before it stay clean.
#include "linear_attention.cuh"

namespace dynconv {
namespace la {

namespace {

constexpr int kC = 128;     // tokens of a chunk
constexpr int kSlice = 64;  // columns of w per CTA
constexpr int kTcThreads = 64 + 4 * 128;
constexpr uint32_t kBox = 64 * kC * 2;  // one TMA box: 128 rows of 64 bf16
// Chunks brought into L2 ahead of their loads: a tile from HBM takes about 2000 cycles, half a
// chunk's time, and the w ring asks for its next tile late.
constexpr int kAhead = 3;
constexpr uint32_t kStageOut = 32 * 64;  // 32 rows x 32 columns of outputs
constexpr int kMaxMaps = kMaxRoles * 4;

// TMEM columns
constexpr uint32_t kColSc = 0, kColA = 128, kColKv = 192, kColO1 = 256, kColO2 = 384, kTmemCols = 512;  // O1, O2: two each

struct TcMaps {
  CUtensorMap m[kMaxMaps];  // [role][x, y, w, out]
};

template <int DX, int NS>
struct Smem {
  // The third part of W' takes the room in which outputs are staged for TMA stores: their rows are
  // then stored directly.
  static constexpr bool kStage = NS == 2;
  static constexpr uint32_t kX = DX / 64 * kBox;
  static constexpr uint32_t kOffX = 0;
  static constexpr uint32_t kOffY = kOffX + 2 * kX;
  static constexpr uint32_t kOffW = kOffY + 2 * kX;
  static constexpr uint32_t kOffH = kOffW + 2 * kBox;  // W': NS boxes, or two and the staged outputs
  static constexpr uint32_t kOffO = kOffH + 2 * kBox;
  static constexpr uint32_t kOffS = kOffH + 3 * kBox;
  // The state pass has no x, no S and no outputs: a second W', in x's place where that is wide enough.
  static constexpr uint32_t kOffH2 = DX == 128 ? kOffX : kOffS + DX * 128;
  static constexpr uint32_t kTotal = kOffS + DX * 128 + (DX == 128 ? 0 : NS * kBox) + 1024;
};

struct Bars {
  uint64_t xy_full[2], xy_empty[2], w_full[2], w_empty[2];
  uint64_t sc_full, a_ready, o_full, o_free[2], o2_full, h_ready[2], kv_full[2], s_ready, kv_free[2], drain;
};

// 16-byte chunk c of row r in a 128-byte-swizzled tile of 128-byte rows.
__device__ __forceinline__ uint32_t sw_off(int r, int c) { return (uint32_t)r * 128u + (uint32_t)((c ^ (r & 7)) << 4); }

// 16-byte chunk c of row r in a 64-byte-swizzled tile of 64-byte rows (a warp's staged outputs).
__device__ __forceinline__ uint32_t out_off(int r, int c) {
  return (uint32_t)r * 64u + (uint32_t)((c ^ ((r >> 1) & 3)) << 4);
}

// Lane by lane max(a, |b|) of two bf16 pairs; NaN if either is.
__device__ __forceinline__ uint32_t max_abs_nan(uint32_t a, uint32_t b) {
  uint32_t m, d;
  asm("abs.bf16x2 %0, %1;" : "=r"(m) : "r"(b));
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(m));
  return d;
}

__device__ __forceinline__ float bf_lo(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float bf_hi(uint32_t u) { return __uint_as_float(u & 0xFFFF0000u); }

template <int DX, int NS, bool STATE_ONLY>
__global__ void __launch_bounds__(kTcThreads, 1)
    la_tc_kernel(const __grid_constant__ Params p, const __grid_constant__ TcMaps maps, int total_slices) {
  using L = Smem<DX, NS>;
  // W' and KV are single in the main pass (their time hides behind the other products) and double in
  // the state pass, which has nothing else to do.
  constexpr int kBuf = STATE_ONLY ? 2 : 1;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align_smem_1024(smem_raw);
  __shared__ Bars bars;
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  // Not-finite values of w in chunk i: bad_any[i % 4] = i + 1, and for each column the first
  // one's scan position a as (i + 1) * 256 + 255 - a (the largest wins, so nothing is ever
  // reset).  The writers may be three chunks ahead of the readers, not four.
  __shared__ unsigned bad_any[4], bad_row[4][kSlice];
  __shared__ float decays[31 + kC + 1];       // 31 zeros, then decay^0 .. decay^kC
  const float* pw = decays + 31;
  __shared__ __align__(16) float far_of[32];  // decays from a column to its 32-column block's far edge

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  // consecutive CTAs: the roles and slices of one batch row and head, which read the same tensors
  int ss = blockIdx.x % total_slices;
  const int64_t rest = blockIdx.x / total_slices;
  const int bh = (int)(rest % ((int64_t)p.B * p.H));
  const int seg = (int)(rest / ((int64_t)p.B * p.H));
  int ri = 0;
  while (ri + 1 < p.n_roles && ss >= (p.role[ri].dw + kSlice - 1) / kSlice) {
    ss -= (p.role[ri].dw + kSlice - 1) / kSlice;
    ++ri;
  }
  if (STATE_ONLY && seg == p.n_seg - 1 && !p.scan_final) return;
  const Role& ro = p.role[ri];
  const int c0 = ss * kSlice;
  const int b = bh / p.H, h = bh % p.H;
  const int64_t n_chunks = (p.T + kC - 1) / kC;
  const int64_t first = (int64_t)seg * p.chunks_per_seg;
  const int n = (int)(min(n_chunks, first + p.chunks_per_seg) - first);
  const int e = ro.reverse ? 0 : 1;

  auto start_of = [&](int i) -> int {  // first token of chunk i's tile (negative: before the sequence)
    const int64_t ch = first + i;
    return (int)(ro.reverse ? p.T - (ch + 1) * kC : ch * kC);
  };

  const CUtensorMap *mx = &maps.m[ri * 4], *my = mx + 1, *mw = mx + 2;
  auto load_xy = [&](int i) {
    const int s = i & 1;
    mbar_arrive_expect_tx(&bars.xy_full[s], STATE_ONLY ? L::kX : 2 * L::kX);
#pragma unroll
    for (int d = 0; d < DX / 64; ++d) {
      if (!STATE_ONLY)
        tma_load_4d(smem + L::kOffX + s * L::kX + d * kBox, mx, &bars.xy_full[s], d * 64, h, start_of(i), b,
                    policy_evict_normal());
      tma_load_4d(smem + L::kOffY + s * L::kX + d * kBox, my, &bars.xy_full[s], d * 64, h, start_of(i), b,
                  policy_evict_normal());
    }
  };
  auto load_w = [&](int i) {
    const int s = i & 1;
    mbar_arrive_expect_tx(&bars.w_full[s], kBox);
    tma_load_4d(smem + L::kOffW + s * kBox, mw, &bars.w_full[s], c0, h, start_of(i), b, policy_evict_normal());
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bars.xy_full[s], 1);
      mbar_init(&bars.xy_empty[s], 1);
      mbar_init(&bars.w_full[s], 1);
      mbar_init(&bars.w_empty[s], STATE_ONLY ? 4 : 1);  // (the state pass needs w only to weight it)
    }
    mbar_init(&bars.sc_full, 1);
    mbar_init(&bars.a_ready, 8);
    mbar_init(&bars.o_full, 1);
    mbar_init(&bars.o_free[0], 8);
    mbar_init(&bars.o_free[1], 8);
    mbar_init(&bars.o2_full, 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bars.h_ready[s], 4);
      mbar_init(&bars.kv_full[s], 1);
      mbar_init(&bars.kv_free[s], 4);
    }
    mbar_init(&bars.s_ready, 4);
    mbar_init(&bars.drain, 1);
    abort_flag = 0;
    fence_barrier_init();
    for (int i = 0; i < 2 && i < n; ++i) {  // the first loads, under way while the CTA sets itself up
      load_xy(i);
      load_w(i);
    }
  }
  if (threadIdx.x < 4 * kSlice) bad_row[threadIdx.x / kSlice][threadIdx.x % kSlice] = 0;
  if (threadIdx.x < 4) bad_any[threadIdx.x] = 0;
  if (threadIdx.x <= kC) {
    const float f = (float)exp2(log2_decay(p.log_decay, h) * threadIdx.x);
    decays[31 + threadIdx.x] = f;
    if (threadIdx.x < 32) {
      far_of[ro.reverse ? threadIdx.x : 31 - threadIdx.x] = f;
      if (threadIdx.x < 31) decays[threadIdx.x] = 0.f;
    }
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  if (warp == 0) {
    // ------------------------------------------------------------------ producer
    if (lane == 0) {
      int xy = min(n, 2), w = xy;  // loads issued
      auto more_xy = [&](int i) -> bool {
        if (!mbar_wait(&bars.xy_empty[i & 1], ((i >> 1) & 1) ^ 1, kErrWaitProducer, &abort_flag)) return false;
        load_xy(i);
        xy = i + 1;
        return true;
      };
      auto more_w = [&](int i) -> bool {
        if (!mbar_wait(&bars.w_empty[i & 1], ((i >> 1) & 1) ^ 1, kErrWaitProducer, &abort_flag)) return false;
        load_w(i);
        w = i + 1;
        return true;
      };
      for (int i = 0; i < n; ++i) {
        // w's tile is free first in the state pass, last in the main pass
        if (i >= 2 && !(STATE_ONLY ? more_w(i) && more_xy(i) : more_xy(i) && more_w(i))) break;
        if (i + kAhead < n) {
          const int t1 = start_of(i + kAhead);
#pragma unroll
          for (int d = 0; d < DX / 64; ++d) {
            if (!STATE_ONLY) tma_prefetch_4d(mx, d * 64, h, t1, b);
            tma_prefetch_4d(my, d * 64, h, t1, b);
          }
          tma_prefetch_4d(mw, c0, h, t1, b);
        }
      }
      if (abort_flag) {  // a wait gave up: the copies in flight land before the shared memory is given back
        for (int i = max(0, xy - 2); i < xy; ++i) mbar_drain(&bars.xy_full[i & 1], (i >> 1) & 1);
        for (int i = max(0, w - 2); i < w; ++i) mbar_drain(&bars.w_full[i & 1], (i >> 1) & 1);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA issuer
    constexpr uint32_t id_sc = make_idesc_bf16(kC, kC, 0, 0);
    constexpr uint32_t id_o = make_idesc_bf16(kC, kSlice, 0, 1);
    constexpr uint32_t id_kv = make_idesc_bf16(kC, kSlice, 1, 1), id_kv2 = make_idesc_bf16(kC, 2 * kSlice, 1, 1);
    const uint32_t sb = smem_u32(smem);
    const uint32_t el = elect_lane();
    auto issue_o1 = [&](int j) -> bool {
      if (!mbar_wait(&bars.a_ready, j & 1, kErrWaitMma, &abort_flag)) return false;
      tc_fence_after();
      const uint32_t w = desc_lo(sb + L::kOffW + (j & 1) * kBox, kBox);
#pragma unroll
      for (int k = 0; k < kC / 16; ++k)
        umma_f16_ts_e(el, tmem + kColO1 + (j & 1) * kSlice, tmem + kColA + k * 8, w + k * (2048 / 16), id_o, k > 0);
      umma_commit_e(el, &bars.w_empty[j & 1]);
      umma_commit_e(el, &bars.o_full);
      __syncwarp();
      return true;
    };
    bool dead = false;
    for (int i = 0; i < n; ++i) {
      const int s = i & 1;
      const uint32_t x = desc_lo(sb + L::kOffX + s * L::kX), yk = desc_lo(sb + L::kOffY + s * L::kX),
                     ym = desc_lo(sb + L::kOffY + s * L::kX, kBox);
      if (!STATE_ONLY && i > 0 && !issue_o1(i - 1)) {
        dead = true;
        break;
      }
      if (!mbar_wait(&bars.xy_full[s], (i >> 1) & 1, kErrWaitMma, &abort_flag)) break;
      tc_fence_after();
      if (!STATE_ONLY) {
#pragma unroll
        for (int k = 0; k < DX / 16; ++k) {
          const uint32_t at = ((k / 4) * kBox + (k % 4) * 32) / 16;
          umma_f16_e(el, tmem + kColSc, x + at, yk + at, id_sc, k > 0);
        }
        umma_commit_e(el, &bars.sc_full);
        __syncwarp();
      }
      const int hb = i % kBuf;
      if (!mbar_wait(&bars.h_ready[hb], (i / kBuf) & 1, kErrWaitMma, &abort_flag)) break;
      // the state group has read what this KV holds (s_ready: and has put down S)
      if (STATE_ONLY ? i >= kBuf && !mbar_wait(&bars.kv_free[hb], (i / kBuf - 1) & 1, kErrWaitMma, &abort_flag)
                     : !mbar_wait(&bars.s_ready, i & 1, kErrWaitMma, &abort_flag))
        break;
      tc_fence_after();
      // rows of Y^T beyond DX = 64 read the next tile: lanes of KV that nobody looks at
      const uint32_t hs = sb + (hb ? L::kOffH2 : L::kOffH);
      if (STATE_ONLY) {
        // the first two parts of W' side by side, the third on top of the second: half as many
        // products as part by part, in columns that the main pass does not have
#pragma unroll
        for (int k = 0; k < kC / 16; ++k)
          umma_f16_e(el, tmem + hb * 2 * kSlice, ym + k * (2048 / 16), desc_lo(hs, kBox) + k * (2048 / 16), id_kv2, k > 0);
        if (NS == 3) {
#pragma unroll
          for (int k = 0; k < kC / 16; ++k)
            umma_f16_e(el, tmem + hb * 2 * kSlice + kSlice, ym + k * (2048 / 16),
                       desc_lo(hs + 2 * kBox, kBox) + k * (2048 / 16), id_kv, 1);
        }
      } else {
#pragma unroll
        for (int part = 0; part < NS; ++part) {
          const uint32_t hw = desc_lo(hs + part * kBox, kBox);
#pragma unroll
          for (int k = 0; k < kC / 16; ++k)
            umma_f16_e(el, tmem + kColKv, ym + k * (2048 / 16), hw + k * (2048 / 16), id_kv, part > 0 || k > 0);
        }
      }
      umma_commit_e(el, &bars.kv_full[hb]);
      if (!STATE_ONLY) {
        // the outputs of chunk i-2 have left this O2 (and the O1 that O1(i) will write)
        if (i > 1 && !mbar_wait(&bars.o_free[s], ((i >> 1) - 1) & 1, kErrWaitMma, &abort_flag)) break;
        tc_fence_after();
        const uint32_t st = desc_lo(sb + L::kOffS, kBox);
#pragma unroll
        for (int k = 0; k < DX / 16; ++k)
          umma_f16_e(el, tmem + kColO2 + s * kSlice, x + ((k / 4) * kBox + (k % 4) * 32) / 16, st + k * (2048 / 16),
                     id_o, k > 0);
        umma_commit_e(el, &bars.o2_full);
      }
      umma_commit_e(el, &bars.xy_empty[s]);
      __syncwarp();
    }
    if (!STATE_ONLY && !dead && !abort_flag) issue_o1(n - 1);
    if (abort_flag) {  // the products in flight, before their accumulators are given back
      umma_commit_e(el, &bars.drain);
      mbar_drain(&bars.drain, 0);
    }
  } else {
    const int q = warp & 3;
    const int row = q * 32 + lane;  // token of the chunk's tile, or row of the state
    const uint32_t lanes = (uint32_t)(q * 32) << 16;
    const int a = ro.reverse ? kC - 1 - row : row;  // scan position of token `row`
    const int group = (warp - 2) >> 2;
    if (group == 1 || (group == 0 && !STATE_ONLY)) {
      // ----------------------------------------------------- outputs and masks
      if (!STATE_ONLY) {
        const bool rev = ro.reverse;
        const int half = group;  // of the outputs' columns, and every other block of the scores
        uint8_t* tile = smem + L::kOffO + (half * 4 + q) * kStageOut;
        const float fo = ro.i_scale * pw[a + e];
        __nv_bfloat16* out = (__nv_bfloat16*)ro.out.p + (int64_t)b * ro.out.sb + (int64_t)h * ro.out.sh + c0;
        // Decays of the scores.  On the diagonal 32 x 32 block: g^|row - column|, read along the
        // diagonals of the table.  d blocks away from it: g^(distance) = near * g^(32 (d - 1)) *
        // far[column], near from the row to its block's edge, far from the column's edge to the
        // column (both at most one, so nothing overflows on the way).
        const float* diag = pw + (rev ? -lane : lane);
        const int step = rev ? 1 : -1;
        const uint32_t seen = rev ? 0xFFFFFFFFu << lane : 0xFFFFFFFFu >> (31 - lane);  // columns of the diagonal block
        const float near = pw[rev ? 32 - lane : lane + 1], g32 = pw[32];
        const int blocks = rev ? 4 - q : q + 1;  // 32-column blocks that are not masked
        {  // the masked blocks of A are zero once and for all
          const uint32_t z[8] = {};
          for (int c = half; c < 4; c += 2)
            if (rev ? c < q : c > q) {
              tmem_st8(tmem + lanes + kColA + c * 16, z);
              tmem_st8(tmem + lanes + kColA + c * 16 + 8, z);
            }
        }
        auto outputs = [&](int i) {
          const int t = start_of(i) + row;
          // a whole chunk leaves through shared memory and a TMA store of each warp's 32 x 32
          const bool staged = L::kStage && p.T - (first + i) * kC >= kC;
          if (lane == 0) bulk_wait_group_read<0>();  // the store of the chunk before has read the tile
          __syncwarp();
          __nv_bfloat16* dst = out + (int64_t)t * ro.out.st;
          const bool in = t >= 0 && t < p.T;
          const bool bad = bad_any[i & 3] == (unsigned)i + 1;
#pragma unroll
          for (int c = 0; c < 32; c += 16) {
            float v[16], u[16];
            tmem_ld16(tmem + lanes + kColO1 + (i & 1) * kSlice + half * 32 + c, v);
            tmem_ld16(tmem + lanes + kColO2 + (i & 1) * kSlice + half * 32 + c, u);
            tmem_ld_wait();
            uint32_t w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float2 r = fma2(make_float2(fo, fo), make_float2(u[2 * j], u[2 * j + 1]),
                                    mul2(make_float2(ro.a_scale, ro.a_scale), make_float2(v[2 * j], v[2 * j + 1])));
              w[j] = pack_bf16x2(r.x, r.y);
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const uint4 o = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
              if (staged)
                *reinterpret_cast<uint4*>(tile + out_off(lane, c / 8 + j)) = o;
              else if (in && c0 + half * 32 + c + 8 * j < ro.dw)
                *reinterpret_cast<uint4*>(dst + half * 32 + c + 8 * j) = o;
            }
          }
          tc_fence_before();
          if (bad) {
#pragma unroll 1
            for (int c = 0; c < 32; ++c) {
              const unsigned key = bad_row[i & 3][half * 32 + c];
              if (key >> 8 != (unsigned)i + 1 || 255 - (int)(key & 255) > a) continue;
              if (staged)
                *reinterpret_cast<uint16_t*>(tile + out_off(lane, c / 8) + (c & 7) * 2) = 0x7FC0;
              else if (in && c0 + half * 32 + c < ro.dw)
                *reinterpret_cast<uint16_t*>(dst + half * 32 + c) = 0x7FC0;
            }
          }
          if (staged) fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&bars.o_free[i & 1]);
            if (staged) {
              tma_store_4d(&maps.m[ri * 4 + 3], tile, c0 + half * 32, h, start_of(i) + q * 32, b);
              bulk_commit_group();
            }
          }
        };
        for (int i = 0; i <= n; ++i) {
          // A's reader, O1(i-1), is done (as is O2(i-1), issued before it)
          if ((i > 0 && !mbar_wait(&bars.o_full, (i - 1) & 1, kErrWaitEpilogue, &abort_flag)) ||
              (i < n && !mbar_wait(&bars.sc_full, i & 1, kErrWaitEpilogue, &abort_flag)))
            break;
          tc_fence_after();
          if (i == n) {
            outputs(n - 1);
            break;
          }
          float f = half ? near : near * g32;  // of this warp's first block off the diagonal: 1 or 2 away
#pragma unroll 1
          for (int k = half; k < blocks; k += 2) {
            const int c = (rev ? q + k : q - k) * 32;
            float v[32];
            uint32_t w[16];
            tmem_ld32(tmem + lanes + kColSc + c, v);
            tmem_ld_wait();
            if (k == 0) {
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                const float2 m = mul2(make_float2(v[2 * j], v[2 * j + 1]), make_float2(diag[step * 2 * j], diag[step * (2 * j + 1)]));
                // (zero whatever a masked score was)
                w[j] = pack_bf16x2(seen & (1u << (2 * j)) ? m.x : 0.f, seen & (2u << (2 * j)) ? m.y : 0.f);
              }
            } else {
#pragma unroll
              for (int j = 0; j < 16; j += 2) {
                const float4 t4 = *reinterpret_cast<const float4*>(&far_of[2 * j]);
                const float2 f2 = make_float2(f, f);
                const float2 m0 = mul2(mul2(f2, make_float2(t4.x, t4.y)), make_float2(v[2 * j], v[2 * j + 1]));
                const float2 m1 = mul2(mul2(f2, make_float2(t4.z, t4.w)), make_float2(v[2 * j + 2], v[2 * j + 3]));
                w[j] = pack_bf16x2(m0.x, m0.y);
                w[j + 1] = pack_bf16x2(m1.x, m1.y);
              }
              f *= g32 * g32;
            }
            const uint32_t at = tmem + lanes + kColA + c / 2;
            tmem_st8(at, {w[0], w[1], w[2], w[3], w[4], w[5], w[6], w[7]});
            tmem_st8(at + 8, {w[8], w[9], w[10], w[11], w[12], w[13], w[14], w[15]});
          }
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars.a_ready);
          if (i > 0) outputs(i - 1);
        }
        if (lane == 0) bulk_wait_group_read<0>();  // (shared memory may go once it has been read)
      }
    } else if (group == 2) {
      // ---------------------------------------------------------------- state
      const int64_t n_state = (int64_t)ro.dx * ro.dw;
      const bool live = row < ro.dx;
      float S[kSlice];
      // Rows of 64 floats per thread would touch 32 lines with every load: states whose w-dimension
      // is dense pass through the warp's part of S's shared memory, a line at a time (rows
      // and columns of a 32 x 32 tile exchanged, column index ^ row against bank conflicts).
      float* tile = reinterpret_cast<float*>(smem + L::kOffS) + q * 1024;
      const int rows_here = min(32, ro.dx - q * 32);  // (none or fewer in the upper warps)
      {
        const float* src = nullptr;
        int64_t si = ro.dw, sj = 1;
        if (!STATE_ONLY) {
          if (p.n_seg > 1)
            src = seg_state(p, ri, seg, bh, n_state);
          else if (ro.s_in)
            src = ro.s_in + (int64_t)bh * n_state, si = ro.si, sj = ro.sj;
        }
        if (src && sj == 1 && rows_here > 0) {
#pragma unroll
          for (int hf = 0; hf < kSlice; hf += 32) {
            const bool in = c0 + hf + lane < ro.dw;
            const float* at = src + (int64_t)q * 32 * si + c0 + hf + lane;
#pragma unroll 8
            for (int r = 0; r < 32; ++r) tile[r * 32 + (lane ^ r)] = in && r < rows_here ? at[r * si] : 0.f;
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 32; ++j) S[hf + j] = tile[lane * 32 + (j ^ lane)];
            __syncwarp();
          }
        } else {
          if (!live) src = nullptr;
          const float* at = src + row * si + c0 * sj;
#pragma unroll
          for (int j = 0; j < kSlice; ++j) S[j] = src && c0 + j < ro.dw ? at[j * sj] : 0.f;
        }
      }
      const double l2d = log2_decay(p.log_decay, h);
      const Factor f_full = decay_factor(l2d, kC);
      bool dead = false;
      for (int i = 0; i <= n; ++i) {
        if (i > 0) {
          const int hb = (i - 1) % kBuf;
          if (!mbar_wait(&bars.kv_full[hb], ((i - 1) / kBuf) & 1, kErrWaitEpilogue, &abort_flag)) {
            dead = true;
            break;
          }
          tc_fence_after();
          const int64_t left = p.T - (first + i - 1) * kC;
          const Factor f = left >= kC ? f_full : decay_factor(l2d, (double)left);
#pragma unroll
          for (int c = 0; c < kSlice; c += 16) {
            float v[16];
            if (STATE_ONLY) {
              float u[16];
              tmem_ld16(tmem + lanes + hb * 2 * kSlice + c, v);
              tmem_ld16(tmem + lanes + hb * 2 * kSlice + kSlice + c, u);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 16; ++j) v[j] += u[j];
            } else {
              tmem_ld16(tmem + lanes + kColKv + c, v);
              tmem_ld_wait();
            }
#pragma unroll
            for (int j = 0; j < 16; j += 2) {  // decay_add of pairs
              const float2 s2 = make_float2(S[c + j], S[c + j + 1]);
              const float2 r = fma2(make_float2(f.hi, f.hi), s2, fma2(make_float2(f.lo, f.lo), s2, make_float2(v[j], v[j + 1])));
              S[c + j] = r.x, S[c + j + 1] = r.y;
            }
          }
          tc_fence_before();
          if (STATE_ONLY) {
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars.kv_free[hb]);
          }
        }
        if (i == n) break;
        if (!STATE_ONLY) {
          if (i > 0 && !mbar_wait(&bars.o2_full, (i - 1) & 1, kErrWaitEpilogue, &abort_flag)) {  // S's reader
            dead = true;
            break;
          }
          if (row < DX) {
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              uint4 w;
              w.x = pack_bf16x2(S[8 * c], S[8 * c + 1]), w.y = pack_bf16x2(S[8 * c + 2], S[8 * c + 3]);
              w.z = pack_bf16x2(S[8 * c + 4], S[8 * c + 5]), w.w = pack_bf16x2(S[8 * c + 6], S[8 * c + 7]);
              *reinterpret_cast<uint4*>(smem + L::kOffS + sw_off(row, c)) = w;
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars.s_ready);
        }
      }
      if (!dead) {
        float* dst = nullptr;
        int64_t si = ro.dw, sj = 1;
        if (STATE_ONLY)
          dst = seg_state(p, ri, seg, bh, n_state);
        else if (seg == p.n_seg - 1 && ro.s_out && !p.scan_final)
          dst = ro.s_out + (int64_t)bh * n_state, si = ro.si, sj = ro.sj;
        if (dst && sj == 1 && rows_here > 0) {
          // S's last reader is O2 of the last chunk
          if (!STATE_ONLY) dead = !mbar_wait(&bars.o2_full, (n - 1) & 1, kErrWaitEpilogue, &abort_flag);
          if (!dead) {
#pragma unroll
            for (int hf = 0; hf < kSlice; hf += 32) {
              __syncwarp();
#pragma unroll
              for (int j = 0; j < 32; ++j) tile[lane * 32 + (j ^ lane)] = S[hf + j];
              __syncwarp();
              float* at = dst + (int64_t)q * 32 * si + c0 + hf + lane;
              if (c0 + hf + lane < ro.dw) {
#pragma unroll 8
                for (int r = 0; r < 32; ++r)
                  if (r < rows_here) at[r * si] = tile[r * 32 + (lane ^ r)];
              }
            }
          }
        } else if (dst && sj != 1 && live) {
          float* at = dst + row * si + c0 * sj;
#pragma unroll
          for (int j = 0; j < kSlice; ++j)
            if (c0 + j < ro.dw) at[j * sj] = S[j];
        }
      }
    } else {
      // -------------------------------------------------------------- weights
      const float fw = ro.w_scale * pw[kC - e - a];
      // (the state pass: two groups, every other chunk each)
      for (int i = STATE_ONLY && group == 0 ? 1 : 0; i < n; i += kBuf) {
        const int sw = i & 1, hb = i % kBuf;
        if (!mbar_wait(&bars.w_full[sw], (i >> 1) & 1, kErrWaitEpilogue, &abort_flag) ||
            (i >= kBuf && !mbar_wait(&bars.kv_full[hb], (i / kBuf - 1) & 1, kErrWaitEpilogue, &abort_flag)))
          break;
        const int64_t left = p.T - (first + i) * kC;
        float f = fw;
        if (left < kC) f = a < left ? ro.w_scale * pw[left - e - a] : 0.f;
        uint8_t* src = smem + L::kOffW + sw * kBox;
        uint8_t* dst = smem + (hb ? L::kOffH2 : L::kOffH);
        uint32_t largest = 0;  // magnitudes of the even and the odd columns, NaN above all
#pragma unroll 4
        for (int c = 0; c < 8; ++c) {
          const uint32_t at = sw_off(row, c);
          const uint4 u = *reinterpret_cast<const uint4*>(src + at);
          const uint32_t w[4] = {u.x, u.y, u.z, u.w};
          uint32_t part[NS][4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            largest = max_abs_nan(largest, w[j]);
            float2 x = mul2(make_float2(bf_lo(w[j]), bf_hi(w[j])), make_float2(f, f));
#pragma unroll
            for (int s = 0; s < NS; ++s) {
              part[s][j] = pack_bf16x2(x.x, x.y);
              if (s + 1 < NS) x = fma2(make_float2(bf_lo(part[s][j]), bf_hi(part[s][j])), make_float2(-1.f, -1.f), x);
            }
          }
#pragma unroll
          for (int s = 0; s < NS; ++s)
            *reinterpret_cast<uint4*>(dst + s * kBox + at) = make_uint4(part[s][0], part[s][1], part[s][2], part[s][3]);
        }
        if (!STATE_ONLY && ((largest & 0x7F80u) == 0x7F80u || (largest & 0x7F800000u) == 0x7F800000u)) {
          // the tile keeps zeros where a value was not finite; rows that may see it become NaN
          __nv_bfloat16* wr = reinterpret_cast<__nv_bfloat16*>(src);
          for (int c = 0; c < kSlice; ++c) {
            __nv_bfloat16* at = wr + (sw_off(row, c >> 3) >> 1) + (c & 7);
            if (!isfinite(__bfloat162float(*at))) {
              *at = __float2bfloat16_rn(0.f);
              atomicMax(&bad_row[i & 3][c], ((unsigned)i + 1) * 256 + 255 - a);
              bad_any[i & 3] = (unsigned)i + 1;
            }
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&bars.h_ready[hb]);
          if (STATE_ONLY) mbar_arrive(&bars.w_empty[sw]);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, kTmemCols);
}

bool mappable(const View& v, int64_t B, int64_t T, int H) {
  if (reinterpret_cast<uintptr_t>(v.p) & 15) return false;
  const int64_t s[3] = {v.sb, v.st, v.sh}, n[3] = {B, T, H};
  for (int i = 0; i < 3; ++i)
    if (n[i] > 1 && (s[i] <= 0 || s[i] % 8 != 0 || s[i] * 2 >= ((int64_t)1 << 40))) return false;
  return true;
}

int view_map(CUtensorMap* map, const View& v, int64_t B, int64_t T, int H, int d, int cols, int rows) {
  const cuuint64_t dims[4] = {(cuuint64_t)d, (cuuint64_t)H, (cuuint64_t)T, (cuuint64_t)B};
  const cuuint64_t strides[3] = {(cuuint64_t)(H > 1 ? v.sh * 2 : 16), (cuuint64_t)(T > 1 ? v.st * 2 : 16),
                                 (cuuint64_t)(B > 1 ? v.sb * 2 : 16)};
  const cuuint32_t box[4] = {(cuuint32_t)cols, 1, (cuuint32_t)rows, 1};
  return encode_tensor_map_bf16(map, v.p, 4, dims, strides, box,
                                cols == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
}

template <int DX, int NS, bool STATE_ONLY>
int go(const Params& p, const TcMaps& maps, cudaStream_t st) {
  using L = Smem<DX, NS>;
  static_assert(L::kTotal <= 232448 - 1024, "shared memory of one CTA");
  int slices = 0;
  for (int r = 0; r < p.n_roles; ++r) slices += (p.role[r].dw + kSlice - 1) / kSlice;
  const int64_t blocks = (int64_t)p.n_seg * p.B * p.H * slices;
  if (blocks > INT32_MAX) return set_error(DYNCONV_ERR_SHAPE, "linear attention: B*H too large");
  cudaError_t e =
      cudaFuncSetAttribute(la_tc_kernel<DX, NS, STATE_ONLY>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::kTotal);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return cuda_status(e, "cudaFuncSetAttribute(la_tc)");
  }
  la_tc_kernel<DX, NS, STATE_ONLY><<<(unsigned)blocks, kTcThreads, L::kTotal, st>>>(p, maps, slices);
  DYNCONV_CHECK_LAUNCH("la_tc_kernel");
  return DYNCONV_OK;
}

// NS = 3 wherever a state goes back to the caller: in the state pass where there is one.
template <int DX>
int passes(const Params& p, const TcMaps& maps, bool states, cudaStream_t st) {
  int s;
  if (p.n_seg > 1) {
    if ((s = states ? go<DX, 3, true>(p, maps, st) : go<DX, 2, true>(p, maps, st))) return s;
    if ((s = scan_launch(p, kC, st))) return s;
  }
  return states && p.n_seg == 1 ? go<DX, 3, false>(p, maps, st) : go<DX, 2, false>(p, maps, st);
}

}  // namespace

// bf16, widths that are multiples of 8 up to 128, and tensors that TMA can address: 16-byte
// aligned, strides positive multiples of 16 bytes.
bool tc_supported(const Params& p, int dtype) {
  if (dtype != DYNCONV_DTYPE_BF16) return false;
  for (int r = 0; r < p.n_roles; ++r) {
    const Role& ro = p.role[r];
    if (ro.dx % 8 || ro.dw % 8 || ro.dx > 128 || ro.dw > 128) return false;
    for (const View* v : {&ro.x, &ro.y, &ro.w, &ro.out})
      if (!mappable(*v, p.B, p.T, p.H)) return false;
  }
  return true;
}

// Measured at 128 x 128, one CTA per SM: a chunk 2 us, 2.9 with the third part of W'; a chunk of the
// state pass 0.9 us, 1.1 with it; 9 us to start and end a round, 6 us for the scan.  So a long chain
// whose last state is wanted is cheaper cut, with the third part in the state pass alone.
void tc_plan(Params* p, bool states) {
  p->scan_final = states;
  plan_segments(p, kC, kSlice, sm_count(), states ? 1.45 : 1.0, states ? 0.55 : 0.45, 4.5, 3.0);
  if (p->n_seg == 1) p->scan_final = 0;
}

int tc_launch(const Params& p, cudaStream_t st) {
  TcMaps maps;
  int s, dx = 0;
  for (int r = 0; r < p.n_roles; ++r) {
    const Role& ro = p.role[r];
    if ((s = view_map(&maps.m[4 * r], ro.x, p.B, p.T, p.H, ro.dx, 64, kC))) return s;
    if ((s = view_map(&maps.m[4 * r + 1], ro.y, p.B, p.T, p.H, ro.dx, 64, kC))) return s;
    if ((s = view_map(&maps.m[4 * r + 2], ro.w, p.B, p.T, p.H, ro.dw, 64, kC))) return s;
    if ((s = view_map(&maps.m[4 * r + 3], ro.out, p.B, p.T, p.H, ro.dw, 32, 32))) return s;
    dx = ro.dx > dx ? ro.dx : dx;
  }
  const bool states = wants_states(p);
  return dx <= 64 ? passes<64>(p, maps, states, st) : passes<128>(p, maps, states, st);
}

}  // namespace la

DYNCONV_DEFINE_ERROR_ACCESSOR(la_tc_error_word)

}  // namespace dynconv
