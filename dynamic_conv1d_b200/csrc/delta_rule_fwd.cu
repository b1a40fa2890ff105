// delta_rule_fwd.cu -- the gated delta rule over whole sequences: the chain over the chunks (formulas:
// delta_rule.cuh; how the warps share the work: delta_chain.cuh).
//
// Each chunk is three products in a row, K S0 and Q S0, then T x, then P U and K^T U.  4 x 4096 tokens, 16 heads of 128 x 128,
// states kept: 278 us, 4.3 us for 64 tokens of four teams.  Bound by shared memory (82% of its throughput; matrix units 45%
// active, issue 43%): each team reads all of K, Q, T and P for its 16 columns, and each of its warps the whole state.
// One row of 32768 tokens, a team to a CTA and an exact state: 1.05 ms, 2.05 us a chunk.  There it is the chunks' order: a
// scheduler has one warp that works, and gets an instruction from it every 4.6 cycles (issue 22%, matrix units 33%, shared
// memory 49%).
#include "delta_chain.cuh"

namespace dynconv {
namespace dr {
namespace {

template <typename G, int KK, bool SAVE>
__global__ void __launch_bounds__(Chain<G, KK>::kMostThreads, 1) delta_fwd_kernel(Forward p, const __grid_constant__ Maps maps, Plan plan) {
  using Ch = Chain<G, KK>;
  using E = typename G::T;
  constexpr int C = G::C, NP = G::NP, PX = G::PX, PP = G::PP, NB = G::kBlocks, NT = Ch::NT, PU = Ch::PU;
  constexpr int PS = PX == 1 ? 1 : 3;  // parts of the state in the outputs' product
  extern __shared__ uint8_t smem_raw[];
  __shared__ typename Ch::Bars bars;
  uint8_t* const smem = align_smem_1024(smem_raw);
  const int64_t bh = blockIdx.y, b = bh / p.H, h = bh % p.H;
  const int chunks = (int)((p.T + C - 1) / C), n_k16 = (p.dk + 15) / 16, first_col = blockIdx.x * plan.teams * 16;
  const int warp = warp_index(), l = threadIdx.x & 31, row = l >> 2, col = 2 * (l & 3);
  Ch::init(bars, Ch::live_teams(plan, p.dv, first_col));
  const typename Ch::Producer producer{smem, bars, plan, maps, p.pre, (int)b, (int)h, chunks, p.dk, p.dv, first_col, bh};
  if (warp == plan.teams * Ch::W) {
    if (l == 0) producer.template walk<false>();
    return;
  }
  const int team = warp / Ch::W, w = (warp + team) % Ch::W;  // (turned, so that the last tokens' warps fall on different schedulers)
  const int d0 = first_col + 16 * team, slices = (p.dv + 15) / 16, slice = d0 / 16;
  if (d0 >= p.dv) return;
  const bool produces = !plan.own_warp && team == 0 && w == 0 && l == 0;  // (of the warp with the fewest blocks of T)
  if (produces) producer.template start<false>();
  const int bytes = Ch::stage_bytes(plan.teams);
  uint4* const state = (uint4*)(smem + plan.stages * bytes + team * Ch::kTeam);
  uint4 *const part_r = state + Ch::kState / 16, *const part_u = part_r + Ch::kBlock / 16, *const part_s = part_u + Ch::kBlock / 16;
  const KeyLane across(false);
  // (the row and piece of a lane in transposed reads and writes of a team's bf16 columns, 16 tokens at a time)
  const int v_row = (l & 7) + 8 * (l >> 4), v_piece = l >> 3 & 1;
  uint32_t down[NT / 2];  // this warp's columns of K, 16 at a time
  {
    const KeyLane lane(true);
#pragma unroll
    for (int m = 0; m < NT / 2; ++m) {
      const int kk = w * NT / 2 + m;
      uint32_t off = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i == (kk & 3)) off = lane.off[i];
      down[m] = off + (kk >> 2) * (C * 128);
    }
  }

  float S[NT][4];  // S^T: rows d0 + row (+ 8), columns 8 (w NT + n) + col (+ 1) of dk
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int d = d0 + row + 8 * (e >> 1), k = 8 * (w * NT + n) + col + (e & 1);
      S[n][e] = p.s_in && d < p.dv && k < p.dk ? p.s_in[(bh * p.dk + k) * p.dv + d] : 0.f;
    }
  // the state before chunk c to the team, and to the backward
  auto publish = [&](int c) {
#pragma unroll
    for (int m = 0; m < NT / 2; ++m) {
      const int kk = w * NT / 2 + m;
      uint32_t a[NP][4];
      operand<NP>(S[2 * m], S[2 * m + 1], a);
      Ch::put(state + kk * NP * 32, a);
      if constexpr (SAVE) {
        if (kk < n_k16 && c < chunks)
#pragma unroll
          for (int i = 0; i < PS; ++i)
            Ch::keep(p.states + ((((i * (int64_t)p.B * p.H + bh) * chunks + c) * slices + slice) * n_k16 + kk) * 256, a[i]);
      }
    }
  };
  publish(0);

  for (int c = 0, stage = 0, parity = 0; c < chunks; ++c) {
    if (!Ch::team_all(team, mbar_wait(&bars.full[stage], parity, kErrWaitMma, &bars.abort_flag))) {
      if (produces) producer.drain(c, c + plan.stages);
      return;
    }
    const typename Ch::Stage s{smem + stage * bytes, plan.teams};
    const Gates<C>& gate = s.gates();
    int bad = gate.bad;
    // (K S0)^T and (Q S0)^T; the operands of the next 16 of dk are asked for before the products of these
    float Z[2][4], O[2][4];
    {
      constexpr int L = 2;
      float z[L][2][4], o[L][2][4];
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int i = 0; i < L; ++i) zero(z[i][m]), zero(o[i][m]);
      uint32_t a[2][NP][4], f[2][PX][4], g[2][PX][4];
      auto fetch = [&](int kk, uint32_t(&a)[NP][4], uint32_t(&f)[PX][4], uint32_t(&g)[PX][4]) {
        Ch::template get<NP>(state + kk * NP * 32, a);
        const uint32_t at = across.at<C>(w, kk);
#pragma unroll
        for (int i = 0; i < PX; ++i) {
          ldsm(f[i], s.k() + at + i * G::kTile * 2);
          ldsm(g[i], s.q() + at + i * G::kTile * 2);
        }
      };
      fetch(0, a[0], f[0], g[0]);
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        if (kk + 1 < KK) fetch(kk + 1, a[(kk + 1) & 1], f[(kk + 1) & 1], g[(kk + 1) & 1]);
        uint32_t a_o[PS][4];
#pragma unroll
        for (int i = 0; i < PS; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) a_o[i][e] = a[kk & 1][i][e];
        mma_levels<NP, PX, NP, L>(z, a[kk & 1], f[kk & 1]);
        mma_levels<PS, PX, PS, L>(o, a_o, g[kk & 1]);
      }
      sum_levels<L>(Z, z), sum_levels<L>(O, o);
    }
    // (V - e^b K S0)^T in Z's place, O scaled
    float odd = 0.f;  // NaN if a value is not finite
    {
      float v[2][4];
      if constexpr (sizeof(E) == 2) {
        uint32_t f[4];
        ldsm_t(f, smem_u32(s.v(team, 16 * w + v_row, v_piece)));
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i >> 1][2 * (i & 1)] = low(f[i]), v[i >> 1][2 * (i & 1) + 1] = high(f[i]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          v[i >> 2][i & 3] = s.value(team, 16 * w + 8 * (i >> 2) + col + (i & 1), row + 8 * ((i >> 1) & 1));
      }
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const float2 eb = *reinterpret_cast<const float2*>(gate.e + 16 * w + 8 * m + col);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          odd = fmaf(v[m][e], 0.f, odd);
          Z[m][e] = fmaf(-(e & 1 ? eb.y : eb.x), Z[m][e], v[m][e]);
          O[m][e] *= p.scale * (e & 1 ? eb.y : eb.x);
        }
      }
    }
    const bool odd_here = __any_sync(0xffffffffu, !(odd == 0.f));
    if (bad < C || odd_here) {  // (rare)
      // What is not finite must not meet the zeros of T and P: values from the first bad token on count as zero.
      bad = min(bad, Ch::bad_row(s, team, false));
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (16 * w + 8 * m + col + (e & 1) >= bad) Z[m][e] = O[m][e] = 0.f;
    }
    {
      uint32_t a[NP][4];
      operand<NP>(Z[0], Z[1], a);
      Ch::put(part_r + w * NP * 32, a);
    }
    // (another warp's tokens may be the bad ones)
    if (!Ch::team_all(team, !odd_here)) bad = min(bad, Ch::bad_row(s, team, false));
    if (produces && c > 0) producer.template refill<false>(c);
    // r^T = (V - e^b K S0)^T T^T, U = beta r
    float U[2][4];
    {
      float u[NP][2][4];
#pragma unroll
      for (int i = 0; i < NP; ++i) zero(u[i][0]), zero(u[i][1]);
      const uint4* const t_at = s.t() + lower(w, 0) * NP * 32;
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        if (j > w) continue;
        uint32_t a[NP][4], f[NP][4];
        Ch::template get<NP>(part_r + j * NP * 32, a);
        Ch::template get<NP>(t_at + j * NP * 32, f);
        mma_levels<NP, NP, NP, NP>(u, a, f);
      }
      sum_levels<NP>(U, u);
      if constexpr (SAVE) {
        uint32_t a[PU][4];
        operand<PU>(U[0], U[1], a);
#pragma unroll
        for (int i = 0; i < PU; ++i)
          Ch::keep(p.rest + ((((i * (int64_t)p.B * p.H + bh) * chunks + c) * slices + slice) * NB + w) * 256, a[i]);
      }
      float x[2][4];
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const float2 beta = *reinterpret_cast<const float2*>(gate.beta + 16 * w + 8 * m + col);
        const float2 out = *reinterpret_cast<const float2*>(gate.out + 16 * w + 8 * m + col);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          U[m][e] *= e & 1 ? beta.y : beta.x;
          x[m][e] = U[m][e] * (e & 1 ? out.y : out.x);
        }
      }
      uint32_t a[NP][4];
      operand<NP>(x[0], x[1], a);
      Ch::put(part_s + w * NP * 32, a);
      uint32_t a_u[PU][4];
      operand<PU>(U[0], U[1], a_u);
      Ch::put(part_u + w * PU * 32, a_u);
    }
    Ch::team_sync(team);
    // S^T <- e^(b_C) S^T + (e^(b_C - b) U)^T K, each chunk's sum by itself first: the instruction's own
    // additions are cut off, not rounded
    const float total = gate.total;
    constexpr int NX = NT < 4 ? NT : 4;
#pragma unroll
    for (int n = 0; n < NT; n += NX) {
      float x[NX][4];
#pragma unroll
      for (int m = 0; m < NX; ++m) zero(x[m]);
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        uint32_t a[NP][4];
        Ch::template get<NP>(part_s + j * NP * 32, a);
#pragma unroll
        for (int m = 0; m < NX; m += 2) {
          uint32_t f[PX][4];
#pragma unroll
          for (int i = 0; i < PX; ++i)
            ldsm_t(f[i], s.k() + 2 * i * G::kTile + j * 2048 + down[(n + m) / 2]);
          mma_parts<NP, PX, NP>(x[m], x[m + 1], a, f);
        }
      }
#pragma unroll
      for (int m = 0; m < NX; ++m)
#pragma unroll
        for (int e = 0; e < 4; ++e) S[n + m][e] = fmaf(total, S[n + m][e], x[m][e]);
    }
    if (bad < C) {
#pragma unroll
      for (int n = 0; n < NT; ++n) S[n][0] = S[n][1] = S[n][2] = S[n][3] = NAN;
    }
    // (the state's readers of this chunk passed the barriers above)
    publish(c + 1);
    // O^T += U^T P^T
    {
      float o[PU][2][4];
#pragma unroll
      for (int i = 0; i < PU; ++i) zero(o[i][0]), zero(o[i][1]);
      const uint4* const p_at = s.p() + lower(w, 0) * PP * 32;
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        if (j > w) continue;
        uint32_t a[PU][4], f[PP][4];
        Ch::template get<PU>(part_u + j * PU * 32, a);
        Ch::template get<PP>(p_at + j * PP * 32, f);
        mma_levels<PU, PP, PU, PU>(o, a, f);
      }
      float x[2][4];
      sum_levels<PU>(x, o);
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int e = 0; e < 4; ++e) O[m][e] += x[m][e];
      if (bad < C) {
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (16 * w + 8 * m + col + (e & 1) >= bad) O[m][e] = NAN;
      }
      // through v's tile, of which nobody else needs these tokens and columns any more
      const int64_t t0 = (int64_t)c * C + 16 * w;
      const int rows = (int)(p.T - t0 < 16 ? p.T - t0 : 16);
      E* const to = (E*)p.o.p + b * p.o.sb + h * p.o.sh + t0 * p.o.st + d0;
      if constexpr (sizeof(E) == 2) {
        stsm_t(smem_u32(s.v(team, 16 * w + v_row, v_piece)), pack(O[0][0], O[0][1]), pack(O[0][2], O[0][3]),
               pack(O[1][0], O[1][1]), pack(O[1][2], O[1][3]));
        __syncwarp();
        if (plan.o_vectors) {
          const int r = l >> 1, d = (l & 1) * 8;
          if (r < rows && d0 + d < p.dv) *reinterpret_cast<uint4*>(to + r * p.o.st + d) = *reinterpret_cast<const uint4*>(s.v(team, 16 * w + r, l & 1));
        } else {
          for (int i = l; i < 16 * rows; i += 32)
            if (d0 + i % 16 < p.dv) to[i / 16 * p.o.st + i % 16] = s.value(team, 16 * w + i / 16, i % 16);
        }
      } else {
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = 8 * m + col + (e & 1), d = row + 8 * (e >> 1);
            if (r < rows && d0 + d < p.dv) to[r * p.o.st + d] = O[m][e];
          }
      }
    }
    if constexpr (sizeof(E) == 2) fence_proxy_async_smem();  // (the outputs went through the tile that is loaded again)
    __syncwarp();
    if (l == 0) mbar_arrive(&bars.empty[stage]);
    if (++stage == plan.stages) stage = 0, parity ^= 1;
  }
  if (p.s_out) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = d0 + row + 8 * (e >> 1), k = 8 * (w * NT + n) + col + (e & 1);
        if (d < p.dv && k < p.dk) p.s_out[(bh * p.dk + k) * p.dv + d] = S[n][e];
      }
  }
}

template <typename G, int KK, bool SAVE>
int go(const Forward& p, Plan plan, cudaStream_t st) {
  using Ch = Chain<G, KK>;
  int s;
  const int slices = (p.dv + 15) / 16;
  plan.o_vectors = vectors_of(p.o, p.dv, sizeof(typename G::T));
  const int smem = Ch::smem_bytes(plan.teams, plan.stages);
  if ((s = allow_shared(delta_fwd_kernel<G, KK, SAVE>, Ch::kMostBytes, "cudaFuncSetAttribute(delta_fwd)"))) return s;
  Maps maps{};
  if ((s = chain_maps<G>(&maps, p.pre, p.k, p.q, p.v, p.B, p.T, p.H, p.dk, p.dv, plan.teams))) return s;
  const dim3 grid((unsigned)((slices + plan.teams - 1) / plan.teams), (unsigned)(p.B * p.H));
  delta_fwd_kernel<G, KK, SAVE><<<grid, 32 * (plan.teams * Ch::W + plan.own_warp), smem, st>>>(p, maps, plan);
  DYNCONV_CHECK_LAUNCH("delta_fwd_kernel");
  return DYNCONV_OK;
}

template <typename G, bool SAVE>
int pick(const Forward& p, cudaStream_t st) {
  const int64_t bh = (int64_t)p.B * p.H;
  if (p.dk <= 64) return go<G, 4, SAVE>(p, plan_of<Chain<G, 4>>(bh, p.dv), st);
  return go<G, 8, SAVE>(p, plan_of<Chain<G, 8>>(bh, p.dv), st);
}

}  // namespace

// bf16 chains hold their numbers as two parts (16 digits: the outputs' own rounding is 8), as three where
// the state after the last token goes back to the caller, who gets it in fp32.
int forward_launch(const Forward& p, int dtype, cudaStream_t st) {
  const bool save = p.states != nullptr, exact = p.s_out != nullptr;
  const int s = prep_launch(p.pre, p.k, p.q, p.v, p.g, p.beta, p.gates32, p.B, p.H, p.T, p.dk, p.dv, p.scale, dtype, exact, false, st);
  if (s) return s;
  if (dtype == DYNCONV_DTYPE_F32) return save ? pick<CfgF32, true>(p, st) : pick<CfgF32, false>(p, st);
  if (exact) return save ? pick<CfgBf16<true, false>, true>(p, st) : pick<CfgBf16<true, false>, false>(p, st);
  return save ? pick<CfgBf16<false, false>, true>(p, st) : pick<CfgBf16<false, false>, false>(p, st);
}

}  // namespace dr

DYNCONV_DEFINE_ERROR_ACCESSOR(dr_fwd_error_word)

}  // namespace dynconv
