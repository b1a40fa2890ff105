// delta_rule_bwd.cu -- the gradients' chain of the gated delta rule: dS of every chunk and dU, from the last chunk to the
// first (formulas: delta_rule.cuh; how the warps share the work: delta_chain.cuh).  The gradients themselves
// follow from these chunk by chunk (delta_grad.cu).
//
// Bound as the forward's chain is, each chunk being P^T dO and K dS, then T^T x, then the products with Q and K that
// the state takes: 264 us for 4 x 4096 tokens, 16 heads of 128 x 128 (shared memory 84%, matrix units 52% active, issue 45%).
#include "delta_chain.cuh"

namespace dynconv {
namespace dr {
namespace {

template <typename G, int KK>
__global__ void __launch_bounds__(Chain<G, KK>::kMostThreads, 1) delta_bwd_kernel(Backward p, const __grid_constant__ Maps maps, Plan plan) {
  using Ch = Chain<G, KK>;
  using E = typename G::T;
  constexpr int C = G::C, NP = G::NP, PX = G::PX, PP = G::PP, NB = G::kBlocks, NT = Ch::NT, PU = Ch::PU;
  constexpr int PS = PX == 1 ? 1 : 3, KX = PX > PP ? PX : PP;
  extern __shared__ uint8_t smem_raw[];
  __shared__ typename Ch::Bars bars;
  uint8_t* const smem = align_smem_1024(smem_raw);
  const int64_t bh = blockIdx.y, b = bh / p.H, h = bh % p.H;
  const int chunks = (int)((p.T + C - 1) / C), n_k16 = (p.dk + 15) / 16, first_col = blockIdx.x * plan.teams * 16;
  const int warp = warp_index(), l = threadIdx.x & 31, row = l >> 2, col = 2 * (l & 3);
  Ch::init(bars, Ch::live_teams(plan, p.dv, first_col));
  const typename Ch::Producer producer{smem, bars, plan, maps, p.pre, (int)b, (int)h, chunks, p.dk, p.dv, first_col, bh};
  if (warp == plan.teams * Ch::W) {
    if (l == 0) producer.template walk<true>();
    return;
  }
  const int team = warp / Ch::W, w = (warp + team) % Ch::W;
  const int d0 = first_col + 16 * team, slices = (p.dv + 15) / 16, slice = d0 / 16;
  if (d0 >= p.dv) return;
  const bool produces = !plan.own_warp && team == 0 && w == Ch::W - 1 && l == 0;  // (of the warp with the fewest blocks of T)
  if (produces) producer.template start<true>();
  const int bytes = Ch::stage_bytes(plan.teams);
  uint4* const state = (uint4*)(smem + plan.stages * bytes + team * Ch::kTeam);
  uint4 *const part_x = state + Ch::kState / 16, *const part_o = part_x + Ch::kBlock / 16, *const part_u = part_o + Ch::kBlock / 16;
  const KeyLane across(false);
  const int v_row = (l & 7) + 8 * (l >> 4), v_piece = l >> 3 & 1;
  uint32_t down[NT / 2];  // this warp's columns of K and Q, 16 at a time
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

  float S[NT][4];  // dS^T, as the state in the forward
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int d = d0 + row + 8 * (e >> 1), k = 8 * (w * NT + n) + col + (e & 1);
      S[n][e] = p.ds_out && d < p.dv && k < p.dk ? p.ds_out[(bh * p.dk + k) * p.dv + d] : 0.f;
    }
  // dS after chunk c to the team, and to the gradients
  auto publish = [&](int c) {
#pragma unroll
    for (int m = 0; m < NT / 2; ++m) {
      const int kk = w * NT / 2 + m;
      uint32_t a[NP][4];
      operand<NP>(S[2 * m], S[2 * m + 1], a);
      Ch::put(state + kk * NP * 32, a);
      if (kk < n_k16 && c >= 0)
#pragma unroll
        for (int i = 0; i < PS; ++i)
          Ch::keep(p.dstates + ((((i * (int64_t)p.B * p.H + bh) * chunks + c) * slices + slice) * n_k16 + kk) * 256, a[i]);
    }
  };
  publish(chunks - 1);

  for (int c = chunks - 1, stage = 0, parity = 0; c >= 0; --c) {
    if (!Ch::team_all(team, mbar_wait(&bars.full[stage], parity, kErrWaitMma, &bars.abort_flag))) {
      if (produces) producer.drain(chunks - 1 - c, chunks - 1 - c + plan.stages);
      return;
    }
    const typename Ch::Stage s{smem + stage * bytes, plan.teams};
    const Gates<C>& gate = s.gates();
    // dO^T of the slice as first operands
    uint32_t dO[NB][PX][4];
    float odd = 0.f;  // NaN if a number of it is not finite
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      if constexpr (sizeof(E) == 2) {
        ldsm_t(dO[j][0], smem_u32(s.v(team, 16 * j + v_row, v_piece)));
#pragma unroll
        for (int e = 0; e < 4; ++e) odd = fmaf(low(dO[j][0][e]), 0.f, fmaf(high(dO[j][0][e]), 0.f, odd));
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int t = 16 * j + 8 * (e >> 1) + col, d = row + 8 * (e & 1);
          const float x = s.value(team, t, d), y = s.value(team, t + 1, d);
          odd = fmaf(x, 0.f, fmaf(y, 0.f, odd));
          uint32_t part[PX];
          split<PX>(x, y, part);
#pragma unroll
          for (int i = 0; i < PX; ++i) dO[j][i][e] = part[i];
        }
      }
    }
    int bad = 0;  // tokens up to the last one of dO that is not finite
    if (__any_sync(0xffffffffu, !(odd == 0.f))) {  // (rare) must not meet the zeros of P: counts as zero, and makes NaN at the end
      bad = Ch::bad_row(s, team, true);
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int i = 0; i < PX; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int t = 16 * j + 8 * (e >> 1) + col;
            dO[j][i][e] &= (t < bad ? 0u : 0x0000ffffu) | (t + 1 < bad ? 0u : 0xffff0000u);
          }
    }
    // (K dS1)^T
    float Z[2][4];
    {
      constexpr int L = 2;
      float z[L][2][4];
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int i = 0; i < L; ++i) zero(z[i][m]);
      uint32_t a[2][NP][4], f[2][PX][4];
      auto fetch = [&](int kk, uint32_t(&a)[NP][4], uint32_t(&f)[PX][4]) {
        Ch::template get<NP>(state + kk * NP * 32, a);
#pragma unroll
        for (int i = 0; i < PX; ++i) ldsm(f[i], s.k() + across.at<C>(w, kk) + i * G::kTile * 2);
      };
      fetch(0, a[0], f[0]);
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        if (kk + 1 < KK) fetch(kk + 1, a[(kk + 1) & 1], f[(kk + 1) & 1]);
        mma_levels<NP, PX, NP, L>(z, a[kk & 1], f[kk & 1]);
      }
      sum_levels<L>(Z, z);
    }
    // what reaches U from outside its own chunk's corrections: P^T dO + e^(b_C - b) K dS1, transposed
    {
      float x[KX][2][4];
#pragma unroll
      for (int i = 0; i < KX; ++i) zero(x[i][0]), zero(x[i][1]);
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        if (i < w) continue;
        uint32_t f[PP][4];
        Ch::template get<PP>(s.p() + lower(i, w) * PP * 32, f);
        mma_levels<PX, PP, KX, KX>(x, dO[i], f);
      }
      float y[2][4];
      sum_levels<KX>(y, x);
      float scaled[2][4];  // scale e^b dO of these tokens
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const float2 out = *reinterpret_cast<const float2*>(gate.out + 16 * w + 8 * m + col);
        const float2 eb = *reinterpret_cast<const float2*>(gate.e + 16 * w + 8 * m + col);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          y[m][e] = fmaf(e & 1 ? out.y : out.x, Z[m][e], y[m][e]);
          float v = 0.f;
#pragma unroll
          for (int i = PX - 1; i >= 0; --i) {
            uint32_t u = 0;
#pragma unroll
            for (int j = 0; j < NB; ++j)
              if (j == w) u = dO[j][i][2 * m + (e >> 1)];
            v += e & 1 ? high(u) : low(u);
          }
          scaled[m][e] = v * (p.scale * (e & 1 ? eb.y : eb.x));
        }
      }
      uint32_t a[NP][4];
      operand<NP>(y[0], y[1], a);
      Ch::put(part_x + w * NP * 32, a);
      operand<NP>(scaled[0], scaled[1], a);
      Ch::put(part_o + w * NP * 32, a);
    }
    Ch::team_sync(team);
    if (produces && c < chunks - 1) producer.template refill<true>(chunks - 1 - c);
    // dU^T = x^T T
    {
      float u[NP][2][4], U[2][4];
#pragma unroll
      for (int i = 0; i < NP; ++i) zero(u[i][0]), zero(u[i][1]);
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        if (i < w) continue;
        uint32_t a[NP][4], f[NP][4];
        Ch::template get<NP>(part_x + i * NP * 32, a);
        Ch::template get<NP>(s.t() + lower(i, w) * NP * 32, f);
        mma_levels<NP, NP, NP, NP>(u, a, f);
      }
      sum_levels<NP>(U, u);
      if (bad > 16 * w) {
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (16 * w + 8 * m + col + (e & 1) < bad) U[m][e] = NAN;
      }
      uint32_t a_u[PU][4];
      operand<PU>(U[0], U[1], a_u);
#pragma unroll
      for (int i = 0; i < PU; ++i)
        Ch::keep(p.du + ((((i * (int64_t)p.B * p.H + bh) * chunks + c) * slices + slice) * NB + w) * 256, a_u[i]);
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const float2 beta = *reinterpret_cast<const float2*>(gate.beta + 16 * w + 8 * m + col);
        const float2 eb = *reinterpret_cast<const float2*>(gate.e + 16 * w + 8 * m + col);
#pragma unroll
        for (int e = 0; e < 4; ++e) U[m][e] *= -(e & 1 ? beta.y * eb.y : beta.x * eb.x);
      }
      uint32_t a[NP][4];
      operand<NP>(U[0], U[1], a);
      Ch::put(part_u + w * NP * 32, a);
    }
    Ch::team_sync(team);
    // dS0^T = e^(b_C) dS1^T + (scale e^b dO)^T Q - (beta e^b dU)^T K
    const float total = gate.total;
    constexpr int NX = NT < 4 ? NT : 4;
#pragma unroll
    for (int n = 0; n < NT; n += NX) {
      float x[NX][4];
#pragma unroll
      for (int m = 0; m < NX; ++m) zero(x[m]);
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        uint32_t a[NP][4], g[NP][4];
        Ch::template get<NP>(part_o + j * NP * 32, a);
        Ch::template get<NP>(part_u + j * NP * 32, g);
#pragma unroll
        for (int m = 0; m < NX; m += 2) {
          uint32_t f[PX][4], k[PX][4];
#pragma unroll
          for (int i = 0; i < PX; ++i) {
            const uint32_t at = 2 * i * G::kTile + j * 2048 + down[(n + m) / 2];
            ldsm_t(f[i], s.q() + at);
            ldsm_t(k[i], s.k() + at);
          }
          mma_parts<NP, PX, NP>(x[m], x[m + 1], a, f);
          mma_parts<NP, PX, NP>(x[m], x[m + 1], g, k);
        }
      }
#pragma unroll
      for (int m = 0; m < NX; ++m)
#pragma unroll
        for (int e = 0; e < 4; ++e) S[n + m][e] = fmaf(total, S[n + m][e], x[m][e]);
    }
    if (bad > 0) {
#pragma unroll
      for (int n = 0; n < NT; ++n) S[n][0] = S[n][1] = S[n][2] = S[n][3] = NAN;
    }
    publish(c - 1);
    __syncwarp();
    if (l == 0) mbar_arrive(&bars.empty[stage]);
    if (++stage == plan.stages) stage = 0, parity ^= 1;
  }
  if (p.ds_in) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = d0 + row + 8 * (e >> 1), k = 8 * (w * NT + n) + col + (e & 1);
        if (d < p.dv && k < p.dk) p.ds_in[(bh * p.dk + k) * p.dv + d] = S[n][e];
      }
  }
}

template <typename G, int KK>
int go(const Backward& p, const Plan& plan, cudaStream_t st) {
  using Ch = Chain<G, KK>;
  int s;
  const int slices = (p.dv + 15) / 16, smem = Ch::smem_bytes(plan.teams, plan.stages);
  if ((s = allow_shared(delta_bwd_kernel<G, KK>, Ch::kMostBytes, "cudaFuncSetAttribute(delta_bwd)"))) return s;
  Maps maps{};
  if ((s = chain_maps<G>(&maps, p.pre, p.k, p.q, p.d_o, p.B, p.T, p.H, p.dk, p.dv, plan.teams))) return s;
  const dim3 grid((unsigned)((slices + plan.teams - 1) / plan.teams), (unsigned)(p.B * p.H));
  delta_bwd_kernel<G, KK><<<grid, 32 * (plan.teams * Ch::W + plan.own_warp), smem, st>>>(p, maps, plan);
  DYNCONV_CHECK_LAUNCH("delta_bwd_kernel");
  return DYNCONV_OK;
}

template <typename G>
int pick(const Backward& p, cudaStream_t st) {
  const int64_t bh = (int64_t)p.B * p.H;
  if (p.dk <= 64) return go<G, 4>(p, plan_of<Chain<G, 4>>(bh, p.dv), st);
  return go<G, 8>(p, plan_of<Chain<G, 8>>(bh, p.dv), st);
}

}  // namespace

// Three parts where the gradient of the first state goes back to the caller, as in the forward.
int backward_launch(const Backward& p, int dtype, cudaStream_t st) {
  const bool exact = p.ds_in != nullptr;
  int s = prep_launch(p.pre, p.k, p.q, p.d_o, p.g, p.beta, p.gates32, p.B, p.H, p.T, p.dk, p.dv, p.scale, dtype, exact, true, st);
  if (s) return s;
  s = dtype == DYNCONV_DTYPE_F32 ? pick<CfgF32>(p, st) : exact ? pick<CfgBf16<true, true>>(p, st) : pick<CfgBf16<false, true>>(p, st);
  return s ? s : grad_launch(p, dtype, st);
}

}  // namespace dr

DYNCONV_DEFINE_ERROR_ACCESSOR(dr_bwd_error_word)

}  // namespace dynconv
