// delta_chain.cuh -- the frame of the two chain kernels of the gated delta rule (formulas: delta_rule.cuh).
//
// A CTA walks the chunks of one (batch row, head) for `teams` slices of 16 of v's columns.  A team of W warps, one for each 16
// tokens of a chunk, holds a slice of the state, transposed: warp w keeps 16 x (128 / W) of it in registers, fp32, in the
// accumulators' layout, and works out what belongs to the tokens from 16 w on.  What the others need of a warp's numbers
// goes through shared memory as bf16 parts in the layout of first operands, 16 bytes per lane.  One thread,
// of a warp of its own or, where the chains' warps take all registers, of the first team's warp with the fewest blocks
// of T, right behind a barrier of the team (before it, the whole team waited for the copies' start: 296 and 270 us
// against 278 and 264 us for the chains at 4 x 4096 tokens, 16 heads of 128 x 128), brings the next chunks' tiles
// by TMA into two or three stages.  (16-byte asynchronous copies by threads, of one warp or four, took longer than a
// chunk's products: 10 to 20 bytes per cycle and SM.  Asking for the chunk after next into L2 as well: 316 and 319 us.)
//
// Why teams: one warp per slice, its numbers all in registers, took 7400 cycles for a chunk of 64 tokens
// and 128 x 128 states, four times what its matrix instructions need: every instruction waited for the one
// before.  More warps hide that, and where there are few chains they bring idle quarters of the SM to bear.
#pragma once

#include "delta_rule.cuh"

namespace dynconv {
namespace dr {

struct Plan {
  int teams, stages;
  int o_vectors;
  int own_warp;  // the producer has one
};

// KK: pieces of 16 of dk that are worked on, 4 or 8 (behind dk there are zeros).
template <typename G, int KK_>
struct Chain {
  static constexpr int C = G::C, NP = G::NP, PX = G::PX, PP = G::PP, NB = G::kBlocks;
  static constexpr int W = NB;                     // warps of a team, one for each block of 16 tokens
  static constexpr int KK = KK_, NT = 2 * KK / W;  // a warp's 8-column tiles of the state
  static constexpr int PU = PX == 1 ? 2 : 3;  // parts of what the backward is given
  using E = typename G::T;
  static constexpr int kMostTeams = NP == 2 ? 4 : 2;  // (three parts: the registers of 8 warps, and shared memory)
  static constexpr int kMostThreads = 32 * W * kMostTeams;

  static constexpr int kKq = PX * G::kTile * 2;  // bytes
  static constexpr int kRow = 16 * (int)sizeof(E), kV = C * kRow;  // of a team's columns: the tile is [C tokens][teams * 16]
  static constexpr int kT = G::kLower * NP * 512, kP = G::kLower * PP * 512, kGates = sizeof(Gates<C>);
  static constexpr int kState = KK * NP * 512, kBlock = NB * NP * 512;  // a team's buffers
  static constexpr int kTeam = kState + 3 * kBlock;
  static __host__ __device__ constexpr int stage_bytes(int teams) {
    return (2 * kKq + teams * kV + kT + kP + kGates + 1023) / 1024 * 1024;
  }
  static constexpr int smem_bytes(int teams, int stages) { return 1024 + stages * stage_bytes(teams) + teams * kTeam; }
  static constexpr int kMostBytes = 227 * 1024 - 1024;  // of any plan (the rest: barriers)
  static_assert(smem_bytes(1, 2) <= kMostBytes, "the smallest plan");

  struct Stage {
    uint8_t* at;
    int teams;
    __device__ __forceinline__ uint32_t k() const { return smem_u32(at); }
    __device__ __forceinline__ uint32_t q() const { return smem_u32(at) + kKq; }
    __device__ __forceinline__ uint8_t* v() const { return at + 2 * kKq; }
    // a token's 16-byte piece of a team's columns
    __device__ __forceinline__ uint8_t* v(int team, int r, int piece) const {
      return v() + row_swizzle(teams * kRow, r, team * (kRow / 16) + piece);
    }
    __device__ __forceinline__ E& value(int team, int r, int d) const {
      return ((E*)v(team, r, d / (16 / (int)sizeof(E))))[d % (16 / (int)sizeof(E))];
    }
    __device__ __forceinline__ uint4* t() const { return (uint4*)(at + 2 * kKq + teams * kV); }
    __device__ __forceinline__ uint4* p() const { return t() + kT / 16; }
    __device__ __forceinline__ Gates<C>& gates() const { return *(Gates<C>*)(p() + kP / 16); }
  };

  struct Bars {
    uint64_t full[3], empty[3];
    int abort_flag;
  };

  // The team's barrier.
  static __device__ __forceinline__ void team_sync(int team) {
    asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "n"(32 * W) : "memory");
  }
  // The barrier with "and" of `ok`: a team whose wait gave up leaves as a whole.
  static __device__ __forceinline__ bool team_all(int team, bool ok) {
    uint32_t all;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %1, 0;\n\tbarrier.cta.red.and.pred p, %2, %3, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(all)
                 : "r"((uint32_t)ok), "r"(team + 1), "n"(32 * W)
                 : "memory");
    return all != 0;
  }
  static __device__ __forceinline__ int live_teams(const Plan& plan, int dv, int first_col) {
    return min(plan.teams, (dv - first_col + 15) / 16);
  }
  static __device__ __forceinline__ void init(Bars& bars, int live) {
    if (threadIdx.x == 0) {
      for (int i = 0; i < 3; ++i) mbar_init(&bars.full[i], 1), mbar_init(&bars.empty[i], live * W);
      bars.abort_flag = 0;
      fence_barrier_init();
    }
    __syncthreads();
  }

  // One thread asks for the tiles of the n-th chunk in the order of the walk (BACK: from the last chunk to the first).
  struct Producer {
    uint8_t* smem;
    Bars& bars;
    const Plan& plan;
    const Maps& maps;
    const Prepared& pre;
    int b, h, chunks, dk, dv, first_col;
    int64_t bh;

    template <bool BACK>
    __device__ __forceinline__ void load(int n, int stage) const {
      const int halves = dk > 64 ? 2 : 1;
      const uint32_t half = C * 128, all = 2 * PX * halves * half + plan.teams * kV + kT + kP + kGates;
      const Stage st{smem + stage * stage_bytes(plan.teams), plan.teams};
      uint8_t *const k = st.at, *const q = st.at + kKq;
      const int c = BACK ? chunks - 1 - n : n;
      const int64_t at = bh * chunks + c;
      uint64_t* const bar = &bars.full[stage];
      mbar_arrive_expect_tx(bar, all);
      if (pre.k) {
        for (int i = 0; i < PX; ++i) {
          const int64_t from = (at * PX + i) * halves * (C * 64);
          bulk_load(k + i * G::kTile * 2, pre.k + from, halves * half, bar);
          bulk_load(q + i * G::kTile * 2, pre.q + from, halves * half, bar);
        }
      } else {
        for (int d = 0; d < halves; ++d) {
          tma_load_4d(k + d * half, &maps.k, bar, 64 * d, h, c * C, b, policy_evict_normal());
          tma_load_4d(q + d * half, &maps.q, bar, 64 * d, h, c * C, b, policy_evict_normal());
        }
      }
      tma_load_4d(st.v(), &maps.v, bar, first_col * (int)(sizeof(E) / 2), h, c * C, b, policy_evict_normal());
      bulk_load(st.t(), pre.t + at * (kT / 16), kT, bar);
      bulk_load(st.p(), pre.p + at * (kP / 16), kP, bar);
      bulk_load(&st.gates(), (const uint8_t*)pre.gates + at * kGates, kGates, bar);
    }
    template <bool BACK>
    __device__ __forceinline__ void start() const {
      for (int n = 0; n < plan.stages && n < chunks; ++n) load<BACK>(n, n);
    }
    // In the n-th chunk, n > 0: refills the stage of the chunk before it, once all warps are done with it.
    template <bool BACK>
    __device__ __forceinline__ void refill(int n) const {
      const int next = n - 1 + plan.stages, stage = (n - 1) % plan.stages, round = (n - 1) / plan.stages;
      if (next < chunks && mbar_wait(&bars.empty[stage], round & 1, kErrWaitProducer, &bars.abort_flag)) load<BACK>(next, stage);
    }
    // The walk of a producer with a warp of its own.
    template <bool BACK>
    __device__ __forceinline__ void walk() const {
      int n = 0;
      for (; n < chunks; ++n) {
        const int stage = n % plan.stages, round = n / plan.stages;
        if (round > 0 && !mbar_wait(&bars.empty[stage], (round - 1) & 1, kErrWaitProducer, &bars.abort_flag)) break;
        load<BACK>(n, stage);
      }
      if (n < chunks) drain(max(0, n - plan.stages), n);
    }
    // The wait for chunk n gave up: what is in flight lands before the shared memory goes.
    __device__ __forceinline__ void drain(int n, int end) const {
      for (int i = n; i < end && i < chunks; ++i) mbar_drain(&bars.full[i % plan.stages], (i / plan.stages) & 1);
    }
  };

  // The first row (last: one more than the last) of a team's columns that holds a number that is not finite; C (0)
  // where there is none.  One warp.
  static __device__ __noinline__ int bad_row(Stage s, int team, bool last) {
    int bad = last ? 0 : C;
    for (int r = threadIdx.x & 31; r < C; r += 32)
      for (int d = 0; d < 16; ++d)
        if (!(fabsf(Elem<E>::to_f(s.value(team, r, d))) < INFINITY)) bad = last ? max(bad, r + 1) : min(bad, r);
    return last ? __reduce_max_sync(0xffffffffu, bad) : __reduce_min_sync(0xffffffffu, bad);
  }

  // A first operand's parts to and from a team's buffer.
  template <int N>
  static __device__ __forceinline__ void put(uint4* to, const uint32_t (&a)[N][4]) {
#pragma unroll
    for (int i = 0; i < N; ++i) to[i * 32 + (threadIdx.x & 31)] = make_uint4(a[i][0], a[i][1], a[i][2], a[i][3]);
  }
  template <int N>
  static __device__ __forceinline__ void get(const uint4* from, uint32_t (&a)[N][4]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint4 u = from[i * 32 + (threadIdx.x & 31)];
      a[i][0] = u.x, a[i][1] = u.y, a[i][2] = u.z, a[i][3] = u.w;
    }
  }
  // The same for the backward, as four matrices of 128 bytes.
  static __device__ __forceinline__ void keep(__nv_bfloat16* to, const uint32_t (&a)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) ((uint32_t*)to)[e * 32 + (threadIdx.x & 31)] = a[e];
  }
};

template <typename G>
int chain_maps(Maps* maps, const Prepared& pre, const View& k, const View& q, const View& v, int B, int64_t T, int H, int dk, int dv, int teams) {
  int s = DYNCONV_OK;
  if (!pre.k && ((s = view_map(&maps->k, k, B, T, H, dk, 2, 64, G::C)) || (s = view_map(&maps->q, q, B, T, H, dk, 2, 64, G::C)))) return s;
  return value_map(&maps->v, pre, v, B, T, H, dv, sizeof(typename G::T), 16 * teams, G::C);
}

// CTAs of as few teams as let all slices run at once, each then having more of its SM's matrix units and shared
// memory; and of no more than there are slices, since a team without columns would only take the copies' own warp and
// a stage (200 chains of 2048 tokens, 64 x 16: 211 us with four teams, 193 with the one that has columns).
template <typename Ch>
Plan plan_of(int64_t bh, int dv) {
  const int slices = (dv + 15) / 16;
  Plan p{};
  p.teams = 1;
  while (2 * p.teams <= Ch::kMostTeams && p.teams < slices && Ch::smem_bytes(2 * p.teams, 2) <= Ch::kMostBytes && bh * ((slices + p.teams - 1) / p.teams) > sm_count())
    p.teams *= 2;
  p.stages = Ch::smem_bytes(p.teams, 3) <= Ch::kMostBytes ? 3 : 2;
  p.own_warp = p.teams < Ch::kMostTeams;
  return p;
}

}  // namespace dr
}  // namespace dynconv
