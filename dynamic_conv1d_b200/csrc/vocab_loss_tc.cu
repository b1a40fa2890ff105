// vocab_loss_tc.cu -- the vocabulary loss's products, on the tensor cores: of bf16 tensors in place, of
// fp32 ones as three bf16 parts, of bf16 rows that TMA cannot address as padded copies.
//
// One persistent kernel computes out(m, n) = sum_k A(m, k) B(n, k) for all four products;
// only the operands' majors and the epilogue differ:
//     forward       A = hidden [N][D],      B = weight [V][D]      -> row maxima and sums
//     logits' grad  A = hidden,             B = weight piece       -> dl (bf16, piece buffer)
//     dhidden       A = dl [N][piece],      B = weight piece^T     -> fp32, added up over pieces
//     dweight       A = dl^T,               B = hidden^T           -> bf16
// K-major operands are TMA boxes of 64 K elements x rows, the transposed ones boxes of 64
// rows x 64 K steps; both land in 128-byte-swizzled tiles that tcgen05.mma reads as they
// are, so nothing is ever transposed in memory.
//
// Two CTAs of a cluster (the two SMs of a TPC) work on one 256 x 256 tile with cta_group::2
// products: each holds its 128 rows of A and half of B's 256 rows, and its 128 rows of the
// accumulator.  A CTA by itself on 128 x 256 would move 24 KB through shared memory for each
// product of 16 inner elements (12 KB written by TMA, 12 KB read by the product), 192 cycles at
// 128 bytes each for 128 cycles of tensor work; a pair moves 16 KB per SM.
// Each CTA runs one producer warp (TMA ring of kStages) and eight epilogue warps (two per TMEM
// lane quarter, half of the columns each); the pair's first CTA issues the products.  Two
// accumulators of 256 TMEM columns let a tile's epilogue run under the next tile's products.
//
// What bounds it: the tensor cores at the clock that the power limit leaves (pipe 88 to 92% active).
// 16384 tokens x 2048 channels over 50001 words (B200, bf16): forward 2.2 ms, logits again 2.3,
// weight gradient 2.15, hidden gradient 2.1 ms: 1.5 PFLOP/s each, 94% of a library product's
// burst rate; back to back under the power limit the pass takes 10.8 ms (1.25 PFLOP/s; that
// library product sustains 1.38).
//
// Copied operands (PARTS) go through the same kernel.  fp32: a small kernel writes each tensor as
// three bf16 parts, the inner dimension is walked once for each of six products of parts, and dl
// leaves the epilogue as parts too.  The sums of 256 inner elements' products are added up in
// registers (the tensor core's sums alone would be off by more than fp32's rounding).  Products at
// 1/6 of the bf16 rate are 3.5 times what the fp32 units could do at their best.  Whole passes, forward
// and backward (B200; in brackets fp32 products on the CUDA cores, in tiles of 128 x 128): 1021 tokens x
// 256 channels over 4999 words 34 + 102 us (90 + 233), 1021 x 1024 x 8000 93 + 269 us (400 + 1226), 4096 x
// 2048 x 65536 5.0 + 16.2 ms (20.8 + 71.1): 1.25 PFLOP/s of bf16 products.  Few rows gain only over
// large vocabularies, as the tensors are written anew: one row of 256 x 4999 25 + 61 us (19 + 40), of
// 2048 x 65536 0.83 + 1.27 ms (0.63 + 1.52), 32 rows of the latter 0.59 + 1.12 (0.65 + 1.67).  Elementary torch
// operations are faster there: whole calls of one row of 2048 x 9000 188 us against 360 here, of 2048 x 20000 240
// against 706; from about 64 rows on, or over 4999 words of 256, they are not.  bf16, 1021 x 257 x 4999: 118 us of
// kernels (430).
#include "vocab_loss.cuh"

namespace dynconv {
namespace vl {

namespace {

constexpr int kM = 256, kN = 256, kKB = 64;  // a pair's tile, and inner elements per stage
constexpr int kHalfM = 128, kHalfB = 128;    // rows of A and of B in one CTA
constexpr int kStages = 6;
constexpr int kEpiWarps = 8;
constexpr int kTcThreads = 64 + 32 * kEpiWarps;
constexpr uint32_t kABytes = kHalfM * kKB * 2, kBBytes = kHalfB * kKB * 2, kStageBytes = kABytes + kBBytes;
constexpr uint32_t kAtom = 64 * kKB * 2;  // one 64 x 64 box
constexpr uint32_t kStageOut = 32 * 128;  // an epilogue warp's 32 rows x 64 columns of bf16, staged for a TMA store
constexpr int kSmem = kStages * (int)kStageBytes + kEpiWarps * (int)kStageOut + 1024;
static_assert(kSmem <= 232448 - 2048, "shared memory of one CTA");
// The tensor core's accumulation truncates: a sum of 4096 products came out 3.8e-6 of itself too
// small, which the loss's 32 bits would show (1.1e-6 of it).  Where the inner dimension is longer
// than kChain blocks (2048 products), the logits are summed that many at a time and those sums added
// up in registers (the long modes; forms of their own, as they need 128 registers more).  The backward does as
// the forward, bit for bit: dl is the difference of a logit and the forward's sums, and where a row's target
// dominates it, dl is smaller than what the two ways of adding differ by.  The gradients' own sums are not
// broken up: over 16384 tokens they lose 2^-16, and are rounded to 2^-8.
constexpr int kChain = 32;
constexpr int kHalf = kN / 2;  // columns of one epilogue warp; a forward tile's partials are per half

enum TcMode { kTcForward, kTcForwardLong, kTcGrad, kTcGradLong, kTcAdd, kTcStore };

struct TcGemm {
  int64_t M, N;        // extents of the output
  int k_blocks;        // 64-element blocks of the inner dimension (COPIED: of each product of parts)
  int m_tiles, n_tiles, z;
  int group;           // m tiles that share a sweep over n: consecutive tiles walk a group's rows first
  int64_t col0;        // kTcGrad: first vocabulary column
  void* out;           // kTcAdd: fp32 [z][M][N] (the bf16 outputs go through a tensor map)
  int64_t out_ld;
  int add;             // kTcAdd: add to what is there
  void* result;        // kTcAdd: not null: the last sums, in the tensors' type
  int vec;             // COPIED kTcAdd: rows of result may be written 16 bytes at a time
};

struct Tile {
  int m, n, z, kb0, kb1;
};

template <int PARTS>
__device__ __forceinline__ Tile tile_at(const TcGemm& g, int t) {
  Tile r;
  const int plane = g.m_tiles * g.n_tiles;
  r.z = t / plane;
  t -= r.z * plane;
  const int grp = t / (g.group * g.n_tiles);
  t -= grp * g.group * g.n_tiles;
  const int rows = min(g.group, g.m_tiles - grp * g.group);
  r.n = t / rows;
  r.m = grp * g.group + (t - r.n * rows);
  if constexpr (PARTS > 0) {  // whole chains
    const int64_t chains = (g.k_blocks + kCopyChain - 1) / kCopyChain;
    constexpr int products = products_of(PARTS);
    r.kb0 = (int)(chains * r.z / g.z) * kCopyChain * products;
    r.kb1 = min((int)(chains * (r.z + 1) / g.z) * kCopyChain, g.k_blocks) * products;
  } else {
    r.kb0 = (int)((int64_t)g.k_blocks * r.z / g.z);
    r.kb1 = (int)((int64_t)g.k_blocks * (r.z + 1) / g.z);
  }
  return r;
}

// What the kb-th block of products of three parts multiplies: kCopyChain blocks' six products at a
// time, the smallest products first.
struct CopyBlock {
  int block, a, b;  // 64 inner elements, parts of A and B
};

__device__ __forceinline__ CopyBlock copy_block(int k_blocks, int kb) {
  const int chain = kb / (kCopyChain * 6), r = kb - chain * kCopyChain * 6;
  const int blocks = min(kCopyChain, k_blocks - chain * kCopyChain), product = r / blocks;
  // parts (0,2), (1,1), (2,0), (0,1), (1,0), (0,0)
  return {chain * kCopyChain + r - product * blocks, 0x010210 >> (4 * product) & 3, 0x001012 >> (4 * product) & 3};
}

// ---- a CTA pair: addresses in the first CTA, products over both

__device__ __forceinline__ uint32_t cta_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
  return r;
}

__device__ __forceinline__ uint32_t in_first_cta(const void* p) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(smem_u32(p)));
  return a;
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ void arrive_in_first_cta(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// Into this CTA's shared memory, counted on the first CTA's barrier.
__device__ __forceinline__ void tma_load_pair(void* dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, "
      "%4}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1)
      : "memory");
}

// The same from one of a copy's parts.
__device__ __forceinline__ void tma_load_pair(void* dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int part) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, "
      "%4, %5}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(part)
      : "memory");
}

__device__ __forceinline__ void umma_pair(uint32_t elected, uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo,
                                          uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 a, b;\n\t"
      "setp.ne.b32 p, %5, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
      "mov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
      "@q tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %4, p;\n\t}" ::"r"(d_tmem),
      "r"(a_lo), "r"(b_lo), "n"(kDescHiSw128), "r"(idesc), "r"(accumulate), "r"(elected)
      : "memory");
}

// Arrives on the barrier at this place in both CTAs when the products issued so far are done.
__device__ __forceinline__ void umma_commit_pair(uint32_t elected, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %2;\n\t}" ::"r"(
          smem_u32(bar)),
      "r"(elected), "h"((uint16_t)3)
      : "memory");
}

__device__ __forceinline__ void tmem_alloc_pair(uint32_t* dst_smem, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst_smem)), "r"(ncols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}

// v[at].  (Selected by masks: an indexed read would put v into local memory.)
template <int n>
__device__ __forceinline__ float pick(const float (&v)[n], int at) {
  uint32_t bits = 0;
#pragma unroll
  for (int j = 0; j < n; ++j) bits |= __float_as_uint(v[j]) & -(uint32_t)(j == at);
  return __uint_as_float(bits);
}

// dl of n columns, in place.  f: the row's factor, at: the target's column among them, own: its gradient (null
// where the row's loss was not kept).  lse2 = lse * log2(e), rounded: an error of 2^-24 lse in each exponent, as the
// logits themselves have.
template <int n>
__device__ __forceinline__ void logits_gradient(float (&v)[n], float f, float lse2, int at, const float* own) {
#pragma unroll
  for (int j = 0; j < n; ++j) v[j] = f != 0.f ? ex2(fmaf(v[j], kLog2e, -lse2)) * f : 0.f;  // (an ignored row's NaN stays out)
  if (at >= 0 && at < n) {
    const float g = own ? *own : pick(v, at) - f;
#pragma unroll
    for (int j = 0; j < n; ++j)
      if (j == at) v[j] = g;
  }
}

// The next bf16 part of two numbers, packed; the numbers keep the rest (exact).
__device__ __forceinline__ uint32_t take_part(float2& x) {
  const uint32_t p = pack_bf16x2(x.x, x.y);
  x = add2(x, make_float2(-__uint_as_float(p << 16), -__uint_as_float(p & 0xFFFF0000u)));
  return p;
}

// A matrix as its parts: fp32 as three, bf16 as it is; rows padded with zeros.  clean: rows of hidden that
// the gradients leave out (dl has zeros there) are zero, whatever they hold: in the weight's gradient a
// product of zero and a value that is not finite would be NaN for the whole vocabulary.
template <typename In>
__global__ void __launch_bounds__(256) vl_copy_kernel(const In* __restrict__ src, int64_t rows, int64_t D, int64_t pitch,
                                                      __nv_bfloat16* __restrict__ copy, const __grid_constant__ Problem p,
                                                      int clean) {
  const int64_t per = pitch / 8, n = rows * per, plane = rows * pitch;
  const bool vec = D % 8 == 0 && (reinterpret_cast<uintptr_t>(src) & 15) == 0;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t row = i / per, c = (i - row * per) * 8;
    const In* s = src + row * D + c;
    __nv_bfloat16* to = copy + row * pitch + c;
    if (clean && row_factor(p, row, p.target[row]) == 0.f) {
#pragma unroll
      for (int k = 0; k < (sizeof(In) == 2 ? 1 : 3); ++k) *reinterpret_cast<uint4*>(to + k * plane) = make_uint4(0, 0, 0, 0);
      continue;
    }
    if constexpr (sizeof(In) == 2) {
      if (vec) {
        *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(s);
        continue;
      }
      uint32_t w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = c + j < D ? reinterpret_cast<const uint16_t*>(s)[j] : 0;
      *reinterpret_cast<uint4*>(to) = make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
    } else {
      float2 v[4];
      if (vec) {
        const float4 lo = reinterpret_cast<const float4*>(s)[0], hi = reinterpret_cast<const float4*>(s)[1];
        v[0] = make_float2(lo.x, lo.y), v[1] = make_float2(lo.z, lo.w);
        v[2] = make_float2(hi.x, hi.y), v[3] = make_float2(hi.z, hi.w);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          v[j] = make_float2(c + 2 * j < D ? s[2 * j] : 0.f, c + 2 * j + 1 < D ? s[2 * j + 1] : 0.f);
      }
      // the first part is cut to bf16's range: a number close to fp32's largest stays finite, an
      // infinity or a NaN becomes a NaN in the parts that follow
      constexpr float kLargest = 3.38953139e38f;
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float2 cut = make_float2(fminf(fmaxf(v[j].x, -kLargest), kLargest), fminf(fmaxf(v[j].y, -kLargest), kLargest));
        const float2 over = make_float2(v[j].x - cut.x, v[j].y - cut.y);  // zero, but for those
        w[j] = take_part(cut);
        v[j] = add2(cut, over);
      }
      *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
#pragma unroll
      for (int k = 1; k < 3; ++k)
        *reinterpret_cast<uint4*>(to + k * plane) = make_uint4(take_part(v[0]), take_part(v[1]), take_part(v[2]), take_part(v[3]));
    }
  }
}

// COPIED: 16 columns of a row of the fp32 sums (rows padded to whole 16 bytes), added up over pieces;
// the last ones are the result in fp32.
__device__ __forceinline__ void add_columns(const TcGemm& g, const float (&v)[16], int64_t row, int64_t col, int z,
                                            float factor) {
  float* o = (float*)g.out + ((int64_t)z * g.M + row) * g.out_ld + col;
  float* r = (float*)g.result + row * g.N + col;
#pragma unroll
  for (int j = 0; j < 16; j += 4) {
    if (col + j >= g.N) break;
    float4 u = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
    if (g.add) {
      const float4 w = *reinterpret_cast<const float4*>(o + j);
      u.x += w.x, u.y += w.y, u.z += w.z, u.w += w.w;
    }
    if (!g.result) {
      *reinterpret_cast<float4*>(o + j) = u;
      continue;
    }
    u.x *= factor, u.y *= factor, u.z *= factor, u.w *= factor;
    if (g.vec) {
      *reinterpret_cast<float4*>(r + j) = u;
    } else {
      r[j] = u.x;
      if (col + j + 1 < g.N) r[j + 1] = u.y;
      if (col + j + 2 < g.N) r[j + 2] = u.z;
      if (col + j + 3 < g.N) r[j + 3] = u.w;
    }
  }
}

// 32 columns of a row of the fp32 sums, added up over pieces; the last piece rounds them into
// the result itself.  Widths are multiples of 8.
__device__ __forceinline__ void add_columns(const TcGemm& g, const float (&v)[32], int64_t row, int64_t col, int z,
                                            float factor) {
  float* o = (float*)g.out + ((int64_t)z * g.M + row) * g.out_ld + col;
  __nv_bfloat16* r = (__nv_bfloat16*)g.result + row * g.out_ld + col;
#pragma unroll
  for (int j = 0; j < 32; j += 8) {
    if (col + j >= g.N) break;
    float4 u0 = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]), u1 = make_float4(v[j + 4], v[j + 5], v[j + 6], v[j + 7]);
    if (g.add) {
      const float4 w0 = *reinterpret_cast<const float4*>(o + j), w1 = *reinterpret_cast<const float4*>(o + j + 4);
      u0.x += w0.x, u0.y += w0.y, u0.z += w0.z, u0.w += w0.w;
      u1.x += w1.x, u1.y += w1.y, u1.z += w1.z, u1.w += w1.w;
    }
    if (g.result) {
      u0.x *= factor, u0.y *= factor, u0.z *= factor, u0.w *= factor;
      u1.x *= factor, u1.y *= factor, u1.z *= factor, u1.w *= factor;
      *reinterpret_cast<uint4*>(r + j) =
          make_uint4(pack_bf16x2(u0.x, u0.y), pack_bf16x2(u0.z, u0.w), pack_bf16x2(u1.x, u1.y), pack_bf16x2(u1.z, u1.w));
    } else {
      *reinterpret_cast<float4*>(o + j) = u0;
      *reinterpret_cast<float4*>(o + j + 4) = u1;
    }
  }
}

// n columns of a row from column c on, rounded into the warp's staged tile (128-byte swizzle).
template <int n>
__device__ __forceinline__ void stage_columns(uint8_t* tile, int row, int c, const float (&v)[n]) {
#pragma unroll
  for (int j = 0; j < n / 8; ++j) {
    const uint4 u = make_uint4(pack_bf16x2(v[8 * j], v[8 * j + 1]), pack_bf16x2(v[8 * j + 2], v[8 * j + 3]),
                               pack_bf16x2(v[8 * j + 4], v[8 * j + 5]), pack_bf16x2(v[8 * j + 6], v[8 * j + 7]));
    *reinterpret_cast<uint4*>(tile + row * 128 + (((c / 8 + j) ^ (row & 7)) << 4)) = u;
  }
}

template <int MODE, bool A_MN, bool B_MN, int PARTS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kTcThreads, 1)
    vl_tc_kernel(const __grid_constant__ CUtensorMap amap, const __grid_constant__ CUtensorMap bmap,
                 const __grid_constant__ CUtensorMap omap, const __grid_constant__ TcGemm g, const __grid_constant__ Problem p) {
  constexpr bool COPIED = PARTS > 0;
  constexpr bool kForward = MODE == kTcForward || MODE == kTcForwardLong;
  constexpr bool kGrad = MODE == kTcGrad || MODE == kTcGradLong;
  constexpr bool kChained = MODE == kTcForwardLong || MODE == kTcGradLong || COPIED;  // sums of kBlocks blocks are added up in registers
  constexpr int kBlocks = COPIED ? kCopyChain * products_of(PARTS) : kChain;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align_smem_1024(smem_raw);
  // full and acce are used in the first CTA only; empty and accf in both
  __shared__ uint64_t full_bar[kStages], empty_bar[kStages], accf_bar[2], acce_bar[2], drain_bar;
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  // kGrad: each row's dl at its target, needed by one column of it (in a register it cost the fp32 backward
  // 2 us of 102 at 1021 x 256 x 4999: beside 128 sums there is none left)
  __shared__ float target_dl[kGrad ? kEpiWarps : 1][32];
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int n_tiles = g.m_tiles * g.n_tiles * g.z;
  const int rank = (int)cta_rank(), pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&accf_bar[a], 1);
      mbar_init(&acce_bar[a], 2 * kEpiWarps);
    }
    mbar_init(&drain_bar, 1);
    abort_flag = 0;
    fence_barrier_init();
    prefetch_tensormap(&amap);
    prefetch_tensormap(&bmap);
  }
  if (warp == 1) tmem_alloc_pair(&tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      int it = 0;
      bool dead = false;
      for (int i = pair; i < n_tiles && !dead; i += pairs) {
        const Tile t = tile_at<PARTS>(g, i);
        const int m0 = t.m * kM + rank * kHalfM, n0 = t.n * kN + rank * kHalfB;
        for (int kb = t.kb0; kb < t.kb1; ++kb, ++it) {
          const int s = it % kStages;
          if (!mbar_wait(&empty_bar[s], ((it / kStages) & 1) ^ 1, kErrWaitProducer, &abort_flag)) {
            dead = true;
            break;
          }
          uint8_t* a = smem + s * kStageBytes;
          uint8_t* b = a + kABytes;
          const uint32_t full = in_first_cta(&full_bar[s]);
          // the first CTA announces both CTAs' bytes (the other's may land before: the phase
          // still waits for this arrival)
          if (rank == 0) mbar_arrive_expect_tx(&full_bar[s], 2 * kStageBytes);
          CopyBlock cb{kb, 0, 0};
          if constexpr (PARTS == 3) cb = copy_block(g.k_blocks, kb);
          auto load = [&](uint8_t* dst, const CUtensorMap* map, int c0, int c1, int part) {
            if constexpr (COPIED)
              tma_load_pair(dst, map, full, c0, c1, part);
            else
              tma_load_pair(dst, map, full, c0, c1);
          };
          if constexpr (A_MN) {
#pragma unroll
            for (int j = 0; j < kHalfM / 64; ++j) load(a + j * kAtom, &amap, m0 + j * 64, cb.block * kKB, cb.a);
          } else {
            load(a, &amap, cb.block * kKB, m0, cb.a);
          }
          if constexpr (B_MN) {
#pragma unroll
            for (int j = 0; j < kHalfB / 64; ++j) load(b + j * kAtom, &bmap, n0 + j * 64, cb.block * kKB, cb.b);
          } else {
            load(b, &bmap, cb.block * kKB, n0, cb.b);
          }
        }
      }
      // a wait gave up: let the copies in flight land before the shared memory is given back (the
      // pair leaves together)
      if (abort_flag && rank == 0)
        for (int j = max(0, it - kStages); j < it; ++j)
          mbar_drain(&full_bar[j % kStages], (j / kStages) & 1);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 0) {
      constexpr uint32_t idesc = make_idesc_bf16(kM, kN, A_MN, B_MN);
      const uint32_t el = elect_lane();
      const uint32_t sb = smem_u32(smem);
      int it = 0, n = 0;
      bool dead = false;
      for (int i = pair; i < n_tiles && !dead; i += pairs, ++n) {
        const Tile t = tile_at<PARTS>(g, i);
        int a = n & 1, first = t.kb0;
        for (int kb = t.kb0; kb < t.kb1; ++kb, ++it) {
          if (kb == t.kb0 || (kChained && kb - first == kBlocks)) {
            if (kb > t.kb0) ++n;
            a = n & 1, first = kb;
            if (!mbar_wait(&acce_bar[a], ((n >> 1) & 1) ^ 1, kErrWaitMma, &abort_flag)) {
              dead = true;
              break;
            }
            asm volatile("fence.acq_rel.cluster;" ::: "memory");  // (half of the arrivals came from the other CTA)
            tc_fence_after();
          }
          const int s = it % kStages;
          if (!mbar_wait(&full_bar[s], (it / kStages) & 1, kErrWaitMma, &abort_flag)) {
            dead = true;
            break;
          }
          tc_fence_after();
          const uint32_t as = sb + s * kStageBytes;
          const uint32_t ad = desc_lo(as, A_MN ? kAtom : 16), bd = desc_lo(as + kABytes, B_MN ? kAtom : 16);
#pragma unroll
          for (int k = 0; k < kKB / 16; ++k)
            umma_pair(el, tmem + a * kN, ad + k * (A_MN ? 2048 : 32) / 16, bd + k * (B_MN ? 2048 : 32) / 16, idesc,
                      (kb > first || k > 0) ? 1u : 0u);
          umma_commit_pair(el, &empty_bar[s]);
          if (kb == t.kb1 - 1 || (kChained && kb - first == kBlocks - 1)) umma_commit_pair(el, &accf_bar[a]);
          __syncwarp();
        }
      }
      if (abort_flag) {  // the products in flight, before their accumulators are given back
        umma_commit_pair(el, &drain_bar);
        mbar_drain(&drain_bar, 0);
      }
    }
  } else {
    const int q = warp & 3, half = (warp - 2) >> 2;
    bool dead = false;
    int n = 0;
    const float factor = MODE == kTcAdd || MODE == kTcStore ? result_factor(p) : 1.f;
    const uint32_t freed[2] = {in_first_cta(&acce_bar[0]), in_first_cta(&acce_bar[1])};
    for (int i = pair; i < n_tiles; i += pairs, ++n) {
      const Tile t = tile_at<PARTS>(g, i);
      int a = n & 1;
      const int64_t row = (int64_t)t.m * kM + rank * kHalfM + q * 32 + lane;
      const int64_t col0 = (int64_t)t.n * kN + half * kHalf;
      const bool row_in = row < g.M;
      float f = 0.f, lse2 = 0.f;
      int64_t target = -1;
      if constexpr (kForward || kGrad) {
        if (row_in) target = p.target[row];
        if constexpr (kGrad) {
          if (row_in) {
            f = row_factor(p, row, target);
            lse2 = p.lse[row] * kLog2e;
            if (p.row_loss) target_dl[warp - 2][lane] = f != 0.f ? f * expm1f(-p.row_loss[row]) : 0.f;
          }
        }
      }
      float chained[kChained ? kHalf : 1];  // the sums of the chains before the last (COPIED: of all)
      if constexpr (kChained) {
        const int chains = (t.kb1 - t.kb0 + kBlocks - 1) / kBlocks, early = COPIED ? chains : chains - 1;
#pragma unroll
        for (int j = 0; j < kHalf; ++j) chained[j] = 0.f;
#pragma unroll 1
        for (int k = 0; k < early; ++k, ++n) {
          a = n & 1;
          if (!dead) dead = !mbar_wait(&accf_bar[a], (n >> 1) & 1, kErrWaitEpilogue, &abort_flag);
          tc_fence_after();
          if (!dead) {
            const uint32_t base = tmem + ((uint32_t)(q * 32) << 16) + a * kN + half * kHalf;
#pragma unroll
            for (int c = 0; c < kHalf; c += 8) {
              float v[8];
              tmem_ld8(base + c, v);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 8; ++j) chained[c + j] += v[j];
            }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive_in_first_cta(freed[a]);
        }
        if constexpr (COPIED) --n;
        a = n & 1;
      }
      if constexpr (!COPIED) {
        if (!dead) dead = !mbar_wait(&accf_bar[a], (n >> 1) & 1, kErrWaitEpilogue, &abort_flag);
        tc_fence_after();
      }
      if (!dead) {
        const uint32_t base = tmem + ((uint32_t)(q * 32) << 16) + a * kN + half * kHalf;
        float m2 = -INFINITY, sum = 0.f;
        const int there = (int)max((int64_t)0, min((int64_t)kHalf, g.N - col0));  // columns that are there
        const int64_t t_col = target - g.col0 - col0;
        const int mine = row_in && t_col >= 0 && t_col < there ? (int)t_col : -1;  // the target's column
        constexpr int kStep = kChained ? 16 : 32;  // columns at a time (registers)
#pragma unroll (kChained ? kHalf / kStep : 1)
        for (int c = 0; c < kHalf; c += kStep) {
          float v[kStep];
          if constexpr (COPIED) {
#pragma unroll
            for (int j = 0; j < kStep; ++j) v[j] = chained[c + j];
          } else if constexpr (kChained) {
            tmem_ld16(base + c, v);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < kStep; ++j) v[j] += chained[c + j];
          } else {
            tmem_ld32(base + c, v);
            tmem_ld_wait();
          }
          if constexpr (kForward) {
            if (mine >= c && mine < c + kStep) {  // the target's logit leaves the others' sum
              p.tgt[row] = pick(v, mine - c);
#pragma unroll
              for (int j = 0; j < kStep; ++j)
                if (j == mine - c) v[j] = -INFINITY;
            }
            const int left = there - c;
            float mx = -INFINITY;
            if (left >= kStep) {
#pragma unroll
              for (int j = 0; j < kStep; ++j) mx = max_nan(mx, v[j]);
            } else {
#pragma unroll
              for (int j = 0; j < kStep; ++j) {
                if (j >= left) v[j] = -INFINITY;
                mx = max_nan(mx, v[j]);
              }
            }
            const float m_new = max_nan(m2, mx * kLog2e);
            if (m_new != -INFINITY) {  // (a NaN goes into the sum)
              float s0 = 0.f, s1 = 0.f;
#pragma unroll
              for (int j = 0; j < kStep; j += 2) {
                s0 += ex2(fmaf(v[j], kLog2e, -m_new));
                s1 += ex2(fmaf(v[j + 1], kLog2e, -m_new));
              }
              sum = fmaf(sum, ex2(m2 - m_new), s0 + s1);
              m2 = m_new;
            }
          } else if constexpr (MODE == kTcAdd) {
            if (row_in) add_columns(g, v, row, col0 + c, t.z, factor);
          } else if constexpr (COPIED) {
            logits_gradient(v, f, lse2, mine - c, p.row_loss ? &target_dl[warp - 2][lane] : nullptr);
#pragma unroll
            for (int j = 0; j < kStep; ++j) chained[c + j] = v[j];
            // 64 columns at a time, part by part, through the staged tile (fp32, 1021 x 256 x 4999: 102 us for the
            // backward, where 16-byte stores from each row's thread take 114)
            if ((c + kStep) % 64 == 0) {
              uint8_t* tile = smem + kStages * kStageBytes + (warp - 2) * kStageOut;
              const int from = c + kStep - 64;
              float2 pr[32];
#pragma unroll
              for (int j = 0; j < 32; ++j) pr[j] = make_float2(chained[from + 2 * j], chained[from + 2 * j + 1]);
#pragma unroll
              for (int k = 0; k < PARTS; ++k) {
                if (lane == 0) bulk_wait_group_read<0>();
                __syncwarp();
#pragma unroll
                for (int j = 0; j < 8; ++j)
                  *reinterpret_cast<uint4*>(tile + lane * 128 + ((j ^ (lane & 7)) << 4)) =
                      make_uint4(take_part(pr[4 * j]), take_part(pr[4 * j + 1]), take_part(pr[4 * j + 2]), take_part(pr[4 * j + 3]));
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                  tma_store_3d(&omap, tile, (int)(col0 + from), t.m * kM + rank * kHalfM + q * 32, k);
                  bulk_commit_group();
                }
              }
            }
          } else {
            // bf16: 64 columns at a time through the warp's staged tile and a TMA store, which
            // leaves out what lies beyond the matrix
            uint8_t* tile = smem + kStages * kStageBytes + (warp - 2) * kStageOut;
            if (c % 64 == 0) {
              if (lane == 0) bulk_wait_group_read<0>();
              __syncwarp();
            }
            if constexpr (kGrad) {
              logits_gradient(v, f, lse2, mine - c, p.row_loss ? &target_dl[warp - 2][lane] : nullptr);
            } else {
#pragma unroll
              for (int j = 0; j < kStep; ++j) v[j] *= factor;
            }
            stage_columns(tile, lane, c % 64, v);
            if ((c + kStep) % 64 == 0) {
              fence_proxy_async_smem();
              __syncwarp();
              if (lane == 0) {
                tma_store_2d(&omap, tile, (int)(col0 + c + kStep - 64), t.m * kM + rank * kHalfM + q * 32);
                bulk_commit_group();
              }
            }
          }
        }
        if constexpr (kForward) {
          if (row_in) p.part[((int64_t)t.n * 2 + half) * g.M + row] = make_float2(m2, sum);
        }
      }
      if constexpr (!COPIED) {  // (COPIED has given its accumulators back one by one)
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_in_first_cta(freed[a]);
      }
    }
    if constexpr (kGrad || MODE == kTcStore) {
      if (lane == 0) bulk_wait_group_read<0>();  // (shared memory may go once it has been read)
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // neither CTA leaves while the other may still use its shared memory
  if (warp == 1) tmem_dealloc_pair(tmem, 512);
}

// A row-major [rows][cols] bf16 matrix as boxes of 64 columns x box_rows rows, 128-byte swizzle; of a
// copy, its parts one behind the other (0: no copy).
int matrix_map(CUtensorMap* map, int parts, const void* base, int64_t cols, int64_t rows, int64_t ld, int box_rows) {
  const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)parts};
  const cuuint64_t strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)(rows * ld) * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)box_rows, 1};
  return encode_tensor_map_bf16(map, base, parts ? 3 : 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int MODE, bool A_MN, bool B_MN, int PARTS>
int launch(const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& o, TcGemm g, const Problem& p, const char* what) {
  const int64_t mt = (g.M + kM - 1) / kM, nt = (g.N + kN - 1) / kN;
  if (mt * nt * g.z > INT32_MAX) return set_error(DYNCONV_ERR_SHAPE, "%s: too many tiles", what);
  g.m_tiles = (int)mt, g.n_tiles = (int)nt;
  if (g.group > g.m_tiles) g.group = g.m_tiles;
  const int tiles = g.m_tiles * g.n_tiles * g.z, most = sm_count() / 2;
  const int grid = 2 * (tiles < most ? tiles : most);
  cudaError_t e =
      cudaFuncSetAttribute(vl_tc_kernel<MODE, A_MN, B_MN, PARTS>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return cuda_status(e, "cudaFuncSetAttribute(vl_tc)");
  }
  vl_tc_kernel<MODE, A_MN, B_MN, PARTS><<<grid, kTcThreads, kSmem, p.st>>>(a, b, o, g, p);
  DYNCONV_CHECK_LAUNCH(what);
  return DYNCONV_OK;
}

int copy_launch(const Problem& p, const void* src, int64_t rows, int dtype, __nv_bfloat16* copy, bool clean = false) {
  const int64_t pitch = copy_pitch(p.D), most = 16 * (int64_t)sm_count();
  int64_t grid = (rows * (pitch / 8) + 255) / 256;
  if (grid > most) grid = most;
  if (dtype == DYNCONV_DTYPE_F32)
    vl_copy_kernel<<<(unsigned)grid, 256, 0, p.st>>>((const float*)src, rows, p.D, pitch, copy, p, clean);
  else
    vl_copy_kernel<<<(unsigned)grid, 256, 0, p.st>>>((const __nv_bfloat16*)src, rows, p.D, pitch, copy, p, clean);
  DYNCONV_CHECK_LAUNCH("vl_copy_kernel");
  return DYNCONV_OK;
}

// Rows of hidden (a group) that stay in L2 while the vocabulary is swept over them: half of it.
int row_group(int64_t D, int dtype) {
  const int64_t g = ((int64_t)64 << 20) / (kM * (int64_t)copy_bytes(1, D, dtype));
  return g < 1 ? 1 : (int)(g < 4096 ? g : 4096);
}

int blocks_of(int64_t n) { return (int)((n + kKB - 1) / kKB); }

template <int PARTS>
int fwd(const Problem& all, int dtype) {
  constexpr bool COPIED = PARTS > 0;
  const int64_t words = COPIED ? words_at_once(all.D, all.V, dtype) : all.V, ld = COPIED ? copy_pitch(all.D) : all.D;
  const int64_t elem = dtype == DYNCONV_DTYPE_F32 ? 4 : 2;
  int s;
  for (int64_t r0 = 0; r0 < all.N; r0 += kRowsAtOnce) {
    const Problem p = rows_from(all, r0, elem);
    if (COPIED && (s = copy_launch(p, p.hidden, p.N, dtype, p.hidden_copy))) return s;
    CUtensorMap a;
    if ((s = matrix_map(&a, PARTS, COPIED ? p.hidden_copy : p.hidden, p.D, p.N, ld, kHalfM))) return s;
    TcGemm g{};
    g.M = p.N, g.k_blocks = blocks_of(p.D), g.z = 1, g.group = row_group(p.D, dtype);
    for (int64_t v0 = 0; v0 < p.V; v0 += words) {  // (words: all, or a multiple of a tile's)
      const void* w = p.weight;
      g.N = p.V - v0 < words ? p.V - v0 : words, g.col0 = v0;
      if constexpr (COPIED) {
        if (r0 == 0 || words < p.V)
          if ((s = copy_launch(p, (const char*)w + v0 * p.D * elem, g.N, dtype, p.weight_copy))) return s;
        w = p.weight_copy;
      }
      CUtensorMap b;
      if ((s = matrix_map(&b, PARTS, w, p.D, g.N, ld, kHalfB))) return s;
      Problem tiles = p;
      tiles.part += v0 / kHalf * p.N;
      s = COPIED || g.k_blocks <= kChain
              ? launch<kTcForward, false, false, PARTS>(a, b, a, g, tiles, "vl_tc_kernel (forward)")
              : launch<kTcForwardLong, false, false, 0>(a, b, a, g, tiles, "vl_tc_kernel (forward)");
      if (s) return s;
    }
    if ((s = merge_launch(p, (p.V + kN - 1) / kN * 2))) return s;
  }
  return total_launch(all);
}

template <int PARTS>
int bwd(const Problem& p, const Plan& pl, int dtype) {
  constexpr bool COPIED = PARTS > 0;
  const int64_t ld = COPIED ? copy_pitch(p.D) : p.D, elem = dtype == DYNCONV_DTYPE_F32 ? 4 : 2;
  // shares of an inner dimension: each has a block, or a chain, at least
  const auto shares = [](int z, int blocks) {
    const int most = COPIED ? (blocks + kCopyChain - 1) / kCopyChain : blocks;
    return z < most ? z : most;
  };
  const auto vec = [&](const void* q) { return COPIED && p.D % 4 == 0 && (reinterpret_cast<uintptr_t>(q) & 15) == 0; };
  // the products' sums are the result itself (fp32, or bf16 rows of whole 16 bytes)
  const bool direct = !COPIED || dtype == DYNCONV_DTYPE_F32;
  int s;
  // The weight's gradient takes hidden without the rows that do not count; so do the logits then, as
  // one tensor stays in L2 better than two.  (bf16 in place: 8.13 ms of backward under sustained load where
  // hidden itself took 8.07 at 16384 x 2048 x 50001; 28.3 against 26.6 us at 32 x 512 x 2000.)
  const void* hidden = p.hidden;
  if (COPIED || p.dweight) {
    if ((s = copy_launch(p, hidden, p.N, dtype, p.hidden_copy, true))) return s;
    hidden = p.hidden_copy;
  }
  CUtensorMap hk, hm;
  if ((s = matrix_map(&hk, PARTS, hidden, p.D, p.N, ld, kHalfM))) return s;
  if ((s = matrix_map(&hm, PARTS, hidden, p.D, p.N, ld, 64))) return s;
  for (int64_t v0 = 0; v0 < p.V; v0 += pl.piece) {
    const int64_t vp = p.V - v0 < pl.piece ? p.V - v0 : pl.piece;
    const void* w = (const char*)p.weight + v0 * p.D * elem;
    if constexpr (COPIED) {
      if ((s = copy_launch(p, w, vp, dtype, p.weight_copy))) return s;
      w = p.weight_copy;
    }
    // maps of exactly this piece: what lies beyond it reads as zero
    CUtensorMap wk, wm, pk, pm, po;
    if ((s = matrix_map(&wk, PARTS, w, p.D, vp, ld, kHalfB))) return s;
    if ((s = matrix_map(&wm, PARTS, w, p.D, vp, ld, 64))) return s;
    if ((s = matrix_map(&pk, PARTS, p.piece, vp, p.N, pl.pitch, kHalfM))) return s;
    if ((s = matrix_map(&pm, PARTS, p.piece, vp, p.N, pl.pitch, 64))) return s;
    if ((s = matrix_map(&po, PARTS, p.piece, vp, p.N, pl.pitch, 32))) return s;
    TcGemm g{};
    g.M = p.N, g.N = vp, g.k_blocks = blocks_of(p.D), g.z = 1, g.group = row_group(p.D, dtype);
    g.col0 = v0;
    s = COPIED || g.k_blocks <= kChain
            ? launch<kTcGrad, false, false, PARTS>(hk, wk, po, g, p, "vl_tc_kernel (logits' gradient)")
            : launch<kTcGradLong, false, false, 0>(hk, wk, po, g, p, "vl_tc_kernel (logits' gradient)");
    if (s) return s;
    if (p.dweight) {
      void* dw = (char*)p.dweight + v0 * p.D * elem;
      const bool finish = pl.z_w > 1 || !direct;
      TcGemm gw{};
      gw.M = vp, gw.N = p.D, gw.k_blocks = blocks_of(p.N), gw.group = 1, gw.out_ld = ld;
      gw.z = shares(pl.z_w, gw.k_blocks);
      gw.out = p.acc_w;
      if (!COPIED && !finish) {
        CUtensorMap wo;
        if ((s = matrix_map(&wo, 0, dw, p.D, vp, p.D, 32))) return s;
        if ((s = launch<kTcStore, true, true, 0>(pm, hm, wo, gw, p, "vl_tc_kernel (weight gradient)"))) return s;
      } else {
        if (!finish) gw.result = dw, gw.vec = vec(dw);
        if ((s = launch<kTcAdd, true, true, PARTS>(pm, hm, pm, gw, p, "vl_tc_kernel (weight gradient)"))) return s;
        if (finish && (s = finish_launch(p, p.acc_w, gw.z, vp, ld, dw, dtype))) return s;
      }
    }
    if (p.dhidden) {
      TcGemm gh{};
      gh.M = p.N, gh.N = p.D, gh.k_blocks = blocks_of(vp), gh.group = 1;
      gh.z = shares(pl.z_h, gh.k_blocks);  // the first piece fills every share; a short last one may not
      gh.out = p.acc_h, gh.out_ld = ld, gh.add = v0 > 0;
      gh.result = direct && pl.z_h == 1 && v0 + vp == p.V ? p.dhidden : nullptr;
      gh.vec = vec(gh.result);
      if ((s = launch<kTcAdd, false, true, PARTS>(pk, wm, pk, gh, p, "vl_tc_kernel (hidden gradient)"))) return s;
    }
  }
  if (!p.dhidden || (direct && pl.z_h == 1)) return DYNCONV_OK;
  return finish_launch(p, p.acc_h, pl.z_h, p.N, ld, p.dhidden, dtype);
}

}  // namespace

int forward(const Problem& p, int dtype) {
  if (!copied(p.D, dtype)) return fwd<0>(p, dtype);
  return parts_of(dtype) == 3 ? fwd<3>(p, dtype) : fwd<1>(p, dtype);
}

int backward(const Problem& p, const Plan& pl, int dtype) {
  if (!copied(p.D, dtype)) return bwd<0>(p, pl, dtype);
  return parts_of(dtype) == 3 ? bwd<3>(p, pl, dtype) : bwd<1>(p, pl, dtype);
}

}  // namespace vl

DYNCONV_DEFINE_ERROR_ACCESSOR(vl_tc_error_word)

}  // namespace dynconv
