// vocab_loss.cu -- the vocabulary loss on the CUDA cores: tiled fp32 products for bf16 tensors that
// TMA cannot address (a width that is no multiple of 8, a base off 16 bytes), the kernels that
// merge the forward's tiles and join partial sums, and the cut of both paths' work.  The
// formulas stand in vocab_loss.cuh.
//
// What bounds the products: the fp32 units, and tiles that do not divide the SMs.  1021 tokens x 257
// channels over 4999 words in bf16 (B200): 93 and 97 us for the two logits' products (320 tiles
// of 128 x 128, 296 at a time), 100 and 120 us for the gradients: 22 to 28 TFLOP/s where the units
// could do 72.
#include "vocab_loss.cuh"

namespace dynconv {
namespace vl {

namespace {

constexpr int kK = 8;       // inner steps staged at once (16 take more registers and 5% longer)
constexpr int kThreads = 256;
using T = __nv_bfloat16;

enum Mode { kForward, kGrad, kAccumulate, kStore };

// out(m, n) = sum_k A[m*am + k*ak] * B[n*bn + k*bk] over one CTA's tile and its share
// blockIdx.z of the inner dimension, fp32 throughout.
struct Gemm {
  const void *A, *B;
  int64_t am, ak, bn, bk;
  int64_t M, N, K, k_share;
  int64_t col0;       // kForward, kGrad: first vocabulary column of the product
  void* out;          // kGrad: piece buffer, kStore: tensor, kAccumulate: fp32 [z][M][N]
  int64_t out_ld;
  int add;            // kAccumulate: add to what is there
};

// One thread's share of TILE rows x kK inner steps: fetched into registers while the stage
// before is multiplied, then put down transposed, [k][row].  Threads follow the dense
// dimension, so that loads coalesce either way.
template <int TILE>
struct Stage {
  static constexpr int kPer = TILE * kK / kThreads;
  const T* at;        // this thread's first element of the current step
  int64_t next, step; // to its next element, to the next step's
  uint32_t rows;      // which of its elements lie in rows that are there
  int k, dk, to, dto; // its first inner index and place in shared memory, and how they go on
  float v[kPer];
  __device__ __forceinline__ Stage(const T* src, int64_t rs, int64_t ks, int64_t r0, int64_t n_rows, int64_t k0) {
    const int t = threadIdx.x;
    const bool k_dense = ks == 1;
    const int r = k_dense ? t / kK : t % TILE, dr = k_dense ? kThreads / kK : 0;
    k = k_dense ? t % kK : t / TILE;
    dk = k_dense ? 0 : kThreads / TILE;
    to = k * (TILE + 4) + r;
    dto = dk * (TILE + 4) + dr;
    at = src + (r0 + r) * rs + (k0 + k) * ks;
    next = dr * rs + dk * ks;
    step = kK * ks;
    rows = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) rows |= (uint32_t)(r0 + r + i * dr < n_rows) << i;
  }
  __device__ __forceinline__ void fetch(int k_left) {  // k_left: inner elements from this step on
    const T* q = at;
#pragma unroll
    for (int i = 0; i < kPer; ++i, q += next)
      v[i] = (rows >> i & 1) && k + i * dk < k_left ? Elem<T>::to_f(*q) : 0.f;
    at += step;
  }
  __device__ __forceinline__ void put(float* s) const {
#pragma unroll
    for (int i = 0; i < kPer; ++i) s[to + i * dto] = v[i];
  }
};

// R x R outputs per thread in groups of four rows and columns, products in packed pairs.
// R = 8: 128 x 128 tiles, 4 bytes of shared memory read for each two multiply-adds; R = 4: 64 x 64
// tiles, for few rows or too few tiles.
template <int MODE, int R>
__global__ void __launch_bounds__(kThreads, 2) vl_gemm_kernel(const Gemm g, const Problem p) {
  constexpr int TILE = 16 * R, LD = TILE + 4, Q = R / 4;
  __shared__ __align__(16) float as[2][kK * LD], bs[2][kK * LD];
  const int64_t m0 = (int64_t)blockIdx.x * TILE, n0 = (int64_t)blockIdx.y * TILE;
  const int64_t k_begin = blockIdx.z * g.k_share, k_end = min(g.K, k_begin + g.k_share);
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
  float2 acc2[R][R / 2] = {};
  Stage<TILE> a_next((const T*)g.A, g.am, g.ak, m0, g.M, k_begin), b_next((const T*)g.B, g.bn, g.bk, n0, g.N, k_begin);
  int left = (int)(k_end - k_begin), buf = 0;  // (a share beyond the end has none)
  a_next.fetch(left);
  b_next.fetch(left);
  for (; left > 0; left -= kK, buf ^= 1) {
    a_next.put(as[buf]);
    b_next.put(bs[buf]);
    __syncthreads();  // (the other buffer's readers passed the barrier before this one)
    a_next.fetch(left - kK);
    b_next.fetch(left - kK);
#pragma unroll
    for (int k = 0; k < kK; ++k) {
      float4 a[Q], b[Q];
#pragma unroll
      for (int i = 0; i < Q; ++i) {
        a[i] = *reinterpret_cast<const float4*>(as[buf] + k * LD + i * 64 + ty * 4);
        b[i] = *reinterpret_cast<const float4*>(bs[buf] + k * LD + i * 64 + tx * 4);
      }
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const float4 a4 = a[i >> 2];
        const float av = (i & 3) == 0 ? a4.x : (i & 3) == 1 ? a4.y : (i & 3) == 2 ? a4.z : a4.w;
        const float2 aa = make_float2(av, av);
#pragma unroll
        for (int j = 0; j < Q; ++j) {
          acc2[i][2 * j] = fma2(aa, make_float2(b[j].x, b[j].y), acc2[i][2 * j]);
          acc2[i][2 * j + 1] = fma2(aa, make_float2(b[j].z, b[j].w), acc2[i][2 * j + 1]);
        }
      }
    }
  }
  const float factor = MODE == kStore ? result_factor(p) : 1.f;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int64_t m = m0 + (i >> 2) * 64 + ty * 4 + (i & 3);
    const bool row = m < g.M;
    float acc[R];
    int64_t col[R];
#pragma unroll
    for (int j = 0; j < R; ++j) {
      acc[j] = j & 1 ? acc2[i][j >> 1].y : acc2[i][j >> 1].x;
      col[j] = n0 + (j >> 2) * 64 + tx * 4 + (j & 3);
    }
    if constexpr (MODE == kForward) {
      // 16 threads (one half warp) share a row: its maximum, then its sum of exponentials
      const int64_t t = row ? p.target[m] : -1;
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < R; ++j) {
        if (col[j] < g.N) mx = fmaxf(mx, acc[j]);
        if (row && col[j] < g.N && col[j] == t) p.tgt[m] = acc[j];
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      mx *= kLog2e;
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < R; ++j)
        if (col[j] < g.N) sum += exp2f(fmaf(acc[j], kLog2e, -mx));
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (row && tx == 0) p.part[(int64_t)blockIdx.y * p.N + m] = make_float2(mx, sum);
    } else if constexpr (MODE == kGrad) {
      if (!row) continue;
      const int64_t t = p.target[m];
      const float f = row_factor(p, m, t), lse = p.lse[m];
#pragma unroll
      for (int j = 0; j < R; ++j) {
        if (col[j] >= g.N) continue;
        const float pr = expf(acc[j] - lse) - (g.col0 + col[j] == t ? 1.f : 0.f);
        ((T*)g.out)[m * g.out_ld + col[j]] = Elem<T>::from_f(f == 0.f ? 0.f : pr * f);
      }
    } else {
      if (!row) continue;
#pragma unroll
      for (int j = 0; j < R; ++j) {
        if (col[j] >= g.N) continue;
        if constexpr (MODE == kAccumulate) {
          float* o = (float*)g.out + ((int64_t)blockIdx.z * g.M + m) * g.out_ld + col[j];
          *o = g.add ? *o + acc[j] : acc[j];
        } else {
          ((T*)g.out)[m * g.out_ld + col[j]] = Elem<T>::from_f(acc[j] * factor);
        }
      }
    }
  }
}

// 128 x 128 tiles where both sides fill them and there are enough for the SMs.
bool large_tiles(int64_t M, int64_t N, int64_t z) {
  return M >= 96 && N >= 96 && ((M + 127) / 128) * ((N + 127) / 128) * z >= sm_count() / 2;
}

template <int MODE, int R>
int gemm_tiles(const Gemm& g, const Problem& p, int z, const char* what) {
  constexpr int TILE = 16 * R;
  const int64_t gx = (g.M + TILE - 1) / TILE, gy = (g.N + TILE - 1) / TILE;
  if (gx > INT32_MAX || gy > 65535) return set_error(DYNCONV_ERR_SHAPE, "%s: too many tiles", what);
  vl_gemm_kernel<MODE, R><<<dim3((unsigned)gx, (unsigned)gy, (unsigned)z), kThreads, 0, p.st>>>(g, p);
  DYNCONV_CHECK_LAUNCH(what);
  return DYNCONV_OK;
}

template <int MODE>
int gemm(Gemm g, const Problem& p, int z, const char* what) {
  g.k_share = ((g.K + z - 1) / z + kK - 1) / kK * kK;
  return large_tiles(g.M, g.N, z) ? gemm_tiles<MODE, 8>(g, p, z, what) : gemm_tiles<MODE, 4>(g, p, z, what);
}

// Merges the tiles' (maximum, sum) of 32 rows per CTA: lane = row, warps take every eighth
// tile; then the rows' losses.
__global__ void __launch_bounds__(256) vl_merge_kernel(const Problem p, int64_t tiles) {
  __shared__ float2 part[8][32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t n = (int64_t)blockIdx.x * 32 + lane;
  float mx = -INFINITY, sum = 0.f;
  if (n < p.N) {
    for (int64_t i = w; i < tiles; i += 8) {
      const float2 v = p.part[i * p.N + n];
      const float m2 = fmaxf(mx, v.x);
      if (m2 == -INFINITY) continue;  // nothing finite so far: exp(-inf) adds nothing
      sum = sum * exp2f(mx - m2) + v.y * exp2f(v.x - m2);
      mx = m2;
    }
  }
  part[w][lane] = make_float2(mx, sum);
  __syncthreads();
  if (w != 0 || n >= p.N) return;
  for (int i = 1; i < 8; ++i) {
    const float2 v = part[i][lane];
    const float m2 = fmaxf(mx, v.x);
    if (m2 == -INFINITY) continue;
    sum = sum * exp2f(mx - m2) + v.y * exp2f(v.x - m2);
    mx = m2;
  }
  const float lse = (float)(((double)mx + (double)log2f(sum)) * 0.6931471805599453);
  p.lse[n] = lse;
  const int64_t t = p.target[n];
  // an ignored row adds nothing; a target outside the vocabulary makes the loss NaN
  float row = 0.f;
  if (t != p.ignore) row = (t >= 0 && t < p.V) ? lse - p.tgt[n] : __int_as_float(0x7fc00000);
  if (p.reduction == kNone)
    p.loss[n] = row;
  else
    p.tgt[n] = row;
}

// Sums the rows' losses in a fixed order (one CTA) and counts the rows that take part.
__global__ void __launch_bounds__(1024) vl_total_kernel(const Problem p) {
  __shared__ double ssum[32];
  __shared__ long long scnt[32];
  double sum = 0.0;
  long long cnt = 0;
  for (int64_t n = threadIdx.x; n < p.N; n += 1024) {
    if (p.reduction != kNone) sum += (double)p.tgt[n];
    cnt += p.target[n] != p.ignore;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    cnt += __shfl_xor_sync(0xffffffffu, cnt, o);
  }
  if ((threadIdx.x & 31) == 0) {
    ssum[threadIdx.x >> 5] = sum;
    scnt[threadIdx.x >> 5] = cnt;
  }
  __syncthreads();
  if (threadIdx.x != 0) return;
  sum = 0.0;
  cnt = 0;
  for (int i = 0; i < 32; ++i) {
    sum += ssum[i];
    cnt += scnt[i];
  }
  p.stats[0] = (float)sum;
  p.stats[1] = (float)cnt;
  if (p.reduction == kSum) p.loss[0] = (float)sum;
  if (p.reduction == kMean) p.loss[0] = (float)(sum / (double)cnt);  // no row left: 0/0, NaN
}

template <typename Out>
__global__ void __launch_bounds__(256) vl_finish_kernel(const Problem p, const float* __restrict__ parts, int n_parts,
                                                        int64_t n, Out* __restrict__ out) {
  const float f = result_factor(p);
  const int64_t step = (int64_t)gridDim.x * blockDim.x;
  int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (n % 4 == 0) {  // (the parts are 256-byte aligned; the output's rows may start anywhere)
    for (; i < n / 4; i += step) {
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (int z = 0; z < n_parts; ++z) {
        const float4 v = __ldg(reinterpret_cast<const float4*>(parts + z * n) + i);
        a.x += v.x, a.y += v.y, a.z += v.z, a.w += v.w;
      }
      const float r[4] = {a.x * f, a.y * f, a.z * f, a.w * f};
      store_span(out + 4 * i, r);
    }
    return;
  }
  for (; i < n; i += step) {
    float a = 0.f;
    for (int z = 0; z < n_parts; ++z) a += __ldg(parts + z * n + i);
    out[i] = Elem<Out>::from_f(a * f);
  }
}

}  // namespace

int finish_launch(const Problem& p, const float* parts, int n_parts, int64_t n, void* out, int dtype) {
  if (n <= 0) return DYNCONV_OK;
  int64_t grid = (n / 4 + 255) / 256 + 1;
  if (grid > 16 * (int64_t)sm_count()) grid = 16 * (int64_t)sm_count();
  if (dtype == DYNCONV_DTYPE_BF16)
    vl_finish_kernel<<<(unsigned)grid, 256, 0, p.st>>>(p, parts, n_parts, n, (__nv_bfloat16*)out);
  else
    vl_finish_kernel<<<(unsigned)grid, 256, 0, p.st>>>(p, parts, n_parts, n, (float*)out);
  DYNCONV_CHECK_LAUNCH("vl_finish_kernel");
  return DYNCONV_OK;
}

int merge_launch(const Problem& p, int64_t tiles) {
  vl_merge_kernel<<<(unsigned)((p.N + 31) / 32), 256, 0, p.st>>>(p, tiles);
  DYNCONV_CHECK_LAUNCH("vl_merge_kernel");
  return DYNCONV_OK;
}

int total_launch(const Problem& p) {
  vl_total_kernel<<<1, 1024, 0, p.st>>>(p);
  DYNCONV_CHECK_LAUNCH("vl_total_kernel");
  return DYNCONV_OK;
}

// The piece's width is the one with the lowest estimated time among those whose buffer stays
// within 512 MB: each product runs in rounds of one tile per SM or SM pair (weight-gradient tiles
// are few and long: at 16384 x 2048 a width of 7168 columns makes 224 of them, three rounds of 74
// and two tiles), each piece costs three launches and one pass over the fp32 sums of dhidden.  Times are
// counted in blocks of 64 inner elements of a tile, 0.46 us each on the tensor cores; an fp32
// tensor's parts make six products of each block.
// Where a product has few tiles its inner dimension is spread over several CTAs, each share at
// least 512 elements (one chain of 256 for fp32 tensors; 128 on the CUDA cores, where they take as
// long).
// The cut rests on sizes and type alone, so that a workspace asked for by size fits every call of
// that size: tensors whose alignment keeps them from the tensor cores are cut the same way.
Plan plan(int64_t N, int64_t D, int64_t V, int dtype) {
  const bool split = dtype == DYNCONV_DTYPE_F32, tc = split || D % 8 == 0;
  const int64_t elem = split ? 2 * kSplitParts : 2, sms = tc ? sm_count() / 2 : sm_count();
  const int64_t tm = tc ? 256 : 128, tn = tc ? 256 : 128;
  const auto up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
  const int64_t least = split ? 64 * kSplitChain : tc ? 512 : 128;
  const auto share = [&](int64_t tiles, int64_t inner) {
    int64_t z = 2 * sms / tiles;
    if (z > inner / least) z = inner / least;
    if (z > 16) z = 16;
    return (int)(z < 1 ? 1 : z);
  };
  // blocks of a tile's inner dimension that one of z shares has
  const auto inner = [&](int64_t n, int z) {
    return split ? up(up(n, 64 * kSplitChain), z) * kSplitChain * kSplitProducts : up(up(n, 64), z);
  };
  const double launch = 10, sums = 0.5 * (double)(N * D) * 8 / 6.5e12 / 0.46e-6;
  const int64_t n_tiles = up(N, tm), d_tiles = up(D, tn);
  const auto cost = [&](int64_t cols, int z_h, int z_w) {
    const double logits = (double)(up(n_tiles * up(cols, tn), sms) * inner(D, 1));
    const double dw = (double)(up(up(cols, tm) * d_tiles * z_w, sms) * inner(N, z_w));
    const double dh = (double)(up(n_tiles * d_tiles * z_h, sms) * inner(cols, z_h));
    return logits + dw + dh + (split ? 4 : 3) * launch + sums * z_h;
  };
  int64_t most = ((int64_t)512 << 20) / (elem * (N > 0 ? N : 1)) / 256 * 256;
  if (most < 1024) most = 1024;
  if (split && most > words_at_once(D, V)) most = words_at_once(D, V);
  Plan best{};
  double best_cost = 1e300;
  const int64_t step = up(up(V, 32), 256) * 256;  // at most about 32 candidates (0.4 us of host time each)
  for (int64_t cols = most < V ? most : up(V, 256) * 256; cols > 0; cols -= step) {
    const int64_t full = V / cols, rest = V - full * cols;
    const int z_h = share(n_tiles * d_tiles, cols < V ? cols : V), z_w = share(up(cols < V ? cols : V, tm) * d_tiles, N);
    const double c = (double)full * cost(cols, z_h, z_w) + (rest ? cost(rest, z_h, z_w) : 0.0);
    if (c < best_cost) {
      best_cost = c;
      best.piece = cols < V ? cols : V;
      best.z_h = z_h, best.z_w = z_w;
    }
    if (up(V, cols) > 64) break;
  }
  best.pitch = up(best.piece, 64) * 64;
  return best;
}

int simple_fwd(const Problem& all) {
  int s;
  for (int64_t r0 = 0; r0 < all.N; r0 += kRowsAtOnce) {
    const Problem p = rows_from(all, r0, sizeof(T));
    Gemm g{};
    g.A = p.hidden, g.am = p.D, g.ak = 1;
    g.B = p.weight, g.bn = p.D, g.bk = 1;
    g.M = p.N, g.N = p.V, g.K = p.D;
    if ((s = gemm<kForward>(g, p, 1, "vl_gemm_kernel (forward)"))) return s;
    const int64_t tile = large_tiles(p.N, p.V, 1) ? 128 : 64;
    if ((s = merge_launch(p, (p.V + tile - 1) / tile))) return s;
  }
  return total_launch(all);
}

int simple_bwd(const Problem& p, const Plan& pl) {
  int s;
  for (int64_t v0 = 0; v0 < p.V; v0 += pl.piece) {
    const int64_t vp = p.V - v0 < pl.piece ? p.V - v0 : pl.piece;
    const T* w = (const T*)p.weight + v0 * p.D;
    Gemm g{};
    g.A = p.hidden, g.am = p.D, g.ak = 1;
    g.B = w, g.bn = p.D, g.bk = 1;
    g.M = p.N, g.N = vp, g.K = p.D, g.col0 = v0;
    g.out = p.piece, g.out_ld = pl.pitch;
    if ((s = gemm<kGrad>(g, p, 1, "vl_gemm_kernel (logits' gradient)"))) return s;
    if (p.dweight) {
      Gemm gw{};
      gw.A = p.piece, gw.am = 1, gw.ak = pl.pitch;
      gw.B = p.hidden, gw.bn = 1, gw.bk = p.D;
      gw.M = vp, gw.N = p.D, gw.K = p.N;
      gw.out_ld = p.D;
      if (pl.z_w == 1) {
        gw.out = (T*)p.dweight + v0 * p.D;
        if ((s = gemm<kStore>(gw, p, 1, "vl_gemm_kernel (weight gradient)"))) return s;
      } else {
        gw.out = p.acc_w;
        if ((s = gemm<kAccumulate>(gw, p, pl.z_w, "vl_gemm_kernel (weight gradient)"))) return s;
        if ((s = finish_launch(p, p.acc_w, pl.z_w, vp * p.D, (T*)p.dweight + v0 * p.D, DYNCONV_DTYPE_BF16))) return s;
      }
    }
    if (p.dhidden) {
      Gemm gh{};
      gh.A = p.piece, gh.am = pl.pitch, gh.ak = 1;
      gh.B = w, gh.bn = 1, gh.bk = p.D;
      gh.M = p.N, gh.N = p.D, gh.K = vp;
      gh.out = p.acc_h, gh.out_ld = p.D, gh.add = v0 > 0;
      if ((s = gemm<kAccumulate>(gh, p, pl.z_h, "vl_gemm_kernel (hidden gradient)"))) return s;
    }
  }
  return p.dhidden ? finish_launch(p, p.acc_h, pl.z_h, p.N * p.D, p.dhidden, DYNCONV_DTYPE_BF16) : DYNCONV_OK;
}

}  // namespace vl
}  // namespace dynconv
