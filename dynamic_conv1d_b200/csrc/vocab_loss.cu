// vocab_loss.cu -- what surrounds the vocabulary loss's products (vocab_loss_tc.cu): the merge of the
// forward's tiles, the join of partial sums, and how the backward is cut.  The formulas stand in
// vocab_loss.cuh.
#include "vocab_loss.cuh"

namespace dynconv {
namespace vl {

namespace {

// Adds a tile's (maximum, sum) to a row's.
__device__ __forceinline__ void merge(float& mx, float& sum, float2 v) {
  const float m2 = max_nan(mx, v.x);
  if (m2 == -INFINITY) return;  // only words of minus infinity so far: exp(-inf) adds nothing
  sum = sum * exp2f(mx - m2) + v.y * exp2f(v.x - m2);
  mx = m2;
}

// Merges the tiles' (maximum, sum) of 32 rows per CTA: lane = row, warps take every eighth
// tile; then the rows' losses.
__global__ void __launch_bounds__(256) vl_merge_kernel(const Problem p, int64_t tiles) {
  __shared__ float2 part[8][32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t n = (int64_t)blockIdx.x * 32 + lane;
  float mx = -INFINITY, sum = 0.f;
  if (n < p.N) {
    constexpr int kFly = 4;  // tiles under way before the first is used
    for (int64_t i = w; i < tiles; i += 8 * kFly) {
      float2 v[kFly];
#pragma unroll
      for (int k = 0; k < kFly; ++k) v[k] = i + 8 * k < tiles ? p.part[(i + 8 * k) * p.N + n] : make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int k = 0; k < kFly; ++k) merge(mx, sum, v[k]);
    }
  }
  part[w][lane] = make_float2(mx, sum);
  __syncthreads();
  if (w != 0 || n >= p.N) return;
  for (int i = 1; i < 8; ++i) merge(mx, sum, part[i][lane]);
  const double others = ((double)mx + (double)log2f(sum)) / (double)kLog2e;  // (the constant that scaled them)
  const int64_t t = p.target[n];
  const bool word = t >= 0 && t < p.V;
  // an ignored row adds nothing; a target outside the vocabulary makes the loss NaN
  const float nan = __int_as_float(0x7fc00000);
  float row = nan;
  float lse = (float)others;
  if (word) {
    const float tgt = p.tgt[n];
    const double l = tgt == INFINITY ? (double)nan : (double)tgt;  // (inf - inf: no softmax)
    const double d = others - l, top = d > 0.0 ? others : l, rest = (double)log1pf(expf((float)-fabs(d)));
    row = (float)((top - l) + rest);
    lse = (float)(top + rest);
  }
  p.lse[n] = lse;
  if (p.row_loss) p.row_loss[n] = row;
  if (t == p.ignore) row = 0.f;
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

// Rows of ld = a multiple of 8 floats, of which D are there.  (The parts are 256-byte aligned; the
// output's rows may start anywhere.)
template <typename Out>
__global__ void __launch_bounds__(256) vl_finish_kernel(const Problem p, const float* __restrict__ parts, int n_parts,
                                                        int64_t rows, int64_t ld, Out* __restrict__ out) {
  const float f = result_factor(p);
  const int64_t n = rows * ld, step = (int64_t)gridDim.x * blockDim.x;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n / 4; i += step) {
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int z = 0; z < n_parts; ++z) {
      const float4 v = __ldg(reinterpret_cast<const float4*>(parts + z * n) + i);
      a.x += v.x, a.y += v.y, a.z += v.z, a.w += v.w;
    }
    const float r[4] = {a.x * f, a.y * f, a.z * f, a.w * f};
    if (ld == p.D) {
      store_span(out + 4 * i, r);
    } else {
      const int64_t row = 4 * i / ld, c = 4 * i - row * ld;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c + j < p.D) out[row * p.D + c + j] = Elem<Out>::from_f(r[j]);
    }
  }
}

}  // namespace

int finish_launch(const Problem& p, const float* parts, int n_parts, int64_t rows, int64_t ld, void* out, int dtype) {
  int64_t grid = (rows * ld / 4 + 255) / 256;
  if (grid > 16 * (int64_t)sm_count()) grid = 16 * (int64_t)sm_count();
  if (dtype == DYNCONV_DTYPE_BF16)
    vl_finish_kernel<<<(unsigned)grid, 256, 0, p.st>>>(p, parts, n_parts, rows, ld, (__nv_bfloat16*)out);
  else
    vl_finish_kernel<<<(unsigned)grid, 256, 0, p.st>>>(p, parts, n_parts, rows, ld, (float*)out);
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
// within 512 MB: each product runs in rounds of one tile per SM pair (weight-gradient tiles
// are few and long: at 16384 x 2048 a width of 7168 columns makes 224 of them, three rounds of 74
// and two tiles), each piece costs three launches (four with a copy of its words) and one pass over the
// fp32 sums of dhidden.  Times are counted in blocks of 64 inner elements of a tile, 0.46 us each; an
// fp32 tensor's parts make six products of each block.
// Where a product has few tiles its inner dimension is spread over several CTAs, each share at
// least 512 elements (one chain of 256 of copied operands).
// The cut rests on sizes and type alone, so that a workspace asked for by size fits every call of
// that size.
Plan plan(int64_t N, int64_t D, int64_t V, int dtype) {
  const bool copy = copied(D, dtype);
  const int64_t products = products_of(parts_of(dtype));
  const int64_t elem = 2 * parts_of(dtype), sms = sm_count() / 2, tm = 256, tn = 256;
  const auto up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
  const int64_t least = copy ? 64 * kCopyChain : 512;
  const auto share = [&](int64_t tiles, int64_t inner) {
    int64_t z = 2 * sms / tiles;
    if (z > inner / least) z = inner / least;
    if (z > 16) z = 16;
    return (int)(z < 1 ? 1 : z);
  };
  // blocks of a tile's inner dimension that one of z shares has
  const auto inner = [&](int64_t n, int z) {
    return copy ? up(up(n, 64 * kCopyChain), z) * kCopyChain * products : up(up(n, 64), z);
  };
  const double launch = 10, sums = 0.5 * (double)(N * D) * 8 / 6.5e12 / 0.46e-6;
  const int64_t n_tiles = up(N, tm), d_tiles = up(D, tn);
  const auto cost = [&](int64_t cols, int z_h, int z_w) {
    const double logits = (double)(up(n_tiles * up(cols, tn), sms) * inner(D, 1));
    const double dw = (double)(up(up(cols, tm) * d_tiles * z_w, sms) * inner(N, z_w));
    const double dh = (double)(up(n_tiles * d_tiles * z_h, sms) * inner(cols, z_h));
    return logits + dw + dh + (copy ? 4 : 3) * launch + sums * z_h;
  };
  int64_t most = ((int64_t)512 << 20) / (elem * (N > 0 ? N : 1)) / 256 * 256;
  if (most < 1024) most = 1024;
  if (copy && most > words_at_once(D, V, dtype)) most = words_at_once(D, V, dtype);
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

}  // namespace vl
}  // namespace dynconv
