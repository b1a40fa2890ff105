// norm.cuh -- arguments of the norms (norm.cu); the formulas stand there.
#pragma once

#include "common.cuh"

namespace dynconv {
namespace norm {

constexpr int kMaxWidth = 16384;

// Rows (n, g), n < N and g < G, of D numbers; x and gate with strides, everything else dense.
struct Gated {
  const void *x, *weight, *gate;
  int64_t x_outer, x_inner, gate_outer, gate_inner;
  void* y;
  const void* dy;
  void *dx, *dgate, *dweight;  // (any may be null)
  float* part;                 // [partial_rows()][D], null without dweight
  int64_t N, G;
  int D;
  float eps, scale;
};

struct Residual {
  const void *x, *residual, *weight, *scale;  // scale: one per channel, or null for `factor`
  void *y, *h;
  const void *dy, *dh;  // (backward: h is read; either gradient may be null)
  void *dx, *dresidual, *dweight, *dscale;
  float *part_w, *part_s;
  int64_t N;
  int D;
  float eps, factor;
};

int64_t partial_rows();
// w32: weight and scale, and their gradients, are float32 whatever the rows' type.
int gated_launch(const Gated& p, int dtype, bool w32, bool backward, cudaStream_t st);
int residual_launch(const Residual& p, int dtype, bool w32, bool backward, cudaStream_t st);

}  // namespace norm
}  // namespace dynconv
