// f32 products of any layout and alignment (gemm_f32.hip).
#pragma once

#include "common.h"

namespace ferrite {

// out[M,N] = op(x) . op(y) over f32: x [M,K], or [K,M] when xt; y [K,N], or [N,K] when yt. Rows are dense and may start at any
// element. With slices > 1 slice s leaves its share of K in out + s slab floats.
struct F32Product {
  const float *x, *y;
  float* out;
  int64_t m, n, k;
  bool xt, yt;
  int slices;
  int64_t slab;
};
// Sizes that it takes: at least four along the contiguous dimension of each operand.
bool f32_any_ok(int64_t m, int64_t n, int64_t k, bool xt, bool yt);
// Slices of K for the CUs, and floats from one slab to the next.
int f32_any_slices(int64_t m, int64_t n, int64_t k, int64_t cus);
inline int64_t f32_any_slab(int64_t m, int64_t n) { return cdiv(m * n, (int64_t)4) * 4; }
int f32_any_launch(const F32Product& p, hipStream_t stream);

}  // namespace ferrite
