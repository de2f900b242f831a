// The elementwise half of a linear layer's backward, for gfx950: du = dy act'(u) and the bias's gradient, the sum of du's rows.
//
// Reference: the autodiff of src/ferrite/model/gpt.py:95-104, whose linear layers have neither bias nor activation of their own. The
// products that follow (du . w^T, x^T . du) are matmul.hip's.
//
// Bound by memory: dy and u are read and du written once. du is rounded to the products' operand type, whose matrix instructions take
// nothing wider at their rate; the bias's sums take it unrounded, in f32 and a fixed order: a thread owns eight columns of every
// eighth row of its workgroup's rows, the workgroup's threads are added through LDS into a partial row, and a second kernel adds the
// partial rows.
#include <algorithm>

#include "common.h"
#include "internal_api.h"
#include "linear.h"
#include "rows.h"

namespace ferrite {
namespace {

constexpr int kUnits = 32, kLanes = 8;  // units of columns and rows under way in a workgroup

// Without u, du is dy and is not written. With one workgroup to a column its sums are the bias's gradient.
template <typename T, int W>
__global__ __launch_bounds__(kUnits* kLanes) void act_grad_kernel(const T* __restrict__ dy, const T* __restrict__ u,
                                                                  T* __restrict__ du, float* __restrict__ part, int64_t rows,
                                                                  int dim, int act, int64_t share, void* db, int db_f32) {
  __shared__ float red[kLanes][kUnits * W + 1];
  const int c = threadIdx.x % kUnits, r = threadIdx.x / kUnits;
  const int unit = (int)blockIdx.x * kUnits + c;
  const int at = column<W>(unit, dim);
  const int64_t first = blockIdx.y * share, end = std::min<int64_t>(rows, first + share);
  float sum[W];
#pragma unroll
  for (int e = 0; e < W; ++e) sum[e] = 0.f;
  constexpr int U = 4;  // rows whose loads go out together
  if (at >= 0)
    for (int64_t row = first + r; row < end; row += kLanes * U) {
      Cols<T, W> g[U], v[U];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int64_t off = std::min<int64_t>(row + k * kLanes, end - 1) * dim + at;
        g[k].load(dy + off);
        if (u) v[k].load(u + off);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int k = 0; k < U; ++k) {
        if (row + k * kLanes >= end) break;
        float x[W], y[W];
        g[k].get(x);
        if (u) {
          v[k].get(y);
#pragma unroll
          for (int e = 0; e < W; ++e) x[e] *= act_slope(y[e], act);
          g[k].set(x);
          g[k].store(du + (row + k * kLanes) * dim + at);
        }
#pragma unroll
        for (int e = 0; e < W; ++e) sum[e] += x[e];
      }
    }
  if (!part && !db) return;
#pragma unroll
  for (int e = 0; e < W; ++e) red[r][c * W + e] = sum[e];
  __syncthreads();
  // Column j of the workgroup is its unit's element j; the last unit of a row may lie over the one before it.
  for (int j = threadIdx.x; j < kUnits * W; j += kUnits * kLanes) {
    const int to = column<W>((int)blockIdx.x * kUnits + j / W, dim);
    if (to < 0 || to + j % W < ((int)blockIdx.x * kUnits + j / W) * W) continue;
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < kLanes; ++k) s += red[k][j];
    if (part)
      part[(int64_t)blockIdx.y * dim + to + j % W] = s;
    else if (db_f32)
      static_cast<float*>(db)[to + j % W] = s;
    else
      static_cast<bf16*>(db)[to + j % W] = (bf16)s;
  }
}

// Rows to a workgroup: about eight workgroups per CU in all, at least 32 rows to one (a load of each thread's four) and at most 512, so
// that no lane adds more than 64 in a line, up to 2^18 rows (512 partial rows). By the first rule alone 65536 x 32768 bf16 had lines of
// 512: 2541 us with GELU and 648 without, now 2484 and 670. 16384 x 2048 bf16 with GELU 44.1 us (4.6 TB/s with the join), with four
// workgroups per CU 52, two 50; with loads of eight rows together 60, of two 47.5 at four and 43.8 at eight.
struct ActPlan {
  int64_t cols, parts, share;
};
ActPlan act_plan(int64_t rows, int64_t dim) {
  ActPlan p{};
  p.cols = cdiv(dim >= 8 ? cdiv(dim, (int64_t)8) : dim, (int64_t)kUnits);
  p.parts = std::clamp<int64_t>(std::max(std::min(2048 / p.cols, cdiv(rows, (int64_t)32)), cdiv(rows, (int64_t)512)), 1, 512);
  p.share = cdiv(cdiv(std::max<int64_t>(rows, 1), p.parts), (int64_t)kLanes) * kLanes;
  p.parts = cdiv(std::max<int64_t>(rows, 1), p.share);
  return p;
}
bool act_ok(int64_t rows, int64_t dim) {
  return rows >= 0 && dim >= 1 && dim <= 0x7fffffff / 64 && rows <= ((int64_t)1 << 58) / dim;
}

}  // namespace
}  // namespace ferrite

extern "C" int64_t ferrite_internal_act_grad_workspace(int64_t rows, int64_t dim) {
  using namespace ferrite;
  if (!act_ok(rows, dim)) return -1;
  const ActPlan p = act_plan(rows, dim);
  return p.parts > 1 ? p.parts * dim * (int64_t)sizeof(float) : 0;
}

extern "C" int ferrite_internal_act_grad(const void* dy, const void* u, void* du, void* db, int64_t rows, int64_t dim, int act,
                                         int dtype, int bias_dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace ferrite;
  if (!valid_dtype(dtype) || (db && !valid_dtype(bias_dtype)) || act < FERRITE_ACT_NONE || act > FERRITE_ACT_SILU)
    return fail(FERRITE_ERR_INVALID_ARGUMENT, "ferrite_linear_bwd: bad dtype or activation");
  if (!act_ok(rows, dim)) return fail(FERRITE_ERR_INVALID_ARGUMENT, "ferrite_linear_bwd: sizes out of range");
  if ((rows && !dy) || (u && rows && !du)) return fail(FERRITE_ERR_INVALID_ARGUMENT, "ferrite_linear_bwd: null pointer");
  const int64_t need = db ? ferrite_internal_act_grad_workspace(rows, dim) : 0;
  if (need && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 3)))
    return fail(FERRITE_ERR_INVALID_ARGUMENT, "ferrite_linear_bwd: workspace too small");
  const ActPlan p = act_plan(rows, dim);
  hipStream_t s = static_cast<hipStream_t>(stream);
  float* part = need ? static_cast<float*>(workspace) : nullptr;
  auto go = [&](auto kernel, auto* t) {
    typedef std::remove_pointer_t<decltype(t)> T;
    hipLaunchKernelGGL(kernel, dim3((unsigned)p.cols, (unsigned)p.parts), dim3(kUnits * kLanes), 0, s,
                       static_cast<const T*>(dy), static_cast<const T*>(u), static_cast<T*>(du), part, rows, (int)dim, act,
                       p.share, need ? nullptr : db, bias_dtype == FERRITE_F32);
  };
  auto typed = [&](auto* t) {
    typedef std::remove_pointer_t<decltype(t)> T;
    if (dim >= 8)
      go(act_grad_kernel<T, 8>, t);
    else
      go(act_grad_kernel<T, 1>, t);
  };
  if (dtype == FERRITE_BF16)
    typed((bf16*)nullptr);
  else
    typed((float*)nullptr);
  if (need) {
    if (bias_dtype == FERRITE_BF16)
      join_parts(part, static_cast<bf16*>(db), (bf16*)nullptr, 1, (int)p.parts, dim, s);
    else
      join_parts(part, static_cast<float*>(db), (float*)nullptr, 1, (int)p.parts, dim, s);
  }
  return check_launch("ferrite_linear_bwd");
}
