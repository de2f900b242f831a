// Clipping of gradients by their global norm, for gfx950.
//
// Reference: src/ferrite/model/train.py:59-66 (the norm and the scale of adamw_update, which optim.hip fuses with the update).
// Here they stand alone, for an optimiser of another kind or a step between:
//   norm = sqrt(sum over all tensors of sum(g^2));  g = g min(1, most / (norm + 1e-6))
//
// Bound by memory: one read of the gradients, and where the factor is below 1 another and a write. Two kernels over tiles of all
// tensors at once: partial sums of squares, and the scaling, whose workgroups each add the partial sums (in one order, from L2) instead of
// waiting for a kernel that would. Tensors travel in the kernel arguments, up to kTensors to a launch, in f32 and bf16 alike. The
// squares are added in 64 bits: those of gradients past 2^64 do not overflow, and the order costs no precision.
//
// Gradients of more than 128 MB in all are read past the caches (kStream): 150 MB of bf16 85 us against 96, 600 MB 320 (5.6 TB/s)
// against 376. Smaller ones are still there for the second read: 26 MB 17.8 us cached against 21.5, 104 MB 62 both ways.
// Scaling the last tiles first, those just read, changed nothing.
#include <math.h>

#include <algorithm>

#include "common.h"
#include "internal_api.h"
#include "rows.h"

namespace ferrite {
namespace {

constexpr int kTensors = 128;      // tensors per launch (kernel-argument table)
constexpr int kTile = 256 * 8 * 4; // elements per workgroup and step: four vectors of eight a thread
constexpr int kParts = 1024;       // partial sums in all
constexpr int64_t kStream = 128 << 20;  // bytes of gradients beyond which no cache keeps them for the second read

struct Tensors {
  void* p[kTensors];
  int64_t n[kTensors];
  int64_t tile0[kTensors + 1];  // tiles before each tensor
  uint32_t f32[kTensors / 32];  // bit i: tensor i is f32
  int count;
};
static_assert(sizeof(Tensors) <= 3500, "kernel arguments stay under 4 KB");

// The tensor of tile t: the last that begins at or before it (empty ones begin where the next does).
__device__ __forceinline__ int tensor_of(const Tensors& s, int64_t t) {
  int lo = 0, hi = s.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (s.tile0[mid] <= t)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ double wave_sum64(double x) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) x += __shfl_xor(x, off, kWave);
  return x;
}
// Sum over the workgroup's 256 threads, in all of them.
__device__ __forceinline__ double block_sum64(double x, double* lds) {
  x = wave_sum64(x);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
  __syncthreads();
  return (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

template <bool Past, typename T>
__device__ __forceinline__ void load_tile(Eight<T> (&v)[4], const T* g) {
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    if (Past)
      v[u].load(g + u * 2048 + threadIdx.x * 8);
    else
      v[u].load_cached(g + u * 2048 + threadIdx.x * 8);
  }
}

template <bool Past, typename T>
__device__ __forceinline__ double tile_squares(const T* g, int64_t first, int64_t n) {
  double acc = 0.0;
  if (first + kTile <= n) {
    Eight<T> v[4];
    load_tile<Past>(v, g + first);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      float x[8];
      v[u].get(x);
#pragma unroll
      for (int e = 0; e < 8; ++e) acc += (double)x[e] * (double)x[e];
    }
  } else {
    for (int64_t i = first + threadIdx.x; i < n; i += 256) {
      const double x = (double)Elem<T>::to_f32(g[i]);
      acc += x * x;
    }
  }
  return acc;
}

template <bool Past>
__global__ __launch_bounds__(256) void clip_norm_kernel(Tensors s, double* __restrict__ part) {
  __shared__ double lds[4];
  double acc = 0.0;
  for (int64_t t = blockIdx.x; t < s.tile0[s.count]; t += gridDim.x) {
    const int i = tensor_of(s, t);
    const int64_t first = (t - s.tile0[i]) * kTile;
    acc += (s.f32[i / 32] >> (i % 32)) & 1 ? tile_squares<Past>(static_cast<const float*>(s.p[i]), first, s.n[i])
                                           : tile_squares<Past>(static_cast<const bf16*>(s.p[i]), first, s.n[i]);
  }
  acc = block_sum64(acc, lds);
  if (threadIdx.x == 0) part[blockIdx.x] = acc;
}

// The factor as a float; one below the normal floats, which would have few bits or none, as a float of [0.5, 1) and a power of two that
// the product takes afterwards. (Products in 64 bits cost bf16 7% of 140 MB.)
struct Factor {
  float head;
  int power;
  __device__ __forceinline__ explicit Factor(double f) : head((float)f), power(0) {
    if (f > 0.0 && f < 0x1p-126) head = (float)frexp(f, &power);
  }
  __device__ __forceinline__ float of(float x) const { return __builtin_amdgcn_ldexpf(x * head, power); }
};

template <bool Past, typename T>
__device__ __forceinline__ void tile_scale(T* g, int64_t first, int64_t n, const Factor& factor) {
  if (first + kTile <= n) {
    Eight<T> v[4];
    load_tile<Past>(v, g + first);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      float x[8];
      v[u].get(x);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = factor.of(x[e]);
      v[u].set(x);
      v[u].store(g + first + u * 2048 + threadIdx.x * 8);
    }
  } else {
    for (int64_t i = first + threadIdx.x; i < n; i += 256) g[i] = Elem<T>::from_f32(factor.of(Elem<T>::to_f32(g[i])));
  }
}

// A norm that is no finite float leaves the gradients as they are: the caller sees it in the norm.
template <bool Past>
__global__ __launch_bounds__(256) void clip_scale_kernel(Tensors s, const double* __restrict__ part, int parts, double most,
                                                         float* __restrict__ norm_out) {
  __shared__ double lds[4];
  double sum = 0.0;
  for (int i = threadIdx.x; i < parts; i += 256) sum += part[i];
  const double norm = sqrt(block_sum64(sum, lds));
  const float rounded = (float)norm;
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = rounded;
  const double factor = most / (norm + 1e-6);
  if (!(rounded < INFINITY) || !(factor < 1.0)) return;
  const Factor scale(factor);
  for (int64_t t = blockIdx.x; t < s.tile0[s.count]; t += gridDim.x) {
    const int i = tensor_of(s, t);
    const int64_t first = (t - s.tile0[i]) * kTile;
    if ((s.f32[i / 32] >> (i % 32)) & 1)
      tile_scale<Past>(static_cast<float*>(s.p[i]), first, s.n[i], scale);
    else
      tile_scale<Past>(static_cast<bf16*>(s.p[i]), first, s.n[i], scale);
  }
}

Tensors make_tensors(int64_t first, int64_t count, void* const* grads, const int64_t* numel, const int32_t* dtypes) {
  Tensors s{};
  s.count = (int)count;
  for (int64_t j = 0; j < count; ++j) {
    s.p[j] = grads[first + j];
    s.n[j] = numel[first + j];
    s.tile0[j + 1] = s.tile0[j] + cdiv(s.n[j], (int64_t)kTile);
    if (dtypes[first + j] == FERRITE_F32) s.f32[j / 32] |= 1u << (j % 32);
  }
  return s;
}

}  // namespace
}  // namespace ferrite

extern "C" int64_t ferrite_internal_clip_workspace(int64_t n_tensors) {
  using namespace ferrite;
  if (n_tensors < 0) return -1;
  return (kParts + cdiv(n_tensors, (int64_t)kTensors)) * (int64_t)sizeof(double);
}

extern "C" int ferrite_internal_clip(int64_t n_tensors, void* const* grads, const int64_t* numel, const int32_t* dtypes,
                                     double most, float* norm, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace ferrite;
  const char* name = "ferrite_clip_grad_norm";
  if (n_tensors < 1 || !(most >= 0.0))
    return fail(FERRITE_ERR_INVALID_ARGUMENT, std::string(name) + ": need tensors and a bound of 0 or more");
  if (!grads || !numel || !dtypes || !norm || !workspace || workspace_bytes < ferrite_internal_clip_workspace(n_tensors) ||
      (reinterpret_cast<uintptr_t>(workspace) & 7))
    return fail(FERRITE_ERR_INVALID_ARGUMENT, std::string(name) + ": null pointer or small workspace");
  int64_t tiles = 0, bytes = 0;
  for (int64_t i = 0; i < n_tensors; ++i) {
    if (!valid_dtype(dtypes[i]))
      return fail(FERRITE_ERR_INVALID_ARGUMENT, std::string(name) + ": dtype must be FERRITE_F32 or FERRITE_BF16");
    if (numel[i] < 0 || numel[i] > ((int64_t)1 << 60) || (numel[i] > 0 && !grads[i]))
      return fail(FERRITE_ERR_INVALID_ARGUMENT, std::string(name) + ": null tensor or bad size");
    tiles += cdiv(numel[i], (int64_t)kTile);
    if (bytes <= kStream) bytes += numel[i] * (dtypes[i] == FERRITE_F32 ? 4 : 2);
  }
  const auto norm_kernel = bytes > kStream ? clip_norm_kernel<true> : clip_norm_kernel<false>;
  const auto scale_kernel = bytes > kStream ? clip_scale_kernel<true> : clip_scale_kernel<false>;
  hipStream_t st = static_cast<hipStream_t>(stream);
  double* part = static_cast<double*>(workspace);
  int parts = 0;
  for (int64_t first = 0; first < n_tensors; first += kTensors) {
    const Tensors s = make_tensors(first, std::min<int64_t>(kTensors, n_tensors - first), grads, numel, dtypes);
    // Its share of the partial sums, at least one (a launch without tiles leaves a zero).
    const int64_t mine = s.tile0[s.count];
    const int blocks = (int)std::max<int64_t>(1, std::min<int64_t>(mine, tiles <= kParts ? mine : kParts * mine / tiles));
    hipLaunchKernelGGL(norm_kernel, dim3((unsigned)blocks), dim3(256), 0, st, s, part + parts);
    parts += blocks;
  }
  for (int64_t first = 0; first < n_tensors; first += kTensors) {
    const Tensors s = make_tensors(first, std::min<int64_t>(kTensors, n_tensors - first), grads, numel, dtypes);
    const int64_t mine = s.tile0[s.count];
    if (mine == 0 && first > 0) continue;  // the first launch leaves the norm
    hipLaunchKernelGGL(scale_kernel, dim3((unsigned)std::clamp<int64_t>(mine, 1, 2048)), dim3(256), 0, st, s, part, parts,
                       most, first == 0 ? norm : nullptr);
  }
  return check_launch(name);
}
