// What follows the product of a linear layer: out = act(x . w + bias) + residual, and act's derivative.
//
// Sums, activation and residual are f32, rounded once to the output's type; the pre-activation that a backward needs (aux) is
// rounded to the type of x. GELU is gelu.h's tanh form. silu(u) = u s with s = 1 / (1 + 2^(-u log2 e)).
#pragma once

#include "common.h"
#include "gelu.h"
#include "internal_api.h"
#include "rows.h"

namespace ferrite {
namespace {

constexpr int kEpiLinear = 3;  // beside gelu.h's

struct LinArgs {
  const void* bias;      // [N], f32 or bf16, or null
  const void* residual;  // [M, N] of the output's type, or null
  int bias_f32, act;
};

__device__ __forceinline__ float silu_gate(float u) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-kLog2e * u));
}
__device__ __forceinline__ float act_of(float u, int act) {
  switch (act) {
    case FERRITE_ACT_RELU:
      return u < 0.f ? 0.f : u;  // NaN stays
    case FERRITE_ACT_GELU:
      return gelu_tanh(u);
    case FERRITE_ACT_SILU:
      return u * silu_gate(u);
    default:
      return u;
  }
}
// The activation of eight values, its kind looked at once.
__device__ __forceinline__ void act_eight(float (&v)[8], int act) {
  if (act == FERRITE_ACT_RELU) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = v[e] < 0.f ? 0.f : v[e];
  } else if (act == FERRITE_ACT_GELU) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = gelu_tanh(v[e]);
  } else if (act == FERRITE_ACT_SILU) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= silu_gate(v[e]);
  }
}
// The same of the sums acc[0 .. YF - 1][i] of a 32 x 32 product.
template <int YF, int XF>
__device__ __forceinline__ void act_sums(f32x16 (&acc)[YF][XF], int i, int act) {
  if (act == FERRITE_ACT_RELU) {
#pragma unroll
    for (int j = 0; j < YF; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[j][i][r] = acc[j][i][r] < 0.f ? 0.f : acc[j][i][r];
  } else if (act == FERRITE_ACT_GELU) {
#pragma unroll
    for (int j = 0; j < YF; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[j][i][r] = gelu_tanh(acc[j][i][r]);
  } else if (act == FERRITE_ACT_SILU) {
#pragma unroll
    for (int j = 0; j < YF; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[j][i][r] *= silu_gate(acc[j][i][r]);
  }
}
// Past |u| = 64 GELU's gate is 0 or 1 in f32, past 128 SiLU's too (1.6e-28 at -64), and the slopes are: there squares could overflow and
// an infinity meet a zero.
__device__ __forceinline__ float act_slope(float u, int act) {
  if (act == FERRITE_ACT_RELU) return u > 0.f ? 1.f : u != u ? u : 0.f;
  const float far = act == FERRITE_ACT_GELU ? 64.f : 128.f;
  const float v = u < -far ? -far : u > far ? far : u;
  if (act == FERRITE_ACT_GELU) return gelu_tanh_grad(v);
  const float s = silu_gate(v);
  return s + v * s * (1.f - s);
}

__device__ __forceinline__ float bias_at(const LinArgs& a, int64_t n) {
  if (!a.bias) return 0.f;
  return a.bias_f32 ? static_cast<const float*>(a.bias)[n] : (float)static_cast<const bf16*>(a.bias)[n];
}
// The biases of eight columns from n.
__device__ __forceinline__ void bias_eight(const LinArgs& a, int64_t n, float (&o)[8]) {
  if (!a.bias) {
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = 0.f;
  } else if (a.bias_f32) {
    Eight<float> v;
    v.load_cached(static_cast<const float*>(a.bias) + n);
    v.get(o);
  } else {
    Eight<bf16> v;
    v.load_cached(static_cast<const bf16*>(a.bias) + n);
    v.get(o);
  }
}

// Four columns from n of N, the last one again past them.
__device__ __forceinline__ void bias_four(const LinArgs& a, int n, int N, float* o) {
  if (n + 4 <= N) {
    if (a.bias_f32) {
      const f32x4 v = *reinterpret_cast<const f32x4_any*>(static_cast<const float*>(a.bias) + n);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = v[e];
    } else {
      typedef bf16x4 bf16x4_any __attribute__((aligned(2)));
      const bf16x4 v = *reinterpret_cast<const bf16x4_any*>(static_cast<const bf16*>(a.bias) + n);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = (float)v[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = bias_at(a, min(n + e, N - 1));
  }
}

// The second pass of a product that is cut along K, or that a kernel without this epilogue leaves in f32: `slices` slabs
// added in order, then the epilogue. Eight elements a thread where rows hold whole eights, else one. With one slice
// part and out may be the same.
template <typename TO, int W>
__global__ __launch_bounds__(256) void linear_pass_kernel(const float* part, int slices, int64_t slab, TO* out,
                                                          TO* __restrict__ aux, LinArgs a, int64_t mn, int N) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * W;
  if (i >= mn) return;
  const int n = (int)(i % N);
  const TO* res = static_cast<const TO*>(a.residual);
  if constexpr (W == 8) {
    float v[8], t[8];
    Eight<float> p;
    p.load_cached(part + i);
    p.get(v);
    for (int s = 1; s < slices; ++s) {
      p.load_cached(part + s * slab + i);
      p.get(t);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += t[e];
    }
    bias_eight(a, n, t);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += t[e];
    Eight<TO> o;
    if (aux) {
      o.set(v);
      o.store(aux + i);
    }
    act_eight(v, a.act);
    if (res) {
      o.load(res + i);
      o.get(t);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += t[e];
    }
    o.set(v);
    o.store(out + i);
  } else {
    float v = part[i];
    for (int s = 1; s < slices; ++s) v += part[s * slab + i];
    v += bias_at(a, n);
    if (aux) aux[i] = Elem<TO>::from_f32(v);
    v = act_of(v, a.act);
    if (res) v += Elem<TO>::to_f32(res[i]);
    out[i] = Elem<TO>::from_f32(v);
  }
}

template <typename TO>
int linear_pass(const float* part, int slices, int64_t slab, void* out, void* aux, const LinArgs& a, int64_t m, int64_t n,
                hipStream_t stream) {
  const int64_t mn = m * n;
  const bool whole = n % 8 == 0;
  const int64_t blocks = cdiv(whole ? mn / 8 : mn, 256);
  if (blocks > 0xffffffff / 256) return fail(FERRITE_ERR_INVALID_ARGUMENT, "ferrite_linear: output too large");
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), 0, stream, part, slices, slab, static_cast<TO*>(out),
                       static_cast<TO*>(aux), a, mn, (int)n);
  };
  if (whole)
    go(linear_pass_kernel<TO, 8>);
  else
    go(linear_pass_kernel<TO, 1>);
  return check_launch("ferrite_linear");
}

}  // namespace
}  // namespace ferrite
