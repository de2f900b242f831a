// Rows of any width and alignment in vectors of W elements (16 bytes, or eight floats), for kernels that hold a row in registers.
//
// Chunk c of a row of dim >= W elements holds elements W c .. W c + W - 1. The last one of a width that is no multiple of W holds
// the row's last W elements instead: the first `skip` of them belong to the chunk before as well, are left
// out of sums, and are stored twice with the same value. So no element is loaded or stored by itself, and rows that start at
// odd elements take the same 16-byte accesses (which this GPU makes at any address) as aligned ones.
#pragma once

#include "common.h"

namespace ferrite {
namespace {

struct Chunk {
  int at, skip;
  bool on;
};
template <int W>
__device__ __forceinline__ Chunk chunk_of(int c, int dim) {
  const int at = min(W * c, dim - W);
  return {at, W * c - at, W * c < dim};
}

// Vectors that may start at any element.
typedef bf16x8 bf16x8_any __attribute__((aligned(2)));
typedef f32x4 f32x4_any __attribute__((aligned(4)));

// Eight elements of T as they lie in memory. Each byte of a row is touched once: the accesses are non-temporal.
template <typename T>
struct Eight;
template <>
struct Eight<bf16> {
  bf16x8 v;
  __device__ __forceinline__ void load(const bf16* p) { v = __builtin_nontemporal_load(reinterpret_cast<const bf16x8_any*>(p)); }
  __device__ __forceinline__ void load_cached(const bf16* p) { v = *reinterpret_cast<const bf16x8_any*>(p); }
  __device__ __forceinline__ void store(bf16* p) const { __builtin_nontemporal_store(v, reinterpret_cast<bf16x8_any*>(p)); }
  __device__ __forceinline__ void get(float (&o)[8]) const {
    const u32x4 w = __builtin_bit_cast(u32x4, v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      o[2 * i] = __uint_as_float(w[i] << 16);
      o[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  __device__ __forceinline__ void set(const float (&x)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (bf16)x[e];
  }
};
template <>
struct Eight<float> {
  f32x4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = __builtin_nontemporal_load(reinterpret_cast<const f32x4_any*>(p));
    b = __builtin_nontemporal_load(reinterpret_cast<const f32x4_any*>(p + 4));
  }
  __device__ __forceinline__ void load_cached(const float* p) {
    a = *reinterpret_cast<const f32x4_any*>(p);
    b = *reinterpret_cast<const f32x4_any*>(p + 4);
  }
  __device__ __forceinline__ void store(float* p) const {
    __builtin_nontemporal_store(a, reinterpret_cast<f32x4_any*>(p));
    __builtin_nontemporal_store(b, reinterpret_cast<f32x4_any*>(p + 4));
  }
  __device__ __forceinline__ void get(float (&o)[8]) const {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      o[e] = a[e];
      o[4 + e] = b[e];
    }
  }
  __device__ __forceinline__ void set(const float (&x)[8]) {
    a = f32x4{x[0], x[1], x[2], x[3]};
    b = f32x4{x[4], x[5], x[6], x[7]};
  }
};

// Columns of W elements in one access (two of 16 bytes for eight floats), or one where a row has fewer.
template <typename T, int W>
struct Cols;
template <typename T>
struct Cols<T, 8> : Eight<T> {};
template <typename T>
struct Cols<T, 4> {
  typedef T vec __attribute__((ext_vector_type(4)));
  typedef vec any __attribute__((aligned(sizeof(T))));
  vec v;
  __device__ __forceinline__ void load(const T* p) { v = __builtin_nontemporal_load(reinterpret_cast<const any*>(p)); }
  __device__ __forceinline__ void load_cached(const T* p) { v = *reinterpret_cast<const any*>(p); }
  __device__ __forceinline__ void store(T* p) const { __builtin_nontemporal_store(v, reinterpret_cast<any*>(p)); }
  __device__ __forceinline__ void get(float (&o)[4]) const {
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = Elem<T>::to_f32(v[e]);
  }
  __device__ __forceinline__ void set(const float (&x)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = Elem<T>::from_f32(x[e]);
  }
};
template <typename T>
struct Cols<T, 1> {
  T v;
  __device__ __forceinline__ void load(const T* p) { v = *p; }
  __device__ __forceinline__ void store(T* p) const { *p = v; }
  __device__ __forceinline__ void get(float (&o)[1]) const { o[0] = Elem<T>::to_f32(v); }
  __device__ __forceinline__ void set(const float (&x)[1]) { v = Elem<T>::from_f32(x[0]); }
};
// First column of unit c of a row of dim >= W; -1 past it. The last unit lies over the one before, as a Chunk does.
template <int W>
__device__ __forceinline__ int column(int c, int dim) {
  return c < (dim + W - 1) / W ? min(W * c, dim - W) : -1;
}

// The sums of partial rows [parts][arrays][dim], array blockIdx.y of them into a or b (or none, where that is null): 64 columns to a
// workgroup, whose 16 waves each add every 16th row in turn; the waves' sums are added in their order.
template <typename T>
__global__ __launch_bounds__(1024) void join_parts_kernel(const float* __restrict__ part, T* __restrict__ a, T* __restrict__ b,
                                                          int parts, int64_t dim) {
  __shared__ float red[16][64];
  T* const out = blockIdx.y ? b : a;
  if (!out) return;
  const int c = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t col = (int64_t)blockIdx.x * 64 + c;
  float acc = 0.f;
  if (col < dim) {
#pragma unroll 8
    for (int p = wave; p < parts; p += 16) acc += part[((int64_t)p * gridDim.y + blockIdx.y) * dim + col];
  }
  red[wave][c] = acc;
  __syncthreads();
  if (wave == 0 && col < dim) {
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) sum += red[k][c];
    out[col] = Elem<T>::from_f32(sum);
  }
}
template <typename T>
void join_parts(const float* part, T* a, T* b, int arrays, int parts, int64_t dim, hipStream_t stream) {
  hipLaunchKernelGGL((join_parts_kernel<T>), dim3((unsigned)cdiv(dim, (int64_t)64), (unsigned)arrays), dim3(1024), 0, stream,
                     part, a, b, parts, dim);
}

// Sum over a group of G threads (a wave, or a whole workgroup of G), in every one of its threads. Two sums share the waits.
template <int G>
__device__ __forceinline__ void rows_sum(float& x, float& y, float (*lds)[16]) {
  x = wave_sum(x);
  y = wave_sum(y);
  if constexpr (G > 64) {
    __syncthreads();  // the previous sums have been read
    if ((threadIdx.x & 63) == 0) {
      lds[0][threadIdx.x >> 6] = x;
      lds[1][threadIdx.x >> 6] = y;
    }
    __syncthreads();
    x = y = 0.f;
#pragma unroll
    for (int w = 0; w < G / 64; ++w) {
      x += lds[0][w];
      y += lds[1][w];
    }
  }
}

}  // namespace
}  // namespace ferrite
