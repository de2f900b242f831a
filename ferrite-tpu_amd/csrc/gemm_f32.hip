// f32 products for a linear layer's passes, for gfx950: any sizes, rows that start at any element, either operand
// given transposed, without copies.
//
// Reference: src/ferrite/kernels/matmul.py:27-38, :99-104 (the blocked matmul and the two products of its VJP).
//
// Bound by the f32 matrix pipes (153 TFLOP/s in torch's product of 8192^3) where there are tiles enough for every CU, by latency and the
// last round of tiles where there are not. matmul.hip's f32 kernels load rows that are not 16-byte aligned by single floats and
// have transposed operands copied first; here every load is 16 bytes, which this GPU makes at any 4-byte address:
//   k-contiguous (x, or y transposed)      staged as [free][k] in 128-byte rows, chunks XOR-swizzled by row; a lane reads its 8 k in two
//   free-contiguous (y, or x transposed)   staged as [k][free] in 256-byte rows; a lane reads its 8 k one by one, a row's 32 lanes 128
//                                          consecutive bytes
// Both give product e of a 16-deep step element e of every lane, k = 8 (lane / 32) + e, so any pair of layouts meets in
// v_mfma_f32_32x32x2_f32. A workgroup of four waves owns 64 x 64 outputs, 32 x 32 to a wave, over two LDS stages of 32 k; four or more
// workgroups share a CU, and K is cut until there are about that many (f32_any_slices), the slabs added in order by the pass that
// follows anyway (linear.h) or by gemm_splitk_reduce_kernel.
#include "gemm_f32.h"

#include <algorithm>

namespace ferrite {
namespace {

constexpr int kTile = 64, kDepth = 32, kThreads = 256, kMostSlices = 32;
constexpr int kOperand = kTile * kDepth * 4;  // bytes of an operand's stage
typedef f32x4 f32x4_any __attribute__((aligned(4)));

__device__ __forceinline__ f32x4 load4(const float* p) { return *reinterpret_cast<const f32x4_any*>(p); }

// One operand of a tile: 64 free indices from f0 (of F) by 32 k, two vectors of four a thread.
template <bool KC>
struct Operand {
  const float* p;
  int64_t ld;
  int f0, F;
  f32x4 v[2];

  // Values past the k of the slice and past K are zeros; free indices past F are anything that is there.
  __device__ __forceinline__ void load(int k0, int kend, int K) {
    const bool whole = k0 + kDepth <= kend && f0 + kTile <= F;  // uniform
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int idx = threadIdx.x + kThreads * i;
      if constexpr (KC) {
        const int f = f0 + idx / 8, k = k0 + idx % 8 * 4;
        if (whole) {
          v[i] = load4(p + (int64_t)f * ld + k);
        } else {
          const int at = min(k, K - 4), skip = k - at;  // the last vector of a row ends with the row
          const f32x4 w = load4(p + (int64_t)min(f, F - 1) * ld + at);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float t = 0.f;
#pragma unroll
            for (int s = 0; s < 4; ++s)
              if (e + s < 4 && s == skip) t = w[e + s];
            v[i][e] = k + e < kend ? t : 0.f;
          }
        }
      } else {
        const int k = k0 + idx / 16, f = f0 + idx % 16 * 4;
        if (whole) {
          v[i] = load4(p + (int64_t)k * ld + f);
        } else {
          const int at = min(f, F - 4), skip = f - at;
          const f32x4 w = load4(p + (int64_t)min(k, K - 1) * ld + at);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float t = 0.f;
#pragma unroll
            for (int s = 0; s < 4; ++s)
              if (e + s < 4 && s == skip) t = w[e + s];
            v[i][e] = k < kend ? t : 0.f;
          }
        }
      }
    }
  }
  static __device__ __forceinline__ int row_off(int row, int chunk) {
    return row * 128 + ((chunk ^ ((row ^ (row >> 3)) & 7)) << 4);
  }
  __device__ __forceinline__ void store(char* lds) const {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int idx = threadIdx.x + kThreads * i;
      *reinterpret_cast<f32x4*>(lds + (KC ? row_off(idx / 8, idx % 8) : idx * 16)) = v[i];
    }
  }
  // The lane's 8 values of free index f (of the tile), k = 16 step + 8 g + e.
  static __device__ __forceinline__ void read(const char* lds, int f, int step, int g, float (&o)[8]) {
    if constexpr (KC) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const f32x4 w = *reinterpret_cast<const f32x4*>(lds + row_off(f, 4 * step + 2 * g + h));
#pragma unroll
        for (int e = 0; e < 4; ++e) o[4 * h + e] = w[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = *reinterpret_cast<const float*>(lds + (16 * step + 8 * g + e) * 256 + f * 4);
    }
  }
};

template <bool XT, bool YT>
__global__ __launch_bounds__(kThreads, 4) void gemm_f32_any_kernel(const float* __restrict__ x, const float* __restrict__ y,
                                                                   float* __restrict__ out, int M, int N, int K, int tiles_m,
                                                                   int tiles_n, int kslice, int64_t slab) {
  __shared__ __attribute__((aligned(16))) char smem[2][2 * kOperand];
  // Blocks are dealt to the 8 XCDs round robin: an XCD's are made consecutive, slices slowest, tiles in groups of 4 tile rows.
  const int total = (int)gridDim.x, xcd = blockIdx.x % 8, q = total / 8, rest = total % 8;
  const int v = xcd * q + min(xcd, rest) + blockIdx.x / 8;
  const int tiles = tiles_m * tiles_n, slice = v / tiles, tile = v % tiles;
  const int first_m = tile / (4 * tiles_n) * 4, gsize = min(tiles_m - first_m, 4), in = tile % (4 * tiles_n);
  const int m0 = (first_m + in % gsize) * kTile, n0 = in / gsize * kTile;
  const int lane = threadIdx.x & 63, l32 = lane & 31, g = lane >> 5, wave = threadIdx.x >> 6;
  const int wm = (wave & 1) * 32, wn = (wave >> 1) * 32;
  Operand<!XT> xo{x, XT ? M : K, m0, M};
  Operand<YT> yo{y, YT ? K : N, n0, N};
  const int kbeg = slice * kslice, kend = min(K, kbeg + kslice);

  f32x16 acc;
#pragma unroll
  for (int r = 0; r < 16; ++r) acc[r] = 0.f;
  xo.load(kbeg, kend, K);
  yo.load(kbeg, kend, K);
  xo.store(smem[0]);
  yo.store(smem[0] + kOperand);
  __syncthreads();
  int at = 0;
  for (int k0 = kbeg; k0 < kend; k0 += kDepth, at ^= 1) {
    const bool more = k0 + kDepth < kend;
    if (more) {
      xo.load(k0 + kDepth, kend, K);
      yo.load(k0 + kDepth, kend, K);
    }
#pragma unroll
    for (int step = 0; step < 2; ++step) {
      float a[8], b[8];
      Operand<YT>::read(smem[at] + kOperand, wn + l32, step, g, a);
      Operand<!XT>::read(smem[at], wm + l32, step, g, b);
#pragma unroll
      for (int e = 0; e < 8; ++e) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], acc, 0, 0, 0);
    }
    if (more) {
      xo.store(smem[at ^ 1]);
      yo.store(smem[at ^ 1] + kOperand);
    }
    __syncthreads();
  }
  // Register r of lane (l32, g): out[m0 + wm + l32][n0 + wn + (r / 4) 8 + 4 g + r % 4].
  const int m = m0 + wm + l32;
  if (m >= M) return;
  float* const row = out + slice * slab + (int64_t)m * N;
#pragma unroll
  for (int qd = 0; qd < 4; ++qd) {
    const int n = n0 + wn + qd * 8 + 4 * g;
    if (n + 4 <= N) {
      *reinterpret_cast<f32x4_any*>(row + n) = f32x4{acc[4 * qd], acc[4 * qd + 1], acc[4 * qd + 2], acc[4 * qd + 3]};
    } else {
#pragma unroll
      for (int e = 0; e < 3; ++e)
        if (n + e < N) row[n + e] = acc[4 * qd + e];
    }
  }
}

}  // namespace

bool f32_any_ok(int64_t m, int64_t n, int64_t k, bool xt, bool yt) {
  return m >= 1 && n >= 1 && k >= 1 && m <= 0x7fffff00 && n <= 0x7fffff00 && k <= 0x7fffff00 && (xt ? m : k) >= 4 &&
         (yt ? k : n) >= 4 && cdiv(m, (int64_t)kTile) * cdiv(n, (int64_t)kTile) < (1 << 24) / kMostSlices &&  // under 2^32 threads
         m <= ((int64_t)1 << 58) / n;
}

// The number of slices with the least estimated time: the rounds of tiles on the fullest CU, at 110 TFLOP/s over the chip and less
// where fewer than three workgroups share a CU, and for more than one slice the slabs' way through memory and the pass that
// adds them. us of the kernel alone, M x K x N by slices: 2100 x 1003 x 515 68 (1), 45 (2), 38.5 (3, taken), 35.5 (8);
// 1003 x 2100 x 515 106 (1), 47 (3), 38 (5, taken), 40.5 (8); 2100 x 515 x 1003 45 (1, taken), 36 (3, and 10 for the slabs). With the
// adding pass, 16 sizes from 100 x 2048 x 70 to 8192 x 768 x 768 in three layouts against each fixed number of up to 32: within 0.7% of the
// best in the mean, 14% at worst (2100 x 515 x 1003 in one slice 44.7, in three 39.3).
int f32_any_slices(int64_t m, int64_t n, int64_t k, int64_t cus) {
  const int64_t tiles = cdiv(m, (int64_t)kTile) * cdiv(n, (int64_t)kTile), most = std::clamp<int64_t>(k / (4 * kDepth), 1, kMostSlices);
  const double tile_us = 18.7e-3 * (double)k, slab_us = (double)m * (double)n * 8 / 5e6;
  int best = 1;
  double least = 1e300;
  for (int64_t g = 1; g <= most; ++g) {
    const double share = (double)(tiles * g) / (double)cus;
    const double us = tile_us * (double)cdiv(tiles * g, cus) / (double)g * (share < 3 ? 1 + 0.25 * (3 - share) : 1) +
                      (g > 1 ? 4 + slab_us * (double)g : 0);
    if (us < least) {
      least = us;
      best = (int)g;
    }
  }
  return best;
}

int f32_any_launch(const F32Product& p, hipStream_t stream) {
  const int64_t tiles_m = cdiv(p.m, (int64_t)kTile), tiles_n = cdiv(p.n, (int64_t)kTile);
  const int kslice = (int)(cdiv(cdiv(p.k, (int64_t)p.slices), (int64_t)kDepth) * kDepth);
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)(tiles_m * tiles_n * p.slices)), dim3(kThreads), 0, stream, p.x, p.y, p.out,
                       (int)p.m, (int)p.n, (int)p.k, (int)tiles_m, (int)tiles_n, kslice, p.slab);
    return check_launch("ferrite_matmul");
  };
  if (p.xt && p.yt) return go(gemm_f32_any_kernel<true, true>);
  if (p.xt) return go(gemm_f32_any_kernel<true, false>);
  if (p.yt) return go(gemm_f32_any_kernel<false, true>);
  return go(gemm_f32_any_kernel<false, false>);
}

}  // namespace ferrite
