// Layer norm, with the residual add before it, forward and backward, for gfx950.
//
// No counterpart in the reference, whose model norms by RMS (src/ferrite/kernels/rmsnorm.py:39-56); the interface is that of
// the RMS norm's kernels (rmsnorm.hip).
//   h   = x + r in f32, rounded to x's type (h = x without r)
//   y   = (h - mean) rstd w + b,  mean = sum(h) / dim,  rstd = 1 / sqrt(sum((h - mean)^2) / dim + eps)
//   g   = dy w,  n = (h - mean) rstd
//   dh  = rstd (g - mean(g) - n mean(g n)) [+ the gradient that h has of its own]
//   dw  = sum over rows of dy n,  db = sum over rows of dy
// The norm is that of the h which is stored, so the backward is the derivative of what the forward computed.
//
// Bound by memory: a row is read once and stays in registers, every input and output moves once. Statistics are f32. The mean is
// corrected by the mean of the differences from it, which costs one more value in the second reduction: a row whose mean is
// 10^4 times its deviation keeps its precision. The forward leaves mean and rstd for the backward.
//
// dw and db have a fixed order: a thread owns the same columns on every row of its group, the groups of a workgroup
// are added through LDS into a partial row each, and a second kernel adds the partial rows.
#include <algorithm>

#include "common.h"
#include "internal_api.h"
#include "rows.h"

namespace ferrite {
namespace {

template <typename TW, int W>
__device__ __forceinline__ void load_params(const TW* p, int at, float (&o)[W]) {
  if (!p) {
#pragma unroll
    for (int e = 0; e < W; ++e) o[e] = 0.f;
    return;
  }
  Cols<TW, W> v;
  v.load_cached(p + at);
  v.get(o);
}

// 1 / sqrt(v). The instruction takes a subnormal v, which small rows have with eps = 0, for zero.
__device__ __forceinline__ float inverse_root(float v) {
  return v < 0x1p-126f ? __builtin_amdgcn_rsqf(v * 0x1p48f) * 0x1p24f : __builtin_amdgcn_rsqf(v);
}

// G threads own a row, VPL chunks of W elements each: chunk t + G i of thread t. W is 16 bytes: eight floats of a lane in two accesses
// would leave every other 16 bytes of a line to the next instruction. A wave (G = 64) takes D rows at a time, whose loads go out together,
// and keeps its weights; wider groups read the weights again for every row, from L2.
template <typename TX, typename TW, bool RES, int W, int VPL, int G, int D>
__global__ __launch_bounds__((G < 256 ? 256 : G)) void layernorm_kernel(
    const TX* __restrict__ x, const TX* __restrict__ r, const TW* __restrict__ w, const TW* __restrict__ b,
    TX* __restrict__ h, TX* __restrict__ y, float* __restrict__ stats, int64_t rows, int dim, float inv_dim, float eps) {
  constexpr int kGroups = G < 256 ? 256 / G : 1;
  constexpr bool kKeep = G == 64 && W * VPL <= 16;
  __shared__ float lds[2][16];
  const int t = threadIdx.x % G;
  Chunk ch[VPL];
  float wv[VPL][W], bv[VPL][W];
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    ch[i] = chunk_of<W>(t + G * i, dim);
    if (kKeep && ch[i].on) {
      load_params(w, ch[i].at, wv[i]);
      load_params(b, ch[i].at, bv[i]);
    }
  }
  for (int64_t row0 = ((int64_t)blockIdx.x * kGroups + threadIdx.x / G) * D; row0 < rows;
       row0 += (int64_t)gridDim.x * kGroups * D) {
    Cols<TX, W> xr[D][VPL], rr[D][VPL];
#pragma unroll
    for (int k = 0; k < D; ++k) {
      const int64_t off = min(row0 + k, rows - 1) * dim;
#pragma unroll
      for (int i = 0; i < VPL; ++i)
        if (ch[i].on) {
          xr[k][i].load(x + off + ch[i].at);
          if constexpr (RES) rr[k][i].load(r + off + ch[i].at);
        }
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int k = 0; k < D; ++k) {
      const int64_t row = row0 + k, off = row * dim;
      if (D > 1 && row >= rows) break;
      float hv[VPL][W];
      float sum = 0.f, none = 0.f;
#pragma unroll
      for (int i = 0; i < VPL; ++i)
        if (ch[i].on) {
          xr[k][i].get(hv[i]);
          if constexpr (RES) {
            float rv[W];
            rr[k][i].get(rv);
#pragma unroll
            for (int e = 0; e < W; ++e) hv[i][e] += rv[e];
            Cols<TX, W> out;
            out.set(hv[i]);
            out.store(h + off + ch[i].at);
            out.get(hv[i]);
          }
#pragma unroll
          for (int e = 0; e < W; ++e) sum += e >= ch[i].skip ? hv[i][e] : 0.f;
        }
      rows_sum<G>(sum, none, lds);
      const float mean = sum * inv_dim;
      float rest = 0.f, square = 0.f;
#pragma unroll
      for (int i = 0; i < VPL; ++i)
        if (ch[i].on)
#pragma unroll
          for (int e = 0; e < W; ++e) {
            hv[i][e] -= mean;
            const float c = e >= ch[i].skip ? hv[i][e] : 0.f;
            rest += c;
            square += c * c;
          }
      rows_sum<G>(rest, square, lds);
      rest *= inv_dim;
      // max(0, NaN) would hide a NaN, so the difference is compared
      float var = square * inv_dim - rest * rest;
      var = var < 0.f ? 0.f : var;
      const float rstd = inverse_root(var + eps);
      if (stats && t == 0) {
        stats[2 * row] = mean + rest;
        stats[2 * row + 1] = rstd;
      }
#pragma unroll
      for (int i = 0; i < VPL; ++i)
        if (ch[i].on) {
          if constexpr (!kKeep) {
            load_params(w, ch[i].at, wv[i]);
            load_params(b, ch[i].at, bv[i]);
          }
          float yv[W];
#pragma unroll
          for (int e = 0; e < W; ++e) yv[e] = (hv[i][e] - rest) * rstd * wv[i][e] + bv[i][e];
          Cols<TX, W> out;
          out.set(yv);
          out.store(y + off + ch[i].at);
        }
    }
  }
}

// Rows of fewer than 8 elements or of more than a group holds: a workgroup to a row, swept three times (from the caches after
// the first).
template <typename TX, typename TW, bool RES>
__global__ __launch_bounds__(256) void layernorm_sweep_kernel(const TX* __restrict__ x, const TX* __restrict__ r,
                                                              const TW* __restrict__ w, const TW* __restrict__ b,
                                                              TX* __restrict__ h, TX* __restrict__ y,
                                                              float* __restrict__ stats, int64_t rows, int64_t dim,
                                                              float inv_dim, float eps) {
  __shared__ float lds[2][16];
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const int64_t off = row * dim;
    auto value = [&](int64_t e) {
      const float v = Elem<TX>::to_f32(x[off + e]);
      return RES ? Elem<TX>::to_f32(Elem<TX>::from_f32(v + Elem<TX>::to_f32(r[off + e]))) : v;
    };
    float sum = 0.f, none = 0.f, rest = 0.f, square = 0.f;
    for (int64_t e = threadIdx.x; e < dim; e += 256) {
      const float v = value(e);
      if constexpr (RES) h[off + e] = Elem<TX>::from_f32(v);
      sum += v;
    }
    rows_sum<256>(sum, none, lds);
    const float mean = sum * inv_dim;
    for (int64_t e = threadIdx.x; e < dim; e += 256) {
      const float c = value(e) - mean;
      rest += c;
      square += c * c;
    }
    rows_sum<256>(rest, square, lds);
    rest *= inv_dim;
    float var = square * inv_dim - rest * rest;
    var = var < 0.f ? 0.f : var;
    const float rstd = inverse_root(var + eps);
    if (stats && threadIdx.x == 0) {
      stats[2 * row] = mean + rest;
      stats[2 * row + 1] = rstd;
    }
    for (int64_t e = threadIdx.x; e < dim; e += 256)
      y[off + e] = Elem<TX>::from_f32((value(e) - mean - rest) * rstd * Elem<TW>::to_f32(w[e]) +
                                      (b ? Elem<TW>::to_f32(b[e]) : 0.f));
  }
}

// Threads to a row and eights of elements to a thread; group 0: the sweeps. Below 8 elements a row goes to them too.
struct NormPlan {
  int group, vpl;
};
NormPlan norm_plan(int64_t dim) {
  if (dim < 8 || dim > 16384) return {0, 0};
  const int64_t chunks = cdiv(dim, 8);
  if (chunks <= 256) return {64, chunks <= 64 ? 1 : chunks <= 128 ? 2 : 4};
  if (chunks <= 1024) return {256, chunks <= 512 ? 2 : 4};
  return {512, 4};
}

// Runs the statement with VPL and G as constants.
#define FERRITE_NORM_CASE(plan, ...)                      \
  do {                                                    \
    auto run = [&](auto vpl, auto group) {                \
      constexpr int W = 16 / sizeof(TX);                  \
      constexpr int VPL = decltype(vpl)::value * 8 / W;   \
      constexpr int G = decltype(group)::value;           \
      __VA_ARGS__;                                        \
    };                                                    \
    const NormPlan& p_ = plan;                            \
    if (p_.group == 64 && p_.vpl == 1)                    \
      run(Int<1>(), Int<64>());                           \
    else if (p_.group == 64 && p_.vpl == 2)               \
      run(Int<2>(), Int<64>());                           \
    else if (p_.group == 64)                              \
      run(Int<4>(), Int<64>());                           \
    else if (p_.group == 256 && p_.vpl == 2)              \
      run(Int<2>(), Int<256>());                          \
    else if (p_.group == 256)                             \
      run(Int<4>(), Int<256>());                          \
    else                                                  \
      run(Int<4>(), Int<512>());                          \
  } while (0)
template <int N>
struct Int {
  static constexpr int value = N;
};

template <typename TX, typename TW, bool RES>
int norm_launch(const TX* x, const TX* r, const TW* w, const TW* b, TX* h, TX* y, float* stats, int64_t rows, int64_t dim,
                float eps, hipStream_t stream) {
  const float inv_dim = (float)(1.0 / (double)dim);
  const NormPlan plan = norm_plan(dim);
  if (!plan.group) {
    hipLaunchKernelGGL((layernorm_sweep_kernel<TX, TW, RES>), dim3((unsigned)std::min<int64_t>(rows, 1 << 20)), dim3(256), 0,
                       stream, x, r, w, b, h, y, stats, rows, dim, inv_dim, eps);
    return check_launch("ferrite_layernorm");
  }
  // Two rows of a wave under way where there are rows for it and they are short in bytes. us, add and norm, a row at a time / two:
  // 8192 x 768 bf16 13.1 / 11.1, 500 x 1024 bf16 4.3 / 6.3, 3001 x 1003 f32 (no add) 7.0 / 7.7. Four of 512 columns: 32768 rows 25.1
  // / 28.1 (4). At most eight workgroups of four waves per CU; with four 8192 x 2048 bf16 33.0 and not 28.6.
  FERRITE_NORM_CASE(plan, constexpr int kGroups = G < 256 ? 256 / G : 1; auto go = [&](auto kernel, int64_t depth) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)std::min<int64_t>(cdiv(rows, kGroups * depth), G > 256 ? 512 : 2048)),
                       dim3(G < 256 ? 256 : G), 0, stream, x, r, w, b, h, y, stats, rows, (int)dim, inv_dim, eps);
  };
                    if constexpr (sizeof(TX) == 2 && VPL == 2 && G == 64) {
                      if (rows >= 4096) return go(layernorm_kernel<TX, TW, RES, W, VPL, G, 2>, 2);
                    };
                    go(layernorm_kernel<TX, TW, RES, W, VPL, G, 1>, 1));
  return check_launch("ferrite_layernorm");
}

// ---------------------------------------------------------------------------
// Backward
// ---------------------------------------------------------------------------
constexpr int kBwdParts = 512;  // partial rows of dw and db

template <typename TX, typename TW, bool DIRECT, int W, int VPL, int G>
__global__ __launch_bounds__((G < 256 ? 256 : G)) void layernorm_bwd_kernel(
    const TX* __restrict__ h, const TW* __restrict__ w, const TX* __restrict__ dy, const TX* __restrict__ dd,
    const float* __restrict__ stats, TX* __restrict__ dh, float* __restrict__ part, int64_t rows, int dim, float inv_dim) {
  constexpr int kGroups = G < 256 ? 256 / G : 1;
  // The widest rows leave no registers for the next row and the weights (up to 180 spilled).
  constexpr bool kAhead = G * W * VPL < 16384;
  extern __shared__ float red[];  // [kGroups][dim] where there is more than one group
  __shared__ float lds[2][16];
  const int t = threadIdx.x % G, grp = threadIdx.x / G;
  Chunk ch[VPL];
  float wv[VPL][W], dw[VPL][W], db[VPL][W];
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    ch[i] = chunk_of<W>(t + G * i, dim);
    if (kAhead && ch[i].on) load_params(w, ch[i].at, wv[i]);
#pragma unroll
    for (int e = 0; e < W; ++e) dw[i][e] = db[i][e] = 0.f;
  }
  Cols<TX, W> hr[VPL], gr[VPL], dr[VPL];
  float mean = 0.f, rstd = 0.f;
  auto load = [&](int64_t row) {
    const int64_t off = row * dim;
    mean = stats[2 * row];
    rstd = stats[2 * row + 1];
#pragma unroll
    for (int i = 0; i < VPL; ++i)
      if (ch[i].on) {
        hr[i].load(h + off + ch[i].at);
        gr[i].load(dy + off + ch[i].at);
        if constexpr (DIRECT && kAhead) dr[i].load(dd + off + ch[i].at);
      }
  };
  const int64_t step = (int64_t)gridDim.x * kGroups;
  int64_t row = (int64_t)blockIdx.x * kGroups + grp;
  if (kAhead && row < rows) load(row);
  for (; row < rows; row += step) {
    if (!kAhead) load(row);
    const int64_t off = row * dim;
    float cv[VPL][W], gv[VPL][W], dv[VPL][W];
    float rest = 0.f, sg = 0.f, sgc = 0.f, none = 0.f;
    const float m = mean, rs = rstd;
#pragma unroll
    for (int i = 0; i < VPL; ++i)
      if (ch[i].on) {
        hr[i].get(cv[i]);
        gr[i].get(gv[i]);
        if constexpr (DIRECT && kAhead) dr[i].get(dv[i]);
      }
    if (kAhead && row + step < rows) load(row + step);  // the next row's, under way during this one's sums
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < VPL; ++i)
      if (ch[i].on) {
        if (!kAhead) {
          __builtin_amdgcn_sched_barrier(0);
          load_params(w, ch[i].at, wv[i]);
        }
#pragma unroll
        for (int e = 0; e < W; ++e) {
          cv[i][e] -= m;
          const bool mine = e >= ch[i].skip;
          const float g = mine ? gv[i][e] * wv[i][e] : 0.f;
          rest += mine ? cv[i][e] : 0.f;
          sg += g;
          sgc += g * cv[i][e];
        }
      }
    rows_sum<G>(rest, sg, lds);
    rows_sum<G>(sgc, none, lds);
    rest *= inv_dim;
    const float mg = sg * inv_dim, mgn = (sgc - rest * sg) * inv_dim * rs;  // mean(g), mean(g n)
#pragma unroll
    for (int i = 0; i < VPL; ++i)
      if (ch[i].on) {
        if constexpr (!kAhead) {
          __builtin_amdgcn_sched_barrier(0);  // a chunk's weights and gradients at a time: all of them spill
          load_params(w, ch[i].at, wv[i]);
          if constexpr (DIRECT) {
            dr[i].load(dd + off + ch[i].at);
            dr[i].get(dv[i]);
          }
        }
        float o[W];
#pragma unroll
        for (int e = 0; e < W; ++e) {
          const float n = (cv[i][e] - rest) * rs;
          o[e] = rs * (gv[i][e] * wv[i][e] - mg - n * mgn);
          if constexpr (DIRECT) o[e] += dv[i][e];
          dw[i][e] += gv[i][e] * n;
          db[i][e] += gv[i][e];
        }
        Cols<TX, W> out;
        out.set(o);
        out.store(dh + off + ch[i].at);
      }
  }
  // The groups' sums, dw's and then db's, through the same LDS.
  float* const mine = part + (int64_t)blockIdx.x * 2 * dim;
  auto put = [&](const float (&acc)[VPL][W], float* dst) {
    float* const to = kGroups > 1 ? red + grp * dim : dst;
#pragma unroll
    for (int i = 0; i < VPL; ++i)
      if (ch[i].on)
#pragma unroll
        for (int e = 0; e < W; ++e)
          if (e >= ch[i].skip) to[ch[i].at + e] = acc[i][e];
    if constexpr (kGroups > 1) {
      __syncthreads();
      for (int col = threadIdx.x; col < dim; col += blockDim.x) {
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < kGroups; ++k) s += red[k * dim + col];
        dst[col] = s;
      }
      __syncthreads();
    }
  };
  put(dw, mine);
  put(db, mine + dim);
}

// The same for the rows that no group takes: sweeps for dh, then a thread to a column for the partial rows. A row's mean as it is stored is
// rounded; the sweep leaves the mean of the differences from it in rests, so that both take the same n.
template <typename TX, typename TW, bool DIRECT>
__global__ __launch_bounds__(256) void layernorm_bwd_sweep_kernel(const TX* __restrict__ h, const TW* __restrict__ w,
                                                                  const TX* __restrict__ dy, const TX* __restrict__ dd,
                                                                  const float* __restrict__ stats, TX* __restrict__ dh,
                                                                  float* __restrict__ rests, int64_t rows, int64_t dim,
                                                                  float inv_dim) {
  __shared__ float lds[2][16];
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const int64_t off = row * dim;
    const float mean = stats[2 * row], rs = stats[2 * row + 1];
    float rest = 0.f, sg = 0.f, sgc = 0.f, none = 0.f;
    for (int64_t e = threadIdx.x; e < dim; e += 256) {
      const float c = Elem<TX>::to_f32(h[off + e]) - mean, g = Elem<TX>::to_f32(dy[off + e]) * Elem<TW>::to_f32(w[e]);
      rest += c;
      sg += g;
      sgc += g * c;
    }
    rows_sum<256>(rest, sg, lds);
    rows_sum<256>(sgc, none, lds);
    rest *= inv_dim;
    if (threadIdx.x == 0) rests[row] = rest;
    const float mg = sg * inv_dim, mgn = (sgc - rest * sg) * inv_dim * rs;
    for (int64_t e = threadIdx.x; e < dim; e += 256) {
      const float n = (Elem<TX>::to_f32(h[off + e]) - mean - rest) * rs;
      float o = rs * (Elem<TX>::to_f32(dy[off + e]) * Elem<TW>::to_f32(w[e]) - mg - n * mgn);
      if constexpr (DIRECT) o += Elem<TX>::to_f32(dd[off + e]);
      dh[off + e] = Elem<TX>::from_f32(o);
    }
  }
}
template <typename TX>
__global__ __launch_bounds__(256) void layernorm_bwd_cols_kernel(const TX* __restrict__ h, const TX* __restrict__ dy,
                                                                 const float* __restrict__ stats,
                                                                 const float* __restrict__ rests,
                                                                 float* __restrict__ part, int64_t rows, int64_t dim) {
  const int64_t col = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (col >= dim) return;
  float dw = 0.f, db = 0.f;
  for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
    const float g = Elem<TX>::to_f32(dy[r * dim + col]);
    dw += g * ((Elem<TX>::to_f32(h[r * dim + col]) - stats[2 * r] - rests[r]) * stats[2 * r + 1]);
    db += g;
  }
  part[(int64_t)blockIdx.y * 2 * dim + col] = dw;
  part[((int64_t)blockIdx.y * 2 + 1) * dim + col] = db;
}

// Partial rows: one to a CU, and two where the columns are few and the rows many; a row to a group at least. More of them cost more
// than they bring. us, one / two to a CU: 8192 x 768 bf16 17.1 / 17.4, 32768 x 512 36 / 30, 8192 x 2048 33.3 / 40.7;
// 64 x 768 in 16 groups of four rows 9.5, of one 6.8.
int bwd_parts(int64_t rows, int64_t dim, const NormPlan& plan) {
  const int64_t groups = plan.group == 64 ? 4 : 1;
  const int64_t one = std::min<int64_t>(cdiv(rows, groups), kBwdParts / 2);
  return (int)std::max<int64_t>(one, dim <= 1024 ? std::min<int64_t>(cdiv(rows, groups * 8), kBwdParts) : 1);
}

template <typename TX, typename TW, bool DIRECT>
int norm_bwd_launch(const TX* h, const TW* w, const TX* dy, const TX* dd, const float* stats, TX* dh, TW* dw, TW* db,
                    float* part, int64_t rows, int64_t dim, hipStream_t stream) {
  const float inv_dim = (float)(1.0 / (double)dim);
  const NormPlan plan = norm_plan(dim);
  const int parts = rows ? bwd_parts(rows, dim, plan) : 0;
  if (rows && plan.group) {
    FERRITE_NORM_CASE(plan, const size_t lds = G < 256 ? (size_t)(256 / G) * dim * 4 : 0;
                      hipLaunchKernelGGL((layernorm_bwd_kernel<TX, TW, DIRECT, W, VPL, G>), dim3((unsigned)parts),
                                         dim3(G < 256 ? 256 : G), lds, stream, h, w, dy, dd, stats, dh, part, rows, (int)dim,
                                         inv_dim));
  } else if (rows) {
    float* const rests = part + (int64_t)parts * 2 * dim;
    hipLaunchKernelGGL((layernorm_bwd_sweep_kernel<TX, TW, DIRECT>), dim3((unsigned)std::min<int64_t>(rows, 1 << 20)),
                       dim3(256), 0, stream, h, w, dy, dd, stats, dh, rests, rows, dim, inv_dim);
    hipLaunchKernelGGL((layernorm_bwd_cols_kernel<TX>), dim3((unsigned)cdiv(dim, 256), (unsigned)parts), dim3(256), 0, stream,
                       h, dy, stats, rests, part, rows, dim);
  }
  join_parts(part, dw, db, 2, parts, dim, stream);
  return check_launch("ferrite_layernorm_bwd");
}

// Rows and columns that the grids, the 32-bit widths and the 64-bit offsets hold.
bool norm_ok(int64_t rows, int64_t dim) {
  return rows >= 0 && dim >= 1 && dim <= 0x7fffffff / 64 && (rows == 0 || rows <= ((int64_t)1 << 60) / dim);
}

template <typename F>
int with_types(int x_dtype, int w_dtype, F&& f) {
  if (x_dtype == FERRITE_BF16) return w_dtype == FERRITE_BF16 ? f((bf16*)nullptr, (bf16*)nullptr) : f((bf16*)nullptr, (float*)nullptr);
  return w_dtype == FERRITE_BF16 ? f((float*)nullptr, (bf16*)nullptr) : f((float*)nullptr, (float*)nullptr);
}

}  // namespace
}  // namespace ferrite

extern "C" int ferrite_internal_layernorm(const void* x, const void* r, const void* w, const void* b, void* h, void* y,
                                          float* stats, int64_t rows, int64_t dim, int x_dtype, int w_dtype, float eps,
                                          void* stream) {
  using namespace ferrite;
  if (!valid_dtype(x_dtype) || !valid_dtype(w_dtype))
    return fail(FERRITE_ERR_INVALID_ARGUMENT, "ferrite_layernorm: dtype must be FERRITE_F32 or FERRITE_BF16");
  if (!norm_ok(rows, dim)) return fail(FERRITE_ERR_INVALID_ARGUMENT, "ferrite_layernorm: need rows >= 0 and 1 <= dim < 2^25");
  if (rows == 0) return FERRITE_OK;
  if (!x || !w || !y || (r && !h)) return fail(FERRITE_ERR_INVALID_ARGUMENT, "ferrite_layernorm: null pointer");
  hipStream_t s = static_cast<hipStream_t>(stream);
  return with_types(x_dtype, w_dtype, [&](auto* tx, auto* tw) {
    typedef std::remove_pointer_t<decltype(tx)> TX;
    typedef std::remove_pointer_t<decltype(tw)> TW;
    auto go = [&](auto residual) {
      return norm_launch<TX, TW, decltype(residual)::value != 0>(
          static_cast<const TX*>(x), static_cast<const TX*>(r), static_cast<const TW*>(w), static_cast<const TW*>(b),
          static_cast<TX*>(h), static_cast<TX*>(y), stats, rows, dim, eps, s);
    };
    return r ? go(Int<1>()) : go(Int<0>());
  });
}

extern "C" int64_t ferrite_internal_layernorm_bwd_workspace(int64_t rows, int64_t dim) {
  using namespace ferrite;
  if (!norm_ok(rows, dim)) return -1;
  const NormPlan plan = norm_plan(dim);
  return rows ? ((int64_t)bwd_parts(rows, dim, plan) * 2 * dim + (plan.group ? 0 : rows)) * 4 : 0;
}

extern "C" int ferrite_internal_layernorm_bwd(const void* h, const void* w, const void* dy, const void* dd,
                                              const float* stats, void* dh, void* dw, void* db, int64_t rows, int64_t dim,
                                              int x_dtype, int w_dtype, void* workspace, int64_t workspace_bytes,
                                              void* stream) {
  using namespace ferrite;
  if (!valid_dtype(x_dtype) || !valid_dtype(w_dtype))
    return fail(FERRITE_ERR_INVALID_ARGUMENT, "ferrite_layernorm_bwd: dtype must be FERRITE_F32 or FERRITE_BF16");
  const int64_t need = ferrite_internal_layernorm_bwd_workspace(rows, dim);
  if (need < 0)
    return fail(FERRITE_ERR_INVALID_ARGUMENT, "ferrite_layernorm_bwd: need rows >= 0 and 1 <= dim < 2^25");
  if (!dw || (rows && (!h || !w || !dy || !stats || !dh)))
    return fail(FERRITE_ERR_INVALID_ARGUMENT, "ferrite_layernorm_bwd: null pointer");
  if (need && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 3)))
    return fail(FERRITE_ERR_INVALID_ARGUMENT, "ferrite_layernorm_bwd: workspace too small");
  hipStream_t s = static_cast<hipStream_t>(stream);
  return with_types(x_dtype, w_dtype, [&](auto* tx, auto* tw) {
    typedef std::remove_pointer_t<decltype(tx)> TX;
    typedef std::remove_pointer_t<decltype(tw)> TW;
    auto go = [&](auto direct) {
      return norm_bwd_launch<TX, TW, decltype(direct)::value != 0>(
          static_cast<const TX*>(h), static_cast<const TW*>(w), static_cast<const TX*>(dy), static_cast<const TX*>(dd), stats,
          static_cast<TX*>(dh), static_cast<TW*>(dw), static_cast<TW*>(db), static_cast<float*>(workspace), rows, dim, s);
    };
    return dd ? go(Int<1>()) : go(Int<0>());
  });
}
