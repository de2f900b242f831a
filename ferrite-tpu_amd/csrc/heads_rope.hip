// Heads of a fused projection, split, normed and rotated in one pass, for gfx950.
//
// qkv [B, S, (H + 2 Hkv) D] holds a token's heads as (q | k | v, head, dim) (the columns of
// model/gpt.py:137). Forward, for every q and k head x of D values at position p:
//   r = rsqrt(mean(x^2) + eps);  u = x r w;  y = rotation of u by the angles of p
// where the rotation turns the pairs (i, i + R/2), or (2 i, 2 i + 1) when interleaved, of the first
// R values: (lo, hi) -> (lo c - hi s, hi c + lo s), c and s from tables [positions, R/2]. v heads are
// moved as they are. Outputs are head-major, q [B, H, S, D], k and v [B, Hkv, S, D], what the
// attention kernels read. Backward, with r formed again from the projection (no statistics kept):
//   du = rotation by the negative angles of dy;  dx = r (du w - x r^2 mean(du w x));  dw = sum du x r
// All of it in f32, rounded once where it is stored.
#include <math.h>

#include <algorithm>

#include "common.h"
#include "internal_api.h"

namespace ferrite {
namespace {

// A head is cut into units of two vectors of V elements: the lo and the hi values of V pairs
// (adjacent vectors when interleaved), so a lane holds both halves of its pairs and the rotation
// needs no lane but its own. L lanes (a power of two) with N units each hold a head; the 64 / L
// lane groups of a wave take consecutive tokens and walk over the same heads, so that every
// token's angles are read once for a chunk of heads, a wave's stores of one head are one
// contiguous stretch of the output, and whether a head is of q, k or v is uniform.
//
// Heads of a wave at most: one reading of the angles for all of them. Backward, 8192 tokens of 12 + 12 + 12 heads of 64: 24.3 us
// with 8, 27.0 with 4, 25.8 with 12, 26.4 with 16.
constexpr int kChunk = 8;

struct HeadsArgs {
  const void* qkv;
  int64_t batch_stride, row_stride;  // of qkv, in elements
  const void *wq, *wk;
  const float *cos, *sin;
  const int32_t* pos;  // [B, S], or null: position s
  void *q, *k, *v;     // forward's outputs, or their gradients [B, heads, S, D] (null: zero)
  void* dqkv;          // backward: dense [B, S, (H + 2 Hkv) D]
  float* part;         // backward: partial weight gradients [chunk, block][D]
  int64_t tokens;
  int S, H, Hkv, D, R, P, chunk;
  float eps;
  int w_bf16;
};

// What chunk `c` of heads holds: kind 0 q, 1 k, 2 v, and heads [from, to) of that kind.
struct Chunk {
  int kind, from, to;
};
__device__ __forceinline__ Chunk chunk_of(const HeadsArgs& a, int c) {
  const int nq = (a.H + a.chunk - 1) / a.chunk, nk = (a.Hkv + a.chunk - 1) / a.chunk;
  const int kind = c < nq ? 0 : c < nq + nk ? 1 : 2;
  const int at = (kind == 0 ? c : kind == 1 ? c - nq : c - nq - nk) * a.chunk;
  return {kind, at, min(at + a.chunk, kind == 0 ? a.H : a.Hkv)};
}

template <typename T, int V>
struct RawOf {
  typedef u32x4 type;
};
template <>
struct RawOf<float, 1> {
  typedef float type;
};
template <>
struct RawOf<bf16, 1> {
  typedef bf16 type;
};

template <typename T, int V>
__device__ __forceinline__ float elem(const typename RawOf<T, V>::type& raw, int e) {
  if constexpr (V == 1)
    return Elem<T>::to_f32(raw);
  else if constexpr (sizeof(T) == 2)
    return (float)__builtin_bit_cast(bf16x8, raw)[e];
  else
    return __builtin_bit_cast(f32x4, raw)[e];
}

template <typename T, int V, bool INTER>
struct Unit {
  typedef typename RawOf<T, V>::type raw_t;
  int lo, hi;  // element offsets of the two vectors
  bool on, turned;
  int angle;  // index of the first pair's angle

  __device__ __forceinline__ void set(int u, int D, int R) {
    on = 2 * u * V < D;
    turned = 2 * u * V < R;
    angle = u * V;
    if (INTER) {
      lo = 2 * u * V;
      hi = lo + V;
    } else if (turned) {
      lo = u * V;
      hi = R / 2 + u * V;
    } else {
      lo = R / 2 + u * V;  // R + (u - R / (2 V)) V
      hi = D / 2 + u * V;  // (D - R) / 2 further
    }
  }
  // The V pairs of two vectors as floats, and back.
  static __device__ __forceinline__ void pairs(const raw_t& A, const raw_t& B, float* a, float* b) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      if (INTER && V > 1) {
        a[e] = e < V / 2 ? elem<T, V>(A, 2 * e) : elem<T, V>(B, 2 * e - V);
        b[e] = e < V / 2 ? elem<T, V>(A, 2 * e + 1) : elem<T, V>(B, 2 * e + 1 - V);
      } else {
        a[e] = elem<T, V>(A, e);
        b[e] = elem<T, V>(B, e);
      }
    }
  }
  static __device__ __forceinline__ raw_t pack(const float* f) {
    if constexpr (V == 1) {
      return Elem<T>::from_f32(f[0]);
    } else if constexpr (sizeof(T) == 2) {
      return u32x4{pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7])};
    } else {
      return __builtin_bit_cast(u32x4, f32x4{f[0], f[1], f[2], f[3]});
    }
  }
  static __device__ __forceinline__ void vectors(const float* a, const float* b, raw_t& A, raw_t& B) {
    if constexpr (INTER && V > 1) {
      float f[2 * V];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        f[2 * e] = a[e];
        f[2 * e + 1] = b[e];
      }
      A = pack(f);
      B = pack(f + V);
    } else {
      A = pack(a);
      B = pack(b);
    }
  }
};

// Floats [V] at index i of a table of floats.
template <int V>
__device__ __forceinline__ void load_floats(const float* p, float* out) {
  if constexpr (V == 1) {
    out[0] = *p;
  } else {
#pragma unroll
    for (int e = 0; e < V; e += 4) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(p + e);
#pragma unroll
      for (int i = 0; i < 4; ++i) out[e + i] = x[i];
    }
  }
}

// The angles of a lane's unit at position p: outside the table NaN, past the rotated values 1 and 0.
template <typename T, int V, bool INTER>
__device__ __forceinline__ void angles(const HeadsArgs& a, const Unit<T, V, INTER>& u, int p, float* c, float* s) {
  const bool known = p >= 0 && p < a.P;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    c[e] = known ? 1.f : NAN;
    s[e] = known ? 0.f : NAN;
  }
  if (known && u.on && u.turned) {
    load_floats<V>(a.cos + (int64_t)p * (a.R / 2) + u.angle, c);
    load_floats<V>(a.sin + (int64_t)p * (a.R / 2) + u.angle, s);
  }
}

// V weights at index i, of w's type.
template <int V>
__device__ __forceinline__ void load_weights(const HeadsArgs& a, const void* w, int i, float* out) {
  if (!a.w_bf16) {
    load_floats<V>(static_cast<const float*>(w) + i, out);
  } else if constexpr (V == 1) {
    out[0] = (float)static_cast<const bf16*>(w)[i];
  } else {
    typedef bf16 __attribute__((ext_vector_type(V))) vec;
    const vec x = *reinterpret_cast<const vec*>(static_cast<const bf16*>(w) + i);
#pragma unroll
    for (int e = 0; e < V; ++e) out[e] = (float)x[e];
  }
}
// The weights of a lane's pairs.
template <typename T, int V, bool INTER>
__device__ __forceinline__ void weights(const HeadsArgs& a, const Unit<T, V, INTER>& u, const void* w, float* lo, float* hi) {
  float x[2][V] = {};
  if (u.on) {
    load_weights<V>(a, w, u.lo, x[0]);
    load_weights<V>(a, w, u.hi, x[1]);
  }
#pragma unroll
  for (int e = 0; e < V; ++e) {
    lo[e] = INTER && V > 1 ? x[2 * e / V][2 * e % V] : x[0][e];
    hi[e] = INTER && V > 1 ? x[(2 * e + 1) / V][(2 * e + 1) % V] : x[1][e];
  }
}

template <int L>
__device__ __forceinline__ float group_sum(float x) {
#pragma unroll
  for (int off = 1; off < L; off <<= 1) x += __shfl_xor(x, off, kWave);
  return x;
}

// grid (blocks of 4 waves of 64 / L tokens, chunks of heads). Bound by HBM: every element is read and written once. 8191 tokens
// of 32 + 8 + 8 heads of 128, bf16: 34.2 us, 6.0 TB/s (heads two or four at a time, for more bytes under way, 37.3 and 40.9: the
// registers that they take cost more waves than they gain loads). 8192 tokens of 12 + 12 + 12 heads of 64: 17.0 us, 4.4 TB/s.
template <typename T, int V, int L, int N, bool INTER>
__global__ __launch_bounds__(256) void heads_rope_kernel(HeadsArgs a) {
  typedef Unit<T, V, INTER> U;
  typedef typename U::raw_t raw_t;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t token = ((int64_t)blockIdx.x * 4 + wave) * (64 / L) + lane / L;
  const Chunk ch = chunk_of(a, blockIdx.y);
  const bool here = token < a.tokens;
  const int64_t b = here ? token / a.S : 0;
  const int s = here ? (int)(token - b * a.S) : 0;
  U u[N];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    u[n].set(lane % L + n * L, a.D, a.R);
    u[n].on = u[n].on && here;
  }
  const int base = ch.kind == 0 ? 0 : ch.kind == 1 ? a.H : a.H + a.Hkv, heads = ch.kind == 0 ? a.H : a.Hkv;
  const T* src = static_cast<const T*>(a.qkv) + b * a.batch_stride + s * a.row_stride + (int64_t)base * a.D;
  T* dst = static_cast<T*>(ch.kind == 0 ? a.q : ch.kind == 1 ? a.k : a.v) + (b * heads * a.S + s) * a.D;
  const int64_t head_step = (int64_t)a.S * a.D;

  float c[N][V], sn[N][V], wl[N][V], wh[N][V];
  if (ch.kind < 2) {
    const int p = a.pos ? (here ? a.pos[token] : 0) : s;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      angles(a, u[n], p, c[n], sn[n]);
      weights(a, u[n], ch.kind == 0 ? a.wq : a.wk, wl[n], wh[n]);
    }
  }
  for (int h = ch.from; h < ch.to; ++h) {
    raw_t A[N], B[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      if (!u[n].on) continue;
      const T* p = src + (int64_t)h * a.D;
      A[n] = *reinterpret_cast<const raw_t*>(p + u[n].lo);
      B[n] = *reinterpret_cast<const raw_t*>(p + u[n].hi);
    }
    if (ch.kind < 2) {
      float lo[N][V], hi[N][V], ss = 0.f;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        if (!u[n].on) continue;
        U::pairs(A[n], B[n], lo[n], hi[n]);
#pragma unroll
        for (int e = 0; e < V; ++e) ss += lo[n][e] * lo[n][e] + hi[n][e] * hi[n][e];
      }
      const float r = rsqrtf(group_sum<L>(ss) / (float)a.D + a.eps);
#pragma unroll
      for (int n = 0; n < N; ++n) {
        if (!u[n].on) continue;
        float yl[V], yh[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float ul = lo[n][e] * r * wl[n][e], uh = hi[n][e] * r * wh[n][e];
          yl[e] = ul * c[n][e] - uh * sn[n][e];
          yh[e] = uh * c[n][e] + ul * sn[n][e];
        }
        U::vectors(yl, yh, A[n], B[n]);
      }
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
      if (!u[n].on) continue;
      T* o = dst + h * head_step;
      *reinterpret_cast<raw_t*>(o + u[n].lo) = A[n];
      *reinterpret_cast<raw_t*>(o + u[n].hi) = B[n];
    }
  }
}

// Bound by HBM (reads dq, dk, dv and the projection's q and k, writes the projection's gradient): 8192 tokens of 12 + 12 + 12
// heads of 64, bf16: 22.2 us, 4.5 TB/s, and 3.9 for the weights' sums.
// grid (blocks, chunks); a wave walks over the token groups of its block's stride and keeps its lanes' share of dw
// in registers. The partial sums [chunk, block][D] are added in their order by heads_rope_dw_kernel.
template <typename T, int V, int L, int N, bool INTER>
__global__ __launch_bounds__(256) void heads_rope_bwd_kernel(HeadsArgs a) {
  typedef Unit<T, V, INTER> U;
  typedef typename U::raw_t raw_t;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const Chunk ch = chunk_of(a, blockIdx.y);
  const int base = ch.kind == 0 ? 0 : ch.kind == 1 ? a.H : a.H + a.Hkv, heads = ch.kind == 0 ? a.H : a.Hkv;
  const T* grad = static_cast<const T*>(ch.kind == 0 ? a.q : ch.kind == 1 ? a.k : a.v);
  const int64_t head_step = (int64_t)a.S * a.D, width = (int64_t)(a.H + 2 * a.Hkv) * a.D;
  U u[N];
#pragma unroll
  for (int n = 0; n < N; ++n) u[n].set(lane % L + n * L, a.D, a.R);
  float wl[N][V], wh[N][V], dl[N][V] = {}, dh[N][V] = {};
  if (ch.kind < 2) {
#pragma unroll
    for (int n = 0; n < N; ++n) weights(a, u[n], ch.kind == 0 ? a.wq : a.wk, wl[n], wh[n]);
  }
  const int64_t step = (int64_t)gridDim.x * 4 * (64 / L);
  for (int64_t first = ((int64_t)blockIdx.x * 4 + wave) * (64 / L); first < a.tokens; first += step) {
    const int64_t token = first + lane / L;
    const bool here = token < a.tokens;
    const int64_t b = here ? token / a.S : 0;
    const int s = here ? (int)(token - b * a.S) : 0;
    const T* src = static_cast<const T*>(a.qkv) + b * a.batch_stride + s * a.row_stride + (int64_t)base * a.D;
    const T* gsrc = grad + (b * heads * a.S + s) * a.D;
    T* dst = static_cast<T*>(a.dqkv) + token * width + (int64_t)base * a.D;
    float c[N][V], sn[N][V];
    if (ch.kind < 2) {
      const int p = a.pos ? (here ? a.pos[token] : 0) : s;
#pragma unroll
      for (int n = 0; n < N; ++n) angles(a, u[n], p, c[n], sn[n]);
    }
    for (int h = ch.from; h < ch.to; ++h) {
      raw_t A[N] = {}, B[N] = {}, GA[N] = {}, GB[N] = {};
#pragma unroll
      for (int n = 0; n < N; ++n) {
        if (!u[n].on || !here) continue;
        const T* p = src + (int64_t)h * a.D;
        const T* g = gsrc + h * head_step;
        if (grad) {
          GA[n] = *reinterpret_cast<const raw_t*>(g + u[n].lo);
          GB[n] = *reinterpret_cast<const raw_t*>(g + u[n].hi);
        }
        if (ch.kind < 2) {
          A[n] = *reinterpret_cast<const raw_t*>(p + u[n].lo);
          B[n] = *reinterpret_cast<const raw_t*>(p + u[n].hi);
        }
      }
      if (ch.kind < 2) {
        float lo[N][V], hi[N][V], ul[N][V], uh[N][V], ss = 0.f, st = 0.f;
#pragma unroll
        for (int n = 0; n < N; ++n) {
          if (!u[n].on || !here) continue;
          float gl[V], gh[V];
          U::pairs(A[n], B[n], lo[n], hi[n]);
          U::pairs(GA[n], GB[n], gl, gh);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            ul[n][e] = gl[e] * c[n][e] + gh[e] * sn[n][e];
            uh[n][e] = gh[e] * c[n][e] - gl[e] * sn[n][e];
            ss += lo[n][e] * lo[n][e] + hi[n][e] * hi[n][e];
            st += ul[n][e] * wl[n][e] * lo[n][e] + uh[n][e] * wh[n][e] * hi[n][e];
          }
        }
        const float r = rsqrtf(group_sum<L>(ss) / (float)a.D + a.eps);
        const float t = group_sum<L>(st) / (float)a.D * r * r;
#pragma unroll
        for (int n = 0; n < N; ++n) {
          if (!u[n].on || !here) continue;
          float xl[V], xh[V];
#pragma unroll
          for (int e = 0; e < V; ++e) {
            dl[n][e] += ul[n][e] * lo[n][e] * r;
            dh[n][e] += uh[n][e] * hi[n][e] * r;
            xl[e] = r * (ul[n][e] * wl[n][e] - lo[n][e] * t);
            xh[e] = r * (uh[n][e] * wh[n][e] - hi[n][e] * t);
          }
          U::vectors(xl, xh, GA[n], GB[n]);
        }
      }
#pragma unroll
      for (int n = 0; n < N; ++n) {
        if (!u[n].on || !here) continue;
        T* o = dst + (int64_t)h * a.D;
        *reinterpret_cast<raw_t*>(o + u[n].lo) = GA[n];
        *reinterpret_cast<raw_t*>(o + u[n].hi) = GB[n];
      }
    }
  }
  if (ch.kind == 2) return;
  // The wave's groups by shuffles, then the waves in their order.
  __shared__ float red[4][2 * V * N * L];
#pragma unroll
  for (int n = 0; n < N; ++n) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
#pragma unroll
      for (int off = L; off < 64; off <<= 1) {
        dl[n][e] += __shfl_xor(dl[n][e], off, kWave);
        dh[n][e] += __shfl_xor(dh[n][e], off, kWave);
      }
      if (lane < L && u[n].on) {
        red[wave][INTER ? u[n].lo + 2 * e : u[n].lo + e] = dl[n][e];
        red[wave][INTER ? u[n].lo + 2 * e + 1 : u[n].hi + e] = dh[n][e];
      }
    }
  }
  __syncthreads();
  float* part = a.part + ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * a.D;
  for (int d = threadIdx.x; d < a.D; d += 256) part[d] = red[0][d] + red[1][d] + red[2][d] + red[3][d];
}

// dw[d] of q (blockIdx.y 0: partial rows [0, nq)) or k (1: [nq, nq + nk)), 16 columns to a block of 64 row slices.
constexpr int kDwCols = 16, kDwSlices = 64;
__global__ __launch_bounds__(1024) void heads_rope_dw_kernel(const float* __restrict__ part, void* dwq, void* dwk,
                                                             int64_t nq, int64_t nk, int D, int w_bf16) {
  __shared__ float red[kDwSlices][kDwCols];
  const int col = threadIdx.x % kDwCols, slice = threadIdx.x / kDwCols, d = (int)blockIdx.x * kDwCols + col;
  const int64_t rows = blockIdx.y ? nk : nq;
  const float* src = part + (blockIdx.y ? nq * D : 0);
  float s = 0.f;
  if (d < D) {
    for (int64_t r = slice; r < rows; r += kDwSlices) s += src[r * D + d];
  }
  red[slice][col] = s;
  __syncthreads();
  for (int n = kDwSlices / 2; n > 0; n /= 2) {
    if (slice < n) red[slice][col] += red[slice + n][col];
    __syncthreads();
  }
  if (slice == 0 && d < D) {
    void* out = blockIdx.y ? dwk : dwq;
    if (w_bf16)
      static_cast<bf16*>(out)[d] = (bf16)red[0][col];
    else
      static_cast<float*>(out)[d] = red[0][col];
  }
}

constexpr int kMaxD = 512;
constexpr int64_t kMostBlocks = 0xffffffff / 256;  // blocks of 256 threads: a launch has under 2^32 threads along x

// Vectors of 16 bytes where the sizes and addresses are whole in them, else elements.
template <typename T, bool INTER, typename F>
int with_layout(bool vec, int D, F&& go) {
  constexpr int V = 16 / (int)sizeof(T);
#define FERRITE_HEADS(LANES) \
  if (D <= 2 * V * LANES) return go(std::integral_constant<int, V>{}, std::integral_constant<int, LANES>{}, std::integral_constant<int, 1>{})
  if (vec) {
    FERRITE_HEADS(2);
    FERRITE_HEADS(4);
    FERRITE_HEADS(8);
    FERRITE_HEADS(16);
    FERRITE_HEADS(32);
    if constexpr (sizeof(T) == 4) FERRITE_HEADS(64);
  }
#undef FERRITE_HEADS
  if (D <= 128)
    return go(std::integral_constant<int, 1>{}, std::integral_constant<int, 16>{}, std::integral_constant<int, 4>{});
  return go(std::integral_constant<int, 1>{}, std::integral_constant<int, 64>{}, std::integral_constant<int, 4>{});
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

bool vectors_fit(const HeadsArgs& a, int esize) {
  const int v = 16 / esize;
  return a.D % (2 * v) == 0 && a.R % (2 * v) == 0 && a.row_stride % v == 0 && a.batch_stride % v == 0 &&
         aligned16(a.qkv) && aligned16(a.q) && aligned16(a.k) && aligned16(a.v) && aligned16(a.cos) && aligned16(a.sin) &&
         aligned16(a.dqkv) && aligned16(a.wq) && aligned16(a.wk);
}

int chunks_of(const HeadsArgs& a) { return (int)(cdiv(a.H, a.chunk) + 2 * cdiv(a.Hkv, a.chunk)); }

// Tokens to a wave are at most 32; with few tokens a wave takes a head or two, so that the heads spread over the CUs. The forward
// kernel's us with 1, 2 and kChunk heads, in turn with the backward, whose data is in the caches: 512 tokens of 36 heads of 64 3.8, 4.4,
// 6.7, 2048 of them 6.0, 6.2, 8.4, 4096 8.7, 8.4, 9.4; 8191 of 48 heads of 128 46.8, 42.4, 39.0 (34.2 with no backward between). The
// heads of one kind are cut evenly.
void set_chunk(HeadsArgs& a) {
  const int64_t all = a.tokens * (a.H + 2 * a.Hkv);
  const int most = all < 32768 ? 1 : all < 196608 ? 2 : kChunk, heads = std::max(a.H, a.Hkv);
  a.chunk = (int)cdiv(heads, cdiv(heads, (int64_t)most));
}

// Blocks along the tokens of the backward: some eight waves a SIMD over all chunks, their groups of tokens (4 waves of 64 / L
// tokens) dealt evenly.
int64_t most_blocks(int64_t tokens, int64_t chunks) {
  return std::max<int64_t>(1, std::min<int64_t>(2048 / chunks, cdiv(tokens, (int64_t)4)));  // a wave takes a token or more
}
int64_t bwd_blocks(int64_t tokens, int64_t chunks, int per_block) {
  const int64_t groups = cdiv(tokens, (int64_t)per_block);
  return cdiv(groups, cdiv(groups, most_blocks(tokens, chunks)));
}

int check_heads(const char* name, int64_t b, int64_t s, int64_t h, int64_t hkv, int64_t d, int64_t rot, int64_t table,
                int dtype, int w_dtype) {
  const std::string n(name);
  if (!valid_dtype(dtype) || !valid_dtype(w_dtype))
    return fail(FERRITE_ERR_INVALID_ARGUMENT, n + ": dtype must be FERRITE_F32 or FERRITE_BF16");
  if (b < 0 || s < 0 || h < 1 || hkv < 1 || h > 16384 || hkv > 16384 || b > 0x7fffffff || s > 0x7fffffff ||
      b * s > 0x7fffffff)
    return fail(FERRITE_ERR_INVALID_ARGUMENT, n + ": need 1 <= heads <= 16384 and under 2^31 tokens");
  if (d < 2 || d > kMaxD || d % 2 || rot < 0 || rot > d || rot % 2)
    return fail(FERRITE_ERR_INVALID_ARGUMENT, n + ": the head dim must be even and at most 512, the rotated part even and within it");
  if (table < 1 || table > 0x7fffffff) return fail(FERRITE_ERR_INVALID_ARGUMENT, n + ": empty angle tables");
  return FERRITE_OK;
}

}  // namespace
}  // namespace ferrite

extern "C" int ferrite_internal_heads_rope(const void* qkv, int64_t batch_stride, int64_t row_stride, const void* wq,
                                           const void* wk, const float* cos, const float* sin, const int32_t* pos,
                                           void* q, void* k, void* v, int64_t b, int64_t s, int64_t h, int64_t hkv,
                                           int64_t d, int64_t rot, int64_t table, int dtype, int w_dtype,
                                           int interleaved, float eps, void* stream) {
  using namespace ferrite;
  const int rc = check_heads("ferrite_heads_rope", b, s, h, hkv, d, rot, table, dtype, w_dtype);
  if (rc != FERRITE_OK) return rc;
  if (b * s == 0) return FERRITE_OK;
  if (!qkv || !wq || !wk || (rot && (!cos || !sin)) || !q || !k || !v)
    return fail(FERRITE_ERR_INVALID_ARGUMENT, "ferrite_heads_rope: null pointer");
  HeadsArgs a{qkv, batch_stride, row_stride, wq, wk, cos, sin, pos, q, k, v, nullptr, nullptr, b * s,
              (int)s, (int)h, (int)hkv, (int)d, (int)rot, (int)table, 0, eps, w_dtype == FERRITE_BF16};
  set_chunk(a);
  hipStream_t st = static_cast<hipStream_t>(stream);
  auto launch = [&](auto* t, auto inter) {
    typedef std::remove_pointer_t<decltype(t)> T;
    return with_layout<T, inter.value>(vectors_fit(a, sizeof(T)), a.D, [&](auto V, auto L, auto N) {
      const int64_t blocks = cdiv(a.tokens, 4 * (64 / L.value));
      if (blocks > kMostBlocks) return fail(FERRITE_ERR_INVALID_ARGUMENT, "ferrite_heads_rope: too many tokens");
      const dim3 grid((unsigned)blocks, (unsigned)chunks_of(a));
      hipLaunchKernelGGL((heads_rope_kernel<T, V.value, L.value, N.value, inter.value>), grid, dim3(256), 0, st, a);
      return check_launch("ferrite_heads_rope");
    });
  };
  if (dtype == FERRITE_BF16)
    return interleaved ? launch((bf16*)nullptr, std::true_type{}) : launch((bf16*)nullptr, std::false_type{});
  return interleaved ? launch((float*)nullptr, std::true_type{}) : launch((float*)nullptr, std::false_type{});
}

extern "C" int64_t ferrite_internal_heads_rope_bwd_workspace(int64_t b, int64_t s, int64_t h, int64_t hkv, int64_t d) {
  using namespace ferrite;
  if (check_heads("ferrite_heads_rope_bwd", b, s, h, hkv, d, 0, 1, FERRITE_F32, FERRITE_F32) != FERRITE_OK) return -1;
  HeadsArgs a{};
  a.tokens = b * s;
  a.H = (int)h;
  a.Hkv = (int)hkv;
  set_chunk(a);
  const int64_t chunks = chunks_of(a), kept = cdiv(a.H, a.chunk) + cdiv(a.Hkv, a.chunk);
  return kept * most_blocks(a.tokens, chunks) * d * (int64_t)sizeof(float);
}

extern "C" int ferrite_internal_heads_rope_bwd(const void* qkv, int64_t batch_stride, int64_t row_stride,
                                               const void* wq, const void* wk, const float* cos, const float* sin,
                                               const int32_t* pos, const void* dq, const void* dk, const void* dv,
                                               void* dqkv, void* dwq, void* dwk, int64_t b, int64_t s, int64_t h,
                                               int64_t hkv, int64_t d, int64_t rot, int64_t table, int dtype,
                                               int w_dtype, int interleaved, float eps, void* workspace,
                                               int64_t workspace_bytes, void* stream) {
  using namespace ferrite;
  const int rc = check_heads("ferrite_heads_rope_bwd", b, s, h, hkv, d, rot, table, dtype, w_dtype);
  if (rc != FERRITE_OK) return rc;
  if (!wq || !wk || !dwq || !dwk || (b * s && (!qkv || (rot && (!cos || !sin)) || !dqkv)))
    return fail(FERRITE_ERR_INVALID_ARGUMENT, "ferrite_heads_rope_bwd: null pointer");
  if (b * s && (!workspace || workspace_bytes < ferrite_internal_heads_rope_bwd_workspace(b, s, h, hkv, d)))
    return fail(FERRITE_ERR_INVALID_ARGUMENT, "ferrite_heads_rope_bwd: workspace too small");
  HeadsArgs a{qkv, batch_stride, row_stride, wq, wk, cos, sin, pos, const_cast<void*>(dq), const_cast<void*>(dk),
              const_cast<void*>(dv), dqkv, static_cast<float*>(workspace), b * s, (int)s, (int)h, (int)hkv, (int)d,
              (int)rot, (int)table, 0, eps, w_dtype == FERRITE_BF16};
  set_chunk(a);
  const int64_t chunks = chunks_of(a);
  int64_t blocks = 0;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (a.tokens) {
    auto launch = [&](auto* t, auto inter) {
      typedef std::remove_pointer_t<decltype(t)> T;
      return with_layout<T, inter.value>(vectors_fit(a, sizeof(T)), a.D, [&](auto V, auto L, auto N) {
        blocks = bwd_blocks(a.tokens, chunks, 4 * (64 / L.value));
        hipLaunchKernelGGL((heads_rope_bwd_kernel<T, V.value, L.value, N.value, inter.value>),
                           dim3((unsigned)blocks, (unsigned)chunks), dim3(256), 0, st, a);
        return check_launch("ferrite_heads_rope_bwd");
      });
    };
    const int done = dtype == FERRITE_BF16
                         ? (interleaved ? launch((bf16*)nullptr, std::true_type{}) : launch((bf16*)nullptr, std::false_type{}))
                         : (interleaved ? launch((float*)nullptr, std::true_type{}) : launch((float*)nullptr, std::false_type{}));
    if (done != FERRITE_OK) return done;
  }
  hipLaunchKernelGGL(heads_rope_dw_kernel, dim3((unsigned)cdiv(d, (int64_t)kDwCols), 2), dim3(1024), 0, st,
                     static_cast<const float*>(workspace), dwq, dwk, blocks * cdiv(h, (int64_t)a.chunk),
                     blocks * cdiv(hkv, (int64_t)a.chunk), (int)d, a.w_bf16);
  return check_launch("ferrite_heads_rope_bwd");
}
