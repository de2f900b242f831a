// Attention of a tree of drafted tokens over a static KV cache, for gfx950.
//
// Reference: src/ferrite/serving/engine.py:89-104 (_cache_attention, _write_cache), which attends one token
// per sequence; here T <= 64 of them, node t of sequence b hanging on node parents[b, t] < t (or on the
// committed tokens, -1):
//   out[t] = softmax(scale q[t] K^T) V  over the cached rows 0 .. pos - 1, the node's ancestors and itself,
// and the nodes' keys and values are written to the cache's rows pos + t. H = G Hkv query heads share Hkv
// key heads: the G T query rows of one key head are one operand, so each cached row is read once for
// all of them.
//
// Bound by reading the cache while G T is up to some tens of rows. Nothing goes through LDS on the way: a wave owns a
// stretch of the keys and computes scores transposed, S^T = K Q^T (16x16 matrix instructions: a lane
// holds keys 4 g .. 4 g + 3 of one query, g = lane / 16), whose accumulator layout is the layout of
// the second product's B operand, O^T = V^T P^T, when that one's k index runs over the keys in the same order. A lane
// loads V of its own keys, 1/16 of a row each, whole rows to the 16 lanes of a group; output row i of
// product j stands for element i D / 16 + j, so the A operands are those loads transposed in registers.
#include <math.h>

#include <algorithm>

#include "common.h"
#include "internal_api.h"

namespace ferrite {
namespace {

constexpr int kMaxNodes = 64;  // a node per lane of a wave, an ancestor per bit

struct TreeArgs {
  const void *q, *kn, *vn;
  void *kc, *vc;
  const int32_t *pos, *parents;
  void* out;    // [B, T, H, D]
  char* part;   // workspace, or null: one chunk, written to out
  int64_t qs[3], ks[3], vs[3];  // element strides of q, k_new and v_new: sequence, head, node
  int64_t items;                // B Hkv chunks
  int H, Hkv, G, T, L, rows;    // rows = G T
  int chunks, row_blocks, wave_rows;
  float c;  // scale log2(e)
};

__device__ __forceinline__ f32x4 mfma16(const u32x4& a, const u32x4& b, f32x4 acc, bf16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), acc, 0, 0, 0);
}
// Four products of one k each: element e of every lane, so the lanes' 16 bytes cover the same k in both operands.
__device__ __forceinline__ f32x4 mfma16(const u32x4& a, const u32x4& b, f32x4 acc, float) {
  const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
  for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e], acc, 0, 0, 0);
  return acc;
}

// Keys of a step: 16 per score tile, and what one matrix instruction of the second product sums.
template <typename T>
constexpr int kTiles = sizeof(T) == 2 ? 2 : 1;

template <typename T, int D>
struct Step {
  static constexpr int NS = kTiles<T>, KEYS = 16 * NS, RB = D * (int)sizeof(T), KB = RB / 64, VD = RB / 64;
  u32x4 k[NS][KB];           // key 16 n + lane % 16, bytes 64 c + 16 (lane / 16)
  uint32_t v[4 * NS][VD];    // key 16 n + 4 (lane / 16) + i, bytes (lane % 16) RB / 16 ..

  // Rows key0 .. of a head's cache; past the descriptor's range they are zeros.
  __device__ __forceinline__ void load_k(__amdgpu_buffer_rsrc_t rs, int key0, int lane) {
    const uint32_t at = (uint32_t)(key0 + (lane & 15)) * RB + (lane >> 4) * 16;
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int c = 0; c < KB; ++c)
        k[n][c] = __builtin_amdgcn_raw_buffer_load_b128(rs, (int)(at + n * 16 * RB + c * 64), 0, 0);
  }
  __device__ __forceinline__ void load_v(__amdgpu_buffer_rsrc_t rs, int key0, int lane) {
    const uint32_t at = (uint32_t)(key0 + 4 * (lane >> 4)) * RB + (lane & 15) * (RB / 16);
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int off = (int)(at + (16 * n + i) * RB);
        if constexpr (VD == 2) {
          const u32x2 x = __builtin_amdgcn_raw_buffer_load_b64(rs, off, 0, 0);
          v[4 * n + i][0] = x[0];
          v[4 * n + i][1] = x[1];
        } else {
#pragma unroll
          for (int w = 0; w < VD; w += 4) {
            const u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(rs, off + 4 * w, 0, 0);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[4 * n + i][w + e] = x[e];
          }
        }
      }
  }
  // The drafted nodes node0 .. ; zeros for one that is not there.
  __device__ __forceinline__ void load_nodes(const T* kn, int64_t kstep, const T* vn, int64_t vstep, int node0, uint64_t there,
                                             int lane) {
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      const int node = node0 + 16 * n + (lane & 15);
      const bool on = node < kMaxNodes && (there >> (node & 63) & 1);
#pragma unroll
      for (int c = 0; c < KB; ++c) {
        k[n][c] = u32x4{0, 0, 0, 0};
        if (on)
          k[n][c] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(kn + node * kstep) + c * 64 + (lane >> 4) * 16);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = node0 + 16 * n + 4 * (lane >> 4) + i;
        const bool von = at < kMaxNodes && (there >> (at & 63) & 1);
        const uint32_t* p = reinterpret_cast<const uint32_t*>(reinterpret_cast<const char*>(vn + at * vstep) + (lane & 15) * (RB / 16));
#pragma unroll
        for (int w = 0; w < VD; ++w) v[4 * n + i][w] = von ? p[w] : 0;
      }
    }
  }
};

// O^T += V^T P^T; o[j] row i stands for element i D / 16 + j.
template <int D>
__device__ __forceinline__ void add_pv(const Step<bf16, D>& st, const f32x4 (&p)[2], f32x4 (&o)[D / 16]) {
  const u32x4 b = {pack_bf16(p[0][0], p[0][1]), pack_bf16(p[0][2], p[0][3]), pack_bf16(p[1][0], p[1][1]),
                   pack_bf16(p[1][2], p[1][3])};
#pragma unroll
  for (int j = 0; j < D / 16; ++j) {
    u32x4 a;
#pragma unroll
    for (int w = 0; w < 4; ++w)
      a[w] = __builtin_amdgcn_perm(st.v[2 * w + 1][j / 2], st.v[2 * w][j / 2], j % 2 ? 0x07060302u : 0x05040100u);
    o[j] = mfma16(a, b, o[j], bf16{});
  }
}
template <int D>
__device__ __forceinline__ void add_pv(const Step<float, D>& st, const f32x4 (&p)[1], f32x4 (&o)[D / 16]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < D / 16; ++j)
      o[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(st.v[i][j]), p[0][i], o[j], 0, 0, 0);
}

// The lanes' nodes: bit s of the result for node `lane` says whether it sees node s (its ancestors and itself); 0
// where the node, or one that it hangs on, is absent (its parent neither -1 nor an earlier node). By doubling: after
// round r a lane holds its 2^r nearest ancestors and points past them.
__device__ __forceinline__ uint64_t ancestors(const int32_t* parents, int t, int lane) {
  int up = lane < t ? parents[lane] : -2;
  if (up < -1 || up >= lane) up = -2;
  uint64_t sees = 1ull << lane;
#pragma unroll
  for (int r = 0; r < 6; ++r) {
    const int from = up < 0 ? lane : up;
    const uint64_t theirs = __shfl((unsigned long long)sees, from, kWave);
    const int next = __shfl(up, from, kWave);
    if (up >= 0) {
      sees |= theirs;
      up = next;
    }
  }
  return up == -1 ? sees : 0;
}

template <typename T>
__device__ __forceinline__ T* uniform_ptr(T* p) {
  const uint64_t a = reinterpret_cast<uint64_t>(p);
  const uint64_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)a);
  const uint64_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32));
  return reinterpret_cast<T*>(lo | (hi << 32));
}

__device__ __forceinline__ float max16(float x) {  // over the four lane groups
  x = fmaxf(x, __shfl_xor(x, 16, kWave));
  return lane32_max(x);
}
__device__ __forceinline__ float sum16(float x) {
  x += __shfl_xor(x, 16, kWave);
  return lane32_sum(x);
}

// Workspace: u64 [B Hkv] which nodes are there, then per chunk and row (m, l), then the unnormalised outputs.
struct Parts {
  uint64_t* there;
  f32x2* ml;   // [B Hkv, chunks, rows]
  float* acc;  // [B Hkv, chunks, rows, D]
};
__host__ __device__ inline int64_t parts_bytes(int64_t heads, int64_t chunks, int64_t rows, int64_t d) {
  return cdiv(heads, 2) * 16 + cdiv(heads * chunks * rows, 2) * 16 + heads * chunks * rows * d * 4;
}
__device__ __forceinline__ Parts parts_of(char* ws, int64_t heads, int64_t chunks, int64_t rows) {
  char* ml = ws + cdiv(heads, 2) * 16;
  return {reinterpret_cast<uint64_t*>(ws), reinterpret_cast<f32x2*>(ml),
          reinterpret_cast<float*>(ml + cdiv(heads * chunks * rows, 2) * 16)};
}

// One row block (16 NT rows) over one chunk of a head's cache; W waves with a stretch of it each. The last
// chunk's last wave takes the drafted nodes too, which come from k_new and v_new: no workgroup reads a row that
// another writes.
template <typename T, int D, int NT, int W>
__global__ __launch_bounds__(64 * W) void tree_attn_kernel(TreeArgs a) {
  typedef Step<T, D> S;
  constexpr int NS = S::NS, KEYS = S::KEYS, KB = S::KB, VE = D / 16;
  constexpr int DP = 512 / W < D ? 512 / W : D, PASSES = D / DP;  // columns per pass of the waves' merge
  __shared__ __attribute__((aligned(16))) float red[W][16][DP + 4];
  __shared__ float red_m[W][16], red_l[W][16];

  // Row blocks of one item lie 8 workgroups apart: on one XCD, whose L2 then holds the chunk for all of them.
  const int64_t group = blockIdx.x / (8 * a.row_blocks);
  const int rest = (int)(blockIdx.x - group * 8 * a.row_blocks), block = rest / 8;
  const int64_t item = group * 8 + rest % 8;
  if (item >= a.items) return;
  const int chunk = (int)(item % a.chunks);
  const int64_t head = item / a.chunks;  // b Hkv + h
  const int64_t b = head / a.Hkv;
  const int h = (int)(head - b * a.Hkv);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, q0 = lane & 15;
  const int p = a.pos[b];
  const bool valid = p >= 0 && p <= a.L - a.T;
  const int cached = valid ? p : 0;
  const bool drafts = chunk == a.chunks - 1;
  if (!drafts && (int64_t)chunk * W * a.wave_rows >= cached) return;  // an empty chunk, which nobody reads

  // Query rows: row r is node r % T of head h G + r / T. Rows past the last read as zeros and are not stored.
  u32x4 q[NT][KB];
  int node[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = (block * NT + n) * 16 + q0;
    const int gh = r / a.T;
    node[n] = r - gh * a.T;
    const char* src = reinterpret_cast<const char*>(static_cast<const T*>(a.q) + b * a.qs[0] + (h * a.G + gh) * a.qs[1] + node[n] * a.qs[2]);
#pragma unroll
    for (int c = 0; c < KB; ++c) {
      q[n][c] = u32x4{0, 0, 0, 0};
      if (r < a.rows) q[n][c] = *reinterpret_cast<const u32x4*>(src + c * 64 + g * 16);
    }
  }

  float m[NT], l[NT];
  f32x4 o[NT][VE];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    m[n] = -INFINITY;
    l[n] = 0.f;
#pragma unroll
    for (int j = 0; j < VE; ++j) o[n][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  S st;
  f32x4 s[NT][NS];
  auto scores = [&] {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int t = 0; t < NS; ++t) {
        s[n][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < KB; ++c) s[n][t] = mfma16(st.k[t][c], q[n][c], s[n][t], T{});
      }
  };
  // sees(n, t, i): whether row tile n's query of this lane sees key 16 t + 4 g + i of the step.
  auto softmax_pv = [&](auto masked, auto&& sees) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float mx = -INFINITY;
#pragma unroll
      for (int t = 0; t < NS; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[n][t][i] *= a.c;
          if (masked.value && !sees(n, t, i)) s[n][t][i] = -INFINITY;
          mx = fmaxf(mx, s[n][t][i]);
        }
      mx = fmaxf(m[n], max16(mx));
      const float ref = mx == -INFINITY ? 0.f : mx;
      if (__any(mx > m[n])) {
        const float f = __builtin_amdgcn_exp2f(m[n] - ref);
        l[n] *= f;
#pragma unroll
        for (int j = 0; j < VE; ++j) o[n][j] *= f;
      }
      m[n] = mx;
#pragma unroll
      for (int t = 0; t < NS; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[n][t][i] = __builtin_amdgcn_exp2f(s[n][t][i] - ref);
          l[n] += s[n][t][i];
        }
      add_pv<D>(st, s[n], o[n]);
    }
  };

  const int64_t base = head * a.L * D;
  const uint32_t bytes = (uint32_t)__builtin_amdgcn_readfirstlane(cached) * (uint32_t)S::RB;
  const __amdgpu_buffer_rsrc_t krs = __builtin_amdgcn_make_buffer_rsrc(uniform_ptr(static_cast<T*>(a.kc) + base), (short)0, (int)bytes, 0x00020000);
  const __amdgpu_buffer_rsrc_t vrs = __builtin_amdgcn_make_buffer_rsrc(uniform_ptr(static_cast<T*>(a.vc) + base), (short)0, (int)bytes, 0x00020000);
  const int from = __builtin_amdgcn_readfirstlane((chunk * W + wave) * a.wave_rows);
  const int to = __builtin_amdgcn_readfirstlane(min(from + a.wave_rows, cached));
  if (from < to) st.load_k(krs, from, lane);
  for (int key = from; key < to; key += KEYS) {
    st.load_v(vrs, key, lane);
    scores();
    if (key + KEYS < to) st.load_k(krs, key + KEYS, lane);
    if (key + KEYS <= cached)
      softmax_pv(std::false_type{}, [](int, int, int) { return true; });
    else
      softmax_pv(std::true_type{}, [&](int, int t, int i) { return key + 16 * t + 4 * g + i < cached; });
  }

  uint64_t there = 0;
  if (drafts && valid) {
    const uint64_t line = ancestors(a.parents + b * a.T, a.T, lane);
    there = __ballot(line != 0);
    const T* kn = static_cast<const T*>(a.kn) + b * a.ks[0] + h * a.ks[1];
    const T* vn = static_cast<const T*>(a.vn) + b * a.vs[0] + h * a.vs[1];
    if (wave == W - 1) {
      uint64_t mine[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) mine[n] = __shfl((unsigned long long)line, node[n], kWave);
      for (int at = 0; at < a.T; at += KEYS) {
        st.load_nodes(kn, a.ks[2], vn, a.vs[2], at, there, lane);
        scores();
        softmax_pv(std::true_type{}, [&](int n, int t, int i) {
          const int k = at + 16 * t + 4 * g + i;
          return k < kMaxNodes && (mine[n] >> (k & 63) & 1);
        });
      }
    }
    if (block == 0) {
      constexpr int VEC = S::RB / 16;
      for (int e = threadIdx.x; e < a.T * VEC; e += 64 * W) {
        const int t = e / VEC, at = e % VEC;
        if (!(there >> t & 1)) continue;
        const int64_t row = (base + (int64_t)(p + t) * D) / (16 / (int)sizeof(T)) + at;
        static_cast<u32x4*>(a.kc)[row] = reinterpret_cast<const u32x4*>(kn + t * a.ks[2])[at];
        static_cast<u32x4*>(a.vc)[row] = reinterpret_cast<const u32x4*>(vn + t * a.vs[2])[at];
      }
    }
  }

  // The waves' states, 16 rows at a time: weights 2^(m_w - max), then the sums over the waves in their order.
  Parts parts{};
  if (a.part) {
    parts = parts_of(a.part, a.items / a.chunks, a.chunks, a.rows);
    if (drafts && block == 0 && threadIdx.x == 0) parts.there[head] = there;
  }
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const float lt = sum16(l[n]);
#pragma unroll
    for (int pass = 0; pass < PASSES; ++pass) {
      __syncthreads();
      if (g == 0) {
        red_m[wave][q0] = m[n];
        red_l[wave][q0] = lt;
      }
      // A lane's elements: 4 VE in a row from g D / 4.
      if (g * (D / 4) / DP == pass) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < VE; ++j) red[wave][q0][g * (D / 4) % DP + i * VE + j] = o[n][j][i];
      }
      __syncthreads();
      for (int e = threadIdx.x; e < 16 * (DP / 4); e += 64 * W) {
        const int row = e / (DP / 4), d = e % (DP / 4) * 4, r = (block * NT + n) * 16 + row;
        if (r >= a.rows) continue;
        float mx = -INFINITY, lsum = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) mx = fmaxf(mx, red_m[w][row]);
        const float ref = mx == -INFINITY ? 0.f : mx;
        f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const float f = __builtin_amdgcn_exp2f(red_m[w][row] - ref);
          lsum += red_l[w][row] * f;
          sum += *reinterpret_cast<const f32x4*>(&red[w][row][d]) * f;
        }
        if (a.part) {
          const int64_t at = (head * a.chunks + chunk) * a.rows + r;
          *reinterpret_cast<f32x4*>(parts.acc + at * D + pass * DP + d) = sum;
          if (pass == 0 && d == 0) parts.ml[at] = f32x2{mx, lsum};
        } else {
          const int gh = r / a.T, t = r - gh * a.T;
          T* out = static_cast<T*>(a.out) + ((b * a.T + t) * a.H + h * a.G + gh) * D + pass * DP + d;
          const bool zero = !(there >> t & 1) || lsum == 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i) out[i] = Elem<T>::from_f32(!valid ? NAN : zero ? 0.f : sum[i] / lsum);
        }
      }
    }
  }
}

// Four elements of a row per thread: the chunks' weights 2^(m_c - max), then the sums in eight lines of chunks.
template <typename T, int D>
__global__ __launch_bounds__(256) void tree_join_kernel(TreeArgs a, int chunk_rows) {
  constexpr int PER = D / 4, ROWS = 256 / PER, N = 8;
  const int64_t head = blockIdx.y + (int64_t)blockIdx.z * a.Hkv;
  const int64_t b = blockIdx.z;
  const int h = blockIdx.y, r = (int)blockIdx.x * ROWS + threadIdx.x / PER, d = threadIdx.x % PER * 4;
  if (r >= a.rows) return;
  const Parts parts = parts_of(a.part, a.items / a.chunks, a.chunks, a.rows);
  const int p = a.pos[b];
  const bool valid = p >= 0 && p <= a.L - a.T;
  const uint64_t there = parts.there[head];
  const int gh = r / a.T, t = r - gh * a.T;
  const int full = valid ? min(a.chunks - 1, (p + chunk_rows - 1) / chunk_rows) : 0, used = full + 1;  // the last: the drafts'
  auto at = [&](int c) { return (head * a.chunks + (c < full ? c : a.chunks - 1)) * a.rows + r; };
  float mx = -INFINITY;
  for (int c = 0; c < used; c += N) {
    float mc[N];
#pragma unroll
    for (int u = 0; u < N; ++u) mc[u] = parts.ml[at(min(c + u, used - 1))][0];
#pragma unroll
    for (int u = 0; u < N; ++u) mx = fmaxf(mx, mc[u]);
  }
  const float ref = mx == -INFINITY ? 0.f : mx;
  float ls[N] = {};
  f32x4 as[N] = {};
  for (int c = 0; c < used; c += N) {
    f32x2 ml[N];
    f32x4 acc[N];
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int64_t i = at(min(c + u, used - 1));
      ml[u] = parts.ml[i];
      acc[u] = *reinterpret_cast<const f32x4*>(parts.acc + i * D + d);
    }
#pragma unroll
    for (int u = 0; u < N; ++u) {
      if (c + u >= used) continue;
      const float f = __builtin_amdgcn_exp2f(ml[u][0] - ref);
      ls[u] += ml[u][1] * f;
      as[u] += acc[u] * f;
    }
  }
#pragma unroll
  for (int n = N / 2; n > 0; n /= 2)
#pragma unroll
    for (int u = 0; u < n; ++u) {
      ls[u] += ls[u + n];
      as[u] += as[u + n];
    }
  T* out = static_cast<T*>(a.out) + ((b * a.T + t) * a.H + h * a.G + gh) * D + d;
  const bool zero = !(there >> t & 1) || ls[0] == 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) out[i] = Elem<T>::from_f32(!valid ? NAN : zero ? 0.f : as[0][i] / ls[0]);
}

constexpr int64_t kGridTarget = 1024;
constexpr int64_t kMostBlocks = 0xffffffff / 512;  // blocks of up to 512 threads: a launch has under 2^32 threads along x

struct Plan {
  int tiles;       // row tiles of 16 a wave
  int waves;
  int64_t row_blocks, chunks, wave_rows;
};
Plan plan_for(int64_t b, int64_t h, int64_t hkv, int64_t t, int64_t max_len, int64_t d, int dtype) {
  const int64_t rows = h / hkv * t, keys = dtype == FERRITE_BF16 ? 32 : 16;
  Plan p;
  p.tiles = rows <= 16 ? 1 : rows <= 32 || d > 128 ? 2 : 4;
  p.row_blocks = cdiv(rows, 16 * p.tiles);
  if (max_len <= 8 * 2 * keys) {
    p.waves = 8;
    p.chunks = 1;
    p.wave_rows = cdiv(cdiv(max_len, 8), keys) * keys;
    return p;
  }
  p.waves = 4;
  int64_t rows_of_chunk = 4 * keys;
  while (rows_of_chunk < max_len && b * hkv * p.row_blocks * cdiv(max_len, rows_of_chunk) > kGridTarget) rows_of_chunk *= 2;
  p.chunks = cdiv(max_len, rows_of_chunk);
  p.wave_rows = rows_of_chunk / 4;
  return p;
}

template <typename T, int D, int NT>
int tree_launch(const TreeArgs& a, const Plan& p, hipStream_t s) {
  const int64_t blocks = cdiv(a.items, 8) * 8 * p.row_blocks;
  if (blocks > kMostBlocks) return fail(FERRITE_ERR_INVALID_ARGUMENT, "ferrite_tree_attention: too many heads");
  if (p.waves == 8)
    hipLaunchKernelGGL((tree_attn_kernel<T, D, NT, 8>), dim3((unsigned)blocks), dim3(512), 0, s, a);
  else
    hipLaunchKernelGGL((tree_attn_kernel<T, D, NT, 4>), dim3((unsigned)blocks), dim3(256), 0, s, a);
  if (p.chunks > 1) {
    const int rc = check_launch("ferrite_tree_attention");
    if (rc != FERRITE_OK) return rc;
    const int64_t B = a.items / p.chunks / a.Hkv;
    hipLaunchKernelGGL((tree_join_kernel<T, D>), dim3((unsigned)cdiv(a.rows, 1024 / D), (unsigned)a.Hkv, (unsigned)B), dim3(256),
                       0, s, a, (int)(4 * p.wave_rows));
  }
  return check_launch("ferrite_tree_attention");
}

int check_tree(int64_t b, int64_t h, int64_t hkv, int64_t t, int64_t max_len, int64_t d, int dtype) {
  const std::string n = "ferrite_tree_attention";
  if (!valid_dtype(dtype)) return fail(FERRITE_ERR_INVALID_ARGUMENT, n + ": dtype must be FERRITE_F32 or FERRITE_BF16");
  if (b < 0 || hkv < 1 || b > 65535 || hkv > 65535 || h < hkv || h > 65535 || h % hkv)
    return fail(FERRITE_ERR_INVALID_ARGUMENT, n + ": need 0 <= b <= 65535 and up to 65535 query heads, a multiple of the key heads");
  if (t < 1 || t > kMaxNodes) return fail(FERRITE_ERR_INVALID_ARGUMENT, n + ": need 1 to 64 nodes");
  if (max_len < 1 || max_len > 0x7fffffff / 512) return fail(FERRITE_ERR_INVALID_ARGUMENT, n + ": need 1 <= max_len < 2^22");
  if (d != 64 && d != 128 && d != 256) return fail(FERRITE_ERR_INVALID_ARGUMENT, n + ": head dim must be 64, 128 or 256");
  return FERRITE_OK;
}

}  // namespace
}  // namespace ferrite

extern "C" int64_t ferrite_internal_tree_attention_workspace(int64_t b, int64_t h, int64_t hkv, int64_t t, int64_t max_len,
                                                             int64_t d, int dtype) {
  using namespace ferrite;
  if (check_tree(b, h, hkv, t, max_len, d, dtype) != FERRITE_OK) return -1;
  const Plan p = plan_for(b, h, hkv, t, max_len, d, dtype);
  return p.chunks > 1 ? parts_bytes(b * hkv, p.chunks, h / hkv * t, d) : 0;
}

extern "C" int ferrite_internal_tree_attention(const void* q, const void* k_new, const void* v_new, void* k_cache,
                                               void* v_cache, const int32_t* pos, const int32_t* parents, void* out,
                                               const int64_t* strides, int64_t b, int64_t h, int64_t hkv, int64_t t,
                                               int64_t max_len, int64_t d, int dtype, float scale, void* workspace,
                                               int64_t workspace_bytes, void* stream) {
  using namespace ferrite;
  const int rc = check_tree(b, h, hkv, t, max_len, d, dtype);
  if (rc != FERRITE_OK) return rc;
  if (b == 0) return FERRITE_OK;
  if (!q || !k_new || !v_new || !k_cache || !v_cache || !pos || !parents || !out || !strides)
    return fail(FERRITE_ERR_INVALID_ARGUMENT, "ferrite_tree_attention: null pointer");
  auto a16 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  bool aligned = a16(q) && a16(k_new) && a16(v_new) && a16(k_cache) && a16(v_cache) && a16(out);
  for (int i = 0; i < 9; ++i) aligned = aligned && strides[i] % (dtype == FERRITE_BF16 ? 8 : 4) == 0;
  if (!aligned) return fail(FERRITE_ERR_INVALID_ARGUMENT, "ferrite_tree_attention: tensors and strides must be 16-byte aligned");
  const Plan p = plan_for(b, h, hkv, t, max_len, d, dtype);
  TreeArgs a{q, k_new, v_new, k_cache, v_cache, pos, parents, out, nullptr, {}, {}, {}, b * hkv * p.chunks, (int)h, (int)hkv,
             (int)(h / hkv), (int)t, (int)max_len, (int)(h / hkv * t), (int)p.chunks, (int)p.row_blocks, (int)p.wave_rows,
             scale * kLog2e};
  for (int i = 0; i < 3; ++i) {
    a.qs[i] = strides[i];
    a.ks[i] = strides[3 + i];
    a.vs[i] = strides[6 + i];
  }
  if (p.chunks > 1) {
    if (!workspace || !a16(workspace) || workspace_bytes < parts_bytes(b * hkv, p.chunks, a.rows, d))
      return fail(FERRITE_ERR_INVALID_ARGUMENT, "ferrite_tree_attention: workspace too small or unaligned");
    a.part = static_cast<char*>(workspace);
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto tiles = [&](auto* e, auto D) {
    typedef std::remove_pointer_t<decltype(e)> T;
    if (p.tiles == 1) return tree_launch<T, D.value, 1>(a, p, s);
    if constexpr (D.value <= 128) {
      if (p.tiles == 4) return tree_launch<T, D.value, 4>(a, p, s);
    }
    return tree_launch<T, D.value, 2>(a, p, s);
  };
  auto dims = [&](auto* e) {
    if (d == 64) return tiles(e, std::integral_constant<int, 64>{});
    if (d == 128) return tiles(e, std::integral_constant<int, 128>{});
    return tiles(e, std::integral_constant<int, 256>{});
  };
  return dtype == FERRITE_BF16 ? dims((bf16*)nullptr) : dims((float*)nullptr);
}
