// After a drafted step, for gfx950: which of a tree's drafted tokens the model itself would have taken,
// and the cache's rows of those put in order.
//
// Reference: src/ferrite/serving/engine.py:98-131, :181-203, which takes one token a step (argmax) and
// stores one row; it drafts nothing. Node 0 of a sequence's tree is the token it already has; a node's
// logits say what follows it, and the walk goes from node 0 to the child that holds their argmax, as long
// as there is one. The rows of the nodes it visits, written at pos + node by the drafted step, then move
// to pos, pos + 1, ...
#include <math.h>

#include <algorithm>

#include "common.h"
#include "internal_api.h"

namespace ferrite {
namespace {

constexpr int kMaxNodes = 64;  // a node per lane of a wave

// (value, index) as one number whose largest is the largest value, of equal ones the lowest index. -0 and 0
// are equal, NaN is larger than any number (as in a tensor library's argmax).
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t b = __float_as_uint(x);
  if (x != x) return 0xffffffffu;
  if (x == 0.f) return 0x80000000u;
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ uint64_t key_of(uint32_t order, int64_t index) {
  return ((uint64_t)order << 32) | (0xffffffffu - (uint32_t)index);
}
__device__ __forceinline__ int64_t index_of(uint64_t key) { return 0xffffffffu - (uint32_t)key; }

template <typename T>
__device__ __forceinline__ float elem_of(const u32x4& raw, int e) {
  if constexpr (sizeof(T) == 2)
    return __uint_as_float(e % 2 ? raw[e / 2] & 0xffff0000u : raw[e / 2] << 16);
  else
    return __builtin_bit_cast(f32x4, raw)[e];
}

// The largest key of vectors t, t + n, .. of v (element 0 is x[first]), BATCH under way. Past the end the last one is read again:
// loads behind branches of their own would be waited for one by one. Numbers are compared as they are (three operations a
// value; orders take ten, which the reads of long rows do not hide): NaN, for which no comparison holds, is looked for
// alongside, and a thread that has one goes over its values again.
template <typename T, int BATCH>
__device__ __forceinline__ uint64_t best_vector(const u32x4* v, int64_t first, int64_t vecs, int t, int n) {
  constexpr int V = 16 / sizeof(T);
  if (t >= vecs) return 0;
  float best = -INFINITY;
  int64_t at = first + (int64_t)t * V;
  bool nan = false;
  for (int64_t i = t; i < vecs; i += BATCH * n) {
    u32x4 raw[BATCH];
#pragma unroll
    for (int u = 0; u < BATCH; ++u) raw[u] = __builtin_nontemporal_load(v + min(i + u * n, vecs - 1));
    int found = -1;  // of equal ones the first: a thread's values come in order
#pragma unroll
    for (int u = 0; u < BATCH; ++u)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float x = elem_of<T>(raw[u], e);
        nan |= x != x;
        if (x > best) {
          best = x;
          found = u * V + e;
        }
      }
    if (found >= 0) at = first + min(i + found / V * n, vecs - 1) * V + found % V;
  }
  uint64_t k = key_of(order_of(best), at);
  if (nan)
    for (int64_t i = t; i < vecs; i += n) {
      const u32x4 raw = v[i];
#pragma unroll
      for (int e = 0; e < V; ++e) k = max(k, key_of(order_of(elem_of<T>(raw, e)), first + i * V + e));
    }
  return k;
}

// The largest key of x[from, to), not empty, that thread t of n threads sees: vectors of 16 bytes between the first and the last
// 16-byte boundary, and an element before and behind them, whose loads go out first.
template <typename T>
__device__ __forceinline__ uint64_t best_of(const T* x, int64_t from, int64_t to, int t, int n) {
  constexpr int V = 16 / sizeof(T);
  const int64_t lead = ((16 - (reinterpret_cast<uintptr_t>(x + from) & 15)) & 15) / sizeof(T);
  const int64_t first = min(from + lead, to), vecs = (to - first) / V, tail = first + vecs * V + t;
  const float head_x = Elem<T>::to_f32(x[min(from + t, to - 1)]), tail_x = Elem<T>::to_f32(x[min(tail, to - 1)]);
  const u32x4* v = reinterpret_cast<const u32x4*>(x + first);
  uint64_t k = vecs <= n ? best_vector<T, 1>(v, first, vecs, t, n) : best_vector<T, 4>(v, first, vecs, t, n);
  if (from + t < first) k = max(k, key_of(order_of(head_x), from + t));
  if (tail < to) k = max(k, key_of(order_of(tail_x), tail));
  return k;
}

__device__ __forceinline__ uint64_t wave_best(uint64_t k) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) k = max(k, (uint64_t)__shfl_xor((unsigned long long)k, off, kWave));
  return k;
}

__device__ __forceinline__ bool node_there(int parent, int node) { return parent >= -1 && parent < node; }

// One wave: from node 0 down, a node per lane. Every step goes to a later node, so it ends.
__device__ __forceinline__ void walk(const int64_t* target, const int64_t* __restrict__ tokens,
                                     const int32_t* __restrict__ parents, int32_t* __restrict__ path,
                                     int32_t* __restrict__ count, int64_t* __restrict__ following, int64_t b, int t) {
  const int lane = threadIdx.x;
  const bool on = lane < t;
  const int parent = on ? parents[b * t + lane] : -2;
  const int64_t token = on ? tokens[b * t + lane] : 0;
  const bool there = on && node_there(parent, lane);
  int n = 0, mine = -1;
  int64_t next = -1;
  if (__shfl(parent, 0, kWave) == -1) {
    int at = 0;
    while (true) {
      if (lane == n) mine = at;
      ++n;
      next = target[at];
      const uint64_t child = __ballot(there && parent == at && token == next);
      if (!child) break;
      at = __builtin_ctzll(child);
    }
  }
  if (on) path[b * t + lane] = mine;
  if (lane == 0) {
    count[b] = n;
    following[b] = next;
  }
}

// A sequence in one workgroup: a wave to a row, then the walk. Bound by two round trips and the launch: 8 rows of 256 floats 2.5 us.
template <typename T>
__global__ __launch_bounds__(1024) void accept_short_kernel(const T* __restrict__ logits, const int64_t* __restrict__ tokens,
                                                            const int32_t* __restrict__ parents, int32_t* __restrict__ path,
                                                            int32_t* __restrict__ count, int64_t* __restrict__ following,
                                                            int t, int64_t v) {
  __shared__ int64_t target[kMaxNodes];
  const int64_t b = blockIdx.x;
  for (int row = threadIdx.x >> 6; row < t; row += 16) {
    if (!node_there(parents[b * t + row], row)) continue;
    const uint64_t k = wave_best(best_of(logits + (b * t + row) * v, 0, v, threadIdx.x & 63, 64));
    if ((threadIdx.x & 63) == 0) target[row] = index_of(k);
  }
  __syncthreads();
  if (threadIdx.x < 64) walk(target, tokens, parents, path, count, following, b, t);
}

// grid (pieces, rows): the best key of a piece of a row. Bound by HBM.
template <typename T>
__global__ __launch_bounds__(256) void accept_rows_kernel(const T* __restrict__ logits, const int32_t* __restrict__ parents,
                                                          uint64_t* __restrict__ part, int t, int64_t v, int64_t piece) {
  const int64_t row = blockIdx.y;
  if (!node_there(parents[row], (int)(row % t))) return;
  const int64_t from = blockIdx.x * piece, to = min(from + piece, v);
  const uint64_t k = wave_best(best_of(logits + row * v, from, to, threadIdx.x, 256));
  __shared__ uint64_t red[4];
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = k;
  __syncthreads();
  if (threadIdx.x == 0) part[row * gridDim.x + blockIdx.x] = max(max(red[0], red[1]), max(red[2], red[3]));
}

__global__ __launch_bounds__(1024) void accept_walk_kernel(const uint64_t* __restrict__ part, const int64_t* __restrict__ tokens,
                                                           const int32_t* __restrict__ parents, int32_t* __restrict__ path,
                                                           int32_t* __restrict__ count, int64_t* __restrict__ following, int t,
                                                           int pieces) {
  __shared__ int64_t target[kMaxNodes];
  const int64_t b = blockIdx.x;
  for (int row = threadIdx.x >> 6; row < t; row += 16) {
    if (!node_there(parents[b * t + row], row)) continue;
    uint64_t k = 0;
    for (int i = threadIdx.x & 63; i < pieces; i += 64) k = max(k, part[(b * t + row) * pieces + i]);
    k = wave_best(k);
    if ((threadIdx.x & 63) == 0) target[row] = index_of(k);
  }
  __syncthreads();
  if (threadIdx.x < 64) walk(target, tokens, parents, path, count, following, b, t);
}

// Whether one workgroup walks a sequence's rows, a wave to each, or they are cut into pieces over the chip and walked by a second
// kernel. One: 8 rows of 4096 floats 6.6 us and not 9.4, of 8192 bf16 7.6 and not 9.3; 32 rows (two to a wave) of 2048 floats
// 6.5 and 10.1; 64 of 1024 8.0 and 10.3 (bf16 12.1 and 10.5). Two: 32 rows of 4096 9.1 us and not 10.7, 64 of 2048 10.3 and
// 10.6 (bf16 10.5 and 13.2), of 4096 9.3 and 20.8.
bool short_rows(int64_t t, int64_t v) { return v <= (t <= 16 ? 8192 : 4096 / cdiv(t, 16)); }
// Pieces of a row: small ones, so that the chip stays full to the end (16 sequences of up to 32 rows of 50257 floats:
// 14.1 us, 5.5 TB/s with the launch; pieces of 8192 14.7, of 16384 17.0), but no more than 8192 workgroups of them.
constexpr int64_t kPiece = 4096;
int64_t piece_of(int64_t rows, int64_t v) {
  int64_t piece = kPiece;
  while (piece < v && rows * cdiv(v, piece) > 8192) piece *= 2;
  return piece;
}

// A thread owns U bytes of a head's rows and moves them one accepted row after another, so no thread reads what
// another writes. Rows go to places at or before their own and their order holds (path[i] > path[i - 1]), so a row's place is
// never one that a later row still has to leave: the loads of kBatch rows go out together. Bound by the launch and two round
// trips: 12 layers of 32 sequences, 12 heads of 64, up to 24 rows, bf16: 5.5 us a call.
constexpr int kBatch = 8;
template <typename U>
__global__ __launch_bounds__(256) void compact_kernel(U* __restrict__ k_cache, U* __restrict__ v_cache,
                                                      const int32_t* __restrict__ pos, const int32_t* __restrict__ path,
                                                      const int32_t* __restrict__ count, int64_t layers, int64_t B, int64_t H,
                                                      int64_t L, int cols, int t) {
  __shared__ int32_t line[kMaxNodes];
  __shared__ int rows;
  const int64_t b = blockIdx.y;
  const int p = pos[b];
  if (threadIdx.x < 64) {
    const int lane = threadIdx.x, n = min(count[b], t);
    const int mine = lane < n ? path[b * t + lane] : -1;
    const int before = __shfl_up(mine, 1, kWave);
    const bool ok = lane < n && p >= 0 && mine > (lane ? before : -1) && mine < L - p;
    const uint64_t bad = ~__ballot(ok);
    line[lane] = mine;
    if (lane == 0) rows = bad ? __builtin_ctzll(bad) : 64;
  }
  __syncthreads();
  const int64_t item = (int64_t)blockIdx.x * 256 + threadIdx.x, heads = layers * H;
  if (item >= 2 * heads * cols) return;
  const int64_t head = item / cols % heads;
  const int col = (int)(item % cols);
  const int64_t at = ((head / H * B + b) * H + head % H) * L + p;
  U* base = (item / cols < heads ? k_cache : v_cache) + at * cols + col;
  for (int i = 0; i < rows; i += kBatch) {
    U x[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
      if (i + u < rows && line[i + u] != i + u) x[u] = base[(int64_t)line[i + u] * cols];
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
      if (i + u < rows && line[i + u] != i + u) base[(int64_t)(i + u) * cols] = x[u];
  }
}

}  // namespace
}  // namespace ferrite

extern "C" int64_t ferrite_internal_accept_drafts_workspace(int64_t b, int64_t t, int64_t v) {
  using namespace ferrite;
  if (b < 0 || t < 1 || t > kMaxNodes || v < 1 || v > 0x7fffffff || b > 65535 / t) return -1;
  return short_rows(t, v) ? 0 : b * t * cdiv(v, piece_of(b * t, v)) * (int64_t)sizeof(uint64_t);
}

extern "C" int ferrite_internal_accept_drafts(const void* logits, const int64_t* tokens, const int32_t* parents,
                                              int32_t* path, int32_t* count, int64_t* following, int64_t b, int64_t t,
                                              int64_t v, int dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace ferrite;
  if (!valid_dtype(dtype))
    return fail(FERRITE_ERR_INVALID_ARGUMENT, "ferrite_accept_drafts: dtype must be FERRITE_F32 or FERRITE_BF16");
  const int64_t need = ferrite_internal_accept_drafts_workspace(b, t, v);
  if (need < 0)
    return fail(FERRITE_ERR_INVALID_ARGUMENT, "ferrite_accept_drafts: need 1 to 64 nodes, at most 65535 of them in all, and 1 <= vocabulary < 2^31");
  if (b == 0) return FERRITE_OK;
  if (!logits || !tokens || !parents || !path || !count || !following)
    return fail(FERRITE_ERR_INVALID_ARGUMENT, "ferrite_accept_drafts: null pointer");
  if (need && (!workspace || workspace_bytes < need))
    return fail(FERRITE_ERR_INVALID_ARGUMENT, "ferrite_accept_drafts: workspace too small");
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto go = [&](auto* x) {
    typedef std::remove_const_t<std::remove_pointer_t<decltype(x)>> T;
    if (!need) {
      hipLaunchKernelGGL((accept_short_kernel<T>), dim3((unsigned)b), dim3(1024), 0, s, x, tokens, parents, path, count,
                         following, (int)t, v);
      return;
    }
    const int64_t piece = piece_of(b * t, v), pieces = cdiv(v, piece);
    uint64_t* part = static_cast<uint64_t*>(workspace);
    hipLaunchKernelGGL((accept_rows_kernel<T>), dim3((unsigned)pieces, (unsigned)(b * t)), dim3(256), 0, s, x, parents,
                       part, (int)t, v, piece);
    hipLaunchKernelGGL(accept_walk_kernel, dim3((unsigned)b), dim3(1024), 0, s, part, tokens, parents, path, count,
                       following, (int)t, (int)pieces);
  };
  if (dtype == FERRITE_BF16)
    go(static_cast<const bf16*>(logits));
  else
    go(static_cast<const float*>(logits));
  return check_launch("ferrite_accept_drafts");
}

extern "C" int ferrite_internal_compact_cache(void* k_cache, void* v_cache, const int32_t* pos, const int32_t* path,
                                              const int32_t* count, int64_t layers, int64_t b, int64_t h, int64_t max_len,
                                              int64_t d, int64_t t, int dtype, void* stream) {
  using namespace ferrite;
  if (!valid_dtype(dtype))
    return fail(FERRITE_ERR_INVALID_ARGUMENT, "ferrite_compact_cache: dtype must be FERRITE_F32 or FERRITE_BF16");
  if (layers < 0 || b < 0 || h < 0 || max_len < 1 || d < 1 || t < 1 || t > kMaxNodes || b > 65535 || layers > 0xffff ||
      h > 0xffff || max_len > 0x7fffffff || d > 0xffff)
    return fail(FERRITE_ERR_INVALID_ARGUMENT, "ferrite_compact_cache: need 1 to 64 nodes, at most 65535 layers, sequences and heads, 1 <= max_len < 2^31 and head dims up to 65535");
  if (layers == 0 || b == 0 || h == 0) return FERRITE_OK;
  if (!k_cache || !v_cache || !pos || !path || !count)
    return fail(FERRITE_ERR_INVALID_ARGUMENT, "ferrite_compact_cache: null pointer");
  const int64_t bytes = d * (dtype == FERRITE_BF16 ? 2 : 4);
  const bool vec = bytes % 16 == 0 && ((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache)) & 15) == 0;
  const int64_t cols = vec ? bytes / 16 : d, blocks = cdiv(2 * layers * h * cols, 256);
  if (blocks > 0xffffffff / 256) return fail(FERRITE_ERR_INVALID_ARGUMENT, "ferrite_compact_cache: too many heads");
  const int64_t all = std::min(layers * b * h, ((int64_t)1 << 62) / (max_len * bytes)) * max_len * bytes;
  if (overlap(k_cache, all, v_cache, all))  // a row could be read behind the other cache's write of it
    return fail(FERRITE_ERR_INVALID_ARGUMENT, "ferrite_compact_cache: the caches overlap");
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto go = [&](auto* unit) {
    typedef std::remove_pointer_t<decltype(unit)> U;
    hipLaunchKernelGGL((compact_kernel<U>), dim3((unsigned)blocks, (unsigned)b), dim3(256), 0, s,
                       static_cast<U*>(k_cache), static_cast<U*>(v_cache), pos, path, count, layers, b, h, max_len,
                       (int)cols, (int)t);
  };
  if (vec)
    go((u32x4*)nullptr);
  else if (dtype == FERRITE_BF16)
    go((uint16_t*)nullptr);
  else
    go((uint32_t*)nullptr);
  return check_launch("ferrite_compact_cache");
}
