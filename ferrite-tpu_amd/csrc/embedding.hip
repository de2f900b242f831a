// Lookup of scaled rows of a table and its gradient, for gfx950.
//
// Reference: src/ferrite/model/gpt.py:124-127 (the token embedding) and its autodiff backward, which XLA runs as a gather and a
// scatter-add. The kernels of layout.hip take vocabularies of up to 1024 tokens with a position table; these any vocabulary.
//   out[i] = scale table[t_i]          dtable[t] = scale sum over i with t_i = t of dout[i]
// A token outside the table gives NaN in its row and nothing to the gradient; the padding's token gives nothing to the gradient. With
// `indexing` (the model's own lookup) negative tokens count from the table's end, and one outside it stops the program.
//
// Both are bound by memory: the rows that are looked up, the output; for the gradient the rows of dout and the whole table, most of whose
// rows are zero where the vocabulary is large. The gradient's rows are brought into the tokens' order, equal ones in the order in
// which they stand, and added along it in f32: no atomics, and one result whatever the launch's timing.
//   order  Up to kRankRows rows: every row's place is the number of rows before it, counted against all of them in LDS (8192 rows:
//          67 million comparisons over the chip) by workgroups of the same launch that fills the table with zeros,
//          behind whose 10 us (50 MB) it disappears. More rows: digits of up to 10 bits, stable, three launches each.
//   sums   A wave adds a piece of 16 or 64 rows of the order, 512 columns at a time, and stores each token's sum where the piece holds
//          all of its rows; the first and the last of a piece may go on in its neighbours and leave a partial row.
//   join   A workgroup adds the partial rows of a token that starts in its piece and goes on.
#include <math.h>

#include <algorithm>

#include "common.h"
#include "internal_api.h"
#include "rows.h"
#include "table_row.h"

namespace ferrite {
namespace {

constexpr int kRankRows = 16384;  // 64 KB of keys in LDS
constexpr int kIndexBits = 14;    // a row's index below its token in a key
constexpr int64_t kRankVocab = (int64_t)1 << (32 - kIndexBits);
static_assert(kRankRows == 1 << kIndexBits, "a key holds a row's index");

// A thread to a unit of a row, units of all rows in line.
template <typename TE, typename TO, int W>
__global__ __launch_bounds__(256) void lookup_kernel(const int64_t* __restrict__ tokens, const TE* __restrict__ table,
                                                     TO* __restrict__ out, int64_t total, int units, int dim, int64_t vocab,
                                                     float scale, bool indexing) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t row = total <= 0xffffffff ? (uint32_t)i / (uint32_t)units : i / units;
    const int at = column<W>((int)(i - row * units), dim);
    const int64_t t = table_row(tokens[row], vocab, indexing);
    if (t == kStopRow) __builtin_trap();
    float v[W];
    if (t >= 0) {
      Cols<TE, W> in;
      in.load(table + t * dim + at);
      in.get(v);
#pragma unroll
      for (int e = 0; e < W; ++e) v[e] *= scale;
    } else {
#pragma unroll
      for (int e = 0; e < W; ++e) v[e] = NAN;
    }
    Cols<TO, W> o;
    o.set(v);
    o.store(out + row * dim + at);
  }
}

// The token of a row in the gradient's order: those without a gradient behind all others.
struct Vocab {
  int64_t size, pad;
  bool indexing;
};
__device__ __forceinline__ uint32_t token_of(int64_t t, const Vocab& v) {
  t = table_row(t, v.size, v.indexing);
  return t < 0 || t == v.pad ? (uint32_t)v.size : (uint32_t)t;
}

// Zeros in `bytes` bytes at p, the workgroup's share of `blocks`.
__device__ __forceinline__ void fill_zero(char* p, int64_t bytes, int64_t block, int64_t blocks) {
  const int64_t lead = std::min<int64_t>((16 - (int64_t)(reinterpret_cast<uintptr_t>(p) & 15)) & 15, bytes);
  const int64_t vecs = (bytes - lead) / 16;
  if (block == 0) {  // what lies before the first and behind the last 16-byte boundary, two bytes at a time
    for (int64_t i = threadIdx.x * 2; i < lead; i += blockDim.x * 2) *reinterpret_cast<uint16_t*>(p + i) = 0;
    for (int64_t i = lead + vecs * 16 + threadIdx.x * 2; i < bytes; i += blockDim.x * 2) *reinterpret_cast<uint16_t*>(p + i) = 0;
  }
  u32x4* v = reinterpret_cast<u32x4*>(p + lead);
  for (int64_t i = block * blockDim.x + threadIdx.x; i < vecs; i += blocks * blockDim.x)
    __builtin_nontemporal_store(u32x4{0u, 0u, 0u, 0u}, v + i);
}

// Workgroups 0 .. ranks - 1 order R rows each, a share of the comparisons to every R lanes; the others fill the table's gradient. R
// goes with the rows so that the comparisons spread over the chip (rank_rows): 8192 rows by 64 17 us with the fill, by 32 12.
template <int R>
__global__ __launch_bounds__(512) void rank_fill_kernel(const int64_t* __restrict__ tokens, uint32_t* __restrict__ keys,
                                                        uint32_t* __restrict__ order, int rows, Vocab vocab, int ranks,
                                                        char* __restrict__ dtable, int64_t bytes) {
  constexpr int kShares = 512 / R;
  extern __shared__ __attribute__((aligned(16))) uint32_t all[];  // [padded]: (token, index), no two alike
  __shared__ uint32_t places[kShares][R];
  if ((int)blockIdx.x >= ranks) {
    fill_zero(dtable, bytes, blockIdx.x - ranks, gridDim.x - ranks);
    return;
  }
  const int share = (rows + 4 * kShares - 1) / (4 * kShares) * 4, padded = share * kShares;
  for (int i0 = 0; i0 < padded; i0 += 8 * 512) {  // eight loads together: one by one they take 16 round trips for 8192 rows
    int64_t t[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) t[u] = tokens[min(i0 + u * 512 + (int)threadIdx.x, rows - 1)];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int i = i0 + u * 512 + (int)threadIdx.x;
      if (i < padded) all[i] = i < rows ? (token_of(t[u], vocab) << kIndexBits) | (uint32_t)i : 0xffffffffu;
    }
  }
  __syncthreads();
  const int r = threadIdx.x % R, part = threadIdx.x / R, mine = (int)blockIdx.x * R + r;
  const uint32_t key = all[min(mine, rows - 1)];
  uint32_t before = 0;
  const u32x4* p = reinterpret_cast<const u32x4*>(all + part * share);
#pragma unroll 4
  for (int j = 0; j < share / 4; ++j) {
    const u32x4 k = p[j];
#pragma unroll
    for (int e = 0; e < 4; ++e) before += k[e] < key;
  }
  places[part][r] = before;
  __syncthreads();
  if (part == 0 && mine < rows) {
    uint32_t place = 0;
#pragma unroll
    for (int w = 0; w < kShares; ++w) place += places[w][r];
    keys[place] = key >> kIndexBits;
    order[place] = key & (kRankRows - 1);
  }
}
int rank_rows(int64_t rows) { return rows > 8192 ? 64 : rows > 4096 ? 32 : 16; }

__global__ __launch_bounds__(512) void fill_kernel(char* __restrict__ dtable, int64_t bytes) {
  fill_zero(dtable, bytes, blockIdx.x, gridDim.x);
}

// ---- more rows: stable passes over digits, least first ----
constexpr int kSortTile = 1024;  // rows to a workgroup: 4 waves of 4 rounds (65536 rows 7.9 us a pass; 8 rounds 11.4)
constexpr int kRounds = kSortTile / 256;
constexpr int kMaxDigits = 1024;

// Where a pass reads a row's token and index: the tokens themselves at first.
struct SortSource {
  const int64_t* tokens;  // or null:
  const uint32_t *keys, *order;
  Vocab vocab;
  __device__ __forceinline__ uint32_t key(int64_t i) const { return tokens ? token_of(tokens[i], vocab) : keys[i]; }
  __device__ __forceinline__ uint32_t index(int64_t i) const { return tokens ? (uint32_t)i : order[i]; }
};

// counts[digit][workgroup]
__global__ __launch_bounds__(256) void sort_count_kernel(SortSource src, uint32_t* __restrict__ counts, int64_t rows, int shift,
                                                         int digits) {
  __shared__ uint32_t hist[kMaxDigits];
  for (int d = threadIdx.x; d < digits; d += 256) hist[d] = 0;
  __syncthreads();
  const int64_t first = (int64_t)blockIdx.x * kSortTile, end = std::min<int64_t>(rows, first + kSortTile);
  for (int64_t i = first + threadIdx.x; i < end; i += 256) atomicAdd(&hist[(src.key(i) >> shift) & (digits - 1)], 1u);
  __syncthreads();
  for (int d = threadIdx.x; d < digits; d += 256) counts[(int64_t)d * gridDim.x + blockIdx.x] = hist[d];
}

// A wave to a digit: how many rows of that digit lie in the workgroups before each, and in all.
__global__ __launch_bounds__(64) void sort_scan_kernel(uint32_t* __restrict__ counts, uint32_t* __restrict__ totals, int blocks) {
  uint32_t* row = counts + (int64_t)blockIdx.x * blocks;
  uint32_t carry = 0;
  for (int b0 = 0; b0 < blocks; b0 += 64) {
    const int b = b0 + (int)threadIdx.x;
    const uint32_t mine = b < blocks ? row[b] : 0;
    uint32_t upto = mine;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const uint32_t v = __shfl_up(upto, off, kWave);
      if ((int)threadIdx.x >= off) upto += v;
    }
    if (b < blocks) row[b] = carry + upto - mine;
    carry += __shfl(upto, 63, kWave);
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = carry;
}

// Rows to their places. A wave owns kSortTile / 4 rows in a row, 64 a round; lanes of one digit find each other by a ballot per bit.
__global__ __launch_bounds__(256) void sort_place_kernel(SortSource src, const uint32_t* __restrict__ counts,
                                                         const uint32_t* __restrict__ totals, uint32_t* __restrict__ keys,
                                                         uint32_t* __restrict__ order, int64_t rows, int shift, int bits) {
  __shared__ uint32_t at[4][kMaxDigits];  // per wave: rows of a digit so far, then their first place
  __shared__ uint32_t sums[256];
  const int digits = 1 << bits, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int d = threadIdx.x; d < 4 * digits; d += 256) at[d >> bits][d & (digits - 1)] = 0;
  __syncthreads();
  const int64_t first = (int64_t)blockIdx.x * kSortTile + wave * (kSortTile / 4);
  uint32_t key[kRounds], rank[kRounds];
#pragma unroll
  for (int u = 0; u < kRounds; ++u) {
    const int64_t i = first + u * 64 + lane;
    const bool on = i < rows;
    key[u] = on ? src.key(i) : 0;
    const uint32_t d = (key[u] >> shift) & (digits - 1);
    uint64_t peers = __ballot(on);
    for (int k = 0; k < bits; ++k) {
      const uint64_t set = __ballot((d >> k) & 1);
      peers &= (d >> k) & 1 ? set : ~set;
    }
    const uint64_t below = lane ? peers & (~0ull >> (64 - lane)) : 0;
    const uint32_t seen = on ? at[wave][d] : 0;
    rank[u] = seen + __builtin_popcountll(below);
    __builtin_amdgcn_wave_barrier();  // every lane has read before the first of each digit writes
    if (on && below == 0) at[wave][d] = seen + __builtin_popcountll(peers);
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();
  // First places: the digits before, the workgroups before, the waves before. A thread sums digits / 256 (at least one) in a row.
  const int per = std::max(1, digits / 256);
  uint32_t sum = 0;
  for (int k = 0; k < per; ++k) {
    const int d = (int)threadIdx.x * per + k;
    if (d < digits) sum += totals[d];
  }
  sums[threadIdx.x] = sum;
  __syncthreads();
  for (int off = 1; off < 256; off <<= 1) {
    const uint32_t v = (int)threadIdx.x >= off ? sums[threadIdx.x - off] : 0;
    __syncthreads();
    sums[threadIdx.x] += v;
    __syncthreads();
  }
  uint32_t base = sums[threadIdx.x] - sum;
  for (int k = 0; k < per; ++k) {
    const int d = (int)threadIdx.x * per + k;
    if (d >= digits) break;
    uint32_t place = base + counts[(int64_t)d * gridDim.x + blockIdx.x];
    base += totals[d];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const uint32_t n = at[w][d];
      at[w][d] = place;
      place += n;
    }
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < kRounds; ++u) {
    const int64_t i = first + u * 64 + lane;
    if (i >= rows) continue;
    const uint32_t place = at[wave][(key[u] >> shift) & (digits - 1)] + rank[u];
    keys[place] = key[u];
    order[place] = src.index(i);
  }
}

// ---- the sums ----
// Rows [first, first + n) of the order and 64 W columns to a wave. slab: two f32 rows a piece, of the token that began before
// it and of the one that goes on behind it. A token that began before and goes on is the former.
template <typename T, typename TO, int W>
__global__ __launch_bounds__(64) void token_sums_kernel(const uint32_t* __restrict__ keys, const uint32_t* __restrict__ order,
                                                        const T* __restrict__ dy, TO* __restrict__ dtable,
                                                        float* __restrict__ slab, int64_t rows, int dim, uint32_t vocab,
                                                        float scale, int piece) {
  constexpr int U = 8;  // rows whose loads go out together
  const int lane = threadIdx.x;
  const int at = column<W>((int)blockIdx.y * 64 + lane, dim);
  const int64_t first = (int64_t)blockIdx.x * piece, end = std::min<int64_t>(rows, first + piece);
  const uint32_t before = first ? keys[first - 1] : vocab, behind = end < rows ? keys[end] : vocab;
  float acc[W];
  uint32_t current = keys[first];
  if (current == vocab) return;  // rows without a gradient, from here on
  bool opened = current == before;  // the current token began in a piece before
  auto leave = [&](bool goes_on) {
    if (at < 0) return;
    if (opened || goes_on) {
      float* to = slab + ((int64_t)blockIdx.x * 2 + (opened ? 0 : 1)) * dim + at;
#pragma unroll
      for (int e = 0; e < W; ++e) to[e] = acc[e];
      return;
    }
    float v[W];
#pragma unroll
    for (int e = 0; e < W; ++e) v[e] = acc[e] * scale;
    Cols<TO, W> o;
    o.set(v);
    o.store(dtable + (int64_t)current * dim + at);
  };
#pragma unroll
  for (int e = 0; e < W; ++e) acc[e] = 0.f;
  for (int64_t p = first; p < end; p += U) {
    const int64_t i = std::min<int64_t>(p + (lane & (U - 1)), end - 1);
    const uint32_t key = keys[i], row = order[i];
    Cols<T, W> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t r = __builtin_amdgcn_readlane(row, u);
      if (at >= 0) v[u].load(dy + (int64_t)r * dim + at);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (p + u >= end) break;
      const uint32_t k = __builtin_amdgcn_readlane(key, u);
      if (k != current) {
        leave(false);
        if (k == vocab) return;
        current = k;
        opened = false;
#pragma unroll
        for (int e = 0; e < W; ++e) acc[e] = 0.f;
      }
      float x[W];
      if (at >= 0) {
        v[u].get(x);
#pragma unroll
        for (int e = 0; e < W; ++e) acc[e] += x[e];
      }
    }
  }
  leave(behind == current);
}

// The token that goes on behind a piece in which it began: its partial rows. Of few pieces each wave adds all of its columns'; of more
// the waves share the pieces 4 or 16 ways, every 4th or 16th to one, and their sums are added in order. us for the 24
// tokens over several pieces of 8192 (up to 50 pieces, 768 columns): 16 ways always 15.0, so 7.
template <typename TO>
__global__ __launch_bounds__(1024) void token_join_kernel(const uint32_t* __restrict__ keys, const float* __restrict__ slab,
                                                          TO* __restrict__ dtable, int64_t rows, int dim, uint32_t vocab,
                                                          float scale, int piece) {
  __shared__ float red[16][64];
  const int64_t first = (int64_t)blockIdx.x * piece, end = first + piece;
  if (end >= rows) return;
  const uint32_t token = keys[end - 1];
  if (token == vocab || keys[end] != token || (first && keys[first - 1] == token)) return;
  // The pieces that it reaches: the last is the first whose last row is another token's (keys go up).
  int64_t lo = blockIdx.x + 1, hi = cdiv(rows, (int64_t)piece) - 1;
  while (lo < hi) {
    const int64_t mid = (lo + hi) / 2;
    if (keys[std::min<int64_t>(rows, (mid + 1) * piece) - 1] == token)
      lo = mid + 1;
    else
      hi = mid;
  }
  // A piece that ends with the token's last row holds it too: the search went one too far if the piece it found begins with another.
  const int64_t last = keys[lo * piece] == token ? lo : lo - 1;
  const int64_t pieces = last - blockIdx.x + 1;
  const int ways = pieces <= 24 ? 1 : pieces <= 256 ? 4 : 16, groups = 16 / ways;
  const int c = threadIdx.x & 63, wave = threadIdx.x >> 6, way = wave / groups;
  for (int col0 = 0; col0 < dim; col0 += 64 * groups) {
    const int col = col0 + wave % groups * 64 + c;
    float acc = 0.f;
    if (col < dim) {
#pragma unroll 8
      for (int64_t p = blockIdx.x + way; p <= last; p += ways)
        acc += slab[(p * 2 + (p == blockIdx.x ? 1 : 0)) * dim + col];
    }
    if (ways > 1) {
      __syncthreads();
      red[wave][c] = acc;
      __syncthreads();
      if (way > 0) continue;
      acc = 0.f;
      for (int w = 0; w < ways; ++w) acc += red[w * groups + wave][c];
    }
    if (col < dim) dtable[(int64_t)token * dim + col] = Elem<TO>::from_f32(acc * scale);
  }
}

struct EmbedPlan {
  bool rank;
  int passes, bits, piece;
  int64_t pieces, sort_blocks;
  // parts of the workspace, in bytes
  int64_t keys, order, keys2, order2, counts, totals, slab, bytes;
};
bool embed_plan(int64_t rows, int64_t dim, int64_t vocab, EmbedPlan& p) {
  // A join of 1024 threads for every 64 rows stays under 2^32 threads.
  if (rows < 0 || rows > 0x7ffffff || dim < 1 || dim > 0x7fffffff / 64 || vocab < 1 || vocab > 0x7ffffffe ||
      vocab > ((int64_t)1 << 58) / dim || rows > ((int64_t)1 << 58) / dim || cdiv(dim, (int64_t)64) > 65535)
    return false;
  p = EmbedPlan{};
  // us of the gradient, bf16, counting / sorting: 512 rows of 768 columns over 32768 tokens 18.7 / 37.7, 4096 21.3 / 44.2, 8192 27.7 / 48.2,
  // 12288 45.1 / 53.9, 16384 52.8 / 55.0 (x 512 over 4096: 47.1 / 44.6). A piece of 16 / 64 rows: 4096 x 768 22.5 / 33.3, 16384 51.8 / 56.9,
  // 32768 70.7 / 70.1, 65536 x 512 73.7 / 65.3, 131072 x 512 115.6 / 87.6, 262144 x 768 228 / 170.
  p.rank = rows <= kRankRows && vocab < kRankVocab;
  int width = 1;
  while (width < 31 && ((int64_t)1 << width) <= vocab) ++width;  // bits of the largest key, vocab
  p.passes = (int)cdiv(width, 10);
  p.bits = (int)cdiv(width, p.passes);
  p.piece = rows <= 1 << 15 ? 16 : 64;
  p.pieces = cdiv(rows, (int64_t)p.piece);
  p.sort_blocks = cdiv(rows, (int64_t)kSortTile);
  int64_t at = 0;
  auto take = [&](int64_t n) {
    const int64_t here = at;
    at += (n + 15) / 16 * 16;
    return here;
  };
  p.keys = take(rows * 4);
  p.order = take(rows * 4);
  if (!p.rank) {
    p.keys2 = take(rows * 4);
    p.order2 = take(rows * 4);
    p.counts = take((p.sort_blocks << p.bits) * 4);
    p.totals = take(((int64_t)1 << p.bits) * 4);
  }
  p.slab = take(p.pieces * 2 * dim * 4);
  p.bytes = at;
  return true;
}

template <typename T, typename TO>
int embed_bwd(const int64_t* tokens, const T* dy, TO* dtable, int64_t rows, int64_t dim, const Vocab& vocab, float scale,
              const EmbedPlan& p, char* ws, hipStream_t s) {
  const int64_t bytes = vocab.size * dim * (int64_t)sizeof(TO);
  const unsigned fills = (unsigned)std::clamp<int64_t>(cdiv(bytes, (int64_t)512 * 16 * 8), 1, 2048);
  auto part = [&](int64_t at) { return reinterpret_cast<uint32_t*>(ws + at); };
  uint32_t *keys = part(p.keys), *order = part(p.order);
  if (rows && p.rank) {
    const int r = rank_rows(rows), ranks = (int)cdiv(rows, (int64_t)r), lds = (int)cdiv(rows, 4 * (512 / r)) * 4 * (512 / r) * 4;
    auto go = [&](auto kernel) {
      if (int rc = allow_lds((const void*)kernel, kRankRows * 4, s, "ferrite_embedding_bwd")) return rc;
      hipLaunchKernelGGL(kernel, dim3(ranks + fills), dim3(512), lds, s, tokens, keys, order, (int)rows, vocab, ranks,
                         reinterpret_cast<char*>(dtable), bytes);
      return (int)FERRITE_OK;
    };
    if (int rc = r == 64 ? go(rank_fill_kernel<64>) : r == 32 ? go(rank_fill_kernel<32>) : go(rank_fill_kernel<16>)) return rc;
  } else {
    hipLaunchKernelGGL(fill_kernel, dim3(fills), dim3(512), 0, s, reinterpret_cast<char*>(dtable), bytes);
    if (rows == 0) return check_launch("ferrite_embedding_bwd");
    const unsigned blocks = (unsigned)p.sort_blocks;
    uint32_t *counts = part(p.counts), *totals = part(p.totals);
    // The last pass leaves its rows in keys and order.
    uint32_t* to[2][2] = {{keys, order}, {part(p.keys2), part(p.order2)}};
    SortSource src{tokens, nullptr, nullptr, vocab};
    for (int k = 0; k < p.passes; ++k) {
      uint32_t** dst = to[(p.passes - 1 - k) & 1];
      const int shift = k * p.bits, digits = 1 << p.bits;
      hipLaunchKernelGGL(sort_count_kernel, dim3(blocks), dim3(256), 0, s, src, counts, rows, shift, digits);
      hipLaunchKernelGGL(sort_scan_kernel, dim3(digits), dim3(64), 0, s, counts, totals, (int)blocks);
      hipLaunchKernelGGL(sort_place_kernel, dim3(blocks), dim3(256), 0, s, src, counts, totals, dst[0], dst[1], rows, shift, p.bits);
      src = SortSource{nullptr, dst[0], dst[1], vocab};
    }
  }
  float* slab = reinterpret_cast<float*>(ws + p.slab);
  auto sums = [&](auto kernel, int64_t units) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)p.pieces, (unsigned)cdiv(units, (int64_t)64)), dim3(64), 0, s, keys, order, dy,
                       dtable, slab, rows, (int)dim, (uint32_t)vocab.size, scale, p.piece);
  };
  constexpr int kWide = sizeof(T) == 2 ? 8 : 4;
  if (dim >= kWide)
    sums(token_sums_kernel<T, TO, kWide>, cdiv(dim, (int64_t)kWide));
  else
    sums(token_sums_kernel<T, TO, 1>, dim);
  if (p.pieces > 1)
    hipLaunchKernelGGL((token_join_kernel<TO>), dim3((unsigned)p.pieces), dim3(1024), 0, s, keys, slab, dtable, rows, (int)dim,
                       (uint32_t)vocab.size, scale, p.piece);
  return check_launch("ferrite_embedding_bwd");
}

template <typename F>
int with_two_types(int a, int b, F&& f) {
  if (a == FERRITE_BF16) return b == FERRITE_BF16 ? f((bf16*)nullptr, (bf16*)nullptr) : f((bf16*)nullptr, (float*)nullptr);
  return b == FERRITE_BF16 ? f((float*)nullptr, (bf16*)nullptr) : f((float*)nullptr, (float*)nullptr);
}

}  // namespace
}  // namespace ferrite

extern "C" int ferrite_internal_embedding(const int64_t* tokens, const void* table, void* out, int64_t rows, int64_t dim,
                                          int64_t vocab, float scale, int indexing, int table_dtype, int out_dtype,
                                          void* stream) {
  using namespace ferrite;
  EmbedPlan p;
  if (!valid_dtype(table_dtype) || !valid_dtype(out_dtype))
    return fail(FERRITE_ERR_INVALID_ARGUMENT, "ferrite_embedding: dtype must be FERRITE_F32 or FERRITE_BF16");
  if (!embed_plan(rows, dim, vocab, p)) return fail(FERRITE_ERR_INVALID_ARGUMENT, "ferrite_embedding: sizes out of range");
  if (rows == 0) return FERRITE_OK;
  if (!tokens || !table || !out) return fail(FERRITE_ERR_INVALID_ARGUMENT, "ferrite_embedding: null pointer");
  hipStream_t s = static_cast<hipStream_t>(stream);
  return with_two_types(table_dtype, out_dtype, [&](auto* te, auto* to) {
    typedef std::remove_pointer_t<decltype(te)> TE;
    typedef std::remove_pointer_t<decltype(to)> TO;
    // Sixteen bytes of the wider type to a thread: eight floats in two accesses leave every other 16 bytes to the next instruction.
    // us, 51690 rows of 1716 floats, in fours / in eights: 109 / 127.
    constexpr int kWide = sizeof(TE) == 2 && sizeof(TO) == 2 ? 8 : 4;
    const int64_t units = dim >= kWide ? cdiv(dim, (int64_t)kWide) : dim, total = rows * units;
    const dim3 grid((unsigned)std::min<int64_t>(cdiv(total, (int64_t)256), 1 << 16));
    auto go = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, tokens, static_cast<const TE*>(table), static_cast<TO*>(out), total,
                         (int)units, (int)dim, vocab, scale, indexing != 0);
    };
    if (dim >= kWide)
      go(lookup_kernel<TE, TO, kWide>);
    else
      go(lookup_kernel<TE, TO, 1>);
    return check_launch("ferrite_embedding");
  });
}

extern "C" int64_t ferrite_internal_embedding_bwd_workspace(int64_t rows, int64_t dim, int64_t vocab) {
  ferrite::EmbedPlan p;
  return ferrite::embed_plan(rows, dim, vocab, p) ? p.bytes : -1;
}

extern "C" int ferrite_internal_embedding_bwd(const int64_t* tokens, const void* dy, void* dtable, int64_t rows, int64_t dim,
                                              int64_t vocab, int64_t padding, float scale, int indexing, int dy_dtype,
                                              int table_dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace ferrite;
  EmbedPlan p;
  if (!valid_dtype(table_dtype) || !valid_dtype(dy_dtype))
    return fail(FERRITE_ERR_INVALID_ARGUMENT, "ferrite_embedding_bwd: dtype must be FERRITE_F32 or FERRITE_BF16");
  if (!embed_plan(rows, dim, vocab, p)) return fail(FERRITE_ERR_INVALID_ARGUMENT, "ferrite_embedding_bwd: sizes out of range");
  if (!dtable || (rows && (!tokens || !dy))) return fail(FERRITE_ERR_INVALID_ARGUMENT, "ferrite_embedding_bwd: null pointer");
  if (p.bytes && (!workspace || workspace_bytes < p.bytes || (reinterpret_cast<uintptr_t>(workspace) & 15)))
    return fail(FERRITE_ERR_INVALID_ARGUMENT, "ferrite_embedding_bwd: null, unaligned or small workspace");
  return with_two_types(dy_dtype, table_dtype, [&](auto* g, auto* d) {
    typedef std::remove_pointer_t<decltype(g)> T;
    typedef std::remove_pointer_t<decltype(d)> TO;
    return embed_bwd(tokens, static_cast<const T*>(dy), static_cast<TO*>(dtable), rows, dim, Vocab{vocab, padding, indexing != 0}, scale, p,
                     static_cast<char*>(workspace), static_cast<hipStream_t>(stream));
  });
}
