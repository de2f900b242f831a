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
  char* part;   // workspace, or null: every workgroup takes one whole head
  int64_t qs[3], ks[3], vs[3];  // element strides of q, k_new and v_new: sequence, head, node
  int B, H, Hkv, G, T, L, rows;  // rows = G T
  int row_groups;                // workgroups' row blocks per head
  int groups, least;             // workgroups that share the work, and steps of one at least
  int begin;                     // what beginning a (head, row group) costs, in steps
  float c;                       // |scale| log2(e)
  uint32_t flip;                 // sign bits to flip in q (a negative scale)
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

// Bytes that a descriptor's range covers at most. What lies past it is past every range: loads there read zeros and touch
// no memory.
constexpr uint32_t kMostBytes = 0xfffe0000u;

// A word of values, infinities and NaN as zeros.
__device__ __forceinline__ uint32_t finite_of(uint32_t x, float) { return (x & 0x7f800000u) == 0x7f800000u ? 0 : x; }
__device__ __forceinline__ uint32_t finite_of(uint32_t x, bf16) {
  return ((x & 0x7f800000u) == 0x7f800000u ? 0 : x & 0xffff0000u) | ((x & 0x7f80u) == 0x7f80u ? 0 : x & 0xffffu);
}

template <typename T, int D>
struct Step {
  static constexpr int NS = kTiles<T>, KEYS = 16 * NS, RB = D * (int)sizeof(T), KB = RB / 64, VD = RB / 64;
  u32x4 k[NS][KB];           // key 16 n + lane % 16, bytes 64 c + 16 (lane / 16)
  uint32_t v[4 * NS][VD];    // key 16 n + 4 (lane / 16) + i, bytes (lane % 16) RB / 16 ..

  // Rows first .. of what the descriptor covers, `bytes` from one to the next; past its range they are zeros. Read once
  // (non-temporal).
  __device__ __forceinline__ void load_k(__amdgpu_buffer_rsrc_t rs, uint32_t first, uint32_t bytes, int lane) {
    const uint32_t at = first + (lane & 15) * bytes + (lane >> 4) * 16;
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int c = 0; c < KB; ++c)
        k[n][c] = __builtin_amdgcn_raw_buffer_load_b128(rs, (int)(at + n * 16 * bytes + c * 64), 0, 2);
  }
  __device__ __forceinline__ void load_v(__amdgpu_buffer_rsrc_t rs, uint32_t first, uint32_t bytes, int lane) {
    const uint32_t at = first + 4 * (lane >> 4) * bytes + (lane & 15) * (RB / 16);
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t off = at + (16 * n + i) * bytes;
        if constexpr (VD == 2) {
          const u32x2 x = __builtin_amdgcn_raw_buffer_load_b64(rs, (int)off, 0, 2);
          v[4 * n + i][0] = x[0];
          v[4 * n + i][1] = x[1];
        } else {
#pragma unroll
          for (int w = 0; w < VD; w += 4) {
            const u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(rs, (int)(off + 4 * w), 0, 2);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[4 * n + i][w + e] = x[e];
          }
        }
      }
  }
  // Values of the keys whose bit of `there` (bit 0: the step's first) is not set, whatever they hold, as zeros.
  __device__ __forceinline__ void drop_absent(uint32_t there, int lane) {
    there >>= 4 * (lane >> 4);
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t keep = there >> (16 * n + i) & 1 ? ~0u : 0u;
#pragma unroll
        for (int w = 0; w < VD; ++w) v[4 * n + i][w] &= keep;
      }
  }
  // Whether any value is infinite or NaN; those as zeros.
  __device__ __forceinline__ bool not_finite() const {
    uint32_t most[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 4 * NS; ++i)
#pragma unroll
      for (int w = 0; w < VD; ++w) {
        most[0] = max(most[0], v[i][w] & 0x7fffffffu);
        if (sizeof(T) == 2) most[1] = max(most[1], v[i][w] << 16 & 0x7fffffffu);
      }
    return max(most[0], most[1]) >= 0x7f800000u;
  }
  __device__ __forceinline__ void drop_not_finite() {
#pragma unroll
    for (int i = 0; i < 4 * NS; ++i)
#pragma unroll
      for (int w = 0; w < VD; ++w) v[i][w] = finite_of(v[i][w], T{});
  }
};

// Two weights as bf16 pairs that together are within 2^-16 of each: `high`, the bits of a float below the weight cut to bf16, and
// the rest of the weight (exact in f32), rounded. A weight's one rounding to bf16 would be off by up to 2^-8, and keys of one score
// would all be off by the same, while l sums the weights as they are. `high` is less than the weight, so the rest is 0 for a weight of 0
// alone, and an infinite value times both stays what it is times the weight.
struct WeightPair {
  uint32_t high, rest;
};
__device__ __forceinline__ WeightPair split_weights(float a, float b) {
  const uint32_t x = __builtin_elementwise_sub_sat(__float_as_uint(a), 1u), y = __builtin_elementwise_sub_sat(__float_as_uint(b), 1u);
  return {__builtin_amdgcn_perm(y, x, 0x07060302u),
          pack_bf16(a - __uint_as_float(x & 0xffff0000u), b - __uint_as_float(y & 0xffff0000u))};
}

// O^T += V^T P^T; o[j] row i stands for element i D / 16 + j.
// bf16 values: two bf16 products, of the weights' high parts and of their rests (f32 ones run at a sixteenth of the rate).
template <int D>
__device__ __forceinline__ void add_pv(const Step<bf16, D>& st, const f32x4 (&p)[2], f32x4 (&o)[D / 16]) {
  u32x4 high, rest;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const WeightPair x = split_weights(p[w / 2][w % 2 * 2], p[w / 2][w % 2 * 2 + 1]);
    high[w] = x.high;
    rest[w] = x.rest;
  }
#pragma unroll
  for (int j = 0; j < D / 16; ++j) {
    u32x4 a;
#pragma unroll
    for (int w = 0; w < 4; ++w)
      a[w] = __builtin_amdgcn_perm(st.v[2 * w + 1][j / 2], st.v[2 * w][j / 2], j % 2 ? 0x07060302u : 0x05040100u);
    o[j] = mfma16(a, high, o[j], bf16{});
    o[j] = mfma16(a, rest, o[j], bf16{});
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

// The lanes' nodes, each with its parent (-2: no node): bit s of the result for node `lane` says whether it sees node s (its ancestors and itself); 0
// where the node, or one that it hangs on, is absent (its parent neither -1 nor an earlier node). By doubling: after
// round r a lane holds its 2^r nearest ancestors and points past them.
__device__ __forceinline__ uint64_t ancestors(int parent, int lane) {
  int up = parent < -1 || parent >= lane ? -2 : parent;
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

// The work is a line of steps: sequence by sequence, (head, row group) by (head, row group), the steps of its cached keys and
// of its nodes (one step for a sequence that has no place in the cache), and in front of them places without work, as many
// as it costs to begin. It is cut evenly over the workgroups, so each has at most one (head, row group) that it shares with
// workgroups before it and one with workgroups behind it; their states go to its two slots of the workspace.
__device__ __forceinline__ int pos_of(const TreeArgs& a, int b) { return a.pos[min(b, a.B - 1)]; }
__device__ __forceinline__ bool in_cache(const TreeArgs& a, int p) { return p >= 0 && p <= a.L - a.T; }
template <int KEYS>
__device__ __forceinline__ int steps_at(const TreeArgs& a, int b, int p) {
  return b >= a.B ? 0 : in_cache(a, p) ? (p + KEYS - 1) / KEYS + (a.T + KEYS - 1) / KEYS : 1;
}
// The sums over the lanes up to each, and over all.
__device__ __forceinline__ int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // rows of 16 lanes: from 1, 2, 4 and 8 lanes below
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // the last lane of rows 0 and 2 to rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // lane 31 to rows 2 and 3
  return x;
}
__device__ __forceinline__ int last_lane(int x) { return __builtin_amdgcn_readlane(x, 63); }

// Steps of a workgroup, and whether every (head, row group) takes whole shares of the line (the last one's end empty): so it is
// where the workgroups suffice for that, and none then has a second one to begin.
struct Shares {
  int share, begin;
  bool apart;
  // Of the first 64 sequences, a lane each: position, steps, and places on the line up to each (of one head and row group).
  int p, steps, upto;
  __device__ __forceinline__ int pieces(int n) const { return (n + share - 1) / share; }
  __device__ __forceinline__ int span(int n) const { return n == 0 ? 0 : apart ? pieces(n) * share : n + begin; }
};
template <int KEYS>
__device__ __forceinline__ Shares shares_of(const TreeArgs& a, int lane) {
  const int per_seq = a.Hkv * a.row_groups;
  Shares s;
  s.p = pos_of(a, lane);
  s.steps = steps_at<KEYS>(a, lane, s.p);
  s.upto = wave_scan(s.steps);
  int total = last_lane(s.upto);
  for (int b0 = 64; b0 < a.B; b0 += 64) total += last_lane(wave_scan(steps_at<KEYS>(a, b0 + lane, pos_of(a, b0 + lane))));
  s.share = __builtin_amdgcn_readfirstlane(max((total * per_seq + a.groups - 1) / a.groups, a.least));
  const int upto = wave_scan(s.pieces(s.steps));
  int pieces = last_lane(upto);
  for (int b0 = 64; b0 < a.B; b0 += 64)
    pieces += last_lane(wave_scan(s.pieces(steps_at<KEYS>(a, b0 + lane, pos_of(a, b0 + lane)))));
  s.apart = (int64_t)pieces * per_seq <= a.groups;
  if (s.apart) {
    s.begin = 0;
    s.upto = upto * s.share;
  } else {
    s.begin = a.begin;
    s.upto += min(lane + 1, a.B) * a.begin;
    s.share = __builtin_amdgcn_readfirstlane(max(((total + a.B * a.begin) * per_seq + a.groups - 1) / a.groups, a.least));
  }
  return s;
}

// Where a workgroup is on the line: steps [s0, s1) of the hr-th (head, row group) of sequence b, [cur, end) its own.
template <int KEYS>
struct Cursor {
  int b, p, steps, hr, s0, cur, end;
  Shares sh;

  // false: nothing to do.
  __device__ __forceinline__ bool start(const TreeArgs& a, int lane) {
    const int per_seq = a.Hkv * a.row_groups;
    int seq_at = 0;  // where on the line the sequence begins
    sh = Shares{1, 0, false, 0, 0, 0};
    if (a.part) {
      sh = shares_of<KEYS>(a, lane);
      cur = (int)blockIdx.x * sh.share;
      end = cur + sh.share;
      int before = 0, x = sh.p, mine = sh.steps, upto = sh.upto;
      for (int b0 = 0;;) {
        const uint64_t past = __ballot((before + upto) * per_seq > cur);
        if (past) {
          const int at = __builtin_ctzll(past);
          b = b0 + at;
          p = __builtin_amdgcn_readlane(x, at);
          steps = __builtin_amdgcn_readlane(mine, at);
          seq_at = (before + __builtin_amdgcn_readlane(upto, at) - sh.span(steps)) * per_seq;
          break;
        }
        before += last_lane(upto);
        if ((b0 += 64) >= a.B) return false;
        x = pos_of(a, b0 + lane);
        mine = steps_at<KEYS>(a, b0 + lane, x);
        upto = wave_scan(sh.span(mine));
      }
    } else {
      b = (int)(blockIdx.x / per_seq);
      p = pos_of(a, b);
      steps = steps_at<KEYS>(a, b, p);
      cur = (int)(blockIdx.x % per_seq) * steps;
      end = cur + steps;
    }
    b = __builtin_amdgcn_readfirstlane(b);
    p = __builtin_amdgcn_readfirstlane(p);
    steps = __builtin_amdgcn_readfirstlane(steps);
    cur = __builtin_amdgcn_readfirstlane(cur);
    end = __builtin_amdgcn_readfirstlane(end);
    const int at = cur - __builtin_amdgcn_readfirstlane(seq_at), span = __builtin_amdgcn_readfirstlane(sh.span(steps));
    hr = __builtin_amdgcn_readfirstlane(at / span);
    s0 = at - hr * span - sh.begin;
    if (s0 < 0) {
      cur -= s0;
      s0 = 0;
    }
    return cur < end;
  }
  __device__ __forceinline__ int s1() const { return min(steps, s0 + end - cur); }
  // To the next (head, row group); false: none left.
  __device__ __forceinline__ bool next(const TreeArgs& a) {
    cur += steps - s0 + sh.begin;  // of shares that stand apart there is no next
    if (sh.apart || cur >= end) return false;
    s0 = 0;
    if (++hr == a.Hkv * a.row_groups) {
      hr = 0;
      if (++b >= a.B) return false;
      p = __builtin_amdgcn_readfirstlane(pos_of(a, b));
      steps = steps_at<KEYS>(a, b, p);
    }
    return true;
  }
};

// A node's value that is infinite or NaN counts for the rows that see it and for no other, but the products would have it times a
// weight of 0 for those: it is left out there, and here is what such values of the nodes from .. to - 1 add to elements
// d .. d + 3 of node t, which is there: along its line of parents. (Their weights, above 0, change nothing of that; one of a score of
// -inf counts as above 0 too.)
template <typename T>
__device__ __forceinline__ f32x4 not_finite_of(const TreeArgs& a, int b, const T* vn, int t, int from, int to, int d) {
  f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
  for (int s = t; s >= from; s = a.parents[(int64_t)b * a.T + s])
    if (s < to)
      for (int i = 0; i < 4; ++i) {
        const float v = (float)vn[s * a.vs[2] + d + i];
        x[i] += __builtin_isfinite(v) ? 0.f : v;
      }
  return x;
}

// Slots of `rows` rows, two to a workgroup, the second for a first piece of a (head, row group): (m, l) of each, then the unnormalised outputs.
struct Parts {
  f32x2* ml;   // [slots, rows]
  float* acc;  // [slots, rows, D]
};
__host__ __device__ inline int64_t parts_bytes(int64_t slots, int64_t rows, int64_t d) { return slots * rows * (8 + 4 * d); }
__device__ __forceinline__ Parts parts_of(char* ws, int64_t slots, int64_t rows) {
  return {reinterpret_cast<f32x2*>(ws), reinterpret_cast<float*>(ws + slots * rows * 8)};
}

// Where the query fragments would not fit in a wave's registers beside O and two steps of keys and values they lie in LDS.
template <typename T, int D, int NT>
constexpr bool kQueriesInLds = NT * D * (int)sizeof(T) / 64 >= 16 || D * (int)sizeof(T) >= 512;
// Two steps of keys and values in registers, one under way, where they fit; else the next step's keys are loaded when the scores
// are done, and its values when it begins.
template <typename T, int D, int NT>
constexpr bool kPingPong = D == 64 || (D == 128 && (sizeof(T) == 2 || NT < 4));
// Waves that a SIMD is to hold.
template <typename T, int D, int NT>
constexpr int kWavesPerSimd = NT == 1 ? (D == 64 ? 3 : D == 128 ? 2 : 1) : NT == 2 && D == 64 ? 2 : 1;
// LDS: the queries, and after the last step the waves' O with its (m, l).
template <typename T, int D, int NT, int W>
constexpr int kTreeLds = std::max(kQueriesInLds<T, D, NT> ? NT * (D * (int)sizeof(T) / 64) * 1024 : 0,
                                  W * NT * 16 * (D + 4 + 2) * 4);

// The nodes' rows of the cache, from element `at` of it, by the workgroup that has the first step of nodes of the head's first
// rows: behind the steps, when those rows are in the L2, where all other waits are over.
template <typename T, int D, int W>
__device__ __forceinline__ void write_nodes(const TreeArgs& a, const T* kn, const T* vn, int64_t at, uint64_t there) {
  constexpr int VEC = D * (int)sizeof(T) / 16, N = 4;
  u32x4* const kc = reinterpret_cast<u32x4*>(static_cast<T*>(a.kc) + at);
  u32x4* const vc = reinterpret_cast<u32x4*>(static_cast<T*>(a.vc) + at);
  for (int e0 = threadIdx.x; e0 < a.T * VEC; e0 += N * 64 * W) {
    u32x4 xk[N], xv[N];
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int e = min(e0 + u * 64 * W, a.T * VEC - 1);
      xk[u] = reinterpret_cast<const u32x4*>(kn + e / VEC * a.ks[2])[e % VEC];
      xv[u] = reinterpret_cast<const u32x4*>(vn + e / VEC * a.vs[2])[e % VEC];
    }
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int e = e0 + u * 64 * W;
      if (e >= a.T * VEC || !(there >> (e / VEC) & 1)) continue;
      kc[e] = xk[u];
      vc[e] = xv[u];
    }
  }
}

// A row group of 16 NT rows, its steps dealt to W waves. Long caches: bound by HBM (8 sequences of 2047 to 8188 keys, 32 heads of
// 128, 4 nodes, bf16: 104 us, 6.5 TB/s; two steps of 16 KB are under way in each of 8 waves a CU). Short ones: by what follows one
// another in a wave with two or three steps. 4 heads of 512 keys of 128, bf16: 10.9 us, of them from inside 9.5: 0.5 to find the place,
// 2.4 until the queries and ancestors are there, 4.7 for the steps (the first one's keys and values are on their way since the place
// is known), 0.7 for the nodes' rows, 1.2 through LDS and out. f32, 39 rows for each of 2 heads of 64 over 747, 1868 and 2988 keys:
// 12.7 us, of them 1.1, 3.5, 3.2, 0.1 and 1.9 (and the join).
template <typename T, int D, int NT, int W>
__global__ __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(kWavesPerSimd<T, D, NT>, kWavesPerSimd<T, D, NT>))) void tree_attn_kernel(TreeArgs a) {
  typedef Step<T, D> S;
  constexpr int NS = S::NS, KEYS = S::KEYS, KB = S::KB, VE = D / 16, ROWS = 16 * NT;
  constexpr bool QL = kQueriesInLds<T, D, NT>;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  u32x4* const queries = reinterpret_cast<u32x4*>(lds);  // [NT KB][64]
  float* const red = reinterpret_cast<float*>(lds);              // [W][16 NT][D + 4]
  float *const red_m = red + W * NT * 16 * (D + 4), *const red_l = red_m + W * NT * 16;  // [W][16 NT]

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, q0 = lane & 15;
  Cursor<KEYS> at;
  if (!at.start(a, lane)) return;
  do {
    // readfirstlane: descriptors must be provably uniform, or every load becomes a loop over the lanes' distinct ones.
    const int b = __builtin_amdgcn_readfirstlane(at.b), p = __builtin_amdgcn_readfirstlane(at.p);
    const int s0 = __builtin_amdgcn_readfirstlane(at.s0), s1 = __builtin_amdgcn_readfirstlane(at.s1());
    const int hr = __builtin_amdgcn_readfirstlane(at.hr), h = hr / a.row_groups, row0 = (hr - h * a.row_groups) * ROWS;
    const bool valid = in_cache(a, p);
    const int cached = valid ? p : 0, cached_steps = (cached + KEYS - 1) / KEYS;

    // This wave's steps: s0 + wave and every W-th after it, below s1. Those before whole_to are 16 NS cached keys each, then come the
    // cache's last keys, from cached_steps on the nodes.
    const int64_t base = ((int64_t)b * a.Hkv + h) * a.L * D;
    const T* kn = static_cast<const T*>(a.kn) + b * a.ks[0] + h * a.ks[1];
    const T* vn = static_cast<const T*>(a.vn) + b * a.vs[0] + h * a.vs[1];
    const uint32_t kbytes = (uint32_t)a.ks[2] * sizeof(T), vbytes = (uint32_t)a.vs[2] * sizeof(T);
    int s = valid ? s0 + wave : s1;
    const int whole_to = cached / KEYS;
    // A load past the last step goes out too, from past every range, which reads nothing: behind a branch the waits would count on
    // none of it and wait for the step under way too.
    auto range = [](const T* x, uint32_t bytes) {
      return __builtin_amdgcn_make_buffer_rsrc(uniform_ptr(const_cast<T*>(x)), (short)0, (int)bytes, 0x00020000);
    };
    auto load_k = [&](S& st, int at) {
      const bool old = at < cached_steps;
      const uint32_t step = old ? S::RB : kbytes, first = (uint32_t)(at - (old ? 0 : cached_steps)) * KEYS * step;
      st.load_k(range(old ? static_cast<const T*>(a.kc) + base : kn, old ? (uint32_t)cached * S::RB : (a.T - 1) * step + S::RB),
                                 at < s1 ? first : kMostBytes, at < s1 ? step : 0, lane);
    };
    auto load_v = [&](S& st, int at) {
      const bool old = at < cached_steps;
      const uint32_t step = old ? S::RB : vbytes, first = (uint32_t)(at - (old ? 0 : cached_steps)) * KEYS * step;
      st.load_v(range(old ? static_cast<const T*>(a.vc) + base : vn, old ? (uint32_t)cached * S::RB : (a.T - 1) * step + S::RB),
                                 at < s1 ? first : kMostBytes, at < s1 ? step : 0, lane);
    };
    const int parent = a.parents[(int64_t)b * a.T + min(lane, a.T - 1)];
    S even;
    load_k(even, s);
    if constexpr (kPingPong<T, D, NT>) load_v(even, s);

    // Query rows: row r is node r % T of head h G + r / T. In place of rows past the last it is read again, and not stored. No load
    // behind a branch of its own: each would be waited for alone.
    u32x4 q[NT][QL ? 1 : KB];
    int node[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = min(row0 + n * 16 + q0, a.rows - 1);
      const int gh = r / a.T;
      node[n] = r - gh * a.T;
      if (QL && wave != 0) continue;
      const char* src = reinterpret_cast<const char*>(static_cast<const T*>(a.q) + b * a.qs[0] + (h * a.G + gh) * a.qs[1] + node[n] * a.qs[2]);
#pragma unroll
      for (int c = 0; c < KB; ++c) {
        const u32x4 x = *reinterpret_cast<const u32x4*>(src + c * 64 + g * 16) ^ a.flip;
        if constexpr (QL)
          queries[(n * KB + c) * 64 + lane] = x;
        else
          q[n][c] = x;
      }
    }
    uint64_t there = 0, line = 0;
    const bool drafts = valid && s1 > cached_steps;
    if (drafts) {
      line = ancestors(lane < a.T ? parent : -2, lane);
      there = __ballot(line != 0);
    }
    if (QL) __syncthreads();

    float m[NT], l[NT];
    int odd_values = 0;  // whether nodes' values that are not finite were left out
    f32x4 o[NT][VE];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n] = -INFINITY;
      l[n] = 0.f;
#pragma unroll
      for (int j = 0; j < VE; ++j) o[n][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    // Step `at`: scores of its keys, the running maximum (m, in units of log2) and sum, O.
    auto add_step = [&](S& st, int at, auto&& after_scores) {
      f32x4 x[NT][NS];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int t = 0; t < NS; ++t) x[n][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < KB; ++c) {
          u32x4 y;
          if constexpr (QL)
            y = queries[(n * KB + c) * 64 + lane];
          else
            y = q[n][c];
#pragma unroll
          for (int t = 0; t < NS; ++t) x[n][t] = mfma16(st.k[t][c], y, x[n][t], T{});
        }
      }
      after_scores();
      if (at >= whole_to) {  // not every row sees every key: bit k of `sees` is the step's key k
        const bool old = at < cached_steps;
        const int first = old ? 0 : (at - cached_steps) * KEYS;
        if (!old) {
          st.drop_absent((uint32_t)(there >> first), lane);
          if (__any(st.not_finite())) {
            st.drop_not_finite();
            odd_values = 1;
          }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const uint64_t mine = __shfl((unsigned long long)line, node[n], kWave) >> first;
          const uint32_t sees = (old ? (1u << (cached - at * KEYS)) - 1 : (uint32_t)mine) >> (4 * g);
#pragma unroll
          for (int t = 0; t < NS; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) x[n][t][i] = sees >> (16 * t + i) & 1 ? x[n][t][i] : -INFINITY;
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float mx = -INFINITY;
#pragma unroll
        for (int t = 0; t < NS; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) mx = fmaxf(mx, x[n][t][i]);
        mx = fmaxf(m[n], max16(mx) * a.c);
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
            x[n][t][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[n][t][i], a.c, -ref));
            l[n] += x[n][t][i];
          }
        add_pv<D>(st, x[n], o[n]);
      }
    };

    // The next step's loads are under way while one is added.
    if constexpr (kPingPong<T, D, NT>) {
      S odd;
      auto load = [&](S& st, int at) {
        asm volatile("" ::: "memory");  // the queries' LDS reads stay in their step
        load_k(st, at);
        load_v(st, at);
      };
      while (s < s1) {
        load(odd, s + W);
        add_step(even, s, [] {});
        s += W;
        if (s >= s1) break;
        load(even, s + W);
        add_step(odd, s, [] {});
        s += W;
      }
    } else {
      for (; s < s1; s += W) {
        asm volatile("" ::: "memory");
        load_v(even, s);
        add_step(even, s, [&] { load_k(even, s + W); });
      }
    }

    if (drafts && s0 <= cached_steps && row0 == 0) write_nodes<T, D, W>(a, kn, vn, base + (int64_t)p * D, there);

    // The waves' states through LDS: weights 2^(m_w - max), then the sums over the waves of a row block in their order, to the
    // output or to this workgroup's slot.
    if (QL) __syncthreads();
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int row = wave * NT * 16 + n * 16 + q0;
      const float lt = sum16(l[n]);
      if (g == 0) {
        red_m[row] = m[n];
        red_l[row] = lt;
      }
      // A lane's elements: 4 VE in a row from g D / 4.
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < VE; j += 4)
          *reinterpret_cast<f32x4*>(&red[row * (D + 4) + g * (D / 4) + i * VE + j]) =
              f32x4{o[n][j][i], o[n][j + 1][i], o[n][j + 2][i], o[n][j + 3][i]};
    }
    if (lane == 0) reinterpret_cast<int*>(red)[wave * ROWS * (D + 4) + D] = odd_values;
    __syncthreads();
    odd_values = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) odd_values |= reinterpret_cast<const int*>(red)[w * ROWS * (D + 4) + D];
    const bool whole = s0 == 0 && s1 == at.steps;
    const Parts parts = parts_of(a.part, 2 * (int64_t)a.groups, ROWS);
    for (int e = threadIdx.x; e < ROWS * (D / 4); e += 64 * W) {
      const int r = e / (D / 4), d = e % (D / 4) * 4;  // row r of the row group
      if (row0 + r >= a.rows) break;
      float mx = -INFINITY, lsum = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) mx = fmaxf(mx, red_m[r + w * ROWS]);
      const float ref = mx == -INFINITY ? 0.f : mx;
      f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float f = __builtin_amdgcn_exp2f(red_m[r + w * ROWS] - ref);
        lsum += red_l[r + w * ROWS] * f;
        sum += *reinterpret_cast<const f32x4*>(&red[(r + w * ROWS) * (D + 4) + d]) * f;
      }
      if (odd_values && there >> (row0 + r) % a.T & 1)
        sum += not_finite_of(a, b, vn, (row0 + r) % a.T, (max(s0, cached_steps) - cached_steps) * KEYS, (s1 - cached_steps) * KEYS, d);
      if (whole) {
        const int gh = (row0 + r) / a.T, t = row0 + r - gh * a.T;
        T* out = static_cast<T*>(a.out) + (((int64_t)b * a.T + t) * a.H + h * a.G + gh) * D + d;
        const bool zero = !(there >> t & 1);
        float y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = !valid ? NAN : zero ? 0.f : sum[i] / lsum;
        if constexpr (sizeof(T) == 2)
          *reinterpret_cast<u32x2*>(out) = u32x2{pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3])};
        else
          *reinterpret_cast<f32x4*>(out) = f32x4{y[0], y[1], y[2], y[3]};
      } else {
        const int64_t i = (2 * (int64_t)blockIdx.x + (s0 == 0)) * ROWS + r;
        *reinterpret_cast<f32x4*>(parts.acc + i * D + d) = sum;
        if (d == 0) parts.ml[i] = f32x2{mx, lsum};
      }
    }
    __syncthreads();

  } while (at.next(a));
}

// Many query rows (bf16): W waves of 32 rows each over the same keys, which go through LDS once for all of them. A stage of KEYS keys
// and values is copied straight into LDS (four stages, up to three under way), 16-byte pieces of a row
// in an order of its own, so that neither the reads of 32 rows' pieces (keys) nor the transposing ones (values) meet in a bank.
// S^T = K Q^T and O^T = V^T P^T in 32x32 tiles: a lane has 16 of a tile's 32 scores of one query.
//
// A step is two clusters, the softmax of its scores (VALU) and its product with V and the next step's with K (matrix units), each
// behind a barrier, and the second half of the waves is one cluster behind the first: of a SIMD's two waves one is on the
// VALU while the other is on the matrix units. Bound by LDS and the matrix units, neither of which is fed without a pause: of a
// step's 2.9 us (256 heads of 1088 to 4160 keys) the reads of keys and values by all eight waves, 128 KB of each, at 128 bytes a clock
// and the transposing ones at 64, take 3100 cycles, 1.3 us, and the products 3000, 1000 of them those of the weights' rests
// (without these a step takes 2.3 us). 64 rows to a wave would halve the reads and leave one wave to a SIMD, and nothing to set against
// its softmax. 16 sequences of 1008 to 4032 keys, 8 key heads of 128, 256 rows each: 84 us (without the rests 72), 34 GFLOP of nodes
// that are there in 81 of products.
template <int D>
struct WideShape {
  static constexpr int W = D == 256 ? 4 : 8, KEYS = D == 256 ? 32 : 64, RB = 2 * D, PIECES = RB / 16, ROWS = 32 * W;
  static constexpr int STAGE = 2 * KEYS * RB;                     // keys, then values
  static constexpr int COPIES = STAGE / 16 / (64 * W);            // per thread
  static constexpr int LDS = std::max(4 * STAGE, ROWS * (D + 4) * 4);
  // Where in its row a piece lies, and which piece lies there.
  static __device__ __forceinline__ int swapped(int row, int piece) { return (piece ^ ((row & 3) << 2 | (row >> 2 & 3))) & (PIECES - 1); }
  static __device__ __forceinline__ int place(int row, int piece) { return row * RB + swapped(row, piece) * 16; }
};

template <int D>
__global__ __launch_bounds__(64 * WideShape<D>::W) void tree_wide_kernel(TreeArgs a) {
  typedef WideShape<D> C;
  constexpr int KEYS = C::KEYS, RB = C::RB, W = C::W, ROWS = C::ROWS, NT = KEYS / 32;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  float* const red = reinterpret_cast<float*>(lds);  // [ROWS][D + 4]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 5, q0 = lane & 31;
  Cursor<KEYS> at;
  if (!at.start(a, lane)) return;
  do {
    // readfirstlane: descriptors must be provably uniform, or every load becomes a loop over the lanes' distinct ones.
    const int b = __builtin_amdgcn_readfirstlane(at.b), p = __builtin_amdgcn_readfirstlane(at.p);
    const int s0 = __builtin_amdgcn_readfirstlane(at.s0), s1 = __builtin_amdgcn_readfirstlane(at.s1());
    const int hr = __builtin_amdgcn_readfirstlane(at.hr), h = hr / a.row_groups, row0 = (hr - h * a.row_groups) * ROWS;
    const bool valid = in_cache(a, p);
    const int cached = valid ? p : 0, cached_steps = (cached + KEYS - 1) / KEYS, whole_to = cached / KEYS;
    const int to = valid ? s1 : s0;
    const int64_t base = ((int64_t)b * a.Hkv + h) * a.L * D;
    const bf16* kn = static_cast<const bf16*>(a.kn) + b * a.ks[0] + h * a.ks[1];
    const bf16* vn = static_cast<const bf16*>(a.vn) + b * a.vs[0] + h * a.vs[1];
    const uint32_t kbytes = (uint32_t)a.ks[2] * 2, vbytes = (uint32_t)a.vs[2] * 2;
    const bool mine = row0 + wave * 32 < a.rows;  // whether this wave has rows; it copies in any case

    const int parent = a.parents[(int64_t)b * a.T + min(lane, a.T - 1)];
    // Query rows, as B operands: row r is node r % T of head h G + r / T; in place of rows past the last it is read again.
    bf16x8 q[D / 16];
    const int r = min(row0 + wave * 32 + q0, a.rows - 1), gh = r / a.T, node = r - gh * a.T;
    {
      const char* src = reinterpret_cast<const char*>(static_cast<const bf16*>(a.q) + b * a.qs[0] + (h * a.G + gh) * a.qs[1] + node * a.qs[2]);
#pragma unroll
      for (int c = 0; c < D / 16; ++c)
        q[c] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(src + c * 32 + g * 16) ^ a.flip);
    }
    uint64_t there = 0, line = 0;
    const bool drafts = valid && s1 > cached_steps;
    if (drafts) {
      line = ancestors(lane < a.T ? parent : -2, lane);
      there = __ballot(line != 0);
      line = __shfl((unsigned long long)line, node, kWave);
    }
    // Step `s` into its stage; one past the last from past every range, so that the copies under way can be counted.
    auto copy = [&](int s) {
      const bool old = s < cached_steps;
      const int from = (s - (old ? 0 : cached_steps)) * KEYS;
      char* const stage = lds + (s - s0) % 4 * C::STAGE;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint32_t step = old ? RB : half ? vbytes : kbytes;
        const bf16* src = old ? static_cast<const bf16*>(half ? a.vc : a.kc) + base : half ? vn : kn;
        const u32x4 rsrc = buffer_rsrc(src, old ? (uint32_t)cached * RB : (a.T - 1) * step + RB);
#pragma unroll
        for (int u = 0; u < C::COPIES / 2; ++u) {
          const int piece = (u * W + wave) * 64 + lane, row = piece / C::PIECES;
          const uint32_t off = (uint32_t)(from + row) * step + C::swapped(row, piece) * 16;
          // Absent nodes, whatever they hold, are zeros: their weight is 0.
          const bool on = s < to && (old || (from + row < kMaxNodes && (there >> ((from + row) & 63) & 1)));
          dma16(rsrc, stage + half * KEYS * RB + (u * W + wave) * 1024, on ? off : kMostBytes);
        }
      }
    };
    const bool leads = wave < W / 2;
    wait_vmem<0>();  // from here on the copies alone are counted
    copy(s0);
    copy(s0 + 1);
    copy(s0 + 2);

    // A lane's places in a stage: of its key row's pieces; of its values, which of 16 keys lie in rows 4 g .. and 8 + 4 g .. (a row's
    // order of pieces is the same 16 rows on).
    int koff[D / 16], voff[D / 32][2];
#pragma unroll
    for (int c = 0; c < D / 16; ++c) koff[c] = C::place(q0, 2 * c + g);
#pragma unroll
    for (int j = 0; j < D / 32; ++j)
#pragma unroll
      for (int hi = 0; hi < 2; ++hi)
        voff[j][hi] = KEYS * RB + C::place(8 * hi + 4 * g + (lane & 15) / 4, 4 * j + (lane >> 4 & 1) * 2 + (lane & 3) / 2) + (lane & 1) * 8;

    int odd_values = 0;  // whether nodes' values that are not finite were left out
    // Of a step of nodes a wave reads the values that it copied (it has waited for them), and makes those zeros.
    auto clean = [&](int s) {
      if (s < cached_steps || s >= to) return;
      char* const values = lds + (s - s0) % 4 * C::STAGE + KEYS * RB + wave * 1024 + lane * 16;
#pragma unroll
      for (int u = 0; u < C::COPIES / 2; ++u) {
        u32x4& at = *reinterpret_cast<u32x4*>(values + u * W * 1024);
        const u32x4 is = at;
        u32x4 fin;
#pragma unroll
        for (int e = 0; e < 4; ++e) fin[e] = finite_of(is[e], bf16{});
        if (fin[0] != is[0] || fin[1] != is[1] || fin[2] != is[2] || fin[3] != is[3]) {
          at = fin;
          odd_values = 1;
        }
      }
    };

    float m = -INFINITY, l = 0.f;
    f32x16 o[D / 32], x[NT];
#pragma unroll
    for (int j = 0; j < D / 32; ++j)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[j][i] = 0.f;

    auto scores = [&](int s) {
      const char* ks = lds + (s - s0) % 4 * C::STAGE;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) x[t][i] = 0.f;
#pragma unroll
      for (int c = 0; c < D / 16; ++c)
#pragma unroll
        for (int t = 0; t < NT; ++t) mma32(*reinterpret_cast<const bf16x8*>(ks + koff[c] + t * 32 * RB), q[c], x[t]);
    };
    // A wave copies step s + 3 when it begins the product of step s with V: all waves have left that of s - 1, whose stage it
    // takes. Before the barrier at which the leading waves begin that product, every wave has waited for its copies of step
    // s + 1: they when they leave the softmax of s, the others when they leave the product of s - 1.
    wait_vmem<2 * C::COPIES>();
    clean(s0);
    lds_barrier();
    if (mine && s0 < to) scores(s0);
    if (!leads) lds_barrier();
    for (int s = s0; s < to; ++s) {
      if (!leads) {
        wait_vmem<C::COPIES>();
        clean(s + 1);
      }
      lds_barrier();
      __builtin_amdgcn_s_setprio(0);
      u32x4 high[KEYS / 16], rest[KEYS / 16];  // the weights' two parts
      if (mine) {
        if (s >= whole_to) {  // not every row sees every key: bit k of `sees` is the step's key k
          const bool old = s < cached_steps;
          const uint64_t sees = (old ? (1ull << (cached - s * KEYS)) - 1 : line >> (s - cached_steps) * KEYS) >> (4 * g);
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) x[t][i] = sees >> (32 * t + 8 * (i / 4) + i % 4) & 1 ? x[t][i] : -INFINITY;
        }
        float mx = -INFINITY;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < 16; ++i) mx = fmaxf(mx, x[t][i]);
        mx = fmaxf(m, lane32_max(mx) * a.c);
        const float ref = mx == -INFINITY ? 0.f : mx;
        if (__any(mx > m)) {
          const float f = __builtin_amdgcn_exp2f(m - ref);
          l *= f;
#pragma unroll
          for (int j = 0; j < D / 32; ++j)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[j][i] *= f;
        }
        m = mx;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            x[t][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[t][i], a.c, -ref));
            l += x[t][i];
          }
        // 16 keys to an operand: a lane's weights are of keys 4 g .. and 8 + 4 g .., and so are its values.
#pragma unroll
        for (int c = 0; c < KEYS / 16; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const WeightPair w = split_weights(x[c / 2][c % 2 * 8 + 2 * e], x[c / 2][c % 2 * 8 + 2 * e + 1]);
            high[c][e] = w.high;
            rest[c][e] = w.rest;
          }
      }
      if (leads) {
        wait_vmem<C::COPIES>();
        clean(s + 1);
      }
      lds_barrier();
      copy(s + 3);
      if (!mine) continue;
      // O, then the scores of the next step (behind the last one of zeros, for nothing), so that the weights are gone when those
      // arrive: reads from LDS are kept AHEAD operands ahead of the one that they feed, in this order (a read's latency is some six
      // products; left to itself the compiler has every product wait for its own read). 4 and 5 are alike, 6 takes five registers more than
      // there are at head dim 128 (the kernel's fastest run 86 us and 84).
      const char *ks = lds + (s + 1 - s0) % 4 * C::STAGE, *vs = lds + (s - s0) % 4 * C::STAGE;
      constexpr int PV = KEYS / 16 * D / 32, ALL = PV + NT * D / 16, AHEAD = 5;
      auto fetch = [&](int i) {
        if (i >= PV) return *reinterpret_cast<const bf16x8*>(ks + koff[(i - PV) / NT] + (i - PV) % NT * 32 * RB);
        typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
        const int c = i / (D / 32), j = i % (D / 32);
        auto half = [&](int hi) {
          return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              reinterpret_cast<lds_i16x4*>(reinterpret_cast<uintptr_t>(vs + voff[j][hi] + c * 16 * RB)));
        };
        const i16x4 lo = half(0), hi = half(1);
        typedef short i16x8 __attribute__((ext_vector_type(8)));
        return __builtin_bit_cast(bf16x8, i16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]});
      };
      __builtin_amdgcn_s_setprio(1);  // before the SIMD's other wave, whose softmax waits for no one
      bf16x8 ring[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) ring[i] = fetch(i);
#pragma unroll
      for (int i = 0; i < ALL; ++i) {
        __builtin_amdgcn_sched_barrier(0);
        if (i < PV) {
          const int c = i / (D / 32), j = i % (D / 32);
          mma32(ring[i % AHEAD], __builtin_bit_cast(bf16x8, high[c]), o[j]);
          mma32(ring[i % AHEAD], __builtin_bit_cast(bf16x8, rest[c]), o[j]);
        } else {
          const int c = (i - PV) / NT, t = (i - PV) % NT;
          if (c == 0) {
#pragma unroll
            for (int e = 0; e < 16; ++e) x[t][e] = 0.f;
          }
          mma32(ring[i % AHEAD], q[c], x[t]);
        }
        if (i + AHEAD < ALL) ring[i % AHEAD] = fetch(i + AHEAD);
      }
    }
    if (leads) lds_barrier();

    // O through LDS, rows whole, to the output or to this workgroup's slot.
    wait_vmem<0>();
    lds_barrier();
    {
      const float lt = lane32_sum(l);
      const int row = wave * 32 + q0;
#pragma unroll
      for (int j = 0; j < D / 32; ++j)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
          *reinterpret_cast<f32x4*>(&red[row * (D + 4) + 32 * j + 2 * i + 4 * g]) = f32x4{o[j][i], o[j][i + 1], o[j][i + 2], o[j][i + 3]};
      if (g == 0) *reinterpret_cast<f32x2*>(&red[row * (D + 4) + D]) = f32x2{m, lt};
      odd_values = __any(odd_values);
      if (lane == 0) reinterpret_cast<int*>(red)[wave * 32 * (D + 4) + D + 2] = odd_values;
    }
    __syncthreads();
    odd_values = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) odd_values |= reinterpret_cast<const int*>(red)[w * 32 * (D + 4) + D + 2];
    if (drafts && s0 <= cached_steps && row0 == 0) write_nodes<bf16, D, W>(a, kn, vn, base + (int64_t)p * D, there);
    const bool whole = s0 == 0 && s1 == at.steps;
    const Parts parts = parts_of(a.part, 2 * (int64_t)a.groups, ROWS);
    for (int e = threadIdx.x; e < ROWS * (D / 4); e += 64 * W) {
      const int r = e / (D / 4), d = e % (D / 4) * 4;  // row r of the row group
      if (row0 + r >= a.rows) break;
      f32x4 sum = *reinterpret_cast<const f32x4*>(&red[r * (D + 4) + d]);
      const f32x2 ml = *reinterpret_cast<const f32x2*>(&red[r * (D + 4) + D]);
      if (odd_values && there >> (row0 + r) % a.T & 1)
        sum += not_finite_of(a, b, vn, (row0 + r) % a.T, (max(s0, cached_steps) - cached_steps) * KEYS, (s1 - cached_steps) * KEYS, d);
      if (whole) {
        const int gh = (row0 + r) / a.T, t = row0 + r - gh * a.T;
        bf16* out = static_cast<bf16*>(a.out) + (((int64_t)b * a.T + t) * a.H + h * a.G + gh) * D + d;
        const bool zero = !(there >> t & 1);
        float y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = !valid ? NAN : zero ? 0.f : sum[i] / ml[1];
        *reinterpret_cast<u32x2*>(out) = u32x2{pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3])};
      } else {
        const int64_t i = (2 * (int64_t)blockIdx.x + (s0 == 0)) * ROWS + r;
        *reinterpret_cast<f32x4*>(parts.acc + i * D + d) = sum;
        if (d == 0) parts.ml[i] = ml;
      }
    }
    __syncthreads();
  } while (at.next(a));
}

// Joins what several workgroups have of a row. The pieces of a row are dealt to LINES threads for every four elements, each adding
// up N at a time under a running maximum; then the lines in their order. A workgroup takes kJoinRows rows, of one row group.
template <int D, int LINES>
constexpr int kJoinRows = LINES == 1 ? 16 : 1024 / D / LINES;
template <typename T, int D, int KEYS, int LINES, int N>
__global__ __launch_bounds__(256) void tree_join_kernel(TreeArgs a, int slot_rows) {
  constexpr int PER = D / 4, ROWS = 256 / PER / LINES;
  __shared__ __attribute__((aligned(16))) float red[LINES][ROWS][D + 4];  // D sums, m, l
  const int b = blockIdx.z, h = blockIdx.y, block = (int)blockIdx.x * kJoinRows<D, LINES>, lane = threadIdx.x & 63;
  const int per_seq = a.Hkv * a.row_groups;
  const int d = threadIdx.x % PER * 4, row = threadIdx.x / PER % ROWS, part = threadIdx.x / PER / ROWS;
  const int p = pos_of(a, b), parent = lane < a.T ? a.parents[(int64_t)b * a.T + lane] : -2;
  const Shares sh = shares_of<KEYS>(a, lane);
  int before = 0;
  for (int b0 = 0; b0 < b; b0 += 64)
    before += last_lane(wave_scan(b0 + lane < b ? sh.span(steps_at<KEYS>(a, b0 + lane, b0 ? pos_of(a, b0 + lane) : sh.p)) : 0));
  const int share = sh.share, steps = steps_at<KEYS>(a, b, p);
  const int x0 = before * per_seq + (h * a.row_groups + block / slot_rows) * sh.span(steps) + sh.begin;
  const int w0 = x0 / share, used = (x0 + steps - 1) / share - w0 + 1;
  if (used == 1) return;  // one workgroup had it all
  const uint64_t there = __ballot(ancestors(parent, lane) != 0);  // divided: the sequence has its place
  const Parts parts = parts_of(a.part, 2 * (int64_t)a.groups, slot_rows);
  const int to = min(block + kJoinRows<D, LINES>, a.rows);
  for (int r0 = block; r0 < to; r0 += ROWS) {
    const int r = min(r0 + row, to - 1);
    auto at = [&](int k) { return (int64_t)(2 * (w0 + k) + (k == 0)) * slot_rows + r % slot_rows; };
    float m = -INFINITY, l = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int c = part; c < used; c += N * LINES) {
      f32x2 ml[N];
      f32x4 x[N];
#pragma unroll
      for (int u = 0; u < N; ++u) {
        const int64_t i = at(min(c + u * LINES, used - 1));
        ml[u] = parts.ml[i];
        x[u] = *reinterpret_cast<const f32x4*>(parts.acc + i * D + d);
      }
      float mx = m;
#pragma unroll
      for (int u = 0; u < N; ++u) mx = fmaxf(mx, ml[u][0]);
      const float ref = mx == -INFINITY ? 0.f : mx, f = __builtin_amdgcn_exp2f(m - ref);
      l *= f;
      acc *= f;
#pragma unroll
      for (int u = 0; u < N; ++u) {
        const bool on = c + u * LINES < used;  // else the last piece again, whose values need not be finite
        const float w = __builtin_amdgcn_exp2f(ml[u][0] - ref);
        l += on ? ml[u][1] * w : 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] += on ? x[u][e] * w : 0.f;
      }
      m = mx;
    }
    if constexpr (LINES > 1) {
      *reinterpret_cast<f32x4*>(&red[part][row][d]) = acc;
      if (d == 0) *reinterpret_cast<f32x2*>(&red[part][row][D]) = f32x2{m, l};
      __syncthreads();
      float mx = -INFINITY;
#pragma unroll
      for (int u = 0; u < LINES; ++u) mx = fmaxf(mx, red[u][row][D]);
      const float ref = mx == -INFINITY ? 0.f : mx;
      l = 0.f;
      acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int u = 0; u < LINES; ++u) {
        const float w = __builtin_amdgcn_exp2f(red[u][row][D] - ref);
        l += red[u][row][D + 1] * w;
        acc += *reinterpret_cast<const f32x4*>(&red[u][row][d]) * w;
      }
      __syncthreads();
    }
    if (part != 0 || r0 + row >= to) continue;
    const int gh = r / a.T, t = r - gh * a.T;
    T* out = static_cast<T*>(a.out) + (((int64_t)b * a.T + t) * a.H + h * a.G + gh) * D + d;
    const bool zero = !(there >> t & 1);
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = zero ? 0.f : acc[i] / l;
    if constexpr (sizeof(T) == 2)
      *reinterpret_cast<u32x2*>(out) = u32x2{pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3])};
    else
      *reinterpret_cast<f32x4*>(out) = f32x4{y[0], y[1], y[2], y[3]};
  }
}

constexpr int64_t kMostSteps = 1 << 30;

struct Plan {
  bool wide;
  int tiles, waves;  // of tree_attn_kernel
  int64_t keys, slot_rows, row_groups, groups, least, begin;
  bool split;
};

Plan plan_for(int64_t b, int64_t h, int64_t hkv, int64_t t, int64_t max_len, int64_t d, int dtype) {
  const bool half = dtype == FERRITE_BF16;
  const int64_t rows = h / hkv * t;
  Plan p;
  // Many rows share keys and values through LDS (the call's us so, and with 32 rows to a wave, 64 of 64 elements): 8 sequences of 4096
  // keys, 4 key heads of 128 elements, 32 rows each 26.6 and 20.6, 48 rows 27.7 and 29.4, 64 rows 28.5 and 30.7, 96 rows 30.8 and
  // 36.5, 128 rows 32.0 and 41.9; of 64 elements 64 rows 21.4 and 19.3, 96 rows 22.4 and 26.6; of 256 elements 24 and 32 rows 39.7 and
  // 40.7 against 33.5 and 35.3, 48 rows 45.1 and 53.5, 64 rows 47.9 and 56.2. Few heads lose by it: 64 rows of one sequence's 4 heads
  // over 2048 keys 19.9 and 15.5.
  p.wide = half && rows > (d == 64 ? 64 : 32);
  p.tiles = rows <= 16 ? 1 : rows <= 32 || d > 128 ? 2 : 4;
  p.waves = 4;
  p.keys = p.wide ? (d == 256 ? 32 : 64) : half ? 32 : 16;
  p.slot_rows = p.wide ? (d == 256 ? 128 : 256) : 16 * p.tiles;
  p.row_groups = cdiv(rows, p.slot_rows);
  const int64_t heads = b * hkv * p.row_groups, steps = cdiv(max_len, p.keys) + cdiv(t, p.keys);
  // Workgroups that are resident together, and steps that one takes at least (one to a wave; with two to a wave one head of
  // 1024 keys takes 15.3 us and not 13.4, f32 with 700 keys of 256 elements 34.9 and not 19.6).
  const int per_cu = p.wide ? 1 : p.tiles == 1 ? (d == 64 ? 3 : d == 128 ? 2 : 1) : p.tiles == 2 && d == 64 ? 2 : 1;
  p.groups = 256 * per_cu;
  p.least = p.wide ? 2 : p.waves;
  // A wide head takes some 12 us to begin and to store, and a step 2.9 (16 sequences of 1008 to 4032 keys, 8 heads each, 256
  // rows, the kernel's fastest run: 85 us; with 0 it takes 101, with 4 85, with 8 87); else it is about a step of each wave (eight heads
  // of 1024 keys 12.3 us and 14.3 with 0, f32, 32 nodes of four heads to each of 16 key heads of 1024 keys 33.4 and 44.3, and none
  // slower).
  p.begin = p.wide ? 6 : p.waves;
  const bool eight = !p.wide && p.tiles == 1 && d <= 128;
  // Whole heads need no second kernel. Short ones, or many, lose less by uneven shares than that one costs: 256 heads of 1024
  // keys of 128 elements take 23.2 us whole and 26.4 cut (f32 46.1 and 47.4), 512 of 64 elements 19.3 and 25.9; but 32 of
  // 128 elements 18.5 whole and 11.3 cut, 128 of them 20.5 and 16.2, f32 64 of 512 keys 24.2 and 16.2.
  // More heads than fill the chip four times are whole too: 2048 heads of 4096 keys 625 us, cut 668; of 8192 1218 and 1284.
  p.split = heads < 4 * p.groups && steps > (p.wide ? 8 : heads >= 256 ? 128 : eight ? 32 : 16);
  if (p.split) {
    p.groups = std::min(p.groups, cdiv(heads * steps, p.least));
  } else {
    p.groups = heads;
    // Eight waves to a head while that brings more waves to a CU (4 heads of 512 keys: 10.6 us, with four waves 13.6); 1024
    // heads of 512 keys fill it with four (32.2 us, with eight 45.6; f32 66.9 and 81.1).
    if (eight && steps > 8 && heads < 512) p.waves = 8;
  }
  return p;
}

template <typename T, int D, int KEYS>
int tree_finish(const TreeArgs& a, const Plan& p, hipStream_t s) {
  const int rc = check_launch("ferrite_tree_attention");
  if (rc != FERRITE_OK || !p.split) return rc;
  auto join = [&](auto lines, auto at_once) {
    hipLaunchKernelGGL((tree_join_kernel<T, D, KEYS, lines.value, at_once.value>),
                       dim3((unsigned)cdiv(a.rows, kJoinRows<D, lines.value>), (unsigned)a.Hkv, (unsigned)a.B), dim3(256), 0, s, a,
                       (int)p.slot_rows);
  };
  // Few heads are cut into many pieces, and four lines add up a row's: one head of 64 rows, 8192 keys 20.2 us and not 34.3, eight of
  // 8 rows, 4096 keys 12.9 and 15.1; of many rows there are lines enough (32 heads of 96 rows 30.3 us and 29.0, of 128 rows 32.6
  // and 30.2).
  const int64_t heads = (int64_t)a.B * a.Hkv;
  if (p.groups >= 8 * heads * a.row_groups && heads * a.rows <= 2048)
    join(std::integral_constant<int, 4>{}, std::integral_constant<int, 8>{});
  else
    join(std::integral_constant<int, 1>{}, std::integral_constant<int, 4>{});
  return check_launch("ferrite_tree_attention");
}

template <typename T, int D, int NT, int W>
int tree_launch(const TreeArgs& a, const Plan& p, hipStream_t s) {
  constexpr int bytes = kTreeLds<T, D, NT, W>;
  if (bytes > (64 << 10)) {
    const int rc = allow_lds(reinterpret_cast<const void*>(&tree_attn_kernel<T, D, NT, W>), bytes, s, "ferrite_tree_attention");
    if (rc != FERRITE_OK) return rc;
  }
  hipLaunchKernelGGL((tree_attn_kernel<T, D, NT, W>), dim3((unsigned)p.groups), dim3(64 * W), bytes, s, a);
  return tree_finish<T, D, Step<T, D>::KEYS>(a, p, s);
}

template <int D>
int tree_wide_launch(const TreeArgs& a, const Plan& p, hipStream_t s) {
  typedef WideShape<D> C;
  const int rc = allow_lds(reinterpret_cast<const void*>(&tree_wide_kernel<D>), C::LDS, s, "ferrite_tree_attention");
  if (rc != FERRITE_OK) return rc;
  hipLaunchKernelGGL(tree_wide_kernel<D>, dim3((unsigned)p.groups), dim3(64 * C::W), C::LDS, s, a);
  return tree_finish<bf16, D, C::KEYS>(a, p, s);
}

int check_tree(int64_t b, int64_t h, int64_t hkv, int64_t t, int64_t max_len, int64_t d, int dtype) {
  const std::string n = "ferrite_tree_attention";
  if (!valid_dtype(dtype)) return fail(FERRITE_ERR_INVALID_ARGUMENT, n + ": dtype must be FERRITE_F32 or FERRITE_BF16");
  if (b < 0 || hkv < 1 || b > 65535 || hkv > 65535 || h < hkv || h > 65535 || h % hkv)
    return fail(FERRITE_ERR_INVALID_ARGUMENT, n + ": need 0 <= b <= 65535 and up to 65535 query heads, a multiple of the key heads");
  if (t < 1 || t > kMaxNodes) return fail(FERRITE_ERR_INVALID_ARGUMENT, n + ": need 1 to 64 nodes");
  if (d != 64 && d != 128 && d != 256) return fail(FERRITE_ERR_INVALID_ARGUMENT, n + ": head dim must be 64, 128 or 256");
  if (max_len < 1 || max_len > kMostBytes / (d * (dtype == FERRITE_BF16 ? 2 : 4)))
    return fail(FERRITE_ERR_INVALID_ARGUMENT, n + ": need max_len >= 1, and a head's cache within 4 GiB less 128 KiB");
  // Places on the line of steps are 32-bit numbers.
  const Plan p = plan_for(b, h, hkv, t, max_len, d, dtype);
  if (b * hkv * p.row_groups > kMostSteps / 512 || b * hkv * p.row_groups * (cdiv(max_len, 16) + 64) > kMostSteps)
    return fail(FERRITE_ERR_INVALID_ARGUMENT, n + ": too many heads for caches of this length");
  return FERRITE_OK;
}

}  // namespace
}  // namespace ferrite

extern "C" int64_t ferrite_internal_tree_attention_workspace(int64_t b, int64_t h, int64_t hkv, int64_t t, int64_t max_len,
                                                             int64_t d, int dtype) {
  using namespace ferrite;
  if (check_tree(b, h, hkv, t, max_len, d, dtype) != FERRITE_OK) return -1;
  const Plan p = plan_for(b, h, hkv, t, max_len, d, dtype);
  return p.split ? parts_bytes(2 * p.groups, p.slot_rows, d) : 0;
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
  for (int i = 5; i < 9; i += 3)
    if (strides[i] < 0 || (t - 1) * strides[i] * (dtype == FERRITE_BF16 ? 2 : 4) > (int64_t)kMostBytes - 1024)
      return fail(FERRITE_ERR_INVALID_ARGUMENT, "ferrite_tree_attention: a head's new keys or values span 4 GiB");
  // Nodes' rows are written while other workgroups read the inputs.
  const int64_t size = dtype == FERRITE_BF16 ? 2 : 4, cache = b * hkv * max_len * d * size;
  bool apart = !overlap(k_cache, cache, v_cache, cache);
  const void* inputs[3] = {q, k_new, v_new};
  for (int i = 0; i < 3; ++i) {
    const int64_t* st = strides + 3 * i;
    const int64_t span = ((b - 1) * st[0] + ((i ? hkv : h) - 1) * st[1] + (t - 1) * st[2] + d) * size;
    apart = apart && !overlap(inputs[i], span, k_cache, cache) && !overlap(inputs[i], span, v_cache, cache);
  }
  const Plan p = plan_for(b, h, hkv, t, max_len, d, dtype);
  TreeArgs a{q, k_new, v_new, k_cache, v_cache, pos, parents, out, nullptr, {}, {}, {}, (int)b, (int)h, (int)hkv, (int)(h / hkv),
             (int)t, (int)max_len, (int)(h / hkv * t), (int)p.row_groups, (int)p.groups, (int)p.least, (int)p.begin,
             std::max(fabsf(scale) * kLog2e, 1e-37f),  // above 0, so that it times -inf is -inf
             scale >= 0 ? 0u : dtype == FERRITE_BF16 ? 0x80008000u : 0x80000000u};
  for (int i = 0; i < 3; ++i) {
    a.qs[i] = strides[i];
    a.ks[i] = strides[3 + i];
    a.vs[i] = strides[6 + i];
  }
  if (p.split) {
    if (!workspace || !a16(workspace) || workspace_bytes < parts_bytes(2 * p.groups, p.slot_rows, d))
      return fail(FERRITE_ERR_INVALID_ARGUMENT, "ferrite_tree_attention: workspace too small or unaligned");
    a.part = static_cast<char*>(workspace);
  }
  if (!apart)
    return fail(FERRITE_ERR_INVALID_ARGUMENT, "ferrite_tree_attention: the caches overlap each other or q, k_new or v_new");
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto tiles = [&](auto* e, auto D) {
    typedef std::remove_pointer_t<decltype(e)> T;
    if constexpr (sizeof(T) == 2) {
      if (p.wide) return tree_wide_launch<D.value>(a, p, s);
    }
    if constexpr (D.value <= 128) {
      if (p.waves == 8) return tree_launch<T, D.value, 1, 8>(a, p, s);
    }
    if constexpr (D.value == 64 || (D.value == 128 && sizeof(T) == 4)) {
      if (p.tiles == 4) return tree_launch<T, D.value, 4, 4>(a, p, s);
    }
    if (p.tiles == 1) return tree_launch<T, D.value, 1, 4>(a, p, s);
    return tree_launch<T, D.value, 2, 4>(a, p, s);
  };
  auto dims = [&](auto* e) {
    if (d == 64) return tiles(e, std::integral_constant<int, 64>{});
    if (d == 128) return tiles(e, std::integral_constant<int, 128>{});
    return tiles(e, std::integral_constant<int, 256>{});
  };
  return dtype == FERRITE_BF16 ? dims((bf16*)nullptr) : dims((float*)nullptr);
}
