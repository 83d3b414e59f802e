// Log probability of one given token per row of logits, the entropy of the row and its most
// probable alternatives, and the gradient of the first two (sm_100a).
//
// Row x with V valid columns, temperature T:  m = max x,  z_j = (x_j - m) / T <= 0,
//   S = sum e^z_j,  A = sum e^z_j z_j,  logp_j = z_j - ln S,  H = ln S - A / S  (both sums have one
// sign, so nothing cancels), and with incoming gradients g (log probability) and h (entropy)
//   dx_j = ((j == token) g - p_j (g + h (logp_j + H))) / T.
// A column of -inf has probability 0 and adds nothing to H.  A row without any finite column is
// empty: log probability -inf, entropy 0, no gradient.  NaN and +inf make the row's results NaN.
// The difference x - m is taken before the scaling, so rows of the type's lowest value neither
// overflow nor become empty.  Every sum is held in 32 bits.
//
// Forward: one pass.  A warp takes tiles of 1 KiB (32 bytes a lane); every lane keeps its own
// running (m, S, A) and rescales S and A once per tile, without a branch.  What bounds it is HBM,
// with the exponentials (16 a clock and SM) close behind: 16-bit logits arrive at 0.7 of their rate.
// A CTA of eight warps takes a row; where rows are few, a cluster of CTAs shares one and joins
// through distributed shared memory (no workspace, no second launch).
//
// Alternatives: by (logit descending, column ascending) the k first columns lie in the k first groups
// of consecutive columns ranked by (their largest logit, their place).  The pass leaves each tile's
// maximum in shared memory; the k first tiles are found by counting how many come before each, and
// read once more: the columns that reach the least of the k maxima (few more than k) are ranked by
// counting, too.  Only where ties or a short row make those many does a selection among the tiles'
// 32-byte vectors come between, which bounds them by k vectors.  (Taking the largest k times over
// cost 1 us an alternative; a binary search for the k-th maximum 6 us.)
#include "wb_logprobs.h"

#include <cooperative_groups.h>
#include <cstdlib>

#include "wb_vec.cuh"

namespace wb {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr float kInf = __builtin_huge_valf();
constexpr float kNaN = __builtin_nanf("");
constexpr float kLowest = -3.402823466e38f;
constexpr float kLn2 = 0.6931471805599453f, kLog2e = 1.4426950408889634f;
constexpr uint32_t kMaxSplits = 8;         // the portable cluster size

template <typename T> constexpr uint32_t kTile = 32u * kVecN<T>;

template <typename T>
__device__ __forceinline__ const T* row_ptr(const LogprobRows& in, uint32_t r) {
  return reinterpret_cast<const T*>(in.logits) + (int64_t)(r / in.inner) * in.stride_outer +
         (int64_t)(r % in.inner) * in.stride_inner;
}

__device__ __forceinline__ int64_t token_of(const LogprobRows& in, uint32_t r) {
  const int64_t o = (int64_t)(r / in.inner) * in.tok_outer + (int64_t)(r % in.inner) * in.tok_inner;
  return in.tokens_i32 ? (int64_t) reinterpret_cast<const int32_t*>(in.tokens)[o]
                       : reinterpret_cast<const int64_t*>(in.tokens)[o];
}

// Elements between the 32-byte boundary at or below a row's first element and that element: tiles
// start at boundaries, so that every tile but the first and the last is read with aligned vectors.
template <typename T>
__device__ __forceinline__ uint32_t misaligned(const T* x) {
  return (uint32_t)(reinterpret_cast<uintptr_t>(x) & 31) / sizeof(T);
}

// Whole numbers in the order of the floats: -0 equals +0, NaN lies above everything; 0 is no number's.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }

// Running maximum and sums, z in units of ln 2.
struct Stats {
  float m = kLowest;
  F2 s{0.f, 0.f}, a{0.f, 0.f};
};

// exp2 of the shift from maximum `from` to `to` >= from; the shift itself, finite, in `shift`
__device__ __forceinline__ float rescale(float from, float to, float c2, float& shift) {
  shift = fmaxf((from - to) * c2, -1e30f);
  return ex2(shift);
}

// The largest element of a vector, NaN left out; -inf where there is nothing else.
template <typename T>
__device__ __forceinline__ float vec_max(const Vec32& v) {
  if constexpr (sizeof(T) == 4) {
    float m = -kInf;
    #pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, __uint_as_float(v.w[i]));
    return m;
  } else {
    using T2 = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
    T2 w[8];
    #pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = *reinterpret_cast<const T2*>(&v.w[i]);
    #pragma unroll
    for (int o = 4; o > 0; o >>= 1) {
      #pragma unroll
      for (int i = 0; i < o; ++i) w[i] = __hmax2(w[i], w[i + o]);
    }
    return fmaxf(fmaxf(to_f32(w[0].x), to_f32(w[0].y)), -kInf);
  }
}

__device__ __forceinline__ void raise(Stats& t, float top, float c2) {
  const float m = fmaxf(t.m, top);
  float shift;
  const float f = rescale(t.m, m, c2, shift);
  t.a = mul2(fma2(t.s, F2{shift, shift}, t.a), F2{f, f});
  t.s = mul2(t.s, F2{f, f});
  t.m = m;
}

template <int N2>
__device__ __forceinline__ void accumulate(Stats& t, const F2 (&x)[N2], float c2) {
  #pragma unroll
  for (int i = 0; i < N2; ++i) {
    const F2 z = mul2(add2(x[i], F2{-t.m, -t.m}), F2{c2, c2});
    const F2 e{ex2(z.x), ex2(z.y)};
    t.s = add2(t.s, e);
    t.a = fma2(e, F2{fmaxf(z.x, -1e30f), fmaxf(z.y, -1e30f)}, t.a);      // 0 * -inf would be NaN
  }
}

struct RowStats { float m, s, a; };

__device__ __forceinline__ RowStats at_max(RowStats t, float m, float c2) {
  float shift;
  const float f = rescale(t.m, m, c2, shift);
  return {m, t.s * f, (t.a + t.s * shift) * f};
}

// Joins the lanes' statistics (all lanes get the result; the order of the additions is fixed).
__device__ __forceinline__ RowStats warp_join(RowStats t, float c2) {
  t = at_max(t, warp_max(t.m), c2);
  return {t.m, warp_sum(t.s), warp_sum(t.a)};
}

template <typename T> constexpr uint32_t kNegInf = sizeof(T) == 4 ? 0xff800000u : 0;
template <> constexpr uint32_t kNegInf<__nv_bfloat16> = 0xff80u;
template <> constexpr uint32_t kNegInf<__half> = 0xfc00u;

// A lane's vector of columns j0 .. j0 + N - 1; what lies outside the row reads as -inf.
template <typename T>
__device__ __forceinline__ Vec32 load_vec(const T* x, uint32_t vocab, int32_t j0) {
  constexpr int N = kVecN<T>;
  Vec32 v;
  if (j0 >= 0 && (uint32_t)j0 + N <= vocab) return load32(x + j0);
  using Bits = std::conditional_t<sizeof(T) == 4, uint32_t, uint16_t>;
  uint32_t e[N];
  #pragma unroll
  for (int i = 0; i < N; ++i) {
    const int32_t j = j0 + i;
    e[i] = j >= 0 && (uint32_t)j < vocab ? (uint32_t) reinterpret_cast<const Bits*>(x)[j] : kNegInf<T>;
  }
  #pragma unroll
  for (int i = 0; i < 8; ++i) v.w[i] = sizeof(T) == 4 ? e[i] : e[2 * i % N] | e[(2 * i + 1) % N] << 16;
  return v;
}

struct RowResult { float m, ln, entropy; bool empty; };

__device__ __forceinline__ RowResult finish(RowStats t) {
  RowResult r;
  r.empty = t.s == 0.f;
  r.m = r.empty ? 0.f : t.m;
  r.ln = r.empty ? kInf : logf(t.s);
  r.entropy = r.empty ? 0.f : r.ln - kLn2 * t.a / t.s;
  return r;
}

__device__ __forceinline__ float logprob(const RowResult& t, float x, float inv_temp) {
  return t.empty ? -kInf : (x - t.m) * inv_temp - t.ln;
}

// The token's logit, loaded before the row: its latency passes under the row's.
template <typename T>
__device__ __forceinline__ float token_logit(const LogprobRows& in, const T* x, int64_t tok) {
  return tok >= 0 && tok < (int64_t)in.vocab ? to_f32(x[tok]) : kNaN;
}

__device__ __forceinline__ void write_row(const LogprobRows& in, const LogprobOut& out, uint32_t r, int64_t tok, float xt, const RowResult& t) {
  out.logprobs[r] = tok >= 0 && tok < (int64_t)in.vocab ? logprob(t, xt, in.inv_temp) : kNaN;
  out.entropy[r] = t.entropy;
  if (out.stats) {
    out.stats[2 * (int64_t)r] = t.m;
    out.stats[2 * (int64_t)r + 1] = t.ln;
  }
}

__device__ __forceinline__ void write_ignored(const LogprobOut& out, uint32_t r) {
  out.logprobs[r] = 0.f;
  out.entropy[r] = 0.f;
  if (out.stats) out.stats[2 * (int64_t)r] = out.stats[2 * (int64_t)r + 1] = 0.f;
}

// Keys of 16-bit types differ in their upper bits only.
template <typename T> constexpr int kKeyShift = 0;
template <> constexpr int kKeyShift<__nv_bfloat16> = 16;
template <> constexpr int kKeyShift<__half> = 13;

// A tile's maximum as it is kept: 16-bit types have room for the tile below the key, lower tiles first.
template <typename T>
__device__ __forceinline__ uint32_t tile_key(uint32_t key, uint32_t tile) {
  constexpr uint32_t kMask = (1u << kKeyShift<T>) - 1;
  return kMask ? (key & ~kMask) | (kMask - tile) : key;
}
static_assert(kLogprobMaxTopVocab / kTile<__half> + 1 < 1u << kKeyShift<__half>);

// Whether tile j comes before tile i.
template <typename T>
__device__ __forceinline__ uint32_t tile_before(uint32_t key_j, uint32_t j, uint32_t key_i, uint32_t i) {
  return kKeyShift<T> ? key_j > key_i : key_j + (j < i) > key_i;
}

// Tiles first, first + step, ... below `end` of a row into this lane's statistics.  Two tiles' loads
// are always under way: one's vector is refilled as soon as it is unpacked.  tops: each tile's
// largest, as a key.
template <typename T, bool TOP>
__device__ __forceinline__ Stats walk(const T* x, uint32_t vocab, uint32_t mis, uint32_t first, uint32_t step, uint32_t end,
                                      uint32_t base, float c2, uint32_t* tops) {
  constexpr int N = kVecN<T>, kDepth = 2;
  const uint32_t lane = threadIdx.x & 31;
  Stats st;
  Vec32 raw[kDepth];
  auto load = [&](int u, uint32_t k) {
    if (k < end) raw[u] = load_vec(x, vocab, (int32_t)(k * kTile<T> + lane * N - mis));
  };
  #pragma unroll
  for (int u = 0; u < kDepth; ++u) load(u, first + u * step);
  #pragma unroll 1
  for (uint32_t t = first; t < end; t += kDepth * step) {
    float top[kDepth];
    #pragma unroll
    for (int u = 0; u < kDepth; ++u) {
      const uint32_t k = t + u * step;
      top[u] = k < end ? vec_max<T>(raw[u]) : -kInf;
      if constexpr (TOP) {
        const uint32_t key = __reduce_max_sync(kFullWarp, order_key(top[u]));
        if (lane == 0 && k < end) tops[k - base] = tile_key<T>(key, k - base);
      }
    }
    raise(st, fmaxf(top[0], top[1]), c2);
    #pragma unroll
    for (int u = 0; u < kDepth; ++u) {
      const uint32_t k = t + u * step;
      if (k >= end) break;
      F2 v[N / 2];
      unpack<T>(raw[u], v);
      load(u, k + kDepth * step);
      accumulate(st, v, c2);
    }
  }
  return st;
}

// Many short rows: a warp takes one after another; the next row's token is under way meanwhile.
template <typename T>
__global__ void __launch_bounds__(kThreads) logprobs_warp_kernel(const LogprobRows in, const LogprobOut out) {
  const uint32_t warps = gridDim.x * kWarps, lane = threadIdx.x & 31;
  const float c2 = in.inv_temp * kLog2e;
  uint32_t r = blockIdx.x * kWarps + threadIdx.x / 32;
  int64_t next = r < in.rows ? token_of(in, r) : 0;
  for (; r < in.rows; r += warps) {
    const int64_t tok = next;
    if (in.rows - r > warps) next = token_of(in, r + warps);
    if (tok == in.ignore_index) {
      if (lane == 0) write_ignored(out, r);
      continue;
    }
    const T* x = row_ptr<T>(in, r);
    const float xt = token_logit(in, x, tok);
    const uint32_t mis = misaligned(x), tiles = (mis + in.vocab + kTile<T> - 1) / kTile<T>;
    const Stats st = walk<T, false>(x, in.vocab, mis, 0, 1, tiles, 0, c2, nullptr);
    const RowStats t = warp_join({st.m, st.s.x + st.s.y, st.a.x + st.a.y}, c2);
    if (lane == 0) write_row(in, out, r, tok, xt, finish(t));
  }
}

// -- alternatives ---------------------------------------------------------------------------------
constexpr uint32_t kTopPerWarp = kLogprobMaxTop / kWarps;                 // selected tiles of one warp
constexpr uint32_t kMaxCandidates = kLogprobMaxTop * kVecN<__nv_bfloat16>;

struct TopShared {
  uint64_t candidates[kMaxCandidates], out[kLogprobMaxTop];   // key << 32 | ~column
  uint32_t picked[kLogprobMaxTop], part[2][kWarps];
  uint32_t n_picked, n_candidates, n_out, least;
};

// A whole number's sum over the CTA; `turn` alternates, so that one barrier a sum is enough.
__device__ __forceinline__ uint32_t cta_count(uint32_t c, TopShared& sh, uint32_t& turn) {
  c = __reduce_add_sync(kFullWarp, c);
  uint32_t* part = sh.part[turn & 1];
  ++turn;
  if ((threadIdx.x & 31) == 0) part[threadIdx.x / 32] = c;
  __syncthreads();
  uint32_t sum = 0;
  #pragma unroll
  for (int i = 0; i < kWarps; ++i) sum += part[i];
  return sum;
}

// Selection of the k first of some groups by (value descending, place ascending): those with a
// value above `value`, and those with that value up to place `last`.  count(f): how many groups f
// holds for.  All are selected where there are at most k of value `low` or more.
struct Selection { uint32_t value, last; };

template <typename Count>
__device__ Selection select_first(uint32_t k, uint32_t low, uint32_t high, uint32_t places, Count count) {
  if (count([&](uint32_t v, uint32_t) { return v >= low; }) <= k) return {low, 0xffffffffu};
  while (low < high) {
    const uint32_t mid = high - (high - low) / 2;
    const uint32_t c = count([&](uint32_t v, uint32_t) { return v >= mid; });
    if (c == k) return {mid, 0xffffffffu};
    if (c > k) low = mid; else high = mid - 1;
  }
  // more than k from `low` on, fewer above it: the first places of that value fill up
  const uint32_t above = count([&](uint32_t v, uint32_t) { return v > low; });
  uint32_t from = 0, to = places;
  while (from < to) {
    const uint32_t mid = from + (to - from) / 2;
    if (above + count([&](uint32_t v, uint32_t p) { return v == low && p <= mid; }) >= k) to = mid; else from = mid + 1;
  }
  return {low, from};
}

// Ranks n distinct candidates by counting; the first k go to `out` in order.
__device__ __forceinline__ void rank_candidates(const uint64_t* c, uint32_t n, uint32_t k, uint64_t* out) {
  for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
    const uint64_t mine = c[i];
    uint32_t rank = 0;
    #pragma unroll 4
    for (uint32_t j = 0; j < n; ++j) rank += c[j] > mine;
    if (rank < k) out[rank] = mine;
  }
}

// The k first columns of tiles [base, base + n), in order, into sh.out.  top: the largest logit of
// these tiles; tops: each tile's, as a key.
template <typename T>
__device__ void find_top(const T* x, uint32_t vocab, uint32_t mis, uint32_t base, uint32_t n, uint32_t k, float top, const uint32_t* tops,
                         TopShared& sh) {
  constexpr int N = kVecN<T>, kShift = kKeyShift<T>;
  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  const uint32_t high = order_key(top) >> kShift;
  uint32_t turn = 0;
  const bool counted = n <= 2 * kThreads;
  if (threadIdx.x == 0) sh.n_picked = sh.n_candidates = 0, sh.least = 1;
  if (counted) {
    __syncthreads();
    const uint32_t i0 = threadIdx.x, i1 = i0 + kThreads;
    const uint32_t key0 = i0 < n ? tops[i0] : 0, key1 = i1 < n ? tops[i1] : 0;
    uint32_t rank0 = 0, rank1 = 0;
    for (uint32_t j = 0; j < n; j += 4) {              // zeros follow the last tile
      const uint4 q = *reinterpret_cast<const uint4*>(tops + j);
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
      #pragma unroll
      for (int u = 0; u < 4; ++u) rank0 += tile_before<T>(w[u], j + u, key0, i0);
      if (n > kThreads) {
        #pragma unroll
        for (int u = 0; u < 4; ++u) rank1 += tile_before<T>(w[u], j + u, key1, i1);
      }
    }
    if (i0 < n && rank0 < k) sh.picked[rank0] = base + i0;
    if (i1 < n && rank1 < k) sh.picked[rank1] = base + i1;
    if (rank0 == k - 1 && i0 < n) sh.least = key0 >> kShift;
    if (rank1 == k - 1 && i1 < n) sh.least = key1 >> kShift;
    if (threadIdx.x == 0) sh.n_picked = min(n, k);
  } else {
    const Selection tiles = select_first(k, 1, high, n, [&](auto holds) {
      uint32_t c = 0;
      for (uint32_t i = threadIdx.x; i < n; i += kThreads) c += holds(tops[i] >> kShift, i);
      return cta_count(c, sh, turn);
    });
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
      const uint32_t v = tops[i] >> kShift;
      if (v > tiles.value || (v == tiles.value && i <= tiles.last)) sh.picked[atomicAdd(&sh.n_picked, 1u)] = base + i;
    }
    if (threadIdx.x == 0) sh.least = tiles.value;
  }
  __syncthreads();
  const uint32_t picked = sh.n_picked, least = sh.least;
  Vec32 raw[kTopPerWarp];
  uint32_t value[kTopPerWarp];                         // the vectors' largest
  int32_t j0[kTopPerWarp];
  #pragma unroll
  for (uint32_t s = 0; s < kTopPerWarp; ++s) {
    const uint32_t p = warp + s * kWarps;
    value[s] = 0;
    if (p >= picked) continue;
    j0[s] = (int32_t)(sh.picked[p] * kTile<T> + lane * N - mis);
    raw[s] = load_vec(x, vocab, j0[s]);
  }
  #pragma unroll
  for (uint32_t s = 0; s < kTopPerWarp; ++s) {
    if (warp + s * kWarps >= picked || j0[s] + N <= 0 || j0[s] >= (int32_t)vocab) continue;      // no column of the row
    value[s] = order_key(vec_max<T>(raw[s])) >> kShift;
  }
  // the columns from `from` on of the vectors that `wanted` takes
  auto collect = [&](uint32_t from, auto wanted) {
    #pragma unroll
    for (uint32_t s = 0; s < kTopPerWarp; ++s) {
      if (value[s] < from || !value[s] || !wanted(value[s], (uint32_t)(j0[s] + N))) continue;
      F2 v[N / 2];
      unpack<T>(raw[s], v);
      #pragma unroll
      for (int e = 0; e < N; ++e) {
        const int32_t j = j0[s] + e;
        const uint32_t key = order_key(e & 1 ? v[e / 2].y : v[e / 2].x);
        if (j >= 0 && j < (int32_t)vocab && key >> kShift >= from) {
          const uint32_t at = atomicAdd(&sh.n_candidates, 1u);
          if (at < kMaxCandidates) sh.candidates[at] = (uint64_t)key << 32 | ~(uint32_t)j;
        }
      }
    }
    __syncthreads();
  };
  collect(least, [](uint32_t, uint32_t) { return true; });
  if (sh.n_candidates > kMaxCandidates) {              // many columns of one value, or fewer than k tiles
    // places: the vectors' first columns, counted from one vector before the row's start
    const Selection vecs = select_first(k, least, high, vocab + N, [&](auto holds) {
      uint32_t c = 0;
      #pragma unroll
      for (uint32_t s = 0; s < kTopPerWarp; ++s) c += value[s] && holds(value[s], (uint32_t)(j0[s] + N));
      return cta_count(c, sh, turn);
    });
    if (threadIdx.x == 0) sh.n_candidates = 0;
    __syncthreads();
    collect(vecs.value, [&](uint32_t v, uint32_t place) { return v > vecs.value || place <= vecs.last; });
  }
  const uint32_t m = sh.n_candidates;
  rank_candidates(sh.candidates, m, k, sh.out);
  if (threadIdx.x == 0) sh.n_out = min(m, k);
  __syncthreads();
}

// A CTA per row, or a cluster of `splits` CTAs.
template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads, 4) logprobs_row_kernel(const LogprobRows in, const LogprobOut out, const uint32_t splits) {
  extern __shared__ __align__(16) uint32_t tops[];       // TOP: the tiles' maxima, and zeros up to a multiple of four
  __shared__ RowStats warps[kWarps], mine;
  __shared__ std::conditional_t<TOP, TopShared, int> shared;
  const uint32_t r = blockIdx.x / splits, split = blockIdx.x % splits;
  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  const int64_t tok = token_of(in, r);
  if (tok == in.ignore_index) {                          // the whole cluster leaves
    if (split == 0) {
      if (threadIdx.x == 0) write_ignored(out, r);
      if ((int)threadIdx.x < out.top_k) {
        out.top_logprobs[(int64_t)r * out.top_k + threadIdx.x] = -kInf;
        out.top_ids[(int64_t)r * out.top_k + threadIdx.x] = -1;
      }
    }
    return;
  }
  const T* x = row_ptr<T>(in, r);
  const float xt = token_logit(in, x, tok);
  const float c2 = in.inv_temp * kLog2e;
  const uint32_t mis = misaligned(x), tiles = (mis + in.vocab + kTile<T> - 1) / kTile<T>;
  const uint32_t per = (tiles + splits - 1) / splits;
  const uint32_t begin = min(split * per, tiles), end = min(begin + per, tiles);
  if (TOP && threadIdx.x < 4) tops[(end - begin) + threadIdx.x] = 0;
  const Stats st = walk<T, TOP>(x, in.vocab, mis, begin + warp, kWarps, end, begin, c2, tops);
  const RowStats w = warp_join({st.m, st.s.x + st.s.y, st.a.x + st.a.y}, c2);
  if (lane == 0) warps[warp] = w;
  __syncthreads();
  // every warp joins the eight: the same operations, the same bits
  RowStats all = warp_join(lane < kWarps ? warps[lane] : RowStats{kLowest, 0.f, 0.f}, c2);
  if constexpr (TOP) find_top(x, in.vocab, mis, begin, end - begin, (uint32_t)out.top_k, all.m, tops, shared);
  if (splits > 1) {
    cg::cluster_group cl = cg::this_cluster();
    if (threadIdx.x == 0) mine = all;
    cl.sync();
    if (split == 0) {
      all = warp_join(lane < splits ? *cl.map_shared_rank(&mine, lane) : RowStats{kLowest, 0.f, 0.f}, c2);
      if constexpr (TOP) {               // at most 8 * 32 candidates, a thread each
        const uint32_t k = (uint32_t)out.top_k, s = threadIdx.x / k, i = threadIdx.x % k;
        uint64_t c = 0;
        if (s < splits) {
          const TopShared* theirs = cl.map_shared_rank(&shared, s);
          if (i < theirs->n_out) c = theirs->out[i];
        }
        if (threadIdx.x == 0) shared.n_candidates = 0;
        __syncthreads();                 // this CTA's own list has been read, too
        if (c) shared.candidates[atomicAdd(&shared.n_candidates, 1u)] = c;
        __syncthreads();
        rank_candidates(shared.candidates, shared.n_candidates, k, shared.out);
        __syncthreads();
      }
    }
    cl.sync();                             // the others' shared memory stays until it has been read
  }
  if (split == 0 && warp == 0) {
    const RowResult t = finish(all);
    if (lane == 0) write_row(in, out, r, tok, xt, t);
    if constexpr (TOP) {
      if (lane < (uint32_t)out.top_k) {
        const uint64_t c = shared.out[lane];
        out.top_logprobs[(int64_t)r * out.top_k + lane] = logprob(t, key_value((uint32_t)(c >> 32)), in.inv_temp);
        out.top_ids[(int64_t)r * out.top_k + lane] = (int64_t)(uint32_t)~(uint32_t)c;
      }
    }
  }
}

// -- gradient -------------------------------------------------------------------------------------
constexpr uint32_t kGradTiles = 16;        // tiles of one warp's work: 16 KiB read, 16 KiB written

// Reads a logit and writes a gradient, once each, at HBM's rate; a warp takes up to 16 tiles of one
// row and shares nothing.  Tiles follow the gradient's alignment.  Where the logits' rows lie
// otherwise (views whose rows are not multiples of 32 bytes), and at the ends of a row, lanes take
// single elements side by side instead of vectors.
template <typename T>
__global__ void __launch_bounds__(kThreads) logprobs_grad_kernel(const LogprobRows in, const LogprobGrad g, const uint32_t segs,
                                                                 const uint64_t units) {
  constexpr int N = kVecN<T>;
  const uint64_t unit = (uint64_t)blockIdx.x * kWarps + threadIdx.x / 32;
  if (unit >= units) return;
  const uint32_t r = (uint32_t)(unit / segs), seg = (uint32_t)(unit % segs), lane = threadIdx.x & 31;
  const int64_t tok = token_of(in, r);
  const T* x = row_ptr<T>(in, r);
  T* d = reinterpret_cast<T*>(g.grad) + (int64_t)r * g.cols;
  const uint32_t mis = misaligned(d);
  const float m = g.stats[2 * (int64_t)r], ln = g.stats[2 * (int64_t)r + 1], h = g.entropy[r];
  float glp = g.g_logprobs ? g.g_logprobs[r * g.g_logprobs_stride] : 0.f;
  float gh = g.g_entropy ? g.g_entropy[r * g.g_entropy_stride] : 0.f;
  const bool dead = tok == in.ignore_index || ln == kInf;
  if (dead) glp = gh = 0.f;
  else if (tok < 0 || tok >= (int64_t)in.vocab) glp = kNaN;
  // dx = p (a + b log2 p), and onehot at the token
  const float c2 = in.inv_temp * kLog2e, l2 = ln * kLog2e;
  const float a = -in.inv_temp * (glp + gh * h), b = -in.inv_temp * gh * kLn2, onehot = glp * in.inv_temp;
  auto grad2 = [&](F2 v) {
    const F2 z = fma2(add2(v, F2{-m, -m}), F2{c2, c2}, F2{-l2, -l2});
    return mul2(F2{ex2(z.x), ex2(z.y)}, fma2(F2{b, b}, F2{fmaxf(z.x, -1e30f), fmaxf(z.y, -1e30f)}, F2{a, a}));
  };
  const bool vectors = misaligned(x) == mis;
  const uint32_t tiles = (mis + g.cols + kTile<T> - 1) / kTile<T>;
  const uint32_t begin = seg * kGradTiles, end = min(begin + kGradTiles, tiles);
  #pragma unroll 2
  for (uint32_t t = begin; t < end; ++t) {
    const int32_t tile0 = (int32_t)(t * kTile<T> - mis), j0 = tile0 + lane * N;
    const bool padding = j0 >= (int32_t)in.vocab;
    if (vectors && j0 >= 0 && (uint32_t)j0 + N <= (padding ? g.cols : in.vocab)) {
      F2 v[N / 2];
      if (dead || padding) {
        #pragma unroll
        for (int i = 0; i < N / 2; ++i) v[i] = {0.f, 0.f};
      } else {
        unpack<T>(load32(x + j0), v);
        #pragma unroll
        for (int i = 0; i < N / 2; ++i) v[i] = grad2(v[i]);
        if (tok >= j0 && tok < j0 + N) {
          #pragma unroll
          for (int i = 0; i < N / 2; ++i) {
            if (tok == j0 + 2 * i) v[i].x += onehot;
            if (tok == j0 + 2 * i + 1) v[i].y += onehot;
          }
        }
      }
      store32(d + j0, pack<T>(v));
    } else {
      // a lane that passes the row's ends: its own elements; rows that lie otherwise: side by side
      const int32_t first = vectors ? j0 : tile0 + (int32_t)lane, step = vectors ? 1 : 32;
      float v[N];
      #pragma unroll
      for (int e = 0; e < N; ++e) {
        const int32_t j = first + e * step;
        v[e] = !dead && j >= 0 && j < (int32_t)in.vocab ? to_f32(x[j]) : -kInf;
      }
      #pragma unroll
      for (int e = 0; e < N; ++e) {
        const int32_t j = first + e * step;
        const float y = j < (int32_t)in.vocab && !dead ? grad2({v[e], v[e]}).x + (j == tok ? onehot : 0.f) : 0.f;
        if (j >= 0 && j < (int32_t)g.cols) d[j] = from_f32<T>(y);
      }
    }
  }
}

template <typename F>
cudaError_t by_type(uint32_t dtype, F f) {
  switch (dtype) {
    case DT_BF16: return f(__nv_bfloat16{});
    case DT_F16: return f(__half{});
    case DT_F32: return f(float{});
    default: return cudaErrorInvalidValue;
  }
}

bool ok(const LogprobRows& in) { return in.rows < 0x7fffffffu && in.vocab >= 1 && in.vocab <= kLogprobMaxColumns && in.inner >= 1; }

template <typename T>
cudaError_t launch_rows(const LogprobRows& in, const LogprobOut& out, int sms, cudaStream_t stream) {
  const uint32_t tiles = (in.vocab + kTile<T> - 1) / kTile<T> + 1;
  // A warp a row: no barrier, no second join.  For rows of up to four tiles, of which a CTA's eight
  // warps would find no two; and for up to 32 where the rows fill half of the GPU's warps.
  if (!out.top_k && (tiles <= 5 || (tiles <= 33 && in.rows >= (uint32_t)sms * 16))) {
    const uint32_t cap = (uint32_t)sms * 4, grid = (in.rows + kWarps - 1) / kWarps;
    logprobs_warp_kernel<T><<<grid < cap ? grid : cap, kThreads, 0, stream>>>(in, out);
    return cudaGetLastError();
  }
  uint32_t splits = 1;
  const uint64_t most = (uint64_t)sms * (out.top_k ? 2 : 4);
  while (splits < kMaxSplits && (uint64_t)in.rows * splits * 2 <= most && tiles >= splits * 2 * kWarps) splits *= 2;
  if (getenv("WB_SPLITS")) splits = atoi(getenv("WB_SPLITS"));
  const uint32_t per = (tiles + splits - 1) / splits;
  const size_t shared = out.top_k ? 4 * (size_t)per + 16 : 0;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(in.rows * splits);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = shared;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = splits;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  auto kernel = out.top_k ? logprobs_row_kernel<T, true> : logprobs_row_kernel<T, false>;
  return cudaLaunchKernelEx(&cfg, kernel, in, out, splits);
}

}  // namespace

cudaError_t launch_token_logprobs(const LogprobRows& in, const LogprobOut& out, int sms, cudaStream_t stream) {
  if (!ok(in) || out.top_k < 0 || out.top_k > kLogprobMaxTop || (uint32_t)out.top_k > in.vocab) return cudaErrorInvalidValue;
  if (out.top_k && in.vocab > kLogprobMaxTopVocab) return cudaErrorInvalidValue;
  if (in.rows == 0) return cudaSuccess;
  return by_type(in.dtype, [&](auto t) { return launch_rows<decltype(t)>(in, out, sms, stream); });
}

cudaError_t launch_token_logprobs_grad(const LogprobRows& in, const LogprobGrad& g, cudaStream_t stream) {
  if (!ok(in) || g.cols < in.vocab || g.cols > kLogprobMaxColumns) return cudaErrorInvalidValue;
  if (in.rows == 0) return cudaSuccess;
  return by_type(in.dtype, [&](auto t) {
    using T = decltype(t);
    const uint32_t tiles = (g.cols + kTile<T> - 1) / kTile<T> + 1, segs = (tiles + kGradTiles - 1) / kGradTiles;
    const uint64_t units = (uint64_t)in.rows * segs, grid = (units + kWarps - 1) / kWarps;
    if (grid > 0x7fffffffull) return cudaErrorInvalidValue;
    logprobs_grad_kernel<T><<<(uint32_t)grid, kThreads, 0, stream>>>(in, g, segs, units);
    return cudaGetLastError();
  });
}

}  // namespace wb
