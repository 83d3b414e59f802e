// Log probability of one given token per row of logits, the entropy of the row and its most
// probable alternatives, and the gradient of the first two (sm_100a).
//
// Row x with V valid columns, temperature T:  m = max x,  z_j = (x_j - m) / T <= 0,
//   S = sum e^z_j,  A = sum e^z_j z_j,  logp_j = z_j - ln S,  H = ln S - A / S,
// and with incoming gradients g (log probability) and h (entropy)
//   dx_j = ((j == token) g - p_j (g + h (logp_j + H))) / T.
// A column of -inf has probability 0 and adds nothing to H.  A row without any finite column is
// empty: log probability -inf, entropy 0, no gradient.  NaN and +inf make the row's results NaN.
// Rows of the type's lowest value neither overflow nor become empty.  Every sum is held in 32 bits.
// Counted from the maximum both sums have one sign and nothing cancels.  The common path counts from
// the first tile's: where one column far above that holds nearly all of the probability, ln S and A / S
// are alike and large, and their difference is off by up to 35 ln 2 half steps a term (some 1e-6).  The
// signs are known, so no log probability comes out above 0 and no entropy below.
//
// Forward: one pass.  A warp takes tiles of 1 KiB (32 bytes a lane), two loads under way; every lane
// keeps its own sums.  What bounds it is HBM, with the exponentials (16 a clock and SM: 16-bit
// logits arrive at 0.7 of their rate) and the instructions around them close behind, so the common
// path takes no running maximum and no clamp (194 -> 186 us for 4096 x 128256 bf16).  A row that needs
// them is read again.
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
constexpr float kModerate = 1048576.f;     // 2^20
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

// What z is counted from, in units of ln 2: z = (x - a) c2 - b with c2 = log2(e) / T.  Of an ordinary
// maximum a = 0 and b is max * c2 rounded to a whole number: z takes one fused operation with one
// rounding, and shifts between references are exact.  Where max * c2 is too large to be rounded so,
// a is the maximum itself and b = 0.
struct Reference {
  float a, b;
  __device__ __forceinline__ bool ordinary() const { return a == 0.f; }
  __device__ __forceinline__ float z(float x, float c2) const { return fmaf(x - a, c2, -b); }
};

__device__ __forceinline__ Reference reference(float m, float c2) {
  const float mc = m * c2;
  const bool ordinary = fabsf(mc) < kModerate;
  return {ordinary ? 0.f : m, ordinary ? rintf(mc) : 0.f};
}

// Running maximum and sums.
struct Stats {
  float m = kLowest;
  Reference ref{kLowest, 0.f};
  F2 s{0.f, 0.f}, a{0.f, 0.f};
};

// exp2 of the shift from one reference to another, of a maximum not below its own; the shift, finite, in `shift`
__device__ __forceinline__ float rescale(Reference from, Reference to, float c2, float& shift) {
  shift = fmaxf(fmaf(from.a - to.a, c2, from.b - to.b), -1e30f);
  return ex2(shift);
}

// The largest element of a vector, NaN left out; -inf where there is nothing else.
template <int N2>
__device__ __forceinline__ float largest(const F2 (&x)[N2]) {
  float m = -kInf;
  #pragma unroll
  for (int i = 0; i < N2; ++i) m = fmaxf(m, fmaxf(x[i].x, x[i].y));
  return m;
}
template <int N2>
__device__ __forceinline__ float least(const F2 (&x)[N2]) {
  float m = kInf;
  #pragma unroll
  for (int i = 0; i < N2; ++i) m = fminf(m, fminf(x[i].x, x[i].y));
  return m;
}

__device__ __forceinline__ void raise(Stats& t, float top, float c2) {
  t.m = fmaxf(t.m, top);
  const Reference to = reference(t.m, c2);
  float shift;
  const float f = rescale(t.ref, to, c2, shift);
  t.a = mul2(fma2(t.s, F2{shift, shift}, t.a), F2{f, f});
  t.s = mul2(t.s, F2{f, f});
  t.ref = to;
}

// PLAIN: an ordinary reference, and nothing so low that z would not be finite (0 * -inf would be NaN).
template <bool PLAIN, int N2>
__device__ __forceinline__ void accumulate(Stats& t, const F2 (&x)[N2], float c2) {
  const float a = t.ref.a, b = t.ref.b;
  #pragma unroll
  for (int i = 0; i < N2; ++i) {
    const F2 z = fma2(PLAIN ? x[i] : add2(x[i], F2{-a, -a}), F2{c2, c2}, F2{-b, -b});
    const F2 e{ex2(z.x), ex2(z.y)};
    t.s = add2(t.s, e);
    t.a = fma2(e, PLAIN ? z : F2{fmaxf(z.x, -1e30f), fmaxf(z.y, -1e30f)}, t.a);
  }
}

// Adds the exponent of S to an ordinary reference (exactly): for sums that have outgrown it.
__device__ __forceinline__ void lift(Stats& t) {
  const int e = (int)(__float_as_uint(t.s.x + t.s.y) >> 23) - 127;
  const float shift = (float)-e, f = __uint_as_float((uint32_t)(127 - e) << 23);
  t.a = mul2(fma2(t.s, F2{shift, shift}, t.a), F2{f, f});
  t.s = mul2(t.s, F2{f, f});
  t.ref.b += (float)e;
}

struct RowStats { float m, s, a; };

__device__ __forceinline__ RowStats at_max(RowStats t, float m, float c2) {
  float shift;
  const float f = rescale(reference(t.m, c2), reference(m, c2), c2, shift);
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

struct RowResult {
  float m, log2_sum, entropy;              // log2_sum: of the exponentials from the reference; +inf: an empty row
  Reference ref;
};

__device__ __forceinline__ RowResult finish(RowStats t, float c2) {
  const bool empty = t.s == 0.f;
  RowResult r;
  r.m = empty ? 0.f : t.m;
  r.ref = reference(r.m, c2);
  r.log2_sum = empty ? kInf : log2f(t.s);
  r.entropy = empty ? 0.f : kLn2 * (r.log2_sum - t.a / t.s);
  if (r.entropy < 0.f) r.entropy = 0.f;    // rounding alone; NaN stays
  return r;
}

// Near the type's lowest value z is out of range where the log probability itself may not be; the sum
// is nothing beside it.
__device__ __forceinline__ float logprob(const RowResult& t, float x, float c2) {
  const float z = t.ref.z(x, c2);
  const float lp = z == -kInf && t.log2_sum < kInf ? (x - t.m) * (c2 * kLn2) : kLn2 * (z - t.log2_sum);
  return lp > 0.f ? 0.f : lp;              // rounding alone; NaN stays
}

// The token's logit, loaded before the row: its latency passes under the row's.
template <typename T>
__device__ __forceinline__ float token_logit(const LogprobRows& in, const T* x, int64_t tok) {
  return tok >= 0 && tok < (int64_t)in.vocab ? to_f32(x[tok]) : kNaN;
}

__device__ __forceinline__ void write_row(const LogprobRows& in, const LogprobOut& out, uint32_t r, int64_t tok, float xt, const RowResult& t,
                                          float c2) {
  out.logprobs[r] = tok >= 0 && tok < (int64_t)in.vocab ? logprob(t, xt, c2) : kNaN;
  out.entropy[r] = t.entropy;
  if (out.stats) {
    out.stats[2 * (int64_t)r] = t.m;
    out.stats[2 * (int64_t)r + 1] = t.log2_sum;
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

// One warp's way through tiles first, first + step, ... below `end` of a row.  Two tiles' loads are
// always under way: one's vector is refilled as soon as it is unpacked.
template <typename T>
struct Walk {
  static constexpr int N = kVecN<T>, kDepth = 2;
  const T* x;
  uint32_t vocab, mis, first, step, end;
  Vec32 raw[kDepth];

  __device__ __forceinline__ void load(int u, uint32_t k) {
    if (k < end) raw[u] = load_vec(x, vocab, (int32_t)(k * kTile<T> + (threadIdx.x & 31) * N - mis));
  }
  // issues the first loads
  __device__ __forceinline__ void start() {
    #pragma unroll
    for (int u = 0; u < kDepth; ++u) load(u, first + u * step);
  }
  // This lane's statistics; tops: each tile's largest as a key, counted from tile `base`.
  template <bool TOP>
  __device__ __forceinline__ Stats run(float c2, uint32_t base, uint32_t* tops) {
    Stats st;
    if (!common<TOP>(st, c2, base, tops)) {
      start();
      careful<TOP>(st, c2, base, tops);
    }
    return st;
  }

 private:
  template <bool TOP>
  __device__ __forceinline__ static void keep_top(const F2 (&v)[N / 2], uint32_t tile, uint32_t* tops) {
    if constexpr (TOP) {
      const uint32_t key = __reduce_max_sync(kFullWarp, order_key(largest(v)));
      if ((threadIdx.x & 31) == 0) tops[tile] = tile_key<T>(key, tile);
    }
  }

  // Ordinary rows: the first tile's largest gives the reference of the whole walk, which is lifted
  // where a sum outgrows it, so no maximum is taken of the other tiles.  False (for the whole warp) at
  // the first sum that is not finite (a masked column: 0 * -inf; NaN), where a logit is some 2^35
  // times as probable as the reference (A, of terms e^z z, would lose the bits of z to it), or where the
  // reference was lifted out of its range.
  template <bool TOP>
  __device__ __forceinline__ bool common(Stats& st, float c2, uint32_t base, uint32_t* tops) {
    if (first >= end) return true;
    {
      F2 v[N / 2];
      unpack<T>(raw[0], v);
      st.ref = reference(warp_max(largest(v)), c2);
    }
    if (!st.ref.ordinary()) return false;
    const uint32_t full_from = mis ? 1 : 0, full_to = (mis + vocab) / kTile<T>;
    #pragma unroll 1
    for (uint32_t t = first; t < end; t += kDepth * step) {
      #pragma unroll
      for (int u = 0; u < kDepth; ++u) {
        const uint32_t k = t + u * step;
        if (k >= end) break;
        F2 v[N / 2];
        unpack<T>(raw[u], v);
        load(u, k + kDepth * step);
        keep_top<TOP>(v, k - base, tops);
        if (k >= full_from && k < full_to) accumulate<true>(st, v, c2);
        else accumulate<false>(st, v, c2);
      }
      const float size = st.a.x + st.a.y;
      if (__any_sync(kFullWarp, !(fabsf(size) < 1.0995116e12f))) return false;       // 2^40
      if (size > 65536.f) lift(st);
    }
    // reference(b / c2) gives b again: within 2^20 the quotient and its product are off by less than 1/8
    if (__any_sync(kFullWarp, !(fabsf(st.ref.b) < kModerate))) return false;
    st.m = st.ref.b / c2;
    return true;
  }

  // Any row: the maximum is kept, the sums rescaled to it, and what is too low to count is clamped.
  template <bool TOP>
  __device__ __forceinline__ void careful(Stats& st, float c2, uint32_t base, uint32_t* tops) {
    st = Stats{};
    #pragma unroll 1
    for (uint32_t t = first; t < end; t += kDepth * step) {
      #pragma unroll
      for (int u = 0; u < kDepth; ++u) {
        const uint32_t k = t + u * step;
        if (k >= end) break;
        F2 v[N / 2];
        unpack<T>(raw[u], v);
        load(u, k + kDepth * step);
        keep_top<TOP>(v, k - base, tops);
        raise(st, largest(v), c2);
        accumulate<false>(st, v, c2);
      }
    }
  }
};

// Many short rows: a warp takes one after another.  The next row's token is under way during a row,
// and its first tiles while this one's lanes are joined.
template <typename T>
__global__ void __launch_bounds__(kThreads) logprobs_warp_kernel(const LogprobRows in, const LogprobOut out) {
  const uint32_t warps = gridDim.x * kWarps, lane = threadIdx.x & 31;
  const float c2 = in.inv_temp * kLog2e;
  uint32_t next = blockIdx.x * kWarps + threadIdx.x / 32;          // the row that `ahead` is the token of
  int64_t ahead = next < in.rows ? token_of(in, next) : 0;
  uint32_t r = 0;
  int64_t tok = 0;
  float xt = 0.f;
  Walk<T> w;
  auto open = [&] {                                                // the next row that is not ignored
    for (; next < in.rows; next += warps) {
      r = next;
      tok = ahead;
      if (in.rows - next > warps) ahead = token_of(in, next + warps);
      if (tok != in.ignore_index) {
        w.x = row_ptr<T>(in, r);
        w.mis = misaligned(w.x);
        w.vocab = in.vocab;
        w.first = 0, w.step = 1, w.end = (w.mis + in.vocab + kTile<T> - 1) / kTile<T>;
        w.start();
        xt = token_logit(in, w.x, tok);
        next += warps;
        return true;
      }
      if (lane == 0) write_ignored(out, r);
    }
    return false;
  };
  bool more = open();
  while (more) {
    const Stats st = w.template run<false>(c2, 0, nullptr);
    const uint32_t row = r;
    const int64_t row_tok = tok;
    const float row_xt = xt;
    more = open();
    const RowStats t = warp_join({st.m, st.s.x + st.s.y, st.a.x + st.a.y}, c2);
    if (lane == 0) write_row(in, out, row, row_tok, row_xt, finish(t, c2), c2);
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

// Ranks n distinct candidates (and zeros, which are none) by counting; the first k go to `out` in order.
__device__ __forceinline__ void rank_candidates(const uint64_t* c, uint32_t n, uint32_t k, uint64_t* out) {
  for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
    const uint64_t mine = c[i];
    uint32_t rank = 0;
    #pragma unroll 8
    for (uint32_t j = 0; j < n; ++j) rank += c[j] > mine;
    if (mine && rank < k) out[rank] = mine;
  }
}

// The k first columns of tiles [base, base + n), in order, into sh.out.  tops: each tile's largest.
template <typename T>
__device__ void find_top(const T* x, uint32_t vocab, uint32_t mis, uint32_t base, uint32_t n, uint32_t k, const uint32_t* tops,
                         TopShared& sh) {
  constexpr int N = kVecN<T>, kShift = kKeyShift<T>;
  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  constexpr uint32_t high = 0xffffffffu >> kShift;
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
    F2 v[N / 2];
    unpack<T>(raw[s], v);
    value[s] = order_key(largest(v)) >> kShift;
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

// A CTA per row, or a cluster of `splits` CTAs.  4096 x 128256 bf16: 177 to 187 us, 0.92 to 0.87 of the
// measured copy rate (one of two GPUs, the other); 64 x 151936 with 20 alternatives: 14.5 us; one row of
// 128256: 4.7 us, with 5 alternatives 7.6.
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
  const float c2 = in.inv_temp * kLog2e;
  const uint32_t mis = misaligned(x), tiles = (mis + in.vocab + kTile<T> - 1) / kTile<T>;
  const uint32_t per = (tiles + splits - 1) / splits;
  const uint32_t begin = min(split * per, tiles), end = min(begin + per, tiles);
  if (TOP && threadIdx.x < 4) tops[(end - begin) + threadIdx.x] = 0;
  Walk<T> walk{x, in.vocab, mis, begin + warp, kWarps, end, {}};
  walk.start();
  const float xt = token_logit(in, x, tok);
  const Stats st = walk.template run<TOP>(c2, begin, tops);
  const RowStats w = warp_join({st.m, st.s.x + st.s.y, st.a.x + st.a.y}, c2);
  if (lane == 0) warps[warp] = w;
  __syncthreads();
  // every warp joins the eight: the same operations, the same bits
  RowStats all = warp_join(lane < kWarps ? warps[lane] : RowStats{kLowest, 0.f, 0.f}, c2);
  if constexpr (TOP) find_top(x, in.vocab, mis, begin, end - begin, (uint32_t)out.top_k, tops, shared);
  if (splits > 1) {
    cg::cluster_group cl = cg::this_cluster();
    if (threadIdx.x == 0) mine = all;
    cl.sync();
    if (split == 0) {
      all = warp_join(lane < splits ? *cl.map_shared_rank(&mine, lane) : RowStats{kLowest, 0.f, 0.f}, c2);
      if constexpr (TOP) {               // at most 8 * 32 candidates, a thread each; 0: none
        const uint32_t k = (uint32_t)out.top_k, s = threadIdx.x / k, i = threadIdx.x % k;
        uint64_t c = 0;
        if (s < splits) {
          const TopShared* theirs = cl.map_shared_rank(&shared, s);
          const uint32_t n = theirs->n_out;
          c = theirs->out[i];
          if (i >= n) c = 0;
          shared.candidates[threadIdx.x] = c;
        }
        __syncthreads();                 // this CTA's own list has been read, too
        rank_candidates(shared.candidates, splits * k, k, shared.out);
        __syncthreads();
      }
    }
    cl.sync();                             // the others' shared memory stays until it has been read
  }
  if (split == 0 && warp == 0) {
    const RowResult t = finish(all, c2);
    if (lane == 0) write_row(in, out, r, tok, xt, t, c2);
    if constexpr (TOP) {
      if (lane < (uint32_t)out.top_k) {
        const uint64_t c = shared.out[lane];
        out.top_logprobs[(int64_t)r * out.top_k + lane] = logprob(t, key_value((uint32_t)(c >> 32)), c2);
        out.top_ids[(int64_t)r * out.top_k + lane] = (int64_t)(uint32_t)~(uint32_t)c;
      }
    }
  }
}

// -- gradient -------------------------------------------------------------------------------------
constexpr uint32_t kGradTiles = 16;        // tiles of one warp's work: 16 KiB read, 16 KiB written

// Reads a logit and writes a gradient, once each, at HBM's rate (4096 x 152064 bf16: 400 us, 0.96 of
// the measured copy rate); a warp takes up to 16 tiles of one
// row and shares nothing.  Tiles follow the gradient's alignment.  Where the logits' rows lie
// otherwise (views whose rows are not multiples of 32 bytes), and at the ends of a row, lanes take
// single elements side by side instead of vectors.
template <typename T>
__global__ void __launch_bounds__(kThreads, 4) logprobs_grad_kernel(const LogprobRows in, const LogprobGrad g, const uint32_t segs,
                                                                 const uint64_t units) {
  constexpr int N = kVecN<T>;
  const uint64_t unit = (uint64_t)blockIdx.x * kWarps + threadIdx.x / 32;
  if (unit >= units) return;
  const uint32_t r = (uint32_t)(unit / segs), seg = (uint32_t)(unit % segs), lane = threadIdx.x & 31;
  const int64_t tok = token_of(in, r);
  const T* x = row_ptr<T>(in, r);
  T* d = reinterpret_cast<T*>(g.grad) + (int64_t)r * g.cols;
  const uint32_t mis = misaligned(d);
  const float c2 = in.inv_temp * kLog2e, m = g.stats[2 * (int64_t)r], log2_sum = g.stats[2 * (int64_t)r + 1], h = g.entropy[r];
  float glp = g.g_logprobs ? g.g_logprobs[r * g.g_logprobs_stride] : 0.f;
  float gh = g.g_entropy ? g.g_entropy[r * g.g_entropy_stride] : 0.f;
  const bool dead = tok == in.ignore_index || log2_sum == kInf;
  if (dead) glp = gh = 0.f;
  else if (tok < 0 || tok >= (int64_t)in.vocab) glp = kNaN;
  // log2 p = z - f, z counted from a whole number more and f the rest of log2_sum: with
  // dx = p (c + d log2 p) = 2^z 2^-f (c - d f + d z) the constants take the rest in
  const Reference ref = reference(m, c2);
  const float whole = dead ? 0.f : rintf(log2_sum), f = dead ? 0.f : log2_sum - whole, k = ex2(-f);
  const float d1 = -k * in.inv_temp * gh * kLn2, c1 = -k * in.inv_temp * (glp + gh * h) - d1 * f, onehot = glp * in.inv_temp;
  const float a = ref.a, b = ref.b + whole, lowest = -kModerate / c2;
  auto plain2 = [&](F2 v) {
    const F2 z = fma2(v, F2{c2, c2}, F2{-b, -b});
    return mul2(F2{ex2(z.x), ex2(z.y)}, fma2(F2{d1, d1}, z, F2{c1, c1}));
  };
  // Any column: one without probability gets 0, whatever c and d z are (1 / T and the incoming gradients may
  // be so large that these pass the range).  NaN stays.
  auto safe2 = [&](F2 v) {
    const F2 z = fma2(add2(v, F2{-a, -a}), F2{c2, c2}, F2{-b, -b});
    const F2 p{ex2(z.x), ex2(z.y)}, d = mul2(p, fma2(F2{d1, d1}, z, F2{c1, c1}));
    return F2{p.x == 0.f ? 0.f : d.x, p.y == 0.f ? 0.f : d.y};
  };
  // of an ordinary reference and logits above `lowest` |z| is below 2^22
  const bool plain = ref.ordinary() && fabsf(d1) < 1.2676506e30f && fabsf(c1) < 1.7014118e38f;   // 2^100, 2^127
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
        if (plain && least(v) > lowest) {
          #pragma unroll
          for (int i = 0; i < N / 2; ++i) v[i] = plain2(v[i]);
        } else {
          #pragma unroll
          for (int i = 0; i < N / 2; ++i) v[i] = safe2(v[i]);
        }
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
      #pragma unroll 1
      for (int e = 0; e < N; e += 8) {
        float v[8];
        #pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int32_t j = first + (e + i) * step;
          v[i] = !dead && j >= 0 && j < (int32_t)in.vocab ? to_f32(x[j]) : -kInf;
        }
        #pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int32_t j = first + (e + i) * step;
          const float y = j < (int32_t)in.vocab && !dead ? safe2({v[i], v[i]}).x + (j == tok ? onehot : 0.f) : 0.f;
          if (j >= 0 && j < (int32_t)g.cols) d[j] = from_f32<T>(y);
        }
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
  // A warp a row where the rows alone fill the GPU: no barrier, no second join.  The more tiles a row
  // has, the more rows it takes until a CTA's eight warps a row lose (bf16, warp against CTA: 1000 x
  // 4000 6.5 and 6.7 us, 2000 x 8000 12.0 and 13.7, 4096 x 16000 31.9 and 36.3, 20000 x 32000 231
  // and 249; the other way 500 x 4000 4.9 and 3.9, 2000 x 32000 36.3 and 30.1, 4096 x 128256 209 and 175).
  if (!out.top_k && tiles <= 65 && (uint64_t)tiles * sms * 2 <= (uint64_t)in.rows * 3) {
    const uint32_t cap = (uint32_t)sms * 4, grid = (in.rows + kWarps - 1) / kWarps;
    logprobs_warp_kernel<T><<<grid < cap ? grid : cap, kThreads, 0, stream>>>(in, out);
    return cudaGetLastError();
  }
  // CTAs of a row: until two (with alternatives, whose search every CTA repeats) or four of the four
  // that an SM holds are taken, and every warp keeps two tiles (bf16, 64 x 151936: 1 CTA 23 us, 2: 15,
  // 4: 11.1, 8: 10.4; 512 rows: 1 CTA 41, 2: 45).
  uint32_t splits = 1;
  const uint64_t most = (uint64_t)sms * (out.top_k ? 2 : 4);
  while (splits < kMaxSplits && (uint64_t)in.rows * splits * 2 <= most && tiles >= splits * 2 * kWarps) splits *= 2;
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
