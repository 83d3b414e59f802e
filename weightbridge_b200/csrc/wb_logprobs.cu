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
// Alternatives: a tile's columns are consecutive, so by (logit descending, column ascending) the
// k first columns lie in the k first tiles ranked by (their largest logit, tile).  The pass leaves
// each tile's maximum in shared memory; k tiles are picked, read once more and searched.
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

template <int N2>
__device__ __forceinline__ float tile_max(const F2 (&x)[N2]) {
  float m = fmaxf(x[0].x, x[0].y);
  #pragma unroll
  for (int i = 1; i < N2; ++i) m = fmaxf(m, fmaxf(x[i].x, x[i].y));
  return m;
}

template <int N2>
__device__ __forceinline__ void accumulate(Stats& t, const F2 (&x)[N2], float top, float c2) {
  const float m = fmaxf(t.m, top);
  float shift;
  const float f = rescale(t.m, m, c2, shift);
  t.a = mul2(fma2(t.s, F2{shift, shift}, t.a), F2{f, f});
  t.s = mul2(t.s, F2{f, f});
  t.m = m;
  #pragma unroll
  for (int i = 0; i < N2; ++i) {
    const F2 z = mul2(add2(x[i], F2{-m, -m}), F2{c2, c2});
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

// A tile that the row does not fill, element by element; what lies outside the row reads as -inf.
template <typename T>
__device__ __forceinline__ void load_edge(const T* x, uint32_t vocab, int64_t j0, F2 (&v)[kVecN<T> / 2]) {
  #pragma unroll
  for (int i = 0; i < kVecN<T>; ++i) {
    const int64_t j = j0 + i;
    const float f = j >= 0 && j < (int64_t)vocab ? to_f32(x[j]) : -kInf;
    if (i & 1) v[i / 2].y = f; else v[i / 2].x = f;
  }
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

template <typename T>
__device__ __forceinline__ void write_row(const LogprobRows& in, const LogprobOut& out, uint32_t r, const T* x, int64_t tok,
                                          const RowResult& t) {
  out.logprobs[r] = tok >= 0 && tok < (int64_t)in.vocab ? logprob(t, to_f32(x[tok]), in.inv_temp) : kNaN;
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

// Tiles [first, first + step, ...) below `end` of a row into this lane's statistics; two at a time,
// so that the second's load runs under the first's arithmetic.  tops: each tile's largest, as a key.
template <typename T, bool TOP>
__device__ __forceinline__ Stats walk(const T* x, uint32_t vocab, uint32_t mis, uint32_t first, uint32_t step, uint32_t end,
                                      uint32_t base, float c2, uint32_t* tops) {
  constexpr int N = kVecN<T>, kDepth = 2;
  const uint32_t lane = threadIdx.x & 31;
  Stats st;
  const T* aligned = x - mis;
  // full tiles: those that begin at or behind the row's start and end at or before its end
  const uint32_t full_from = mis ? 1 : 0, full_to = (mis + vocab) / kTile<T>;
  for (uint32_t t = first; t < end; t += kDepth * step) {
    Vec32 raw[kDepth];
    bool full[kDepth];
    #pragma unroll
    for (int u = 0; u < kDepth; ++u) {
      const uint32_t k = t + u * step;
      full[u] = k >= full_from && k < full_to && k < end;
      if (full[u]) raw[u] = load32(aligned + (int64_t)k * kTile<T> + lane * N);
    }
    #pragma unroll
    for (int u = 0; u < kDepth; ++u) {
      const uint32_t k = t + u * step;
      if (k >= end) break;
      F2 v[N / 2];
      if (full[u]) unpack<T>(raw[u], v);
      else load_edge(x, vocab, (int64_t)k * kTile<T> + lane * N - mis, v);
      const float top = tile_max(v);
      accumulate(st, v, top, c2);
      if constexpr (TOP) {
        const uint32_t key = __reduce_max_sync(kFullWarp, order_key(top));
        if (lane == 0) tops[k - base] = key;
      }
    }
  }
  return st;
}

// Many short rows: a warp each.
template <typename T>
__global__ void __launch_bounds__(kThreads) logprobs_warp_kernel(const LogprobRows in, const LogprobOut out) {
  const uint32_t r = blockIdx.x * kWarps + threadIdx.x / 32;
  if (r >= in.rows) return;
  const int64_t tok = token_of(in, r);
  if (tok == in.ignore_index) {
    if (threadIdx.x % 32 == 0) write_ignored(out, r);
    return;
  }
  const T* x = row_ptr<T>(in, r);
  const float c2 = in.inv_temp * kLog2e;
  const uint32_t mis = misaligned(x), tiles = (mis + in.vocab + kTile<T> - 1) / kTile<T>;
  const Stats st = walk<T, false>(x, in.vocab, mis, 0, 1, tiles, 0, c2, nullptr);
  const RowStats t = warp_join({st.m, st.s.x + st.s.y, st.a.x + st.a.y}, c2);
  if (threadIdx.x % 32 == 0) write_row(in, out, r, x, tok, finish(t));
}

// -- alternatives ---------------------------------------------------------------------------------
// The largest (key, lowest index) over the warp; key 0: none.
__device__ __forceinline__ bool warp_best(uint32_t key, uint32_t idx, uint32_t& best_key, uint32_t& best_idx) {
  best_key = __reduce_max_sync(kFullWarp, key);
  best_idx = __reduce_min_sync(kFullWarp, key == best_key ? idx : 0xffffffffu);
  return best_key != 0;
}

// Shared memory of the search, in words: the tiles' maxima, then the keys of the picked tiles.
template <typename T>
struct TopShared {
  uint32_t picked[kLogprobMaxTop], key[kLogprobMaxTop], col[kLogprobMaxTop];   // per picked tile: its best column left
  uint32_t out_key[kLogprobMaxTop], out_col[kLogprobMaxTop];                   // the result, in order
  uint32_t n_picked, n_out;
};

// The k first columns of tiles [base, base + n): whole CTA; the result in sh.out_*.
template <typename T>
__device__ void find_top(const T* x, uint32_t vocab, uint32_t mis, uint32_t base, uint32_t n, uint32_t k, uint32_t* tops, uint32_t* keys,
                         TopShared<T>& sh) {
  constexpr int N = kVecN<T>;
  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  if (warp == 0) {                         // pick k tiles by (maximum, lowest tile)
    uint32_t key = 0, idx = 0xffffffffu, picked = 0;
    auto scan = [&] {
      key = 0, idx = 0xffffffffu;
      for (uint32_t i = lane; i < n; i += 32)
        if (tops[i] > key) key = tops[i], idx = i;
    };
    scan();
    for (; picked < k; ++picked) {
      uint32_t bk, bi;
      if (!warp_best(key, idx, bk, bi)) break;
      if (lane == 0) sh.picked[picked] = bi;
      if (idx == bi) {
        tops[bi] = 0;
        scan();
      }
    }
    if (lane == 0) sh.n_picked = picked;
  }
  __syncthreads();
  const uint32_t picked = sh.n_picked;
  for (uint32_t s = warp; s < picked; s += kWarps) {         // their columns' keys, element-major
    const int64_t j0 = (int64_t)(base + sh.picked[s]) * kTile<T> + lane * N - mis;
    uint32_t key = 0, col = 0xffffffffu;
    #pragma unroll
    for (int e = 0; e < N; ++e) {
      const int64_t j = j0 + e;
      const uint32_t v = j >= 0 && j < (int64_t)vocab ? order_key(to_f32(x[j])) : 0;
      keys[s * kTile<T> + e * 32 + lane] = v;
      if (v > key) key = v, col = (uint32_t)j;
    }
    uint32_t bk, bc;
    warp_best(key, col, bk, bc);
    if (lane == 0) sh.key[s] = bk, sh.col[s] = bc;
  }
  __syncthreads();
  if (warp == 0) {                         // k times the best of the picked tiles' bests
    uint32_t key = lane < picked ? sh.key[lane] : 0, col = lane < picked ? sh.col[lane] : 0xffffffffu;
    uint32_t found = 0;
    for (; found < k; ++found) {
      uint32_t bk, bc;
      if (!warp_best(key, col, bk, bc)) break;
      if (lane == 0) sh.out_key[found] = bk, sh.out_col[found] = bc;
      const uint32_t s = __ffs(__ballot_sync(kFullWarp, key == bk && col == bc)) - 1;
      const uint32_t tile = sh.picked[s] + base, at = bc + mis - tile * kTile<T>;
      uint32_t nk = 0, nc = 0xffffffffu;
      #pragma unroll
      for (int e = 0; e < N; ++e) {        // columns behind the one taken: a lower key, or the same and a higher column
        const uint32_t v = keys[s * kTile<T> + e * 32 + lane], p = lane * N + e;
        if ((v < bk || (v == bk && p > at)) && v > nk) nk = v, nc = tile * kTile<T> + p - mis;
      }
      uint32_t gk, gc;
      warp_best(nk, nc, gk, gc);
      if (lane == s) key = gk, col = gc;
    }
    if (lane == 0) sh.n_out = found;
  }
  __syncthreads();
}

// A CTA per row, or a cluster of `splits` CTAs.
template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads) logprobs_row_kernel(const LogprobRows in, const LogprobOut out, const uint32_t splits) {
  extern __shared__ uint32_t dyn[];                      // TOP: tile maxima, then keys
  __shared__ RowStats warps[kWarps], mine;
  __shared__ TopShared<T> sh;
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
  const Stats st = walk<T, TOP>(x, in.vocab, mis, begin + warp, kWarps, end, begin, c2, dyn);
  const RowStats w = warp_join({st.m, st.s.x + st.s.y, st.a.x + st.a.y}, c2);
  if (lane == 0) warps[warp] = w;
  __syncthreads();
  if (warp == 0) {
    const RowStats t = warp_join(lane < kWarps ? warps[lane] : RowStats{kLowest, 0.f, 0.f}, c2);
    if (lane == 0) mine = t;
  }
  if constexpr (TOP) find_top(x, in.vocab, mis, begin, end - begin, (uint32_t)out.top_k, dyn, dyn + per, sh);
  else __syncthreads();
  RowStats all = mine;
  if (splits > 1) {
    cg::cluster_group cl = cg::this_cluster();
    cl.sync();
    if (split == 0 && warp == 0) {
      all = warp_join(lane < splits ? *cl.map_shared_rank(&mine, lane) : RowStats{kLowest, 0.f, 0.f}, c2);
      if constexpr (TOP) {
        // every CTA's list is in order: lane s stands at the head of CTA s's list
        TopShared<T>* theirs = lane < splits ? cl.map_shared_rank(&sh, lane) : &sh;
        const uint32_t n = lane < splits ? theirs->n_out : 0;
        uint32_t at = 0, key = n ? theirs->out_key[0] : 0, col = n ? theirs->out_col[0] : 0xffffffffu;
        for (uint32_t i = 0; i < (uint32_t)out.top_k; ++i) {
          uint32_t bk, bc;
          warp_best(key, col, bk, bc);
          if (lane == 0) dyn[2 * i] = bk, dyn[2 * i + 1] = bc;     // the maxima are no longer needed
          if (key == bk && col == bc) {
            ++at;
            key = at < n ? theirs->out_key[at] : 0;
            col = at < n ? theirs->out_col[at] : 0xffffffffu;
          }
        }
        __syncwarp();
        if (lane < (uint32_t)out.top_k) sh.out_key[lane] = dyn[2 * lane], sh.out_col[lane] = dyn[2 * lane + 1];
        __syncwarp();
      }
    }
    cl.sync();                             // the others' shared memory stays until it has been read
  }
  if (split == 0 && warp == 0) {
    const RowResult t = finish(all);
    if (lane == 0) write_row(in, out, r, x, tok, t);
    if (TOP && lane < (uint32_t)out.top_k) {
      out.top_logprobs[(int64_t)r * out.top_k + lane] = logprob(t, key_value(sh.out_key[lane]), in.inv_temp);
      out.top_ids[(int64_t)r * out.top_k + lane] = sh.out_col[lane];
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
  const uint32_t full_from = mis ? 1 : 0, full_to = vectors ? (mis + in.vocab) / kTile<T> : 0;
  #pragma unroll 2
  for (uint32_t t = begin; t < end; ++t) {
    if (t >= full_from && t < full_to) {
      const int64_t j0 = (int64_t)t * kTile<T> + lane * N - mis;
      F2 v[N / 2];
      if (dead) {
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
      for (int e = 0; e < N; ++e) {
        const int64_t j = (int64_t)t * kTile<T> + e * 32 + lane - mis;
        if (j < 0 || j >= (int64_t)g.cols) continue;
        float v = 0.f;
        if (!dead && j < (int64_t)in.vocab) v = grad2({to_f32(x[j]), 0.f}).x + (j == tok ? onehot : 0.f);
        d[j] = from_f32<T>(v);
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

bool ok(const LogprobRows& in) { return in.rows < 0x7fffffffu && in.vocab >= 1 && in.vocab < 0x7fffffffu && in.inner >= 1; }

// Rows of up to this many columns are read by one warp where nothing else asks for a CTA.
constexpr uint32_t kWarpRow = 2048;

template <typename T>
cudaError_t launch_rows(const LogprobRows& in, const LogprobOut& out, int sms, cudaStream_t stream) {
  const uint32_t tiles = (in.vocab + kTile<T> - 1) / kTile<T> + 1;
  if (!out.top_k && in.vocab <= kWarpRow) {
    logprobs_warp_kernel<T><<<(in.rows + kWarps - 1) / kWarps, kThreads, 0, stream>>>(in, out);
    return cudaGetLastError();
  }
  uint32_t splits = 1;
  while (splits < kMaxSplits && (uint64_t)in.rows * splits * 2 <= (uint64_t)sms * 2 && tiles >= splits * 2 * kWarps) splits *= 2;
  const uint32_t per = (tiles + splits - 1) / splits;
  const size_t shared = out.top_k ? 4 * (per + (size_t)out.top_k * kTile<T>) : 0;
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
  if (shared > 40 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)shared);
    if (e != cudaSuccess) return e;
  }
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
  if (!ok(in) || g.cols < in.vocab || g.cols >= 0x7fffffffu) return cudaErrorInvalidValue;
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
