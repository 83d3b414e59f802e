// The AdamW step over many tensors in one launch, and the global gradient norm (sm_100a).
//
// With c = min(1, max_norm / (norm + 1e-6)), g' = c g, t the number of the step:
//   m = b1 m + (1 - b1) g',  v = b2 v + (1 - b2) g'^2,
//   p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps),
// all in 32 bits; p is rounded to nearest once, to the parameter's type (with fp32 master weights p
// is the master weight and the parameter its rounded copy, so small steps are not lost).
//
// 8-bit states: 128 consecutive elements of a tensor share an fp32 scale = amax / 448; m and the
// root r of v are held as e4m3 codes q = RN(x / scale).  The root halves the exponents that a
// block has to span (e4m3 holds 2^-9 .. 448, so v spans 2^35 within a block).  A positive r never
// takes the code 0 but at least the smallest, 2^-9: a zero denominator would let the step grow
// without bound, a denominator rounded up only shortens it.
// What bounds it: HBM.  Of the measured copy rate, over 200M elements: fp32 states 0.94 to 0.98 (0.85 to
// 0.95 at odd addresses), 8-bit states 0.83 to 0.89 (0.46 to 0.76): their arithmetic, 29 instructions
// an element, runs close behind.  The norm: 604M bf16 gradients in 174 us, as fast as they are read.
#include "wb_optim.h"

#include <cuda_fp8.h>

#include "wb_vec.cuh"

namespace wb {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr double kMaxDouble = 1.7976931348623157e308;

// A sum over the CTA in a fixed order; all threads get it.
__device__ __forceinline__ double cta_sum(double v, double* red) {
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0;
  for (int i = 0; i < kWarps; ++i) v += red[i];
  return v;
}

// -- the step -------------------------------------------------------------------------------------
struct StepScalars { float b1, om_b1, b2, om_b2, step_size, root_c2, eps, coef, lr; };

template <bool FP8> constexpr int kAdamCtas = FP8 ? 2 : 4;       // CTAs an SM holds

template <int N>
struct Grads {
  uint64_t p[N];
  uint32_t first_tensor, first_chunk, n_chunks, last;
};

// Hardware approximations with relative errors of 2^-23; numbers below 2^-126 count as 0.
__device__ __forceinline__ float root(float x) {
  float r;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float reciprocal(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ F2 both(float x) { return {x, x}; }

// Two elements: the new moments, the new values and r = sqrt(v).
__device__ __forceinline__ void update2(const StepScalars& s, float keep, F2 grad, F2& m, F2& v, F2& p, F2& r) {
  const F2 g = mul2(grad, both(s.coef));
  m = fma2(both(s.b1), m, mul2(both(s.om_b1), g));
  v = fma2(both(s.b2), v, mul2(mul2(both(s.om_b2), g), g));
  r = {root(v.x), root(v.y)};
  const F2 d = fma2(r, both(s.root_c2), both(s.eps));
  const F2 u = mul2(m, F2{reciprocal(d.x), reciprocal(d.y)});
  p = fma2(both(-s.step_size), u, mul2(p, both(keep)));
}

__device__ __forceinline__ F2 decode2(uint32_t q) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(q & 0xffffu), __NV_E4M3);
  const float2 f = __half22float2(__half2(h));
  return {f.x, f.y};
}

__device__ __forceinline__ uint32_t encode2(F2 x) { return __nv_cvt_float2_to_fp8x2(make_float2(x.x, x.y), __NV_SATFINITE, __NV_E4M3); }

// Scale of a block, amax / 448, and 448 / amax, each a product with an approximate reciprocal and one
// Newton step of the quotient: q + (a - b q) / b, whose residual a fused multiply-add leaves exact but for one
// rounding (the reciprocal of the rounded scale would round once more).  A block of tiny values keeps a
// normal scale, whose reciprocal is finite; a block of zeros has scale 1.
__device__ __forceinline__ float block_scale(float amax) {
  constexpr float kInv = 1.f / kE4M3Max;
  float q = amax * kInv;
  q = fmaf(fmaf(-kE4M3Max, q, amax), kInv, q);
  if (!(amax <= 3.402823466e38f)) q = amax;              // an infinite moment stays one
  return amax > 0.f ? fmaxf(q, 1.17549435e-38f) : 1.f;
}
__device__ __forceinline__ float block_inverse(float amax) {
  const float r = reciprocal(0.25f * amax);  // 4 / amax: a normal number up to the largest amax
  float q = 0.25f * kE4M3Max * r;
  q = fmaf(fmaf(-amax, q, kE4M3Max), 0.25f * r, q);
  return fminf(q, 8.507059173e37f);         // 2^126, also where the above is not a number (zero and tiny blocks)
}

// r in units of the scale; a positive r keeps at least the smallest code, NaN stays
__device__ __forceinline__ F2 root_codes(F2 r, float inv) {
  const F2 q = mul2(r, both(inv));
  return {r.x > 0.f ? fmaxf(q.x, 0.001953125f) : q.x, r.y > 0.f ? fmaxf(q.y, 0.001953125f) : q.y};
}

// The states of E consecutive elements of one lane as they come from memory.
template <bool FP8, int E> struct RawStates;

template <int E>
struct RawStates<true, E> {
  uint32_t m[E / 4], v[E / 4];              // codes
  float ms, vs;
  __device__ __forceinline__ void load(const AdamArgs& a, uint64_t si) {
    static_assert(E == 4);                  // longer ones come through shared memory
    m[0] = *reinterpret_cast<const uint32_t*>(reinterpret_cast<const uint8_t*>(a.m) + si);
    v[0] = *reinterpret_cast<const uint32_t*>(reinterpret_cast<const uint8_t*>(a.v) + si);
    ms = a.m_scale[si / kStateBlock];
    vs = a.v_scale[si / kStateBlock];
  }
};

template <int E>
struct RawStates<false, E> {
  F2 m[E / 2], v[E / 2];
  __device__ __forceinline__ void load(const AdamArgs& a, uint64_t si) {
    load_pairs<E>(reinterpret_cast<const float*>(a.m) + si, m);
    load_pairs<E>(reinterpret_cast<const float*>(a.v) + si, v);
  }
};

// The states of E consecutive elements of one lane, as pairs.  Slices of the flat buffers are
// padded to whole blocks, so a lane may pass the tensor's end: there the states are and stay 0.
template <bool FP8, int E>
struct States {
  F2 m[E / 2], v[E / 2];

  __device__ __forceinline__ void decode(const RawStates<FP8, E>& raw) {
    #pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      if constexpr (FP8) {
        m[i] = mul2(decode2(i & 1 ? raw.m[i / 2] >> 16 : raw.m[i / 2]), both(raw.ms));
        const F2 r = mul2(decode2(i & 1 ? raw.v[i / 2] >> 16 : raw.v[i / 2]), both(raw.vs));
        v[i] = mul2(r, r);
      } else {
        m[i] = raw.m[i];
        v[i] = raw.v[i];
      }
    }
  }

  // r: the roots of v
  __device__ __forceinline__ void store(const AdamArgs& a, uint64_t si, const F2 (&r)[E / 2]) {
    if constexpr (FP8) {
      constexpr int kLanes = kStateBlock / E;            // lanes that share a block
      float ma = 0.f, ra = 0.f;
      #pragma unroll
      for (int i = 0; i < E / 2; ++i) {
        ma = fmaxf(ma, fmaxf(fabsf(m[i].x), fabsf(m[i].y)));
        ra = fmaxf(ra, fmaxf(r[i].x, r[i].y));
      }
      #pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) {
        ma = fmaxf(ma, __shfl_xor_sync(kFullWarp, ma, o));
        ra = fmaxf(ra, __shfl_xor_sync(kFullWarp, ra, o));
      }
      const float mi = block_inverse(ma), ri = block_inverse(ra);
      uint32_t mq[E / 4], vq[E / 4];
      #pragma unroll
      for (int i = 0; i < E / 4; ++i) {
        mq[i] = encode2(mul2(m[2 * i], both(mi))) | encode2(mul2(m[2 * i + 1], both(mi))) << 16;
        vq[i] = encode2(root_codes(r[2 * i], ri)) | encode2(root_codes(r[2 * i + 1], ri)) << 16;
      }
      write_codes(reinterpret_cast<uint8_t*>(a.m) + si, mq);
      write_codes(reinterpret_cast<uint8_t*>(a.v) + si, vq);
      if ((threadIdx.x & (kLanes - 1)) == 0) {           // the lanes' shuffles came after their loads of the old scales
        a.m_scale[si / kStateBlock] = block_scale(ma);
        a.v_scale[si / kStateBlock] = block_scale(ra);
      }
    } else {
      store_pairs<E>(reinterpret_cast<float*>(a.m) + si, m);
      store_pairs<E>(reinterpret_cast<float*>(a.v) + si, v);
    }
  }

 private:
  __device__ __forceinline__ static void write_codes(uint8_t* p, const uint32_t (&q)[E / 4]) {
    if constexpr (E == 16) store16(p, make_uint4(q[0], q[1], q[2], q[3]));
    else if constexpr (E == 8) store8(p, make_uint2(q[0], q[1]));
    else *reinterpret_cast<uint32_t*>(p) = q[0];
  }
};

// Elements a lane takes at once with vectors: eight, and sixteen of 8-bit states (one 16-byte load of
// codes, eight lanes a block) unless parameter or master weight and gradient are both fp32 (W: their
// bytes), which the copies' slots do not hold.
template <bool FP8, int W> constexpr int kLaneElems = FP8 && W <= 6 ? 16 : 8;

// One lane's vectors of a step; V: what the new value is computed from, the parameter's type or fp32.
template <bool FP8, typename P, typename G, typename V>
struct Lane {
  static constexpr int E = kLaneElems<FP8, sizeof(V) + sizeof(G)>;
  RawVec<V, E> p;
  RawVec<G, E> g;
  RawStates<FP8, E> st;

  __device__ __forceinline__ void load(const AdamArgs& a, const V* from, const G* grad, uint64_t si) {
    g.load(grad);
    p.load(from);
    st.load(a, si);
  }

  __device__ __forceinline__ void step(const AdamArgs& a, const StepScalars& s, float keep, P* param, V* from, uint64_t si) const {
    F2 grad[E / 2], value[E / 2], r[E / 2];
    States<FP8, E> states;
    g.pairs(grad);
    p.pairs(value);
    states.decode(st);
    #pragma unroll
    for (int i = 0; i < E / 2; ++i) update2(s, keep, grad[i], states.m[i], states.v[i], value[i], r[i]);
    if constexpr (!std::is_same_v<P, V>) store_pairs<E>(from, value);
    if constexpr (FP8) store_pairs16<E>(param, value);
    else store_pairs<E>(param, value);
    states.store(a, si, r);
  }
};

// Copies of a warp's next vectors into its own shared memory, kStages steps ahead (8-bit states).
// The arithmetic of sixteen elements needs the registers that a register prefetch would take.
// Lanes copy 16 bytes side by side (every sector once) and read back their own elements, so a
// warp's barrier stands after the wait for the copies and before a stage is filled again.
constexpr int kStages = 3, kMaxSlots = 8;
constexpr size_t kStageBytes = (size_t)kStages * kMaxSlots * kThreads * 16;

__device__ __forceinline__ void copy_async16(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory"); }

template <typename P, typename G, typename V>
struct Ahead {
  using L = Lane<true, P, G, V>;
  static constexpr int E = L::E, kP = E * (int)sizeof(V) / 16, kG = E * (int)sizeof(G) / 16;
  static_assert(kP + kG + E / 8 <= kMaxSlots);
  float ms[kStages], vs[kStages];

  // the warp's part of a stage, 512 bytes a slot
  __device__ __forceinline__ static uint4* slot(int stage, int i) {
    extern __shared__ uint4 slots[];
    return slots + ((stage * kWarps + (threadIdx.x >> 5)) * kMaxSlots + i) * 32;
  }
  __device__ __forceinline__ static uint32_t at(int stage, int i) {
    return (uint32_t)__cvta_generic_to_shared(slot(stage, i) + (threadIdx.x & 31));
  }

  // from, grad, si: the warp's first element
  __device__ __forceinline__ void issue(int stage, const AdamArgs& a, const V* from, const G* grad, uint64_t si) {
    const uint32_t lane = threadIdx.x & 31;
    #pragma unroll
    for (int i = 0; i < kP; ++i) copy_async16(at(stage, i), reinterpret_cast<const uint4*>(from) + 32 * i + lane);
    #pragma unroll
    for (int i = 0; i < kG; ++i) copy_async16(at(stage, kP + i), reinterpret_cast<const uint4*>(grad) + 32 * i + lane);
    const uint8_t *m = reinterpret_cast<const uint8_t*>(a.m) + si, *v = reinterpret_cast<const uint8_t*>(a.v) + si;
    if constexpr (E == 16) {
      copy_async16(at(stage, kP + kG), m + 16 * lane);
      copy_async16(at(stage, kP + kG + 1), v + 16 * lane);
    } else {                            // 256 bytes each: half a slot
      copy_async16(at(stage, kP + kG), lane < 16 ? m + 16 * lane : v + 16 * (lane - 16));
    }
    ms[stage] = a.m_scale[(si + lane * E) / kStateBlock];
    vs[stage] = a.v_scale[(si + lane * E) / kStateBlock];
  }

  __device__ __forceinline__ L take(int stage) const {
    L l;
    const uint32_t lane = threadIdx.x & 31;
    #pragma unroll
    for (int i = 0; i < kP; ++i) put(l.p.w + 4 * i, slot(stage, 0)[kP * lane + i]);
    #pragma unroll
    for (int i = 0; i < kG; ++i) put(l.g.w + 4 * i, slot(stage, kP)[kG * lane + i]);
    if constexpr (E == 16) {
      put(l.st.m, slot(stage, kP + kG)[lane]);
      put(l.st.v, slot(stage, kP + kG + 1)[lane]);
    } else {
      const uint2 *m = reinterpret_cast<const uint2*>(slot(stage, kP + kG)) + lane, *v = m + 32;
      l.st.m[0] = m->x, l.st.m[1] = m->y, l.st.v[0] = v->x, l.st.v[1] = v->y;
    }
    l.st.ms = ms[stage];
    l.st.vs = vs[stage];
    return l;
  }

 private:
  __device__ __forceinline__ static void put(uint32_t* w, uint4 v) { w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w; }
};

// Elements a warp takes at once of tensors at odd addresses: as many as the registers hold.
template <bool FP8> constexpr uint32_t kOddSpan = FP8 ? 512 : 256;

// B blocks of 128 elements, four elements a lane and block: parameters and gradients one by one,
// for tensors at odd addresses (FULL) and for the ends of tensors.  The states keep their vectors.
// All loads come before the first store, so that several blocks' are in flight.
template <bool FP8, int B, bool FULL, typename P, typename G, typename V>
__device__ __forceinline__ void step_blocks(const AdamArgs& a, const StepScalars& s, float keep, P* param, V* from, const G* grad, uint64_t si,
                                            uint32_t left) {
  constexpr bool kMaster = !std::is_same_v<P, V>;
  F2 g[B][2], p[B][2], r[2];
  RawStates<FP8, 4> raw[B];
  #pragma unroll
  for (int b = 0; b < B; ++b) {
    const uint32_t at = b * kStateBlock;
    auto one = [&](auto* from, uint32_t k) { return FULL || k < left ? to_f32(from[at + k]) : 0.f; };
    g[b][0] = {one(grad, 0), one(grad, 1)};
    g[b][1] = {one(grad, 2), one(grad, 3)};
    if constexpr (kMaster) {
      load_pairs<4>(from + at, p[b]);
    } else {
      p[b][0] = {one(param, 0), one(param, 1)};
      p[b][1] = {one(param, 2), one(param, 3)};
    }
    raw[b].load(a, si + at);
  }
  #pragma unroll
  for (int b = 0; b < B; ++b) {
    const uint32_t at = b * kStateBlock;
    States<FP8, 4> st;
    st.decode(raw[b]);
    #pragma unroll
    for (int i = 0; i < 2; ++i) update2(s, keep, g[b][i], st.m[i], st.v[i], p[b][i], r[i]);
    if constexpr (kMaster) store_pairs<4>(from + at, p[b]);
    #pragma unroll
    for (int k = 0; k < 4; ++k)
      if (FULL || k < left) param[at + k] = from_f32<P>(k & 1 ? p[b][k / 2].y : p[b][k / 2].x);
    st.store(a, si + at, r);
  }
}

template <bool FP8, typename P, typename G, typename V>
__device__ __forceinline__ void step_chunk(const AdamArgs& a, const StepScalars& s, float keep, const AdamTensor& t, V* from, uint64_t grad,
                                           uint64_t begin, uint64_t end) {
  using L = Lane<FP8, P, G, V>;
  constexpr uint32_t kSpan = 32 * L::E, kStep = kWarps * kSpan;     // elements a warp, a CTA takes at once
  const uint32_t lane = threadIdx.x & 31, off = lane * L::E;
  P* param = reinterpret_cast<P*>(t.param);
  const G* gp = reinterpret_cast<const G*>(grad);
  // 8-bit states: copies and stores of 16 bytes; otherwise vectors of eight elements
  const bool aligned = (t.param & (FP8 ? 15 : 8 * sizeof(P) - 1)) == 0 && (grad & (FP8 ? 15 : 8 * sizeof(G) - 1)) == 0;
  const uint32_t span = aligned ? kSpan : kOddSpan<FP8>;
  uint64_t i = begin + (threadIdx.x >> 5) * span;
  if (!aligned) {
    #pragma unroll 1
    for (; i + kOddSpan<FP8> <= end; i += kWarps * kOddSpan<FP8>) {
      const uint64_t j = i + lane * 4;
      step_blocks<FP8, (int)(kOddSpan<FP8> / kStateBlock), true>(a, s, keep, param + j, from + j, gp + j, t.state + j, 4);
    }
  } else if constexpr (FP8) {
    Ahead<P, G, V> ahead;
    #pragma unroll
    for (int k = 0; k < kStages; ++k) {
      const uint64_t j = i + k * kStep;
      if (j + kSpan <= end) ahead.issue(k, a, from + j, gp + j, t.state + j);
      copies_commit();
    }
    while (i + kSpan <= end) {
      #pragma unroll
      for (int k = 0; k < kStages; ++k) {
        if (i + kSpan > end) break;
        copies_wait();
        __syncwarp();
        ahead.take(k).step(a, s, keep, param + i + off, from + i + off, t.state + i + off);
        __syncwarp();
        const uint64_t j = i + kStages * kStep;
        if (j + kSpan <= end) ahead.issue(k, a, from + j, gp + j, t.state + j);
        copies_commit();
        i += kStep;
      }
    }
  } else {
    #pragma unroll 1
    for (; i + kSpan <= end; i += kStep) {
      const uint64_t j = i + off;
      L cur;
      cur.load(a, from + j, gp + j, t.state + j);
      cur.step(a, s, keep, param + j, from + j, t.state + j);
    }
  }
  // what is left of the tensor is less than a span, of one warp
  const uint64_t stop = min(i + span, end);
  #pragma unroll 1
  for (; i < stop; i += kStateBlock) {
    const uint64_t j = i + lane * 4;
    step_blocks<FP8, 1, false>(a, s, keep, param + j, from + j, gp + j, t.state + j, j < end ? (uint32_t)min(end - j, (uint64_t)4) : 0u);
  }
}

template <bool FP8, bool MASTER, typename P, typename G>
__device__ __forceinline__ void step_chunk_of(const AdamArgs& a, const StepScalars& s, float keep, const AdamTensor& t, uint64_t grad,
                                              uint64_t begin, uint64_t end) {
  if constexpr (MASTER && sizeof(P) == 2) step_chunk<FP8, P, G, float>(a, s, keep, t, a.master + t.state, grad, begin, end);
  else step_chunk<FP8, P, G, P>(a, s, keep, t, reinterpret_cast<P*>(t.param), grad, begin, end);
}

template <bool FP8, bool MASTER, int N>
__global__ void __launch_bounds__(kThreads, kAdamCtas<FP8>) adamw_kernel(const AdamArgs a, const __grid_constant__ Grads<N> g) {
  __shared__ StepScalars shared;
  __shared__ double red[kWarps];
  double sum_sq = 0.0;
  if (a.partial) {
    for (uint32_t i = threadIdx.x; i < a.n_partial; i += kThreads) sum_sq += a.partial[i];
    sum_sq = cta_sum(sum_sq, red);
    if (blockIdx.x == 0 && threadIdx.x == 0 && g.first_tensor == 0) *a.norm = (float)sqrt(sum_sq);
    if (!(sum_sq <= kMaxDouble)) return;              // a step on gradients that are not finite is not taken
  }
  if (threadIdx.x == 0) {
    const double lr = !a.lr_ptr ? a.lr : a.lr_f64 ? *reinterpret_cast<const double*>(a.lr_ptr) : (double)*reinterpret_cast<const float*>(a.lr_ptr);
    const double c1 = 1.0 - a.clock->b1t * a.beta1, c2 = 1.0 - a.clock->b2t * a.beta2;
    const double coef = a.partial ? fmin(1.0, a.max_norm / (sqrt(sum_sq) + 1e-6)) : 1.0;
    shared = StepScalars{(float)a.beta1, (float)(1.0 - a.beta1), (float)a.beta2, (float)(1.0 - a.beta2), (float)(lr / c1),
                         (float)sqrt(1.0 / c2), (float)a.eps, (float)coef, (float)lr};
  }
  __syncthreads();
  const StepScalars s = shared;
  for (uint32_t c = blockIdx.x; c < g.n_chunks; c += gridDim.x) {
    const AdamChunk ch = a.chunks[g.first_chunk + c];
    const uint64_t gp = g.p[ch.tensor - g.first_tensor], grad = gp & ~1ull;
    if (gp == 0) continue;
    const AdamTensor t = a.tensors[ch.tensor];
    const float keep = (float)(1.0 - (double)s.lr * t.weight_decay);
    const uint64_t begin = (uint64_t)ch.chunk * a.chunk, end = begin + a.chunk < t.numel ? begin + a.chunk : t.numel;
    if (t.dtype == DT_F32) step_chunk_of<FP8, MASTER, float, float>(a, s, keep, t, grad, begin, end);
    else if (t.dtype == DT_BF16 && (gp & 1)) step_chunk_of<FP8, MASTER, __nv_bfloat16, float>(a, s, keep, t, grad, begin, end);
    else if (t.dtype == DT_BF16) step_chunk_of<FP8, MASTER, __nv_bfloat16, __nv_bfloat16>(a, s, keep, t, grad, begin, end);
    else if (gp & 1) step_chunk_of<FP8, MASTER, __half, float>(a, s, keep, t, grad, begin, end);
    else step_chunk_of<FP8, MASTER, __half, __half>(a, s, keep, t, grad, begin, end);
  }
  // the last CTA of a step's last launch advances the clock; all others have read it by then
  if (g.last && threadIdx.x == 0) {
    __threadfence();
    if (atomicAdd(&a.clock->done, 1u) == gridDim.x - 1) {
      a.clock->done = 0;
      a.clock->step += 1;
      a.clock->b1t *= a.beta1;
      a.clock->b2t *= a.beta2;
    }
  }
}

template <bool FP8, bool MASTER, int N>
cudaError_t adamw_launch_n(const AdamArgs& a, const uint64_t* grads, const uint32_t* chunk_start, uint32_t first, uint32_t n,
                           int sms, cudaStream_t stream) {
  Grads<N> g;
  for (uint32_t i = 0; i < n; ++i) g.p[i] = grads[first + i];
  g.first_tensor = first;
  g.first_chunk = chunk_start[first];
  g.n_chunks = chunk_start[first + n] - g.first_chunk;
  g.last = first + n == a.n_tensors;
  // 8-bit states: all CTAs resident at once; fp32 states: twice as many as are, 1 % faster
  const uint32_t cap = (uint32_t)(sms * (FP8 ? kAdamCtas<FP8> : 2 * kAdamCtas<FP8>));
  const uint32_t grid = g.n_chunks < 1 ? 1 : g.n_chunks < cap ? g.n_chunks : cap;
  const size_t shared = FP8 ? kStageBytes : 0;
  if (FP8) {
    const cudaError_t e = cudaFuncSetAttribute(adamw_kernel<FP8, MASTER, N>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)shared);
    if (e != cudaSuccess) return e;
  }
  adamw_kernel<FP8, MASTER, N><<<grid, kThreads, shared, stream>>>(a, g);
  return cudaGetLastError();
}

template <bool FP8, bool MASTER>
cudaError_t adamw_launch(const AdamArgs& a, const uint64_t* grads, const uint32_t* chunk_start, int sms, cudaStream_t stream) {
  for (uint32_t first = 0; first < a.n_tensors; first += kGradsPerLaunch) {
    const uint32_t n = a.n_tensors - first < kGradsPerLaunch ? a.n_tensors - first : kGradsPerLaunch;
    // launch arguments are copied per launch: a small optimizer does not pay for thousands of addresses
    const cudaError_t e = n <= 64 ? adamw_launch_n<FP8, MASTER, 64>(a, grads, chunk_start, first, n, sms, stream)
                          : n <= 512 ? adamw_launch_n<FP8, MASTER, 512>(a, grads, chunk_start, first, n, sms, stream)
                                     : adamw_launch_n<FP8, MASTER, kGradsPerLaunch>(a, grads, chunk_start, first, n, sms, stream);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

// -- sum of squares -------------------------------------------------------------------------------
template <int N>
struct NormTable {
  NormTensor t[N];
  uint32_t n, n_chunks;
};

// Elements [begin, end) counted from the 32-byte boundary at or below the tensor's start, of which
// [mis, mis + numel) are the tensor's.  Each thread adds at most 64 squares in 32 bits.
template <typename T>
__device__ __forceinline__ float chunk_squares(const NormTensor& t, uint64_t begin) {
  constexpr int V = kVecN<T>, kDepth = 4;
  const T* x = reinterpret_cast<const T*>(t.ptr);
  const uint32_t mis = (uint32_t)(t.ptr & 31) / sizeof(T);
  const uint64_t end = t.numel + mis;
  float sum = 0.f;
  F2 acc{0.f, 0.f};
  if (begin >= mis && begin + kNormChunk <= end) {
    const T* p = x + (begin - mis) + threadIdx.x * V;
    #pragma unroll
    for (uint32_t k = 0; k < kNormChunk; k += kDepth * kThreads * V) {
      Vec32 raw[kDepth];
      #pragma unroll
      for (int u = 0; u < kDepth; ++u) raw[u] = load32(p + k + u * kThreads * V);
      #pragma unroll
      for (int u = 0; u < kDepth; ++u) {
        F2 v[V / 2];
        unpack<T>(raw[u], v);
        #pragma unroll
        for (int i = 0; i < V / 2; ++i) acc = fma2(v[i], v[i], acc);
      }
    }
    sum = acc.x + acc.y;
  } else {
    for (uint64_t i = begin + threadIdx.x; i < begin + kNormChunk && i < end; i += kThreads)
      if (i >= mis) {
        const float f = to_f32(x[i - mis]);
        sum += f * f;
      }
  }
  return sum;
}

template <int N>
__global__ void __launch_bounds__(kThreads) partial_sums_kernel(const __grid_constant__ NormTable<N> tab, double* partial) {
  __shared__ double red[kWarps];
  double acc = 0.0;
  for (uint32_t c = blockIdx.x; c < tab.n_chunks; c += gridDim.x) {
    uint32_t lo = 0, hi = tab.n;                  // the tensor whose chunks hold c
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) / 2;
      if (tab.t[mid].first_chunk <= c) lo = mid; else hi = mid;
    }
    const NormTensor& t = tab.t[lo];
    const uint64_t begin = (uint64_t)(c - t.first_chunk) * kNormChunk;
    acc += t.dtype == DT_F32 ? chunk_squares<float>(t, begin)
           : t.dtype == DT_BF16 ? chunk_squares<__nv_bfloat16>(t, begin) : chunk_squares<__half>(t, begin);
  }
  acc = cta_sum(acc, red);
  if (threadIdx.x == 0) partial[blockIdx.x] = acc;
}

__global__ void __launch_bounds__(kThreads) norm_kernel(const double* partial, uint32_t n, double* sum_sq, float* norm) {
  __shared__ double red[kWarps];
  double acc = 0.0;
  for (uint32_t i = threadIdx.x; i < n; i += kThreads) acc += partial[i];
  acc = cta_sum(acc, red);
  if (threadIdx.x == 0) {
    *sum_sq = acc;
    *norm = (float)sqrt(acc);
  }
}

constexpr uint32_t kNormCtas = 4;         // per SM

uint32_t chunks_of(const NormTensor& t) {
  const uint64_t mis = (t.ptr & 31) / dtype_bytes(t.dtype);
  return (uint32_t)((t.numel + mis + kNormChunk - 1) / kNormChunk);
}

template <int N>
uint32_t partial_sums_launch(NormTensor* t, uint32_t n, double* partial, int sms, cudaStream_t stream) {
  NormTable<N> tab;
  tab.n_chunks = 0;
  for (uint32_t i = 0; i < n; ++i) {
    t[i].first_chunk = tab.n_chunks;
    tab.n_chunks += chunks_of(t[i]);
    tab.t[i] = t[i];
  }
  tab.n = n;
  const uint32_t cap = (uint32_t)sms * kNormCtas, grid = tab.n_chunks < cap ? tab.n_chunks : cap;
  if (grid) partial_sums_kernel<N><<<grid, kThreads, 0, stream>>>(tab, partial);
  return grid;
}

}  // namespace

cudaError_t launch_adamw(const AdamArgs& a, const uint64_t* grads, const uint32_t* chunk_start, int sms, cudaStream_t stream) {
  const auto launch = a.m_scale ? (a.master ? adamw_launch<true, true> : adamw_launch<true, false>)
                                : (a.master ? adamw_launch<false, true> : adamw_launch<false, false>);
  return launch(a, grads, chunk_start, sms, stream);
}

uint64_t partial_sums_size(uint32_t n, int sms) {
  return (uint64_t)((n + kNormTensorsPerLaunch - 1) / kNormTensorsPerLaunch) * (uint64_t)sms * kNormCtas;
}

cudaError_t launch_partial_sums(NormTensor* t, uint32_t n, double* partial, uint32_t* n_partial, int sms, cudaStream_t stream) {
  *n_partial = 0;
  for (uint32_t first = 0; first < n; first += kNormTensorsPerLaunch) {
    const uint32_t k = n - first < kNormTensorsPerLaunch ? n - first : kNormTensorsPerLaunch;
    *n_partial += k <= 128 ? partial_sums_launch<128>(t + first, k, partial + *n_partial, sms, stream)
                  : k <= 512 ? partial_sums_launch<512>(t + first, k, partial + *n_partial, sms, stream)
                             : partial_sums_launch<kNormTensorsPerLaunch>(t + first, k, partial + *n_partial, sms, stream);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

cudaError_t launch_norm(const double* partial, uint32_t n_partial, double* sum_sq, float* norm, cudaStream_t stream) {
  norm_kernel<<<1, kThreads, 0, stream>>>(partial, n_partial, sum_sq, norm);
  return cudaGetLastError();
}

}  // namespace wb
