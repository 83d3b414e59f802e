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
#include "wb_optim.h"

#include <cuda_fp8.h>

#include "wb_vec.cuh"

namespace wb {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr double kMaxDouble = 1.7976931348623157e308;

__device__ __forceinline__ float load_as_f32(uint64_t p, uint32_t dtype, uint64_t i) {
  if (dtype == DT_F32) return reinterpret_cast<const float*>(p)[i];
  if (dtype == DT_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(reinterpret_cast<const __half*>(p)[i]);
}

__device__ __forceinline__ void store_from_f32(uint64_t p, uint32_t dtype, uint64_t i, float x) {
  if (dtype == DT_F32) reinterpret_cast<float*>(p)[i] = x;
  else if (dtype == DT_BF16) reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
  else reinterpret_cast<__half*>(p)[i] = __float2half_rn(x);
}

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

// Scale of a block, amax / 448, and 448 / amax, each with one correction step after the product
// (the reciprocal of the rounded scale would round once more).  A block of tiny values keeps a
// normal scale, whose reciprocal is finite; a block of zeros has scale 1.
__device__ __forceinline__ float block_scale(float amax) {
  constexpr float kInv = 1.f / kE4M3Max;
  float q = amax * kInv;
  q = fmaf(fmaf(-kE4M3Max, q, amax), kInv, q);
  return amax > 0.f ? fmaxf(q, 1.17549435e-38f) : 1.f;
}
__device__ __forceinline__ float block_inverse(float amax) {
  const float r = reciprocal(amax);
  float q = kE4M3Max * r;
  q = fmaf(fmaf(-amax, q, kE4M3Max), r, q);
  return fminf(q, 8.507059173e37f);         // 2^126, also where the above is not a number (zero and tiny blocks)
}

// r in units of the scale; a positive r keeps at least the smallest code
__device__ __forceinline__ F2 root_codes(F2 r, float inv) {
  const F2 q = mul2(r, both(inv));
  return {fmaxf(q.x, r.x > 0.f ? 0.001953125f : 0.f), fmaxf(q.y, r.y > 0.f ? 0.001953125f : 0.f)};
}

// E consecutive elements of the states of one lane, as pairs.  Slices of the flat buffers are
// padded to whole blocks, so a lane may pass the tensor's end: there the states are and stay 0.
template <bool FP8, int E>
struct States {
  F2 m[E / 2], v[E / 2];

  __device__ __forceinline__ void load(const AdamArgs& a, uint64_t si) {
    if constexpr (FP8) {
      uint32_t mq[E / 4], vq[E / 4];
      read_codes(reinterpret_cast<const uint8_t*>(a.m) + si, mq);
      read_codes(reinterpret_cast<const uint8_t*>(a.v) + si, vq);
      const F2 ms = both(a.m_scale[si / kStateBlock]), vs = both(a.v_scale[si / kStateBlock]);
      #pragma unroll
      for (int i = 0; i < E / 2; ++i) {
        m[i] = mul2(decode2(i & 1 ? mq[i / 2] >> 16 : mq[i / 2]), ms);
        const F2 r = mul2(decode2(i & 1 ? vq[i / 2] >> 16 : vq[i / 2]), vs);
        v[i] = mul2(r, r);
      }
    } else {
      load_pairs<E>(reinterpret_cast<const float*>(a.m) + si, m);
      load_pairs<E>(reinterpret_cast<const float*>(a.v) + si, v);
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
  __device__ __forceinline__ static void read_codes(const uint8_t* p, uint32_t (&q)[E / 4]) {
    if constexpr (E == 16) {
      const uint4 w = load16(p);
      q[0] = w.x, q[1] = w.y, q[2] = w.z, q[3] = w.w;
    } else {
      static_assert(E == 4);
      q[0] = *reinterpret_cast<const uint32_t*>(p);
    }
  }
  __device__ __forceinline__ static void write_codes(uint8_t* p, const uint32_t (&q)[E / 4]) {
    if constexpr (E == 16) store16(p, make_uint4(q[0], q[1], q[2], q[3]));
    else *reinterpret_cast<uint32_t*>(p) = q[0];
  }
};

// E elements a lane with vectors, all addresses aligned to them.  Eight for fp32 states (64 bytes
// of them in flight a lane), sixteen for 8-bit ones (16-byte loads of codes, eight lanes a block).
template <bool FP8> constexpr int kLaneElems = FP8 ? 16 : 8;

template <bool FP8, typename P, typename G>
__device__ __forceinline__ void step_vector(const AdamArgs& a, const StepScalars& s, float keep, P* param, const G* grad, uint64_t si) {
  constexpr int E = kLaneElems<FP8>;
  F2 g[E / 2], p[E / 2], r[E / 2];
  States<FP8, E> st;
  load_pairs<E>(grad, g);
  if (a.master) load_pairs<E>(a.master + si, p);
  else load_pairs<E>(param, p);
  st.load(a, si);
  #pragma unroll
  for (int i = 0; i < E / 2; ++i) update2(s, keep, g[i], st.m[i], st.v[i], p[i], r[i]);
  if (a.master) store_pairs<E>(a.master + si, p);
  store_pairs<E>(param, p);
  st.store(a, si, r);
}

// A block of 128 elements, four a lane: parameters and gradients one by one, for tensors at odd
// addresses (FULL) and for the ends of tensors.  The states keep their vectors.
template <bool FP8, bool FULL, typename P, typename G>
__device__ __forceinline__ void step_block(const AdamArgs& a, const StepScalars& s, float keep, P* param, const G* grad, uint64_t si, uint32_t left) {
  float g[4], p[4];
  States<FP8, 4> st;
  #pragma unroll
  for (int k = 0; k < 4; ++k) g[k] = FULL || k < left ? to_f32(grad[k]) : 0.f;
  if (a.master) {
    F2 w[2];
    load_pairs<4>(a.master + si, w);
    p[0] = w[0].x, p[1] = w[0].y, p[2] = w[1].x, p[3] = w[1].y;
  } else {
    #pragma unroll
    for (int k = 0; k < 4; ++k) p[k] = FULL || k < left ? to_f32(param[k]) : 0.f;
  }
  st.load(a, si);
  F2 w[2] = {{p[0], p[1]}, {p[2], p[3]}}, r[2];
  update2(s, keep, {g[0], g[1]}, st.m[0], st.v[0], w[0], r[0]);
  update2(s, keep, {g[2], g[3]}, st.m[1], st.v[1], w[1], r[1]);
  if (a.master) store_pairs<4>(a.master + si, w);
  p[0] = w[0].x, p[1] = w[0].y, p[2] = w[1].x, p[3] = w[1].y;
  #pragma unroll
  for (int k = 0; k < 4; ++k)
    if (FULL || k < left) param[k] = from_f32<P>(p[k]);
  st.store(a, si, r);
}

template <bool FP8, typename P, typename G>
__device__ __forceinline__ void step_chunk(const AdamArgs& a, const StepScalars& s, float keep, const AdamTensor& t, uint64_t grad,
                                           uint64_t begin, uint64_t end) {
  constexpr uint32_t kSpan = 32 * kLaneElems<FP8>;        // elements of a warp's step
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  P* param = reinterpret_cast<P*>(t.param);
  const G* gp = reinterpret_cast<const G*>(grad);
  const bool aligned = ((t.param | grad) & 31) == 0;
  for (uint64_t i = begin + warp * kSpan; i < end; i += kWarps * kSpan) {
    if (aligned && i + kSpan <= end) {
      const uint64_t j = i + lane * kLaneElems<FP8>;
      step_vector<FP8>(a, s, keep, param + j, gp + j, t.state + j);
    } else {
      for (uint64_t b = i; b < i + kSpan && b < end; b += kStateBlock) {
        const uint64_t j = b + lane * 4;
        if (b + kStateBlock <= end) step_block<FP8, true>(a, s, keep, param + j, gp + j, t.state + j, 4);
        else step_block<FP8, false>(a, s, keep, param + j, gp + j, t.state + j, j < end ? (uint32_t)(end - j) : 0u);
      }
    }
  }
}

template <bool FP8, int N>
__global__ void __launch_bounds__(kThreads) adamw_kernel(const AdamArgs a, const __grid_constant__ Grads<N> g) {
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
    if (t.dtype == DT_F32) step_chunk<FP8, float, float>(a, s, keep, t, grad, begin, end);
    else if (t.dtype == DT_BF16 && (gp & 1)) step_chunk<FP8, __nv_bfloat16, float>(a, s, keep, t, grad, begin, end);
    else if (t.dtype == DT_BF16) step_chunk<FP8, __nv_bfloat16, __nv_bfloat16>(a, s, keep, t, grad, begin, end);
    else if (gp & 1) step_chunk<FP8, __half, float>(a, s, keep, t, grad, begin, end);
    else step_chunk<FP8, __half, __half>(a, s, keep, t, grad, begin, end);
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

template <bool FP8, int N>
cudaError_t adamw_launch_n(const AdamArgs& a, const uint64_t* grads, const uint32_t* chunk_start, uint32_t first, uint32_t n,
                           int sms, cudaStream_t stream) {
  Grads<N> g;
  for (uint32_t i = 0; i < n; ++i) g.p[i] = grads[first + i];
  g.first_tensor = first;
  g.first_chunk = chunk_start[first];
  g.n_chunks = chunk_start[first + n] - g.first_chunk;
  g.last = first + n == a.n_tensors;
  const uint32_t cap = (uint32_t)sms * 8u;
  const uint32_t grid = g.n_chunks < 1 ? 1 : g.n_chunks < cap ? g.n_chunks : cap;
  adamw_kernel<FP8, N><<<grid, kThreads, 0, stream>>>(a, g);
  return cudaGetLastError();
}

template <bool FP8>
cudaError_t adamw_launch(const AdamArgs& a, const uint64_t* grads, const uint32_t* chunk_start, int sms, cudaStream_t stream) {
  for (uint32_t first = 0; first < a.n_tensors; first += kGradsPerLaunch) {
    const uint32_t n = a.n_tensors - first < kGradsPerLaunch ? a.n_tensors - first : kGradsPerLaunch;
    // launch arguments are copied per launch: a small optimizer does not pay for thousands of addresses
    const cudaError_t e = n <= 64 ? adamw_launch_n<FP8, 64>(a, grads, chunk_start, first, n, sms, stream)
                          : n <= 512 ? adamw_launch_n<FP8, 512>(a, grads, chunk_start, first, n, sms, stream)
                                     : adamw_launch_n<FP8, kGradsPerLaunch>(a, grads, chunk_start, first, n, sms, stream);
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
  return a.m_scale ? adamw_launch<true>(a, grads, chunk_start, sms, stream) : adamw_launch<false>(a, grads, chunk_start, sms, stream);
}

uint64_t partial_sums_size(uint32_t n, int sms) {
  return (uint64_t)((n + kNormTensorsPerLaunch - 1) / kNormTensorsPerLaunch) * (uint64_t)sms * kNormCtas;
}

cudaError_t launch_partial_sums(NormTensor* t, uint32_t n, double* partial, uint32_t* n_partial, int sms, cudaStream_t stream) {
  *n_partial = 0;
  for (uint32_t first = 0; first < n; first += kNormTensorsPerLaunch) {
    const uint32_t k = n - first < kNormTensorsPerLaunch ? n - first : kNormTensorsPerLaunch;
    *n_partial += k <= 128 ? partial_sums_launch<128>(t + first, k, partial + *n_partial, sms, stream)
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
