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

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

namespace wb {
namespace {

constexpr int kThreads = 256;

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

__device__ __forceinline__ float e4m3_to_f32(uint8_t q) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(q, __NV_E4M3)));
}

struct StepScalars { float b1, om_b1, b2, om_b2, step_size, inv_c2, eps, coef; double lr; };

template <int N>
struct Grads {
  uint64_t p[N];
  uint32_t first_tensor, first_chunk, n_chunks, last;
};

__device__ __forceinline__ float warp_max(float v) {
  #pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, o));
  return v;
}

// scale of a block; tiny blocks keep a normal scale, whose reciprocal is finite
__device__ __forceinline__ float block_scale(float amax) {
  return amax > 0.f ? fmaxf(__fdiv_rn(amax, kE4M3Max), 1.17549435e-38f) : 1.f;
}

template <bool FP8, int N>
__global__ void __launch_bounds__(kThreads) adamw_kernel(const AdamArgs a, const __grid_constant__ Grads<N> g) {
  __shared__ StepScalars s;
  __shared__ bool skip;
  if (threadIdx.x == 0) {
    const double lr = !a.lr_ptr ? a.lr : a.lr_f64 ? *reinterpret_cast<const double*>(a.lr_ptr) : (double)*reinterpret_cast<const float*>(a.lr_ptr);
    const double c1 = 1.0 - a.clock->b1t * a.beta1, c2 = 1.0 - a.clock->b2t * a.beta2;
    double coef = 1.0;
    skip = false;
    if (a.sum_sq) {
      const double norm = sqrt(*a.sum_sq);
      coef = fmin(1.0, a.max_norm / (norm + 1e-6));
      skip = !(norm <= 1.7976931348623157e308);       // a step on gradients that are not finite is not taken
      if (blockIdx.x == 0 && g.first_tensor == 0) *a.norm = (float)norm;
    }
    s = StepScalars{(float)a.beta1, (float)(1.0 - a.beta1), (float)a.beta2, (float)(1.0 - a.beta2), (float)(lr / c1),
                    (float)(1.0 / c2), (float)a.eps, (float)coef, lr};
  }
  __syncthreads();
  if (skip) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (uint32_t c = blockIdx.x; c < g.n_chunks; c += gridDim.x) {
    const AdamChunk ch = a.chunks[g.first_chunk + c];
    const AdamTensor t = a.tensors[ch.tensor];
    const uint64_t gp = g.p[ch.tensor - g.first_tensor];
    if (gp == 0) continue;
    const uint32_t gtype = gp & 1 ? (uint32_t)DT_F32 : t.dtype;
    const float keep = (float)(1.0 - s.lr * t.weight_decay);
    const uint64_t begin = (uint64_t)ch.chunk * kAdamChunk;
    const uint64_t end = begin + kAdamChunk < t.numel ? begin + kAdamChunk : t.numel;
    for (uint64_t b = begin + warp * kStateBlock; b < end; b += kThreads / 32 * kStateBlock) {
      const uint64_t blk = (t.state + b) / kStateBlock;
      float m[4], r[4], ma = 0.f, ra = 0.f;
      #pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint64_t i = b + lane + 32 * k, si = t.state + i;
        m[k] = r[k] = 0.f;
        if (i >= end) continue;
        const float grad = load_as_f32(gp & ~1ull, gtype, i) * s.coef;
        float m0, v0;
        if constexpr (FP8) {
          m0 = e4m3_to_f32(reinterpret_cast<const uint8_t*>(a.m)[si]) * a.m_scale[blk];
          const float r0 = e4m3_to_f32(reinterpret_cast<const uint8_t*>(a.v)[si]) * a.v_scale[blk];
          v0 = r0 * r0;
        } else {
          m0 = reinterpret_cast<const float*>(a.m)[si];
          v0 = reinterpret_cast<const float*>(a.v)[si];
        }
        m[k] = s.b1 * m0 + s.om_b1 * grad;
        const float v = s.b2 * v0 + s.om_b2 * grad * grad;
        float p = a.master ? a.master[si] : load_as_f32(t.param, t.dtype, i);
        p = p * keep - s.step_size * (m[k] / (sqrtf(v * s.inv_c2) + s.eps));
        if (a.master) a.master[si] = p;
        store_from_f32(t.param, t.dtype, i, p);
        if constexpr (FP8) {
          r[k] = sqrtf(v);
          ma = fmaxf(ma, fabsf(m[k]));
          ra = fmaxf(ra, r[k]);
        } else {
          reinterpret_cast<float*>(a.m)[si] = m[k];
          reinterpret_cast<float*>(a.v)[si] = v;
        }
      }
      if constexpr (FP8) {
        const float ms = block_scale(warp_max(ma)), rs = block_scale(warp_max(ra));
        const float mi = __frcp_rn(ms), ri = __frcp_rn(rs);
        #pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint64_t i = b + lane + 32 * k, si = t.state + i;
          if (i >= end) continue;
          reinterpret_cast<uint8_t*>(a.m)[si] = __nv_cvt_float_to_fp8(m[k] * mi, __NV_SATFINITE, __NV_E4M3);
          uint8_t q = __nv_cvt_float_to_fp8(r[k] * ri, __NV_SATFINITE, __NV_E4M3);
          if (r[k] > 0.f && q == 0) q = 1;
          reinterpret_cast<uint8_t*>(a.v)[si] = q;
        }
        __syncwarp();       // every lane has read the old scales
        if (lane == 0) {
          a.m_scale[blk] = ms;
          a.v_scale[blk] = rs;
        }
      }
    }
  }
  // the last CTA of a step's last launch advances the clock; all others have read it by then
  if (!g.last) return;
  __syncthreads();
  if (threadIdx.x == 0) {
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
  Grads<N> g{};
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

// -- sum of squares -----------------------------------------------------------------------------
template <int N>
struct NormTable {
  NormTensor t[N];
  uint32_t n, n_chunks;
};

__device__ __forceinline__ double cta_sum(double v, double* red) {
  #pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0;
  for (int i = 0; i < kThreads / 32; ++i) v += red[i];
  return v;
}

template <int N>
__global__ void __launch_bounds__(kThreads) sum_sq_kernel(const __grid_constant__ NormTable<N> tab, double* partial) {
  __shared__ double red[kThreads / 32];
  double acc = 0.0;
  for (uint32_t c = blockIdx.x; c < tab.n_chunks; c += gridDim.x) {
    uint32_t lo = 0, hi = tab.n;                  // the tensor whose chunks hold c
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) / 2;
      if (tab.t[mid].first_chunk <= c) lo = mid; else hi = mid;
    }
    const NormTensor& t = tab.t[lo];
    const uint64_t begin = (uint64_t)(c - t.first_chunk) * kNormChunk;
    const uint64_t end = begin + kNormChunk < t.numel ? begin + kNormChunk : t.numel;
    float s = 0.f;                                // at most 64 squares; sums of those in 64 bits
    for (uint64_t i = begin + threadIdx.x; i < end; i += kThreads) {
      const float x = load_as_f32(t.ptr, t.dtype, i);
      s += x * x;
    }
    acc += s;
  }
  acc = cta_sum(acc, red);
  if (threadIdx.x == 0) partial[blockIdx.x] = acc;
}

__global__ void __launch_bounds__(kThreads) sum_sq_final_kernel(const double* partial, uint32_t n, double* sum_sq, float* norm) {
  __shared__ double red[kThreads / 32];
  double acc = 0.0;
  for (uint32_t i = threadIdx.x; i < n; i += kThreads) acc += partial[i];
  acc = cta_sum(acc, red);
  if (threadIdx.x == 0) {
    *sum_sq = acc;
    *norm = (float)sqrt(acc);
  }
}

uint32_t norm_grid(uint32_t n_chunks, int sms) {
  const uint32_t cap = (uint32_t)sms * 8u;
  return n_chunks < cap ? n_chunks : cap;
}

uint32_t chunks_of(const NormTensor& t) { return (uint32_t)((t.numel + kNormChunk - 1) / kNormChunk); }

template <int N>
uint32_t sum_sq_launch_n(NormTensor* t, uint32_t n, double* partial, int sms, cudaStream_t stream) {
  NormTable<N> tab{};
  for (uint32_t i = 0; i < n; ++i) {
    t[i].first_chunk = tab.n_chunks;
    tab.n_chunks += chunks_of(t[i]);
    tab.t[i] = t[i];
  }
  tab.n = n;
  const uint32_t grid = norm_grid(tab.n_chunks, sms);
  if (grid) sum_sq_kernel<N><<<grid, kThreads, 0, stream>>>(tab, partial);
  return grid;
}

}  // namespace

cudaError_t launch_adamw(const AdamArgs& a, const uint64_t* grads, const uint32_t* chunk_start, int sms, cudaStream_t stream) {
  return a.m_scale ? adamw_launch<true>(a, grads, chunk_start, sms, stream) : adamw_launch<false>(a, grads, chunk_start, sms, stream);
}

uint64_t sum_sq_scratch(const NormTensor* t, uint32_t n, int sms) {
  const uint64_t launches = (n + kNormTensorsPerLaunch - 1) / kNormTensorsPerLaunch;
  return launches * (uint64_t)sms * 8u + 1;
}

cudaError_t launch_sum_sq(NormTensor* t, uint32_t n, double* scratch, double* sum_sq, float* norm, int sms, cudaStream_t stream) {
  uint32_t used = 0;
  for (uint32_t first = 0; first < n; first += kNormTensorsPerLaunch) {
    const uint32_t k = n - first < kNormTensorsPerLaunch ? n - first : kNormTensorsPerLaunch;
    used += k <= 128 ? sum_sq_launch_n<128>(t + first, k, scratch + used, sms, stream)
                     : sum_sq_launch_n<kNormTensorsPerLaunch>(t + first, k, scratch + used, sms, stream);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
  }
  sum_sq_final_kernel<<<1, kThreads, 0, stream>>>(scratch, used, sum_sq, norm);
  return cudaGetLastError();
}

}  // namespace wb
