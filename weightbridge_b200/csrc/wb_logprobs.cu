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
#include "wb_logprobs.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace wb {
namespace {

constexpr int kThreads = 256;
constexpr float kInf = __builtin_huge_valf();

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }

template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }

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

// Whole numbers in the order of the floats: -0 equals +0, NaN lies above everything.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

struct Sum2 { float s, a; };

template <typename V, typename F>
__device__ __forceinline__ V cta_reduce(V v, V* red, F op) {
  #pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    V w;
    if constexpr (sizeof(V) == 8 && !std::is_same_v<V, unsigned long long>) {
      w = V{__shfl_xor_sync(~0u, v.s, o), __shfl_xor_sync(~0u, v.a, o)};
    } else {
      w = __shfl_xor_sync(~0u, v, o);
    }
    v = op(v, w);
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
  for (int i = 1; i < kThreads / 32; ++i) v = op(v, red[i]);
  return v;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) logprobs_kernel(const LogprobRows in, const LogprobOut out) {
  __shared__ unsigned long long red[kThreads / 32];
  const uint32_t r = blockIdx.x;
  const int64_t tok = token_of(in, r);
  if (tok == in.ignore_index) {
    if (threadIdx.x == 0) {
      out.logprobs[r] = 0.f;
      out.entropy[r] = 0.f;
      if (out.stats) out.stats[2 * r] = out.stats[2 * r + 1] = 0.f;
    }
    if ((int)threadIdx.x < out.top_k) {
      out.top_logprobs[(int64_t)r * out.top_k + threadIdx.x] = -kInf;
      out.top_ids[(int64_t)r * out.top_k + threadIdx.x] = -1;
    }
    return;
  }
  const T* x = row_ptr<T>(in, r);
  float m = -kInf;
  for (uint32_t j = threadIdx.x; j < in.vocab; j += kThreads) m = fmaxf(m, to_f32(x[j]));
  m = cta_reduce(m, reinterpret_cast<float*>(red), [](float a, float b) { return fmaxf(a, b); });
  if (m == -kInf) m = 0.f;
  Sum2 t{0.f, 0.f};
  for (uint32_t j = threadIdx.x; j < in.vocab; j += kThreads) {
    const float z = (to_f32(x[j]) - m) * in.inv_temp, e = __expf(z);
    t.s += e;
    t.a += e * fmaxf(z, -1e30f);
  }
  t = cta_reduce(t, reinterpret_cast<Sum2*>(red), [](Sum2 a, Sum2 b) { return Sum2{a.s + b.s, a.a + b.a}; });
  const bool empty = t.s == 0.f;
  const float ln = empty ? kInf : logf(t.s);
  if (threadIdx.x == 0) {
    float lp = __int_as_float(0x7fffffff);
    if (tok >= 0 && tok < (int64_t)in.vocab) lp = empty ? -kInf : (to_f32(x[tok]) - m) * in.inv_temp - ln;
    out.logprobs[r] = lp;
    out.entropy[r] = empty ? 0.f : ln - t.a / t.s;
    if (out.stats) {
      out.stats[2 * r] = m;
      out.stats[2 * r + 1] = ln;
    }
  }
  unsigned long long last = ~0ull;
  for (int k = 0; k < out.top_k; ++k) {
    // the largest of what lies below the one before: the logit's order, then the lower column first
    unsigned long long best = 0;
    for (uint32_t j = threadIdx.x; j < in.vocab; j += kThreads) {
      const unsigned long long key = (unsigned long long)order_key(to_f32(x[j])) << 32 | (0xffffffffu - j);
      if (key < last && key > best) best = key;
    }
    best = cta_reduce(best, red, [](unsigned long long a, unsigned long long b) { return a > b ? a : b; });
    last = best;
    if (threadIdx.x == 0) {
      const uint32_t j = 0xffffffffu - (uint32_t)best;
      out.top_ids[(int64_t)r * out.top_k + k] = j;
      out.top_logprobs[(int64_t)r * out.top_k + k] = empty ? -kInf : (to_f32(x[j]) - m) * in.inv_temp - ln;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) logprobs_grad_kernel(const LogprobRows in, const LogprobGrad g) {
  const uint32_t r = blockIdx.x;
  const int64_t tok = token_of(in, r);
  const T* x = row_ptr<T>(in, r);
  T* d = reinterpret_cast<T*>(g.grad) + (int64_t)r * g.cols;
  const float m = g.stats[2 * r], ln = g.stats[2 * r + 1], h = g.entropy[r];
  float glp = g.g_logprobs ? g.g_logprobs[r * g.g_logprobs_stride] : 0.f;
  const float gh = g.g_entropy ? g.g_entropy[r * g.g_entropy_stride] : 0.f;
  const bool dead = tok == in.ignore_index || ln == kInf;
  if (tok < 0 || tok >= (int64_t)in.vocab) glp = __int_as_float(0x7fffffff);
  for (uint32_t j = threadIdx.x; j < g.cols; j += kThreads) {
    float v = 0.f;
    if (!dead && j < in.vocab) {
      const float lp = (to_f32(x[j]) - m) * in.inv_temp - ln, p = __expf(lp);
      v = -p * (glp + gh * (fmaxf(lp, -1e30f) + h));
      if ((int64_t)j == tok) v += glp;
      v *= in.inv_temp;
    }
    d[j] = from_f32<T>(v);
  }
}

template <typename F>
cudaError_t by_type(uint32_t dtype, F f) {
  switch (dtype) {
    case DT_BF16: f(__nv_bfloat16{}); break;
    case DT_F16: f(__half{}); break;
    case DT_F32: f(float{}); break;
    default: return cudaErrorInvalidValue;
  }
  return cudaGetLastError();
}

bool ok(const LogprobRows& in) { return in.rows < 0x7fffffffu && in.vocab >= 1 && in.inner >= 1; }

}  // namespace

cudaError_t launch_token_logprobs(const LogprobRows& in, const LogprobOut& out, cudaStream_t stream) {
  if (!ok(in) || out.top_k < 0 || out.top_k > kLogprobMaxTop || (uint32_t)out.top_k > in.vocab) return cudaErrorInvalidValue;
  if (in.rows == 0) return cudaSuccess;
  return by_type(in.dtype, [&](auto t) { logprobs_kernel<decltype(t)><<<in.rows, kThreads, 0, stream>>>(in, out); });
}

cudaError_t launch_token_logprobs_grad(const LogprobRows& in, const LogprobGrad& g, cudaStream_t stream) {
  if (!ok(in) || g.cols < in.vocab) return cudaErrorInvalidValue;
  if (in.rows == 0) return cudaSuccess;
  return by_type(in.dtype, [&](auto t) { logprobs_grad_kernel<decltype(t)><<<in.rows, kThreads, 0, stream>>>(in, g); });
}

}  // namespace wb
