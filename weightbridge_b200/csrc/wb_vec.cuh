// 32-byte vectors of elements and packed fp32 arithmetic, shared by the operator kernels.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cstdint>
#include <type_traits>

namespace wb {

constexpr uint32_t kFullWarp = 0xffffffffu;

// 32 bytes: one load or store instruction a lane, 1 KiB a warp.
struct Vec32 { uint32_t w[8]; };

__device__ __forceinline__ Vec32 load32(const void* p) {
  Vec32 v;
  asm volatile("ld.global.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(v.w[0]), "=r"(v.w[1]), "=r"(v.w[2]), "=r"(v.w[3]), "=r"(v.w[4]), "=r"(v.w[5]), "=r"(v.w[6]), "=r"(v.w[7])
               : "l"(p) : "memory");
  return v;
}

__device__ __forceinline__ void store32(void* p, const Vec32& v) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(v.w[0]), "r"(v.w[1]), "r"(v.w[2]), "r"(v.w[3]),
               "r"(v.w[4]), "r"(v.w[5]), "r"(v.w[6]), "r"(v.w[7]) : "memory");
}

__device__ __forceinline__ uint4 load16(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ void store16(void* p, uint4 v) {
  asm volatile("st.global.v4.b32 [%0], {%1,%2,%3,%4};" ::"l"(p), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void store8(void* p, uint2 v) {
  asm volatile("st.global.v2.b32 [%0], {%1,%2};" ::"l"(p), "r"(v.x), "r"(v.y) : "memory");
}

template <typename T> constexpr int kVecN = 32 / (int)sizeof(T);

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }

template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }

// Two fp32 values in one 64-bit register: Blackwell adds, multiplies and fuses both in one instruction.
struct F2 { float x, y; };

__device__ __forceinline__ uint64_t bits(F2 v) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(v.x), "f"(v.y));
  return r;
}
__device__ __forceinline__ F2 pair(uint64_t r) {
  F2 v;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(r));
  return v;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)));
  return pair(r);
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)));
  return pair(r);
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)), "l"(bits(c)));
  return pair(r);
}

__device__ __forceinline__ F2 unpack2(uint32_t w, __nv_bfloat16) { return {__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)}; }
__device__ __forceinline__ F2 unpack2(uint32_t w, __half) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  return {f.x, f.y};
}

// The elements of a vector as pairs of fp32.
template <typename T>
__device__ __forceinline__ void unpack(const Vec32& v, F2 (&x)[kVecN<T> / 2]) {
  #pragma unroll
  for (int i = 0; i < kVecN<T> / 2; ++i) {
    if constexpr (sizeof(T) == 4) x[i] = {__uint_as_float(v.w[2 * i]), __uint_as_float(v.w[2 * i + 1])};
    else x[i] = unpack2(v.w[i], T{});
  }
}

__device__ __forceinline__ uint32_t pack2(F2 v, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(F2 v, __half) {
  const __half2 h = __floats2half2_rn(v.x, v.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T>
__device__ __forceinline__ Vec32 pack(const F2 (&x)[kVecN<T> / 2]) {
  Vec32 v;
  #pragma unroll
  for (int i = 0; i < kVecN<T> / 2; ++i) {
    if constexpr (sizeof(T) == 4) {
      v.w[2 * i] = __float_as_uint(x[i].x);
      v.w[2 * i + 1] = __float_as_uint(x[i].y);
    } else {
      v.w[i] = pack2(x[i], T{});
    }
  }
  return v;
}

// E consecutive elements of one lane as they come from memory, in the widest vectors that they fill;
// the address is aligned to them, or to 32 bytes where they are longer.
template <typename T, int E>
struct RawVec {
  static constexpr int kWords = E * (int)sizeof(T) / 4;
  uint32_t w[kWords];

  __device__ __forceinline__ void load(const T* p) {
    if constexpr (kWords >= 8) {
      #pragma unroll
      for (int k = 0; k < kWords / 8; ++k) {
        const Vec32 v = load32(p + k * kVecN<T>);
        #pragma unroll
        for (int i = 0; i < 8; ++i) w[8 * k + i] = v.w[i];
      }
    } else {
      static_assert(kWords == 4);
      const uint4 v = load16(p);
      w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    }
  }
  __device__ __forceinline__ void pairs(F2 (&x)[E / 2]) const {
    #pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      if constexpr (sizeof(T) == 4) x[i] = {__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1])};
      else x[i] = unpack2(w[i], T{});
    }
  }
};

template <int E, typename T>
__device__ __forceinline__ void load_pairs(const T* p, F2 (&x)[E / 2]) {
  RawVec<T, E> v;
  v.load(p);
  v.pairs(x);
}

template <int E, typename T>
__device__ __forceinline__ void store_pairs(T* p, const F2 (&x)[E / 2]) {
  constexpr int kBytes = E * (int)sizeof(T);
  if constexpr (kBytes >= 32) {
    #pragma unroll
    for (int k = 0; k < kBytes / 32; ++k) {
      F2 part[kVecN<T> / 2];
      #pragma unroll
      for (int i = 0; i < kVecN<T> / 2; ++i) part[i] = x[k * (kVecN<T> / 2) + i];
      store32(p + k * kVecN<T>, pack<T>(part));
    }
  } else {
    static_assert(kBytes == 16);
    if constexpr (sizeof(T) == 4) {
      store16(p, make_uint4(__float_as_uint(x[0].x), __float_as_uint(x[0].y), __float_as_uint(x[1].x), __float_as_uint(x[1].y)));
    } else {
      store16(p, make_uint4(pack2(x[0], T{}), pack2(x[1], T{}), pack2(x[2], T{}), pack2(x[3], T{})));
    }
  }
}

// The same for addresses aligned to 16 bytes only.
template <int E, typename T>
__device__ __forceinline__ void store_pairs16(T* p, const F2 (&x)[E / 2]) {
  constexpr int N = 16 / (int)sizeof(T);
  #pragma unroll
  for (int k = 0; k < E / N; ++k) {
    F2 part[N / 2];
    #pragma unroll
    for (int i = 0; i < N / 2; ++i) part[i] = x[k * (N / 2) + i];
    store_pairs<N>(p + k * N, part);
  }
}

// 2^x by the hardware's approximation (relative error 2^-22; results below 2^-126 become 0).
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ float warp_max(float v) {
  #pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kFullWarp, v, o));
  return v;
}

template <typename T>
__device__ __forceinline__ T warp_sum(T v) {
  #pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFullWarp, v, o);
  return v;
}

}  // namespace wb
