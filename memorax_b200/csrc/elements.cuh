// Element types of the kernels that take bf16, fp16 and fp32 alike: conversions to float, and accesses of N neighbours at once.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "mxk_common.cuh"

namespace mxk {

inline bool known_type(int type) { return type == MXK_F32 || type == MXK_BF16 || type == MXK_F16; }
inline int type_bytes(int type) { return type == MXK_F32 ? 4 : 2; }

__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float as_float(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }

// Two of 16 bits in a word: one instruction each for an element on the way in, one for both on the way out.
__device__ __forceinline__ void unpack2(uint32_t w, __nv_bfloat16, float* x) {
  x[0] = __uint_as_float(w << 16);
  x[1] = __uint_as_float(w & 0xffff0000u);
}
__device__ __forceinline__ void unpack2(uint32_t w, __half, float* x) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  x[0] = f.x;
  x[1] = f.y;
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&p);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
  const __half2 p = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&p);
}

template <int kBytes> struct Raw;
template <> struct Raw<16> { using type = uint4; };
template <> struct Raw<8> { using type = uint2; };
template <> struct Raw<4> { using type = uint32_t; };
template <> struct Raw<2> { using type = uint16_t; };
template <> struct Raw<1> { using type = uint8_t; };

// N neighbours that one access moves: N * sizeof(T) bytes, aligned to as many.
template <typename T, int N>
struct Vec {
  using raw = typename Raw<N * sizeof(T)>::type;
  raw bits;
  __device__ __forceinline__ static Vec load(const T* p) { return {*reinterpret_cast<const raw*>(p)}; }
  __device__ __forceinline__ static Vec load_stream(const T* p) { return {__ldcs(reinterpret_cast<const raw*>(p))}; }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<raw*>(p) = bits; }
  __device__ __forceinline__ void store_stream(T* p) const { __stcs(reinterpret_cast<raw*>(p), bits); }
  __device__ __forceinline__ void unpack(float* x) const {
    if constexpr (sizeof(T) == 2 && N > 1) {
      const uint32_t* w = reinterpret_cast<const uint32_t*>(&bits);
#pragma unroll
      for (int i = 0; i < N / 2; ++i) unpack2(w[i], T(), x + 2 * i);
    } else {
      const T* e = reinterpret_cast<const T*>(&bits);
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = as_float(e[i]);
    }
  }
  __device__ __forceinline__ static Vec pack(const float* x) {
    Vec v;
    if constexpr (sizeof(T) == 2 && N > 1) {
      uint32_t* w = reinterpret_cast<uint32_t*>(&v.bits);
#pragma unroll
      for (int i = 0; i < N / 2; ++i) w[i] = pack2(x[2 * i], x[2 * i + 1], T());
    } else {
      T* e = reinterpret_cast<T*>(&v.bits);
#pragma unroll
      for (int i = 0; i < N; ++i) e[i] = from_float<T>(x[i]);
    }
    return v;
  }
};

// Widest access (bytes, at most 16 and at least an element) that addresses and strides of these low bits allow.
inline int access_bytes(uintptr_t bits) { return bits % 16 == 0 ? 16 : bits % 8 == 0 ? 8 : bits % 4 == 0 ? 4 : 2; }
inline uintptr_t address(const void* p) { return reinterpret_cast<uintptr_t>(p); }

}  // namespace mxk
