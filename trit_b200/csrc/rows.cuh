// Values of a row's type as f32 and back: one, or the two 16-bit ones of a word.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

namespace trit {

template <class T>
__device__ __forceinline__ float to_f32(T v) {
  if constexpr (sizeof(T) == 4) return v;
  else if constexpr (__is_same(T, __half)) return __half2float(v);
  else return __bfloat162float(v);
}
template <class T>
__device__ __forceinline__ T from_f32(float v) {
  if constexpr (sizeof(T) == 4) return v;
  else if constexpr (__is_same(T, __half)) return __float2half_rn(v);
  else return __float2bfloat16_rn(v);
}
template <class T>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (__is_same(T, __half)) return __half22float2(*(const __half2*)&w);
  else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <class T>
__device__ __forceinline__ uint32_t pack2(float2 v) {
  if constexpr (__is_same(T, __half)) {
    const __half2 h = __float22half2_rn(v);
    return *(const uint32_t*)&h;
  } else {
    const __nv_bfloat162 h = __float22bfloat162_rn(v);
    return *(const uint32_t*)&h;
  }
}

}  // namespace trit
