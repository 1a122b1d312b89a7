// RMSNorm of rows with the residual's addition in front and rows of 8 bits
// behind it:
//   h = x + residual, rounded to the rows' type (what the residual then holds)
//   s = f32(1 / sqrt(mean h^2 + eps)),  y = h * f32(s * w)
//   out = y rounded to the rows' type;  a group of 128 of y as e4m3 numbers:
//   scale = max(f32(max |y| / 448), 2^-126) (1 for zeros),
//   code = e4m3(f32(y * f32(1 / scale)))
// The sum of squares is 64 bits wide, so that s, and with it every code, does
// not depend on the order of the sum (an order's error of 1e-16 moves an f32
// s once in 1e8 rows), and rows of any size of values have an answer. The
// floor of the scale keeps 1 / scale finite. A group with a NaN or an infinity
// gets the scale NaN.
//
// Bound by bytes: a row is read once and stays in registers between the sum
// and the output. A thread holds 8 neighbouring values at a time, so 16
// threads hold a group and share its maximum with shuffles.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "rows.h"

namespace trit {
namespace {

template <class T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// 8 values at p, those from `left` on zero. VEC: p is 16-byte aligned and
// left is 8 or less than 1.
template <class T, bool VEC>
__device__ __forceinline__ void load8(const T* p, int left, float (&v)[8]) {
  if constexpr (VEC) {
    if (left <= 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.0f;
      return;
    }
    if constexpr (sizeof(T) == 4) {
      const float4 a = *(const float4*)p, b = *(const float4*)(p + 4);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
      v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
      const uint4 a = *(const uint4*)p;
      const T* h = (const T*)&a;
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = to_f32(h[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < left ? to_f32(p[i]) : 0.0f;
  }
}
template <class T, bool VEC>
__device__ __forceinline__ void store8(T* p, int left, const float (&v)[8]) {
  if constexpr (VEC) {
    if (left <= 0) return;
    if constexpr (sizeof(T) == 4) {
      *(float4*)p = make_float4(v[0], v[1], v[2], v[3]);
      *(float4*)(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      uint4 a;
      T* h = (T*)&a;
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = from_f32<T>(v[i]);
      *(uint4*)p = a;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) p[i] = from_f32<T>(v[i]);
  }
}

__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Two e4m3 numbers, the first in the low byte.
__device__ __forceinline__ uint32_t e4m3x2(float a, float b) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
  return r;
}

// The codes and the scale of 8 values whose group the 16 threads of this half
// warp hold. Every thread of the warp takes part.
template <bool VEC>
__device__ __forceinline__ void put_codes(const float (&y)[8], uint8_t* codes, float* scale_at, int left) {
  uint32_t most = 0;  // the bits of |y| are ordered as its values, infinity and NaN above all
#pragma unroll
  for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(y[i]) & 0x7fffffffu);
#pragma unroll
  for (int o = 8; o; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
  float scale = 1.0f;
  if (most >= 0x7f800000u) scale = __uint_as_float(0x7fffffffu);
  else if (most) scale = fmaxf(__fdiv_rn(__uint_as_float(most), 448.0f), 1.17549435e-38f);
  if (left <= 0) return;
  const float inv = __fdiv_rn(1.0f, scale);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = e4m3x2(__fmul_rn(y[2 * i], inv), __fmul_rn(y[2 * i + 1], inv));
  if constexpr (VEC) {
    *(uint2*)codes = make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) codes[i] = (uint8_t)(w[i / 2] >> (8 * (i & 1)));
  }
  if ((threadIdx.x & 15) == 0) *scale_at = scale;
}

template <class T, bool VEC>
__device__ __forceinline__ void finish8(const NormArgs& a, size_t row, int at, int left, const float (&y)[8]) {
  if (a.out) store8<T, VEC>((T*)a.out + row * a.out_stride + at, left, y);
  if (a.codes)
    put_codes<VEC>(y, a.codes + row * a.width + at,
                   a.scales + row * ((a.width + kFp8Group - 1) / kFp8Group) + at / kFp8Group, left);
}

// h of 8 values: x, or its sum with the residual, which is stored.
template <class T, bool VEC>
__device__ __forceinline__ void sum8(const NormArgs& a, size_t row, int at, int left, float (&h)[8], const float (&r)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) h[i] = to_f32(from_f32<T>(__fadd_rn(h[i], r[i])));
  store8<T, VEC>((T*)a.sum + row * a.sum_stride + at, left, h);
}

// The block's (TEAM threads') sum of a value a thread.
template <int TEAM>
__device__ __forceinline__ double team_sum(double v) {
  v = warp_sum_f64(v);
  if constexpr (TEAM > 32) {
    __shared__ double part[TEAM / 32];
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = warp_sum_f64((threadIdx.x & 31) < TEAM / 32 ? part[threadIdx.x & 31] : 0.0);
  }
  return v;
}
// s as f32(s 2^e) and 2^-e, e = 0 but where s or its product with h's bits
// would leave f32's exponents: rows of f32 beyond 2^100 or, without eps, below
// 2^-100.
struct Factor {
  float s = 1.0f, h = 1.0f;
};
__device__ __forceinline__ Factor norm_factor(double sum, const NormArgs& a) {
  const double s = rsqrt(sum / a.width + a.eps);
  if (s < 0x1p-100 && s > 0.0) return Factor{(float)(s * 0x1p64), 0x1p-64f};
  if (s > 0x1p100) return Factor{(float)(s * 0x1p-64), 0x1p64f};
  return Factor{(float)s, 1.0f};
}

// y from h: the norm's factor times the weights, or the rows as they are.
template <class T, bool VEC>
__device__ __forceinline__ void norm8(const NormArgs& a, int at, int left, const Factor& f, float (&v)[8]) {
  if (!a.weight) return;
  float w[8];
  if (a.weight_f32) load8<float, VEC>((const float*)a.weight + at, left, w);
  else load8<T, VEC>((const T*)a.weight + at, left, w);
  if (f.h != 1.0f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= f.h;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __fmul_rn(v[i], __fmul_rn(f.s, w[i]));
}

// A row of up to TEAM * 8 * VPT values, held in registers. A team of one warp
// shares its block with seven others.
template <class T, int TEAM, int VPT, bool VEC>
__global__ void __launch_bounds__(TEAM == 32 ? 256 : TEAM) k_norm(const __grid_constant__ NormArgs a) {
  const int t = TEAM == 32 ? threadIdx.x & 31 : threadIdx.x;
  const size_t row = TEAM == 32 ? blockIdx.x * (size_t)8 + (threadIdx.x >> 5) : blockIdx.x;
  if (row >= (size_t)a.rows) return;  // a whole warp
  float h[VPT][8];
  const T* x = (const T*)a.x + row * a.x_stride;
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const int at = (t + j * TEAM) * 8;
    load8<T, VEC>(x + at, a.width - at, h[j]);
  }
  if (a.residual) {
    const T* res = (const T*)a.residual + row * a.residual_stride;
    float r[VPT][8];
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int at = (t + j * TEAM) * 8;
      load8<T, VEC>(res + at, a.width - at, r[j]);
    }
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int at = (t + j * TEAM) * 8;
      sum8<T, VEC>(a, row, at, a.width - at, h[j], r[j]);
    }
  }
  Factor f;
  if (a.weight) {
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < VPT; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) sum = fma((double)h[j][i], (double)h[j][i], sum);
    f = norm_factor(team_sum<TEAM>(sum), a);
  }
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const int at = (t + j * TEAM) * 8, left = a.width - at;
    norm8<T, VEC>(a, at, left, f, h[j]);
    finish8<T, VEC>(a, row, at, left, h[j]);
  }
}

// Rows of any width: the second pass reads h again (the sum where there is a
// residual), each thread what it read or wrote itself.
template <class T, bool VEC>
__global__ void __launch_bounds__(1024) k_norm_long(const __grid_constant__ NormArgs a) {
  const size_t row = blockIdx.x;
  const T* x = (const T*)a.x + row * a.x_stride;
  const int all = (a.width + 8 * 1024 - 1) / (8 * 1024) * (8 * 1024);  // every thread takes every turn
  double sum = 0.0;
  for (int at = threadIdx.x * 8; at < all; at += 8 * 1024) {
    float h[8];
    load8<T, VEC>(x + at, a.width - at, h);
    if (a.residual) {
      float r[8];
      load8<T, VEC>((const T*)a.residual + row * a.residual_stride + at, a.width - at, r);
      sum8<T, VEC>(a, row, at, a.width - at, h, r);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = fma((double)h[i], (double)h[i], sum);
  }
  const Factor f = a.weight ? norm_factor(team_sum<1024>(sum), a) : Factor();
  const T* from = a.residual ? (const T*)a.sum + row * a.sum_stride : x;
  for (int at = threadIdx.x * 8; at < all; at += 8 * 1024) {
    const int left = a.width - at;
    float h[8];
    load8<T, VEC>(from + at, left, h);
    norm8<T, VEC>(a, at, left, f, h);
    finish8<T, VEC>(a, row, at, left, h);
  }
}

template <class T, int TEAM, int VPT, bool VEC>
cudaError_t run(const NormArgs& a, cudaStream_t s) {
  const int per = TEAM == 32 ? 8 : 1;
  k_norm<T, TEAM, VPT, VEC><<<(a.rows + per - 1) / per, TEAM == 32 ? 256 : TEAM, 0, s>>>(a);
  return cudaGetLastError();
}

template <class T, bool VEC>
cudaError_t dispatch(const NormArgs& a, cudaStream_t s) {
  const int w = a.width;
  if (w <= 256) return run<T, 32, 1, VEC>(a, s);
  if (w <= 1024) return run<T, 32, 4, VEC>(a, s);
  if (w <= 2048) return run<T, 256, 1, VEC>(a, s);
  if (w <= 4096) return run<T, 256, 2, VEC>(a, s);
  if (w <= 8192) return run<T, 512, 2, VEC>(a, s);
  k_norm_long<T, VEC><<<a.rows, 1024, 0, s>>>(a);
  return cudaGetLastError();
}

template <class T>
cudaError_t by_alignment(const NormArgs& a, cudaStream_t s) {
  const uintptr_t at = (uintptr_t)a.x | (uintptr_t)a.residual | (uintptr_t)a.sum | (uintptr_t)a.weight | (uintptr_t)a.out;
  const size_t strides = a.x_stride | a.residual_stride | a.sum_stride | a.out_stride | (size_t)a.width;
  const bool vec = at % 16 == 0 && strides % 8 == 0 && (uintptr_t)a.codes % 8 == 0;
  return vec ? dispatch<T, true>(a, s) : dispatch<T, false>(a, s);
}

}  // namespace

cudaError_t launch_rms_norm(const NormArgs& a, cudaStream_t s) {
  if (a.rows <= 0) return cudaSuccess;
  if (a.type == kRowF32) return by_alignment<float>(a, s);
  if (a.type == kRowF16) return by_alignment<__half>(a, s);
  return by_alignment<__nv_bfloat16>(a, s);
}

}  // namespace trit
