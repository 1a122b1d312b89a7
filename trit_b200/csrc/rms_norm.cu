// RMSNorm of rows with the residual's addition in front and rows of 8 bits
// behind it:
//   h = x + residual, rounded to the rows' type (what the residual then holds)
//   s = f32(1 / sqrt(mean h^2 + eps)),  y = h * f32(s * w)
//   out = y rounded to the rows' type;  a group of 128 of y as e4m3 numbers:
//   scale = max(f32(max |y| / 448), 2^-126) (1 for zeros),
//   code = e4m3(f32(y * f32(1 / scale)))
// The sum of squares is 64 bits wide, so that s, and with it every code, all but
// never depends on the order of the sum (an order's error of 1e-16 moves an f32
// s once in 1e8 rows; the order goes by the width and the alignment, not by the
// rows beside), and rows of any size of values have an answer. The
// floor of the scale keeps 1 / scale finite. A group with a NaN or an infinity
// gets the scale NaN.
//
// Bound by bytes: a row is read once and stays in registers between the sum
// and the output. It takes few instructions to be so: a thread holds 16 values
// of a group (two runs of 8, so that a warp's loads are whole lines), 8 threads
// share the group's maximum with shuffles, and the two quotients, the row's
// root and the products are written with what is exact and cheap.
#include <cuda_runtime.h>

#include <algorithm>

#include "device.cuh"
#include "launch.cuh"
#include "rows.cuh"
#include "rows.h"

namespace trit {
namespace {

template <class T>
__device__ __forceinline__ void unpack8(const uint32_t (&w)[4], float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 x = unpack2<T>(w[i]);
    v[2 * i] = x.x;
    v[2 * i + 1] = x.y;
  }
}
// 8 values at p (16-byte aligned), or zeros.
template <class T>
__device__ __forceinline__ void load8(const T* p, int left, float (&v)[8]) {
  if (left <= 0) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.0f;
  } else if constexpr (sizeof(T) == 4) {
    const float4 a = *(const float4*)p, b = *(const float4*)(p + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    const uint4 a = *(const uint4*)p;
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
    unpack8<T>(w, v);
  }
}
template <class T>
__device__ __forceinline__ void store8(T* p, int left, const float (&v)[8]) {
  if (left <= 0) return;
  if constexpr (sizeof(T) == 4) {
    *(float4*)p = make_float4(v[0], v[1], v[2], v[3]);
    *(float4*)(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    *(uint4*)p = make_uint4(pack2<T>(make_float2(v[0], v[1])), pack2<T>(make_float2(v[2], v[3])),
                            pack2<T>(make_float2(v[4], v[5])), pack2<T>(make_float2(v[6], v[7])));
  }
}

// The sum over TEAM threads (a power of two, up to a warp).
template <int TEAM>
__device__ __forceinline__ double lanes_sum(double v) {
#pragma unroll
  for (int o = TEAM / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// The sum of a value a thread over the team: a part of a warp, or the block.
// `turn` counts the block's sums: two in a row use different memory, so one
// barrier a sum is enough.
template <int TEAM>
__device__ __forceinline__ double team_sum(double v, int turn) {
  if constexpr (TEAM <= 32) {
    return lanes_sum<TEAM>(v);
  } else {
    __shared__ double part[2][TEAM / 32];
    v = lanes_sum<32>(v);
    if ((threadIdx.x & 31) == 0) part[turn & 1][threadIdx.x >> 5] = v;
    __syncthreads();
    return lanes_sum<TEAM / 32>(part[turn & 1][threadIdx.x & (TEAM / 32 - 1)]);
  }
}

// s as f32(s 2^e) and 2^-e, e = 0 but where s or its product with h's bits
// would leave f32's exponents: rows of f32 beyond 2^100 or, without eps, below
// 2^-100.
struct Factor {
  float s = 1.0f, h = 1.0f;
};
__device__ __forceinline__ Factor norm_factor(double sum, const NormArgs& a) {
  const double d = sum * a.inv_width + a.eps;
  if (d > 0x1p-90 && d < 0x1p90) {
    // From the f32 approximation y (off by 2^-22): with e = 1 - d y^2,
    // 1 / sqrt(d) = y (1 - e)^(-1/2) = y (1 + e / 2 + 3 e^2 / 8 + ...); the
    // next term is below 2^-63.
    const double y = (double)rsqrtf((float)d), e = fma(-d * y, y, 1.0);
    return Factor{(float)fma(y * e, fma(e, 0.375, 0.5), y), 1.0f};
  }
  const double s = rsqrt(d);
  if (s < 0x1p-100 && s > 0.0) return Factor{(float)(s * 0x1p64), 0x1p-64f};
  if (s > 0x1p100) return Factor{(float)(s * 0x1p-64), 0x1p64f};
  return Factor{(float)s, 1.0f};
}

template <class T>
__device__ __forceinline__ uint32_t add_packed(uint32_t a, uint32_t b) {
  if constexpr (__is_same(T, __half)) {
    const __half2 v = __hadd2(*(const __half2*)&a, *(const __half2*)&b);
    return *(const uint32_t*)&v;
  } else if constexpr (__is_same(T, __nv_bfloat16)) {
    const __nv_bfloat162 v = __hadd2(*(const __nv_bfloat162*)&a, *(const __nv_bfloat162*)&b);
    return *(const uint32_t*)&v;
  } else {
    return 0;  // f32 is not packed
  }
}

// The largest |v|; NaN where there is one.
__device__ __forceinline__ float max_abs(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// Two e4m3 numbers, the first in the low byte.
__device__ __forceinline__ uint32_t e4m3x2(float2 v) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(v.y), "f"(v.x));
  return r;
}

// A thread's 16 values of a group. VEC: runs of 8 from `at` and from at + 64 of
// the row, there are left0 and left1 values from each on (8 or more, or none).
// Otherwise every eighth value from `at` on, so that neighbouring threads have
// neighbouring values, and left0 values of the row from there on.
template <bool VEC>
struct Place {
  int at, left0, left1;
  __device__ __forceinline__ Place(int unit, int width)
      : at((unit >> 3) * kFp8Group + (unit & 7) * (VEC ? 8 : 1)), left0(width - at), left1(width - at - 64) {}
};
template <class T, bool VEC>
__device__ __forceinline__ void load16(const T* p, const Place<VEC>& u, float (&v)[16]) {
  if constexpr (VEC) {
    load8(p + u.at, u.left0, *(float (*)[8])v);
    load8(p + u.at + 64, u.left1, *(float (*)[8])(v + 8));
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = 8 * i < u.left0 ? to_f32(p[u.at + 8 * i]) : 0.0f;
  }
}
template <class T, bool VEC>
__device__ __forceinline__ void store16(T* p, const Place<VEC>& u, const float (&v)[16]) {
  if constexpr (VEC) {
    store8(p + u.at, u.left0, *(const float (*)[8])v);
    store8(p + u.at + 64, u.left1, *(const float (*)[8])(v + 8));
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (8 * i < u.left0) p[u.at + 8 * i] = from_f32<T>(v[i]);
  }
}
// Codes of values 2 i and 2 i + 1 in the low half of w[i].
template <bool VEC>
__device__ __forceinline__ void store_codes16(uint8_t* p, const Place<VEC>& u, const uint32_t (&w)[8]) {
  if constexpr (VEC) {
    if (u.left0 > 0) *(uint2*)(p + u.at) = make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
    if (u.left1 > 0) *(uint2*)(p + u.at + 64) = make_uint2(w[4] | w[5] << 16, w[6] | w[7] << 16);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (8 * i < u.left0) p[u.at + 8 * i] = (uint8_t)(w[i / 2] >> (8 * (i & 1)));
  }
}

// The codes and the scale of a group that 8 neighbouring threads hold. Every
// thread of the warp takes part.
template <bool VEC>
__device__ __forceinline__ void put_codes(const float (&y)[16], const Place<VEC>& u, uint8_t* codes, float* scales) {
  float most = max_abs(y[0], y[1], y[2]);
#pragma unroll
  for (int i = 3; i < 15; i += 2) most = max_abs(most, y[i], y[i + 1]);
  most = max_abs(most, y[15], 0.0f);
#pragma unroll
  for (int o = 4; o; o >>= 1) most = max_abs(most, __shfl_xor_sync(0xffffffffu, most, o), 0.0f);
  // max / 448 through 64 bits: with X the 24 bits of max, the quotient lies at
  // least 1 / 14 of an f32 step from the border between two f32 (2 X 2^s is
  // even, 7 (2 j + 1) odd), the 64-bit product within 2^-28 of a step.
  float scale = fmaxf((float)((double)most * (1.0 / 448.0)), 1.17549435e-38f);
  if (most == 0.0f) scale = 1.0f;
  if (!(most < __uint_as_float(0x7f800000u))) scale = __uint_as_float(0x7fffffffu);
  const float inv = __frcp_rn(scale);
  const float2 i2 = make_float2(inv, inv);
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = e4m3x2(mul2(make_float2(y[2 * i], y[2 * i + 1]), i2));
  store_codes16(codes, u, w);
  if ((threadIdx.x & 7) == 0 && u.left0 > 0) scales[u.at / kFp8Group] = scale;
}

template <class T, bool VEC>
__device__ __forceinline__ void weights16(const NormArgs& a, const Place<VEC>& u, float (&w)[16]) {
  if (a.weight_f32) load16((const float*)a.weight, u, w);
  else load16((const T*)a.weight, u, w);
}
// y: h times the norm's factor and the weights.
__device__ __forceinline__ void norm16(const Factor& f, const float (&w)[16], float (&v)[16]) {
  if (f.h != 1.0f) {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] *= f.h;
  }
  const float2 s2 = make_float2(f.s, f.s);
#pragma unroll
  for (int i = 0; i < 16; i += 2) {
    const float2 y = mul2(make_float2(v[i], v[i + 1]), mul2(s2, make_float2(w[i], w[i + 1])));
    v[i] = y.x;
    v[i + 1] = y.y;
  }
}

// A thread's values of x and of the residual as they lie in memory: 16-bit
// values stay packed, so that the next row's can be on their way meanwhile.
template <class T, bool VEC>
struct Loaded {
  static constexpr bool PACKED = VEC && sizeof(T) == 2;
  uint4 x[PACKED ? 2 : 1], r[PACKED ? 2 : 1];
  __device__ __forceinline__ void load(const NormArgs& a, size_t row, const Place<VEC>& u) {
    if constexpr (PACKED) {
      const T* p = (const T*)a.x + row * a.x_stride + u.at;
      const uint4 zero = make_uint4(0, 0, 0, 0);
      x[0] = u.left0 > 0 ? *(const uint4*)p : zero;
      x[1] = u.left1 > 0 ? *(const uint4*)(p + 64) : zero;
      if (a.residual) {
        const T* q = (const T*)a.residual + row * a.residual_stride + u.at;
        r[0] = u.left0 > 0 ? *(const uint4*)q : zero;
        r[1] = u.left1 > 0 ? *(const uint4*)(q + 64) : zero;
      }
    }
  }
  // h: x, or its sum with the residual, which is stored. A packed addition
  // rounds once; in f32 first the sum is either exact (up to 24 bits from the
  // larger value's first to the smaller one's last), or the smaller value lies
  // below a quarter of the larger one's last place: the same number.
  __device__ __forceinline__ void sum(const NormArgs& a, size_t row, const Place<VEC>& u, float (&h)[16]) {
    if constexpr (PACKED) {
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        uint32_t v[4] = {x[g].x, x[g].y, x[g].z, x[g].w};
        if (a.residual) {
          const uint32_t w[4] = {r[g].x, r[g].y, r[g].z, r[g].w};
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] = add_packed<T>(v[i], w[i]);
          if ((g ? u.left1 : u.left0) > 0)
            *(uint4*)((T*)a.sum + row * a.sum_stride + u.at + g * 64) = make_uint4(v[0], v[1], v[2], v[3]);
        }
        unpack8<T>(v, *(float (*)[8])(h + g * 8));
      }
    } else {
      load16((const T*)a.x + row * a.x_stride, u, h);
      if (!a.residual) return;
      float q[16];
      load16((const T*)a.residual + row * a.residual_stride, u, q);
#pragma unroll
      for (int i = 0; i < 16; ++i) h[i] = to_f32(from_f32<T>(__fadd_rn(h[i], q[i])));
      store16((T*)a.sum + row * a.sum_stride, u, h);
    }
  }
};
template <class T, bool VEC>
__device__ __forceinline__ void finish16(const NormArgs& a, size_t row, const Place<VEC>& u, const float (&y)[16]) {
  if (a.out) store16((T*)a.out + row * a.out_stride, u, y);
  if (a.codes)
    put_codes(y, u, a.codes + row * a.width, a.scales + row * ((a.width + kFp8Group - 1) / kFp8Group));
}
__device__ __forceinline__ double add_squares(const float (&h)[16], double sum) {
#pragma unroll
  for (int i = 0; i < 16; ++i) sum = fma((double)h[i], (double)h[i], sum);
  return sum;
}

// Rows of up to TEAM * 16 * U values, held in registers. Teams of a warp or
// less share a block. A team takes row after row: the weights are read once,
// and the next row is on its way while this one is worked on.
template <class T, int TEAM, int U, bool VEC>
__global__ void __launch_bounds__(TEAM <= 32 ? 256 : TEAM) k_norm(const __grid_constant__ NormArgs a) {
  constexpr int PER = TEAM <= 32 ? 256 / TEAM : 1;  // teams of a block
  let_next_start();
  after_kernel_before();
  const int t = threadIdx.x % TEAM;
  // A team behind the last row has no values, but takes part in the shuffles.
  const auto place = [&](int j, int row) { return Place<VEC>(t + j * TEAM, row < a.rows ? a.width : 0); };
  const int first = blockIdx.x * PER + (PER > 1 ? threadIdx.x / TEAM : 0), step = gridDim.x * PER;
  Loaded<T, VEC> next[U];
#pragma unroll
  for (int j = 0; j < U; ++j) next[j].load(a, first, place(j, first));
  float w[U][16];
  if (a.weight) {
#pragma unroll
    for (int j = 0; j < U; ++j) weights16<T, VEC>(a, place(j, 0), w[j]);
  }
  const int turns = (a.rows - blockIdx.x * PER + step - 1) / step;  // the block's
  for (int i = 0; i < turns; ++i) {
    const int row = first + i * step;
    float h[U][16];
#pragma unroll
    for (int j = 0; j < U; ++j) next[j].sum(a, row, place(j, row), h[j]);
    if (i + 1 < turns) {
#pragma unroll
      for (int j = 0; j < U; ++j) next[j].load(a, row + step, place(j, row + step));
    }
    if (a.weight) {
      double sum = 0.0;
#pragma unroll
      for (int j = 0; j < U; ++j) sum = add_squares(h[j], sum);
      const Factor f = norm_factor(team_sum<TEAM>(sum, i), a);
#pragma unroll
      for (int j = 0; j < U; ++j) norm16(f, w[j], h[j]);
    }
#pragma unroll
    for (int j = 0; j < U; ++j) finish16<T, VEC>(a, row, place(j, row), h[j]);
  }
}

// Rows of any width: the second pass reads h again (the sum where there is a
// residual), each thread what it read or wrote itself.
template <class T, bool VEC>
__global__ void __launch_bounds__(1024) k_norm_long(const __grid_constant__ NormArgs a) {
  let_next_start();
  after_kernel_before();
  const size_t row = blockIdx.x;
  const int turns = (a.width + 16 * 1024 - 1) / (16 * 1024);  // every thread takes every turn
  double sum = 0.0;
  for (int j = 0; j < turns; ++j) {
    const Place<VEC> u(j * 1024 + threadIdx.x, a.width);
    float h[16];
    Loaded<T, VEC> in;
    in.load(a, row, u);
    in.sum(a, row, u, h);
    sum = add_squares(h, sum);
  }
  const Factor f = a.weight ? norm_factor(team_sum<1024>(sum, 0), a) : Factor();
  const T* from = a.residual ? (const T*)a.sum + row * a.sum_stride : (const T*)a.x + row * a.x_stride;
  for (int j = 0; j < turns; ++j) {
    const Place<VEC> u(j * 1024 + threadIdx.x, a.width);
    float h[16];
    load16(from, u, h);
    if (a.weight) {
      float w[16];
      weights16<T, VEC>(a, u, w);
      norm16(f, w, h);
    }
    finish16<T, VEC>(a, row, u, h);
  }
}

template <class T, int TEAM, int U, bool VEC>
cudaError_t run(const NormArgs& a, cudaStream_t s) {
  constexpr int threads = TEAM <= 32 ? 256 : TEAM, per = threads / TEAM;
  // As many blocks as the SMs hold beside each other.
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  static DeviceOnce once;
  static int resident[kMaxDevices];
  e = once.run(dev, [dev] {
    return cudaOccupancyMaxActiveBlocksPerMultiprocessor(&resident[dev], k_norm<T, TEAM, U, VEC>, threads, 0);
  });
  if (e != cudaSuccess) return e;
  const long long most = (long long)current_sm_count() * std::max(1, resident[dev]);
  const int blocks = (int)std::min((a.rows + per - 1LL) / per, most);
  return launch_early(k_norm<T, TEAM, U, VEC>, dim3(blocks), dim3(threads), 0, s, 1, a);
}

template <class T, bool VEC>
cudaError_t dispatch(const NormArgs& a, cudaStream_t s) {
  const int w = a.width;
  if (w <= 128) return run<T, 8, 1, VEC>(a, s);
  if (w <= 512) return run<T, 32, 1, VEC>(a, s);
  if (w <= 1024) return run<T, 64, 1, VEC>(a, s);
  if (w <= 2048) return run<T, 128, 1, VEC>(a, s);
  if (w <= 4096) return run<T, 256, 1, VEC>(a, s);
  if (w <= 8192) return run<T, 512, 1, VEC>(a, s);
  if (w <= 16384) return run<T, 1024, 1, VEC>(a, s);
  return launch_early(k_norm_long<T, VEC>, dim3(a.rows), dim3(1024), 0, s, 1, a);
}

template <class T>
cudaError_t by_alignment(const NormArgs& a, cudaStream_t s) {
  const uintptr_t at = (uintptr_t)a.x | (uintptr_t)a.residual | (uintptr_t)a.sum | (uintptr_t)a.weight | (uintptr_t)a.out;
  const size_t strides = a.x_stride | a.residual_stride | a.sum_stride | a.out_stride | (size_t)a.width;
  const bool vec = at % 16 == 0 && strides % 8 == 0 && (uintptr_t)a.codes % 8 == 0;
  return vec ? dispatch<T, true>(a, s) : dispatch<T, false>(a, s);
}

}  // namespace

cudaError_t launch_rms_norm(const NormArgs& args, cudaStream_t s) {
  if (args.rows <= 0) return cudaSuccess;
  NormArgs a = args;
  a.inv_width = 1.0 / a.width;
  if (a.type == kRowF32) return by_alignment<float>(a, s);
  if (a.type == kRowF16) return by_alignment<__half>(a, s);
  return by_alignment<__nv_bfloat16>(a, s);
}

}  // namespace trit
