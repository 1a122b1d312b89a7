// Device helpers of the 8-bit key/value cache (kv8.h): addresses, types, codes
// and the softmax's constants.
#pragma once

#include <cuda_bf16.h>

#include "kv8.h"

namespace trit {
namespace {

constexpr float kF16Max = 65504.0f;
// "No key yet": finite, so that differences are no NaN, and below every score
// (the lowest f32).
constexpr float kMInit = -3.4028234663852886e38f;

__host__ __device__ __forceinline__ size_t kv_block(const KvView& kv, int page_or_seq, int layer, int which, int head) {
  return (((size_t)page_or_seq * kv.layers + layer) * 2 + which) * kv.kv_heads + head;
}

__device__ __forceinline__ float kv_load(const void* p, size_t i, int type) {
  if (type == kKvF32) return ((const float*)p)[i];
  if (type == kKvF16) return __half2float(((const __half*)p)[i]);
  return __bfloat162float(((const __nv_bfloat16*)p)[i]);
}
__device__ __forceinline__ void kv_store(void* p, size_t i, int type, float v) {
  if (type == kKvF32) ((float*)p)[i] = v;
  else if (type == kKvF16) ((__half*)p)[i] = __float2half_rn(v);
  else ((__nv_bfloat16*)p)[i] = __float2bfloat16_rn(v);
}
__device__ __forceinline__ __half to_cache_f16(float v) {
  if (v != v) v = 0.0f;
  return __float2half_rn(fminf(fmaxf(v, -kF16Max), kF16Max));
}

// 8 values at p (any alignment of the type; `vec`: 16-byte aligned).
__device__ __forceinline__ void kv_load8(const void* p, size_t i, int type, bool vec, float (&v)[8]) {
  if (!vec) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = kv_load(p, i + j, type);
  } else if (type == kKvF32) {
    const float4 a = *(const float4*)((const float*)p + i), b = *(const float4*)((const float*)p + i + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    const uint4 a = *(const uint4*)((const __half*)p + i);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (type == kKvF16) {
        const float2 f = __half22float2(*(const __half2*)&w[j]);
        v[2 * j] = f.x;
        v[2 * j + 1] = f.y;
      } else {
        v[2 * j] = __uint_as_float(w[j] << 16);
        v[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
      }
    }
  }
}
__device__ __forceinline__ void kv_load4(const void* p, size_t i, int type, bool vec, float (&v)[4]) {
  if (!vec) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = kv_load(p, i + j, type);
  } else if (type == kKvF32) {
    const float4 a = *(const float4*)((const float*)p + i);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  } else {
    const uint2 a = *(const uint2*)((const __half*)p + i);
    const uint32_t w[2] = {a.x, a.y};
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (type == kKvF16) {
        const float2 f = __half22float2(*(const __half2*)&w[j]);
        v[2 * j] = f.x;
        v[2 * j + 1] = f.y;
      } else {
        v[2 * j] = __uint_as_float(w[j] << 16);
        v[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
      }
    }
  }
}
__device__ __forceinline__ void kv_store4(void* p, size_t i, int type, bool vec, const float (&v)[4]) {
  if (!vec) {
#pragma unroll
    for (int j = 0; j < 4; ++j) kv_store(p, i + j, type, v[j]);
  } else if (type == kKvF32) {
    *(float4*)((float*)p + i) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    uint32_t w[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (type == kKvF16) {
        const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
        w[j] = *(const uint32_t*)&h;
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
        w[j] = *(const uint32_t*)&h;
      }
    }
    *(uint2*)((__half*)p + i) = make_uint2(w[0], w[1]);
  }
}
__device__ __forceinline__ void kv_store8(void* p, size_t i, int type, bool vec, const float (&v)[8]) {
  if (!vec) {
#pragma unroll
    for (int j = 0; j < 8; ++j) kv_store(p, i + j, type, v[j]);
  } else if (type == kKvF32) {
    *(float4*)((float*)p + i) = make_float4(v[0], v[1], v[2], v[3]);
    *(float4*)((float*)p + i + 4) = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (type == kKvF16) {
        const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
        w[j] = *(const uint32_t*)&h;
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
        w[j] = *(const uint32_t*)&h;
      }
    }
    *(uint4*)((__half*)p + i) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}
__device__ __forceinline__ void halves8(uint4 h, float (&v)[8]) {
  const uint32_t w[4] = {h.x, h.y, h.z, h.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = __half22float2(*(const __half2*)&w[j]);
    v[2 * j] = f.x;
    v[2 * j + 1] = f.y;
  }
}

constexpr float kRaise = 14.0f, kBelow = 7.0f;
// Positions whose values f32 rows sum up on the tensor cores in one go: their
// sums are cut short, not rounded, and lose up to 2^-24 of themselves with
// every product, 2^-25 on average (60000 positions in one chain of k_kv_attend: 1.4e-5).
constexpr int kKvChain = 256;
constexpr float kZeroScaleLog2 = -31.0f;  // below every f16 page's scale (6e-8 / 127)

// Two codes (bytes 0, 1 or 2, 3 of w, each code + 128) as exact f16.
__device__ __forceinline__ uint32_t codes_lo(uint32_t w) {
  const uint32_t x = __byte_perm(w, 0x64646464u, 0x4140);
  const __half2 h = __hsub2(*(const __half2*)&x, __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480)));
  return *(const uint32_t*)&h;
}
__device__ __forceinline__ uint32_t codes_hi(uint32_t w) {
  const uint32_t x = __byte_perm(w, 0x64646464u, 0x4342);
  const __half2 h = __hsub2(*(const __half2*)&x, __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480)));
  return *(const uint32_t*)&h;
}
// 2^x to 2 units in the last place (0 below 2^-126).
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *(const uint32_t*)&h;
}

// The run and its place among the blocks of a kv head.
__device__ __forceinline__ void find_run(const KvRuns& runs, int block, int chunks, int splits, KvRun& run, int& chunk,
                                         int& split) {
  if (runs.row_seq) {
    const int row = block / (chunks * splits);
    run.seq = runs.row_seq[row];
    run.first = runs.row_pos[row];
    run.row0 = row;
    run.count = 1;
    run.len = run.first + 1;
    run.block0 = row * chunks * splits;
    run.splits = splits;
  } else {
    int lo = 0, hi = runs.n - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (runs.run[mid].block0 <= block) lo = mid;
      else hi = mid - 1;
    }
    run = runs.run[lo];
  }
  const int at = block - run.block0;
  chunk = at / run.splits;
  split = at % run.splits;
}

// Four values of a column, joined over its shares in their order: share i's
// values at first + i * step + at, its (m, l) at first + i * step + ml.
__device__ __forceinline__ void join_shares(const float* first, size_t step, int at, int ml, int shares, float& sum,
                                            float4& v) {
  float top = kMInit;
  for (int i0 = 0; i0 < shares; i0 += 4) {
    float4 x[4];
    float2 s[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i0 + j < shares) {
        x[j] = __ldcg((const float4*)(first + (size_t)(i0 + j) * step + at));
        s[j] = __ldcg((const float2*)(first + (size_t)(i0 + j) * step + ml));
      }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i0 + j < shares) {
        const float to = fmaxf(top, s[j].x), fa = exp2_fast(top - to), fb = exp2_fast(s[j].x - to);
        sum = fmaf(sum, fa, s[j].y * fb);
        v = make_float4(fmaf(v.x, fa, x[j].x * fb), fmaf(v.y, fa, x[j].y * fb), fmaf(v.z, fa, x[j].z * fb),
                        fmaf(v.w, fa, x[j].w * fb));
        top = to;
      }
  }
}

}  // namespace
}  // namespace trit
