// Products with 4-bit weights and a scale per 32 (ggml Q4_0 blocks: an f16
// scale d and 32 codes c, the weight d (c - 8)):
//   y[m][i] = sum over groups b of d[i][b] * sum over the group (c - 8) x[m]
// for a few rows of x, the products of a greedy step. Each weight is read
// once for all rows of a pass; bound by 18 bytes a 32 weights.
//
// The group sums run on mma m16n8k16 (M 16 matrix rows, N 8 columns): a code
// becomes an exact f16 with one bitwise operation and one subtraction (or
// fused multiply-add) for two codes, and a row of x is two f16 columns: each
// group of 32 values scaled by a power of two (its largest in [1, 2)) and the
// remainders, 22 bits in all. A row rounded to 8 bits first is its codes,
// exact in one column. The group's factor (the power of two, or the codes'
// scale) joins d where the group sums, exact or in f32, are added in f32.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "device.cuh"
#include "kernels.h"

namespace trit {
namespace {

constexpr int kQ4Warps = 8;
constexpr int kQ4Threads = kQ4Warps * 32;
constexpr int kQ4Ahead = 3;  // chunks a warp has in flight
constexpr int kQ4Chunk = 128;

__device__ __forceinline__ void q4_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Codes of the low halves of bytes 0 and 2 (shift w right by 8 for bytes 1
// and 3) as f16 c - 8: 0x6400 | c is 1024 + c.
__device__ __forceinline__ uint32_t q4_low(uint32_t w) {
  const uint32_t x = (w & 0x000F000Fu) | 0x64006400u;
  const __half2 b = __halves2half2(__ushort_as_half(0x6408), __ushort_as_half(0x6408));
  const __half2 h = __hsub2(*(const __half2*)&x, b);
  return *(const uint32_t*)&h;
}
// The high halves: 0x6400 | 16 c is 1024 + 16 c; / 16 - 72 is c - 8, exactly.
__device__ __forceinline__ uint32_t q4_high(uint32_t w) {
  const uint32_t x = (w & 0x00F000F0u) | 0x64006400u;
  const __half2 a = __halves2half2(__ushort_as_half(0x2C00), __ushort_as_half(0x2C00));
  const __half2 b = __halves2half2(__ushort_as_half(0xD480), __ushort_as_half(0xD480));
  const __half2 h = __hfma2(*(const __half2*)&x, a, b);
  return *(const uint32_t*)&h;
}
__device__ __forceinline__ uint4 q4_load(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// One pass: up to 4 * NT rows of x. A block stages the rows' operand in
// shared memory ([group][n-tile][lane] 16 bytes: both steps of 16) while its
// first weights are on the way, then takes tiles of 16 matrix rows, whose
// chunks of 128 values its warps share; their sums meet in shared memory.
template <int NT>
__global__ void __launch_bounds__(kQ4Threads) k_q4(const __grid_constant__ DQ4 W, const float* x, int m, int quantize,
                                                   int k0, int k1, int vec, float* y, int add) {
  extern __shared__ __align__(16) uint8_t q4_smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, j = lane & 3;
  const int row0 = blockIdx.y * 4 * NT, rows = min(4 * NT, m - row0);
  const int c0 = k0 / kQ4Chunk, c1 = (k1 + kQ4Chunk - 1) / kQ4Chunk, nc = c1 - c0;  // this segment's chunks
  uint4* xf = (uint4*)q4_smem;
  float* factors = (float*)(xf + (size_t)nc * 4 * NT * 32);  // [group][4 * NT]
  __shared__ float s_sum[2][kQ4Warps][NT][64];

  // This warp's chunks: chunk (i % per) * warps + warp of tile i / per.
  const int tiles = (W.n + 15) / 16, mine = tiles > (int)blockIdx.x ? (tiles - 1 - blockIdx.x) / gridDim.x + 1 : 0;
  const int per = warp < nc ? (nc - 1 - warp) / kQ4Warps + 1 : 0, total = per * mine;
  const uint4* codes = (const uint4*)W.codes;
  const uint2* scales = (const uint2*)W.scales;
  uint4 w[kQ4Ahead][2];
  uint2 sc[kQ4Ahead][2];
  int ft = blockIdx.x, fc = warp;  // the next chunk to fetch
  auto fetch = [&](int slot) {
    const size_t at = (size_t)ft * W.chunks + c0 + fc;
    w[slot][0] = q4_load(codes + at * 64 + lane);
    w[slot][1] = q4_load(codes + at * 64 + 32 + lane);
    sc[slot][0] = __ldg(scales + at * 16 + r);
    sc[slot][1] = __ldg(scales + at * 16 + r + 8);
    fc += kQ4Warps;
    if (fc >= nc) {
      fc = warp;
      ft += gridDim.x;
    }
  };
#pragma unroll
  for (int i = 0; i < kQ4Ahead; ++i)
    if (i < total) fetch(i);

  // The rows' operand: a thread takes 8 values of a group, four threads the
  // group. Value i = 16 step + 4 jj + z of a group is half z / 2 of word
  // (step, z % 2) of lanes (columns 2 (q % 4) and 2 (q % 4) + 1, jj).
  const int units = nc * 16;  // of 8 values, a row
  for (int u0 = 0; u0 < 4 * NT * units; u0 += kQ4Threads) {
    const int u = u0 + threadIdx.x;  // row-major; units is a multiple of 16, so a group's threads stay together
    const int q = u / units, at = u % units, b = at >> 2, first = k0 + at * 8;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    if (q < rows && first < k1) {  // k1 is k or whole chunks: whole groups of 32
      const float* src = x + (size_t)(row0 + q) * W.k + first;
      if (vec) {
        const float4 a = *(const float4*)src, c = *(const float4*)(src + 4);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = c.x; v[5] = c.y; v[6] = c.z; v[7] = c.w;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = src[i];
      }
    }
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v[i]));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    if (q >= 4 * NT) continue;
    float factor;
    __half hi[8], lo[8];
    if (quantize) {
      const float scale = group_scale(top), inv = __fdiv_rn(1.0f, scale);
      factor = round_f16(scale);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        // A value that is no number stays none.
        const float c = v[i] * inv;
        hi[i] = __float2half_rn(c == c ? (float)quantize_value(v[i], inv) : c);
        lo[i] = __ushort_as_half(0);
      }
    } else {
      int e = 0;
      if (top > 0.0f && top <= 3.4e38f) e = max(-126, min(126, (int)((__float_as_uint(top) >> 23) & 255) - 127));
      factor = __uint_as_float((uint32_t)(127 + e) << 23);
      const float down = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float a = v[i] * down;
        hi[i] = __float2half_rn(a);
        lo[i] = __float2half_rn(a - __half2float(hi[i]));
      }
    }
    if ((at & 3) == 0) factors[b * 4 * NT + q] = factor;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      // Values 4 jj .. 4 jj + 3 of step `step`.
      const int t = (at & 3) * 2 + h, step = t >> 2, jj = t & 3;
      uint32_t* to = (uint32_t*)(xf + ((size_t)b * NT + (q >> 2)) * 32 + (2 * (q & 3)) * 4 + jj) + 2 * step;
      const __half2 a0 = __halves2half2(hi[4 * h], hi[4 * h + 2]), a1 = __halves2half2(hi[4 * h + 1], hi[4 * h + 3]);
      const __half2 b0 = __halves2half2(lo[4 * h], lo[4 * h + 2]), b1 = __halves2half2(lo[4 * h + 1], lo[4 * h + 3]);
      *(uint2*)to = make_uint2(*(const uint32_t*)&a0, *(const uint32_t*)&a1);
      *(uint2*)(to + 4 * 4) = make_uint2(*(const uint32_t*)&b0, *(const uint32_t*)&b1);
    }
  }
  __syncthreads();

  int i = 0;
  for (int t = 0; t < mine; ++t) {
    const int tile = blockIdx.x + t * gridDim.x;
    float acc[NT][2];
#pragma unroll
    for (int a = 0; a < NT; ++a) acc[a][0] = acc[a][1] = 0.0f;
    for (int c = 0; c < per; ++c, ++i) {
      const uint4 wa = w[0][0], wb = w[0][1];
      const uint2 sa = sc[0][0], sb = sc[0][1];
#pragma unroll
      for (int z = 0; z + 1 < kQ4Ahead; ++z) {
        w[z][0] = w[z + 1][0];
        w[z][1] = w[z + 1][1];
        sc[z][0] = sc[z + 1][0];
        sc[z][1] = sc[z + 1][1];
      }
      if (i + kQ4Ahead < total) fetch(kQ4Ahead - 1);
      const uint32_t ra[4] = {wa.x, wa.y, wa.z, wa.w}, rb[4] = {wb.x, wb.y, wb.z, wb.w};
      const float2 s0 = __half22float2(*(const __half2*)&sa.x), s1 = __half22float2(*(const __half2*)&sa.y);
      const float2 s2 = __half22float2(*(const __half2*)&sb.x), s3 = __half22float2(*(const __half2*)&sb.y);
      const float fa[4] = {s0.x, s0.y, s1.x, s1.y}, fb[4] = {s2.x, s2.y, s3.x, s3.y};
      const int group = (warp + c * kQ4Warps) * 4;
      const uint4* xg = xf + (size_t)group * NT * 32 + lane;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const uint32_t ha = ra[b] >> 8, hb = rb[b] >> 8;
        const uint32_t a00 = q4_low(ra[b]), a01 = q4_low(rb[b]), a02 = q4_low(ha), a03 = q4_low(hb);
        const uint32_t a10 = q4_high(ra[b]), a11 = q4_high(rb[b]), a12 = q4_high(ha), a13 = q4_high(hb);
#pragma unroll
        for (int a = 0; a < NT; ++a) {
          const uint4 f = xg[(b * NT + a) * 32];
          const float factor = factors[(group + b) * 4 * NT + 4 * a + j];
          float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
          q4_mma(d, a00, a01, a02, a03, f.x, f.y);
          q4_mma(d, a10, a11, a12, a13, f.z, f.w);
          // Columns 2 j and 2 j + 1 are one row's values and remainders.
          acc[a][0] = fmaf(fa[b] * factor, d[0] + d[1], acc[a][0]);
          acc[a][1] = fmaf(fb[b] * factor, d[2] + d[3], acc[a][1]);
        }
      }
    }
    float (*sum)[NT][64] = s_sum[t & 1];
#pragma unroll
    for (int a = 0; a < NT; ++a) {
      sum[warp][a][r * 4 + j] = acc[a][0];
      sum[warp][a][(r + 8) * 4 + j] = acc[a][1];
    }
    __syncthreads();
    for (int o = threadIdx.x; o < NT * 64; o += kQ4Threads) {
      const int a = o / 64, row = o % 64 / 4, q = a * 4 + o % 4, at = tile * 16 + row;
      float v = 0.0f;
#pragma unroll
      for (int z = 0; z < kQ4Warps; ++z) v += sum[z][a][o % 64];
      if (q < rows && at < W.n) {
        float* out = y + (size_t)(row0 + q) * W.n + at;
        *out = add ? *out + v : v;
      }
    }
  }
}

// Q4_0 blocks in file order to the tiles that k_q4 reads: codes
// [tile of 16 rows][chunk][half of the rows][lane] 16 bytes (word b: bytes
// 4 j .. 4 j + 3 of group b of the chunk), scales [tile][chunk][row][4].
// Rows and groups past the matrix are zero.
__global__ void __launch_bounds__(256) k_q4_pack(const uint8_t* blocks, DQ4 W, uint32_t* codes, __half* scales) {
  const int groups = W.k / 32, tiles = (W.n + 15) / 16;
  const size_t n = (size_t)tiles * 16 * W.chunks * 4;
  for (size_t i = blockIdx.x * (size_t)256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) {
    const int b = (int)(i % 4), row = (int)(i / 4 % 16);
    const size_t tc = i / 64;  // tile * chunks + chunk
    const int chunk = (int)(tc % W.chunks);
    const size_t at = tc / W.chunks * 16 + row;
    const int group = chunk * 4 + b;
    const bool live = at < (size_t)W.n && group < groups;
    const uint16_t* src = (const uint16_t*)(blocks + (at * groups + group) * 18);
    uint16_t h[9] = {0, 0, 0, 0, 0, 0, 0, 0, 0};
    if (live)
#pragma unroll
      for (int z = 0; z < 9; ++z) h[z] = src[z];
    scales[i] = __ushort_as_half(h[0]);
    const int half = row >> 3, r = row & 7;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      codes[((tc * 2 + half) * 32 + r * 4 + j) * 4 + b] = (uint32_t)h[1 + 2 * j] | ((uint32_t)h[2 + 2 * j] << 16);
  }
}

// The packed weights as Q8_0 ones (codes c - 8 in int8, row-major) for the
// tensor-core product of many rows.
__global__ void __launch_bounds__(256) k_q4_expand(DQ4 W, int8_t* codes, __half* scales) {
  const int groups = W.k / 32;
  const size_t n = (size_t)W.n * groups;
  for (size_t i = blockIdx.x * (size_t)256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) {
    const size_t row = i / groups;
    const int group = (int)(i % groups), half = (int)(row >> 3 & 1), r = (int)(row & 7);
    const size_t tc = row / 16 * W.chunks + group / 4;
    const uint32_t* src = (const uint32_t*)W.codes + ((tc * 2 + half) * 32 + r * 4) * 4 + group % 4;
    uint32_t lo[4], hi[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t w = src[j * 4];
      lo[j] = __vsub4(w & 0x0F0F0F0Fu, 0x08080808u);
      hi[j] = __vsub4((w >> 4) & 0x0F0F0F0Fu, 0x08080808u);
    }
    uint4* out = (uint4*)(codes + row * W.k + group * 32);
    out[0] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    out[1] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    scales[i] = ((const __half*)W.scales)[(tc * 16 + row % 16) * 4 + group % 4];
  }
}

constexpr int kQ4Segment = 8192;  // values of k a pass stages (128 KB at 4 rows)

template <int NT>
cudaError_t pass(const DQ4& W, const float* x, int m, bool quantize, float* y, cudaStream_t s) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  static DeviceOnce once;
  static int by_registers = 1;  // blocks an SM (every device is the same GPU)
  e = once.run(dev, [] {
    cudaFuncAttributes attr{};
    cudaError_t r = cudaFuncGetAttributes(&attr, k_q4<NT>);
    if (r != cudaSuccess) return r;
    by_registers = std::max(1, 65536 / (attr.numRegs * kQ4Threads));
    return cudaFuncSetAttribute(k_q4<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, 190 * 1024);
  });
  if (e != cudaSuccess) return e;
  const int segment = kQ4Segment / NT, tiles = (W.n + 15) / 16, passes = (m + 4 * NT - 1) / (4 * NT);
  const int vec = ((uintptr_t)x & 15) == 0;  // rows are multiples of 32 values
  for (int p0 = 0; p0 < passes; p0 += 65535) {
    const int np = std::min(passes - p0, 65535);
    for (int k0 = 0; k0 < W.k; k0 += segment) {
      const int k1 = std::min(W.k, k0 + segment);
      const size_t smem = (size_t)((k1 - k0 + kQ4Chunk - 1) / kQ4Chunk) * 4 * NT * (512 + 16);
      const size_t fixed = sizeof(float) * 2 * kQ4Warps * NT * 64 + 1024;
      const int per_sm = std::max<int>(1, (int)std::min<size_t>(by_registers, 227 * 1024 / (smem + fixed)));
      const int grid = std::min(tiles, per_sm * current_sm_count());
      k_q4<NT><<<dim3(grid, np), kQ4Threads, smem, s>>>(W, x + (size_t)p0 * 4 * NT * W.k, m - p0 * 4 * NT, quantize ? 1 : 0,
                                                       k0, k1, vec, y + (size_t)p0 * 4 * NT * W.n, k0 > 0 ? 1 : 0);
      e = cudaGetLastError();
      if (e != cudaSuccess) return e;
    }
  }
  return cudaSuccess;
}

}  // namespace

cudaError_t launch_q4(const DQ4& W, const float* x, int m, bool quantize, float* y, cudaStream_t s) {
  if (m <= 0) return cudaSuccess;
  if (m <= 4) return pass<1>(W, x, m, quantize, y, s);
  if (m <= 8) return pass<2>(W, x, m, quantize, y, s);
  return pass<4>(W, x, m, quantize, y, s);
}

cudaError_t launch_q4_pack(const void* blocks, const DQ4& W, void* codes, void* scales, cudaStream_t s) {
  k_q4_pack<<<148 * 8, 256, 0, s>>>((const uint8_t*)blocks, W, (uint32_t*)codes, (__half*)scales);
  return cudaGetLastError();
}

cudaError_t launch_q4_expand(const DQ4& W, int8_t* codes, void* scales, cudaStream_t s) {
  k_q4_expand<<<148 * 8, 256, 0, s>>>(W, codes, (__half*)scales);
  return cudaGetLastError();
}

}  // namespace trit
