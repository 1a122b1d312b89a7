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
// scale) joins d where the group sums are added in f32. (Codes as subnormals
// as they lie in the word, the 8 taken off the sum, save the subtractions but
// lose seven bits: the tensor cores align products by the operands'
// exponents.) Limited by instructions, about 190 a warp for 2048 weights:
// 151936 x 2048 and three f32 rows 45 us (3.9 TB/s; issue slots 69 % busy),
// 12288 x 2048 and one row 12.4 us (10.4 with the weights in L2), of which the
// launch and the rows' operand are most. More than 16 rows read the weights
// again for every 16: 512 f32 rows of 12288 x 2048 take 380 us, 68 TFLOP/s.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "device.cuh"
#include "kernels.h"

namespace trit {
namespace {

constexpr int kQ4Warps = 8;
constexpr int kQ4Threads = kQ4Warps * 32;
constexpr int kQ4Chunk = 128;
// A warp's ring of chunks (16 rows x 128 values: 1 KB of codes, 128 bytes of
// scales), all but one of them on the way.
constexpr int kQ4Stages = 8, kQ4Stage = 1024 + 128;
constexpr int kQ4Ring = kQ4Warps * kQ4Stages * kQ4Stage;

// D = A B and D += A B.
__device__ __forceinline__ void q4_mma0(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void q4_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// (w & mask) | one, one instruction while `one` is in a register (the compiler
// would make two of two immediates).
template <uint32_t MASK>
__device__ __forceinline__ uint32_t q4_pick(uint32_t w, uint32_t one) {
  uint32_t x;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(x) : "r"(w), "n"(MASK), "r"(one));
  return x;
}
// Codes of the low halves of bytes 0 and 2 (shift w right by 8 for bytes 1
// and 3) as f16 c - 8: 0x6400 | c is 1024 + c. `one`: 0x64006400.
__device__ __forceinline__ uint32_t q4_low(uint32_t w, uint32_t one) {
  const uint32_t x = q4_pick<0x000F000Fu>(w, one);
  const __half2 b = __halves2half2(__ushort_as_half(0x6408), __ushort_as_half(0x6408));
  const __half2 h = __hsub2(*(const __half2*)&x, b);
  return *(const uint32_t*)&h;
}
// The high halves: 0x6400 | 16 c is 1024 + 16 c; / 16 - 72 is c - 8, exactly.
__device__ __forceinline__ uint32_t q4_high(uint32_t w, uint32_t one) {
  const uint32_t x = q4_pick<0x00F000F0u>(w, one);
  const __half2 a = __halves2half2(__ushort_as_half(0x2C00), __ushort_as_half(0x2C00));
  const __half2 b = __halves2half2(__ushort_as_half(0xD480), __ushort_as_half(0xD480));
  const __half2 h = __hfma2(*(const __half2*)&x, a, b);
  return *(const uint32_t*)&h;
}

// One pass: up to 4 * NT rows of x. A block stages the rows' operand in
// shared memory ([group][n-tile][lane] 16 bytes: both steps of 16) while its
// first weights are on the way. `split` warps share a tile of 16 matrix rows,
// each taking every split-th chunk of 128 values; their sums meet in shared
// memory. Weights come by asynchronous copies into each warp's own ring.
template <int NT>
__global__ void __launch_bounds__(kQ4Threads, 2) k_q4(const __grid_constant__ DQ4 W, const float* x, int m, int quantize,
                                                      int k0, int k1, int vec, int split, float* y, int add) {
  extern __shared__ __align__(16) uint8_t q4_smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, j = lane & 3;
  const int row0 = blockIdx.y * 4 * NT, rows = min(4 * NT, m - row0);
  const int c0 = k0 / kQ4Chunk, c1 = (k1 + kQ4Chunk - 1) / kQ4Chunk, nc = c1 - c0;  // this segment's chunks
  uint4* xf = (uint4*)(q4_smem + kQ4Ring);
  float* factors = (float*)(xf + (size_t)nc * 4 * NT * 32);  // [group][4 * NT]
  __shared__ float s_sum[2][kQ4Warps][NT][64];

  const int part = warp % split, team = warp / split;
  const int teams = gridDim.x * (kQ4Warps / split), first = blockIdx.x * (kQ4Warps / split) + team;
  const int tiles = (W.n + 15) / 16, mine = tiles > first ? (tiles - 1 - first) / teams + 1 : 0;
  const int per = part < nc ? (nc - 1 - part) / split + 1 : 0, total = per * mine;
  uint8_t* ring = q4_smem + warp * (kQ4Stages * kQ4Stage);
  const uint32_t ring32 = (uint32_t)__cvta_generic_to_shared(ring);
  // The next chunk to fetch: its bytes, its place in the ring.
  const uint8_t* codes = (const uint8_t*)W.codes + ((size_t)first * W.chunks + c0 + part) * 1024 + lane * 16;
  const uint8_t* scales = (const uint8_t*)W.scales + ((size_t)first * W.chunks + c0 + part) * 128 + lane * 4;
  const size_t turn = (size_t)teams * W.chunks - (size_t)per * split;  // chunks to the next tile's first
  int left = total, fc = per, slot_in = 0;
  auto fetch = [&]() {
    if (left > 0) {
      const uint32_t to = ring32 + slot_in;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + lane * 16), "l"(codes) : "memory");
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + 512 + lane * 16), "l"(codes + 512) : "memory");
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to + 1024 + lane * 4), "l"(scales) : "memory");
      codes += (size_t)split * 1024;
      scales += (size_t)split * 128;
      if (--fc == 0) {
        fc = per;
        codes += turn * 1024;
        scales += turn * 128;
      }
      --left;
      slot_in = slot_in == (kQ4Stages - 1) * kQ4Stage ? 0 : slot_in + kQ4Stage;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < kQ4Stages - 1; ++i) fetch();

  // The rows' operand: a thread takes 8 values of a group, four threads the
  // group. Value i = 16 step + 4 jj + z of a group is half z / 2 of word
  // (step, z % 2) of lanes (columns 2 (q % 4) and 2 (q % 4) + 1, jj).
  const int units = nc * 16;  // of 8 values, a row
  for (int u0 = 0; u0 < 4 * NT * units; u0 += kQ4Threads) {
    const int u = u0 + threadIdx.x;  // row-major; units is a multiple of 16, so a group's threads stay together
    const int q = u / units, at = u % units, b = at >> 2, from = k0 + at * 8;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    if (q < rows && from < k1) {  // k1 is k or whole chunks: whole groups of 32
      const float* src = x + (size_t)(row0 + q) * W.k + from;
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
    float factor;
    __half hi[8], lo[8];
    if (quantize) {
      const float scale = group_scale(top), inv = __fdiv_rn(1.0f, scale);
      factor = round_f16(scale);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        // NaN stays NaN; a zero is code 0 although `inv` may be infinite (a
        // largest value below 3.8e-37).
        hi[i] = __float2half_rn(v[i] == v[i] ? (float)quantize_value(v[i], inv) : v[i]);
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
    if (q >= 4 * NT) continue;
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

  uint32_t one;
  asm volatile("mov.b32 %0, 0x64006400;" : "=r"(one));
  int slot = 0;
  for (int t = 0; t < mine; ++t) {
    const int tile = first + t * teams;
    // Rows r and r + 8 of the tile, columns 2 j and 2 j + 1 (a row's values
    // and remainders).
    float acc[NT][4];
#pragma unroll
    for (int a = 0; a < NT; ++a) acc[a][0] = acc[a][1] = acc[a][2] = acc[a][3] = 0.0f;
    const uint4* xg = xf + (size_t)part * 4 * NT * 32 + lane;
    const float* fg = factors + part * 16 * NT + j;
    for (int c = 0; c < per; ++c) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kQ4Stages - 2) : "memory");
      __syncwarp();  // the scales are other lanes' copies; the slot before is free
      fetch();
      const uint8_t* in = ring + slot;
      slot = slot == (kQ4Stages - 1) * kQ4Stage ? 0 : slot + kQ4Stage;
      const uint4 wa = *(const uint4*)(in + lane * 16), wb = *(const uint4*)(in + 512 + lane * 16);
      const uint2 sa = *(const uint2*)(in + 1024 + r * 8), sb = *(const uint2*)(in + 1024 + r * 8 + 64);
      const uint32_t ra[4] = {wa.x, wa.y, wa.z, wa.w}, rb[4] = {wb.x, wb.y, wb.z, wb.w};
      const float2 s0 = __half22float2(*(const __half2*)&sa.x), s1 = __half22float2(*(const __half2*)&sa.y);
      const float2 s2 = __half22float2(*(const __half2*)&sb.x), s3 = __half22float2(*(const __half2*)&sb.y);
      const float fa[4] = {s0.x, s0.y, s1.x, s1.y}, fb[4] = {s2.x, s2.y, s3.x, s3.y};
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const uint32_t ha = ra[b] >> 8, hb = rb[b] >> 8;
        const uint32_t a0[4] = {q4_low(ra[b], one), q4_low(rb[b], one), q4_low(ha, one), q4_low(hb, one)};
        const uint32_t a1[4] = {q4_high(ra[b], one), q4_high(rb[b], one), q4_high(ha, one), q4_high(hb, one)};
#pragma unroll
        for (int a = 0; a < NT; ++a) {
          const uint4 f = xg[(b * NT + a) * 32];
          const float factor = fg[b * 4 * NT + 4 * a];
          float d[4];
          q4_mma0(d, a0[0], a0[1], a0[2], a0[3], f.x, f.y);
          q4_mma(d, a1[0], a1[1], a1[2], a1[3], f.z, f.w);
          const float da = fa[b] * factor, db = fb[b] * factor;
          acc[a][0] = fmaf(da, d[0], acc[a][0]);
          acc[a][1] = fmaf(da, d[1], acc[a][1]);
          acc[a][2] = fmaf(db, d[2], acc[a][2]);
          acc[a][3] = fmaf(db, d[3], acc[a][3]);
        }
      }
      xg += (size_t)split * 4 * NT * 32;
      fg += split * 16 * NT;
    }
    auto put = [&](int q, int at, float v) {
      if (q < rows && at < W.n) {
        float* out = y + (size_t)(row0 + q) * W.n + at;
        *out = add ? *out + v : v;
      }
    };
    if (split == 1) {
#pragma unroll
      for (int a = 0; a < NT; ++a) {
        put(4 * a + j, tile * 16 + r, acc[a][0] + acc[a][1]);
        put(4 * a + j, tile * 16 + r + 8, acc[a][2] + acc[a][3]);
      }
      continue;
    }
    float (*sum)[NT][64] = s_sum[t & 1];
#pragma unroll
    for (int a = 0; a < NT; ++a) {
      sum[warp][a][r * 4 + j] = acc[a][0] + acc[a][1];
      sum[warp][a][(r + 8) * 4 + j] = acc[a][2] + acc[a][3];
    }
    // The team's barrier (every warp of it has the same tiles).
    asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "r"(split * 32) : "memory");
    for (int o = part * 32 + lane; o < NT * 64; o += split * 32) {
      const int a = o / 64;
      float v = 0.0f;
      for (int z = 0; z < split; ++z) v += sum[team * split + z][a][o % 64];
      put(a * 4 + o % 4, tile * 16 + o % 64 / 4, v);
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
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

// Values of k that a launch stages in what its ring and joins leave of shared
// memory; longer rows take several, which add up in y.
constexpr int kQ4Segment[5] = {0, 8192, 4096, 0, 2048};  // by NT

template <int NT>
cudaError_t pass(const DQ4& W, const float* x, int m, bool quantize, float* y, cudaStream_t s) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  static DeviceOnce once;
  e = once.run(dev, [] {
    return cudaFuncSetAttribute(k_q4<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                227 * 1024 - (int)sizeof(float) * 2 * kQ4Warps * NT * 64);
  });
  if (e != cudaSuccess) return e;
  constexpr int segment = kQ4Segment[NT];
  const int tiles = (W.n + 15) / 16, passes = (m + 4 * NT - 1) / (4 * NT);
  const int vec = ((uintptr_t)x & 15) == 0;  // rows are multiples of 32 values
  for (int p0 = 0; p0 < passes; p0 += 65535) {
    const int np = std::min(passes - p0, 65535);
    for (int k0 = 0; k0 < W.k; k0 += segment) {
      const int k1 = std::min(W.k, k0 + segment);
      const int nc = (k1 - k0 + kQ4Chunk - 1) / kQ4Chunk;
      const size_t smem = kQ4Ring + (size_t)nc * 4 * NT * (512 + 16);
      const size_t fixed = sizeof(float) * 2 * kQ4Warps * NT * 64 + 1024;
      const int blocks = current_sm_count() * (2 * (smem + fixed) <= 227 * 1024 ? 2 : 1);
      // Warps a tile: the least for the busiest warp, a join counted as two
      // chunks (151936 x 2048: eight warps a tile 56 us, one 47).
      int split = 1;
      long best = -1;
      for (int z = 1; z <= kQ4Warps; z *= 2) {
        const long teams = (long)blocks * (kQ4Warps / z);
        const long longest = ((tiles + teams - 1) / teams) * ((nc + z - 1) / z + (z > 1 ? 2 : 0));
        if (best < 0 || longest < best) {
          best = longest;
          split = z;
        }
      }
      const int per_block = kQ4Warps / split, grid = std::min((tiles + per_block - 1) / per_block, blocks);
      k_q4<NT><<<dim3(grid, np), kQ4Threads, smem, s>>>(W, x + (size_t)p0 * 4 * NT * W.k, m - p0 * 4 * NT, quantize ? 1 : 0,
                                                       k0, k1, vec, split, y + (size_t)p0 * 4 * NT * W.n, k0 > 0 ? 1 : 0);
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
