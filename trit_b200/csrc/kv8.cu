// Kernels of the key/value cache held in 8 bits (kv8.h): the quantizing
// write, attention over codes, reads, and page moves.
//
// Values: a key or value is rounded to f16 on arrival (infinities to the
// largest f16, NaN to 0, so nothing the cache holds can spoil a masked
// place). A page that is not full holds f16; when its last position arrives,
// each (layer, keys or values, kv head) block of the page gets one f32 scale
// max|x| / 127 and codes nearest x / scale. Codes depend on the positions'
// values alone, not on how many calls brought them.
#include "kv8.h"

#include <cuda_bf16.h>

#include <algorithm>

#include "kernels.h"

namespace trit {
namespace {

constexpr float kF16Max = 65504.0f;
constexpr float kMInit = -1e30f;  // "no key yet": finite, so that differences stay numbers

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

// The whole number nearest x / scale, ties to even, decided exactly: the
// estimate is at most one off, and fma gives the sign of x - (q +- 1/2)
// scale without rounding error (its result is the exact difference, rounded
// once). |x| <= 127 scale up to the scale's own rounding, so q <= 127.
__device__ __forceinline__ int nearest_code(float x, float scale, float inv) {
  const float t = fabsf(x);
  float q = rintf(t * inv);
  const float up = __fmaf_rn(-(q + 0.5f), scale, t), down = __fmaf_rn(-(q - 0.5f), scale, t);
  const bool odd = ((int)q & 1) != 0;
  if (up > 0.0f || (up == 0.0f && odd)) q += 1.0f;
  else if (down < 0.0f || (down == 0.0f && odd)) q -= 1.0f;
  const int c = (int)q;
  return x < 0.0f ? -c : c;
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

// Codes + 128 of 8 values, packed in order. x * inv is within 4e-5 of
// x / scale (two roundings of a number below 128), so rounding it is exact
// unless it lands within 1e-4 of a border; those go through nearest_code.
// Adding 1.5 * 2^23 rounds, and leaves the code in the low bits.
__device__ __forceinline__ uint2 codes8(const float (&v)[8], float scale, float inv) {
  uint32_t c[8];
  float far = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float y = __fmul_rn(v[j], inv), r = __fadd_rn(y, 12582912.0f + 128.0f);
    c[j] = __float_as_uint(r);
    far = fmaxf(far, fabsf(__fsub_rn(y, __fsub_rn(r, 12582912.0f + 128.0f))));
  }
  if (far > 0.4999f) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c[j] = (uint32_t)(nearest_code(v[j], scale, inv) + 128);
  }
  uint2 w;
  w.x = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
  w.y = __byte_perm(__byte_perm(c[4], c[5], 0x0040), __byte_perm(c[6], c[7], 0x0040), 0x5410);
  return w;
}

// ------------------------------------------------------------- append ----
// One block writes one page's share of a run, for one (keys or values, kv
// head). Block 0 takes the run's first page, which may begin in the open
// buffer, and then the last, partial page, which ends there: the same block,
// so that the second does not overwrite what the first still reads. The
// page's share passes through shared memory as f16, eight values a thread
// and turn, while its largest value is found.
// Bound by bytes: rows in (2 or 4 bytes a value), codes out.
constexpr int kAppendThreads = 256;

template <int HD>
__global__ void __launch_bounds__(kAppendThreads) k_kv_append(const __grid_constant__ KvView kv,
                                                              const __grid_constant__ KvRuns runs, int layer,
                                                              const void* k, size_t k_stride, const void* v,
                                                              size_t v_stride, int type, int vec, int run0) {
  constexpr int U = HD / 8;  // 8-value units of a position
  extern __shared__ __align__(16) uint4 held[];  // [page][U] f16
  __shared__ float warp_top[kAppendThreads / 32];
  const int which = blockIdx.y & 1, head = blockIdx.y >> 1, P = kv.page;
  KvRun run;
  const int ri = run0 + blockIdx.z;
  if (runs.row_seq) {
    run.seq = runs.row_seq[ri];
    run.first = runs.row_pos[ri];
    run.row0 = ri;
    run.count = 1;
  } else {
    run = runs.run[ri];
  }
  if (run.count <= 0) return;
  const int end = run.first + run.count;
  const int first_page = run.first / P, last_page = (end - 1) / P;
  const void* src = which ? v : k;
  const size_t stride = which ? v_stride : k_stride;
  __half* open = kv.open + kv_block(kv, run.seq, layer, which, head) * (size_t)(P * HD);
  int page = first_page + blockIdx.x;
  if (page > last_page) return;
  if (blockIdx.x > 0 && (page + 1) * P > end) return;  // the partial last page is block 0's
  for (;;) {
    const int a = max(run.first - page * P, 0), b = min(end - page * P, P);  // the call's positions in the page
    const bool full = b == P;
    float top = 0.0f;
    for (int i = threadIdx.x + (full ? 0 : a * U); i < b * U; i += kAppendThreads) {
      const int t = i / U, u = i % U;
      uint4 h;
      if (t < a) {
        // Of this page's earlier positions, which a full page needs.
        if (which) {
          const uint4 x = *(const uint4*)(open + ((t >> 1) * HD + 8 * u) * 2),
                      y = *(const uint4*)(open + ((t >> 1) * HD + 8 * u) * 2 + 8);
          const uint32_t sel = (t & 1) ? 0x7632 : 0x5410;
          h = make_uint4(__byte_perm(x.x, x.y, sel), __byte_perm(x.z, x.w, sel), __byte_perm(y.x, y.y, sel),
                         __byte_perm(y.z, y.w, sel));
        } else {
          h = *(const uint4*)(open + t * HD + 8 * u);
        }
      } else {
        float f[8];
        kv_load8(src, (size_t)(run.row0 + page * P + t - run.first) * stride + (size_t)head * HD + 8 * u, type, vec, f);
        __half x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = to_cache_f16(f[j]);
        h = *(const uint4*)x;
      }
      held[i] = h;
      const uint32_t w[4] = {h.x, h.y, h.z, h.w};
      __half2 m = __habs2(*(const __half2*)&w[0]);
#pragma unroll
      for (int j = 1; j < 4; ++j) m = __hmax2(m, __habs2(*(const __half2*)&w[j]));
      top = fmaxf(top, fmaxf(__low2float(m), __high2float(m)));
    }
    if (full) {
#pragma unroll
      for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      if ((threadIdx.x & 31) == 0) warp_top[threadIdx.x >> 5] = top;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kAppendThreads / 32; ++w) top = fmaxf(top, warp_top[w]);
      const float scale = __fdiv_rn(top, 127.0f), inv = scale > 0.0f ? __fdiv_rn(1.0f, scale) : 0.0f;
      const int phys = kv.table[(size_t)run.seq * kv.pages_per_seq + page];
      const size_t block = kv_block(kv, phys, layer, which, head);
      if (threadIdx.x == 0) kv.scales[block] = scale;
      uint4* out = (uint4*)(kv.codes + block * (size_t)(P * HD));
      for (int i = threadIdx.x; i < P * HD / 16; i += kAppendThreads) {
        // 16 codes: two units of a key, or one unit of two values.
        float x[8], y[8];
        if (which) {
          const int t = i / U * 2, u = i % U;
          halves8(held[t * U + u], x);
          halves8(held[(t + 1) * U + u], y);
        } else {
          halves8(held[2 * i], x);
          halves8(held[2 * i + 1], y);
        }
        const uint2 cx = codes8(x, scale, inv), cy = codes8(y, scale, inv);
        out[i] = which ? make_uint4(__byte_perm(cx.x, cy.x, 0x5140), __byte_perm(cx.x, cy.x, 0x7362),
                                    __byte_perm(cx.y, cy.y, 0x5140), __byte_perm(cx.y, cy.y, 0x7362))
                       : make_uint4(cx.x, cx.y, cy.x, cy.y);
      }
    } else if (!which) {
      // A thread's own units, straight on.
      for (int i = threadIdx.x + a * U; i < b * U; i += kAppendThreads) ((uint4*)open)[i] = held[i];
    } else {
      __syncthreads();
      // Values lie in pairs of positions; a pair that this call brings half
      // of keeps its other half.
      for (int i = threadIdx.x + (a >> 1) * U; i < ((b + 1) >> 1) * U; i += kAppendThreads) {
        const int t = i / U * 2, u = i % U;
        __half* to = open + ((t >> 1) * HD + 8 * u) * 2;
        if (t >= a && t + 1 < b) {
          const uint4 x = held[t * U + u], y = held[(t + 1) * U + u];
          ((uint4*)to)[0] = make_uint4(__byte_perm(x.x, y.x, 0x5410), __byte_perm(x.x, y.x, 0x7632),
                                       __byte_perm(x.y, y.y, 0x5410), __byte_perm(x.y, y.y, 0x7632));
          ((uint4*)to)[1] = make_uint4(__byte_perm(x.z, y.z, 0x5410), __byte_perm(x.z, y.z, 0x7632),
                                       __byte_perm(x.w, y.w, 0x5410), __byte_perm(x.w, y.w, 0x7632));
        } else {
          const int mine = t >= a ? t : t + 1;
          const __half* x = (const __half*)&held[mine * U + u];
#pragma unroll
          for (int j = 0; j < 8; ++j) to[2 * j + (mine & 1)] = x[j];
        }
      }
    }
    if (blockIdx.x > 0 || page == last_page || end % P == 0) return;
    page = last_page;
    __syncthreads();
  }
}

// ---------------------------------------------------------- attention ----
// One block of four warps takes a tile of query columns (a column is one
// query row of one head of the kv head's group), one kv head and a share of
// the positions; a warp walks its positions 16 at a time:
//   S^T = K Q^T   mma m16n8k16, M 16 positions, N 8 columns, K the head
//   O^T += V^T P^T               M 16 of the head's values, K 16 positions
// with codes loaded straight into the registers that hold an operand (16
// bytes a lane, whole 32-byte sectors), one byte permute and one subtraction
// turning two codes into two exact f16 (0x6400 | u is 1024 + u). The order of
// a product's inner index is free, so it is taken as the loads bring it.
//
// The products are exact in f16 but for Q and P. A query is scaled by a
// power of two into [1, 2) and, for f32 rows, split into two f16 columns
// (value and remainder: 22 bits); P likewise. For f16 and bf16 rows P is one
// f16 (2^-11, below the rounding of the output). Sums are f32.
//
// Softmax: p = 2^(t - M) with t = log2(e) scale q.k + log2(value scale), so
// the page's value scale rides in the exponent and the value product takes
// the bare codes; the denominator adds p / value scale. M is raised only when
// a t passes it by 14 (p stays below 2^14 in f16), which a vote of the warp
// finds; then M becomes the top less 7.
//
// Bound by the codes' bytes: 2 hd bytes a position and kv head.
constexpr int kAttendWarps = 4;
constexpr float kRaise = 14.0f, kBelow = 7.0f;
constexpr float kZeroScaleLog2 = -31.0f;  // below every f16 page's scale (6e-8 / 127)

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
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
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *(const uint32_t*)&h;
}
__device__ __forceinline__ uint4 load16(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

template <int HD, bool SPLIT, int NT>
__global__ void __launch_bounds__(kAttendWarps * 32) k_kv_attend(const __grid_constant__ KvView kv,
                                                                 const __grid_constant__ KvRuns runs,
                                                                 const __grid_constant__ KvAttendArgs a, int chunks,
                                                                 int splits, float* part) {
  constexpr int CL = NT * (SPLIT ? 4 : 8);   // columns a block
  constexpr int LT = SPLIT ? 1 : 2;          // columns a thread holds in an n-tile
  constexpr int KB = HD / 64;                // 64-wide blocks of a key
  constexpr int MT = HD / 16;                // 16-row tiles of the values
  __shared__ float s_o[kAttendWarps][CL][HD];
  __shared__ float s_m[kAttendWarps][CL], s_l[kAttendWarps][CL];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, j = lane & 3;
  const int head = blockIdx.y, g = a.heads / kv.kv_heads, P = kv.page;

  KvRun run;
  int chunk;
  if (runs.row_seq) {
    const int row = blockIdx.x / chunks;
    chunk = blockIdx.x % chunks;
    run.seq = runs.row_seq[row];
    run.first = runs.row_pos[row];
    run.row0 = row;
    run.count = 1;
    run.len = run.first + 1;
  } else {
    int lo = 0, hi = runs.n - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (runs.run[mid].tile0 <= (int)blockIdx.x) lo = mid;
      else hi = mid - 1;
    }
    run = runs.run[lo];
    chunk = blockIdx.x - run.tile0;
  }
  const int cols = run.count * g, c0 = chunk * CL;

  // The query columns' operand: thread (r, j) holds column r of every n-tile,
  // values 64 b + 16 j + 4 s + {0..3} of step (b, s).
  uint32_t qf[NT][KB][4][2];
  float factor[NT][LT];  // log2(e) scale 2^e of the thread's softmax columns
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int c = c0 + (SPLIT ? t * 4 + (r >> 1) : t * 8 + r);
    const bool live = c < cols;
    const size_t at = live ? (size_t)(run.row0 + c / g) * a.q_stride + (size_t)(head * g + c % g) * HD : 0;
    float v[KB * 16];
    float top = 0.0f;
#pragma unroll
    for (int b = 0; b < KB; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        v[b * 16 + i] = live ? kv_load(a.q, at + b * 64 + j * 16 + i, a.type) : 0.0f;
        top = fmaxf(top, fabsf(v[b * 16 + i]));
      }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    int e = 0;
    if (top > 0.0f && top <= 3.4e38f) e = max(-126, min(126, (int)((__float_as_uint(top) >> 23) & 255) - 127));
    const float down = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
    for (int b = 0; b < KB; ++b)
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        float x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[i] = v[b * 16 + 4 * s + i] * down;
          if (SPLIT && (r & 1)) x[i] -= __half2float(__float2half_rn(x[i]));
        }
        qf[t][b][s][0] = pack_f16(x[0], x[1]);
        qf[t][b][s][1] = pack_f16(x[2], x[3]);
      }
    const float f = a.scale * 1.4426950408889634f * __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
    for (int i = 0; i < LT; ++i) factor[t][i] = __shfl_sync(0xffffffffu, f, 4 * (2 * j + i));
  }
  // The positions a softmax column sees: [0, limit).
  int limit[NT][LT];
  int kend = 0;
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int i = 0; i < LT; ++i) {
      const int c = c0 + (SPLIT ? t * 4 + j : t * 8 + 2 * j + i);
      limit[t][i] = c >= cols ? 0 : a.causal ? min(run.len, run.first + c / g + 1) : run.len;
      kend = max(kend, limit[t][i]);
    }
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) kend = max(kend, __shfl_xor_sync(0xffffffffu, kend, o));

  // This warp's share, in steps of 16 positions.
  const int steps = (kend + 15) / 16, shares = splits * kAttendWarps;
  const int per = (steps + shares - 1) / shares;
  const int s0 = min(steps, ((int)blockIdx.z * kAttendWarps + warp) * per), s1 = min(steps, s0 + per);
  const int full = run.len / P * P / 16;  // steps that lie in full pages

  float o[NT][MT][4], m[NT][LT], l[NT][LT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int x = 0; x < 4; ++x) o[t][i][x] = 0.0f;
#pragma unroll
    for (int i = 0; i < LT; ++i) {
      m[t][i] = kMInit;
      l[t][i] = 0.0f;
    }
  }

  // Scores of 16 positions to P^T and the running sums. s[t]: positions
  // key0 + r and key0 + r + 8 of the thread's columns.
  auto softmax = [&](float (&s)[NT][4], int key0, float key_scale, float log2_value_scale, float inv_value_scale,
                     uint32_t (&p)[NT][2]) {
    float x[NT][LT][2];
    bool raise = false;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < LT; ++i) {
        const float f = factor[t][i] * key_scale;
        const float d0 = SPLIT ? s[t][0] + s[t][1] : s[t][i], d1 = SPLIT ? s[t][2] + s[t][3] : s[t][2 + i];
        x[t][i][0] = key0 + r < limit[t][i] ? fmaf(d0, f, log2_value_scale) : -INFINITY;
        x[t][i][1] = key0 + r + 8 < limit[t][i] ? fmaf(d1, f, log2_value_scale) : -INFINITY;
        raise |= fmaxf(x[t][i][0], x[t][i][1]) > m[t][i] + kRaise;
      }
    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < LT; ++i) {
          float top = fmaxf(x[t][i][0], x[t][i][1]);
#pragma unroll
          for (int w = 4; w < 32; w <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
          if (top > m[t][i] + kRaise) {
            const float to = top - kBelow, alpha = exp2f(m[t][i] - to);
            m[t][i] = to;
            l[t][i] *= alpha;
#pragma unroll
            for (int k = 0; k < MT; ++k) {
              if (SPLIT) {
#pragma unroll
                for (int y = 0; y < 4; ++y) o[t][k][y] *= alpha;
              } else {
                o[t][k][i] *= alpha;
                o[t][k][2 + i] *= alpha;
              }
            }
          }
        }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float e[LT][2];
#pragma unroll
      for (int i = 0; i < LT; ++i) {
        e[i][0] = exp2f(x[t][i][0] - m[t][i]);
        e[i][1] = exp2f(x[t][i][1] - m[t][i]);
        l[t][i] = fmaf(e[i][0] + e[i][1], inv_value_scale, l[t][i]);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t w;
        if (SPLIT) {
          const float hi = __half2float(__float2half_rn(e[0][h]));
          w = pack_f16(hi, e[0][h] - hi);
        } else {
          w = pack_f16(e[0][h], e[LT - 1][h]);
        }
        p[t][h] = transpose8(w);
      }
    }
  };

  const int steps_page = P / 16;
  const size_t table0 = (size_t)run.seq * kv.pages_per_seq;
  const size_t bytes = (size_t)P * HD;
  const int f1 = min(s1, full);
  if (s0 < f1) {
    // Lane i keeps the page number and scales of page base + i.
    int base = s0 / steps_page, pid = 0;
    float ksc = 0.0f, vsc = 0.0f;
    const int last = (f1 - 1) / steps_page;
    auto refill = [&]() {
      const int pg = base + lane;
      if (pg <= last) {
        pid = kv.table[table0 + pg];
        const size_t block = kv_block(kv, pid, a.layer, 0, head);
        ksc = kv.scales[block];
        vsc = kv.scales[block + kv.kv_heads];
      }
    };
    refill();
    uint4 kn[KB][2], vn[KB][2];  // the next step's codes
    float ksn, vsn;
    auto fetch = [&](int step) {
      int pg = step / steps_page - base;
      if (pg == 32) {
        base += 32;
        pg = 0;
        refill();
      }
      const int page = __shfl_sync(0xffffffffu, pid, pg);
      ksn = __shfl_sync(0xffffffffu, ksc, pg);
      vsn = __shfl_sync(0xffffffffu, vsc, pg);
      const int tok = step % steps_page * 16;
      const uint8_t* kp = kv.codes + kv_block(kv, page, a.layer, 0, head) * bytes + (size_t)(tok + r) * HD + 16 * j;
      const uint8_t* vp =
          kv.codes + kv_block(kv, page, a.layer, 1, head) * bytes + (size_t)(tok / 2 + j) * (2 * HD) + 16 * r;
#pragma unroll
      for (int b = 0; b < KB; ++b) {
        kn[b][0] = load16(kp + 64 * b);
        kn[b][1] = load16(kp + 64 * b + 8 * HD);
        vn[b][0] = load16(vp + 128 * b);
        vn[b][1] = load16(vp + 128 * b + 4 * 2 * HD);
      }
    };
    fetch(s0);
    for (int step = s0; step < f1; ++step) {
      uint4 kc[KB][2], vc[KB][2];
#pragma unroll
      for (int b = 0; b < KB; ++b)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          kc[b][h] = kn[b][h];
          vc[b][h] = vn[b][h];
        }
      const float ks = ksn, vs = vsn;
      if (step + 1 < f1) fetch(step + 1);
      float s[NT][4];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int x = 0; x < 4; ++x) s[t][x] = 0.0f;
#pragma unroll
      for (int b = 0; b < KB; ++b) {
        const uint32_t w0[4] = {kc[b][0].x, kc[b][0].y, kc[b][0].z, kc[b][0].w};
        const uint32_t w1[4] = {kc[b][1].x, kc[b][1].y, kc[b][1].z, kc[b][1].w};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint32_t a0 = codes_lo(w0[q]), a1 = codes_lo(w1[q]), a2 = codes_hi(w0[q]), a3 = codes_hi(w1[q]);
#pragma unroll
          for (int t = 0; t < NT; ++t) mma16816(s[t], a0, a1, a2, a3, qf[t][b][q][0], qf[t][b][q][1]);
        }
      }
      uint32_t p[NT][2];
      const bool some = vs > 0.0f;
      softmax(s, step * 16, ks, some ? __log2f(vs) : kZeroScaleLog2, some ? 1.0f / vs : 2147483648.0f, p);
#pragma unroll
      for (int b = 0; b < KB; ++b) {
        const uint32_t w0[4] = {vc[b][0].x, vc[b][0].y, vc[b][0].z, vc[b][0].w};
        const uint32_t w1[4] = {vc[b][1].x, vc[b][1].y, vc[b][1].z, vc[b][1].w};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint32_t a0 = codes_lo(w0[q]), a1 = codes_hi(w0[q]), a2 = codes_lo(w1[q]), a3 = codes_hi(w1[q]);
#pragma unroll
          for (int t = 0; t < NT; ++t) mma16816(o[t][4 * b + q], a0, a1, a2, a3, p[t][0], p[t][1]);
        }
      }
    }
  }
  // The open page's positions, f16.
  const __half* ko = kv.open + kv_block(kv, run.seq, a.layer, 0, head) * bytes;
  const __half* vo = kv.open + kv_block(kv, run.seq, a.layer, 1, head) * bytes;
  for (int step = max(s0, full); step < s1; ++step) {
    const int tok = (step - full) * 16;
    float s[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int x = 0; x < 4; ++x) s[t][x] = 0.0f;
#pragma unroll
    for (int b = 0; b < KB; ++b) {
      const __half* k0 = ko + (size_t)(tok + r) * HD + 64 * b + 16 * j;
      uint32_t w0[8], w1[8];
      *(uint4*)w0 = *(const uint4*)k0;
      *(uint4*)(w0 + 4) = *(const uint4*)(k0 + 8);
      *(uint4*)w1 = *(const uint4*)(k0 + 8 * HD);
      *(uint4*)(w1 + 4) = *(const uint4*)(k0 + 8 * HD + 8);
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int t = 0; t < NT; ++t)
          mma16816(s[t], w0[2 * q], w1[2 * q], w0[2 * q + 1], w1[2 * q + 1], qf[t][b][q][0], qf[t][b][q][1]);
    }
    uint32_t p[NT][2];
    softmax(s, step * 16, 1.0f, 0.0f, 1.0f, p);
#pragma unroll
    for (int b = 0; b < KB; ++b) {
      const __half* v0 = vo + (size_t)(tok / 2 + j) * (2 * HD) + 128 * b + 16 * r;
      uint32_t w0[8], w1[8];
      *(uint4*)w0 = *(const uint4*)v0;
      *(uint4*)(w0 + 4) = *(const uint4*)(v0 + 8);
      *(uint4*)w1 = *(const uint4*)(v0 + 4 * 2 * HD);
      *(uint4*)(w1 + 4) = *(const uint4*)(v0 + 4 * 2 * HD + 8);
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int t = 0; t < NT; ++t)
          mma16816(o[t][4 * b + q], w0[2 * q], w0[2 * q + 1], w1[2 * q], w1[2 * q + 1], p[t][0], p[t][1]);
    }
  }

  // The warps' sums meet in shared memory.
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int i = 0; i < LT; ++i) {
      float sum = l[t][i];
#pragma unroll
      for (int w = 4; w < 32; w <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
      const int c = SPLIT ? t * 4 + j : t * 8 + 2 * j + i;
      if (r == 0) {
        s_m[warp][c] = m[t][i];
        s_l[warp][c] = sum;
      }
#pragma unroll
      for (int k = 0; k < MT; ++k) {
        const int d = KB == 1 ? 8 * r + 2 * k : 64 * (k >> 2) + 8 * r + 2 * (k & 3);
        s_o[warp][c][d] = SPLIT ? o[t][k][0] + o[t][k][1] : o[t][k][i];
        s_o[warp][c][d + 1] = SPLIT ? o[t][k][2] + o[t][k][3] : o[t][k][2 + i];
      }
    }
  __syncthreads();
  for (int x = threadIdx.x; x < CL * HD; x += kAttendWarps * 32) {
    const int lc = x / HD, d = x % HD, c = c0 + lc;
    if (c >= cols) break;
    float top = kMInit;
#pragma unroll
    for (int w = 0; w < kAttendWarps; ++w) top = fmaxf(top, s_m[w][lc]);
    float sum = 0.0f, val = 0.0f;
#pragma unroll
    for (int w = 0; w < kAttendWarps; ++w) {
      const float f = exp2f(s_m[w][lc] - top);
      sum = fmaf(f, s_l[w][lc], sum);
      val = fmaf(f, s_o[w][lc][d], val);
    }
    if (splits == 1) {
      const size_t at = (size_t)(run.row0 + c / g) * a.out_stride + (size_t)(head * g + c % g) * HD + d;
      kv_store(a.out, at, a.type, sum == 0.0f ? 0.0f : val / sum);
    } else {
      // [tile][kv head][split][column][hd + 2]
      float* to = part + ((((size_t)blockIdx.x * gridDim.y + head) * splits + blockIdx.z) * CL + lc) * (HD + 2);
      to[d] = val;
      if (d == 0) {
        to[HD] = top;
        to[HD + 1] = sum;
      }
    }
  }
}

// Joins the splits of a (tile, kv head): one thread a value.
__global__ void __launch_bounds__(128) k_kv_join(const __grid_constant__ KvView kv, const __grid_constant__ KvRuns runs,
                                                 const __grid_constant__ KvAttendArgs a, int chunks, int splits, int CL,
                                                 const float* part) {
  const int head = blockIdx.y, g = a.heads / kv.kv_heads, hd = kv.hd;
  int row0, count, chunk;
  if (runs.row_seq) {
    row0 = blockIdx.x / chunks;
    chunk = blockIdx.x % chunks;
    count = 1;
  } else {
    int lo = 0, hi = runs.n - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (runs.run[mid].tile0 <= (int)blockIdx.x) lo = mid;
      else hi = mid - 1;
    }
    row0 = runs.run[lo].row0;
    count = runs.run[lo].count;
    chunk = blockIdx.x - runs.run[lo].tile0;
  }
  const int x = blockIdx.z * 128 + threadIdx.x, lc = x / hd, d = x % hd, c = chunk * CL + lc;
  if (lc >= CL || c >= count * g) return;
  const float* p = part + (((size_t)blockIdx.x * gridDim.y + head) * splits * CL + lc) * (hd + 2);
  const size_t step = (size_t)CL * (hd + 2);
  float top = kMInit;
  for (int s = 0; s < splits; ++s) top = fmaxf(top, p[s * step + hd]);
  float sum = 0.0f, val = 0.0f;
  for (int s = 0; s < splits; ++s) {
    const float f = exp2f(p[s * step + hd] - top);
    sum = fmaf(f, p[s * step + hd + 1], sum);
    val = fmaf(f, p[s * step + d], val);
  }
  kv_store(a.out, (size_t)(row0 + c / g) * a.out_stride + (size_t)(head * g + c % g) * hd + d, a.type,
           sum == 0.0f ? 0.0f : val / sum);
}

// ---------------------------------------------------------- read, fork ----
// The value that the cache holds at a position of a sequence.
__device__ __forceinline__ float kv_value(const KvView& kv, int seq, int len, int pos, int layer, int which, int head,
                                          int d) {
  const int P = kv.page, page = pos / P, t = pos % P;
  const int at = which ? ((t >> 1) * kv.hd + d) * 2 + (t & 1) : t * kv.hd + d;
  const size_t bytes = (size_t)P * kv.hd;
  if ((page + 1) * P > len) return __half2float(kv.open[kv_block(kv, seq, layer, which, head) * bytes + at]);
  const size_t block = kv_block(kv, kv.table[(size_t)seq * kv.pages_per_seq + page], layer, which, head);
  return __fmul_rn((float)((int)kv.codes[block * bytes + at] - 128), kv.scales[block]);
}

// A unit is 8 values of a pair of positions: the 16 codes that lie together.
template <int HD>
__global__ void __launch_bounds__(256) k_kv_read(const __grid_constant__ KvView kv, const __grid_constant__ KvRuns runs,
                                                 int layer, void* k, void* v, int type, int vec) {
  constexpr int U = HD / 8;
  const KvRun& run = runs.run[blockIdx.z];
  const int which = blockIdx.y & 1, head = blockIdx.y >> 1, P = kv.page;
  void* dst = which ? v : k;
  if (!dst) return;
  const int p0 = run.first >> 1, p1 = (run.first + run.count + 1) >> 1;  // pairs
  const size_t bytes = (size_t)P * HD;
  for (int i = blockIdx.x * 256 + threadIdx.x; i < (p1 - p0) * U; i += gridDim.x * 256) {
    const int pos = (p0 + i / U) * 2, u = i % U, page = pos / P, t = pos % P;
    float x[2][8];
    if ((page + 1) * P > run.len) {
      const __half* open = kv.open + kv_block(kv, run.seq, layer, which, head) * bytes;
      if (which) {
        const uint4* h = (const uint4*)(open + ((t >> 1) * HD + 8 * u) * 2);
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          float f[8];
          halves8(h[z], f);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            x[0][4 * z + j] = f[2 * j];
            x[1][4 * z + j] = f[2 * j + 1];
          }
        }
      } else {
        halves8(*(const uint4*)(open + t * HD + 8 * u), x[0]);
        halves8(*(const uint4*)(open + (t + 1) * HD + 8 * u), x[1]);
      }
    } else {
      const size_t block = kv_block(kv, kv.table[(size_t)run.seq * kv.pages_per_seq + page], layer, which, head);
      const uint8_t* c = kv.codes + block * bytes;
      const float scale = kv.scales[block];
      uint32_t w[2][2];
      if (which) {
        const uint4 q = *(const uint4*)(c + ((t >> 1) * HD + 8 * u) * 2);
        w[0][0] = __byte_perm(q.x, q.y, 0x6420);
        w[1][0] = __byte_perm(q.x, q.y, 0x7531);
        w[0][1] = __byte_perm(q.z, q.w, 0x6420);
        w[1][1] = __byte_perm(q.z, q.w, 0x7531);
      } else {
        const uint2 q0 = *(const uint2*)(c + t * HD + 8 * u), q1 = *(const uint2*)(c + (t + 1) * HD + 8 * u);
        w[0][0] = q0.x;
        w[0][1] = q0.y;
        w[1][0] = q1.x;
        w[1][1] = q1.y;
      }
#pragma unroll
      for (int z = 0; z < 2; ++z)
#pragma unroll
        for (int j = 0; j < 8; ++j)
          x[z][j] = __fmul_rn((float)((int)(w[z][j >> 2] >> (8 * (j & 3)) & 255u) - 128), scale);
    }
#pragma unroll
    for (int z = 0; z < 2; ++z) {
      const int row = pos + z - run.first;
      if (row >= 0 && row < run.count)
        kv_store8(dst, ((size_t)(run.row0 + row) * kv.kv_heads + head) * HD + 8 * u, type, vec, x[z]);
    }
  }
}

// Block (x, run): one (layer, keys or values, head) of the open page.
__global__ void __launch_bounds__(256) k_kv_fork(const __grid_constant__ KvView kv, const __grid_constant__ KvRuns runs,
                                                 int copy_table) {
  const KvRun& run = runs.run[blockIdx.y];
  const int child = run.seq, parent = run.first, P = kv.page, full = run.count / P, rest = run.count % P;
  if (copy_table && blockIdx.x == 0)
    for (int i = threadIdx.x; i < full; i += 256)
      kv.table[(size_t)child * kv.pages_per_seq + i] = kv.table[(size_t)parent * kv.pages_per_seq + i];
  const int head = blockIdx.x % kv.kv_heads, which = blockIdx.x / kv.kv_heads % 2, layer = blockIdx.x / kv.kv_heads / 2;
  __half* to = kv.open + kv_block(kv, child, layer, which, head) * (size_t)(P * kv.hd);
  for (int i = threadIdx.x; i < rest * kv.hd; i += 256) {
    const int t = i / kv.hd, d = i % kv.hd;
    to[which ? ((t >> 1) * kv.hd + d) * 2 + (t & 1) : t * kv.hd + d] =
        __float2half_rn(kv_value(kv, parent, run.len, full * P + t, layer, which, head, d));
  }
}

__global__ void k_kv_table(int* table, const __grid_constant__ KvEntries e) {
  for (int i = threadIdx.x; i < e.n; i += blockDim.x) table[e.index[i]] = e.page[i];
}

// ---------------------------------------------------------- page moves ----
__global__ void __launch_bounds__(256) k_kv_move(const __grid_constant__ KvView kv, const int* moves) {
  const int src = moves[2 * blockIdx.y], dst = moves[2 * blockIdx.y + 1];
  const size_t blocks = (size_t)kv.layers * 2 * kv.kv_heads, n = blocks * kv.page * kv.hd / 16;
  const uint4* a = (const uint4*)(kv.codes + (size_t)src * n * 16);
  uint4* b = (uint4*)(kv.codes + (size_t)dst * n * 16);
  // Eight loads a thread in flight; n is a multiple of 64.
  for (size_t i0 = (size_t)blockIdx.x * 2048; i0 < n; i0 += (size_t)gridDim.x * 2048) {
    uint4 x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i0 + j * 256 + threadIdx.x < n) x[j] = load16(a + i0 + j * 256 + threadIdx.x);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i0 + j * 256 + threadIdx.x < n) b[i0 + j * 256 + threadIdx.x] = x[j];
  }
  if (blockIdx.x == 0)
    for (size_t i = threadIdx.x; i < blocks; i += 256) kv.scales[dst * blocks + i] = kv.scales[src * blocks + i];
}

__global__ void k_kv_remap_init(int* remap, int pages) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i < pages) remap[i] = i;
}
__global__ void k_kv_remap_set(int* remap, const int* moves, int n) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i < n) remap[moves[2 * i]] = moves[2 * i + 1];
}
__global__ void k_kv_remap(int* table, const int* remap, size_t entries) {
  const size_t i = blockIdx.x * (size_t)blockDim.x + threadIdx.x;
  if (i < entries) table[i] = remap[table[i]];
}

template <int HD, bool SPLIT, int NT>
cudaError_t attend(const KvView& kv, const KvRuns& runs, const KvAttendArgs& a, const KvAttendPlan& p, float* ws,
                   cudaStream_t s) {
  k_kv_attend<HD, SPLIT, NT>
      <<<dim3(p.tiles, kv.kv_heads, p.splits), kAttendWarps * 32, 0, s>>>(kv, runs, a, p.chunks, p.splits, ws);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_kv_append(const KvView& kv, const KvRuns& runs, int layer, const void* k, size_t k_stride,
                             const void* v, size_t v_stride, int type, int max_count, cudaStream_t s) {
  if (runs.n <= 0 || max_count <= 0) return cudaSuccess;
  // A run of c rows touches at most (c - 2) / page + 2 pages.
  const int pages = max_count == 1 ? 1 : (max_count - 2) / kv.page + 2;
  const size_t size = type == kKvF32 ? 4 : 2;
  const int vec = ((uintptr_t)k | (uintptr_t)v | k_stride * size | v_stride * size) % 16 == 0;
  for (int r0 = 0; r0 < runs.n; r0 += 65535) {
    const dim3 grid(pages, 2 * kv.kv_heads, std::min(runs.n - r0, 65535));
    const size_t smem = (size_t)kv.page * kv.hd * 2;
    if (kv.hd == 128)
      k_kv_append<128><<<grid, kAppendThreads, smem, s>>>(kv, runs, layer, k, k_stride, v, v_stride, type, vec, r0);
    else
      k_kv_append<64><<<grid, kAppendThreads, smem, s>>>(kv, runs, layer, k, k_stride, v, v_stride, type, vec, r0);
  }
  return cudaGetLastError();
}

KvAttendPlan plan_kv_attend(const KvView& kv, KvRuns& runs, const KvAttendArgs& a) {
  KvAttendPlan p;
  const int g = a.heads / kv.kv_heads, unit = a.type == kKvF32 ? 4 : 8;
  int most = 1;
  for (int i = 0; i < runs.n && !runs.row_seq; ++i) most = std::max(most, runs.run[i].count);
  // One or two n-tiles of columns a block: two when the columns need them
  // (a block reads its positions once for all of its columns).
  p.cols = (size_t)most * g > (size_t)unit ? 2 * unit : unit;
  if (runs.row_seq) {
    p.chunks = (g + p.cols - 1) / p.cols;
    p.tiles = runs.n * p.chunks;
  } else {
    for (int i = 0; i < runs.n; ++i) {
      runs.run[i].tile0 = p.tiles;
      p.tiles += (int)(((size_t)runs.run[i].count * g + p.cols - 1) / p.cols);
    }
  }
  // Splits of the positions until the blocks fill the GPU twice over, each
  // warp keeping at least four steps of 16 positions.
  const int want = 2 * 3 * current_sm_count(), blocks = std::max(1, p.tiles * kv.kv_heads);
  const int most_splits = std::max(1, a.max_len / (16 * 4 * kAttendWarps));
  p.splits = std::max(1, std::min(std::min((want + blocks - 1) / blocks, most_splits), 1024));
  const size_t one = (size_t)p.tiles * kv.kv_heads * p.cols * (kv.hd + 2) * 4;
  if (p.splits > 1) p.splits = std::max<int>(1, (int)std::min<size_t>(p.splits, kKvWorkspace / std::max<size_t>(one, 1)));
  if (p.splits > 1) p.workspace = one * p.splits;
  return p;
}

cudaError_t launch_kv_attend(const KvView& kv, const KvRuns& runs, const KvAttendArgs& a, const KvAttendPlan& p,
                             float* ws, cudaStream_t s) {
  if (p.tiles <= 0) return cudaSuccess;
  if (p.splits > 1 && !ws) return cudaErrorInvalidValue;
  const bool two = p.cols == (a.type == kKvF32 ? 8 : 16);
  cudaError_t e;
  if (kv.hd == 128) {
    if (a.type == kKvF32) e = two ? attend<128, true, 2>(kv, runs, a, p, ws, s) : attend<128, true, 1>(kv, runs, a, p, ws, s);
    else e = two ? attend<128, false, 2>(kv, runs, a, p, ws, s) : attend<128, false, 1>(kv, runs, a, p, ws, s);
  } else {
    if (a.type == kKvF32) e = two ? attend<64, true, 2>(kv, runs, a, p, ws, s) : attend<64, true, 1>(kv, runs, a, p, ws, s);
    else e = two ? attend<64, false, 2>(kv, runs, a, p, ws, s) : attend<64, false, 1>(kv, runs, a, p, ws, s);
  }
  if (e != cudaSuccess || p.splits == 1) return e;
  k_kv_join<<<dim3(p.tiles, kv.kv_heads, (p.cols * kv.hd + 127) / 128), 128, 0, s>>>(kv, runs, a, p.chunks, p.splits,
                                                                                   p.cols, ws);
  return cudaGetLastError();
}

cudaError_t launch_kv_read(const KvView& kv, const KvRuns& runs, int layer, void* k, void* v, int type, int max_count,
                           cudaStream_t s) {
  if (runs.n <= 0 || max_count <= 0) return cudaSuccess;
  const int x = (int)std::min<size_t>((((size_t)max_count / 2 + 1) * (kv.hd / 8) + 255) / 256, 1024);
  const int vec = ((uintptr_t)k | (uintptr_t)v) % 16 == 0;
  const dim3 grid(x, 2 * kv.kv_heads, runs.n);
  if (kv.hd == 128) k_kv_read<128><<<grid, 256, 0, s>>>(kv, runs, layer, k, v, type, vec);
  else k_kv_read<64><<<grid, 256, 0, s>>>(kv, runs, layer, k, v, type, vec);
  return cudaGetLastError();
}

cudaError_t launch_kv_fork(const KvView& kv, const KvRuns& runs, bool copy_table, cudaStream_t s) {
  if (runs.n <= 0) return cudaSuccess;
  k_kv_fork<<<dim3(kv.layers * 2 * kv.kv_heads, runs.n), 256, 0, s>>>(kv, runs, copy_table ? 1 : 0);
  return cudaGetLastError();
}

cudaError_t launch_kv_table(const KvView& kv, const KvEntries& e, cudaStream_t s) {
  if (e.n <= 0) return cudaSuccess;
  k_kv_table<<<1, 256, 0, s>>>(kv.table, e);
  return cudaGetLastError();
}

cudaError_t launch_kv_move(const KvView& kv, const int* moves, int n, cudaStream_t s) {
  const size_t vec = (size_t)kv.layers * 2 * kv.kv_heads * kv.page * kv.hd / 16;
  const int x = (int)std::max<size_t>(1, std::min<size_t>((vec + 2047) / 2048, 64));
  for (int i = 0; i < n; i += 65535) k_kv_move<<<dim3(x, std::min(n - i, 65535)), 256, 0, s>>>(kv, moves + 2 * i);
  return cudaGetLastError();
}

cudaError_t launch_kv_remap(const KvView& kv, const int* moves, int n, int* remap, int pages, int sequences,
                            cudaStream_t s) {
  const size_t entries = (size_t)sequences * kv.pages_per_seq;
  k_kv_remap_init<<<(pages + 255) / 256, 256, 0, s>>>(remap, pages);
  k_kv_remap_set<<<(n + 255) / 256, 256, 0, s>>>(remap, moves, n);
  k_kv_remap<<<(unsigned)((entries + 255) / 256), 256, 0, s>>>(kv.table, remap, entries);
  return cudaGetLastError();
}

}  // namespace trit
