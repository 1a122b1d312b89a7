// Kernels of the key/value cache held in 8 bits (kv8.h): the quantizing
// write, attention over codes, reads, and page moves.
//
// Values: a key or value is rounded to f16 on arrival (infinities to the
// largest f16, NaN to 0, so nothing the cache holds can spoil a masked
// place). A page that is not full holds f16; when its last position arrives,
// each (layer, keys or values, kv head) block of the page gets one f32 scale
// max|x| / 127 and codes nearest x / scale. Codes depend on the positions'
// values alone, not on how many calls brought them.
#include <algorithm>

#include "device.cuh"
#include "kernels.h"
#include "kv8.cuh"

namespace trit {
namespace {

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

// Codes + 128 of 8 values, packed in order. Adding 1.5 * 2^23 rounds x * inv
// to the nearest whole number t and leaves the code in the low bits. x * inv
// is within 127 * 2^-24 (8e-6) of x / scale, so t is the nearest code unless
// x * inv lies within 1e-5 of a border; units with a value within 2e-5 of one
// go through nearest_code.
__device__ __forceinline__ uint2 codes8(const float (&v)[8], float scale, float inv) {
  constexpr float kRound = 12582912.0f + 128.0f;
  const float2 by = make_float2(inv, inv), up = make_float2(kRound, kRound), back = make_float2(kRound, kRound);
  uint32_t c[8];
  float far = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const float2 x = make_float2(v[j], v[j + 1]), r = fma2(x, by, up), t = sub2(back, r), d = fma2(x, by, t);
    c[j] = __float_as_uint(r.x);
    c[j + 1] = __float_as_uint(r.y);
    far = fmaxf(fmaxf(far, fabsf(d.x)), fabsf(d.y));
  }
  if (far > 0.49998f) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c[j] = (uint32_t)(nearest_code(v[j], scale, inv) + 128);
  }
  uint2 w;
  w.x = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
  w.y = __byte_perm(__byte_perm(c[4], c[5], 0x0040), __byte_perm(c[6], c[7], 0x0040), 0x5410);
  return w;
}

// The largest magnitudes of 8 f16, even and odd places; NaN if one is.
__device__ __forceinline__ __half2 largest8(uint4 h) {
  const uint32_t w[4] = {h.x, h.y, h.z, h.w};
  __half2 m = __habs2(*(const __half2*)&w[0]);
#pragma unroll
  for (int j = 1; j < 4; ++j) m = __hmax2_nan(m, __habs2(*(const __half2*)&w[j]));
  return m;
}

// ------------------------------------------------------------- append ----
// One block writes one page's share of a run, for one (keys or values, kv
// head). Block 0 takes the run's first page, which may begin in the open
// buffer, and then the last, partial page, which ends there: the same block,
// so that the second does not overwrite what the first still reads. The
// page's share passes through shared memory as f16, eight values a thread
// and turn, while its largest value is found.
// Its bytes are the rows in (2 or 4 a value) and the codes out; a block waits
// for its rows, then rounds them, so few rows cost latency (64 streams, one
// row each, 9 us) and many cost instructions as well: 5 streams of 1301 bf16
// rows on 8 heads 128 wide 19 us a layer, 2.1 TB/s (256 threads a block: four
// layers and their reads 132 us, with 128 threads 137; when rounding took
// twice the instructions 147, with 512 threads 179).
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
        h = make_uint4(pack_f16(f[0], f[1]), pack_f16(f[2], f[3]), pack_f16(f[4], f[5]), pack_f16(f[6], f[7]));
        const __half2 far = largest8(h);
        if (!(__low2float(far) <= kF16Max && __high2float(far) <= kF16Max)) {  // an infinity or NaN among them
          __half x[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = to_cache_f16(f[j]);
          h = *(const uint4*)x;
        }
      }
      held[i] = h;
      const __half2 m = largest8(h);
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
// two steps an iteration. Codes come by asynchronous copies of whole lines
// into the warp's own ring in shared memory, 4 or 6 steps deep, and from
// there 16 bytes a lane; one byte permute and one subtraction turn two codes
// into two exact f16 (0x6400 | u is 1024 + u). The order of a product's inner
// index is free, so it is taken as the bytes lie.
//
// The products are exact in f16 but for Q and P. A query is scaled by a
// power of two into [1, 2) and, for f32 rows, split into two f16 columns
// (value and remainder: 22 bits); P likewise. f16 rows are f16 in one column,
// and their P has its remainder in a second operand of the same columns (one
// f16, 2^-11 of a weight, is as much as the output's own rounding: 24 streams
// of up to 1500 positions were 2.9e-4 off instead of 2.0e-4, at 20.5 us instead
// of 22.6). For bf16 rows P is one f16, an eighth of the output's rounding:
// 1.7e-3 off with either. Sums are f32.
//
// Softmax: p = 2^(t - M) with t = log2(e) scale q.k + log2(value scale), so
// the page's value scale rides in the exponent and the value product takes
// the bare codes; the denominator adds p / value scale. M is raised only when
// a t passes it by 14 (p stays below 2^14 in f16), which a vote of the warp
// finds; then M becomes the top's whole part less 7 (whole, so that a raise
// scales the sums exactly).
//
// Bound by the codes' bytes, 2 hd a position and kv head, where contexts are
// long: 32 heads on 8, 128 wide, 6 streams of 40001 to 65535 positions take
// 129 us, 5.0 TB/s. 64 streams of 601 to 1279 take 39 us (3.3 TB/s): starting
// and joining blocks and uneven lengths. One of 217 takes 7.5 us, latency.
constexpr int kAttendWarps = 4;
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
__device__ __forceinline__ uint4 load16(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

__device__ __forceinline__ void copy16(void* smem, const void* global) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(smem)), "l"(global)
               : "memory");
}

// TYPE (KvType): f32 rows split Q and P, f16 rows P.
template <int HD, int TYPE, int NT>
struct AttendShape {
  static constexpr bool SPLIT = TYPE == kKvF32;
  static constexpr int UNIT = HD * 32;  // bytes of 16 positions' codes, or of their f16 keys (or values)
  static constexpr int STAGES = HD == 128 && NT == 1 ? 4 : 6;
  static constexpr int BLOCKS = HD == 128 && NT == 2 ? 2 : 3;  // an SM (registers)
  static constexpr int STAGE_BYTES = kAttendWarps * STAGES * UNIT;
  // Sums that f32 rows put aside (see kKvChain): HD / 8 values a lane and tile.
  static constexpr int SMEM = STAGE_BYTES + (SPLIT ? kAttendWarps * NT * HD / 8 * 32 * 4 : 0);
};

template <int HD, int TYPE, int NT>
__global__ void __launch_bounds__(kAttendWarps * 32, AttendShape<HD, TYPE, NT>::BLOCKS)
    k_kv_attend(const __grid_constant__ KvView kv, const __grid_constant__ KvRuns runs,
                const __grid_constant__ KvAttendArgs a, int chunks, int splits, int vec, int vec_out, void* workspace) {
  using Shape = AttendShape<HD, TYPE, NT>;
  constexpr bool SPLIT = Shape::SPLIT;
  constexpr int PB = TYPE == kKvF16 ? 2 : 1;  // operands of P: with its remainder
  constexpr int CL = NT * (SPLIT ? 4 : 8);   // columns a block
  constexpr int LT = SPLIT ? 1 : 2;          // columns a thread holds in an n-tile
  constexpr int KB = HD / 64;                // 64-wide blocks of a key
  constexpr int MT = HD / 16;                // 16-row tiles of the values
  constexpr int STAGES = Shape::STAGES;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float s_m[kAttendWarps][CL], s_l[kAttendWarps][CL];
  __shared__ int s_last;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, j = lane & 3;
  const int head = blockIdx.y, g = a.heads / kv.kv_heads, P = kv.page;

  KvRun run;
  int chunk, split;
  find_run(runs, blockIdx.x, chunks, splits, run, chunk, split);
  const int cols = run.count * g, c0 = chunk * CL;
  // The last column sees most: positions [0, kend).
  const int last_row = (min(cols, c0 + CL) - 1) / g;
  const int kend = a.causal ? min(run.len, run.first + last_row + 1) : run.len;

  // This warp's share, in steps of 16 positions; a step of codes is one unit
  // of loads, a step of the open page two (its keys, then its values).
  const int steps = (kend + 15) / 16, shares = run.splits * kAttendWarps;
  const int per = (steps + shares - 1) / shares;
  const int s0 = min(steps, (split * kAttendWarps + warp) * per), s1 = min(steps, s0 + per);
  const int full = run.len / P * P / 16;  // steps that lie in full pages
  const int f1 = max(s0, min(s1, full)), ncode = f1 - s0, units = ncode + 2 * (s1 - f1);

  const int page_steps = kv.page_shift - 4;  // log2 of a page's steps
  const int* table = kv.table + (size_t)run.seq * kv.pages_per_seq;
  const size_t bytes = (size_t)P * HD;
  const size_t head_scale = ((size_t)a.layer * 2) * kv.kv_heads + head;  // of a page's blocks
  const uint32_t page_blocks = (uint32_t)kv.layers * 2 * kv.kv_heads, page_bytes = page_blocks * (uint32_t)bytes;
  const int last_page = ncode ? (f1 - 1) >> page_steps : 0;
  // Lane i keeps the page number of page fbase + i for the loads, and the
  // scales of page base + i (with the values' logarithm and inverse) for the
  // sums.
  int fbase = s0 >> page_steps, base = fbase, pid = 0;
  float ksc = 0.0f, vlog = kZeroScaleLog2, vinv = 2147483648.0f;
  auto scales = [&](int page) {
    const float* sc = kv.scales + (size_t)page * page_blocks + head_scale;
    const float vs = sc[kv.kv_heads];
    ksc = sc[0];
    vlog = vs > 0.0f ? __log2f(vs) : kZeroScaleLog2;
    vinv = vs > 0.0f ? __fdividef(1.0f, vs) : 2147483648.0f;
  };
  if (ncode && fbase + lane <= last_page) pid = table[fbase + lane];
  // A unit of codes is two runs of 16 HD bytes, each copied as it lies, 512
  // bytes an instruction (whole lines: copies by operand, half lines at a
  // time, reached 4.3 of 6.5 TB/s). In shared memory 16-byte chunks swap
  // places within a row so that operands are read without conflicts: chunk c
  // of key r at c ^ 4 (r % 2) (128 wide), of value pair p at c ^ 2 (p % 4).
  uint8_t* stages = smem + (size_t)warp * STAGES * Shape::UNIT;
  const uint8_t* codes_k = kv.codes + head_scale * bytes + lane * 16;
  const uint8_t* codes_v = codes_k + (size_t)kv.kv_heads * bytes;
  const int put_k = HD == 128 ? (lane >> 3) * 128 + ((lane & 7) ^ ((lane >> 3 & 1) << 2)) * 16 : lane * 16;
  const int put_v = HD * 16 + (HD == 128 ? (lane >> 4) * 256 + ((lane & 15) ^ ((lane >> 4) << 1)) * 16
                                         : (lane >> 3) * 128 + ((lane & 7) ^ ((lane >> 3) << 1)) * 16);
  const int get_k = HD == 128 ? r * 128 + (j ^ ((r & 1) << 2)) * 16 : r * 64 + j * 16;
  const int get_v = HD * 16 + j * (2 * HD) + (r ^ (j << 1)) * 16;
  // Of the open page every lane copies the bytes that it will itself take.
  int slot_in = 0, slot_out = 0, ahead = 0;  // ahead: units fetched
  auto fetch = [&]() {
    const int unit = ahead++;
    if (unit < units) {
      uint8_t* to = stages + slot_in * Shape::UNIT;
      slot_in = slot_in == STAGES - 1 ? 0 : slot_in + 1;
      if (unit < ncode) {
        const int step = s0 + unit;
        int pg = (step >> page_steps) - fbase;
        if (pg == 32) {
          fbase += 32;
          pg = 0;
          if (fbase + lane <= last_page) pid = table[fbase + lane];
        }
        const uint32_t page = (uint32_t)__shfl_sync(0xffffffffu, pid, pg);
        const size_t at = (size_t)page * page_bytes + (uint32_t)(step & ((1 << page_steps) - 1)) * (16 * HD);
        const uint8_t *kp = codes_k + at, *vp = codes_v + at;
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) copy16(to + put_k + i * 512, kp + i * 512);
#pragma unroll
        for (int i = 0; i < HD / 32; ++i)
          copy16(to + (HD == 128 ? (put_v ^ ((i & 1) << 6)) : put_v) + i * 512, vp + i * 512);
      } else {
        const int tok = (f1 - full + (unit - ncode) / 2) * 16, which = (unit - ncode) & 1;
        const __half* x = kv.open + kv_block(kv, run.seq, a.layer, which, head) * bytes;
        x += which ? (size_t)(tok / 2 + j) * (2 * HD) + 16 * r : (size_t)(tok + r) * HD + 16 * j;
        const int half = which ? 4 * 2 * HD : 8 * HD, wide = which ? 128 : 64;
        to += lane * 16;
#pragma unroll
        for (int b = 0; b < KB; ++b) {
          copy16(to + (4 * b) * 512, x + wide * b);
          copy16(to + (4 * b + 1) * 512, x + wide * b + 8);
          copy16(to + (4 * b + 2) * 512, x + wide * b + half);
          copy16(to + (4 * b + 3) * 512, x + wide * b + half + 8);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  auto next = [&]() {  // the unit that is consumed next
    const uint8_t* in = stages + slot_out * Shape::UNIT;
    slot_out = slot_out == STAGES - 1 ? 0 : slot_out + 1;
    return in;
  };
#pragma unroll
  for (int i = 0; i < STAGES - 2; ++i) fetch();
  if (ncode && fbase + lane <= last_page) scales(pid);

  // The query columns' operand: thread (r, j) holds column r of every n-tile,
  // values 64 b + 16 j + 4 s + {0..3} of step (b, s).
  uint32_t qf[NT][KB][4][2];
  float factor[NT][LT];  // log2(e) scale 2^e of the thread's softmax columns
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int c = c0 + (SPLIT ? t * 4 + (r >> 1) : t * 8 + r);
    const bool live = c < cols;
    const size_t at = live ? (size_t)(run.row0 + c / g) * a.q_stride + (size_t)(head * g + c % g) * HD : 0;
    float v[KB * 2][8];
    float top = 0.0f;
#pragma unroll
    for (int b = 0; b < KB * 2; ++b) {
      if (live) {
        kv_load8(a.q, at + (b >> 1) * 64 + j * 16 + (b & 1) * 8, a.type, vec, v[b]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[b][i] = 0.0f;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v[b][i]));
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
          x[i] = v[2 * b + (s >> 1)][4 * (s & 1) + i] * down;
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
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int i = 0; i < LT; ++i) {
      const int c = c0 + (SPLIT ? t * 4 + j : t * 8 + 2 * j + i);
      limit[t][i] = c >= cols ? 0 : a.causal ? min(run.len, run.first + c / g + 1) : run.len;
    }

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

  // f32 rows: the tensor cores cut what they add to a sum short, so a sum
  // loses up to 2^-24 of itself with every product, 2^-25 on average; after
  // kKvChain positions it is put aside in shared memory and begun anew.
  float* aside = (float*)(smem + Shape::STAGE_BYTES) + warp * (NT * HD / 8 * 32) + lane;
  auto put_aside = [&](bool add) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int k = 0; k < MT; ++k)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          float* to = aside + ((t * MT + k) * 2 + y) * 32;
          const float v = o[t][k][2 * y] + o[t][k][2 * y + 1];
          *to = add ? *to + v : v;
          o[t][k][2 * y] = o[t][k][2 * y + 1] = 0.0f;
        }
  };
  if (SPLIT) put_aside(false);

  // Scores of two steps of 16 positions to P^T and the running sums. s[z][t]:
  // positions key0[z] + r and key0[z] + r + 8 of the thread's columns.
  auto softmax = [&](float (&s)[2][NT][4], const int (&key0)[2], const float (&ks)[2], const float (&lv)[2],
                     const float (&iv)[2], uint32_t (&p)[2][NT][PB][2]) {
    float x[2][NT][LT][2];
    bool raise = false;
#pragma unroll
    for (int z = 0; z < 2; ++z)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < LT; ++i) {
          const float f = factor[t][i] * ks[z];
          const float d0 = SPLIT ? s[z][t][0] + s[z][t][1] : s[z][t][i];
          const float d1 = SPLIT ? s[z][t][2] + s[z][t][3] : s[z][t][2 + i];
          x[z][t][i][0] = key0[z] + r < limit[t][i] ? fmaf(d0, f, lv[z]) : -INFINITY;
          x[z][t][i][1] = key0[z] + r + 8 < limit[t][i] ? fmaf(d1, f, lv[z]) : -INFINITY;
          raise |= fmaxf(x[z][t][i][0], x[z][t][i][1]) > m[t][i] + kRaise;
        }
    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < LT; ++i) {
          float top = fmaxf(fmaxf(x[0][t][i][0], x[0][t][i][1]), fmaxf(x[1][t][i][0], x[1][t][i][1]));
#pragma unroll
          for (int w = 4; w < 32; w <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
          if (top > m[t][i] + kRaise) {
            const float to = floorf(top) - kBelow, alpha = exp2_fast(m[t][i] - to);
            m[t][i] = to;
            l[t][i] *= alpha;
#pragma unroll
            for (int k = 0; k < MT; ++k) {
              if (SPLIT) {
#pragma unroll
                for (int y = 0; y < 4; ++y) o[t][k][y] *= alpha;
#pragma unroll
                for (int y = 0; y < 2; ++y) aside[((t * MT + k) * 2 + y) * 32] *= alpha;
              } else {
                o[t][k][i] *= alpha;
                o[t][k][2 + i] *= alpha;
              }
            }
          }
        }
    }
#pragma unroll
    for (int z = 0; z < 2; ++z)
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float e[LT][2];
#pragma unroll
        for (int i = 0; i < LT; ++i) {
          e[i][0] = exp2_fast(x[z][t][i][0] - m[t][i]);
          e[i][1] = exp2_fast(x[z][t][i][1] - m[t][i]);
          l[t][i] = fmaf(e[i][0] + e[i][1], iv[z], l[t][i]);
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
          p[z][t][0][h] = transpose8(w);
          if (PB == 2) {
            const float2 hi = __half22float2(*(const __half2*)&w);
            p[z][t][PB - 1][h] = transpose8(pack_f16(e[0][h] - hi.x, e[LT - 1][h] - hi.y));
          }
        }
      }
  };

  uint32_t p[2][NT][PB][2];
  float s[2][NT][4];
  auto clear = [&]() {
#pragma unroll
    for (int z = 0; z < 2; ++z)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int x = 0; x < 4; ++x) s[z][t][x] = 0.0f;
  };
  // Steps of codes, two at a time (two chains of products in flight).
  int unit = 0;
  for (; unit < ncode; unit += 2) {
    const bool two = unit + 1 < ncode;
    if (SPLIT && unit > 0 && unit % (kKvChain / 16) == 0) put_aside(true);
    __syncwarp();  // the units before are read
    fetch();
    fetch();
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
    __syncwarp();
    float ks[2], lv[2], iv[2];
    int key0[2];
    const uint8_t* in[2];
#pragma unroll
    for (int z = 0; z < 2; ++z) {
      const int step = s0 + unit + z;
      if (z == 0 || two) {
        int pg = (step >> page_steps) - base;
        if (pg == 32) {
          base += 32;
          pg = 0;
          if (base + lane <= last_page) scales(table[base + lane]);
        }
        ks[z] = __shfl_sync(0xffffffffu, ksc, pg);
        lv[z] = __shfl_sync(0xffffffffu, vlog, pg);
        iv[z] = __shfl_sync(0xffffffffu, vinv, pg);
        key0[z] = step * 16;
        in[z] = next();
      } else {
        ks[z] = lv[z] = iv[z] = 0.0f;
        key0[z] = 0x3fffffff;  // past every limit
        in[z] = in[0];
      }
    }
    clear();
    float s2[2][NT][4] = {};  // the second half of 128-wide keys (f32 rows: shorter chains)
#pragma unroll
    for (int b = 0; b < KB; ++b)
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        const uint8_t* at = in[z] + (get_k ^ (b << 6));
        const uint4 k0 = *(const uint4*)at, k1 = *(const uint4*)(at + 8 * HD);
        const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint32_t a0 = codes_lo(w0[q]), a1 = codes_lo(w1[q]), a2 = codes_hi(w0[q]), a3 = codes_hi(w1[q]);
#pragma unroll
          for (int t = 0; t < NT; ++t)
            mma16816(SPLIT && b ? s2[z][t] : s[z][t], a0, a1, a2, a3, qf[t][b][q][0], qf[t][b][q][1]);
        }
      }
    if (SPLIT && KB == 2) {
#pragma unroll
      for (int z = 0; z < 2; ++z)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int x = 0; x < 4; ++x) s[z][t][x] += s2[z][t][x];
    }
    softmax(s, key0, ks, lv, iv, p);
#pragma unroll
    for (int z = 0; z < 2; ++z)
#pragma unroll
      for (int b = 0; b < KB; ++b) {
        const uint8_t* at = in[z] + get_v + b * 128;
        const uint4 v0 = *(const uint4*)at, v1 = *(const uint4*)(at + 8 * HD);
        const uint32_t w0[4] = {v0.x, v0.y, v0.z, v0.w}, w1[4] = {v1.x, v1.y, v1.z, v1.w};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint32_t a0 = codes_lo(w0[q]), a1 = codes_hi(w0[q]), a2 = codes_lo(w1[q]), a3 = codes_hi(w1[q]);
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int x = 0; x < PB; ++x) mma16816(o[t][4 * b + q], a0, a1, a2, a3, p[z][t][x][0], p[z][t][x][1]);
        }
      }
  }
  // The open page, f16: a unit of keys, then one of values.
  for (unit = ncode; unit < units; ++unit) {
    const bool keys = ((unit - ncode) & 1) == 0;
    if (keys) {
      __syncwarp();
      while (ahead < min(units, unit + STAGES)) fetch();
      asm volatile("cp.async.wait_all;" ::: "memory");
      clear();
    }
    const uint4* in = (const uint4*)(next() + lane * 16);
#pragma unroll
    for (int b = 0; b < KB; ++b)
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        const uint4 x0 = in[(4 * b + z) * 32], x1 = in[(4 * b + 2 + z) * 32];
        const uint32_t w0[4] = {x0.x, x0.y, x0.z, x0.w}, w1[4] = {x1.x, x1.y, x1.z, x1.w};
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const int q = 2 * z + y;
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            if (keys) {
              mma16816(s[0][t], w0[2 * y], w1[2 * y], w0[2 * y + 1], w1[2 * y + 1], qf[t][b][q][0], qf[t][b][q][1]);
            } else {
#pragma unroll
              for (int x = 0; x < PB; ++x)
                mma16816(o[t][4 * b + q], w0[2 * y], w0[2 * y + 1], w1[2 * y], w1[2 * y + 1], p[0][t][x][0], p[0][t][x][1]);
            }
          }
        }
      }
    if (keys) {
      const int key0[2] = {(f1 + (unit - ncode) / 2) * 16, 0x3fffffff};
      const float one[2] = {1.0f, 1.0f}, none[2] = {0.0f, 0.0f};
      softmax(s, key0, one, none, one, p);
    }
  }

  // The warps' sums meet in shared memory, where their loads were.
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
  float* s_o = (float*)smem;  // [warps][CL][HD]
  static_assert(Shape::STAGE_BYTES >= kAttendWarps * CL * HD * 4, "the sums fit where the loads were");
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
      float* to = s_o + ((size_t)warp * CL + c) * HD;
#pragma unroll
      for (int k = 0; k < MT; ++k) {
        const int d = KB == 1 ? 8 * r + 2 * k : 64 * (k >> 2) + 8 * r + 2 * (k & 3);
        float2 v = make_float2(o[t][k][i], o[t][k][2 + i]);
        if (SPLIT)
          v = make_float2(o[t][k][0] + o[t][k][1] + aside[(t * MT + k) * 64],
                          o[t][k][2] + o[t][k][3] + aside[(t * MT + k) * 64 + 32]);
        *(float2*)(to + d) = v;
      }
    }
  __syncthreads();
  const int nsplit = run.splits;
  // Partial results of a (kv head, block) behind the counters: [column][HD],
  // then (m, l) of each column.
  float* part = (float*)workspace + kKvHead + ((size_t)head * gridDim.x + blockIdx.x) * CL * (HD + 2);
  auto put = [&](int c, int d, float sum, float4 v) {
    const size_t at = (size_t)(run.row0 + c / g) * a.out_stride + (size_t)(head * g + c % g) * HD + d;
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    const float x[4] = {sum == 0.0f ? 0.0f : v.x * inv, sum == 0.0f ? 0.0f : v.y * inv, sum == 0.0f ? 0.0f : v.z * inv,
                        sum == 0.0f ? 0.0f : v.w * inv};
    kv_store4(a.out, at, a.type, vec_out, x);
  };
  for (int x = 4 * threadIdx.x; x < CL * HD; x += 4 * kAttendWarps * 32) {
    const int lc = x / HD, d = x % HD, c = c0 + lc;
    if (c >= cols) break;
    float top = kMInit;
#pragma unroll
    for (int w = 0; w < kAttendWarps; ++w) top = fmaxf(top, s_m[w][lc]);
    float sum = 0.0f;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < kAttendWarps; ++w) {
      const float f = exp2_fast(s_m[w][lc] - top);
      const float4 q = *(const float4*)(s_o + ((size_t)w * CL + lc) * HD + d);
      sum = fmaf(f, s_l[w][lc], sum);
      v = make_float4(fmaf(f, q.x, v.x), fmaf(f, q.y, v.y), fmaf(f, q.z, v.z), fmaf(f, q.w, v.w));
    }
    if (nsplit == 1) {
      put(c, d, sum, v);
    } else {
      *(float4*)(part + x) = v;
      if (d == 0) *(float2*)(part + CL * HD + 2 * lc) = make_float2(top, sum);
    }
  }
  if (nsplit == 1) return;
  // The block that comes last of a tile's shares joins them, in their order
  // (so the result does not depend on which it is). The counter wraps back
  // to zero.
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    unsigned* counter = (unsigned*)workspace + ((size_t)head * gridDim.x + blockIdx.x - split) % kKvCounters;
    s_last = atomicInc(counter, nsplit - 1) == (unsigned)nsplit - 1;
  }
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  const float* first = part - (size_t)split * CL * (HD + 2);
  for (int x = 4 * threadIdx.x; x < CL * HD; x += 4 * kAttendWarps * 32) {
    const int lc = x / HD, d = x % HD, c = c0 + lc;
    if (c >= cols) break;
    float sum = 0.0f;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    join_shares(first, (size_t)CL * (HD + 2), x, CL * HD + 2 * lc, nsplit, sum, v);
    put(c, d, sum, v);
  }
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
// Bound by codes in and values out; 6505 positions on 8 heads 128 wide as
// bf16 take 10 us (4 TB/s of both), 64 short reads 8.5 us, latency.
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
      // 0x4B000000 | c is 2^23 + c; both steps are exact up to the product's
      // rounding.
      const float2 base = make_float2(-8388736.0f, -8388736.0f), by = make_float2(scale, scale);
#pragma unroll
      for (int z = 0; z < 2; ++z)
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          const uint32_t q = w[z][j >> 2];
          const float2 y = mul2(add2(make_float2(__uint_as_float(__byte_perm(q, 0x4B000000u, 0x7540 + (j & 3))),
                                                 __uint_as_float(__byte_perm(q, 0x4B000000u, 0x7541 + (j & 3)))),
                                     base),
                                by);
          x[z][j] = y.x;
          x[z][j + 1] = y.y;
        }
    }
#pragma unroll
    for (int z = 0; z < 2; ++z) {
      const int row = pos + z - run.first;
      if (row >= 0 && row < run.count)
        kv_store8(dst, ((size_t)(run.row0 + row) * kv.kv_heads + head) * HD + 8 * u, type, vec, x[z]);
    }
  }
}

// Block (x, run): one (layer, keys or values, head) of the open page. A fork
// moves at most one page, so it is latency: 5 to 6 us.
__global__ void __launch_bounds__(256) k_kv_fork(const __grid_constant__ KvView kv, const __grid_constant__ KvRuns runs,
                                                 int copy_table) {
  const KvRun& run = runs.run[blockIdx.y];
  const int child = run.seq, parent = run.first, P = kv.page, full = run.count / P, rest = run.count % P;
  if (copy_table && blockIdx.x == 0)
    for (int i = threadIdx.x; i < full; i += 256)
      kv.table[(size_t)child * kv.pages_per_seq + i] = kv.table[(size_t)parent * kv.pages_per_seq + i];
  const int head = blockIdx.x % kv.kv_heads, which = blockIdx.x / kv.kv_heads % 2, layer = blockIdx.x / kv.kv_heads / 2;
  __half* to = kv.open + kv_block(kv, child, layer, which, head) * (size_t)(P * kv.hd);
  if ((full + 1) * P > run.len) {
    // The cut lies in the parent's open page: its f16 as they are (of values
    // whole pairs of positions).
    const uint4* from = (const uint4*)(kv.open + kv_block(kv, parent, layer, which, head) * (size_t)(P * kv.hd));
    const int n = (which ? (rest + 1) / 2 * 2 : rest) * kv.hd / 8;
    for (int i0 = 0; i0 < n; i0 += 1024) {
      uint4 x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (i0 + j * 256 + threadIdx.x < n) x[j] = from[i0 + j * 256 + threadIdx.x];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (i0 + j * 256 + threadIdx.x < n) ((uint4*)to)[i0 + j * 256 + threadIdx.x] = x[j];
    }
    return;
  }
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
// Bound by bytes, each read and written once: 163 us for 0.5 GB of pages (6.6
// TB/s of DRAM traffic both ways, what a plain copy reaches).
__global__ void __launch_bounds__(256) k_kv_move(const __grid_constant__ KvView kv, const int* moves,
                                                 unsigned long long* remap, unsigned epoch) {
  const int src = moves[2 * blockIdx.y], dst = moves[2 * blockIdx.y + 1];
  if (remap && blockIdx.x == 0 && threadIdx.x == 0) remap[src] = (unsigned long long)epoch << 32 | (unsigned)dst;
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

// Table entries follow the moves: remap[page] holds (epoch, target) for the
// pages that this compaction moved, and an older epoch for all others.
__global__ void k_kv_remap(int* table, const unsigned long long* remap, unsigned epoch, size_t entries) {
  const size_t i = blockIdx.x * (size_t)blockDim.x + threadIdx.x;
  if (i >= entries) return;
  const unsigned long long to = remap[table[i]];
  if ((unsigned)(to >> 32) == epoch) table[i] = (int)(unsigned)to;
}

template <int HD, int TYPE, int NT>
cudaError_t attend(const KvView& kv, const KvRuns& runs, const KvAttendArgs& a, const KvAttendPlan& p, int vec,
                   int vec_out, void* ws, cudaStream_t s) {
  constexpr int smem = AttendShape<HD, TYPE, NT>::SMEM;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  static DeviceOnce once;
  e = once.run(dev, [] {
    return cudaFuncSetAttribute(k_kv_attend<HD, TYPE, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  });
  if (e != cudaSuccess) return e;
  k_kv_attend<HD, TYPE, NT>
      <<<dim3(p.blocks, kv.kv_heads), kAttendWarps * 32, smem, s>>>(kv, runs, a, p.chunks, p.splits, vec, vec_out, ws);
  return cudaGetLastError();
}
template <int TYPE>
cudaError_t attend(const KvView& kv, const KvRuns& runs, const KvAttendArgs& a, const KvAttendPlan& p, int vec,
                   int vec_out, void* ws, cudaStream_t s) {
  const bool two = p.cols == (TYPE == kKvF32 ? 8 : 16);
  if (kv.hd == 128)
    return two ? attend<128, TYPE, 2>(kv, runs, a, p, vec, vec_out, ws, s)
               : attend<128, TYPE, 1>(kv, runs, a, p, vec, vec_out, ws, s);
  return two ? attend<64, TYPE, 2>(kv, runs, a, p, vec, vec_out, ws, s)
             : attend<64, TYPE, 1>(kv, runs, a, p, vec, vec_out, ws, s);
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

// One or two n-tiles of columns a block, two when the columns need them (a
// block reads its positions once for all of its columns).
//
// Positions are cut into shares of `c` steps a block, for one to four rounds
// of blocks over the GPU: fewer rounds waste less on starting and joining,
// more even out lengths that differ. A round costs its longest share and
// kStart steps. Measured with kStart at 12 / 24 / 48 / 96, us: 64 streams of
// 601 to 1279 positions, 32 heads on 8 and 128 wide, 45.5 / 40.4 / 40.5 / 40.6;
// 6 of 40001 to 65535, bf16, 130 / 122 / 122 / 122; 24 of up to 1500, four rows
// each, 16 on 16 and 64 wide, 20.8 / 18.2 / 18.2 / 18.2; 128 of 100 to 600, 16 on
// 2 and 64 wide, 25.5 / 26.2 / 25.6 / 26.7.
KvAttendPlan plan_kv_attend(const KvView& kv, KvRuns& runs, const KvAttendArgs& a) {
  KvAttendPlan p;
  const int g = a.heads / kv.kv_heads, unit = a.type == kKvF32 ? 4 : 8;
  int most = 1;
  for (int i = 0; i < runs.n && !runs.row_seq; ++i) most = std::max(most, runs.run[i].count);
  p.cols = (size_t)most * g > (size_t)unit ? 2 * unit : unit;
  const int slots = current_sm_count() * (kv.hd == 128 && p.cols > unit ? 2 : 3);
  // Tiles and steps of the runs (of the longest row for a decode step, whose
  // positions only the device knows).
  double tiles = 0, work = 0;
  int longest = 1;
  p.chunks = (g + p.cols - 1) / p.cols;
  if (runs.row_seq) {
    tiles = (double)runs.n * p.chunks;
    longest = (a.max_len + 15) / 16;
    work = tiles * longest;
  } else {
    for (int i = 0; i < runs.n; ++i) {
      const double t = (double)(((size_t)runs.run[i].count * g + p.cols - 1) / p.cols);
      const int steps = (runs.run[i].len + 15) / 16;
      tiles += t;
      work += t * steps;
      longest = std::max(longest, steps);
    }
  }
  tiles *= kv.kv_heads;
  work *= kv.kv_heads;
  auto blocks = [&](int c) {
    long n = 0;
    if (runs.row_seq) return (long)tiles * ((longest + c - 1) / c);
    for (int i = 0; i < runs.n; ++i)
      n += (long)(((size_t)runs.run[i].count * g + p.cols - 1) / p.cols) * (((runs.run[i].len + 15) / 16 + c - 1) / c);
    return n * kv.kv_heads;
  };
  constexpr double kStart = 48.0;
  int share = longest;
  if (tiles < 4.0 * slots && tiles <= kKvCounters) {
    double best = (double)((int)((tiles + slots - 1) / slots)) * (longest + kStart);
    for (int rounds = 1; rounds <= 4; ++rounds) {
      // sum ceil(steps / c) over the tiles is about work / c + tiles / 2; the
      // count must not pass the rounds, or a last round of a few blocks comes.
      const double room = (double)rounds * slots - 0.5 * tiles;
      if (room <= 0) continue;
      int c = std::max(16, (int)(work / room) + 1);
      while (c < longest && blocks(c) > (long)rounds * slots) c += std::max(1, c / 32);
      if (c < longest && rounds * (c + kStart) < best) {
        best = rounds * (c + kStart);
        share = c;
      }
    }
  }
  const size_t bytes = (size_t)kv.kv_heads * p.cols * (kv.hd + 2) * 4;
  for (;; share = std::min(longest, 2 * share)) {
    p.blocks = 0;
    p.joins = false;
    if (runs.row_seq) {
      p.splits = (longest + share - 1) / share;
      p.blocks = runs.n * p.chunks * p.splits;
      p.joins = p.splits > 1;
    } else {
      for (int i = 0; i < runs.n; ++i) {
        KvRun& r = runs.run[i];
        r.block0 = p.blocks;
        r.splits = std::max(1, ((r.len + 15) / 16 + share - 1) / share);
        p.joins |= r.splits > 1;
        p.blocks += (int)(((size_t)r.count * g + p.cols - 1) / p.cols) * r.splits;
      }
    }
    p.workspace = p.joins ? kKvHead * 4 + p.blocks * bytes : 0;
    if (!p.joins || ((size_t)p.blocks * kv.kv_heads <= kKvCounters && p.workspace <= kKvWorkspace)) break;
  }
  return p;
}

cudaError_t launch_kv_attend(const KvView& kv, const KvRuns& runs, const KvAttendArgs& a, const KvAttendPlan& p, void* ws,
                             cudaStream_t s) {
  if (p.blocks <= 0) return cudaSuccess;
  if (p.joins && !ws) return cudaErrorInvalidValue;
  const size_t size = a.type == kKvF32 ? 4 : 2;
  const int vec = ((uintptr_t)a.q | a.q_stride * size) % 16 == 0;
  const int vec_out = ((uintptr_t)a.out | a.out_stride * size) % 16 == 0;
  if (a.type == kKvF32) return attend<kKvF32>(kv, runs, a, p, vec, vec_out, ws, s);
  if (a.type == kKvF16) return attend<kKvF16>(kv, runs, a, p, vec, vec_out, ws, s);
  return attend<kKvBF16>(kv, runs, a, p, vec, vec_out, ws, s);
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

cudaError_t launch_kv_move(const KvView& kv, const int* moves, int n, unsigned long long* remap, unsigned epoch,
                           cudaStream_t s) {
  const size_t vec = (size_t)kv.layers * 2 * kv.kv_heads * kv.page * kv.hd / 16;
  const int x = (int)std::max<size_t>(1, std::min<size_t>((vec + 2047) / 2048, 64));
  for (int i = 0; i < n; i += 65535)
    k_kv_move<<<dim3(x, std::min(n - i, 65535)), 256, 0, s>>>(kv, moves + 2 * i, remap, epoch);
  return cudaGetLastError();
}

cudaError_t launch_kv_remap(const KvView& kv, const unsigned long long* remap, unsigned epoch, int sequences,
                            cudaStream_t s) {
  const size_t entries = (size_t)sequences * kv.pages_per_seq;
  k_kv_remap<<<(unsigned)((entries + 255) / 256), 256, 0, s>>>(kv.table, remap, epoch, entries);
  return cudaGetLastError();
}

}  // namespace trit
