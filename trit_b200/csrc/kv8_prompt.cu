// Attention of many query rows over the 8-bit cache on the fifth-generation
// tensor cores. A block takes 128 query columns (a column is one query row of
// one head of the kv head's group) and walks the positions 128 at a time:
//   S = Q K^T    tcgen05.mma kind::f16, M 128 columns, N 128 positions
//   O += P V     M 128 columns, N the head's values, K 128 positions
// Roles:
//   warps 0-3   widen the codes of a tile to f16 (exact: a byte permute and a
//               subtraction for two codes) into swizzled shared memory, keys
//               and values each in two buffers; the open page's f16 is
//               copied. Codes are loaded half a tile ahead in registers.
//   warps 4-11  softmax: a thread owns one query column and half of a tile's
//               positions (and half of O's values); the two threads of a
//               column agree on the tile's largest score.
//   warp 12     owns TMEM and issues the products.
// P goes to TMEM, where the second product takes it as its first operand, so
// shared memory carries only K, V and Q.
//
// f32 rows take two products each (Q and P as f16 value and remainder, 22
// bits, summed in one accumulator), f16 and bf16 rows one (a row scaled by a
// power of two; P rounded to 2^-11, below the output's rounding). Scales are
// applied as in k_kv_attend: the key scale to S, the value scale in the
// exponent of P. Bound by the tensor cores: 4 * 128 * 128 * hd operations a
// tile, twice that for f32 rows.
#include <algorithm>

#include "kernels.h"
#include "kv8.cuh"
#include "tc.cuh"

namespace trit {
namespace {

constexpr int kTile = 128;  // query columns, and positions a step
constexpr int kConvThreads = 128, kSoftThreads = 256;
constexpr int kPromptThreads = kConvThreads + kSoftThreads + 32;
// TMEM columns: S (two buffers), O, P (value, remainder).
constexpr uint32_t kColO = 256, kColP = 384, kColPLow = 448;

struct PromptSmem {
  uint64_t kfull[2], kempty[2], vfull[2], vempty[2], sfull[2], sfree[2], qfull, pfull, ofull, pair[4], drain;
  // Of a tile's groups of 16 positions: key scale, log2 and inverse of the
  // value scale. Four tiles deep: a buffer is written again only when S of
  // the tile two later is made, which waits for the softmax of this one.
  float scales[4][8][4];
  float top[2][2][kTile];  // by parity, half and column
  uint32_t tmem;
  int abort, last;
};

// D = A B (+ D when `accumulate`), A in TMEM.
__device__ __forceinline__ void mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b, uint32_t idesc,
                                           uint32_t accumulate) {
  uint32_t mask0 = 0, mask1 = 0, mask2 = 0, mask3 = 0;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %6, %7, %8}, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b), "r"(idesc), "r"(accumulate), "r"(mask0), "r"(mask1), "r"(mask2), "r"(mask3));
}

// Two codes of bytes (0, 2) or (1, 3): one position's of a value word.
__device__ __forceinline__ uint32_t codes_even(uint32_t w) {
  const uint32_t x = __byte_perm(w, 0x64646464u, 0x4240);
  const __half2 h = __hsub2(*(const __half2*)&x, __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480)));
  return *(const uint32_t*)&h;
}
__device__ __forceinline__ uint32_t codes_odd(uint32_t w) {
  const uint32_t x = __byte_perm(w, 0x64646464u, 0x4341);
  const __half2 h = __hsub2(*(const __half2*)&x, __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480)));
  return *(const uint32_t*)&h;
}
// Where 16-byte chunk c (8 values) of row r lies in a tile of 128 rows:
// 64-value halves of 128-byte rows, swizzled.
__device__ __forceinline__ int tile_at(int r, int c) {
  return (c >> 3) * (kTile * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4);
}

template <int HD, bool LOW>
constexpr int prompt_smem() {
  return 1024 + (LOW ? 2 : 1) * kTile * HD * 2 + 4 * kTile * HD * 2 + (int)sizeof(PromptSmem);
}

template <int HD, bool LOW>
__global__ void __launch_bounds__(kPromptThreads, 1)
    k_kv_prompt(const __grid_constant__ KvView kv, const __grid_constant__ KvRuns runs,
                const __grid_constant__ KvAttendArgs a, int vec, int vec_out, void* workspace, int* status) {
  constexpr int TILE = kTile * HD * 2;  // bytes of an f16 tile
  constexpr int UH = HD / 2;            // values of O a softmax thread holds
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* base = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* q_s = base;
  uint8_t* k_s = q_s + (LOW ? 2 : 1) * TILE;  // [2]
  uint8_t* v_s = k_s + 2 * TILE;              // [2]
  PromptSmem* S = (PromptSmem*)(v_s + 2 * TILE);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int head = blockIdx.y, g = a.heads / kv.kv_heads, P = kv.page;

  KvRun run;
  int chunk, split;
  // The last tiles of a causal prompt see most: they start first.
  const int block = gridDim.x - 1 - blockIdx.x;
  find_run(runs, block, 1, 1, run, chunk, split);
  const int cols = run.count * g, c0 = chunk * kTile;
  const int last_row = (min(cols, c0 + kTile) - 1) / g;
  const int kend = a.causal ? min(run.len, run.first + last_row + 1) : run.len;
  const int tiles = (kend + kTile - 1) / kTile, per = (tiles + run.splits - 1) / run.splits;
  const int t0 = min(tiles, split * per), nt = min(tiles, t0 + per) - t0;
  const int full = run.len & ~(P - 1);  // positions in full pages
  const size_t bytes = (size_t)P * HD;
  volatile int* abort = &S->abort;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&S->kfull[i], kConvThreads);
      mbar_init(&S->kempty[i], 1);
      mbar_init(&S->vfull[i], kConvThreads);
      mbar_init(&S->vempty[i], 1);
      mbar_init(&S->sfull[i], 1);
      mbar_init(&S->sfree[i], kSoftThreads);
    }
    for (int i = 0; i < 4; ++i) mbar_init(&S->pair[i], 64);
    mbar_init(&S->qfull, kSoftThreads);
    mbar_init(&S->pfull, kSoftThreads);
    mbar_init(&S->ofull, 1);
    mbar_init(&S->drain, 1);
    S->abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 12) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&S->tmem)), "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = S->tmem;

  if (warp < 4) {
    // ---- codes to f16 ----
    constexpr int KU = HD / 16;          // 16-code units of a key
    constexpr int N = kTile * KU / 128;  // units a thread takes of a tile's keys (of its values as many)
    const int* table = kv.table + (size_t)run.seq * kv.pages_per_seq;
    const __half* open_k = kv.open + kv_block(kv, run.seq, a.layer, 0, head) * bytes;
    const __half* open_v = kv.open + kv_block(kv, run.seq, a.layer, 1, head) * bytes;
    // Keys: unit i of a thread is row kr(i) and values 16 ku .. of it; eight
    // lanes take eight rows, so that their stores spread over the banks.
    // Values: pair vr(i) of positions and values 8 vu .. of both.
    const int kr0 = (warp * 8 + (lane & 7)), ku0 = lane >> 3;
    const int vr0 = warp * 4 + (lane & 3), vu0 = lane >> 2;
    constexpr int KSTEP = KU / 4;  // a warp covers 8 rows x 4 units: turns over the units
    auto key_row = [&](int i) { return kr0 + i / KSTEP * 32; };
    auto key_unit = [&](int i) { return ku0 + i % KSTEP * 4; };
    constexpr int VU = HD / 8;  // 8-value units of a pair
    constexpr int VSTEP = VU / 8;
    auto val_pair = [&](int i) { return vr0 + i / VSTEP * 16; };
    auto val_unit = [&](int i) { return vu0 + i % VSTEP * 8; };
    uint4 kc[N], vc[N];
    auto load_keys = [&](int tile) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int pos = tile * kTile + key_row(i);
        kc[i] = make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);
        if (pos < kend && pos < full) {
          const size_t b = kv_block(kv, table[pos >> kv.page_shift], a.layer, 0, head) * bytes;
          kc[i] = __ldg((const uint4*)(kv.codes + b + (size_t)(pos & (P - 1)) * HD + 16 * key_unit(i)));
        }
      }
    };
    auto load_values = [&](int tile) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int pos = tile * kTile + 2 * val_pair(i);
        vc[i] = make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);
        if (pos < kend && pos < full) {
          const size_t b = kv_block(kv, table[pos >> kv.page_shift], a.layer, 1, head) * bytes;
          vc[i] = __ldg((const uint4*)(kv.codes + b + (size_t)((pos & (P - 1)) >> 1) * (2 * HD) + 16 * val_unit(i)));
        }
      }
    };
    if (nt > 0) load_keys(t0);
    for (int j = 0; j < nt; ++j) {
      const int s = j & 1, tile = t0 + j;
      load_values(tile);
      // Scales of the tile's groups (thread i: group i).
      float ks = 0.0f, vl = 0.0f, vi = 0.0f;
      if (threadIdx.x < 8) {
        const int pos = tile * kTile + 16 * threadIdx.x;
        if (pos < kend) {
          ks = 1.0f;
          vi = 1.0f;
          if (pos < full) {
            const size_t b = kv_block(kv, table[pos >> kv.page_shift], a.layer, 0, head);
            ks = kv.scales[b];
            const float vs = kv.scales[b + kv.kv_heads];
            vl = vs > 0.0f ? __log2f(vs) : kZeroScaleLog2;
            vi = vs > 0.0f ? __fdividef(1.0f, vs) : 2147483648.0f;
          }
        }
      }
      if (!mbar_wait(&S->kempty[s], ((j >> 1) & 1) ^ 1, abort)) break;
      if (threadIdx.x < 8) {
        float* to = S->scales[j & 3][threadIdx.x];
        to[0] = ks;
        to[1] = vl;
        to[2] = vi;
      }
      uint8_t* kt = k_s + s * TILE;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int r = key_row(i), u = key_unit(i), pos = tile * kTile + r;
        uint4 x, y;
        if (pos >= full && pos < kend) {
          const uint4* src = (const uint4*)(open_k + (size_t)(pos - full) * HD + 16 * u);
          x = src[0];
          y = src[1];
        } else {
          x = make_uint4(codes_lo(kc[i].x), codes_hi(kc[i].x), codes_lo(kc[i].y), codes_hi(kc[i].y));
          y = make_uint4(codes_lo(kc[i].z), codes_hi(kc[i].z), codes_lo(kc[i].w), codes_hi(kc[i].w));
        }
        *(uint4*)(kt + tile_at(r, 2 * u)) = x;
        *(uint4*)(kt + tile_at(r, 2 * u + 1)) = y;
      }
      fence_async_smem();
      mbar_arrive(&S->kfull[s]);
      if (j + 1 < nt) load_keys(tile + 1);
      if (!mbar_wait(&S->vempty[s], ((j >> 1) & 1) ^ 1, abort)) break;
      uint8_t* vt = v_s + s * TILE;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int r = 2 * val_pair(i), u = val_unit(i), pos = tile * kTile + r;
        uint4 x, y;
        if (pos >= full && pos < kend) {
          // Pairs of the open page: words (position 0, position 1) of a value.
          const uint4* src = (const uint4*)(open_v + (size_t)(pos - full) * HD + 16 * u);
          const uint4 p = src[0], q = src[1];
          x = make_uint4(__byte_perm(p.x, p.y, 0x5410), __byte_perm(p.z, p.w, 0x5410), __byte_perm(q.x, q.y, 0x5410),
                         __byte_perm(q.z, q.w, 0x5410));
          y = make_uint4(__byte_perm(p.x, p.y, 0x7632), __byte_perm(p.z, p.w, 0x7632), __byte_perm(q.x, q.y, 0x7632),
                         __byte_perm(q.z, q.w, 0x7632));
        } else {
          x = make_uint4(codes_even(vc[i].x), codes_even(vc[i].y), codes_even(vc[i].z), codes_even(vc[i].w));
          y = make_uint4(codes_odd(vc[i].x), codes_odd(vc[i].y), codes_odd(vc[i].z), codes_odd(vc[i].w));
        }
        *(uint4*)(vt + tile_at(r, u)) = x;
        *(uint4*)(vt + tile_at(r + 1, u)) = y;
      }
      fence_async_smem();
      mbar_arrive(&S->vfull[s]);
    }
  } else if (warp == 12) {
    if (lane == 0 && nt > 0) {
      const uint32_t qa = smem_u32(q_s), ka = smem_u32(k_s), va = smem_u32(v_s);
      auto pv = [&](int j) -> bool {
        if (!mbar_wait(&S->pfull, j & 1, abort) || !mbar_wait(&S->vfull[j & 1], (j >> 1) & 1, abort)) return false;
        fence_after();
        const uint32_t v = va + (j & 1) * TILE;
#pragma unroll
        for (int i = 0; i < kTile / 16; ++i) {
          const uint64_t b = smem_desc_sw128_mn(v + i * 2048, kTile * 128);
          mma_f16_ts(tmem + kColO, tmem + kColP + i * 8, b, idesc_f16n(HD, true), (j > 0 || i > 0) ? 1u : 0u);
          if (LOW) mma_f16_ts(tmem + kColO, tmem + kColPLow + i * 8, b, idesc_f16n(HD, true), 1u);
        }
        mma_commit(&S->ofull);
        mma_commit(&S->vempty[j & 1]);
        return true;
      };
      bool ok = mbar_wait(&S->qfull, 0, abort);
      for (int j = 0; j < nt && ok; ++j) {
        const int s = j & 1;
        if (!mbar_wait(&S->kfull[s], (j >> 1) & 1, abort) || !mbar_wait(&S->sfree[s], ((j >> 1) & 1) ^ 1, abort)) {
          ok = false;
          break;
        }
        fence_after();
        const uint32_t k = ka + s * TILE;
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) {
          const uint32_t at = (i >> 2) * (kTile * 128) + (i & 3) * 32;
          const uint64_t b = smem_desc_sw128(k + at);
          mma_f16(tmem + s * kTile, smem_desc_sw128(qa + at), b, idesc_f16n(kTile), i > 0 ? 1u : 0u);
          if (LOW) mma_f16(tmem + s * kTile, smem_desc_sw128(qa + TILE + at), b, idesc_f16n(kTile), 1u);
        }
        mma_commit(&S->sfull[s]);
        mma_commit(&S->kempty[s]);
        if (j > 0) ok = pv(j - 1);
      }
      if (ok) pv(nt - 1);
      mma_commit(&S->drain);
      const long long start = now_ns();
      while (!mbar_test(&S->drain, 0) && now_ns() - start < TC_WAIT_NS) {
      }
    }
  } else {
    // ---- softmax ----
    const int quarter = warp & 3, half = (warp - 4) >> 2, q = quarter * 32 + lane;
    const int c = c0 + q;
    const bool live = c < cols;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
    const int limit = !live ? 0 : a.causal ? min(run.len, run.first + c / g + 1) : run.len;
    int low_limit = live ? limit : 0x7fffffff;  // of the warp's rows: below it no mask is needed
#pragma unroll
    for (int o = 16; o; o >>= 1) low_limit = min(low_limit, __shfl_xor_sync(0xffffffffu, low_limit, o));
    int pairs = 0;
    // The two threads of a column tell each other a number.
    auto both_max = [&](float x, bool& ok) {
      S->top[pairs & 1][half][q] = x;
      mbar_arrive(&S->pair[quarter]);
      ok = __all_sync(0xffffffffu, mbar_wait(&S->pair[quarter], pairs & 1, abort));
      const float y = S->top[pairs & 1][half ^ 1][q];
      ++pairs;
      return fmaxf(x, y);
    };
    bool ok = true;
    float factor;
    {
      // This thread's half of the row: values UH * half ..
      const size_t at = live ? (size_t)(run.row0 + c / g) * a.q_stride + (size_t)(head * g + c % g) * HD + UH * half : 0;
      float v[UH / 8][8];
      float top = 0.0f;
#pragma unroll
      for (int i = 0; i < UH / 8; ++i) {
        if (live) {
          kv_load8(a.q, at + 8 * i, a.type, vec, v[i]);
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k) v[i][k] = 0.0f;
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) top = fmaxf(top, fabsf(v[i][k]));
      }
      top = both_max(top, ok);
      int e = 0;
      if (top > 0.0f && top <= 3.4e38f) e = max(-126, min(126, (int)((__float_as_uint(top) >> 23) & 255) - 127));
      const float down = __uint_as_float((uint32_t)(127 - e) << 23);
      factor = a.scale * 1.4426950408889634f * __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
      for (int i = 0; i < UH / 8; ++i) {
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float x = v[i][2 * k] * down, y = v[i][2 * k + 1] * down;
          const __half2 h = __floats2half2_rn(x, y);
          hi[k] = *(const uint32_t*)&h;
          lo[k] = pack_f16(x - __low2float(h), y - __high2float(h));
        }
        const int to = tile_at(q, UH / 8 * half + i);
        *(uint4*)(q_s + to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        if (LOW) *(uint4*)(q_s + TILE + to) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
    }
    fence_async_smem();
    mbar_arrive(&S->qfull);
    float m = kMInit, l = 0.0f;
    for (int j = 0; j < nt && ok; ++j) {
      const int s = j & 1, key0 = (t0 + j) * kTile + 64 * half;
      // Warp-uniform waits: the TMEM loads and stores below are warp-wide.
      if (!__all_sync(0xffffffffu, mbar_wait(&S->sfull[s], (j >> 1) & 1, abort))) {
        ok = false;
        break;
      }
      fence_after();
      float v[64];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        uint32_t r[32];
        tmem_ld<32>(lanes + s * kTile + 64 * half + 32 * b, r);
        tmem_wait_ld();
#pragma unroll
        for (int k = 0; k < 32; ++k) v[32 * b + k] = __uint_as_float(r[k]);
      }
      float f[4], vl[4], vi[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 x = *(const float4*)S->scales[j & 3][4 * half + i];
        f[i] = factor * x.x;
        vl[i] = x.y;
        vi[i] = x.z;
      }
      fence_before();
      mbar_arrive(&S->sfree[s]);
      float top = kMInit;
#pragma unroll
      for (int k = 0; k < 64; ++k) v[k] = fmaf(v[k], f[k >> 4], vl[k >> 4]);
      if (key0 + 64 > low_limit) {
#pragma unroll
        for (int k = 0; k < 64; ++k)
          if (key0 + k >= limit) v[k] = -INFINITY;
      }
#pragma unroll
      for (int k = 0; k < 64; ++k) top = fmaxf(top, v[k]);
      top = both_max(top, ok);
      if (!ok) break;
      float alpha = 1.0f;
      if (top > m + kRaise) {
        alpha = exp2_fast(m - (top - kBelow));
        m = top - kBelow;
        l *= alpha;
      }
      // P and O are free when the product before is done.
      if (j > 0) {
        if (!__all_sync(0xffffffffu, mbar_wait(&S->ofull, (j - 1) & 1, abort))) {
          ok = false;
          break;
        }
        fence_after();
        if (__any_sync(0xffffffffu, alpha != 1.0f)) {
#pragma unroll
          for (int b = 0; b < UH / 32; ++b) {
            uint32_t r[32];
            tmem_ld<32>(lanes + kColO + UH * half + 32 * b, r);
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 32; ++k) r[k] = __float_as_uint(__uint_as_float(r[k]) * alpha);
            tmem_st32(lanes + kColO + UH * half + 32 * b, r);
          }
        }
      }
      uint32_t hi[32];
#pragma unroll
      for (int k = 0; k < 32; ++k) {
        const float x = exp2_fast(v[2 * k] - m), y = exp2_fast(v[2 * k + 1] - m);
        l = fmaf(x + y, vi[k >> 3], l);
        const __half2 h = __floats2half2_rn(x, y);
        hi[k] = *(const uint32_t*)&h;
        if (LOW) {
          v[2 * k] = x - __low2float(h);
          v[2 * k + 1] = y - __high2float(h);
        }
      }
      tmem_st32(lanes + kColP + 32 * half, hi);
      if (LOW) {
#pragma unroll
        for (int k = 0; k < 32; ++k) hi[k] = pack_f16(v[2 * k], v[2 * k + 1]);
        tmem_st32(lanes + kColPLow + 32 * half, hi);
      }
      tmem_wait_st();
      fence_before();
      mbar_arrive(&S->pfull);
    }
    // The column's sums, joined over its two threads.
    if (ok) {
      S->top[pairs & 1][half][q] = l;
      mbar_arrive(&S->pair[quarter]);
      ok = __all_sync(0xffffffffu, mbar_wait(&S->pair[quarter], pairs & 1, abort));
      l += S->top[pairs & 1][half ^ 1][q];
    }
    if (ok && nt > 0) ok = __all_sync(0xffffffffu, mbar_wait(&S->ofull, (nt - 1) & 1, abort));
    if (ok) {
      fence_after();
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      float* part = (float*)workspace + kKvCounters + (((size_t)head * gridDim.x + block) * kTile + q) * (HD + 2);
#pragma unroll
      for (int b = 0; b < UH / 32; ++b) {
        uint32_t r[32];
        if (nt > 0) {
          tmem_ld<32>(lanes + kColO + UH * half + 32 * b, r);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int k = 0; k < 32; ++k) r[k] = 0;
        }
        if (!live) continue;
        if (run.splits == 1) {
          const size_t to = (size_t)(run.row0 + c / g) * a.out_stride + (size_t)(head * g + c % g) * HD + UH * half + 32 * b;
#pragma unroll
          for (int k = 0; k < 32; k += 8) {
            float x[8];
#pragma unroll
            for (int z = 0; z < 8; ++z) x[z] = l == 0.0f ? 0.0f : __uint_as_float(r[k + z]) * inv;
            kv_store8(a.out, to + k, a.type, vec_out, x);
          }
        } else {
#pragma unroll
          for (int k = 0; k < 32; ++k) part[UH * half + 32 * b + k] = __uint_as_float(r[k]);
        }
      }
      if (run.splits > 1 && live && half == 0) {
        part[HD] = m;
        part[HD + 1] = l;
      }
    }
  }
  if (run.splits > 1) __threadfence();
  fence_before();
  __syncthreads();
  if (warp == 12) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
  if (threadIdx.x == 0 && S->abort) *(volatile int*)status = 1;
  if (run.splits == 1) return;
  // The block that comes last of a tile's shares joins them, in their order.
  if (threadIdx.x == 0) {
    unsigned* counter = (unsigned*)workspace + ((size_t)head * gridDim.x + block - split) % kKvCounters;
    S->last = atomicInc(counter, run.splits - 1) == (unsigned)run.splits - 1;
  }
  __syncthreads();
  if (!S->last) return;
  __threadfence();
  const float* first = (const float*)workspace + kKvCounters + ((size_t)head * gridDim.x + block - split) * kTile * (HD + 2);
  for (int x = threadIdx.x; x < kTile * HD; x += kPromptThreads) {
    const int lc = x / HD, d = x % HD, c = c0 + lc;
    if (c >= cols) break;
    float top = kMInit, sum = 0.0f, val = 0.0f;
    for (int i = 0; i < run.splits; ++i) {
      const float* p = first + ((size_t)i * kTile + lc) * (HD + 2);
      const float pm = __ldcg(p + HD), pl = __ldcg(p + HD + 1), pv = __ldcg(p + d);
      const float to = fmaxf(top, pm), fa = exp2_fast(top - to), fb = exp2_fast(pm - to);
      sum = fmaf(sum, fa, pl * fb);
      val = fmaf(val, fa, pv * fb);
      top = to;
    }
    kv_store(a.out, (size_t)(run.row0 + c / g) * a.out_stride + (size_t)(head * g + c % g) * HD + d, a.type,
             sum == 0.0f ? 0.0f : val / sum);
  }
}

template <int HD, bool LOW>
cudaError_t prompt(const KvView& kv, const KvRuns& runs, const KvAttendArgs& a, const KvAttendPlan& p, int vec,
                   int vec_out, void* ws, int* status, cudaStream_t s) {
  constexpr int smem = prompt_smem<HD, LOW>();
  static_assert(smem <= 227 * 1024, "the tiles fit in shared memory");
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  static DeviceOnce once;
  e = once.run(dev, [] {
    return cudaFuncSetAttribute(k_kv_prompt<HD, LOW>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  });
  if (e != cudaSuccess) return e;
  k_kv_prompt<HD, LOW><<<dim3(p.blocks, kv.kv_heads), kPromptThreads, smem, s>>>(kv, runs, a, vec, vec_out, ws, status);
  return cudaGetLastError();
}

}  // namespace

// A tile's positions are cut into shares only while the tiles leave SMs idle;
// a share costs about a step and a half to start and to join (measured).
KvAttendPlan plan_kv_prompt(const KvView& kv, KvRuns& runs, const KvAttendArgs& a) {
  KvAttendPlan p;
  p.cols = kTile;
  const int g = a.heads / kv.kv_heads, slots = current_sm_count();
  double tiles = 0, work = 0;
  int longest = 1;
  for (int i = 0; i < runs.n; ++i) {
    const double t = (double)(((size_t)runs.run[i].count * g + kTile - 1) / kTile);
    const int steps = (runs.run[i].len + kTile - 1) / kTile;
    tiles += t;
    work += t * steps;
    longest = std::max(longest, steps);
  }
  tiles *= kv.kv_heads;
  work *= kv.kv_heads;
  int share = longest;
  if (tiles < 2.0 * slots) {
    double best = (double)((int)((tiles + slots - 1) / slots)) * (longest + 1.5);
    for (int rounds = 1; rounds <= 2; ++rounds) {
      const double room = (double)rounds * slots - 0.5 * tiles;
      if (room <= 0) continue;
      const int c = std::max(2, (int)(work / room) + 1);
      if (c < longest && rounds * (c + 1.5) < best) {
        best = rounds * (c + 1.5);
        share = c;
      }
    }
  }
  const size_t bytes = (size_t)kv.kv_heads * kTile * (kv.hd + 2) * 4;
  for (;; share = std::min(longest, 2 * share)) {
    p.blocks = 0;
    p.joins = false;
    for (int i = 0; i < runs.n; ++i) {
      KvRun& r = runs.run[i];
      r.block0 = p.blocks;
      r.splits = std::max(1, ((r.len + kTile - 1) / kTile + share - 1) / share);
      p.joins |= r.splits > 1;
      p.blocks += (int)(((size_t)r.count * g + kTile - 1) / kTile) * r.splits;
    }
    p.workspace = kKvCounters * 4 + p.blocks * bytes;
    if (!p.joins || ((size_t)p.blocks * kv.kv_heads <= kKvCounters && p.workspace <= kKvWorkspace)) break;
  }
  return p;
}

cudaError_t launch_kv_prompt(const KvView& kv, const KvRuns& runs, const KvAttendArgs& a, const KvAttendPlan& p, void* ws,
                             int* status, cudaStream_t s) {
  if (p.blocks <= 0) return cudaSuccess;
  if (runs.row_seq || (p.joins && !ws)) return cudaErrorInvalidValue;
  const size_t size = a.type == kKvF32 ? 4 : 2;
  const int vec = ((uintptr_t)a.q | a.q_stride * size) % 16 == 0, vec_out = ((uintptr_t)a.out | a.out_stride * size) % 16 == 0;
  const bool low = a.type == kKvF32;
  if (kv.hd == 128)
    return low ? prompt<128, true>(kv, runs, a, p, vec, vec_out, ws, status, s)
               : prompt<128, false>(kv, runs, a, p, vec, vec_out, ws, status, s);
  return low ? prompt<64, true>(kv, runs, a, p, vec, vec_out, ws, status, s)
             : prompt<64, false>(kv, runs, a, p, vec, vec_out, ws, status, s);
}

}  // namespace trit
