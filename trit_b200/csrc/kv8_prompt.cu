// Attention of many query rows over the 8-bit cache on the fifth-generation
// tensor cores. A block takes one or two tiles of 128 query columns (a column
// is one query row of one head of the kv head's group) and walks the positions
// 128 at a time:
//   S = Q K^T    tcgen05.mma kind::f16, M 128 columns, N 128 positions
//   O += P V     M 128 columns, N the head's values, K 128 positions
// Roles:
//   warps 0-3   widen the codes of a step to f16 (exact: a byte permute and a
//               subtraction for two codes) into swizzled shared memory; the
//               open page's f16 is copied. Codes are loaded half a step ahead
//               in registers, page numbers a step ahead.
//   warps 4-    softmax, four warps a tile: a thread owns one query column
//               (one TMEM lane). One pass over its scores in TMEM; P takes
//               their place and is the second product's first operand.
//   last warp   owns TMEM and issues the products, for two tiles in turn: while
//               one tile's run, the other's softmax does.
//
// f32 rows take two products each (Q and P as f16 value and remainder, 22
// bits, summed in one accumulator), f16 rows two for P V only (they are f16
// already), bf16 rows one (P rounded to 2^-11, an eighth of the output's
// rounding); 16-bit rows are scaled by a power of two. Scales are applied as
// in k_kv_attend: the key scale to S, the value scale in the
// exponent of P. The floor is the tensor cores' 4 * 128 * 128 * hd operations
// a tile and step, twice that for f32 rows. What bounds it is the softmax: one
// thread a column takes about 5400 cycles a step's tile, the products of two
// tiles 4100, and a step of two tiles about 8400. 4000 causal f32 rows, 32
// heads on 8, 128 wide: 475 us, 276 TFLOP/s (552 as multiplied), the tensor
// pipe busy 31 %; putting sums aside is 50 us of it. As f16 rows 342 us (275
// without P's remainder), as bf16 rows 276 us, 475 TFLOP/s.
#include <algorithm>

#include "device.cuh"
#include "kernels.h"
#include "kv8.cuh"
#include "tc.cuh"

namespace trit {
namespace {

constexpr int kTile = 128;  // query columns of a tile, and positions a step
constexpr int kConvThreads = 128;

// QT: query tiles a block. V is in one buffer where two do not fit. TYPE
// (KvType): f32 rows have remainders of Q and P, f16 rows of P.
template <int HD, int TYPE, int QT>
struct PromptShape {
  static constexpr bool LOW = TYPE == kKvF32;
  static constexpr int TILE = kTile * HD * 2;  // bytes of an f16 tile
  static constexpr int BLOCKS = QT == 1 && !(LOW && HD == 128) ? 2 : 1;  // an SM
  static constexpr int KS = QT == 1 && HD == 128 ? 1 : 2, VS = (QT == 1 || LOW) && HD == 128 ? 1 : 2;
  static constexpr int THREADS = kConvThreads + QT * 128 + 32;
  static constexpr uint32_t COL_O = QT * kTile;  // TMEM columns: S (then P) of each tile, O of each
  static constexpr uint32_t COLS = QT == 2 ? 512 : 256;
};

struct PromptSmem {
  uint64_t kfull[2], kempty[2], vfull[2], vempty[2], sfull[2], pfull[2], qfull, done;
  // Of a step's groups of 16 positions: key scale, log2 and inverse of the
  // value scale. Four steps deep: a buffer is written again when the keys
  // of the step two later are in use, which the softmax of this one precedes.
  float scales[4][8][4];
  uint32_t tmem;
  int abort, last, place;
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

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// A row's scores (128 TMEM columns from s_col) to P in their place, 32 at a
// time: t = log2 of a weight over the value scale, P = 2^(t - m) as f16 (and
// its remainder where LOW: 16 columns of each in turn), `sum` of P over the value
// scales. When a t passes m by kRaise (a vote of the warp: its rows share the
// branch) m becomes a whole number near the largest, so that what is scaled by
// the difference, the sum, O and this row's earlier P, keeps its bits (of P
// those from 2^-32 of the new largest on, f16's last place).
// Positions from `limit` on get no weight.
template <int HD, bool MASK, bool LOW>
__device__ __forceinline__ void tile_weights(uint32_t s_col, uint32_t o_col, bool scale_o, const float (*scales)[4],
                                             float factor, int key0, int limit, float& m, float2& sum, float& carry) {
  float2 part[2] = {sum, make_float2(0.0f, 0.0f)};
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    uint32_t r[32];
    tmem_ld<32>(s_col + 32 * b, r);
    tmem_wait_ld();
    float2 x[16];
    float top[4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float2 sc = *(const float2*)scales[2 * b + h];
      const float f = factor * sc.x;
      const float2 f2 = make_float2(f, f), d2 = make_float2(sc.y, sc.y);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        float2 t = fma2(make_float2(__uint_as_float(r[16 * h + 2 * k]), __uint_as_float(r[16 * h + 2 * k + 1])), f2, d2);
        if (MASK) {
          const int key = key0 + 32 * b + 16 * h + 2 * k;
          if (key >= limit) t.x = -INFINITY;
          if (key + 1 >= limit) t.y = -INFINITY;
        }
        x[8 * h + k] = t;
        const float y = fmaxf(t.x, t.y);
        top[k & 3] = h == 0 && k < 4 ? y : fmaxf(top[k & 3], y);
      }
    }
    const float most = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
    if (__any_sync(0xffffffffu, most > m + kRaise)) {
      // Stores to TMEM are asynchronous: the P of the blocks before, and O
      // where one of them raised m too, are read back below.
      tmem_wait_st();
      float alpha = 1.0f;
      if (most > m + kRaise) {
        const float to = floorf(most) - kBelow;
        alpha = exp2_fast(m - to);
        m = to;
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) part[i] = make_float2(part[i].x * alpha, part[i].y * alpha);
      carry *= alpha;
      // P is scaled in f32: alpha falls below f16 (2^-25 and less) where P
      // times alpha need not.
#pragma unroll 1
      for (int c = 0; c < (LOW ? 32 : 16) * b; c += 16) {
        uint32_t p[16];
        tmem_ld<16>(s_col + c, p);
        tmem_wait_ld();
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const float2 f = __half22float2(*(const __half2*)&p[k]);
          p[k] = pack_f16(f.x * alpha, f.y * alpha);
        }
        tmem_st16(s_col + c, p);
      }
#pragma unroll 1
      for (int c = 0; c < (scale_o ? HD : 0); c += 16) {
        uint32_t p[16];
        tmem_ld<16>(o_col + c, p);
        tmem_wait_ld();
#pragma unroll
        for (int k = 0; k < 16; ++k) p[k] = __float_as_uint(__uint_as_float(p[k]) * alpha);
        tmem_st16(o_col + c, p);
      }
    }
    uint32_t out[32];
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const float iv = scales[2 * b + (k >> 3)][2];
      float2 e = make_float2(exp2_fast(x[k].x - m), exp2_fast(x[k].y - m));
      part[k & 1] = fma2(e, make_float2(iv, iv), part[k & 1]);
      const __half2 p = __floats2half2_rn(e.x, e.y);
      out[k] = *(const uint32_t*)&p;
      if (LOW) {
        const float2 low = sub2(e, __half22float2(p));
        out[16 + k] = pack_f16(low.x, low.y);
      }
    }
    // The sums are due here: put off, they would keep every weight alive.
    asm volatile("" : "+f"(part[0].x), "+f"(part[0].y), "+f"(part[1].x), "+f"(part[1].y));
    if (LOW) tmem_st32(s_col + 32 * b, out);
    else tmem_st16(s_col + 16 * b, out);
  }
  sum = make_float2(part[0].x + part[1].x, part[0].y + part[1].y);
}

template <int HD, int TYPE, int QT>
constexpr int prompt_smem() {
  using Shape = PromptShape<HD, TYPE, QT>;
  return 1024 + (QT * (Shape::LOW ? 2 : 1) + Shape::KS + Shape::VS) * Shape::TILE + (int)sizeof(PromptSmem);
}

template <int HD, int TYPE, int QT>
__global__ void __launch_bounds__(PromptShape<HD, TYPE, QT>::THREADS, PromptShape<HD, TYPE, QT>::BLOCKS)
    k_kv_prompt(const __grid_constant__ KvView kv, const __grid_constant__ KvRuns runs,
                const __grid_constant__ KvAttendArgs a, int vec, int vec_out, void* workspace, size_t aside_at,
                int places, int* status) {
  using Shape = PromptShape<HD, TYPE, QT>;
  constexpr bool LOW = Shape::LOW, LOWP = TYPE != kKvBF16;
  constexpr int TILE = Shape::TILE, KS = Shape::KS, VS = Shape::VS, QB = (LOW ? 2 : 1) * TILE;
  constexpr int COLS = QT * kTile;
  // Steps whose values are summed in one go: f32 rows add O up in the
  // workspace (in a place that the block takes for its time; 32 columns of a
  // warp side by side) and begin anew.
  constexpr int CHAIN = LOW ? kKvChain / kTile : 1 << 30;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* base = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* q_s = base;                  // [QT][value, remainder]
  uint8_t* k_s = q_s + QT * QB;         // [KS]
  uint8_t* v_s = k_s + KS * TILE;       // [VS]
  PromptSmem* S = (PromptSmem*)(v_s + VS * TILE);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int MMA_WARP = 4 + 4 * QT;
  const int head = blockIdx.y, g = a.heads / kv.kv_heads, P = kv.page;

  KvRun run;
  int chunk, split;
  // The last tiles of a causal prompt see most: they start first.
  const int block = gridDim.x - 1 - blockIdx.x;
  find_run(runs, block, 1, 1, run, chunk, split);
  const int cols = run.count * g, c0 = chunk * COLS;
  const int groups = QT == 2 && c0 + kTile < cols ? 2 : 1;  // tiles with columns
  const int last_row = (min(cols, c0 + COLS) - 1) / g;
  const int kend = a.causal ? min(run.len, run.first + last_row + 1) : run.len;
  const int tiles = (kend + kTile - 1) / kTile, per = (tiles + run.splits - 1) / run.splits;
  const int t0 = min(tiles, split * per), nt = min(tiles, t0 + per) - t0;
  const int full = run.len & ~(P - 1);  // positions in full pages
  volatile int* abort = &S->abort;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&S->kfull[i], kConvThreads);
      mbar_init(&S->kempty[i], 1);
      mbar_init(&S->vfull[i], kConvThreads);
      mbar_init(&S->vempty[i], 1);
      mbar_init(&S->sfull[i], 1);
      mbar_init(&S->pfull[i], 128);
    }
    mbar_init(&S->qfull, QT * 128);
    mbar_init(&S->done, 1);
    S->abort = 0;
    S->place = -1;
    if (LOW && nt > CHAIN) {
      // As many places as blocks run at once: one is free.
      unsigned* flags = (unsigned*)workspace + kKvCounters;
      int at = (int)(blockIdx.x + blockIdx.y * gridDim.x) % places;
      for (int i = 0; i < 1 << 20 && S->place < 0; ++i) {
        if (atomicExch(flags + at, 1u) == 0) S->place = at;
        at = at + 1 == places ? 0 : at + 1;
      }
      if (S->place < 0) S->abort = 1;
      __threadfence();
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == MMA_WARP) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&S->tmem)),
                 "r"(Shape::COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = S->tmem;

  if (warp < 4) {
    // ---- codes to f16 ----
    const uint32_t bytes = (uint32_t)P * HD, page_blocks = (uint32_t)kv.layers * 2 * kv.kv_heads;
    const uint32_t page_bytes = page_blocks * bytes;
    const size_t head_block = (size_t)a.layer * 2 * kv.kv_heads + head;
    const uint8_t *codes_k = kv.codes + head_block * bytes, *codes_v = codes_k + (size_t)kv.kv_heads * bytes;
    const __half* open_k = kv.open + kv_block(kv, run.seq, a.layer, 0, head) * (size_t)bytes;
    const __half* open_v = open_k + (size_t)kv.kv_heads * bytes;
    const int* table = kv.table + (size_t)run.seq * kv.pages_per_seq;
    constexpr int KU = HD / 16;          // 16-code units of a key
    constexpr int N = kTile * KU / 128;  // units a thread takes of a step's keys (of its values as many)
    // Keys: unit i of a thread is row key_row(i) and values 16 key_unit(i) ..
    // of it; eight lanes take eight rows, so that their stores spread over
    // the banks. Values: pair val_pair(i) of positions and values 8
    // val_unit(i) .. of both, four pairs and two units in eight lanes.
    const int kr0 = warp * 8 + (lane & 7), ku0 = lane >> 3;
    const int vr0 = warp * 4 + (lane & 3), vu0 = lane >> 2;
    constexpr int KSTEP = KU / 4, VSTEP = HD / 64;
    auto key_row = [&](int i) { return kr0 + i / KSTEP * 32; };
    auto key_unit = [&](int i) { return ku0 + i % KSTEP * 4; };
    auto val_pair = [&](int i) { return vr0 + i / VSTEP * 16; };
    auto val_unit = [&](int i) { return vu0 + i % VSTEP * 8; };
    // Lanes 0-7: the page of each group of 16 positions of a step, or -1
    // (not in a full page, or past the end).
    auto pages_of = [&](int step) {
      const int pos = step * kTile + 16 * (lane & 7);
      return pos < kend && pos < full ? table[pos >> kv.page_shift] : -1;
    };
    uint4 kc[N], vc[N];
    const uint4 none = make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);
    auto load_keys = [&](int step, int pg) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int r = key_row(i), page = __shfl_sync(0xffffffffu, pg, r >> 4);
        const uint32_t at = (uint32_t)((step * kTile + r) & (P - 1)) * HD + 16 * key_unit(i);
        kc[i] = page < 0 ? none : __ldg((const uint4*)(codes_k + (size_t)(uint32_t)page * page_bytes + at));
      }
    };
    auto load_values = [&](int step, int pg) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int r = 2 * val_pair(i), page = __shfl_sync(0xffffffffu, pg, r >> 4);
        const uint32_t at = (uint32_t)((step * kTile + r) & (P - 1)) * HD + 16 * val_unit(i);
        vc[i] = page < 0 ? none : __ldg((const uint4*)(codes_v + (size_t)(uint32_t)page * page_bytes + at));
      }
    };
    // Lanes 0-7 of warp 0: the scales of a step's groups.
    auto scales_of = [&](int step, int pg) {
      float4 sc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (threadIdx.x < 8) {
        if (pg >= 0) {
          const float* x = kv.scales + (size_t)(uint32_t)pg * page_blocks + head_block;
          sc.x = x[0];
          sc.z = x[kv.kv_heads];
        } else if (step * kTile + 16 * (int)threadIdx.x < kend) {
          sc = make_float4(1.0f, 0.0f, 1.0f, 0.0f);  // f16
        }
      }
      return sc;
    };
    auto put_keys = [&](int j, float4 sc) -> bool {
      const int step = t0 + j;
      const bool tail = (step + 1) * kTile > full && full < kend;  // some of it in the open page
      if (!mbar_wait(&S->kempty[j % KS], (j / KS & 1) ^ 1, abort)) return false;
      if (threadIdx.x < 8) {
        const float vs = sc.z;
        sc.y = vs > 0.0f ? __log2f(vs) : kZeroScaleLog2;
        sc.z = vs > 0.0f ? __fdividef(1.0f, vs) : 2147483648.0f;
        *(float4*)S->scales[j & 3][threadIdx.x] = sc;
      }
      uint8_t* kt = k_s + j % KS * TILE;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int r = key_row(i), u = key_unit(i), pos = step * kTile + r;
        uint4 x = make_uint4(codes_lo(kc[i].x), codes_hi(kc[i].x), codes_lo(kc[i].y), codes_hi(kc[i].y));
        uint4 y = make_uint4(codes_lo(kc[i].z), codes_hi(kc[i].z), codes_lo(kc[i].w), codes_hi(kc[i].w));
        if (tail && pos >= full && pos < kend) {
          const uint4* src = (const uint4*)(open_k + (size_t)(pos - full) * HD + 16 * u);
          x = src[0];
          y = src[1];
        }
        *(uint4*)(kt + tile_at(r, 2 * u)) = x;
        *(uint4*)(kt + tile_at(r, 2 * u + 1)) = y;
      }
      fence_async_smem();
      mbar_arrive(&S->kfull[j % KS]);
      return true;
    };
    auto put_values = [&](int j) -> bool {
      const int step = t0 + j;
      const bool tail = (step + 1) * kTile > full && full < kend;
      if (!mbar_wait(&S->vempty[j % VS], (j / VS & 1) ^ 1, abort)) return false;
      uint8_t* vt = v_s + j % VS * TILE;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int r = 2 * val_pair(i), u = val_unit(i), pos = step * kTile + r;
        uint4 x = make_uint4(codes_even(vc[i].x), codes_even(vc[i].y), codes_even(vc[i].z), codes_even(vc[i].w));
        uint4 y = make_uint4(codes_odd(vc[i].x), codes_odd(vc[i].y), codes_odd(vc[i].z), codes_odd(vc[i].w));
        if (tail && pos >= full && pos < kend) {
          // Pairs of the open page: words (position 0, position 1) of a value.
          const uint4* src = (const uint4*)(open_v + (size_t)(pos - full) * HD + 16 * u);
          const uint4 p = src[0], q = src[1];
          x = make_uint4(__byte_perm(p.x, p.y, 0x5410), __byte_perm(p.z, p.w, 0x5410), __byte_perm(q.x, q.y, 0x5410),
                         __byte_perm(q.z, q.w, 0x5410));
          y = make_uint4(__byte_perm(p.x, p.y, 0x7632), __byte_perm(p.z, p.w, 0x7632), __byte_perm(q.x, q.y, 0x7632),
                         __byte_perm(q.z, q.w, 0x7632));
        }
        *(uint4*)(vt + tile_at(r, u)) = x;
        *(uint4*)(vt + tile_at(r + 1, u)) = y;
      }
      fence_async_smem();
      mbar_arrive(&S->vfull[j % VS]);
      return true;
    };
    // Keys run a step ahead of values where they have two buffers: the next
    // step's scores come before this step's values are given back.
    constexpr int LEAD = KS - 1;
    int pgk = nt > 0 ? pages_of(t0) : -1, pgv = pgk;
    float4 sc = scales_of(t0, pgk);
    if (nt > 0) load_keys(t0, pgk);
    for (int i = 0; i < nt + LEAD; ++i) {
      const int jv = i - LEAD;  // values of step jv after keys of step i
      const int pgk_next = i + 1 < nt ? pages_of(t0 + i + 1) : -1;
      if (jv >= 0) load_values(t0 + jv, pgv);
      if (i < nt && !put_keys(i, sc)) break;
      pgv = LEAD ? pgk : pgk_next;
      pgk = pgk_next;
      if (i + 1 < nt) {
        load_keys(t0 + i + 1, pgk);
        sc = scales_of(t0 + i + 1, pgk);
      }
      if (jv >= 0 && !put_values(jv)) break;
    }
  } else if (warp == MMA_WARP) {
    if (lane == 0 && nt > 0) {
      const uint32_t qa = smem_u32(q_s), ka = smem_u32(k_s), va = smem_u32(v_s);
      auto scores = [&](int j, int t) {
        const uint32_t k = ka + j % KS * TILE, q = qa + t * QB;
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) {
          const uint32_t at = (i >> 2) * (kTile * 128) + (i & 3) * 32;
          const uint64_t b = smem_desc_sw128(k + at);
          mma_f16(tmem + t * kTile, smem_desc_sw128(q + at), b, idesc_f16n(kTile), i > 0 ? 1u : 0u);
          if (LOW) mma_f16(tmem + t * kTile, smem_desc_sw128(q + TILE + at), b, idesc_f16n(kTile), 1u);
        }
        mma_commit(&S->sfull[t]);
      };
      auto values = [&](int j, int t) {
        const uint32_t v = va + j % VS * TILE, o = tmem + Shape::COL_O + t * kTile;
#pragma unroll
        for (int i = 0; i < kTile / 16; ++i) {
          const uint64_t b = smem_desc_sw128_mn(v + i * 2048, kTile * 128);
          const uint32_t p = tmem + t * kTile + (LOWP ? 32 * (i >> 1) + 8 * (i & 1) : 8 * i);
          mma_f16_ts(o, p, b, idesc_f16n(HD, true), (j % CHAIN > 0 || i > 0) ? 1u : 0u);
          if (LOWP) mma_f16_ts(o, p + 16, b, idesc_f16n(HD, true), 1u);
        }
      };
      bool ok = mbar_wait(&S->qfull, 0, abort) && mbar_wait(&S->kfull[0], 0, abort);
      if (ok) {
        fence_after();
        for (int t = 0; t < groups; ++t) scores(0, t);
        mma_commit(&S->kempty[0]);
      }
      for (int j = 0; j < nt && ok; ++j) {
        if (!mbar_wait(&S->vfull[j % VS], j / VS & 1, abort)) break;
        for (int t = 0; t < groups && ok; ++t) {
          // A tile's P is ready; its product, then the next step's scores in
          // the same place.
          if (!mbar_wait(&S->pfull[t], j & 1, abort)) {
            ok = false;
            break;
          }
          fence_after();
          values(j, t);
          if (t == groups - 1) mma_commit(&S->vempty[j % VS]);
          if (j + 1 < nt) {
            if (t == 0 && !mbar_wait(&S->kfull[(j + 1) % KS], (j + 1) / KS & 1, abort)) {
              ok = false;
              break;
            }
            fence_after();
            scores(j + 1, t);
            if (t == groups - 1) mma_commit(&S->kempty[(j + 1) % KS]);
          }
        }
      }
      mma_commit(&S->done);
      const long long start = now_ns();
      while (!mbar_test(&S->done, 0) && now_ns() - start < TC_WAIT_NS) {
      }
    }
  } else {
    // ---- softmax ----
    const int t = (warp - 4) >> 2, q = (warp & 3) * 32 + lane, c = c0 + t * kTile + q;
    const bool live = c < cols;
    const uint32_t s_col = tmem + ((uint32_t)((warp & 3) * 32) << 16) + t * kTile;
    const uint32_t o_col = s_col - t * kTile + Shape::COL_O + t * kTile;
    const int limit = !live ? 0 : a.causal ? min(run.len, run.first + c / g + 1) : run.len;
    int low_limit = live ? limit : 0x7fffffff;  // of the warp's rows: below it no mask is needed
#pragma unroll
    for (int o = 16; o; o >>= 1) low_limit = min(low_limit, __shfl_xor_sync(0xffffffffu, low_limit, o));
    // The warp's 32 rows, each scaled into [1, 2) (its sign taken from the
    // scale, so that the largest product is the largest score), as f16 value
    // and remainder. Lanes share rows, so that loads are whole lines.
    float factor = 0.0f;
    {
      constexpr int RL = HD / 4, RW = 32 / RL;  // lanes a row, rows a turn
      const int lr = lane / RL, d = lane % RL * 4;
#pragma unroll 1
      for (int i0 = 0; i0 < 32; i0 += 8 * RW) {
        float v[8][4];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int cc = c - lane + i0 + i * RW + lr;
#pragma unroll
          for (int k = 0; k < 4; ++k) v[i][k] = 0.0f;
          if (cc < cols)
            kv_load4(a.q, (size_t)(run.row0 + cc / g) * a.q_stride + (size_t)(head * g + cc % g) * HD + d, a.type, vec, v[i]);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float top = fmaxf(fmaxf(fabsf(v[i][0]), fabsf(v[i][1])), fmaxf(fabsf(v[i][2]), fabsf(v[i][3])));
#pragma unroll
          for (int o = RL / 2; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          int e = 0;
          if (top > 0.0f && top <= 3.4e38f) e = max(-126, min(126, (int)((__float_as_uint(top) >> 23) & 255) - 127));
          float down = __uint_as_float((uint32_t)(127 - e) << 23);
          if (a.scale < 0.0f) down = -down;
          const float f = fabsf(a.scale) * 1.4426950408889634f * __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
          for (int z = 0; z < RW; ++z) {
            const float fz = __shfl_sync(0xffffffffu, f, z * RL);
            if (lane == i0 + i * RW + z) factor = fz;
          }
          const int r = (warp & 3) * 32 + i0 + i * RW + lr;
          const __half2 h0 = __floats2half2_rn(v[i][0] * down, v[i][1] * down);
          const __half2 h1 = __floats2half2_rn(v[i][2] * down, v[i][3] * down);
          uint8_t* to = q_s + t * QB + tile_at(r, d >> 3) + (d & 4) * 2;
          *(uint2*)to = make_uint2(*(const uint32_t*)&h0, *(const uint32_t*)&h1);
          if (LOW)
            *(uint2*)(to + TILE) = make_uint2(pack_f16(v[i][0] * down - __low2float(h0), v[i][1] * down - __high2float(h0)),
                                              pack_f16(v[i][2] * down - __low2float(h1), v[i][3] * down - __high2float(h1)));
        }
      }
    }
    fence_async_smem();
    mbar_arrive(&S->qfull);
    float m = kMInit, carry = 1.0f;  // carry: what O put aside is to be scaled by
    float2 l2 = make_float2(0.0f, 0.0f);
    bool ok = true, aside = false;
    float* part = (float*)workspace + kKvHead + ((size_t)head * gridDim.x + block) * COLS * (HD + 2);
    float* total = (float*)workspace + aside_at + ((size_t)max(S->place, 0) * COLS + t * kTile + (warp & 3) * 32) * HD + lane;
    // 32 values of O, with what was put aside of them.
    auto whole = [&](int b, uint32_t (&r)[32]) {
      tmem_ld<32>(o_col + 32 * b, r);
      if (LOW && aside) {
        float x[32];
#pragma unroll
        for (int k = 0; k < 32; ++k) x[k] = __ldcg(total + (32 * b + k) * 32);
        tmem_wait_ld();
#pragma unroll
        for (int k = 0; k < 32; ++k) r[k] = __float_as_uint(fmaf(x[k], carry, __uint_as_float(r[k])));
      } else {
        tmem_wait_ld();
      }
    };
    for (int j = 0; j < nt && t < groups; ++j) {
      const int key0 = (t0 + j) * kTile;
      // Warp-uniform waits: the TMEM loads and stores below are warp-wide.
      // The scores are ready, and the tile's products before them are done.
      if (!__all_sync(0xffffffffu, mbar_wait(&S->sfull[t], j & 1, abort))) {
        ok = false;
        break;
      }
      fence_after();
      if (LOW && j > 0 && j % CHAIN == 0) {
        const bool add = aside && __all_sync(0xffffffffu, carry == 1.0f);
#pragma unroll 1
        for (int b = 0; b < HD / 32; ++b) {
          uint32_t r[32];
          if (add) {
            tmem_ld<32>(o_col + 32 * b, r);
            tmem_wait_ld();
            // Nothing waits for these; the same thread reads them back.
#pragma unroll
            for (int k = 0; k < 32; ++k)
              asm volatile("red.relaxed.gpu.global.add.f32 [%0], %1;" ::"l"(total + (32 * b + k) * 32),
                           "f"(__uint_as_float(r[k]))
                           : "memory");
          } else {
            whole(b, r);
#pragma unroll
            for (int k = 0; k < 32; ++k) __stcg(total + (32 * b + k) * 32, __uint_as_float(r[k]));
          }
        }
        aside = true;
        carry = 1.0f;
      }
      const bool mask = key0 + kTile > low_limit;
      const float(*scales)[4] = S->scales[j & 3];
      if (mask) tile_weights<HD, true, LOWP>(s_col, o_col, j % CHAIN > 0, scales, factor, key0, limit, m, l2, carry);
      else tile_weights<HD, false, LOWP>(s_col, o_col, j % CHAIN > 0, scales, factor, key0, limit, m, l2, carry);
      tmem_wait_st();
      fence_before();
      mbar_arrive(&S->pfull[t]);
    }
    if (t < groups && ok && nt > 0) ok = __all_sync(0xffffffffu, mbar_wait(&S->done, 0, abort));
    if (t < groups && ok) {
      fence_after();
      const float l = l2.x + l2.y, inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll 1
      for (int b = 0; b < HD / 32; ++b) {
        uint32_t r[32];
        if (nt > 0) {
          whole(b, r);
        } else {
#pragma unroll
          for (int k = 0; k < 32; ++k) r[k] = 0;
        }
        if (!live) continue;
        if (run.splits == 1) {
          const size_t out_at = (size_t)(run.row0 + c / g) * a.out_stride + (size_t)(head * g + c % g) * HD;
#pragma unroll
          for (int k = 0; k < 32; k += 8) {
            float x[8];
#pragma unroll
            for (int z = 0; z < 8; ++z) x[z] = l == 0.0f ? 0.0f : __uint_as_float(r[k + z]) * inv;
            kv_store8(a.out, out_at + 32 * b + k, a.type, vec_out, x);
          }
        } else {
#pragma unroll
          for (int k = 0; k < 32; k += 4)
            *(uint4*)(part + (t * kTile + q) * HD + 32 * b + k) = make_uint4(r[k], r[k + 1], r[k + 2], r[k + 3]);
        }
      }
      if (run.splits > 1 && live) *(float2*)(part + COLS * HD + 2 * (t * kTile + q)) = make_float2(m, l);
    }
  }
  if (run.splits > 1 || S->place >= 0) __threadfence();
  fence_before();
  __syncthreads();
  if (warp == MMA_WARP) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Shape::COLS) : "memory");
  }
  if (threadIdx.x == 0 && S->abort) *(volatile int*)status = 1;
  if (threadIdx.x == 0 && S->place >= 0) atomicExch((unsigned*)workspace + kKvCounters + S->place, 0u);
  if (run.splits == 1) return;
  // The block that comes last of a tile's shares joins them, in their order.
  if (threadIdx.x == 0) {
    unsigned* counter = (unsigned*)workspace + ((size_t)head * gridDim.x + block - split) % kKvCounters;
    S->last = atomicInc(counter, run.splits - 1) == (unsigned)run.splits - 1;
  }
  __syncthreads();
  if (!S->last) return;
  __threadfence();
  const float* first = (const float*)workspace + kKvHead + ((size_t)head * gridDim.x + block - split) * COLS * (HD + 2);
  for (int x = 4 * threadIdx.x; x < COLS * HD; x += 4 * Shape::THREADS) {
    const int lc = x / HD, d = x % HD, c = c0 + lc;
    if (c >= cols) break;
    float sum = 0.0f;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    join_shares(first, (size_t)COLS * (HD + 2), x, COLS * HD + 2 * lc, run.splits, sum, v);
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    const float y[4] = {sum == 0.0f ? 0.0f : v.x * inv, sum == 0.0f ? 0.0f : v.y * inv, sum == 0.0f ? 0.0f : v.z * inv,
                        sum == 0.0f ? 0.0f : v.w * inv};
    kv_store4(a.out, (size_t)(run.row0 + c / g) * a.out_stride + (size_t)(head * g + c % g) * HD + d, a.type, vec_out, y);
  }
}

template <int HD, int TYPE, int QT>
cudaError_t prompt(const KvView& kv, const KvRuns& runs, const KvAttendArgs& a, const KvAttendPlan& p, int vec,
                   int vec_out, void* ws, int* status, cudaStream_t s) {
  constexpr int smem = prompt_smem<HD, TYPE, QT>();
  static_assert(smem <= 227 * 1024, "the tiles fit in shared memory");
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  static DeviceOnce once;
  e = once.run(dev, [] {
    return cudaFuncSetAttribute(k_kv_prompt<HD, TYPE, QT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  });
  if (e != cudaSuccess) return e;
  k_kv_prompt<HD, TYPE, QT><<<dim3(p.blocks, kv.kv_heads), PromptShape<HD, TYPE, QT>::THREADS, smem, s>>>(
      kv, runs, a, vec, vec_out, ws, p.aside, p.places, status);
  return cudaGetLastError();
}
template <int TYPE>
cudaError_t prompt(const KvView& kv, const KvRuns& runs, const KvAttendArgs& a, const KvAttendPlan& p, int vec,
                   int vec_out, void* ws, int* status, cudaStream_t s) {
  const bool two = p.cols == 2 * kTile;
  if (kv.hd == 128)
    return two ? prompt<128, TYPE, 2>(kv, runs, a, p, vec, vec_out, ws, status, s)
               : prompt<128, TYPE, 1>(kv, runs, a, p, vec, vec_out, ws, status, s);
  return two ? prompt<64, TYPE, 2>(kv, runs, a, p, vec, vec_out, ws, status, s)
             : prompt<64, TYPE, 1>(kv, runs, a, p, vec, vec_out, ws, status, s);
}

}  // namespace

// Two tiles a block while that leaves no SM idle (the two share the widened
// codes, and one's products hide the other's softmax); positions are cut into
// shares while blocks leave SMs idle. A share costs what 12 steps do to start
// and to join (measured: 7 streams of 300 to 2111 positions, 33 to 300 rows
// each, 53.5 us whole, 50 in shares of 9 steps, 63 of 6, 67 of 4).
KvAttendPlan plan_kv_prompt(const KvView& kv, KvRuns& runs, const KvAttendArgs& a) {
  KvAttendPlan p;
  const int g = a.heads / kv.kv_heads;
  int slots = current_sm_count();
  double tiles = 0, work = 0;
  int longest = 1;
  for (int pass = 0; pass < 2; ++pass) {
    p.cols = pass == 0 ? 2 * kTile : kTile;
    tiles = work = 0;
    for (int i = 0; i < runs.n; ++i) {
      const double t = (double)(((size_t)runs.run[i].count * g + p.cols - 1) / p.cols);
      const int steps = (runs.run[i].len + kTile - 1) / kTile;
      tiles += t;
      work += t * steps;
      longest = std::max(longest, steps);
    }
    tiles *= kv.kv_heads;
    work *= kv.kv_heads;
    if (tiles >= slots) break;
  }
  if (p.cols == kTile && !(a.type == kKvF32 && kv.hd == 128)) slots *= 2;  // two blocks an SM
  int share = longest;
  if (tiles < 2.0 * slots) {
    double best = (double)((int)((tiles + slots - 1) / slots)) * (longest + 12.0);
    for (int rounds = 1; rounds <= 2; ++rounds) {
      const double room = (double)rounds * slots - 0.5 * tiles;
      if (room <= 0) continue;
      const int c = std::max(2, (int)(work / room) + 1);
      if (c < longest && rounds * (c + 12.0) < best) {
        best = rounds * (c + 12.0);
        share = c;
      }
    }
  }
  const size_t bytes = (size_t)kv.kv_heads * p.cols * (kv.hd + 2) * 4;
  for (;; share = std::min(longest, 2 * share)) {
    p.blocks = 0;
    p.joins = false;
    for (int i = 0; i < runs.n; ++i) {
      KvRun& r = runs.run[i];
      r.block0 = p.blocks;
      r.splits = std::max(1, ((r.len + kTile - 1) / kTile + share - 1) / share);
      p.joins |= r.splits > 1;
      p.blocks += (int)(((size_t)r.count * g + p.cols - 1) / p.cols) * r.splits;
    }
    // The partial results of shares, then the sums that f32 rows put aside.
    const size_t partial = p.joins ? p.blocks * bytes : 0;
    p.aside = a.type == kKvF32 ? kKvHead + partial / 4 : 0;
    p.workspace = p.aside || p.joins ? kKvHead * 4 + partial : 0;
    p.places = std::min<int>(kKvPlaces, 2 * current_sm_count());  // at most two blocks run on an SM
    if (p.aside) p.workspace += (size_t)p.places * p.cols * kv.hd * 4;
    if (!p.joins || ((size_t)p.blocks * kv.kv_heads <= kKvCounters && p.workspace <= kKvWorkspace)) break;
  }
  return p;
}

cudaError_t launch_kv_prompt(const KvView& kv, const KvRuns& runs, const KvAttendArgs& a, const KvAttendPlan& p, void* ws,
                             int* status, cudaStream_t s) {
  if (p.blocks <= 0) return cudaSuccess;
  if (runs.row_seq || (p.workspace && !ws)) return cudaErrorInvalidValue;
  const size_t size = a.type == kKvF32 ? 4 : 2;
  const int vec = ((uintptr_t)a.q | a.q_stride * size) % 16 == 0, vec_out = ((uintptr_t)a.out | a.out_stride * size) % 16 == 0;
  if (a.type == kKvF32) return prompt<kKvF32>(kv, runs, a, p, vec, vec_out, ws, status, s);
  if (a.type == kKvF16) return prompt<kKvF16>(kv, runs, a, p, vec, vec_out, ws, status, s);
  return prompt<kKvBF16>(kv, runs, a, p, vec, vec_out, ws, status, s);
}

}  // namespace trit
