// Products of 8-bit floating point with block scales:
//   out[r][i] = sum over blocks b of 128 of  sx[r][b] sw[i / 128][b]  (x_b[r] . w_b[i])
// with x and w in e4m3. The dot products of a block run on the tensor cores
// (tcgen05 kind::f8f6f4, f32 accumulators in TMEM); the blocks' sums leave
// TMEM one after another, are scaled and added in f32 registers, since every
// block has scales of its own.
//
// Rows of x are the MMA's M (a TMEM lane each), so a thread's scale of x is one
// register a block and that of w the same for all its columns: one packed
// multiply-add for two sums. The two scales' product is an f32 of its own and has
// to be in range (looking at it, to take it apart where it is not, is a vote in
// the epilogue's chain: 13.5 -> 14.1 us for 64 rows of 16384 x 4096, 52.3 -> 53.7 for
// 1000 of 12288 x 4096). Warp roles:
//   warp 0     producer: a stage is 128 values of k of the tile's rows of x (a
//              tensor copy) and w (bulk copies: w is kept in units of 64 rows x
//              128 values as the MMA reads them, a unit's next ones behind it,
//              so that a tile of w is one run of memory);
//   warp 1     issues four MMAs (K = 32) a stage into one of the TMEM buffers;
//   warps 4..  epilogue: load a block's sums from TMEM, add them up, and write
//              the tile through shared memory in whole lines.
// Every wait is bounded in time and reports through a status word. A block
// takes tile after tile; where tiles are few, a cluster of up to eight blocks
// shares one, each with a part of k, and adds the parts up in order through
// distributed shared memory. Weights do not depend on the kernel in front, so a
// block has its first stages of them on their way while that one still runs.
//
// With CTAS = 2 a pair of blocks shares a tile of 256 x 256: each holds its own
// 128 rows of x and half of the tile's rows of w, and the first one's MMAs
// (cta_group::2) read both. An SM takes 64 bytes a clock from L2, 48 KB a block of
// k of a tile of 128 x 256 and 32 KB of the pair's. Where such tiles leave many
// rows or SMs unused, two blocks an SM take tiles of 128 x 128, one each: one
// copies and starts while the other ends (600 rows of 4096 x 4096: 23.4 us with
// one block an SM, 19.9 with two).
//
// Few rows are bound by the bytes of w: 151936 x 2048 and three rows 53 us (5.9
// TB/s), 16384 x 4096 and 64 f32 rows 17.1 us with their rounding (4.2 TB/s),
// 12288 x 2048 and one row 7.4 us, of which about 4 are a launch, the first copy
// and the join. Many rows: 1000 of 12288 x 4096 52 us (1.9 PFLOP/s, the tensor pipe
// busy half of the time), 8000 of them 370 to 450 us with the clocks that the
// power limit leaves (2.9 PFLOP/s with neither loads from TMEM nor additions).
// What holds them up is an epilogue warp's chain (wait, load, load, add) and the
// round trip of a TMEM buffer, of which 512 columns hold two of 256. Measured and
// left: tiles of 128 x 256 a block (55 us for the 1000 rows), MMAs and buffers of
// half the columns (68), 16 epilogue warps (64, for want of registers), the next
// block's first load ahead of the last additions (60), waits that poll (61), pairs of
// 256 x 128 two an SM (61; 8000 rows 424 beside 365).

#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "device.cuh"
#include "launch.cuh"
#include "rows.cuh"
#include "rows.h"
#include "tc.cuh"

namespace trit {
namespace {

constexpr int F8_K = 128;  // values (bytes) of k a stage: one swizzle line, one scale block
constexpr int F8_UNIT = 64, F8_UNIT_BYTES = F8_UNIT * F8_K;  // rows of a unit of w

// CTAS blocks a tile. AR rows of x are loaded a block (the MMA's other rows read what lies behind them,
// and nobody reads their sums); BN rows of w a tile. Up to 64 rows take MMAs of
// M = 64: under the power limit the arithmetic that nobody reads costs clocks
// (151936 x 2048, three rows, seconds on end: 60 us with M = 128, 57 so).
template <int CTAS, int AR, int BN, int BLOCKS_>
struct F8Shape {
  static constexpr int BR = BN / CTAS;  // rows of w a block holds
  static constexpr int STAGE = (AR + BR) * F8_K;
  static constexpr int COLUMN_WARPS = BN >= 128 && BLOCKS_ == 1 ? 2 : 1;  // epilogue warps that share a tile's columns
  static constexpr int CW = BN / COLUMN_WARPS;                // columns of each
  static constexpr int M = AR <= 64 ? 64 : 128;               // of the MMA
  static constexpr int LANES = M / 4;                         // rows in a quarter of TMEM: its first lanes
  static constexpr int ROW_WARPS = (AR + LANES - 1) / LANES;  // of the four quarters, those with rows
  // Epilogue warps read the quarter of TMEM that their number names; where one
  // quarter has all rows, warp 0 is the epilogue beside the two others.
  static constexpr bool LONE = ROW_WARPS == 1 && COLUMN_WARPS == 1;
  static constexpr int THREADS = LONE ? 96 : 128 + 128 * COLUMN_WARPS;
  static constexpr int LOADER = LONE ? 2 : 0, ISSUER = 1, EPILOGUE = LONE ? 0 : 4;
  static constexpr int BUFS = BN * 4 * BLOCKS_ > 512 ? 2 : 4;
  static constexpr int COLS = BUFS * BN;                      // of TMEM
  // Two blocks of 128 x 128 an SM: each takes one tile, so that its rows leave
  // through the stages' memory, which is free by then.
  static constexpr bool ONE_TILE = BN >= 128 && BLOCKS_ == 2;
  static constexpr int STAGING = ONE_TILE ? 0 : ROW_WARPS * COLUMN_WARPS * 4096;
  static_assert(STAGE % 1024 == 0, "swizzled rows begin at whole kilobytes");
  static constexpr int TAIL = (M - AR) * F8_K > STAGING ? (M - AR) * F8_K : STAGING;  // behind the stages
  static constexpr int BLOCKS = BLOCKS_;                      // an SM holds
  static constexpr int EPILOGUE_THREADS = LONE ? 32 : THREADS - 128;
  static constexpr int SCALES = LONE ? 0 : 2 * 16 * EPILOGUE_THREADS;  // of x, eight of each thread's row
  static constexpr int ROOM = 226 * 1024 / BLOCKS - 2048 - 1024 - TAIL - SCALES;  // (a block's own 1 KB, and its static memory)
  static constexpr int STAGES = ROOM / STAGE < 12 ? ROOM / STAGE : 12;
  static constexpr int SMEM = 1024 + STAGES * STAGE + TAIL + SCALES;
  // 128 sums and two loads a thread do not fit the block's even share of the
  // registers: the epilogue takes what the other roles do not need. The shares
  // add up to the launch's 384 threads x 168, or 256 x 128.
  static constexpr bool SPLITS = BLOCKS_ > 1;  // k may be split over a cluster
  static constexpr int LOAD = ONE_TILE || CTAS == 2 ? 16 : 32;  // columns a load from TMEM (as registers allow)
  static constexpr bool SPLIT = CW == 128;
  static constexpr int REGS = ONE_TILE ? 128 : 168, REGS_FEW = ONE_TILE ? 48 : 40, REGS_MANY = ONE_TILE ? 208 : 232;
  static_assert(!SPLIT || 128 * REGS_FEW + (THREADS - 128) * REGS_MANY == THREADS * REGS, "register shares");
};
struct F8Sync {
  uint64_t full[12], empty[12], tfull[4], tempty[4], drain;
  uint32_t tmem;
  int abort;
};

// One lane of the warp, in a form that the compiler knows to be one: the
// instructions behind it take uniform registers (0.30 -> 0.17 us a stage of
// small MMAs against `lane == 0`).
__device__ __forceinline__ bool elected() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}

template <int CTAS>
__device__ __forceinline__ void mma_f8(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (CTAS == 1)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
}
// The MMAs issued so far arrive at *bar once they are done; of a pair, at both
// blocks' (the same place in each).
template <int CTAS>
__device__ __forceinline__ void commit_f8(uint64_t* bar) {
  if constexpr (CTAS == 1)
    mma_commit(bar);
  else
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                     smem_u32(bar)),
                 "h"((uint16_t)3)
                 : "memory");
}
// The address of the pair's first block's copy of a shared variable.
__device__ __forceinline__ uint32_t first_of_pair(const void* p) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_u32(p)));
  return r;
}
// A tensor copy whose bytes count at the first block's barrier.
__device__ __forceinline__ void tma_load_pair(void* dst, const void* map, uint32_t bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4}], "
      "[%2];" ::"r"(smem_u32(dst)),
      "l"((uint64_t)map), "r"(bar), "r"(x), "r"(y)
      : "memory");
}
// Instruction descriptor of kind::f8f6f4: D f32 (bits 4-5 = 1), A and B e4m3
// (bits 7-9, 10-12 = 0), both K-major, N >> 3 at bit 17, M >> 4 at bit 24.
__host__ __device__ constexpr uint32_t idesc_f8(int m, int n) {
  return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// `bytes` consecutive bytes to shared memory.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// Tiles in groups of 8 row tiles, so that the tiles in work at a time share
// their rows of x and w in L2.
__device__ __forceinline__ void tile_place(uint32_t t, uint32_t row_tiles, uint32_t col_tiles, int* r, int* c) {
  const uint32_t group = t / (8 * col_tiles), rows = min(8u, row_tiles - group * 8), at = t - group * 8 * col_tiles;
  *r = (int)(group * 8 + at % rows);
  *c = (int)(at / rows);
}

// The scales of x of a row's blocks b to b + 3; those past the end are not used.
// (Not through the read-only path: the kernel before may write them while this
// one waits.)
__device__ __forceinline__ float4 scales4(const float* sx, int b, int blocks, bool live, bool vec) {
  float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (!live || b >= blocks) return v;
  if (vec) return *(const float4*)(sx + b);
  v.x = sx[b];
  if (b + 1 < blocks) v.y = sx[b + 1];
  if (b + 2 < blocks) v.z = sx[b + 2];
  if (b + 3 < blocks) v.w = sx[b + 3];
  return v;
}
// The same on their way to shared memory. Loads to registers four blocks ahead
// hold up a warp with many other loads all the same (64 rows of 16384 x 4096 15.3
// us, 14.6 so); the one warp of up to 16 rows is faster with them (three rows of
// 151936 x 2048 52.2 us, 53.8 so).
__device__ __forceinline__ void fetch_scales(float4* to, const float* sx, int b, int blocks, bool live, bool vec) {
  if (vec) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(to)), "l"(live && b < blocks ? sx + b : sx),
                 "r"(live && b < blocks ? 16 : 0)
                 : "memory");
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(to) + 4 * j),
                   "l"(live && b + j < blocks ? sx + b + j : sx), "r"(live && b + j < blocks ? 4 : 0)
                   : "memory");
  }
  asm volatile("cp.async.commit_group;" ::: "memory");
}

__device__ __forceinline__ uint32_t pack16(float a, float b, bool f16) {
  return f16 ? pack2<__half>(make_float2(a, b)) : pack2<__nv_bfloat16>(make_float2(a, b));
}

// A warp's rows (one in each of its first LANES lanes) x CW columns to out, in chunks of 128 bytes a
// row through 4 KB of shared memory of its own: 16-byte unit u of row r lies at
// u ^ (r % 8), as the tensor copies' 128-byte swizzle has it. Where out's rows
// begin and end at whole 16 bytes (a.tma), a chunk leaves by one tensor copy, which ends at
// out's last row and column by itself, and the warp goes on meanwhile.
template <int CW, int LANES>
__device__ __forceinline__ void store_tile(const float2 (&acc)[CW / 2], uint8_t* staging, const CUtensorMap& omap,
                                           const Fp8Args& a, int row0, int col0, int lane) {
  const int rows = min(LANES, a.m - row0);
  const bool f32 = a.type == kRowF32, f16 = a.type == kRowF16;
  const int size = f32 ? 4 : 2;
  uint8_t* const out = (uint8_t*)a.out + (size_t)row0 * a.out_stride * size;
  // The chunk before has left the staging memory.
  auto begin = [&]() {
    if (a.tma && lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    __syncwarp();
  };
  auto chunk = [&](int col) {
    if (a.tma) {
      fence_async_smem();
      __syncwarp();
      if (lane == 0 && col < a.n) {
        asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"((uint64_t)&omap),
                     "r"(smem_u32(staging)), "r"(col), "r"(row0)
                     : "memory");
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
      }
      return;
    }
    __syncwarp();
    // Plain stores, a row's word from each lane; eight rows' words are read
    // before the first is stored, and only whole words are (a branch a row for
    // what a word leaves over took 3 us more of 333 rows of 5001 x 2064 in f16).
    const int live = min(128 / size, a.n - col);
    const size_t pitch = a.out_stride * size;
    uint8_t* p = out + (size_t)col * size;
    const int odd0 = (int)((uintptr_t)p >> 1 & 1), odd_step = f32 ? 0 : (int)(a.out_stride & 1);
#pragma unroll 1
    for (int r0 = 0; r0 < rows; r0 += 8) {
      uint32_t w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = *(const uint32_t*)(staging + (r0 + j) * 128 + ((lane / 4 ^ j) << 4) + (lane & 3) * 4);
#pragma unroll
      for (int j = 0; j < 8; ++j, p += pitch) {
        // (A word of a row that starts on an odd place: see below.)
        const int e = f32 ? lane : 2 * lane - (odd0 ^ (odd_step & j));
        if (r0 + j < rows && e >= 0 && (f32 ? e : e + 1) < live) *(uint32_t*)(p + e * size) = w[j];
      }
    }
    // What whole words leave over of its row stores each lane.
    if (!f32 && lane < rows && live > 0) {
      const int odd = odd0 ^ (odd_step & lane);
      uint16_t* q = (uint16_t*)(out + ((size_t)lane * a.out_stride + col) * size);
      const auto word = [&](int i) { return *(const uint32_t*)(staging + lane * 128 + ((i / 4 ^ (lane & 7)) << 4) + (i & 3) * 4); };
      if (odd) q[0] = (uint16_t)(word(0) >> 16);
      if ((live ^ odd) & 1 && live > odd) q[live - 1] = (uint16_t)word(odd ? live / 2 % 32 : live / 2);
    }
    __syncwarp();
  };
  if (f32) {
#pragma unroll
    for (int c = 0; c < CW; c += 32) {
      begin();
#pragma unroll
      for (int u = 0; u < 8; ++u)
        *(float4*)(staging + lane * 128 + ((u ^ (lane & 7)) << 4)) =
            make_float4(acc[c / 2 + 2 * u].x, acc[c / 2 + 2 * u].y, acc[c / 2 + 2 * u + 1].x, acc[c / 2 + 2 * u + 1].y);
      chunk(col0 + c);
    }
  } else {
#pragma unroll
    for (int c = 0; c < CW; c += 64) {
      begin();
      // A row that starts between two words has its values one half further
      // on: word i holds values 2 i - 1 and 2 i, the first one the last value
      // and value 0.
      const bool odd = !a.tma && ((((uintptr_t)out >> 1) + (size_t)lane * a.out_stride + col0 + c) & 1);
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 v = acc[c / 2 + 4 * u + i];
          const float before = acc[c / 2 + (4 * u + i + 31) % 32].y;
          w[i] = odd ? pack16(before, v.x, f16) : pack16(v.x, v.y, f16);
        }
        *(uint4*)(staging + lane * 128 + ((u ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
      }
      chunk(col0 + c);
    }
  }
}

__device__ __forceinline__ int cluster_size() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
  return (int)r;
}
__device__ __forceinline__ int cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctaid.x;" : "=r"(r));
  return (int)r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// A split's sums in shared memory, [row][BN] f32, over the stages, which are
// all read by then: 16-byte unit u of row r lies at u ^ (r % 8).
template <int CW, int BN>
__device__ __forceinline__ void put_part(const float2 (&acc)[CW / 2], uint8_t* part, int row, int col0) {
#pragma unroll
  for (int u = 0; u < CW / 4; ++u)
    *(float4*)(part + (size_t)row * BN * 4 + (((col0 / 4 + u) ^ (row & 7)) << 4)) =
        make_float4(acc[2 * u].x, acc[2 * u].y, acc[2 * u + 1].x, acc[2 * u + 1].y);
}
// Each block of the cluster adds up its share of the tile, always from the
// first split to the last, and writes it out.
template <int BN>
__device__ __forceinline__ void join_parts(const uint8_t* part, const Fp8Args& a, int row0, int rows, int col0, int split,
                                           int splits) {
  const int units = rows * (BN / 4), u0 = units * split / splits, u1 = units * (split + 1) / splits;
  const bool f32 = a.type == kRowF32, f16 = a.type == kRowF16;
  const int size = f32 ? 4 : 2;
  const bool vec = (((uintptr_t)a.out | a.out_stride * size) & (4 * size - 1)) == 0;
  for (int i = u0 + (int)threadIdx.x; i < u1; i += (int)blockDim.x) {
    const int r = i / (BN / 4), u = i % (BN / 4), at = col0 + u * 4;
    const uint32_t mine = smem_u32(part) + r * BN * 4 + ((u ^ (r & 7)) << 4);
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int z = 0; z < splits; ++z) {
      uint32_t from;
      float w[4];
      asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(from) : "r"(mine), "r"(z));
      asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                   : "=f"(w[0]), "=f"(w[1]), "=f"(w[2]), "=f"(w[3])
                   : "r"(from)
                   : "memory");
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] += w[j];
    }
    uint8_t* p = (uint8_t*)a.out + ((size_t)(row0 + r) * a.out_stride + at) * size;
    if (vec && at + 4 <= a.n) {
      if (f32) *(float4*)p = make_float4(v[0], v[1], v[2], v[3]);
      else *(uint2*)p = make_uint2(pack16(v[0], v[1], f16), pack16(v[2], v[3], f16));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (at + j >= a.n) break;
        if (f32) ((float*)p)[j] = v[j];
        else ((uint16_t*)p)[j] = (uint16_t)pack16(v[j], 0.0f, f16);
      }
    }
  }
}

template <int CTAS, int AR, int BN, int BLOCKS>
__global__ void __launch_bounds__(F8Shape<CTAS, AR, BN, BLOCKS>::THREADS, BLOCKS)
    k_fp8(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap,
          const __grid_constant__ CUtensorMap omap, const __grid_constant__ Fp8Args a) {
  using S = F8Shape<CTAS, AR, BN, BLOCKS>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* base = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  __shared__ F8Sync sync;
  F8Sync* y = &sync;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t row_tiles = ((uint32_t)a.m + CTAS * 128 - 1) / (CTAS * 128), col_tiles = ((uint32_t)a.n + BN - 1) / BN, tiles = row_tiles * col_tiles;
  // The blocks of a cluster share a tile, each with a part of k.
  const int splits = S::SPLITS ? cluster_size() : 1, split = S::SPLITS ? cluster_rank() : 0;
  const int lo = S::SPLITS ? (int)((long long)a.blocks * split / splits) : 0;
  const int hi = S::SPLITS ? (int)((long long)a.blocks * (split + 1) / splits) : a.blocks;
  const int rank = CTAS == 2 ? cluster_rank() : 0;
  const uint32_t first = blockIdx.x / (splits * CTAS), step = gridDim.x / (splits * CTAS);
  volatile int* abort = &y->abort;

  if (threadIdx.x == 0) {
    for (int i = 0; i < S::STAGES; ++i) {
      mbar_init(&y->full[i], 1);
      mbar_init(&y->empty[i], 1);
    }
    for (int i = 0; i < S::BUFS; ++i) {
      mbar_init(&y->tfull[i], 1);
      mbar_init(&y->tempty[i], CTAS * S::ROW_WARPS * S::COLUMN_WARPS);
    }
    mbar_init(&y->drain, 1);
    y->abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == S::ISSUER) {
    if constexpr (CTAS == 1) {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&y->tmem)), "r"(S::COLS)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&y->tmem)), "r"(S::COLS)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
  }
  fence_before();
  __syncthreads();
  if constexpr (CTAS == 2) cluster_sync();
  fence_after();
  const uint32_t tmem = y->tmem;
  let_next_start();

  if (S::LONE ? warp != 0 : warp < 4) {
    if constexpr (S::SPLIT) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::REGS_FEW));
    if (warp == S::LOADER && elected()) {
      uint32_t it = 0;
      bool ok = true;
      // What does not depend on the kernel before, the first stages' weights,
      // is on its way before that kernel has ended.
      uint32_t early = 0;
      for (uint32_t t = first; t < tiles && ok; t += step) {
        int r, c;
        tile_place(t, row_tiles, col_tiles, &r, &c);
        // The tile's units of w; of a pair, each block has half of them.
        const int left = (a.n + F8_UNIT - 1) / F8_UNIT - c * (BN / F8_UNIT);
        const int all = min(BN / F8_UNIT, left), units = min(S::BR / F8_UNIT, left - rank * (S::BR / F8_UNIT));
        const size_t unit0 = ((size_t)c * (BN / F8_UNIT) + rank * (S::BR / F8_UNIT)) * a.blocks;
        auto weights = [&](int b, uint32_t i) {
          uint8_t* to = base + i * S::STAGE + AR * F8_K;
          if (rank == 0) mbar_expect_tx(&y->full[i], CTAS * AR * F8_K + all * F8_UNIT_BYTES);
          for (int z = 0; z < units; ++z) {
            const size_t unit = unit0 + (size_t)z * a.blocks + b;
            if constexpr (CTAS == 1)
              bulk_load(to + z * F8_UNIT_BYTES, a.w + unit * F8_UNIT_BYTES, F8_UNIT_BYTES, &y->full[i]);
            else
              tma_load_pair(to + z * F8_UNIT_BYTES, &wmap, first_of_pair(&y->full[i]), 0, (int)unit * F8_UNIT);
          }
        };
        if (it == 0) {
          for (; early < S::STAGES && lo + (int)early < hi; ++early) weights(lo + early, early);
          after_kernel_before();
        }
        for (int b = lo; b < hi; ++b, ++it) {
          const uint32_t i = it % S::STAGES;
          if (it >= early) {
            if (!mbar_wait(&y->empty[i], ((it / S::STAGES) & 1) ^ 1, abort)) {
              ok = false;
              break;
            }
            weights(b, i);
          }
          if constexpr (CTAS == 1)
            tma_load_2d(base + i * S::STAGE, &xmap, &y->full[i], b * F8_K, r * 128);
          else
            tma_load_pair(base + i * S::STAGE, &xmap, first_of_pair(&y->full[i]), b * F8_K, (r * 2 + rank) * 128);
        }
      }
      if (!ok) {
        // Let the copies in flight land before the block's memory is released
        // (a stage whose rows were not asked for any more does not fill; a pair's
        // second block has no barrier to ask: a copy waits for nothing, 20 ms are ample).
        const long long t0 = now_ns();
        const uint32_t end = max(it, early);
        for (uint32_t z = end > S::STAGES ? end - S::STAGES : 0; z < end; ++z)
          while ((rank || !mbar_test(&y->full[z % S::STAGES], (z / S::STAGES) & 1)) && now_ns() - t0 < (rank ? 20000000ll : TC_WAIT_NS)) {
          }
      }
      if constexpr (CTAS == 2) {
        // The first block's MMAs arrive at both blocks' barriers. A barrier of this
        // block says nothing about the other's copy, so each block sees its own
        // last arrivals before it ends: one that is still on its way would land in
        // memory that belongs to the next block by then.
        for (uint32_t z = it > S::STAGES ? it - S::STAGES : 0; z < it && ok; ++z)
          ok = mbar_wait(&y->empty[z % S::STAGES], (z / S::STAGES) & 1, abort);
        const long long t0 = now_ns();
        while (!mbar_test(&y->drain, 0) && now_ns() - t0 < TC_WAIT_NS) {
        }
      }
    } else if (warp == S::ISSUER && rank == 0 && elected()) {
      after_kernel_before();  // however long that one takes, the limits of the waits run from its end
      const uint32_t s0 = smem_u32(base);
      uint32_t it = 0;
      bool ok = true;
      for (uint32_t t = first; t < tiles && ok; t += step) {
        for (int b = lo; b < hi; ++b, ++it) {
          const uint32_t i = it % S::STAGES, u = it % S::BUFS;
          if (!mbar_wait(&y->tempty[u], ((it / S::BUFS) & 1) ^ 1, abort) ||
              !mbar_wait(&y->full[i], (it / S::STAGES) & 1, abort)) {
            ok = false;
            break;
          }
          fence_after();
#pragma unroll
          for (int j = 0; j < F8_K / 32; ++j)
            mma_f8<CTAS>(tmem + u * BN, smem_desc_sw128(s0 + i * S::STAGE + j * 32),
                   smem_desc_sw128(s0 + i * S::STAGE + AR * F8_K + j * 32), idesc_f8(CTAS * S::M, BN), j ? 1u : 0u);
          commit_f8<CTAS>(&y->tfull[u]);
          commit_f8<CTAS>(&y->empty[i]);
        }
      }
      // Every MMA issued has finished once `drain` completes.
      commit_f8<CTAS>(&y->drain);
      const long long t0 = now_ns();
      while (!mbar_test(&y->drain, 0) && now_ns() - t0 < TC_WAIT_NS) {
      }
    }
  } else {
    if constexpr (S::SPLIT) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(S::REGS_MANY));
    const int quarter = warp & 3, part = (warp - S::EPILOGUE) >> 2;
    after_kernel_before();
    if (quarter < S::ROW_WARPS) {
      uint8_t* staging = base + (S::ONE_TILE ? 0 : S::STAGES * S::STAGE) + (part * S::ROW_WARPS + quarter) * 4096;
      const uint32_t tl = tmem + ((uint32_t)(quarter * 32) << 16) + part * S::CW;
      float4* scales = (float4*)(base + S::STAGES * S::STAGE + S::TAIL) + (threadIdx.x - S::EPILOGUE * 32);
      const bool vec = a.blocks % 4 == 0 && ((uintptr_t)a.x_scales & 15) == 0;
      uint32_t it = 0;
      bool ok = true;
      for (uint32_t t = first; t < tiles && ok; t += step) {
        int r, c;
        tile_place(t, row_tiles, col_tiles, &r, &c);
        const int row0 = (r * CTAS + rank) * 128 + quarter * S::LANES;  // m is at most 2^31 - 256
        const int col0 = c * BN + part * S::CW;
        const bool live = lane < S::LANES && row0 + lane < a.m;
        const float* sx = a.x_scales + (size_t)(live ? row0 + lane : 0) * a.blocks;
        // Every 32 blocks a lane loads the scale of w of one of them. A warp's
        // columns lie in one block of w; past n they read the last block's.
        const float* sw = a.w_scales + (size_t)min(col0 / 128, (a.n - 1) / 128) * a.blocks;
        float2 acc[S::CW / 2];
#pragma unroll
        for (int i = 0; i < S::CW / 2; ++i) acc[i] = make_float2(0.0f, 0.0f);
        float4 now = make_float4(0.0f, 0.0f, 0.0f, 0.0f), next = now;
        if constexpr (S::LONE) next = scales4(sx, lo & ~3, hi, live, vec);
        else fetch_scales(scales + (lo >> 2 & 1) * S::EPILOGUE_THREADS, sx, lo & ~3, hi, live, vec);
        float sws = lo + lane < hi ? __ldg(sw + lo + lane) : 0.0f;
        for (int b = lo; b < hi; ++b, ++it) {
          if ((b & 3) == 0 || b == lo) {
            if constexpr (S::LONE) {
              now = next;
              for (int i = 0; i < (b & 3); ++i) now = make_float4(now.y, now.z, now.w, 0.0f);
              next = scales4(sx, (b & ~3) + 4, hi, live, vec);
            } else {
              asm volatile("cp.async.wait_group 0;" ::: "memory");
              if ((b & ~3) + 4 < hi) fetch_scales(scales + ((b >> 2 & 1) ^ 1) * S::EPILOGUE_THREADS, sx, (b & ~3) + 4, hi, live, vec);
            }
          }
          if (b > lo && ((b - lo) & 31) == 0) sws = b + lane < hi ? __ldg(sw + b + lane) : 0.0f;
          float scale;
          if constexpr (S::LONE) {
            scale = now.x;
            now = make_float4(now.y, now.z, now.w, 0.0f);
          } else {
            scale = ((const float*)(scales + (b >> 2 & 1) * S::EPILOGUE_THREADS))[b & 3];
          }
          scale *= __shfl_sync(0xffffffffu, sws, (b - lo) & 31);
          const float2 s2 = make_float2(scale, scale);
          const uint32_t u = it % S::BUFS;
          if (!__all_sync(0xffffffffu, mbar_wait(&y->tfull[u], (it / S::BUFS) & 1, abort))) {
            ok = false;
            break;
          }
          fence_after();
          // The next columns are on the way while these are added.
          const uint32_t from = tl + u * BN;
          uint32_t v[2][S::LOAD];
          tmem_ld<S::LOAD>(from, v[0]);
#pragma unroll
          for (int q = 0; q < S::CW / S::LOAD; ++q) {
            tmem_wait_ld();
            if (q + 1 < S::CW / S::LOAD) {
              tmem_ld<S::LOAD>(from + (q + 1) * S::LOAD, v[(q + 1) & 1]);
            } else {
              fence_before();
              if (lane == 0) {
                // (No memory is handed over, so the default scope will do across the
                // pair too: an arrival with .release.cluster took it from 428 to 780 us.)
                if constexpr (CTAS == 1) mbar_arrive(&y->tempty[u]);
                else asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(first_of_pair(&y->tempty[u])) : "memory");
              }
            }
#pragma unroll
            for (int i = 0; i < S::LOAD / 2; ++i) {
              float2& sum = acc[q * (S::LOAD / 2) + i];
              sum = fma2(make_float2(__uint_as_float(v[q & 1][2 * i]), __uint_as_float(v[q & 1][2 * i + 1])), s2, sum);
            }
          }
        }
        if (S::SPLITS && splits > 1) {
          if (lane < S::LANES) put_part<S::CW, BN>(acc, base, quarter * S::LANES + lane, part * S::CW);
        } else if (ok && row0 < a.m) store_tile<S::CW, S::LANES>(acc, staging, omap, a, row0, col0, lane);
      }
      // Copies to and from shared memory have ended before it is given back.
      asm volatile("cp.async.wait_all;" ::: "memory");
      if (a.tma && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
  }
  fence_before();
  __syncthreads();
  if (S::SPLITS && splits > 1) {
    cluster_sync();
    int r, c;
    tile_place(first, row_tiles, col_tiles, &r, &c);
    join_parts<BN>(base, a, r * 128, min(AR, a.m - r * 128), c * BN, split, splits);
    cluster_sync();  // nobody leaves while others read its part
  }
  // A pair ends together: the first block's MMAs read the second's memory, whose epilogue arrives at the first's barriers.
  if constexpr (CTAS == 2) cluster_sync();
  if (warp == S::ISSUER) {
    fence_after();
    if constexpr (CTAS == 1)
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::COLS) : "memory");
    else
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::COLS) : "memory");
  }
  if (threadIdx.x == 0 && y->abort) *(volatile int*)a.status = 1;
}

template <int CTAS, int AR, int BN, int BLOCKS>
cudaError_t run(const TcMap& x, const TcMap& w, const TcMap& out, const Fp8Args& a, int splits, cudaStream_t s) {
  using S = F8Shape<CTAS, AR, BN, BLOCKS>;
  static_assert(S::STAGES >= 3 && S::STAGES <= 12 && S::SMEM + (int)sizeof(F8Sync) <= 227 * 1024, "shared memory");
  static_assert(AR * BN * 4 <= S::STAGES * S::STAGE, "a split's sums");
  static_assert(S::COLS * S::BLOCKS <= 512 && (S::COLS & (S::COLS - 1)) == 0, "TMEM");
  static_assert(S::CW <= 128 && S::CW % 64 == 0 && BN % F8_UNIT == 0, "columns of an epilogue warp");
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  static DeviceOnce once;
  e = once.run(dev, [] {
    cudaFuncAttributes f;
    cudaError_t r = cudaFuncGetAttributes(&f, k_fp8<CTAS, AR, BN, BLOCKS>);
    // A launch with fewer registers than the shares add up to would wait for them without end.
    if (r == cudaSuccess && S::SPLIT && f.numRegs != S::REGS) r = cudaErrorInvalidKernelImage;
    if (r != cudaSuccess) return r;
    return cudaFuncSetAttribute(k_fp8<CTAS, AR, BN, BLOCKS>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
  });
  if (e != cudaSuccess) return e;
  const long long tiles = (a.m + CTAS * 128 - 1LL) / (CTAS * 128) * ((a.n + BN - 1) / BN);
  if (tiles >> 30) return cudaErrorInvalidValue;  // an output of 2^42 values or more
  // Blocks take tile after tile; those of a cluster have one.
  const long long grid = splits > 1 || S::ONE_TILE ? tiles * splits : CTAS * std::min<long long>(tiles, current_sm_count() * BLOCKS / CTAS);
  return launch_early(k_fp8<CTAS, AR, BN, BLOCKS>, dim3((unsigned)grid), dim3(S::THREADS), S::SMEM, s,
                      (unsigned)(splits * CTAS), *(const CUtensorMap*)&x, *(const CUtensorMap*)&w, *(const CUtensorMap*)&out, a);
}

// Rows of bytes to the units that k_fp8 reads: [n / 64][k / 128][64 rows][128
// bytes], 16-byte chunk c of row r at c ^ (r % 8), zero past either end. One
// thread a chunk.
__global__ void __launch_bounds__(256) k_fp8_pack(const uint8_t* codes, size_t n, size_t k, uint8_t* w) {
  const size_t blocks = (k + F8_K - 1) / F8_K, chunks = (n + F8_UNIT - 1) / F8_UNIT * blocks * (F8_UNIT_BYTES / 16);
  for (size_t i = blockIdx.x * (size_t)256 + threadIdx.x; i < chunks; i += (size_t)gridDim.x * 256) {
    const size_t unit = i / (F8_UNIT_BYTES / 16);
    const int at = (int)(i % (F8_UNIT_BYTES / 16)), r = at / 8, c = (at % 8) ^ (r & 7);
    const size_t row = unit / blocks * F8_UNIT + r, col = unit % blocks * F8_K + c * 16;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (row < n && col < k) v = *(const uint4*)(codes + row * k + col);  // k is a multiple of 16
    ((uint4*)w)[i] = v;
  }
}

}  // namespace

int fp8_row_box(int m) { return m <= 16 ? 16 : m <= 64 ? 64 : 128; }
int fp8_out_box(int m) { return m <= 64 ? 16 : 32; }
size_t fp8_packed_bytes(size_t n, size_t k) {
  return (n + F8_UNIT - 1) / F8_UNIT * ((k + F8_K - 1) / F8_K) * F8_UNIT_BYTES;
}
cudaError_t launch_fp8_pack(const uint8_t* codes, size_t n, size_t k, uint8_t* w, cudaStream_t s) {
  k_fp8_pack<<<148 * 8, 256, 0, s>>>(codes, n, k, w);
  return cudaGetLastError();
}

cudaError_t launch_fp8(const TcMap& x, const TcMap& w, const TcMap& out, const Fp8Args& a, cudaStream_t s) {
  if (a.m <= 0) return cudaSuccess;
  const long long sms = current_sm_count();
  const auto tiles = [&](int bn) { return (a.m + 127LL) / 128 * ((a.n + bn - 1) / bn); };
  // As many blocks of a cluster as there is room for beside each other, with at
  // least two blocks of k, six where eight share (4096 x 4096, three rows: a
  // cluster of 1 12.7 us, 2 8.9, 4 6.8, 8 7.7; 2048 x 6144: 16.8, 10.7, 7.3, 5.8;
  // 12288 x 2048: 7.6, 7.4, 12.5, 19.2). The parts of the chip that a cluster stays
  // within hold no whole number of large ones: of 296 blocks 70 clusters of four
  // and 33 of eight (k = 6400, 40 rows: 70 tiles in four 15.1 us, 72 23.3).
  const auto splits = [&](long long tiles, long long room) {
    int z = 1;
    while (z < 8 && tiles * z * 2 <= room * (z == 1 ? 16 : z == 2 ? 15 : 14) / 16 && a.blocks / (z * 2) >= (z < 4 ? 2 : 6)) z *= 2;
    return z;
  };
  const int box = fp8_row_box(a.m);
  // Few rows: four blocks an SM, of three warps, so that the next call's blocks
  // find room (two an SM: 151936 x 2048 57.1 us, 32768 x 8192 46.7; four: 53.6, 43.1).
  if (box == 16) return run<1, 16, 64, 4>(x, w, out, a, splits(tiles(64), 4 * sms), s);
  // More rows: 128 columns, one block or two an SM (these have fewer warps and
  // stages each; one copies while the other ends), or tiles of 256 x 256 by pairs.
  // What each takes, in us: a call, whole turns of the SMs, and a turn's blocks of
  // k, as measured. us by one, two and pairs (8-bit rows, bf16 out, replays of a
  // recorded graph), 64 rows: 16384 x 4096 13.4, 15.9; 151936 x 2048 56, 60; 32768 x
  // 8192 46, 44; 8192 x 4096 12.1, 10.6 (k in four). More: 333 rows of 5001 x 2064
  // 9.4, 13.5, 13.3; 128 of 12288 x 2048 9.0, 12.4, 11.9; 512 of 2048 x 6144 17.5,
  // 14.0 (k in four), 24.7; 300 of 20000 x 4096 44, 40, 49; 1140 of 14746 x 528 27,
  // 31, 25; 1000 of 12288 x 4096 69, 61, 52 to 57; 8000 of them 549, 474, 385. The
  // constants are from before the scales of x went through shared memory, which
  // took up to 15 % off one and pairs; two are chosen a little too often since (600
  // of 4096 x 4096 23.4, 19.9, 18.7; 129 of 16384 x 4096 23.7, 21.2, 19.5).
  const auto us = [&](double call, double turn, double block, int blocks, long long work, long long room) {
    return call + (turn + block * blocks) * (double)((work + room - 1) / room);
  };
  const int z = splits(tiles(128), 2 * sms), part = (a.blocks + z - 1) / z;
  if (box == 64) {
    const double one = us(2.3, 0.0, 0.40, a.blocks, tiles(128), sms);
    const double two = us(z > 1 ? 2.2 : 1.0, 3.0, 0.62, part, tiles(128) * z, 2 * sms);
    if (one <= two) return run<1, 64, 128, 1>(x, w, out, a, 1, s);
    return run<1, 64, 128, 2>(x, w, out, a, z, s);
  }
  const double one = us(3.0, 1.0, 0.385, a.blocks, tiles(128), sms);
  const double two = us(z > 1 ? 4.0 : 1.0, 3.0, 0.58, part, tiles(128) * z, 2 * sms);
  const double pairs = us(4.0, 1.5, 0.545, a.blocks, (a.m + 255LL) / 256 * ((a.n + 255LL) / 256), std::max(1LL, sms / 2));
  if (one <= two && one <= pairs) return run<1, 128, 128, 1>(x, w, out, a, 1, s);
  if (two <= pairs) return run<1, 128, 128, 2>(x, w, out, a, z, s);
  return run<2, 128, 256, 1>(x, w, out, a, 1, s);
}

}  // namespace trit
