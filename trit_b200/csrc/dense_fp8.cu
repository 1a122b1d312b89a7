// Products of 8-bit floating point with block scales:
//   out[r][i] = sum over blocks b of 128 of  sx[r][b] sw[i / 128][b]  (x_b[r] . w_b[i])
// with x and w in e4m3. The dot products of a block run on the tensor cores
// (tcgen05 kind::f8f6f4, f32 accumulators in TMEM); the blocks' sums leave
// TMEM one after another, are scaled and added in f32 registers, since every
// block has scales of its own.
//
// Rows of x are the MMA's M (a TMEM lane each), so a thread's scale of x is one
// register a block and that of w the same for all its columns: one packed
// multiply-add for two sums. Warp roles:
//   warp 0     TMA producer: a stage is 128 values of k of the tile's rows of
//              x and w, with the 128-byte swizzle;
//   warp 1     issues four MMAs (K = 32) a stage into one of the TMEM buffers;
//   warps 4..  epilogue: load a block's sums from TMEM, add them up, and write
//              the tile through shared memory in whole lines.
// Every wait is bounded in time and reports through a status word.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "device.cuh"
#include "rows.h"
#include "tc.cuh"

namespace trit {
namespace {

constexpr int F8_K = 128;  // values (bytes) of k a stage: one swizzle line, one scale block

// AR rows of x are loaded (the MMA's other rows read what lies behind them,
// and nobody reads their sums); BN rows of w a tile.
template <int AR, int BN>
struct F8Shape {
  static constexpr int STAGE = (AR + BN) * F8_K;
  static constexpr int COLUMN_WARPS = BN >= 128 ? 2 : 1;      // epilogue warps that share a tile's columns
  static constexpr int CW = BN / COLUMN_WARPS;                // columns of each
  static constexpr int ROW_WARPS = (AR + 31) / 32;            // of the four TMEM quarters, those with rows
  static constexpr int THREADS = 128 + 128 * COLUMN_WARPS;
  static constexpr int BUFS = BN >= 256 ? 2 : 4;
  static constexpr int COLS = BUFS * BN;                      // of TMEM
  static constexpr int STAGING = ROW_WARPS * COLUMN_WARPS * 4096;
  static constexpr int TAIL = (128 - AR) * F8_K > STAGING ? (128 - AR) * F8_K : STAGING;  // behind the stages
  static constexpr int BLOCKS = BN >= 128 ? 1 : 2;            // an SM holds
  static constexpr int ROOM = (BLOCKS == 1 ? 226 : 113) * 1024 - 1024 - TAIL;
  static constexpr int STAGES = ROOM / STAGE < 12 ? ROOM / STAGE : 12;
  static constexpr int SMEM = 1024 + STAGES * STAGE + TAIL;
  // 128 sums and two loads of 32 a thread do not fit the block's even share of
  // the registers: the epilogue takes what the other roles do not need. The
  // shares add up to the launch's 384 threads x 168.
  static constexpr bool SPLIT = CW == 128;
  static constexpr int REGS = 168, REGS_FEW = 72, REGS_MANY = 216;
  static_assert(!SPLIT || (THREADS == 384 && 128 * REGS_FEW + 256 * REGS_MANY == THREADS * REGS), "register shares");
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

__device__ __forceinline__ void mma_f8(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
}
// Instruction descriptor of kind::f8f6f4: D f32 (bits 4-5 = 1), A and B e4m3
// (bits 7-9, 10-12 = 0), both K-major, N >> 3 at bit 17, M >> 4 at bit 24.
__host__ __device__ constexpr uint32_t idesc_f8(int m, int n) {
  return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// Tiles in groups of 8 row tiles, so that the tiles in work at a time share
// their rows of x and w in L2.
__device__ __forceinline__ void tile_place(long long t, int row_tiles, int col_tiles, int* r, int* c) {
  const long long group = t / (8LL * col_tiles);
  const int rows = min(8LL, row_tiles - group * 8);
  const long long at = t - group * 8 * col_tiles;
  *r = (int)(group * 8 + at % rows);
  *c = (int)(at / rows);
}

// The scales of x of four blocks of a row; those past the end are not used.
__device__ __forceinline__ float4 scales4(const float* sx, int b, int blocks, bool live, bool vec) {
  float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (!live || b >= blocks) return v;
  if (vec) return __ldg((const float4*)(sx + b));
  v.x = __ldg(sx + b);
  if (b + 1 < blocks) v.y = __ldg(sx + b + 1);
  if (b + 2 < blocks) v.z = __ldg(sx + b + 2);
  if (b + 3 < blocks) v.w = __ldg(sx + b + 3);
  return v;
}

__device__ __forceinline__ uint32_t pack2(float a, float b, bool f16) {
  if (f16) {
    const __half2 h = __floats2half2_rn(a, b);
    return *(const uint32_t*)&h;
  }
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *(const uint32_t*)&h;
}

// A warp's 32 rows (a lane each) x CW columns to out, through 4 KB of shared
// memory of its own: 16-byte unit u of row r lies at u ^ (r % 8).
template <int CW>
__device__ __forceinline__ void store_tile(const float2 (&acc)[CW / 2], uint8_t* staging, const Fp8Args& a, long long row0,
                                           int col0, int lane) {
  const int rows = (int)min(32LL, a.m - row0);
  const bool f32 = a.type == kRowF32, f16 = a.type == kRowF16;
  const int size = f32 ? 4 : 2;
  const bool vec = (((uintptr_t)a.out | a.out_stride * size) & 15) == 0;
  uint8_t* out = (uint8_t*)a.out + (size_t)row0 * a.out_stride * size;
  // A chunk is up to 128 bytes of every row.
  auto chunk = [&](int col, int units) {
    __syncwarp();
    if (vec) {
      const int u = lane % units, per = 32 / units, values = 16 / size;
      for (int r = lane / units; r < rows; r += per) {
        const uint4 v = *(const uint4*)(staging + r * 128 + ((u ^ (r & 7)) << 4));
        const int at = col + u * values;
        uint8_t* p = out + ((size_t)r * a.out_stride + at) * size;
        if (at + values <= a.n) {
          *(uint4*)p = v;
        } else {
          const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (f32 && i < 4 && at + i < a.n) ((uint32_t*)p)[i] = w[i & 3];
            if (!f32 && at + i < a.n) ((uint16_t*)p)[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
          }
        }
      }
    } else {
      const int values = units * 16 / size;
      for (int r = 0; r < rows; ++r) {
        for (int i = lane; i < values && col + i < a.n; i += 32) {
          const uint8_t* from = staging + r * 128 + (((i * size >> 4) ^ (r & 7)) << 4) + (i * size & 15);
          uint8_t* p = out + ((size_t)r * a.out_stride + col + i) * size;
          if (f32) *(uint32_t*)p = *(const uint32_t*)from;
          else *(uint16_t*)p = *(const uint16_t*)from;
        }
      }
    }
    __syncwarp();
  };
  if (f32) {
#pragma unroll
    for (int c = 0; c < CW; c += 32) {
#pragma unroll
      for (int u = 0; u < 8; ++u)
        *(float4*)(staging + lane * 128 + ((u ^ (lane & 7)) << 4)) =
            make_float4(acc[c / 2 + 2 * u].x, acc[c / 2 + 2 * u].y, acc[c / 2 + 2 * u + 1].x, acc[c / 2 + 2 * u + 1].y);
      chunk(col0 + c, 8);
    }
  } else {
    constexpr int CC = CW < 64 ? CW : 64;
#pragma unroll
    for (int c = 0; c < CW; c += CC) {
#pragma unroll
      for (int u = 0; u < CC / 8; ++u) {
        const float2* v = &acc[c / 2 + 4 * u];
        *(uint4*)(staging + lane * 128 + ((u ^ (lane & 7)) << 4)) =
            make_uint4(pack2(v[0].x, v[0].y, f16), pack2(v[1].x, v[1].y, f16), pack2(v[2].x, v[2].y, f16), pack2(v[3].x, v[3].y, f16));
      }
      chunk(col0 + c, CC / 8);
    }
  }
}

template <int AR, int BN>
__global__ void __launch_bounds__(F8Shape<AR, BN>::THREADS, F8Shape<AR, BN>::BLOCKS)
    k_fp8(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap, const __grid_constant__ Fp8Args a) {
  using S = F8Shape<AR, BN>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* base = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  __shared__ F8Sync sync;
  F8Sync* y = &sync;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row_tiles = (a.m + 127) / 128, col_tiles = (a.n + BN - 1) / BN;
  const long long tiles = (long long)row_tiles * col_tiles;
  volatile int* abort = &y->abort;

  if (threadIdx.x == 0) {
    for (int i = 0; i < S::STAGES; ++i) {
      mbar_init(&y->full[i], 1);
      mbar_init(&y->empty[i], 1);
    }
    for (int i = 0; i < S::BUFS; ++i) {
      mbar_init(&y->tfull[i], 1);
      mbar_init(&y->tempty[i], S::ROW_WARPS * S::COLUMN_WARPS);
    }
    mbar_init(&y->drain, 1);
    y->abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&y->tmem)), "r"(S::COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = y->tmem;

  if (warp < 4) {
    if constexpr (S::SPLIT) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::REGS_FEW));
    if (warp == 0 && elected()) {
      uint32_t it = 0;
      bool ok = true;
      for (long long t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
        int r, c;
        tile_place(t, row_tiles, col_tiles, &r, &c);
        for (int b = 0; b < a.blocks; ++b, ++it) {
          const uint32_t i = it % S::STAGES;
          if (!mbar_wait(&y->empty[i], ((it / S::STAGES) & 1) ^ 1, abort)) {
            ok = false;
            break;
          }
          uint8_t* to = base + i * S::STAGE;
          mbar_expect_tx(&y->full[i], S::STAGE);
          tma_load_2d(to, &xmap, &y->full[i], b * F8_K, r * 128);
          tma_load_2d(to + AR * F8_K, &wmap, &y->full[i], b * F8_K, c * BN);
        }
      }
      if (!ok) {
        // Let the copies in flight land before the block's memory is released.
        for (uint32_t z = it > S::STAGES ? it - S::STAGES : 0; z < it; ++z) {
          const long long t0 = now_ns();
          while (!mbar_test(&y->full[z % S::STAGES], (z / S::STAGES) & 1) && now_ns() - t0 < TC_WAIT_NS) {
          }
        }
      }
    } else if (warp == 1 && elected()) {
      const uint32_t s0 = smem_u32(base);
      uint32_t it = 0;
      bool ok = true;
      for (long long t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
        for (int b = 0; b < a.blocks; ++b, ++it) {
          const uint32_t i = it % S::STAGES, u = it % S::BUFS;
          if (!mbar_wait(&y->tempty[u], ((it / S::BUFS) & 1) ^ 1, abort) ||
              !mbar_wait(&y->full[i], (it / S::STAGES) & 1, abort)) {
            ok = false;
            break;
          }
          fence_after();
#pragma unroll
          for (int j = 0; j < F8_K / 32; ++j)
            mma_f8(tmem + u * BN, smem_desc_sw128(s0 + i * S::STAGE + j * 32),
                   smem_desc_sw128(s0 + i * S::STAGE + AR * F8_K + j * 32), idesc_f8(128, BN), j ? 1u : 0u);
          mma_commit(&y->tfull[u]);
          mma_commit(&y->empty[i]);
        }
      }
      // Every MMA issued has finished once `drain` completes.
      mma_commit(&y->drain);
      const long long t0 = now_ns();
      while (!mbar_test(&y->drain, 0) && now_ns() - t0 < TC_WAIT_NS) {
      }
    }
  } else {
    if constexpr (S::SPLIT) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(S::REGS_MANY));
    const int quarter = warp & 3, part = (warp - 4) >> 2;
    if (quarter < S::ROW_WARPS) {
      constexpr int LD = S::CW >= 64 ? 32 : 16;  // columns a load; the next ones are on the way while these are added
      uint8_t* staging = base + S::STAGES * S::STAGE + (part * S::ROW_WARPS + quarter) * 4096;
      const uint32_t tl = tmem + ((uint32_t)(quarter * 32) << 16) + part * S::CW;
      const bool vec = a.blocks % 4 == 0 && ((uintptr_t)a.x_scales & 15) == 0;
      uint32_t it = 0;
      bool ok = true;
      for (long long t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
        int r, c;
        tile_place(t, row_tiles, col_tiles, &r, &c);
        const long long row0 = (long long)r * 128 + quarter * 32;
        const int col0 = c * BN + part * S::CW;
        const bool live = row0 + lane < a.m;
        const float* sx = a.x_scales + (size_t)(live ? row0 + lane : 0) * a.blocks;
        // Every 32 blocks a lane loads the scale of w of one of them. A warp's
        // columns lie in one block of w; past n they read the last block's.
        const float* sw = a.w_scales + (size_t)min(col0 / 128, (a.n - 1) / 128) * a.blocks;
        float2 acc[S::CW / 2];
#pragma unroll
        for (int i = 0; i < S::CW / 2; ++i) acc[i] = make_float2(0.0f, 0.0f);
        float4 next = scales4(sx, 0, a.blocks, live, vec);
        float sws = 0.0f;
        for (int b0 = 0; b0 < a.blocks && ok; b0 += 4) {
          if ((b0 & 31) == 0) sws = b0 + lane < a.blocks ? __ldg(sw + b0 + lane) : 0.0f;
          const float4 now = next;
          next = scales4(sx, b0 + 4, a.blocks, live, vec);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (b0 + j >= a.blocks) break;
            const float xj = j == 0 ? now.x : j == 1 ? now.y : j == 2 ? now.z : now.w;
            const float scale = xj * __shfl_sync(0xffffffffu, sws, (b0 + j) & 31);
            const float2 s2 = make_float2(scale, scale);
            const uint32_t u = it % S::BUFS;
            if (!__all_sync(0xffffffffu, mbar_wait(&y->tfull[u], (it / S::BUFS) & 1, abort))) {
              ok = false;
              break;
            }
            ++it;
            fence_after();
            const uint32_t from = tl + u * BN;
            uint32_t v[2][LD];
            tmem_ld<LD>(from, v[0]);
#pragma unroll
            for (int q = 0; q < S::CW / LD; ++q) {
              tmem_wait_ld();
              if (q + 1 < S::CW / LD) {
                tmem_ld<LD>(from + (q + 1) * LD, v[(q + 1) & 1]);
              } else {
                fence_before();
                if (lane == 0) mbar_arrive(&y->tempty[u]);
              }
#pragma unroll
              for (int i = 0; i < LD / 2; ++i)
                acc[q * (LD / 2) + i] = fma2(make_float2(__uint_as_float(v[q & 1][2 * i]), __uint_as_float(v[q & 1][2 * i + 1])),
                                             s2, acc[q * (LD / 2) + i]);
            }
          }
        }
        if (ok && row0 < a.m) store_tile<S::CW>(acc, staging, a, row0, col0, lane);
      }
    }
  }
  fence_before();
  __syncthreads();
  if (warp == 1) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::COLS) : "memory");
  }
  if (threadIdx.x == 0 && y->abort) *(volatile int*)a.status = 1;
}

template <int AR, int BN>
cudaError_t run(const TcMap* w, const TcMap& x, const Fp8Args& a, cudaStream_t s) {
  using S = F8Shape<AR, BN>;
  static_assert(S::STAGES >= 3 && S::STAGES <= 12 && S::SMEM + (int)sizeof(F8Sync) <= 227 * 1024, "shared memory");
  static_assert(S::COLS * S::BLOCKS <= 512 && (S::COLS & (S::COLS - 1)) == 0, "TMEM");
  static_assert(S::CW <= 128 && S::CW % 32 == 0, "columns of an epilogue warp");
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  static DeviceOnce once;
  e = once.run(dev, [] {
    cudaFuncAttributes f;
    cudaError_t r = cudaFuncGetAttributes(&f, k_fp8<AR, BN>);
    // A launch with fewer registers than the shares add up to would wait for them without end.
    if (r == cudaSuccess && S::SPLIT && f.numRegs != S::REGS) r = cudaErrorInvalidKernelImage;
    if (r != cudaSuccess) return r;
    return cudaFuncSetAttribute(k_fp8<AR, BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
  });
  if (e != cudaSuccess) return e;
  const long long tiles = (a.m + 127LL) / 128 * ((a.n + BN - 1) / BN);
  const int grid = (int)std::min<long long>(tiles, current_sm_count() * S::BLOCKS);
  constexpr int box = BN == 32 ? 0 : BN == 64 ? 1 : BN == 128 ? 2 : 3;
  k_fp8<AR, BN><<<grid, S::THREADS, S::SMEM, s>>>(*(const CUtensorMap*)&x, *(const CUtensorMap*)&w[box], a);
  return cudaGetLastError();
}

}  // namespace

int fp8_weight_box(int index) { return 32 << index; }
int fp8_row_box(int m) { return m <= 16 ? 16 : m <= 32 ? 32 : m <= 64 ? 64 : 128; }

cudaError_t launch_fp8(const TcMap* w, const TcMap& x, const Fp8Args& a, cudaStream_t s) {
  if (a.m <= 0) return cudaSuccess;
  switch (fp8_row_box(a.m)) {
    case 16: return run<16, 32>(w, x, a, s);
    case 32: return run<32, 32>(w, x, a, s);
    case 64: return run<64, 64>(w, x, a, s);
  }
  if (a.m <= 512) return run<128, 128>(w, x, a, s);
  return run<128, 256>(w, x, a, s);
}

}  // namespace trit
