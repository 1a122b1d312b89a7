// Products of 8-bit floating point with block scales:
//   out[r][i] = sum over blocks b of 128 of  sx[r][b] sw[i / 128][b]  (x_b[r] . w_b[i])
// with x and w in e4m3. The dot products of a block run on the tensor cores
// (tcgen05 kind::f8f6f4, f32 accumulators in TMEM); the blocks' sums leave
// TMEM one after another, are scaled and added in f32 registers, since every
// block has scales of its own.
//
// Rows of x are the MMA's M (a TMEM lane each), rows of w its N. Warp roles:
//   warp 0     TMA producer: a stage is 128 values of k of the tile's rows of
//              x and w, with the 128-byte swizzle;
//   warp 1     issues four MMAs (K = 32) a stage into one of the TMEM buffers;
//   warps 4..  epilogue: load a block's sums from TMEM, add them up.
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

constexpr int F8_BYTES = 128;  // of k a stage: one swizzle line, one scale block

__device__ __forceinline__ void mma_f8(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  uint32_t z = 0;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(d_tmem),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(z));
}
// Instruction descriptor of kind::f8f6f4: D f32 (bits 4-5 = 1), A and B e4m3
// (bits 7-9, 10-12 = 0), both K-major, N >> 3 at bit 17, M >> 4 at bit 24.
__host__ __device__ constexpr uint32_t idesc_f8(int m, int n) {
  return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// AR rows of x are loaded (the MMA's other rows read what lies behind them,
// and nobody reads their sums), BN rows of w.
template <int AR, int BN>
struct F8Shape {
  static constexpr int STAGE = (AR + BN) * F8_BYTES;
  static constexpr int STAGES = AR + BN >= 256 ? 5 : AR + BN >= 128 ? 6 : 8;
  static constexpr int BUFS = BN <= 64 ? 4 : 2;
  static constexpr int COLS = BUFS * BN;
  // The MMA reads 128 rows of A: what it reads behind the last stage's has to be shared memory of the block.
  static constexpr int SMEM = 1024 + STAGES * STAGE + (128 - AR) * F8_BYTES;
};
struct F8Sync {
  uint64_t full[8], empty[8], tfull[4], tempty[4], drain;
  uint32_t tmem;
  int abort;
};

__device__ __forceinline__ void put(void* out, size_t at, int type, float v) {
  if (type == kRowF32) ((float*)out)[at] = v;
  else if (type == kRowF16) ((__half*)out)[at] = __float2half_rn(v);
  else ((__nv_bfloat16*)out)[at] = __float2bfloat16_rn(v);
}

template <int AR, int BN>
__global__ void __launch_bounds__(256) k_fp8(const __grid_constant__ CUtensorMap xmap,
                                             const __grid_constant__ CUtensorMap wmap, const __grid_constant__ Fp8Args a) {
  using S = F8Shape<AR, BN>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* base = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  __shared__ F8Sync sync;
  F8Sync* y = &sync;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n0 = blockIdx.x * BN, m0 = blockIdx.y * 128;
  volatile int* abort = &y->abort;

  if (threadIdx.x == 0) {
    for (int i = 0; i < S::STAGES; ++i) {
      mbar_init(&y->full[i], 1);
      mbar_init(&y->empty[i], 1);
    }
    for (int i = 0; i < S::BUFS; ++i) {
      mbar_init(&y->tfull[i], 1);
      mbar_init(&y->tempty[i], 128);
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

  if (warp == 0) {
    if (lane == 0) {
      int issued = 0;
      for (int b = 0; b < a.blocks; ++b) {
        const int i = b % S::STAGES;
        if (!mbar_wait(&y->empty[i], ((b / S::STAGES) & 1) ^ 1, abort)) break;
        mbar_expect_tx(&y->full[i], S::STAGE);
        tma_load_2d(base + i * S::STAGE, &xmap, &y->full[i], b * F8_BYTES, m0);
        tma_load_2d(base + i * S::STAGE + AR * F8_BYTES, &wmap, &y->full[i], b * F8_BYTES, n0);
        issued = b + 1;
      }
      if (*abort) {
        // Let the copies in flight land before the block's memory is released.
        for (int b = max(0, issued - S::STAGES); b < issued; ++b) {
          const long long t0 = now_ns();
          while (!mbar_test(&y->full[b % S::STAGES], (b / S::STAGES) & 1) && now_ns() - t0 < TC_WAIT_NS) {
          }
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t s0 = smem_u32(base);
      for (int b = 0; b < a.blocks; ++b) {
        const int i = b % S::STAGES, u = b % S::BUFS;
        if (!mbar_wait(&y->full[i], (b / S::STAGES) & 1, abort)) break;
        if (!mbar_wait(&y->tempty[u], ((b / S::BUFS) & 1) ^ 1, abort)) break;
        fence_after();
#pragma unroll
        for (int j = 0; j < F8_BYTES / 32; ++j)
          mma_f8(tmem + u * BN, smem_desc_sw128(s0 + i * S::STAGE + j * 32),
                 smem_desc_sw128(s0 + i * S::STAGE + AR * F8_BYTES + j * 32), idesc_f8(128, BN), j ? 1u : 0u);
        mma_commit(&y->tfull[u]);
        mma_commit(&y->empty[i]);
      }
      mma_commit(&y->drain);
      const long long t0 = now_ns();
      while (!mbar_test(&y->drain, 0) && now_ns() - t0 < TC_WAIT_NS) {
      }
    }
  } else if (warp >= 4) {
    const int r = (warp - 4) * 32 + lane, row = m0 + r;
    const bool live = r < AR && row < a.m;
    const uint32_t tl = tmem + ((uint32_t)((warp - 4) * 32) << 16);
    const float* sx = a.x_scales + (size_t)row * a.blocks;
    const float* sw = a.w_scales + (size_t)(n0 / 128) * a.blocks;
    float2 acc[BN / 2];
#pragma unroll
    for (int i = 0; i < BN / 2; ++i) acc[i] = make_float2(0.0f, 0.0f);
    bool ok = true;
    for (int b = 0; b < a.blocks; ++b) {
      const int u = b % S::BUFS;
      const float scale = live ? __ldg(sx + b) * __ldg(sw + b) : 0.0f;
      const float2 s2 = make_float2(scale, scale);
      if (!__all_sync(0xffffffffu, mbar_wait(&y->tfull[u], (b / S::BUFS) & 1, abort))) {
        ok = false;
        break;
      }
      fence_after();
#pragma unroll
      for (int c = 0; c < BN; c += 32) {
        uint32_t v[32];
        tmem_ld<32>(tl + u * BN + c, v);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 16; ++i)
          acc[c / 2 + i] = fma2(make_float2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), s2, acc[c / 2 + i]);
      }
      fence_before();
      mbar_arrive(&y->tempty[u]);
    }
    if (ok && live) {
#pragma unroll
      for (int i = 0; i < BN; ++i)
        if (n0 + i < a.n) put(a.out, (size_t)row * a.out_stride + n0 + i, a.type, (i & 1) ? acc[i / 2].y : acc[i / 2].x);
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
cudaError_t run(const TcMap& w, const TcMap& x, const Fp8Args& a, cudaStream_t s) {
  using S = F8Shape<AR, BN>;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  static DeviceOnce once;
  e = once.run(dev, [] { return cudaFuncSetAttribute(k_fp8<AR, BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM); });
  if (e != cudaSuccess) return e;
  const dim3 grid((a.n + BN - 1) / BN, (a.m + 127) / 128);
  k_fp8<AR, BN><<<grid, 256, S::SMEM, s>>>(*(const CUtensorMap*)&x, *(const CUtensorMap*)&w, a);
  return cudaGetLastError();
}

}  // namespace

int fp8_weight_box(int index) { return 32 << index; }
int fp8_row_box(int m) { return m <= 16 ? 16 : m <= 32 ? 32 : m <= 64 ? 64 : 128; }

cudaError_t launch_fp8(const TcMap* w, const TcMap& x, const Fp8Args& a, cudaStream_t s) {
  if (a.m <= 0) return cudaSuccess;
  switch (fp8_row_box(a.m)) {
    case 16: return run<16, 32>(w[0], x, a, s);
    case 32: return run<32, 32>(w[0], x, a, s);
    case 64: return run<64, 64>(w[1], x, a, s);
    default: return run<128, 128>(w[2], x, a, s);
  }
}

}  // namespace trit
