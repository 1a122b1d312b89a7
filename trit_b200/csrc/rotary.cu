// Rotary positions of queries and keys in one pass: pair i of a head at
// position p turns by the angle p f_i,
//   (a, b) -> f (a cos - b sin, b cos + a sin),
// pairs (i, i + d / 2) or (2 i, 2 i + 1) of the head's first d values; values
// behind them are copied, bit for bit.
//
// p f_i is formed exactly, in two 64-bit numbers, and brought to an eighth of a
// turn around a quarter turn before anything is rounded to f32: an angle of A
// radians is off by 2^-49 + A 2^-104, so positions of up to 2^53 lose nothing. A
// block computes the angles of its rows once for all heads, while its values
// load. Bound by bytes, each read and written once.
#include <cuda_runtime.h>

#include <algorithm>

#include "device.cuh"
#include "launch.cuh"
#include "rows.cuh"
#include "rows.h"

namespace trit {
namespace {

constexpr int kRotaryThreads = 256;

// V values: f32 ones as they are, pairs of 16-bit ones as words, a lone one in
// a word of its own.
template <class T, int V>
struct Pack {
  static constexpr bool F32 = sizeof(T) == 4;
  static constexpr int N = F32 ? V : (V + 1) / 2;
  uint32_t w[N];
  __device__ __forceinline__ float get() const {  // of a lone value
    if constexpr (F32) return __uint_as_float(w[0]);
    else return to_f32(*(const T*)w);
  }
  __device__ __forceinline__ void put(float x) {
    if constexpr (F32) w[0] = __float_as_uint(x);
    else *(T*)w = from_f32<T>(x);
  }
  // Values 2 i and 2 i + 1.
  __device__ __forceinline__ float2 get2(int i) const {
    if constexpr (F32) return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
    else return unpack2<T>(w[i]);
  }
  __device__ __forceinline__ void put2(int i, float2 x) {
    if constexpr (F32) {
      w[2 * i] = __float_as_uint(x.x);
      w[2 * i + 1] = __float_as_uint(x.y);
    } else {
      w[i] = pack2<T>(x);
    }
  }
};
// One load or store where ALIGNED; values of a pair one after another where not.
template <class T, int V, bool ALIGNED>
__device__ __forceinline__ Pack<T, V> load(const T* p) {
  Pack<T, V> r;
  if constexpr (!ALIGNED) {
    static_assert(V == 2, "unaligned units are pairs");
    if constexpr (sizeof(T) == 4) {
      r.w[0] = *(const uint32_t*)p;
      r.w[1] = *(const uint32_t*)(p + 1);
    } else {
      r.w[0] = *(const uint16_t*)p | (uint32_t)*(const uint16_t*)(p + 1) << 16;
    }
  } else if constexpr (sizeof(T) * V == 16) {
    const uint4 v = *(const uint4*)p;
    r.w[0] = v.x; r.w[1] = v.y; r.w[2] = v.z; r.w[3] = v.w;
  } else if constexpr (sizeof(T) * V == 8) {
    const uint2 v = *(const uint2*)p;
    r.w[0] = v.x; r.w[1] = v.y;
  } else if constexpr (sizeof(T) * V == 4) {
    r.w[0] = *(const uint32_t*)p;
  } else {
    r.w[0] = *(const uint16_t*)p;
  }
  return r;
}
template <class T, int V, bool ALIGNED>
__device__ __forceinline__ void store(T* p, const Pack<T, V>& r) {
  if constexpr (!ALIGNED) {
    if constexpr (sizeof(T) == 4) {
      *(uint32_t*)p = r.w[0];
      *(uint32_t*)(p + 1) = r.w[1];
    } else {
      *(uint16_t*)p = (uint16_t)r.w[0];
      *(uint16_t*)(p + 1) = (uint16_t)(r.w[0] >> 16);
    }
  } else if constexpr (sizeof(T) * V == 16) {
    *(uint4*)p = make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]);
  } else if constexpr (sizeof(T) * V == 8) {
    *(uint2*)p = make_uint2(r.w[0], r.w[1]);
  } else if constexpr (sizeof(T) * V == 4) {
    *(uint32_t*)p = r.w[0];
  } else {
    *(uint16_t*)p = (uint16_t)r.w[0];
  }
}

// A unit is V values, or V pairs of halves. Threads of a block: (unit of a head,
// head, row); a thread has two heads.
// All of it is passed by value: a call needs nothing on the device that outlives
// it. PAIRS: 64 where they are enough, since a launch copies its parameters
// (2 KB of them cost 3 us of the host's call).
template <int PAIRS>
struct RotaryWork {
  RotaryArgs a;
  int head_dim, rotary_dim;
  float factor;
  int turning, per_head;  // units of a head that turn, which come first, and all of them
  double frequency[PAIRS];  // radians a position
};

// cos and sin of p w radians, times f: in turns, the nearest quarter turn, and
// the Taylor series of what is left, up to an eighth of a turn (|x| <= pi / 4: the
// first terms left out are x^11 / 11! < 2e-9 and x^12 / 12! < 2e-10). Short, so
// that it keeps few registers from the values on their way.
__device__ __forceinline__ float2 turn(double p, double w, float f) {
  // 1 / (2 pi) is kTurn + kTurnRest, and p w is u + (the rest) exactly; whole
  // turns leave the product with kTurn before it is rounded. (u is not to be
  // fused with what is subtracted from it.)
  constexpr double kTurn = 0x1.45f306dc9c883p-3, kTurnRest = -0x1.6b01ec5417056p-57;
  const double u = __dmul_rn(p, w);
  double t = fma(u, kTurn, -rint(__dmul_rn(u, kTurn)));
  t = fma(u, kTurnRest, t);
  t = fma(fma(p, w, -u), kTurn, t);
  t -= rint(t);                     // [-1/2, 1/2]
  const double q = rint(4.0 * t);   // the quarter turn
  const float x = (float)(fma(-0.25, q, t) * 6.283185307179586), z = x * x;
  float s = fmaf(z, 1.0f / 362880.0f, -1.0f / 5040.0f), c = fmaf(z, -1.0f / 3628800.0f, 1.0f / 40320.0f);
  s = fmaf(z, s, 1.0f / 120.0f);
  c = fmaf(z, c, -1.0f / 720.0f);
  s = fmaf(z, s, -1.0f / 6.0f);
  c = fmaf(z, c, 1.0f / 24.0f);
  s = fmaf(x * z, s, x);
  c = fmaf(z, fmaf(z, c, -0.5f), 1.0f);
  const int n = (int)q;             // -2 .. 2
  const float a = n & 1 ? s : c, b = n & 1 ? c : s;
  return make_float2(((n + 1) & 2) ? -a * f : a * f, (n & 2) ? -b * f : b * f);
}

// PV consecutive values of cos or sin in shared memory.
template <int PV>
__device__ __forceinline__ void read_angles(const float* from, float (&v)[PV]) {
  if constexpr (PV % 4 == 0) {
#pragma unroll
    for (int i = 0; i < PV; i += 4) *(float4*)(v + i) = *(const float4*)(from + i);
  } else {
#pragma unroll
    for (int i = 0; i < PV; ++i) v[i] = from[i];
  }
}

template <class T, int V, bool INTER, bool ALIGNED, int PAIRS>
__global__ void __launch_bounds__(kRotaryThreads, 4) k_rotary(const __grid_constant__ RotaryWork<PAIRS> w) {
  constexpr int PV = INTER ? V / 2 : V;  // pairs of a unit
  extern __shared__ float4 angles[];     // [row][cos, sin][pair]
  const RotaryArgs& a = w.a;
  const int hd = w.head_dim, rd = w.rotary_dim, pairs = rd / 2, slots = (w.turning * PV + 3) / 4 * 4;
  const int heads = a.q_heads + a.k_heads;
  const int row0 = blockIdx.x * blockDim.z, row = row0 + threadIdx.z;
  const int head0 = blockIdx.y * 2 * blockDim.y + threadIdx.y, head1 = head0 + blockDim.y;
  const bool live0 = row < a.rows && head0 < heads, live1 = row < a.rows && head1 < heads;
  const size_t at_row = row;
  const T* const q = (const T*)a.q + at_row * a.q_stride;
  const T* const k = (const T*)a.k + at_row * a.k_stride - (ptrdiff_t)a.q_heads * hd;  // (heads counted from q's first)
  T* const qo = (T*)a.q_out + at_row * a.q_out_stride;
  T* const ko = (T*)a.k_out + at_row * a.k_out_stride - (ptrdiff_t)a.q_heads * hd;
  const T* const from0 = (head0 < a.q_heads ? q : k) + head0 * hd;
  const T* const from1 = (head1 < a.q_heads ? q : k) + head1 * hd;
  T* const to0 = (head0 < a.q_heads ? qo : ko) + head0 * hd;
  T* const to1 = (head1 < a.q_heads ? qo : ko) + head1 * hd;

  using P = Pack<T, V>;
  P lo0, hi0, lo1, hi1;
  const auto fetch = [&](int at, const T* from, P& lo, P& hi) {
    const bool turns = INTER || at < w.turning;
    from += at * V + (turns ? 0 : rd - w.turning * V);
    lo = load<T, V, ALIGNED>(from);
    if (!INTER && turns) hi = load<T, V, ALIGNED>(from + pairs);
  };
  let_next_start();
  after_kernel_before();
  if ((int)threadIdx.x < w.per_head) {
    if (live0) fetch(threadIdx.x, from0, lo0, hi0);
    if (live1) fetch(threadIdx.x, from1, lo1, hi1);
  }
  const int threads = blockDim.x * blockDim.y * blockDim.z;
  const int thread = (threadIdx.z * blockDim.y + threadIdx.y) * blockDim.x + threadIdx.x;
#pragma unroll 1
  for (int z = 0; z < (int)blockDim.z && row0 + z < a.rows; ++z) {
    float* to = (float*)angles + z * 2 * slots;
#pragma unroll 1  // (the values on their way need the registers)
    for (int p = thread; p < pairs; p += threads) {
      const float2 cs = turn((double)a.positions[row0 + z], w.frequency[p], w.factor);
      to[p] = cs.x;
      to[slots + p] = cs.y;
    }
  }
  __syncthreads();
  const float* const cos_at = (const float*)angles + threadIdx.z * 2 * slots;
#pragma unroll 1
  for (int at = threadIdx.x; at < w.per_head; at += blockDim.x) {
    if (at != (int)threadIdx.x) {
      if (live0) fetch(at, from0, lo0, hi0);
      if (live1) fetch(at, from1, lo1, hi1);
    }
    if (at >= w.turning) {
      const int place = at * V + (INTER ? 0 : rd - w.turning * V);
      if (live0) store<T, V, ALIGNED>(to0 + place, lo0);
      if (live1) store<T, V, ALIGNED>(to1 + place, lo1);
      continue;
    }
    float c[PV], s[PV];
    read_angles<PV>(cos_at + at * PV, c);
    read_angles<PV>(cos_at + slots + at * PV, s);
    const auto put = [&](T* to, const P& lo, const P& hi) {
      if constexpr (INTER) {
        // A unit may reach behind the last pair: those values stay.
        const int turns = pairs - at * PV;
        P o = lo;
#pragma unroll
        for (int j = 0; j < PV; ++j) {
          const float2 x = lo.get2(j);
          if (j < turns) o.put2(j, make_float2(x.x * c[j] - x.y * s[j], x.y * c[j] + x.x * s[j]));
        }
        store<T, V, ALIGNED>(to + at * V, o);
      } else {
        P o, q;
        if constexpr (PV % 2 == 0) {
#pragma unroll
          for (int j = 0; j < PV; j += 2) {
            const float2 u = lo.get2(j / 2), v = hi.get2(j / 2);
            const float2 cc = make_float2(c[j], c[j + 1]), ss = make_float2(s[j], s[j + 1]);
            o.put2(j / 2, fma2(v, make_float2(-ss.x, -ss.y), mul2(u, cc)));
            q.put2(j / 2, fma2(u, ss, mul2(v, cc)));
          }
        } else {
          const float u = lo.get(), v = hi.get();
          o.put(u * c[0] - v * s[0]);
          q.put(v * c[0] + u * s[0]);
        }
        store<T, V, ALIGNED>(to + at * V, o);
        store<T, V, ALIGNED>(to + at * V + pairs, q);
      }
    };
    if (live0) put(to0, lo0, hi0);
    if (live1) put(to1, lo1, hi1);
  }
}

template <class T, int V, bool INTER, bool ALIGNED, int PAIRS>
cudaError_t run_sized(const RotaryTable& t, const RotaryArgs& a, cudaStream_t s) {
  constexpr int PV = INTER ? V / 2 : V;
  const int pairs = t.rotary_dim / 2, heads = a.q_heads + a.k_heads;
  // In place, the values behind the pairs stay as they are.
  const bool still = a.q == a.q_out && a.k == a.k_out;
  RotaryWork<PAIRS> w;
  w.a = a;
  w.head_dim = t.head_dim;
  w.rotary_dim = t.rotary_dim;
  w.factor = t.factor;
  std::copy(t.frequency, t.frequency + pairs, w.frequency);
  w.turning = INTER ? (t.rotary_dim + V - 1) / V : pairs / V;
  w.per_head = still ? w.turning : INTER ? t.head_dim / V : w.turning + (t.head_dim - t.rotary_dim) / V;
  const int lanes = std::min(w.per_head, kRotaryThreads);
  // Two heads a thread, the heads in parts as even as they go; several rows
  // where that leaves a block small and the rows are many.
  const int teams = kRotaryThreads / lanes, two = (heads + 1) / 2, parts = (two + teams - 1) / teams;
  const int head_lanes = (two + parts - 1) / parts;
  int rows = std::min(std::max(1, teams / head_lanes), 8);
  if ((long long)a.rows * parts < 8LL * current_sm_count()) rows = 1;
  const size_t smem = (size_t)rows * 2 * ((w.turning * PV + 3) / 4 * 4) * sizeof(float);
  return launch_early(k_rotary<T, V, INTER, ALIGNED, PAIRS>, dim3((a.rows + rows - 1) / rows, parts), dim3(lanes, head_lanes, rows),
                      smem, s, 1, w);
}
template <class T, int V, bool INTER, bool ALIGNED>
cudaError_t run(const RotaryTable& t, const RotaryArgs& a, cudaStream_t s) {
  return t.rotary_dim <= 128 ? run_sized<T, V, INTER, ALIGNED, 64>(t, a, s)
                             : run_sized<T, V, INTER, ALIGNED, kRotaryPairs>(t, a, s);
}

// The widest units that the sizes, strides and addresses allow.
template <class T>
cudaError_t by_alignment(const RotaryTable& t, const RotaryArgs& a, cudaStream_t s) {
  const uintptr_t at = (uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.q_out | (uintptr_t)a.k_out;
  const size_t strides = a.q_stride | a.k_stride | a.q_out_stride | a.k_out_stride | (size_t)t.head_dim;
  const auto fits = [&](int v) { return at % (v * sizeof(T)) == 0 && strides % v == 0; };
  constexpr int V = 16 / sizeof(T);
  if (t.interleaved) {
    if (fits(V)) return run<T, V, true, true>(t, a, s);
    return run<T, 2, true, false>(t, a, s);  // head_dim is even
  }
  const int half = t.rotary_dim / 2, rest = t.head_dim - t.rotary_dim;
  if (fits(V) && half % V == 0 && rest % V == 0) return run<T, V, false, true>(t, a, s);
  if (fits(2) && half % 2 == 0 && rest % 2 == 0) return run<T, 2, false, true>(t, a, s);
  return run<T, 1, false, true>(t, a, s);
}

}  // namespace

cudaError_t launch_rotary(const RotaryTable& t, const RotaryArgs& a, cudaStream_t s) {
  if (a.rows <= 0 || a.q_heads + a.k_heads <= 0) return cudaSuccess;
  if (a.type == kRowF32) return by_alignment<float>(t, a, s);
  if (a.type == kRowF16) return by_alignment<__half>(t, a, s);
  return by_alignment<__nv_bfloat16>(t, a, s);
}

}  // namespace trit
