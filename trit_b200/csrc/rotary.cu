// Rotary positions of queries and keys in one pass: pair i of a head at
// position p turns by the angle 2 pi p t_i, t_i in turns a position,
//   (a, b) -> f (a cos - b sin, b cos + a sin),
// pairs (i, i + d / 2) or (2 i, 2 i + 1) of the head's first d values; values
// behind them are copied, bit for bit.
//
// p t_i is formed in 64 bits and brought to an eighth of a turn around a
// quarter turn before anything is rounded to f32, so positions of any size
// lose nothing. A block computes the angles of its rows once for all heads
// while its first values load; a thread then keeps those of its pairs in
// registers. Bound by bytes, each read and written once.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "launch.cuh"
#include "rows.h"

namespace trit {
namespace {

constexpr int kRotaryThreads = 256;
constexpr int kRotaryAhead = 4;  // heads a thread loads before it works on the first

template <class T>
__device__ __forceinline__ float wide(T v) {
  if constexpr (sizeof(T) == 4) return v;
  else if constexpr (__is_same(T, __half)) return __half2float(v);
  else return __bfloat162float(v);
}
template <class T>
__device__ __forceinline__ T narrow(float v) {
  if constexpr (sizeof(T) == 4) return v;
  else if constexpr (__is_same(T, __half)) return __float2half_rn(v);
  else return __float2bfloat16_rn(v);
}

// V values as one load or store where ALIGNED.
template <class T, int V>
struct __align__(sizeof(T) * V) Pack {
  T v[V];
};
template <class T, int V, bool ALIGNED>
__device__ __forceinline__ Pack<T, V> load(const T* p) {
  if constexpr (ALIGNED) return *(const Pack<T, V>*)p;
  Pack<T, V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) r.v[i] = p[i];
  return r;
}
template <class T, int V, bool ALIGNED>
__device__ __forceinline__ void store(T* p, const Pack<T, V>& r) {
  if constexpr (ALIGNED) {
    *(Pack<T, V>*)p = r;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) p[i] = r.v[i];
  }
}

// How a block of threads shares out its rows and heads. A unit is V values, or
// V pairs of halves; `at` counts a head's units, those that turn first. A
// thread keeps one unit's place and row, so that it reads its angles once, and
// goes through every `head_lanes`-th head.
struct RotaryWork {
  RotaryArgs a;
  int turning, per_head;  // units of a head that turn, and all of them
  int lanes;              // units of a head side by side: per_head, at most the block
  int rows, head_lanes;   // rows of a block; threads a unit and row
  int heads;              // of a block
};

// cos and sin of t turns, times f.
__device__ __forceinline__ float2 turn(double t, float f) {
  t -= rint(t);                     // [-1/2, 1/2]
  const double q = rint(4.0 * t);   // the quarter turn
  float s, c;
  sincospif(2.0f * (float)(t - 0.25 * q), &s, &c);
  const int z = (int)q;
  if (z == 1) { const float o = c; c = -s; s = o; }
  else if (z == -1) { const float o = c; c = s; s = -o; }
  else if (z) { c = -c; s = -s; }   // half a turn either way
  return make_float2(c * f, s * f);
}

template <class T, int V, bool INTER, bool ALIGNED>
__global__ void __launch_bounds__(kRotaryThreads) k_rotary(const __grid_constant__ RotaryTable table,
                                                           const __grid_constant__ RotaryWork w) {
  constexpr int PV = INTER ? V / 2 : V;  // pairs of a unit
  extern __shared__ float2 angles[];     // [row][pair of its unit][unit]: a warp's units lie side by side
  const RotaryArgs& a = w.a;
  const int pairs = table.rotary_dim / 2, slots = w.turning * PV;
  const int row0 = blockIdx.x * w.rows, rows = min(w.rows, a.rows - row0);
  const int head_end = min((int)(blockIdx.y + 1) * w.heads, a.q_heads + a.k_heads);
  const int lane = threadIdx.x % w.lanes, team = threadIdx.x / w.lanes, r = team % w.rows, head_lane = team / w.rows;
  const int first = r < rows && head_lane < w.head_lanes ? (int)blockIdx.y * w.heads + head_lane : head_end;
  const T* const q = (const T*)a.q + (size_t)(row0 + r) * a.q_stride;
  const T* const k = (const T*)a.k + (size_t)(row0 + r) * a.k_stride;
  T* const qo = (T*)a.q_out + (size_t)(row0 + r) * a.q_out_stride;
  T* const ko = (T*)a.k_out + (size_t)(row0 + r) * a.k_out_stride;
  const int hd = table.head_dim, rd = table.rotary_dim;

  using P = Pack<T, V>;
  P lo[kRotaryAhead], hi[kRotaryAhead];
  // The unit's values of the next heads from h on.
  auto fetch = [&](int at, int h) {
#pragma unroll
    for (int i = 0; i < kRotaryAhead; ++i) {
      const int head = h + i * w.head_lanes;
      if (head >= head_end) break;
      const T* from = head < a.q_heads ? q + head * hd : k + (head - a.q_heads) * hd;
      if (INTER || at < w.turning) from += at * V;
      else from += rd + (at - w.turning) * V;
      lo[i] = load<T, V, ALIGNED>(from);
      if (!INTER && at < w.turning) hi[i] = load<T, V, ALIGNED>(from + pairs);
    }
  };
  let_next_start();
  after_kernel_before();
  if (first < head_end && lane < w.per_head) fetch(lane, first);
  for (int i = threadIdx.x; i < rows * pairs; i += kRotaryThreads) {
    const int row = i / pairs, p = i - row * pairs;
    angles[row * slots + p % PV * w.turning + p / PV] =
        turn((double)__ldg(a.positions + row0 + row) * table.turns[p], table.factor);
  }
  __syncthreads();
  for (int at = lane; at < w.per_head; at += w.lanes) {
    float2 cs[PV];
    // An interleaved unit may reach behind the last pair: those values stay.
    const int turns = at < w.turning ? min(PV, pairs - at * PV) : 0;
#pragma unroll
    for (int j = 0; j < PV; ++j)
      cs[j] = j < turns ? angles[r * slots + j * w.turning + at] : make_float2(1.0f, 0.0f);
    for (int h = first; h < head_end; h += kRotaryAhead * w.head_lanes) {
      if (at != lane || h != first) fetch(at, h);
#pragma unroll
      for (int i = 0; i < kRotaryAhead; ++i) {
        const int head = h + i * w.head_lanes;
        if (head >= head_end) break;
        T* to = head < a.q_heads ? qo + head * hd : ko + (head - a.q_heads) * hd;
        if (INTER) {
          P o = lo[i];
#pragma unroll
          for (int j = 0; j < PV; ++j) {
            const float x = wide(lo[i].v[2 * j]), y = wide(lo[i].v[2 * j + 1]);
            if (j < turns) {
              o.v[2 * j] = narrow<T>(x * cs[j].x - y * cs[j].y);
              o.v[2 * j + 1] = narrow<T>(y * cs[j].x + x * cs[j].y);
            }
          }
          store<T, V, ALIGNED>(to + at * V, o);
        } else if (at < w.turning) {
          P x, y;
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float u = wide(lo[i].v[j]), v = wide(hi[i].v[j]);
            x.v[j] = narrow<T>(u * cs[j].x - v * cs[j].y);
            y.v[j] = narrow<T>(v * cs[j].x + u * cs[j].y);
          }
          store<T, V, ALIGNED>(to + at * V, x);
          store<T, V, ALIGNED>(to + at * V + pairs, y);
        } else {
          store<T, V, ALIGNED>(to + rd + (at - w.turning) * V, lo[i]);
        }
      }
    }
  }
}

template <class T, int V, bool INTER, bool ALIGNED>
cudaError_t run(const RotaryTable& t, const RotaryArgs& a, cudaStream_t s) {
  const int pairs = t.rotary_dim / 2, heads = a.q_heads + a.k_heads;
  // In place, the values behind the pairs stay as they are.
  const bool still = a.q == a.q_out && a.k == a.k_out;
  RotaryWork w{a};
  w.turning = INTER ? (t.rotary_dim + V - 1) / V : pairs / V;
  w.per_head = still ? w.turning : INTER ? t.head_dim / V : w.turning + (t.head_dim - t.rotary_dim) / V;
  w.lanes = std::min(w.per_head, kRotaryThreads);
  const int teams = kRotaryThreads / w.lanes;
  // Many rows: a thread goes through about eight heads. Few: a block has one
  // row, and its heads are cut so that the blocks fill the SMs.
  const long long threads = (long long)a.rows * heads * w.lanes / 8;
  if (threads >= (long long)current_sm_count() * 512) {
    w.head_lanes = std::min(teams, (heads + 7) / 8);
    w.rows = std::min(std::min(teams / w.head_lanes, 8), a.rows);
    w.heads = heads;
  } else {
    w.rows = 1;
    const int parts = std::max(1, std::min((heads + teams - 1) / teams * kRotaryAhead, 2 * current_sm_count() / a.rows));
    w.heads = (heads + parts - 1) / parts;
    w.head_lanes = std::min(teams, w.heads);
  }
  return launch_early(k_rotary<T, V, INTER, ALIGNED>,
                      dim3((a.rows + w.rows - 1) / w.rows, (heads + w.heads - 1) / w.heads), dim3(kRotaryThreads),
                      (size_t)w.rows * w.turning * (INTER ? V / 2 : V) * sizeof(float2), s, 1, t, w);
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
