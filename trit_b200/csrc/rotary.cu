// Rotary positions of queries and keys in one pass: pair i of a head at
// position p turns by the angle 2 pi p t_i, t_i in turns a position,
//   (a, b) -> f (a cos - b sin, b cos + a sin),
// pairs (i, i + d / 2) or (2 i, 2 i + 1) of the head's first d values; values
// behind them are copied, bit for bit.
//
// p t_i is formed in 64 bits and brought to an eighth of a turn around a
// quarter turn before anything is rounded to f32, so positions of any size
// lose nothing. A block computes the angles of its rows once for all heads
// while its first values load. Bound by bytes, each read and written once.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "rows.h"

namespace trit {
namespace {

constexpr int kRotaryThreads = 256;
constexpr int kRotaryAhead = 2;  // units a thread loads before it works on the first

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

// n / d for n < 2^31 by a multiplication.
struct Divide {
  uint32_t by = 1, mul = 0, shift = 0;
  explicit Divide(uint32_t d) : by(d) {
    // ceil(2^(32 + shift) / d) with 2^shift >= d: the error stays below 1 / d.
    while ((1ull << shift) < d) ++shift;
    mul = (uint32_t)(((1ull << (32 + shift)) + d - 1) / d - (1ull << 32));
  }
  __device__ __forceinline__ uint32_t operator()(uint32_t n) const {
    return (uint32_t)(((unsigned long long)__umulhi(n, mul) + n) >> shift);
  }
};

// The work on a row: `units` of V values (halves: V pairs, both their halves),
// head after head, queries before keys, and behind the rotated units of a
// head the copied ones.
struct RotaryWork {
  RotaryArgs a;
  int hd, rd, turning, per_head;  // units of a head that turn, and all of them
  int rows_per_block, heads_per_block;
  Divide by_row, by_head, by_pairs;
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
  extern __shared__ float2 angles[];  // [rows of the block][pairs]
  const RotaryArgs& a = w.a;
  const int row0 = blockIdx.x * w.rows_per_block, rows = min(w.rows_per_block, a.rows - row0);
  const int head0 = blockIdx.y * w.heads_per_block, heads = min(w.heads_per_block, a.q_heads + a.k_heads - head0);
  const int pairs = w.rd / 2, row_units = heads * w.per_head, units = rows * row_units;
  // by_row is for a full set of heads; the last blocks of a row divide.
  const bool full = heads == w.heads_per_block;

  struct Unit {
    const T* from;
    T* to;
    int row, at;  // the unit's place in its head; -1: none
  };
  auto find = [&](int u) {
    Unit r;
    r.at = -1;
    if (u >= units) return r;
    r.row = full ? w.by_row(u) : u / row_units;
    const int rem = u - r.row * row_units, h = w.by_head(rem);
    r.at = rem - h * w.per_head;
    const int head = head0 + h;
    const size_t row = row0 + r.row;
    if (head < a.q_heads) {
      r.from = (const T*)a.q + row * a.q_stride + (size_t)head * w.hd;
      r.to = (T*)a.q_out + row * a.q_out_stride + (size_t)head * w.hd;
    } else {
      r.from = (const T*)a.k + row * a.k_stride + (size_t)(head - a.q_heads) * w.hd;
      r.to = (T*)a.k_out + row * a.k_out_stride + (size_t)(head - a.q_heads) * w.hd;
    }
    return r;
  };
  using P = Pack<T, V>;
  auto fetch = [&](const Unit& r, P& lo, P& hi) {
    if (r.at < 0) return;
    if (INTER) {
      lo = load<T, V, ALIGNED>(r.from + r.at * V);
    } else if (r.at < w.turning) {
      lo = load<T, V, ALIGNED>(r.from + r.at * V);
      hi = load<T, V, ALIGNED>(r.from + r.at * V + pairs);
    } else {
      lo = load<T, V, ALIGNED>(r.from + w.rd + (r.at - w.turning) * V);
    }
  };
  Unit unit[kRotaryAhead];
  P lo[kRotaryAhead], hi[kRotaryAhead];
#pragma unroll
  for (int i = 0; i < kRotaryAhead; ++i) {
    unit[i] = find(threadIdx.x + i * kRotaryThreads);
    fetch(unit[i], lo[i], hi[i]);
  }
  for (int i = threadIdx.x; i < rows * pairs; i += kRotaryThreads) {
    const int r = w.by_pairs(i);
    angles[i] = turn((double)a.positions[row0 + r] * table.turns[i - r * pairs], table.factor);
  }
  __syncthreads();
  for (int u0 = 0; u0 < units; u0 += kRotaryAhead * kRotaryThreads) {
#pragma unroll
    for (int i = 0; i < kRotaryAhead; ++i) {
      const Unit& r = unit[i];
      if (r.at < 0) continue;
      const float2* cs = angles + r.row * pairs;
      if (INTER) {
        P o = lo[i];
        const int first = r.at * V;
#pragma unroll
        for (int j = 0; j < V; j += 2) {
          if (first + j >= w.rd) break;  // rd is even: a pair turns as a whole
          const float2 t = cs[(first + j) / 2];
          const float x = wide(lo[i].v[j]), y = wide(lo[i].v[j + 1]);
          o.v[j] = narrow<T>(x * t.x - y * t.y);
          o.v[j + 1] = narrow<T>(y * t.x + x * t.y);
        }
        store<T, V, ALIGNED>(r.to + first, o);
      } else if (r.at < w.turning) {
        P p, q;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float2 t = cs[r.at * V + j];
          const float x = wide(lo[i].v[j]), y = wide(hi[i].v[j]);
          p.v[j] = narrow<T>(x * t.x - y * t.y);
          q.v[j] = narrow<T>(y * t.x + x * t.y);
        }
        store<T, V, ALIGNED>(r.to + r.at * V, p);
        store<T, V, ALIGNED>(r.to + r.at * V + pairs, q);
      } else {
        store<T, V, ALIGNED>(r.to + w.rd + (r.at - w.turning) * V, lo[i]);
      }
    }
    if (u0 + kRotaryAhead * kRotaryThreads >= units) break;
#pragma unroll
    for (int i = 0; i < kRotaryAhead; ++i) {
      unit[i] = find(u0 + (kRotaryAhead + i) * kRotaryThreads + threadIdx.x);
      fetch(unit[i], lo[i], hi[i]);
    }
  }
}

template <class T, int V, bool INTER, bool ALIGNED>
cudaError_t run(const RotaryTable& t, const RotaryArgs& a, cudaStream_t s) {
  const int pairs = t.rotary_dim / 2, heads = a.q_heads + a.k_heads;
  // In place, the values behind the pairs stay as they are.
  const bool still = a.q == a.q_out && a.k == a.k_out;
  const int turning = INTER ? ((still ? t.rotary_dim : t.head_dim) + V - 1) / V : pairs / V;
  const int per_head = INTER || still ? turning : turning + (t.head_dim - t.rotary_dim) / V;
  // Blocks of several rows, so that a thread has a few units; where the rows
  // alone do not fill the SMs, a block takes a part of the heads.
  const int row_units = heads * per_head;
  const int rows = std::max(1, std::min(std::min(4, 4 * kRotaryThreads / std::max(1, row_units)), a.rows));
  const int row_blocks = (a.rows + rows - 1) / rows;
  const int wanted = 2 * current_sm_count();
  int parts = std::max(1, std::min(heads, wanted / row_blocks));
  while (parts > 1 && (heads + parts - 1) / parts * per_head * rows < kRotaryThreads / 2) --parts;
  const int heads_per_block = (heads + parts - 1) / parts;
  const RotaryWork w{a, t.head_dim, t.rotary_dim, turning, per_head, rows, heads_per_block,
                     Divide(heads_per_block * per_head), Divide(per_head), Divide(pairs)};
  k_rotary<T, V, INTER, ALIGNED><<<dim3(row_blocks, (heads + heads_per_block - 1) / heads_per_block), kRotaryThreads,
                                   (size_t)rows * pairs * sizeof(float2), s>>>(t, w);
  return cudaGetLastError();
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
