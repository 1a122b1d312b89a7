// Operators on rows between a caller's products and its cache: the norm into
// 8-bit rows (rms_norm.cu), rotary positions (rotary.cu), products with
// weights in 8-bit floating point (dense_fp8.cu), and their host side
// (rows.cpp).
//
// 8-bit rows are e4m3 numbers [rows][width] with one f32 scale for each group
// of 128, [rows][ceil(width / 128)].
#pragma once

#include <cuda_runtime.h>

#include <cstdint>
#include <memory>
#include <mutex>
#include <string>
#include <vector>

#include "kernels.h"

namespace trit {

enum RowType : int { kRowF32 = 0, kRowF16 = 1, kRowBF16 = 2 };
constexpr int kFp8Group = 128;
inline size_t row_type_size(int type) { return type == kRowF32 ? 4 : 2; }

// The device that a call's pointers are on is current for the call.
class OnDevice {
 public:
  explicit OnDevice(int device);
  ~OnDevice();
  OnDevice(const OnDevice&) = delete;
  OnDevice& operator=(const OnDevice&) = delete;

 private:
  int before_ = 0, device_ = 0;
};
// The CUDA device whose memory p is in; throws when p is not aligned to
// `align` bytes or is not device memory.
int pointer_device(const void* p, size_t align, const char* what);
// Throws unless p is aligned and on `device`.
void check_on_device(const void* p, size_t align, const char* what, int device);

// ------------------------------------------------------------------ norm
struct NormArgs {
  const void* x = nullptr;
  const void* residual = nullptr;  // null: none
  void* sum = nullptr;             // x + residual, with a residual
  const void* weight = nullptr;    // null: the rows as they are, no norm
  void* out = nullptr;             // values, or null
  uint8_t* codes = nullptr;        // 8-bit rows, or null
  float* scales = nullptr;
  size_t x_stride = 0, residual_stride = 0, sum_stride = 0, out_stride = 0;
  int rows = 0, width = 0;
  int type = 0, weight_f32 = 0;
  double eps = 0.0, inv_width = 0.0;  // (the latter set by the launch)
};
cudaError_t launch_rms_norm(const NormArgs& a, cudaStream_t s);
// The arguments of a caller's norm, checked, and the norm.
void rms_norm(NormArgs a, size_t rows, size_t width, cudaStream_t s);

// ---------------------------------------------------------------- rotary
constexpr int kRotaryPairs = 256;
struct RotaryTable {
  int head_dim = 0, rotary_dim = 0, interleaved = 0;
  float factor = 1.0f;
  double frequency[kRotaryPairs];  // radians a position, per pair
};
struct RotaryArgs {
  const int64_t* positions = nullptr;
  const void *q = nullptr, *k = nullptr;
  void *q_out = nullptr, *k_out = nullptr;
  size_t q_stride = 0, k_stride = 0, q_out_stride = 0, k_out_stride = 0;
  int rows = 0, q_heads = 0, k_heads = 0, type = 0;
};
cudaError_t launch_rotary(const RotaryTable& t, const RotaryArgs& a, cudaStream_t s);

struct Rotary {
  RotaryTable table;
  std::vector<double> frequencies;  // radians a position
  static std::unique_ptr<Rotary> parse(const char* options_json);
  // A caller's arguments, checked, and the rotation.
  void apply(RotaryArgs a, size_t rows, cudaStream_t s) const;
};

// -------------------------------------------------------------- products
struct ScratchPool;
// A layer with e4m3 weights and an f32 scale for each block of 128 x 128.
class DenseFp8 {
 public:
  DenseFp8(const void* codes, const float* scales, size_t n, size_t k, int device);
  ~DenseFp8();
  // out (m x n) from 8-bit rows, or from values that are rounded to them.
  void forward_codes(const void* codes, const float* scales, size_t m, void* out, size_t out_stride, int type,
                     cudaStream_t s);
  void forward_host(const float* x, size_t m, float* out);
  void forward_rows(const void* x, size_t x_stride, size_t m, void* out, size_t out_stride, int type, cudaStream_t s);
  size_t n() const { return n_; }
  size_t k() const { return k_; }
  int device() const { return device_; }
  cudaStream_t stream() const { return stream_; }
  // Throws when a wait in a product that has ended ran out.
  void check_status();

 private:
  void release();
  void check(size_t m, const void* out, size_t* out_stride, int type) const;
  void product(const void* codes, const float* scales, size_t m, void* out, size_t out_stride, int type, cudaStream_t s);

  int device_;
  size_t n_, k_;
  uint8_t* codes_ = nullptr;  // packed (launch_fp8_pack)
  float* scales_ = nullptr;   // [ceil(n / 128)][ceil(k / 128)]
  cudaStream_t stream_ = nullptr;
  std::shared_ptr<ScratchPool> scratch_;  // from the first call that rounds its rows
  bool captured_ = false;
  TcMap map_;                 // of the packed weights
  int* status_ = nullptr;     // pinned: a wait inside a product ran out
};

struct Fp8Args {
  const uint8_t* w = nullptr;  // packed (launch_fp8_pack)
  const float* x_scales = nullptr;
  const float* w_scales = nullptr;
  void* out = nullptr;
  size_t out_stride = 0;
  int m = 0, n = 0, blocks = 0;  // blocks of 128 values of k
  int type = 0, tma = 0;         // tma: out has a map (make_fp8_out_map)
  int* status = nullptr;
};
// A TMA map of 8-bit numbers [rows][k], row stride k, boxes of 128 values x
// box_rows rows with the 128-byte swizzle; past either end reads zero.
cudaError_t make_fp8_map(TcMap* out, const void* base, size_t rows, size_t k, int box_rows);
// A TMA map of out, boxes of 128 bytes x box_rows with the same swizzle; its rows
// have to begin and end at whole 16 bytes.
cudaError_t make_fp8_out_map(TcMap* out, void* base, size_t rows, size_t n, size_t stride, int type, int box_rows);
int fp8_out_box(int m);
int fp8_row_box(int m);  // its box rows for m rows
// The weights [n][k] in the order that the product reads them.
size_t fp8_packed_bytes(size_t n, size_t k);
cudaError_t launch_fp8_pack(const uint8_t* codes, size_t n, size_t k, uint8_t* w, cudaStream_t s);
cudaError_t launch_fp8(const TcMap& x, const TcMap& w, const TcMap& out, const Fp8Args& a, cudaStream_t s);
// A TMA map of the packed weights: rows of 128 bytes, boxes of a unit's 64.
cudaError_t make_fp8_packed_map(TcMap* out, const void* base, size_t bytes);

}  // namespace trit
