// The host side of the row operators (rows.h): argument checks, the
// frequencies of rotary positions, and the fp8 layer's memory.
#include "rows.h"

#include <algorithm>
#include <cmath>
#include <cstring>

#include "engine.h"
#include "host.h"

namespace trit {

OnDevice::OnDevice(int device) : device_(device) {
  TRIT_CUDA(cudaGetDevice(&before_));
  if (before_ != device_) TRIT_CUDA(cudaSetDevice(device_));
}
OnDevice::~OnDevice() {
  if (before_ != device_) cudaSetDevice(before_);
}

int pointer_device(const void* p, size_t align, const char* what) {
  if (!p) throw Error(std::string(what) + " is NULL");
  if ((uintptr_t)p % align) throw Error(std::string(what) + " is not aligned to " + std::to_string(align) + " bytes");
  cudaPointerAttributes attr{};
  TRIT_CUDA(cudaPointerGetAttributes(&attr, p));
  if (attr.type != cudaMemoryTypeDevice && attr.type != cudaMemoryTypeManaged)
    throw Error(std::string(what) + " is not device memory");
  return attr.device;
}
void check_on_device(const void* p, size_t align, const char* what, int device) {
  if (pointer_device(p, align, what) != device)
    throw Error(std::string(what) + " is not device memory of CUDA device " + std::to_string(device));
}

namespace {
void check_type(int type) {
  if (type < kRowF32 || type > kRowBF16) throw Error("the type is 0 (f32), 1 (f16) or 2 (bf16)");
}
// A stride of 0 stands for packed rows.
void check_stride(size_t* stride, size_t width, const char* what) {
  if (!*stride) *stride = width;
  if (*stride < width) throw Error(std::string(what) + " is shorter than a row of " + std::to_string(width));
  if (*stride >> 40) throw Error(std::string(what) + " is 2^40 or more");
}
int check_rows(size_t rows) {
  if (rows > (size_t)INT32_MAX - 255) throw Error("a call has at most 2^31 - 256 rows");
  return (int)rows;
}
// Two tensors of a call: the same rows, or apart (rows that lie between the
// other's are the caller's to keep apart).
void check_same(const void* a, size_t a_stride, const void* b, size_t b_stride, const char* what) {
  if (a == b && a_stride != b_stride) throw Error(std::string(what) + " are one tensor with two strides");
}
}  // namespace

// ------------------------------------------------------------------ norm
void rms_norm(NormArgs a, size_t rows, size_t width, cudaStream_t s) {
  check_type(a.type);
  if (width == 0 || width > (1u << 24)) throw Error("the width is from 1 to 2^24");
  a.rows = check_rows(rows);
  a.width = (int)width;
  if (!(a.eps >= 0.0) || std::isinf(a.eps)) throw Error("eps is a number from 0 on");
  check_stride(&a.x_stride, width, "x_stride");
  if (!a.residual && a.sum) throw Error("sum without a residual");
  if (!a.residual && a.residual_stride) throw Error("residual_stride without a residual");
  if (!a.sum && a.sum_stride) throw Error("sum_stride without sum");
  if (a.residual) {
    check_stride(&a.residual_stride, width, "residual_stride");
    if (!a.sum) {
      a.sum = const_cast<void*>(a.residual);
      a.sum_stride = a.residual_stride;
    }
    check_stride(&a.sum_stride, width, "sum_stride");
    check_same(a.x, a.x_stride, a.sum, a.sum_stride, "x and sum");
    check_same(a.residual, a.residual_stride, a.sum, a.sum_stride, "residual and sum");
  }
  if (!a.weight) throw Error("weight is NULL");
  if (!a.out && !a.codes) throw Error("neither out nor codes is given");
  if (!a.codes != !a.scales) throw Error("codes and scales come together");
  if (a.out) {
    check_stride(&a.out_stride, width, "out_stride");
    check_same(a.x, a.x_stride, a.out, a.out_stride, "x and out");
    if (a.residual && a.out == a.sum) throw Error("out and sum are one tensor");
    if (a.residual && a.out == a.residual) throw Error("out and residual are one tensor");
  } else if (a.out_stride) throw Error("out_stride without out");
  if (!rows) return;
  const size_t size = row_type_size(a.type);
  const int device = pointer_device(a.x, size, "x");
  check_on_device(a.weight, a.weight_f32 ? 4 : size, "weight", device);
  if (a.residual) {
    check_on_device(a.residual, size, "residual", device);
    check_on_device(a.sum, size, "sum", device);
  }
  if (a.out) check_on_device(a.out, size, "out", device);
  if (a.codes) {
    check_on_device(a.codes, 1, "codes", device);
    check_on_device(a.scales, 4, "scales", device);
  }
  OnDevice on(device);
  TRIT_CUDA(launch_rms_norm(a, s));
}

// ---------------------------------------------------------------- rotary
namespace {

double number(const Json& v, const std::string& key, double lo, double hi) {
  if (v.kind != Json::Number || !(v.num >= lo && v.num <= hi)) {
    char text[96];
    std::snprintf(text, sizeof text, " must be a number from %g to %g", lo, hi);
    throw Error("options: " + key + text);
  }
  return v.num;
}
int whole(const Json& v, const std::string& key, int lo, int hi) {
  if (v.kind != Json::Number || v.num != std::floor(v.num) || v.num < lo || v.num > hi)
    throw Error("options: " + key + " must be a whole number from " + std::to_string(lo) + " to " + std::to_string(hi));
  return (int)v.num;
}
std::string word(const Json& v, const std::string& key) {
  if (v.kind != Json::String) throw Error("options: " + key + " must be a string");
  return v.str;
}

constexpr double kPi = 3.14159265358979323846;

}  // namespace

// Frequencies of pair i of d / 2, f_i = theta^(-2 i / d) radians a position:
//   linear  f_i / factor
//   ntk     theta * factor^(d / (d - 2)) in place of theta
//   yarn    pairs that turn more than `fast` times over `trained` positions as
//           they are, those with fewer than `slow` turns / factor, a straight
//           line over the pairs between; values times 0.1 ln(factor) + 1
//   bands   wavelengths below trained / high as they are, those above
//           trained / low / factor, a straight line over f_i between
std::unique_ptr<Rotary> Rotary::parse(const char* text) {
  if (!text || !*text) throw Error("options: head_dim is needed");
  const Json j = Json::parse(text);
  if (j.kind != Json::Object) throw Error("options: not a JSON object");
  auto r = std::make_unique<Rotary>();
  RotaryTable& t = r->table;
  int dim = 0;
  double theta = 1e6, factor = 0, trained = 0, fast = 32, slow = 1, low = 1, high = 4, attention = 0;
  std::string layout = "halves", scaling = "none";
  std::vector<std::string> given;
  bool listed = false;
  for (auto& f : j.fields) {
    const std::string& k = f.first;
    const Json& v = f.second;
    given.push_back(k);
    if (k == "head_dim") t.head_dim = whole(v, k, 2, 2 * kRotaryPairs);
    else if (k == "rotary_dim") dim = whole(v, k, 2, 2 * kRotaryPairs);
    else if (k == "theta") theta = number(v, k, 1.0 + 1e-9, 1e30);
    else if (k == "layout") layout = word(v, k);
    else if (k == "scaling") scaling = word(v, k);
    else if (k == "factor") factor = number(v, k, 1e-6, 1e6);
    else if (k == "trained") trained = number(v, k, 1, 1e12);
    else if (k == "fast") fast = number(v, k, 1e-6, 1e9);
    else if (k == "slow") slow = number(v, k, 1e-6, 1e9);
    else if (k == "low") low = number(v, k, 1e-6, 1e9);
    else if (k == "high") high = number(v, k, 1e-6, 1e9);
    else if (k == "attention_factor") attention = number(v, k, 1e-6, 1e6);
    else if (k == "frequencies") {
      if (v.kind != Json::Array) throw Error("options: frequencies must be an array");
      listed = true;
      for (auto& x : v.items) r->frequencies.push_back(number(x, "each of frequencies", -1e9, 1e9));
    } else throw Error("options: unknown key " + k);
  }
  if (!t.head_dim) throw Error("options: head_dim is needed");
  if (t.head_dim % 2) throw Error("options: head_dim must be even");
  if (!dim) dim = t.head_dim;
  if (dim % 2 || dim > t.head_dim) throw Error("options: rotary_dim must be even and at most head_dim");
  if (layout != "halves" && layout != "interleaved") throw Error("options: layout is \"halves\" or \"interleaved\"");
  const bool linear = scaling == "linear", ntk = scaling == "ntk", yarn = scaling == "yarn", bands = scaling == "bands";
  if (scaling != "none" && !linear && !ntk && !yarn && !bands)
    throw Error("options: scaling is \"none\", \"linear\", \"ntk\", \"yarn\" or \"bands\"");
  // A key that the scaling does not read would be lost without a word.
  const auto only = [&](const char* key, bool read) {
    if (!read && std::find(given.begin(), given.end(), key) != given.end())
      throw Error(std::string("options: ") + key + " is not a setting of " + (listed ? "given frequencies" : "scaling \"" + scaling + "\""));
  };
  if (listed && scaling != "none") throw Error("options: given frequencies are not scaled");
  only("theta", !listed);
  only("factor", linear || ntk || yarn || bands);
  only("trained", yarn || bands);
  only("fast", yarn);
  only("slow", yarn);
  only("low", bands);
  only("high", bands);
  if (scaling != "none" && factor == 0) throw Error("options: scaling \"" + scaling + "\" needs factor");
  if ((yarn || bands) && trained == 0) throw Error("options: scaling \"" + scaling + "\" needs trained");
  if (yarn && fast <= slow) throw Error("options: fast must be more than slow");
  if (bands && high <= low) throw Error("options: high must be more than low");

  const int pairs = dim / 2;
  t.rotary_dim = dim;
  t.interleaved = layout == "interleaved";
  t.factor = 1.0f;
  if (listed) {
    if ((int)r->frequencies.size() != pairs)
      throw Error("options: " + std::to_string(r->frequencies.size()) + " frequencies for " + std::to_string(pairs) + " pairs");
  } else {
    // Two values are one pair, of frequency 1 whatever the base.
    if (ntk && dim > 2) theta *= std::pow(factor, (double)dim / (dim - 2));
    const auto pair_of = [&](double turns) { return dim * std::log(trained / (turns * 2 * kPi)) / (2 * std::log(theta)); };
    const double first = yarn ? std::max(std::floor(pair_of(fast)), 0.0) : 0;
    const double last = yarn ? std::min(std::ceil(pair_of(slow)), dim - 1.0) : 0;
    for (int i = 0; i < pairs; ++i) {
      const double f = std::pow(theta, -2.0 * i / dim);
      double keep = 1;  // the part of f that is not scaled
      if (linear) keep = 0;
      if (yarn) keep = 1 - std::min(std::max((i - first) / std::max(last - first, 0.001), 0.0), 1.0);
      if (bands) keep = std::min(std::max((trained * f / (2 * kPi) - low) / (high - low), 0.0), 1.0);
      r->frequencies.push_back(scaling == "none" || ntk ? f : f / factor * (1 - keep) + f * keep);
    }
    if (yarn) t.factor = (float)(0.1 * std::log(factor) + 1);
    if (yarn && factor < 1) t.factor = 1.0f;
  }
  if (attention > 0) t.factor = (float)attention;
  std::copy(r->frequencies.begin(), r->frequencies.end(), t.frequency);
  return r;
}

void Rotary::apply(RotaryArgs a, size_t rows, cudaStream_t s) const {
  check_type(a.type);
  a.rows = check_rows(rows);
  // (Two heads a thread and as little as a team a block: 65535 blocks in y.)
  if (a.q_heads < 0 || a.k_heads < 0 || a.q_heads > 65535 || a.k_heads > 65535) throw Error("heads are from 0 to 65535");
  if (!a.q_heads && !a.k_heads) throw Error("neither q nor k has heads");
  int device = -1;
  const size_t size = row_type_size(a.type);
  const auto tensor = [&](const void*& x, size_t& x_stride, void*& out, size_t& out_stride, int heads, const char* name) {
    const std::string n = name;
    if (!heads) {
      if (x || out) throw Error(n + " is given with no heads");
      x_stride = out_stride = 0;
      return;
    }
    const size_t width = (size_t)heads * table.head_dim;
    check_stride(&x_stride, width, (n + "_stride").c_str());
    if (!out) {
      if (out_stride) throw Error(n + "_out_stride without " + n + "_out");
      out = const_cast<void*>(x);
      out_stride = x_stride;
    }
    check_stride(&out_stride, width, (n + "_out_stride").c_str());
    check_same(x, x_stride, out, out_stride, (n + " and " + n + "_out").c_str());
    if (!rows) return;
    if (device < 0) device = pointer_device(x, size, name);
    else check_on_device(x, size, name, device);
    check_on_device(out, size, (n + "_out").c_str(), device);
  };
  tensor(a.q, a.q_stride, a.q_out, a.q_out_stride, a.q_heads, "q");
  tensor(a.k, a.k_stride, a.k_out, a.k_out_stride, a.k_heads, "k");
  if (a.q_out && a.q_out == a.k_out) throw Error("q_out and k_out are one tensor");
  if (a.q_out && a.q_out == a.k) throw Error("q_out and k are one tensor");
  if (a.k_out && a.k_out == a.q) throw Error("k_out and q are one tensor");
  if (!rows) return;
  check_on_device(a.positions, 8, "positions", device);
  OnDevice on(device);
  TRIT_CUDA(launch_rotary(table, a, s));
}

// -------------------------------------------------------------- products
// Scratch of calls that round their rows first, shared by a device's layers and
// given back with the last of them. Memory of a pool comes and goes in the
// order of the call's stream, so calls on several streams may overlap; the pool
// keeps what it has across synchronisations.
struct ScratchPool {
  cudaMemPool_t pool = nullptr;
  explicit ScratchPool(int device) {
    cudaMemPoolProps props{};
    props.allocType = cudaMemAllocationTypePinned;
    props.location.type = cudaMemLocationTypeDevice;
    props.location.id = device;
    TRIT_CUDA(cudaMemPoolCreate(&pool, &props));
    uint64_t keep = UINT64_MAX;
    cudaMemPoolSetAttribute(pool, cudaMemPoolAttrReleaseThreshold, &keep);
  }
  ~ScratchPool() { cudaMemPoolDestroy(pool); }
  ScratchPool(const ScratchPool&) = delete;
  ScratchPool& operator=(const ScratchPool&) = delete;
  static std::shared_ptr<ScratchPool> of(int device) {
    static std::mutex mu;
    static std::weak_ptr<ScratchPool> pools[kMaxDevices];
    if (device < 0 || device >= kMaxDevices) throw Error("device index out of range");
    std::lock_guard<std::mutex> lock(mu);
    std::shared_ptr<ScratchPool> p = pools[device].lock();
    if (!p) pools[device] = p = std::make_shared<ScratchPool>(device);
    return p;
  }
};

namespace {
bool is_capturing(cudaStream_t s) {
  cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
  TRIT_CUDA(cudaStreamIsCapturing(s, &st));
  return st != cudaStreamCaptureStatusNone;
}
}  // namespace

DenseFp8::DenseFp8(const void* codes, const float* scales, size_t n, size_t k, int device) : device_(device), n_(n), k_(k) {
  if (!n || n > (size_t)INT32_MAX - 255) throw Error("n is from 1 to 2^31 - 256");
  if (!k || k % 16 || k > (1u << 24)) throw Error("k is a multiple of 16 up to 2^24");
  OnDevice on(device);
  const size_t blocks = ((n + 127) / 128) * ((k + 127) / 128);
  try {
    TRIT_CUDA(cudaMalloc(&codes_, fp8_packed_bytes(n, k)));
    TRIT_CUDA(cudaMalloc(&scales_, blocks * 4));
    TRIT_CUDA(cudaStreamCreateWithFlags(&stream_, cudaStreamNonBlocking));
    TRIT_CUDA(cudaHostAlloc(&status_, 4, cudaHostAllocDefault));
    *status_ = 0;
    // On the layer's stream: a plain cudaMemcpy may return before its last
    // bytes are there, and that stream does not wait for it.
    uint8_t* raw = nullptr;
    TRIT_CUDA(cudaMalloc(&raw, n * k));
    cudaError_t e = cudaMemcpyAsync(scales_, scales, blocks * 4, cudaMemcpyHostToDevice, stream_);
    if (e == cudaSuccess) e = cudaMemcpyAsync(raw, codes, n * k, cudaMemcpyHostToDevice, stream_);
    if (e == cudaSuccess) e = launch_fp8_pack(raw, n, k, codes_, stream_);
    if (e == cudaSuccess) e = cudaStreamSynchronize(stream_);
    cudaFree(raw);
    TRIT_CUDA(e);
    TRIT_CUDA(make_fp8_packed_map(&map_, codes_, fp8_packed_bytes(n, k)));
  } catch (...) {
    release();
    throw;
  }
}
DenseFp8::~DenseFp8() {
  int before = 0;
  cudaGetDevice(&before);
  cudaSetDevice(device_);
  release();
  scratch_.reset();
  // What graphs that are gone had as scratch.
  if (captured_) cudaDeviceGraphMemTrim(device_);
  cudaSetDevice(before);
}
void DenseFp8::release() {
  if (codes_) cudaFree(codes_);
  if (scales_) cudaFree(scales_);
  if (status_) cudaFreeHost(status_);
  if (stream_) cudaStreamDestroy(stream_);
}

void DenseFp8::check(size_t m, const void* out, size_t* out_stride, int type) const {
  check_type(type);
  check_stride(out_stride, n_, "out_stride");
  check_rows(m);
  if (m) check_on_device(out, row_type_size(type), "out", device_);
}

void DenseFp8::check_status() {
  if (!*(volatile int*)status_) return;
  *(volatile int*)status_ = 0;
  throw Error("a product before this one gave up waiting for its pipeline");
}

void DenseFp8::product(const void* codes, const float* scales, size_t m, void* out, size_t out_stride, int type,
                       cudaStream_t s) {
  check_status();
  TcMap map;
  TRIT_CUDA(make_fp8_map(&map, codes, m, k_, fp8_row_box((int)m)));
  Fp8Args a;
  a.w = codes_;
  a.x_scales = scales;
  a.w_scales = scales_;
  a.out = out;
  a.out_stride = out_stride;
  a.m = (int)m;
  a.n = (int)n_;
  a.blocks = (int)((k_ + kFp8Group - 1) / kFp8Group);
  a.type = type;
  a.status = status_;
  TcMap out_map{};
  a.tma = make_fp8_out_map(&out_map, out, m, n_, out_stride, type, fp8_out_box((int)m)) == cudaSuccess;
  TRIT_CUDA(launch_fp8(map, map_, out_map, a, s));
}

void DenseFp8::forward_codes(const void* codes, const float* scales, size_t m, void* out, size_t out_stride, int type,
                             cudaStream_t s) {
  check(m, out, &out_stride, type);
  if (!m) return;
  check_on_device(codes, 16, "codes", device_);
  check_on_device(scales, 4, "scales", device_);
  OnDevice on(device_);
  product(codes, scales, m, out, out_stride, type, s);
}

void DenseFp8::forward_rows(const void* x, size_t x_stride, size_t m, void* out, size_t out_stride, int type,
                            cudaStream_t s) {
  check(m, out, &out_stride, type);
  check_stride(&x_stride, k_, "x_stride");
  if (!m) return;
  check_on_device(x, row_type_size(type), "x", device_);
  OnDevice on(device_);
  const size_t codes = (m * k_ + 255) / 256 * 256, bytes = codes + m * ((k_ + kFp8Group - 1) / kFp8Group) * 4;
  uint8_t* scratch = nullptr;
  // A captured call's scratch belongs to its graph.
  if (is_capturing(s)) {
    TRIT_CUDA(cudaMallocAsync(&scratch, bytes, s));
    captured_ = true;
  } else {
    if (!scratch_) scratch_ = ScratchPool::of(device_);
    TRIT_CUDA(cudaMallocFromPoolAsync(&scratch, bytes, scratch_->pool, s));
  }
  NormArgs q;
  q.x = x;
  q.x_stride = x_stride;
  q.rows = (int)m;
  q.width = (int)k_;
  q.type = type;
  q.codes = scratch;
  q.scales = (float*)(scratch + codes);
  try {
    TRIT_CUDA(launch_rms_norm(q, s));
    product(scratch, q.scales, m, out, out_stride, type, s);
  } catch (...) {
    cudaFreeAsync(scratch, s);
    throw;
  }
  TRIT_CUDA(cudaFreeAsync(scratch, s));
}

// Rows and outputs in host memory; waits.
void DenseFp8::forward_host(const float* x, size_t m, float* out) {
  check_rows(m);
  if (!m) return;
  OnDevice on(device_);
  struct Buffers {
    float *x = nullptr, *y = nullptr;
    ~Buffers() {
      if (x) cudaFree(x);
      if (y) cudaFree(y);
    }
  } b;
  TRIT_CUDA(cudaMalloc(&b.x, m * k_ * 4));
  TRIT_CUDA(cudaMalloc(&b.y, m * n_ * 4));
  TRIT_CUDA(cudaMemcpyAsync(b.x, x, m * k_ * 4, cudaMemcpyHostToDevice, stream_));
  forward_rows(b.x, 0, m, b.y, 0, kRowF32, stream_);
  TRIT_CUDA(cudaMemcpyAsync(out, b.y, m * n_ * 4, cudaMemcpyDeviceToHost, stream_));
  TRIT_CUDA(cudaStreamSynchronize(stream_));
  check_status();
}

}  // namespace trit
