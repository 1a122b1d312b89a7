// The host side of the 8-bit key/value cache (kv8.h): pages, sequences,
// argument checks, and the order of work on different streams.
#include <algorithm>
#include <cmath>

#include "engine.h"
#include "kv8.h"

namespace trit {

KvOptions KvOptions::parse(const char* text) {
  if (!text || !*text) throw Error("options: layers, kv_heads and pages are needed");
  Json j = Json::parse(text);
  if (j.kind != Json::Object) throw Error("options: not a JSON object");
  KvOptions o;
  for (auto& f : j.fields) {
    const std::string& k = f.first;
    auto count = [&](int lo, int hi) {
      const Json& v = f.second;
      if (v.kind != Json::Number || v.num != std::floor(v.num) || v.num < lo || v.num > hi)
        throw Error("options: " + k + " must be a whole number from " + std::to_string(lo) + " to " + std::to_string(hi));
      return (int)v.num;
    };
    if (k == "device") o.device = count(0, 63);
    else if (k == "layers") o.layers = count(1, 4096);
    else if (k == "kv_heads") o.kv_heads = count(1, 1024);
    else if (k == "head_dim") o.hd = count(1, 1024);
    else if (k == "page_tokens") o.page = count(1, 4096);
    else if (k == "pages") o.pages = count(1, 1 << 26);
    else if (k == "sequences") o.sequences = count(1, 65536);
    else if (k == "max_tokens") o.max_tokens = count(1, 1 << 26);
    else throw Error("options: unknown key " + k);
  }
  if (!o.kv_heads) throw Error("options: kv_heads is needed");
  if (!o.pages) throw Error("options: pages is needed");
  if (o.hd != 64 && o.hd != 128) throw Error("options: head_dim is 64 or 128");
  if (o.page != 16 && o.page != 32 && o.page != 64 && o.page != 128)
    throw Error("options: page_tokens is 16, 32, 64 or 128");
  if ((size_t)o.layers * 2 * o.kv_heads * o.page * o.hd >> 32)
    throw Error("options: a page of all layers and heads holds 4 GB or more");
  if ((size_t)o.sequences * std::max(1, o.max_tokens / o.page) > (size_t)INT32_MAX)
    throw Error("options: sequences * max_tokens / page_tokens is 2^31 or more");
  return o;
}

KvCache::KvCache(const KvOptions& o) : opt_(o) {
  TRIT_CUDA(cudaSetDevice(o.device));
  view_.layers = o.layers;
  view_.kv_heads = o.kv_heads;
  view_.hd = o.hd;
  view_.page = o.page;
  while ((1 << view_.page_shift) < o.page) ++view_.page_shift;
  view_.pages_per_seq = std::max(1, o.max_tokens / o.page);
  const size_t blocks = (size_t)o.layers * 2 * o.kv_heads, block = (size_t)o.page * o.hd;
  const size_t open = (size_t)o.sequences * blocks * block * 2, table = (size_t)o.sequences * view_.pages_per_seq * 4;
  try {
    TRIT_CUDA(cudaMalloc(&view_.codes, (size_t)o.pages * blocks * block));
    TRIT_CUDA(cudaMalloc(&view_.scales, (size_t)o.pages * blocks * 4));
    TRIT_CUDA(cudaMalloc(&view_.open, open));
    TRIT_CUDA(cudaMalloc(&view_.table, table));
    TRIT_CUDA(cudaMalloc(&moves_, (size_t)o.pages * 8));
    TRIT_CUDA(cudaMalloc(&remap_, (size_t)o.pages * 8));
    TRIT_CUDA(cudaMemset(remap_, 0, (size_t)o.pages * 8));
    TRIT_CUDA(cudaMalloc(&workspace_, kKvWorkspace));
    TRIT_CUDA(cudaHostAlloc(&status_, 4, cudaHostAllocDefault));
    *status_ = 0;
    // The attention reads whole steps of 16 positions of an open page, also
    // those behind its end: they must hold numbers from the start.
    TRIT_CUDA(cudaMemset(view_.open, 0, open));
    TRIT_CUDA(cudaMemset(workspace_, 0, kKvHead * 4));
    TRIT_CUDA(cudaMemset(view_.table, 0, table));
    TRIT_CUDA(cudaDeviceSynchronize());
    TRIT_CUDA(cudaEventCreateWithFlags(&order_, cudaEventDisableTiming));
  } catch (...) {
    release_memory();
    throw;
  }
  seqs_.resize(o.sequences);
  refs_.assign(o.pages, 0);
  for (int i = 0; i < o.sequences; ++i) free_seqs_.push(i);
  for (int i = 0; i < o.pages; ++i) free_pages_.push(i);
}

KvCache::~KvCache() { release_memory(); }

void KvCache::release_memory() {
  cudaSetDevice(opt_.device);
  void* bufs[] = {view_.codes, view_.scales, view_.open, view_.table, moves_, remap_, workspace_};
  for (void* b : bufs)
    if (b) cudaFree(b);
  if (status_) cudaFreeHost(status_);
  if (order_) cudaEventDestroy(order_);
}

KvCache::Seq& KvCache::seq(int id) {
  if (id < 0 || id >= opt_.sequences || !seqs_[id].live) throw Error("sequence " + std::to_string(id) + " is not open");
  return seqs_[id];
}
const KvCache::Seq& KvCache::seq(int id) const { return const_cast<KvCache*>(this)->seq(id); }

int KvCache::new_seq() {
  const int id = free_seqs_.top();
  free_seqs_.pop();
  Seq& q = seqs_[id];
  q.live = true;
  q.len = 0;
  q.pages.clear();
  q.filled.assign(opt_.layers, 0);
  return id;
}

void KvCache::share(Seq& c, const Seq& p, int64_t tokens) {
  c.len = tokens;
  c.pages.assign(p.pages.begin(), p.pages.begin() + tokens / opt_.page);
  c.filled.assign(opt_.layers, tokens);
  for (int pg : c.pages) ++refs_[pg];
}

void KvCache::check_filled(int id) const {
  const Seq& q = seq(id);
  for (int64_t f : q.filled)
    if (f != q.len) throw Error("sequence " + std::to_string(id) + " has positions that were not appended yet");
}

void KvCache::drop_pages(Seq& q) {
  for (int p : q.pages)
    if (--refs_[p] == 0) free_pages_.push(p);
  q.pages.clear();
}

void KvCache::check_layer(int layer) const {
  if (layer < 0 || layer >= opt_.layers)
    throw Error("layer " + std::to_string(layer) + " of a cache of " + std::to_string(opt_.layers) + " layers");
}

namespace {
bool is_capturing(cudaStream_t s) {
  cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
  TRIT_CUDA(cudaStreamIsCapturing(s, &st));
  return st != cudaStreamCaptureStatusNone;
}
}  // namespace

void KvCache::refuse_capture(cudaStream_t s, const char* what) {
  TRIT_CUDA(cudaSetDevice(opt_.device));
  capturing_ = false;
  if (is_capturing(s))
    throw Error(std::string(what) + ": the stream is being captured, and a replay would write the same positions again");
}

void KvCache::enter(cudaStream_t s, const char* what, bool may_capture) {
  TRIT_CUDA(cudaSetDevice(opt_.device));
  if (take_failure()) throw Error("an attention call before this one gave up waiting for its pipeline");
  if (may_capture) capturing_ = is_capturing(s);
  else refuse_capture(s, what);
  if (capturing_ || !used_) return;
  unsigned long long id = 0;
  TRIT_CUDA(cudaStreamGetId(s, &id));
  if (id != last_stream_) TRIT_CUDA(cudaStreamWaitEvent(s, order_, 0));
}

void KvCache::leave(cudaStream_t s) {
  if (capturing_) return;
  TRIT_CUDA(cudaEventRecord(order_, s));
  TRIT_CUDA(cudaStreamGetId(s, &last_stream_));
  used_ = true;
}

void KvCache::set_entries(const std::vector<std::pair<int, int>>& entries, cudaStream_t s) {
  KvEntries e;
  for (size_t i = 0; i < entries.size(); ++i) {
    e.index[e.n] = entries[i].first;
    e.page[e.n] = entries[i].second;
    if (++e.n == kKvRuns * 3 || i + 1 == entries.size()) {
      TRIT_CUDA(launch_kv_table(view_, e, s));
      e.n = 0;
    }
  }
}

int64_t KvCache::length(int id) const { return seq(id).len; }

void KvCache::open(size_t n, int* out) {
  if (n > free_seqs_.size())
    throw Error(std::to_string(n) + " sequences asked, " + std::to_string(free_seqs_.size()) + " of " +
                std::to_string(opt_.sequences) + " are free");
  for (size_t i = 0; i < n; ++i) out[i] = new_seq();
}

void KvCache::fork(const int* ids, const int64_t* tokens, size_t n, int* out, cudaStream_t s) {
  if (n > free_seqs_.size())
    throw Error(std::to_string(n) + " sequences asked, " + std::to_string(free_seqs_.size()) + " of " +
                std::to_string(opt_.sequences) + " are free");
  for (size_t i = 0; i < n; ++i) {
    const Seq& p = seq(ids[i]);
    if (tokens && (tokens[i] < 0 || tokens[i] > p.len))
      throw Error("a fork at " + std::to_string(tokens[i]) + " of a sequence of " + std::to_string(p.len) + " positions");
    check_filled(ids[i]);
  }
  if (!n) return;
  enter(s, "fork");
  KvRuns runs;
  for (size_t i = 0; i < n; ++i) {
    const int id = new_seq();
    out[i] = id;
    Seq& c = seqs_[id];
    const Seq& p = seqs_[ids[i]];
    share(c, p, tokens ? tokens[i] : p.len);
    runs.run[runs.n++] = KvRun{id, ids[i], 0, (int)c.len, (int)p.len};
    if (runs.n == kKvRuns || i + 1 == n) {
      TRIT_CUDA(launch_kv_fork(view_, runs, true, s));
      runs.n = 0;
    }
  }
  leave(s);
}

void KvCache::copy(const int* ids, size_t n, int* out, cudaStream_t s) {
  size_t pages = 0;
  for (size_t i = 0; i < n; ++i) {
    const Seq& p = seq(ids[i]);
    check_filled(ids[i]);
    pages += p.pages.size();
  }
  if (n > free_seqs_.size())
    throw Error(std::to_string(n) + " sequences asked, " + std::to_string(free_seqs_.size()) + " of " +
                std::to_string(opt_.sequences) + " are free");
  if (pages > free_pages_.size())
    throw Error(std::to_string(pages) + " pages asked, " + std::to_string(free_pages_.size()) + " of " +
                std::to_string(opt_.pages) + " are free");
  if (!n) return;
  enter(s, "copy");
  std::vector<int> moves;
  std::vector<std::pair<int, int>> entries;
  moves.reserve(2 * pages);
  KvRuns runs;
  for (size_t i = 0; i < n; ++i) {
    const int id = new_seq();
    out[i] = id;
    Seq& c = seqs_[id];
    const Seq& p = seqs_[ids[i]];
    c.len = p.len;
    c.filled.assign(opt_.layers, c.len);
    for (size_t k = 0; k < p.pages.size(); ++k) {
      const int pg = free_pages_.top();
      free_pages_.pop();
      refs_[pg] = 1;
      c.pages.push_back(pg);
      moves.push_back(p.pages[k]);
      moves.push_back(pg);
      entries.emplace_back(id * view_.pages_per_seq + (int)k, pg);
    }
    runs.run[runs.n++] = KvRun{id, ids[i], 0, (int)c.len, (int)p.len};
    if (runs.n == kKvRuns || i + 1 == n) {
      TRIT_CUDA(launch_kv_fork(view_, runs, false, s));
      runs.n = 0;
    }
  }
  // The list's copy is staged before cudaMemcpyAsync returns (pageable
  // memory), and no page is both read and written.
  if (pages) {
    TRIT_CUDA(cudaMemcpyAsync(moves_, moves.data(), moves.size() * 4, cudaMemcpyHostToDevice, s));
    TRIT_CUDA(launch_kv_move(view_, moves_, (int)pages, nullptr, 0, s));
    set_entries(entries, s);
  }
  leave(s);
}

void KvCache::release(const int* ids, size_t n) {
  std::vector<char> seen(opt_.sequences, 0);
  for (size_t i = 0; i < n; ++i) {
    seq(ids[i]);
    if (seen[ids[i]]++) throw Error("sequence " + std::to_string(ids[i]) + " is released twice");
  }
  for (size_t i = 0; i < n; ++i) {
    Seq& q = seqs_[ids[i]];
    drop_pages(q);
    q.live = false;
    free_seqs_.push(ids[i]);
  }
}

void KvCache::extend(const int* ids, const int64_t* counts, size_t n, cudaStream_t s) {
  std::vector<char> seen(opt_.sequences, 0);
  size_t pages = 0;
  bool grows = false;
  for (size_t i = 0; i < n; ++i) {
    const Seq& q = seq(ids[i]);
    if (seen[ids[i]]++) throw Error("sequence " + std::to_string(ids[i]) + " is named twice");
    if (counts[i] < 0) throw Error("a negative count");
    if (counts[i] > opt_.max_tokens - q.len)
      throw Error("sequence " + std::to_string(ids[i]) + ": " + std::to_string(q.len) + " + " + std::to_string(counts[i]) +
                  " positions exceed max_tokens " + std::to_string(opt_.max_tokens));
    pages += (q.len + counts[i]) / opt_.page - q.pages.size();
    grows |= counts[i] > 0;
  }
  if (pages > free_pages_.size())
    throw Error(std::to_string(pages) + " pages asked, " + std::to_string(free_pages_.size()) + " of " +
                std::to_string(opt_.pages) + " are free");
  if (pages) enter(s, "extend");
  else if (grows) refuse_capture(s, "extend");
  std::vector<std::pair<int, int>> entries;
  for (size_t i = 0; i < n; ++i) {
    Seq& q = seqs_[ids[i]];
    q.len += counts[i];
    while ((int64_t)q.pages.size() < q.len / opt_.page) {
      const int pg = free_pages_.top();
      free_pages_.pop();
      refs_[pg] = 1;
      entries.emplace_back(ids[i] * view_.pages_per_seq + (int)q.pages.size(), pg);
      q.pages.push_back(pg);
    }
  }
  if (!pages) return;
  set_entries(entries, s);
  leave(s);
}

namespace {
void check_type(int type) {
  if (type < kKvF32 || type > kKvBF16) throw Error("the type is 0 (f32), 1 (f16) or 2 (bf16)");
}
size_t type_size(int type) { return type == kKvF32 ? 4 : 2; }
void check_pointer(const void* p, int type, const char* what, int device) {
  if (!p) throw Error(std::string(what) + " is NULL");
  if ((uintptr_t)p % type_size(type)) throw Error(std::string(what) + " is not aligned to its type");
  cudaPointerAttributes attr{};
  TRIT_CUDA(cudaPointerGetAttributes(&attr, p));
  if ((attr.type != cudaMemoryTypeDevice && attr.type != cudaMemoryTypeManaged) || attr.device != device)
    throw Error(std::string(what) + " is not device memory of CUDA device " + std::to_string(device));
}
}  // namespace

void KvCache::append(int layer, const int* ids, const int64_t* counts, size_t n, const void* k, size_t k_stride,
                     const void* v, size_t v_stride, int type, cudaStream_t s) {
  check_layer(layer);
  check_type(type);
  const size_t width = (size_t)opt_.kv_heads * opt_.hd;
  if (!k_stride) k_stride = width;
  if (!v_stride) v_stride = width;
  if (k_stride < width || v_stride < width) throw Error("a stride is shorter than a row of " + std::to_string(width));
  std::vector<char> seen(opt_.sequences, 0);
  int64_t total = 0;
  for (size_t i = 0; i < n; ++i) {
    const Seq& q = seq(ids[i]);
    if (seen[ids[i]]++) throw Error("sequence " + std::to_string(ids[i]) + " is named twice");
    if (counts[i] < 0 || counts[i] > q.len) throw Error("a count of " + std::to_string(counts[i]) + " for a sequence of " +
                                                        std::to_string(q.len) + " positions");
    if (q.filled[layer] != q.len - counts[i])
      throw Error("sequence " + std::to_string(ids[i]) + ", layer " + std::to_string(layer) + ": positions " +
                  std::to_string(q.len - counts[i]) + " on are appended, the cache holds " +
                  std::to_string(q.filled[layer]) + " (extend first, then append every position once)");
    total += counts[i];
  }
  if (total > INT32_MAX) throw Error("more than 2^31 rows in a call");
  if (!total) return;
  check_pointer(k, type, "k", opt_.device);
  check_pointer(v, type, "v", opt_.device);
  enter(s, "append");
  KvRuns runs;
  int row = 0, most = 0;
  for (size_t i = 0; i < n; ++i) {
    Seq& q = seqs_[ids[i]];
    if (counts[i]) {
      runs.run[runs.n++] = KvRun{ids[i], (int)(q.len - counts[i]), row, (int)counts[i], (int)q.len};
      most = std::max(most, (int)counts[i]);
      row += (int)counts[i];
      q.filled[layer] = q.len;
    }
    if (runs.n == kKvRuns || i + 1 == n) {
      TRIT_CUDA(launch_kv_append(view_, runs, layer, k, k_stride, v, v_stride, type, most, s));
      runs.n = most = 0;
    }
  }
  leave(s);
}

void KvCache::attend(int layer, const int* ids, const int64_t* counts, size_t n, const void* q, size_t q_stride,
                     int heads, int type, float scale, bool causal, void* out, size_t out_stride, cudaStream_t s) {
  check_layer(layer);
  check_type(type);
  if (heads <= 0 || heads % opt_.kv_heads || heads > 65536)
    throw Error(std::to_string(heads) + " query heads do not share " + std::to_string(opt_.kv_heads) +
                " key heads evenly");
  const size_t width = (size_t)heads * opt_.hd;
  if (!q_stride) q_stride = width;
  if (!out_stride) out_stride = width;
  if (q_stride < width || out_stride < width)
    throw Error("a stride is shorter than a row of " + std::to_string(width));
  int64_t total = 0;
  for (size_t i = 0; i < n; ++i) {
    const Seq& p = seq(ids[i]);
    if (counts[i] < 0) throw Error("a negative count");
    if (causal && counts[i] > p.len)
      throw Error(std::to_string(counts[i]) + " causal rows for a sequence of " + std::to_string(p.len) + " positions");
    if (p.filled[layer] != p.len)
      throw Error("sequence " + std::to_string(ids[i]) + " has positions that were not appended yet");
    // Rows without causal order are not bounded by the sequence: checked
    // before they add up past 64 bits.
    if (counts[i] > INT32_MAX || (total += counts[i]) > INT32_MAX) throw Error("more than 2^31 rows in a call");
  }
  if (total * (heads / opt_.kv_heads) > INT32_MAX) throw Error("more than 2^31 rows of heads in a call");
  if (!total) return;
  check_pointer(q, type, "q", opt_.device);
  check_pointer(out, type, "out", opt_.device);
  enter(s, "attend", true);
  KvAttendArgs a;
  a.q = q;
  a.out = out;
  a.q_stride = q_stride;
  a.out_stride = out_stride;
  a.type = type;
  a.heads = heads;
  a.layer = layer;
  a.causal = causal ? 1 : 0;
  a.scale = scale;
  const int group = heads / opt_.kv_heads;
  KvRuns few, many;
  int row = 0;
  for (size_t i = 0; i < n; ++i) {
    const Seq& p = seqs_[ids[i]];
    if (!counts[i]) continue;
    KvRuns& to = kv_prompt_run(counts[i], group, type, total * heads) ? many : few;
    to.run[to.n++] = KvRun{ids[i], (int)(p.len - counts[i]), row, (int)counts[i], (int)p.len};
    row += (int)counts[i];
    if (to.n == kKvRuns) attend_runs(to, a, &to == &many, s);
  }
  attend_runs(few, a, false, s);
  attend_runs(many, a, true, s);
  leave(s);
}

void KvCache::attend_runs(KvRuns& runs, KvAttendArgs& a, bool prompt, cudaStream_t s) {
  if (!runs.n) return;
  a.max_len = 0;
  for (int i = 0; i < runs.n; ++i) a.max_len = std::max(a.max_len, runs.run[i].len);
  const KvAttendPlan plan = prompt ? plan_kv_prompt(view_, runs, a) : plan_kv_attend(view_, runs, a);
  void* ws = workspace_;
  if (capturing_ && plan.workspace) {
    // A captured call's workspace belongs to its graph: two graphs of one
    // cache, or a graph and a call, may then run at once.
    TRIT_CUDA(cudaMallocAsync(&ws, plan.workspace, s));
    TRIT_CUDA(cudaMemsetAsync(ws, 0, kKvHead * 4, s));
  }
  if (prompt) TRIT_CUDA(launch_kv_prompt(view_, runs, a, plan, ws, status_, s));
  else TRIT_CUDA(launch_kv_attend(view_, runs, a, plan, ws, s));
  if (capturing_ && plan.workspace) TRIT_CUDA(cudaFreeAsync(ws, s));
  runs.n = 0;
}

bool KvCache::take_failure() {
  const bool failed = *(volatile int*)status_ != 0;
  *(volatile int*)status_ = 0;
  return failed;
}

void KvCache::read(int layer, const int* ids, const int64_t* firsts, const int64_t* counts, size_t n, void* k, void* v,
                   int type, cudaStream_t s) {
  check_layer(layer);
  check_type(type);
  int64_t total = 0;
  for (size_t i = 0; i < n; ++i) {
    const Seq& p = seq(ids[i]);
    if (firsts[i] < 0 || counts[i] < 0 || counts[i] > p.filled[layer] || firsts[i] > p.filled[layer] - counts[i])
      throw Error("positions " + std::to_string(firsts[i]) + " + " + std::to_string(counts[i]) + " of a sequence with " +
                  std::to_string(p.filled[layer]) + " in layer " + std::to_string(layer));
    total += counts[i];
  }
  if (total > INT32_MAX) throw Error("more than 2^31 rows in a call");
  if (!total || (!k && !v)) return;
  if (k) check_pointer(k, type, "k", opt_.device);
  if (v) check_pointer(v, type, "v", opt_.device);
  enter(s, "read", true);
  KvRuns runs;
  int row = 0, most = 0;
  for (size_t i = 0; i < n; ++i) {
    if (counts[i]) {
      runs.run[runs.n++] = KvRun{ids[i], (int)firsts[i], row, (int)counts[i],
                                  (int)seqs_[ids[i]].filled[layer]};
      most = std::max(most, (int)counts[i]);
      row += (int)counts[i];
    }
    if (runs.n == kKvRuns || i + 1 == n) {
      TRIT_CUDA(launch_kv_read(view_, runs, layer, k, v, type, most, s));
      runs.n = most = 0;
    }
  }
  leave(s);
}

// The pages in use move to the front of the pool: each one behind the count
// of used pages takes a free place before it, so no page is both a source
// and a target.
int64_t KvCache::compact(cudaStream_t s) {
  const int used = pages_used();
  std::vector<int> to(opt_.pages, -1), moves;
  int hole = 0;
  for (int p = used; p < opt_.pages; ++p) {
    if (!refs_[p]) continue;
    while (refs_[hole]) ++hole;
    to[p] = hole;
    moves.push_back(p);
    moves.push_back(hole++);
  }
  if (moves.empty()) return 0;
  enter(s, "compact");
  const int n = (int)(moves.size() / 2);
  TRIT_CUDA(cudaMemcpyAsync(moves_, moves.data(), moves.size() * 4, cudaMemcpyHostToDevice, s));
  ++epoch_;
  TRIT_CUDA(launch_kv_move(view_, moves_, n, remap_, epoch_, s));
  TRIT_CUDA(launch_kv_remap(view_, remap_, epoch_, opt_.sequences, s));
  for (int i = 0; i < n; ++i) {
    refs_[moves[2 * i + 1]] = refs_[moves[2 * i]];
    refs_[moves[2 * i]] = 0;
  }
  for (Seq& q : seqs_)
    if (q.live)
      for (int& p : q.pages)
        if (to[p] >= 0) p = to[p];
  free_pages_ = MinHeap();
  for (int p = used; p < opt_.pages; ++p) free_pages_.push(p);
  leave(s);
  return n;
}

void KvCache::reset(int id) {
  Seq& q = seq(id);
  drop_pages(q);
  q.len = 0;
  q.filled.assign(opt_.layers, 0);
}

void KvCache::fork_into(int parent, int64_t tokens, int child, cudaStream_t s) {
  Seq& c = seq(child);
  const Seq& p = seq(parent);
  check_filled(parent);
  if (c.len || tokens < 0 || tokens > p.len) throw Error("internal: a fork into a sequence with positions");
  enter(s, "fork");
  share(c, p, tokens);
  KvRuns runs;
  runs.run[runs.n++] = KvRun{child, parent, 0, (int)tokens, (int)p.len};
  TRIT_CUDA(launch_kv_fork(view_, runs, true, s));
  leave(s);
}

void KvCache::settle(int id, int64_t tokens) {
  Seq& q = seq(id);
  if (tokens < 0 || tokens > q.len) throw Error("internal: a sequence settled past its positions");
  while ((int64_t)q.pages.size() > tokens / opt_.page) {
    if (--refs_[q.pages.back()] == 0) free_pages_.push(q.pages.back());
    q.pages.pop_back();
  }
  q.len = tokens;
  q.filled.assign(opt_.layers, tokens);
}

}  // namespace trit
