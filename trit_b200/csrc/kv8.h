// The paged key/value cache held in 8 bits: its device layout, the kernels'
// launchers (kv8.cu) and the host side that hands out pages and sequences
// (kv_cache.cpp).
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <mutex>
#include <queue>
#include <string>
#include <vector>

namespace trit {

enum KvType : int { kKvF32 = 0, kKvF16 = 1, kKvBF16 = 2 };

// Device memory of a cache. A (page, layer, which, head) block is page * hd
// codes, each stored as code + 128:
//   keys    [token][hd]
//   values  [token / 2][hd][token % 2]  (the two keys that share a register
//           of the value product lie side by side)
// with one f32 scale a block. A sequence's open page (the positions behind
// its last full page) is f16 in the same order, in the sequence's own buffer.
struct KvView {
  uint8_t* codes = nullptr;   // [pages][layers][2][kv_heads][page * hd]
  float* scales = nullptr;    // [pages][layers][2][kv_heads]
  __half* open = nullptr;     // [sequences][layers][2][kv_heads][page * hd]
  int* table = nullptr;       // [sequences][pages_per_seq] physical page numbers
  int layers = 0, kv_heads = 0, hd = 0, page = 0;
  int page_shift = 0;  // page = 1 << page_shift
  int pages_per_seq = 0;
};

// Consecutive rows of one sequence: rows row0 .. row0 + count of the call's
// tensors are its positions first .. first + count; `len` positions are in
// the cache. block0, splits: the attention's blocks of the runs before, and the
// shares that this run's positions are cut into.
struct KvRun {
  int seq, first, row0, count, len, block0 = 0, splits = 1;
};
// Runs travel as a kernel parameter: a call needs no copy to the device and
// leaves nothing behind that a later call could overwrite.
constexpr int kKvRuns = 120;  // 28 bytes each, in a parameter space of 4 KB
struct KvRuns {
  int n = 0;
  // Rows of a decode step instead of runs: row r is position row_pos[r] of
  // sequence row_seq[r], which then has row_pos[r] + 1 positions.
  const int* row_seq = nullptr;
  const int* row_pos = nullptr;
  KvRun run[kKvRuns];
};

struct KvAttendArgs {
  const void* q = nullptr;
  void* out = nullptr;
  size_t q_stride = 0, out_stride = 0;  // elements between rows
  int type = kKvF32;
  int heads = 0;
  int layer = 0;
  int causal = 1;
  float scale = 1.0f;
  int max_len = 0;  // the longest run's positions
};

// Writes the runs' rows of one layer; pages that fill up become codes.
cudaError_t launch_kv_append(const KvView& kv, const KvRuns& runs, int layer, const void* k, size_t k_stride,
                             const void* v, size_t v_stride, int type, int max_count, cudaStream_t s);
// How launch_kv_attend will run: blocks for each kv head, query columns a
// block, and whether shares of the positions meet in the workspace. `chunks`
// and `splits` are for rows of a decode step (the same for each).
struct KvAttendPlan {
  int blocks = 0, cols = 0, chunks = 1, splits = 1;
  bool joins = false;
  // Bytes of workspace, and where in it (in floats) sums are put aside, in how
  // many places.
  size_t workspace = 0, aside = 0;
  int places = 0;
};
// The workspace begins with words that are zero between calls: a counter a
// tile whose shares meet, and a flag a place where a block of many rows puts
// sums aside. No plan needs more.
constexpr size_t kKvCounters = 8192, kKvPlaces = 1024, kKvHead = kKvCounters + kKvPlaces;
constexpr size_t kKvWorkspace = 64u << 20;
KvAttendPlan plan_kv_attend(const KvView& kv, KvRuns& runs, const KvAttendArgs& a);
cudaError_t launch_kv_attend(const KvView& kv, const KvRuns& runs, const KvAttendArgs& a, const KvAttendPlan& plan,
                             void* workspace, cudaStream_t s);
// Attention of runs with many query rows (kv8_prompt.cu). *status is set
// when a wait inside the kernel ran out.
KvAttendPlan plan_kv_prompt(const KvView& kv, KvRuns& runs, const KvAttendArgs& a);
cudaError_t launch_kv_prompt(const KvView& kv, const KvRuns& runs, const KvAttendArgs& a, const KvAttendPlan& plan,
                             void* workspace, int* status, cudaStream_t s);
// Whether a run's rows are worth the kernel of many rows. It takes 128 or 256
// query columns (a row of a head of the group) at the cost of one, the other
// reads the positions again for every 4 to 16; but it starts late, so the call
// has to bring enough columns over all kv heads as well. Measured on 32 heads
// on 8, 40 on 8 and 8 on 8, 128 wide, and 16 on 4, 32 on 4 and 16 on 16, 64
// wide, over 500 to 4000 positions; us for few / many:
// - columns a run, 24 runs of 1500 positions: f32, 32 on 8, 48 columns 112 /
//   132, 64 154 / 133; 16 on 4, 48 39 / 39, 64 43 / 39; 16 on 16, 64 142 / 147,
//   80 174 / 147. bf16, 32 on 8, 64 87 / 96, 96 118 / 99; 16 on 4, 64 26 / 32,
//   96 41 / 34; 16 on 16, 64 84 / 109, 96 119 / 112. The lengths move the
//   border by a quarter either way.
// - columns a call, one run: f32, 32 on 8, over 2000 positions 2048 37 / 43,
//   4096 65 / 46; over 500 4096 30 / 35, 8192 48 / 35. bf16 over 2000 4096 37 /
//   56, 8192 66 / 57; over 500 8192 31 / 39, 16384 49 / 46; over 6000 4096 85 / 74.
inline bool kv_prompt_run(int64_t count, int group, int type, int64_t columns) {
  return type == kKvF32 ? count * group >= 64 && columns >= 4096 : count * group >= 96 && columns >= 8192;
}
// Positions first .. first + count of each run as values, rows of
// [kv_heads][hd] from row0 on.
cudaError_t launch_kv_read(const KvView& kv, const KvRuns& runs, int layer, void* k, void* v, int type, int max_count,
                           cudaStream_t s);
// Sequence moves: run i makes sequence `seq` start as `count` positions of
// sequence `first`: the open page's values (dequantized where the cut lies
// inside a full page) and, with copy_table, the table entries of its full
// pages.
cudaError_t launch_kv_fork(const KvView& kv, const KvRuns& runs, bool copy_table, cudaStream_t s);
// table[index[i]] = page[i]; up to kKvRuns * 3 entries ride in a parameter.
struct KvEntries {
  int n = 0;
  int index[kKvRuns * 3], page[kKvRuns * 3];
};
cudaError_t launch_kv_table(const KvView& kv, const KvEntries& e, cudaStream_t s);
// Page moves[2i] -> moves[2i + 1] (device pairs; no page is both read and
// written); with `remap`, the moved pages' targets are noted there under
// `epoch`, and launch_kv_remap makes the table's entries follow.
cudaError_t launch_kv_move(const KvView& kv, const int* moves, int n, unsigned long long* remap, unsigned epoch,
                           cudaStream_t s);
cudaError_t launch_kv_remap(const KvView& kv, const unsigned long long* remap, unsigned epoch, int sequences,
                            cudaStream_t s);

struct KvOptions {
  int device = 0, layers = 1, kv_heads = 0, hd = 128, page = 64, pages = 0, sequences = 64, max_tokens = 4096;
  static KvOptions parse(const char* json);
};

// The host side of one cache: which sequence holds which pages. Calls on it
// take turns (the caller holds mutex()); work on different streams is put in
// order with events.
class KvCache {
 public:
  explicit KvCache(const KvOptions& o);
  ~KvCache();
  KvCache(const KvCache&) = delete;
  KvCache& operator=(const KvCache&) = delete;

  std::mutex& mutex() { return mu_; }
  const KvOptions& options() const { return opt_; }
  const KvView& view() const { return view_; }

  void open(size_t n, int* out);
  void fork(const int* seqs, const int64_t* tokens, size_t n, int* out, cudaStream_t s);
  void copy(const int* seqs, size_t n, int* out, cudaStream_t s);
  void release(const int* seqs, size_t n);
  void extend(const int* seqs, const int64_t* counts, size_t n, cudaStream_t s);
  void append(int layer, const int* seqs, const int64_t* counts, size_t n, const void* k, size_t k_stride,
              const void* v, size_t v_stride, int type, cudaStream_t s);
  void attend(int layer, const int* seqs, const int64_t* counts, size_t n, const void* q, size_t q_stride, int heads,
              int type, float scale, bool causal, void* out, size_t out_stride, cudaStream_t s);
  void read(int layer, const int* seqs, const int64_t* firsts, const int64_t* counts, size_t n, void* k, void* v,
            int type, cudaStream_t s);
  int64_t compact(cudaStream_t s);
  int64_t length(int seq) const;
  int pages_used() const { return opt_.pages - (int)free_pages_.size(); }

  // For a decoder that runs the kernels itself on its one stream (Lm): a
  // sequence without positions again; the first `tokens` positions of
  // `parent` for such a sequence; a sequence of which `tokens` positions were
  // written and the rest only set aside.
  void reset(int seq);
  void fork_into(int parent, int64_t tokens, int child, cudaStream_t s);
  void settle(int seq, int64_t tokens);
  // Whether an attention kernel gave up waiting since the last call, and the
  // word that says so (host memory that kernels write).
  bool take_failure();
  int* status() const { return status_; }
  // Memory for the joins of any one attention call.
  void* workspace() const { return workspace_; }

 private:
  struct Seq {
    bool live = false;
    int64_t len = 0;
    std::vector<int> pages;       // one entry for every page begun (len positions)
    std::vector<int64_t> filled;  // positions appended, by layer
  };
  using MinHeap = std::priority_queue<int, std::vector<int>, std::greater<int>>;

  void release_memory();
  Seq& seq(int id);
  const Seq& seq(int id) const;
  int new_seq();
  void share(Seq& child, const Seq& parent, int64_t tokens);
  void check_filled(int id) const;
  void drop_pages(Seq& q);
  void check_layer(int layer) const;
  // Orders stream s behind everything this cache queued on other streams.
  void enter(cudaStream_t s, const char* what, bool may_capture = false);
  void refuse_capture(cudaStream_t s, const char* what);
  void leave(cudaStream_t s);
  void attend_runs(KvRuns& runs, KvAttendArgs& a, bool prompt, cudaStream_t s);
  void set_entries(const std::vector<std::pair<int, int>>& entries, cudaStream_t s);

  KvOptions opt_;
  KvView view_;
  std::mutex mu_;
  std::vector<Seq> seqs_;
  MinHeap free_seqs_, free_pages_;
  std::vector<int> refs_;  // sequences that hold each page
  void* workspace_ = nullptr;
  int *moves_ = nullptr, *status_ = nullptr;
  unsigned long long* remap_ = nullptr;  // [pages] (epoch, target) of the last compaction that moved it
  unsigned epoch_ = 0;
  cudaEvent_t order_ = nullptr;
  unsigned long long last_stream_ = 0;
  bool used_ = false, capturing_ = false;
};

}  // namespace trit
