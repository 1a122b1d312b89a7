/* trit_cuda: the greedy token loop of Trit's decoder language model
 * (CausalLm: Qwen3 / Llama / Mistral / Granite) on NVIDIA B200 (sm_100a).
 * C ABI of libtrit_cuda.so.
 *
 * It replaces the CPU decoder behind src/models/parts/causal_lm.rs of
 * Hi9841/trit; the entry points follow that interface (each cites the
 * function it stands for) and the rules of include/trit.h:7-18:
 * - Strings are UTF-8 and NUL-terminated.
 * - A call that fails returns NULL or -1; trit_cuda_last_error() then gives
 *   the reason, for the calling thread. No C++ exception crosses the ABI.
 * - Every exported name starts with trit_cuda_, trit_lm_ or trit_dense_, so
 *   the library can share a process with the reference's own libtrit,
 *   whose trit_last_error and trit_free_text (ffi/src/lib.rs:186,641) keep
 *   their meaning; nothing else is exported.
 * - One model handle may be used from several threads; calls on it take
 *   turns (a mutex), as calls on one Trit engine share one worker team.
 *   Do not free a handle while another thread is in a call on it.
 * - The caller owns every buffer it passes, for the length of the call;
 *   the library owns the device memory of a handle until trit_lm_free.
 * - There is no CPU fallback: without a usable GPU the load fails.
 *
 * A model is a folder in one of three forms (src/models/gguf/mod.rs,
 * src/cpu/tensors.rs):
 * - config.json (Hugging Face keys, as Config::parse reads them,
 *   causal_lm.rs:41-77) and model.gguf with the tensors under their
 *   Hugging Face names;
 * - config.json and safetensors files (model.safetensors, the shards of
 *   model.safetensors.index.json, or every *.safetensors);
 * - one GGUF file as transcribe.cpp writes it (no config.json): the decoder
 *   settings come from its stt.<arch>.decoder.* metadata and its dec.*
 *   tensor names are mapped as the reference maps them (architectures
 *   qwen3_asr, moss, funasr_nano, canary_qwen, voxtral, voxtral_realtime,
 *   granite_speech; src/models/gguf/qwen3_asr.rs:103-136).
 * Products are Q8_0 (ggml blocks of 32 codes and an f16 scale), float (F32,
 * F16, BF16: quantized to Q8_0 at load as ggml quantizes, gemm.rs:53-76),
 * per-row int8 (`.weight` I8 + `.scales` F32 per row), or ternary
 * (`.qweight`, five base-3 codes a byte, + `.scales` F32 per 128 inputs, as
 * src/models/parts/fastconformer.rs:440-452 reads them); norms F32/F16/BF16;
 * token tables Q8_0, float (quantized to Q8_0) or int8 with per-32 F32
 * scales.
 */
#ifndef TRIT_CUDA_H
#define TRIT_CUDA_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct TritLm TritLm;
typedef struct TritLmPrefix TritLmPrefix;
typedef struct TritDense TritDense;
typedef struct TritKv TritKv;
typedef struct TritRotary TritRotary;

/* A tensor-parallel group's id (NCCL's unique id as 256 hex characters
 * and a NUL, into out of cap >= 257 bytes), made once on one rank and
 * passed to every rank's trit_lm_load as "tp_id". Returns 0, or -1. No
 * counterpart in the reference, which runs on one CPU. */
int trit_cuda_tp_id(char *out, size_t cap);

/* The library version, for example "0.1.0". Static; do not free.
 * (trit_version, include/trit.h:41.) */
const char *trit_cuda_version(void);

/* The error of the last failed call on this thread, or "" after a success.
 * Valid until the next call on this thread; do not free.
 * (trit_last_error, include/trit.h:44-46; ffi/src/lib.rs:20-45,186.) */
const char *trit_cuda_last_error(void);

/* A model folder described without a GPU, as JSON text: its settings as
 * Config::parse reads them (causal_lm.rs:41-77: q/k norms iff model_type
 * is "qwen3", head_dim defaulting to hidden / heads, eps 1e-6, rope_theta
 * 1e6, the Granite multipliers, tie_word_embeddings), the storage of its
 * products and token tables, and the bytes a greedy step reads from device
 * memory for the products and the output table. `options_json` takes the
 * "config_at" and "prefix" keys of trit_lm_load (others are ignored).
 * Free the text with trit_cuda_free_text. NULL on failure. */
char *trit_lm_inspect(const char *model_dir, const char *options_json);

/* Frees text returned by this library (and only by it: the reference's
 * trit_free_text frees with its own allocator). NULL is a no-op.
 * (trit_free_text, include/trit.h:11; ffi/src/lib.rs:641.) */
void trit_cuda_free_text(char *text);

/* Loads a decoder onto a GPU. `options_json` is NULL, "" or an object;
 * every key is optional and an unknown key fails (as trit_load_json,
 * include/trit.h:76-87):
 *   "device":       CUDA device index (0)
 *   "kv":           "f16" (default), "f32" or "q8": the element type of the
 *                   paged KV cache; "f32" holds what the reference holds;
 *                   "q8" holds 8-bit codes with a scale a page and kv head
 *                   (see trit_cuda_kv_new), about half the memory and bytes
 *                   of "f16": logits drift (a value by about 1 %), decoding
 *                   runs layered (slower than "f16" for one stream, faster
 *                   for a batch), pages of 16, 32, 64 or 128 positions, at
 *                   most 16 prefixes at once
 *   "max_context":  positions per stream (4096)
 *   "max_streams":  stream slots for trit_lm_generate_batch (1)
 *   "page_tokens":  positions per KV page (64)
 *   "prefill_rows": prompt rows per prefill pass (512)
 *   "prefix_pages": KV pages kept for trit_lm_prefix (max_context /
 *                   page_tokens: one stream's worth)
 *   "decode":       "persistent" (default: one kernel runs every greedy
 *                   step of a batch-1 generation) or "layered" (a kernel
 *                   per operation and step)
 *   "tensor_cores": true (default on sm_100) or false: products of
 *                   "tc_rows" rows or more on the tensor cores
 *   "tc_rows":      rows from which a product uses the tensor cores (64)
 *   "tc_f16":       false (default) or true: Q8_0 products on the tensor
 *                   cores take their codes as f16 (exact; the MMA makes the
 *                   group dots as exact f32), at the cost of an f16 copy of
 *                   the Q8_0 layers' codes (2 bytes a weight); measured
 *                   slower than the int8 MMA on C5 (5045 against 5268 tok/s)
 *   "tp_size", "tp_rank", "tp_id": tensor parallelism over tp_size ranks,
 *                   one process (or thread) and GPU each: every rank loads
 *                   with the same tp_id (trit_cuda_tp_id's text, made once
 *                   on one rank and shared) and its own tp_rank, and then
 *                   makes the same calls; a rank holds its query heads
 *                   with their key/value heads, its FFN units and its rows
 *                   of the output table, and the ranks sum the o_proj and
 *                   down_proj partials and take the best token of their
 *                   output rows through NCCL (all-reduce). Greedy steps run
 *                   the layered kernels; logit traces, generate_additive
 *                   and bidirectional_tokens are not available
 *   "tp_timeout_s": seconds a rank waits for the others (joining, or a call
 *                   whose collectives they must answer) before it aborts
 *                   the communicator and the call fails (120); the handle
 *                   is unusable afterwards
 *   "weight_cache": false (default) or true: keep the weights' device
 *                   layout in a file (in "cache_dir", default
 *                   <model_dir>/.trit_cuda) on the first load and read it
 *                   straight into device memory on later loads, with no
 *                   parsing or conversion; a file that does not match the
 *                   model's files byte for byte is rewritten, and one that
 *                   cannot be written is skipped (as src/cpu/store.rs:1-16)
 *   "cache_dir":    the folder of the weight cache
 *   "exact":        true (default) or false. true: every floating-point
 *                   step in the order of the reference's CPU decoder, so
 *                   logits equal its logits bit for bit. false: the batch-1
 *                   decode sums in tree order and splits attention and
 *                   o_proj by kv head; the int8 activation codes can then
 *                   move where a value sits on a rounding boundary, so
 *                   logits drift (measured up to 5e-2 max-abs, cosine
 *                   >= 0.9999; the reference restatement with only its
 *                   RmsNorm sum reordered drifts as much) while tokens
 *                   stayed the reference's on every tested config
 *   "tc_attention": false (default) or true (with "exact": false): prompt
 *                   attention as f16 flash attention on the tensor cores
 *                   (f16 cache, pages of a multiple of 64 positions); its
 *                   sums are not the reference's, so logits drift and a
 *                   token can differ where the reference's top two logits
 *                   are close
 *   "config_at":    key path of the decoder settings in config.json ("";
 *                   "thinker_config.text_config." in Qwen3-ASR)
 *   "prefix":       start of every tensor name ("", "thinker.", "llm.")
 * NULL on failure. (CausalLm::load / from_tensors, causal_lm.rs:124-198.) */
TritLm *trit_lm_load(const char *model_dir, const char *options_json);

/* Frees a model and its device memory. NULL is a no-op. (trit_free,
 * include/trit.h:115-116.) */
void trit_lm_free(TritLm *lm);

/* What a load did, as JSON text: "source" (the files' form: "gguf",
 * "gguf-transcribe" or "safetensors"), "weights_from" ("files", or "cache"
 * when the weight cache supplied the device layout), "weight_cache" (its
 * file, or null), "arena_bytes", the KV and decode settings and the
 * prefix pages in use. Free with trit_cuda_free_text. NULL on failure. */
char *trit_lm_status(const TritLm *lm);

/* hidden_size, num_hidden_layers, vocab_size; -1 for NULL.
 * (CausalLm::width / layers, causal_lm.rs:307-313,343-345.) */
int64_t trit_lm_width(const TritLm *lm);
int64_t trit_lm_layers(const TritLm *lm);
int64_t trit_lm_vocab(const TritLm *lm);

/* Runs a prompt start that many calls share (a system prompt) once; a
 * trit_lm_generate or trit_lm_generate_batch_prefix stream whose prompt
 * begins with it and is longer starts from its cache. The prefix's full KV
 * pages are kept read-only in pages the model holds for prefixes (load
 * option "prefix_pages") and every call reads them in place (the page
 * tables of its streams point at them); only the page the prefix ends
 * inside is copied, once per stream and call. NULL on failure (also when
 * the kept pages are used up). (CausalLm::prefix, causal_lm.rs:200-215.) */
TritLmPrefix *trit_lm_prefix(TritLm *lm, const int32_t *ids, size_t n);

/* Frees a prefix and returns its pages. NULL is a no-op. Not while a call
 * on its model uses it. */
void trit_lm_prefix_free(TritLmPrefix *prefix);

/* The KV pages kept for prefixes: in use (by live prefixes) and in all.
 * Returns 0, or -1. */
int trit_lm_prefix_pages(const TritLm *lm, int64_t *used, int64_t *total);

/* Greedy tokens after `prompt` (n ids), until a token of `stop` (nstop ids,
 * not kept) or `max_new` tokens; writes at most `cap` of them to `out`.
 * Returns the number of tokens made, or -1. `prefix` may be NULL.
 * (CausalLm::generate + greedy, causal_lm.rs:217-249,284-302.) */
int64_t trit_lm_generate(TritLm *lm, const TritLmPrefix *prefix, const int32_t *prompt, size_t n,
                         int32_t max_new, const int32_t *stop, size_t nstop, int32_t *out, size_t cap);

/* Greedy tokens after a prompt given as embeddings, `nrows` rows of
 * trit_lm_width() floats (some rows from another model, such as audio
 * frames). Returns the count, or -1. (CausalLm::generate_rows,
 * causal_lm.rs:251-262.) */
int64_t trit_lm_generate_rows(TritLm *lm, const float *rows, size_t nrows, int32_t max_new,
                              const int32_t *stop, size_t nstop, int32_t *out, size_t cap);

/* generate_rows after the prompt `head` (ids), the rows `audio` (naudio
 * rows of trit_lm_width() floats) and the prompt `tail` (ids). Returns the
 * count, or -1. (CausalLm::answer, causal_lm.rs:264-282.) */
int64_t trit_lm_answer(TritLm *lm, const int32_t *head, size_t nhead, const float *audio, size_t naudio,
                       const int32_t *tail, size_t ntail, int32_t max_new, const int32_t *stop,
                       size_t nstop, int32_t *out, size_t cap);

/* trit_lm_generate_rows and trit_lm_answer with the rows in device memory
 * of the model's GPU (an encoder's output that stays on the GPU: no copy
 * through the host). The rows are read after the work queued so far on
 * `cuda_stream` (a cudaStream_t; NULL: the legacy default stream), as
 * device-to-device copies; the call returns when the tokens are on the
 * host, so the caller may reuse the rows' memory then. Fails when the
 * pointer is not device memory of that GPU. Returns the count, or -1.
 * (CausalLm::generate_rows / answer, causal_lm.rs:251-282, fed by
 * Qwen3Asr's encoder rows, src/models/families/qwen3_asr.rs:321-372.) */
int64_t trit_lm_generate_rows_device(TritLm *lm, const float *rows_device, size_t nrows, int32_t max_new,
                                     const int32_t *stop, size_t nstop, int32_t *out, size_t cap,
                                     void *cuda_stream);
int64_t trit_lm_answer_device(TritLm *lm, const int32_t *head, size_t nhead, const float *audio_device,
                              size_t naudio, const int32_t *tail, size_t ntail, int32_t max_new,
                              const int32_t *stop, size_t nstop, int32_t *out, size_t cap, void *cuda_stream);

/* The embeddings of `n` ids, n x trit_lm_width() floats, into `out`.
 * Returns 0, or -1. (CausalLm::embed, causal_lm.rs:347-355.) */
int trit_lm_embed(TritLm *lm, const int32_t *ids, size_t n, float *out);

/* trit_lm_generate with the logits each token came from: `logits` holds
 * max_new x trit_lm_vocab() floats; row i is written for every token made
 * and for a stopping token. For parity checks; slower than
 * trit_lm_generate. (The logits of forward_rows, causal_lm.rs:366-389.) */
int64_t trit_lm_generate_traced(TritLm *lm, const TritLmPrefix *prefix, const int32_t *prompt, size_t n,
                                int32_t max_new, const int32_t *stop, size_t nstop, int32_t *out,
                                size_t cap, float *logits);

/* trit_lm_answer with the logits trace of trit_lm_generate_traced. */
int64_t trit_lm_answer_traced(TritLm *lm, const int32_t *head, size_t nhead, const float *audio,
                              size_t naudio, const int32_t *tail, size_t ntail, int32_t max_new,
                              const int32_t *stop, size_t nstop, int32_t *out, size_t cap,
                              float *logits);

/* Independent greedy generations, one per stream (at most "max_streams"),
 * decoded side by side: stream s starts from prompts[s] (lens[s] ids) and
 * writes its tokens to out[s * max_new ...] and their count to counts[s].
 * Returns 0, or -1. (CausalLm::generate for each stream; the streams share
 * the weights, as the reference's callers share one model.) */
int trit_lm_generate_batch(TritLm *lm, size_t streams, const int32_t *const *prompts, const size_t *lens,
                           int32_t max_new, const int32_t *stop, size_t nstop, int32_t *out,
                           int64_t *counts);

/* trit_lm_generate_batch where the streams whose prompt begins with
 * `prefix` (and is longer) read its pages and run only the rest of their
 * prompt, as S1-mini's cleanup calls share one system prompt
 * (src/cleanup.rs:208,297-299). `prefix` may be NULL. Returns 0, or -1. */
int trit_lm_generate_batch_prefix(TritLm *lm, const TritLmPrefix *prefix, size_t streams,
                                  const int32_t *const *prompts, const size_t *lens, int32_t max_new,
                                  const int32_t *stop, size_t nstop, int32_t *out, int64_t *counts);

/* CausalLm::set_ffn_scales (causal_lm.rs:305-307): the normed MLP input of
 * layer l is multiplied by scales[l * width ...] (layers x width floats,
 * copied); NULL clears the scales. Returns 0, or -1. */
int trit_lm_set_ffn_scales(TritLm *lm, const float *scales, size_t layers, size_t width);

/* CausalLm::generate_additive (causal_lm.rs:317-345), Voxtral Realtime's
 * loop: the prompt's embeddings plus audio rows 0..n, then each new token's
 * embedding plus the next row (`audio`: rows x width floats), until a token
 * of `stop` or the rows end; at most rows - n + 1 tokens, written to `out`
 * (cap of them). Returns the count, or -1. */
int64_t trit_lm_generate_additive(TritLm *lm, const int32_t *prompt, size_t n, const float *audio, size_t rows,
                                  const int32_t *stop, size_t nstop, int32_t *out, size_t cap);

/* CausalLm::bidirectional_tokens (causal_lm.rs:393-408), Granite Speech
 * NAR's editor: one pass over `m` rows (m x width floats) with no causal
 * mask, then the best token of each row from `from` on, m - from ids into
 * `out`. The rows must fit one prefill pass ("prefill_rows"). Returns
 * m - from, or -1. */
int64_t trit_lm_bidirectional_tokens(TritLm *lm, const float *rows, size_t m, size_t from, int32_t *out);

/* The device time of the last generation on this handle, from CUDA events:
 * the prompt (prefill) and the greedy steps after it, in ms, the number of
 * decode steps, and the kernel launches it made. Returns 0, or -1. */
int trit_lm_last_timing(const TritLm *lm, double *prefill_ms, double *decode_ms, int64_t *decode_steps,
                        int64_t *launches);

/* ---- single product layers (Dense, src/cpu/gemm.rs:14-542) ---- */

/* A layer from ggml Q8_0 blocks of an `n x k` row-major matrix (34 bytes a
 * block: f16 scale, 32 codes). table = 0: int8 activations in groups of 32
 * with f16-rounded scales, i8 x i8 products (Dense::q8_0 -> Int8::from_q8_0,
 * gemm.rs:212-231, int8.rs:234-289); table = 1: a token table, f32 math
 * (Dense::table -> Weights::Q8, gemm.rs:383-409). NULL on failure. */
TritDense *trit_dense_q8_0(const void *blocks, size_t n, size_t k, int table, int device);

/* A layer from ggml Q4_0 blocks of an `n x k` row-major matrix (18 bytes a
 * block of 32 weights: an f16 scale d and 32 codes c of 4 bits, code i in the
 * low half of byte i and code 16 + i in its high half; the weight is
 * d (c - 8)), kept in 4 bits on the GPU. k is a multiple of 32; n and k are at
 * most 2^31 - 16384. table = 0: rows of x are rounded to int8 codes in groups
 * of 32 with f16-rounded scales, as in a Q8_0 layer; table = 1: f32 rows as
 * they are. A row with a NaN gives NaN (a Q8_0 layer takes it for 0). Sums are
 * f32, in another order than a Q8_0 layer's. A call of more than 32 rows with table = 0 (n a
 * multiple of 32, k of 128) runs on the int8 tensor cores from an int8 copy of
 * the weights that the first such call makes (n x k bytes more; refused in a
 * capture). Outside of a capture such calls share scratch memory, as a Q8_0
 * layer's do: order them on one stream; a captured one's belongs to its graph.
 * The other calls use none: they may overlap, and may be captured after the
 * first. NULL on failure. (The reference expands Q4_0 tensors when it loads
 * them, src/cpu/ggml_quants.rs:1-6.) */
TritDense *trit_dense_q4_0(const void *blocks, size_t n, size_t k, int table, int device);

/* A layer of 8-bit floating point from an `n x k` row-major matrix of e4m3
 * numbers (`codes`, a byte each: 1 sign, 4 exponent and 3 fraction bits, largest
 * 448, no infinities) with an f32 scale for each block of 128 x 128 (`scales`,
 * ceil(n / 128) x ceil(k / 128), row-major), both in host memory. A weight is
 * code * scale. k is a multiple of 16 up to 2^24, n at most 2^31 - 256. Rows of
 * x are 8-bit rows: e4m3 numbers with an f32 scale for each 128 of a row, which
 * trit_cuda_rms_norm writes; rows of values are rounded to such first, in memory
 * that a call takes and gives back in its stream's order (a captured one has its
 * graph's). Each block's products are summed on the tensor cores, the blocks in
 * f32, each by f32(scale of x * scale of w): where that is no normal number of f32
 * (below 2^-126 and not 0, or 2^128 and more), a block loses bits, or is infinite
 * or NaN, also if its part of the result would be in range. Calls share no memory
 * but the weights, so they may overlap and be captured.
 * NULL on failure. (No counterpart in the reference.) */
TritDense *trit_dense_fp8(const void *codes, const float *scales, size_t n, size_t k, int device);

/* out (rows x n) from 8-bit rows (`codes` rows x k bytes, 16-byte aligned, and
 * `scales` rows x ceil(k / 128)), in device memory, for a layer of
 * trit_dense_fp8. `type` is that of out: 0 for f32, 1 for f16, 2 for bf16;
 * out_stride is in elements between rows (0: packed). Queued on `cuda_stream`
 * (NULL: the default stream); does not wait. Returns 0, or -1. */
int trit_dense_forward_codes(TritDense *layer, const void *codes, const float *scales, size_t rows, void *out,
                             size_t out_stride, int type, void *cuda_stream);

/* trit_dense_forward_codes of rows of values (of `type`, as out), which are
 * rounded to 8-bit rows first, as trit_cuda_rms_norm rounds them. */
int trit_dense_forward_rows(TritDense *layer, const void *x, size_t x_stride, size_t rows, void *out, size_t out_stride,
                            int type, void *cuda_stream);

/* out (rows x n) = x (rows x k) times the layer, both in host memory.
 * Returns 0, or -1. (Dense::forward, gemm.rs:500-542.) */
int trit_dense_forward(TritDense *layer, const float *x, size_t rows, float *out);

/* trit_dense_forward on device pointers, queued on `cuda_stream` (a
 * cudaStream_t, or NULL for the layer's own stream); does not wait. */
int trit_dense_forward_device(TritDense *layer, const float *x, size_t rows, float *out, void *cuda_stream);

/* Whether the layer's products that have ended are whole: every wait inside a
 * tensor-core product is bounded in time, and one that ran out leaves outputs that
 * are not. Returns 0, or -1 if that has happened since it was last reported: here,
 * or as the failure of a call of the layer (trit_dense_forward, and any further
 * product of a trit_dense_fp8 layer). A caller of the calls that do not wait asks
 * after synchronising its stream, and after replays of a recorded graph. */
int trit_dense_check(TritDense *layer);

/* Frees a layer. NULL is a no-op. */
void trit_dense_free(TritDense *layer);

/* A Q8_0 W8A8 product that allocates nothing, for callers that cannot
 * call cudaMalloc when they run it (inside another party's graph capture,
 * on a real-time thread, or with every byte of device memory owned by
 * their own pool). No counterpart in the reference: Trit runs on the CPU
 * and allocates freely. It computes what trit_dense_forward_device
 * computes, on device pointers: `codes` (n x k int8, row-major) and
 * `scales` (n x k/32 f16 bits) are the split form of ggml Q8_0 blocks
 * (block b of row r: scales[r * k/32 + b], codes[r * k + 32 b ...]); x is
 * rows x k f32; out is rows x n f32; k is a multiple of 128 from 128 to
 * 8192 and n a positive multiple of 32. Its scratch (the int8 activations and
 * their scales) is one 1 MiB device array that the library holds on every
 * GPU it is loaded on until the process exits, so rows * k * 9 / 8 must stay
 * within 1 MiB (larger calls fail). All calls share that array and leave
 * their contents in it: calls that overlap on the GPU (other streams,
 * other threads) race; order them on one stream. The first call on a
 * device looks up the array's device address (cudaGetSymbolAddress); make
 * that first call before any stream capture. Returns 0, or -1 with
 * trit_cuda_last_error(). Queued on `cuda_stream` (NULL: the default stream);
 * does not wait. */
int trit_dense_q8_0_forward_static(const void *codes, const void *scales, size_t n, size_t k, const float *x,
                                   size_t rows, float *out, void *cuda_stream);

/* ---- a key/value cache held in 8 bits ----
 *
 * The paged cache of an attention layer stack, for callers that run their
 * own decoder or encoder (trit_lm_load's "kv": "q8" uses the same kernels).
 * A sequence is a list of positions; `page_tokens` consecutive positions make
 * a page. Keys and values are rounded to f16 on arrival (beyond +-65504 to
 * that, NaN to 0). A page that is not full yet stays f16 (one buffer a
 * sequence); when its last position arrives, the page's keys of each layer
 * and kv head, and its values, become int8 codes with one f32 scale,
 *   scale = max|x| / 127,  code = the whole number nearest x / scale
 * (ties to even), and count as code * scale from then on. What the cache
 * holds depends on the values only, not on how many calls brought them.
 * No counterpart in the reference, whose cache is f32 (layers.rs:343-504).
 *
 * A step of a decoder: trit_cuda_kv_extend once, then for every layer
 * trit_cuda_kv_append and trit_cuda_kv_attend, all with the same sequences
 * and counts. Device pointers throughout; rows of several sequences are
 * packed, sequence after sequence. `stream` is a cudaStream_t (NULL: the
 * default stream); calls queue their work there and do not wait. Work on
 * different streams is put in the order of the calls. `type` is 0 for f32, 1
 * for f16, 2 for bf16. Strides are elements between rows (0: packed).
 *
 * In a stream capture only trit_cuda_kv_attend and trit_cuda_kv_read are
 * taken; a replay reads the positions that the sequences had when it was
 * captured, and the caller orders it after the calls it depends on. The
 * graph owns the memory it works in. The cache must outlive the graph, and
 * the sequences must stay as they were: a replay after a
 * trit_cuda_kv_release, trit_cuda_kv_compact or trit_cuda_kv_append of them
 * reads what now lies there.
 *
 * A call that fails on its arguments changes nothing. */

/* A cache. `options_json` is an object: "layers" (1), "kv_heads" and "pages"
 * (needed; "pages" counts full pages, each of every layer), "head_dim" (128;
 * 64 or 128), "page_tokens" (64; 16, 32, 64 or 128), "sequences" (64: how many
 * may be open at once), "max_tokens" (4096: positions a sequence), "device"
 * (0). NULL on failure. */
TritKv *trit_cuda_kv_new(const char *options_json);

/* Frees a cache and its device memory. NULL is a no-op. */
void trit_cuda_kv_free(TritKv *kv);

/* n new sequences without positions, their ids into out. Returns 0, or -1. */
int trit_cuda_kv_open(TritKv *kv, size_t n, int32_t *out);

/* n new sequences, out[i] starting as the first tokens[i] positions of
 * seqs[i] (tokens NULL: all of them). Full pages are shared until their last
 * holder is released (they never change); only the open page is copied. A cut
 * inside a full page keeps that page's values as f16. Returns 0, or -1. */
int trit_cuda_kv_fork(TritKv *kv, const int32_t *seqs, const int64_t *tokens, size_t n, int32_t *out, void *stream);

/* n new sequences equal to seqs[i], on pages of their own. Returns 0, or -1. */
int trit_cuda_kv_copy(TritKv *kv, const int32_t *seqs, size_t n, int32_t *out, void *stream);

/* The sequences go, and with them the pages that no other holds. Returns 0,
 * or -1. */
int trit_cuda_kv_release(TritKv *kv, const int32_t *seqs, size_t n);

/* counts[i] more positions for seqs[i] (each named once), to be appended in
 * every layer. Returns 0, or -1 (and then no sequence has grown). */
int trit_cuda_kv_extend(TritKv *kv, const int32_t *seqs, const int64_t *counts, size_t n, void *stream);

/* The keys and values of the last counts[i] positions of seqs[i] in one
 * layer: rows of kv_heads x head_dim values. Every position is appended once
 * in every layer, in order. Returns 0, or -1. */
int trit_cuda_kv_append(TritKv *kv, int32_t layer, const int32_t *seqs, const int64_t *counts, size_t n, const void *k,
                        size_t k_stride, const void *v, size_t v_stride, int type, void *stream);

/* Attention of counts[i] query rows of heads x head_dim values against
 * seqs[i]: softmax(scale q k) v, query head h on kv head
 * h / (heads / kv_heads). causal = 1: the rows stand at the sequence's last
 * counts[i] positions, each seeing the positions up to its own; causal = 0:
 * every row sees all positions (an encoder's states). Zeros where there is
 * none. Sums are f32; a weight of the softmax holds 22 bits, of bf16 rows 11. A
 * query with a NaN gives NaN. `out` may be `q`, with the same stride. Returns 0, or -1. */
int trit_cuda_kv_attend(TritKv *kv, int32_t layer, const int32_t *seqs, const int64_t *counts, size_t n, const void *q,
                        size_t q_stride, int32_t heads, int type, float scale, int causal, void *out,
                        size_t out_stride, void *stream);

/* What the cache holds of positions firsts[i] .. firsts[i] + counts[i] of
 * seqs[i] in one layer, packed rows of kv_heads x head_dim values; k or v may
 * be NULL. Returns 0, or -1. */
int trit_cuda_kv_read(TritKv *kv, int32_t layer, const int32_t *seqs, const int64_t *firsts, const int64_t *counts,
                      size_t n, void *k, void *v, int type, void *stream);

/* Moves the pages in use to the front of the pool. Returns the number of
 * pages moved, or -1. */
int64_t trit_cuda_kv_compact(TritKv *kv, void *stream);

/* A sequence's positions, or -1. */
int64_t trit_cuda_kv_length(const TritKv *kv, int32_t seq);

/* Full pages in use and in all. Returns 0, or -1. */
int trit_cuda_kv_pages(const TritKv *kv, int64_t *used, int64_t *total);

/* ---- rows between the products and the cache ----
 *
 * For callers that run their own decoder beside trit_cuda_kv_* and layers of
 * trit_dense_fp8. Device pointers throughout, all on one GPU, which is found
 * from them; `type` is 0 for f32, 1 for f16, 2 for bf16; strides are elements
 * between rows (0: packed); `cuda_stream` is a cudaStream_t of that GPU (NULL:
 * the default stream). Calls queue their work there, do not wait, allocate
 * nothing and keep nothing, so any of them may overlap and be captured. A
 * call that fails on its arguments changes nothing. Two tensors of a call are
 * the same (pointer and stride) or share no element. No counterpart in the
 * reference, whose decoder does these steps inside CausalLm. */

/* RMSNorm of rows of `width` values (up to 2^24), behind the residual's
 * addition and in front of 8-bit rows:
 *   h = x + residual, rounded to `type` and written to `sum` (NULL: to
 *       `residual`); without a residual (NULL) h = x, and sum is NULL
 *   s = f32(1 / sqrt(mean(h^2) + eps)), its sum in 64 bits
 *   y = h * f32(s * weight), in f32 (a power of two goes from s to h first
 *       where s is beyond 2^100 or 2^-100, so that s keeps its bits)
 *   out (NULL: none) = y rounded to `type`; out may be x
 *   codes, scales (NULL: none) = y as 8-bit rows: rows x width e4m3 numbers and
 *       an f32 scale for each 128 of a row (rows x ceil(width / 128)),
 *       scale = max(f32(max|y| / 448), 2^-126), 1 where all are zero,
 *       code = e4m3(f32(y * f32(1 / scale))), ties to even
 * A group of 128 with a NaN or an infinity has the scale NaN. `weight` is f32
 * (weight_type 0) or of `type`. x and residual may be one tensor. Returns 0, or -1. (RmsNorm,
 * src/layers.rs:128-153.) */
int trit_cuda_rms_norm(const void *x, size_t x_stride, const void *residual, size_t residual_stride, void *sum,
                       size_t sum_stride, const void *weight, int weight_type, size_t rows, size_t width, int type,
                       double eps, void *out, size_t out_stride, void *codes, float *scales, void *cuda_stream);

/* Rotary positions. `options_json` is an object: "head_dim" (needed; even, up
 * to 512), "rotary_dim" (head_dim: how many of a head's first values turn;
 * even), "layout" ("halves": pairs i, i + rotary_dim / 2; or "interleaved":
 * pairs 2 i, 2 i + 1), "theta" (1e6), "scaling", and its settings. The
 * frequency of pair i is f = theta^(-2 i / rotary_dim) radians a position, or
 *   "linear":  f / factor
 *   "ntk":     that of theta * factor^(d / (d - 2)), d = rotary_dim
 *   "yarn":    between the pairs that turn `fast` (32) and `slow` (1) times
 *              over `trained` positions, rounded outwards and to pairs that there
 *              are, a straight line from f to f / factor; rotated values times
 *              0.1 ln(factor) + 1 (1 for factors below 1)
 *   "bands":   f for wavelengths below trained / high (4), f / factor for those
 *              above trained / low (1), a straight line over f between
 * "frequencies" gives them instead (rotary_dim / 2 numbers), and
 * "attention_factor" the factor of the rotated values. The handle holds no
 * device memory and serves every GPU, also several threads at once. NULL on
 * failure. (Rotary::halves, src/layers.rs:276-335.) */
TritRotary *trit_cuda_rotary_new(const char *options_json);

/* Frees a handle. NULL is a no-op. */
void trit_cuda_rotary_free(TritRotary *rotary);

/* The frequencies, at most `cap` of them into `out`, and the factor of the
 * rotated values (NULL: not wanted). Returns their count, or -1. */
int64_t trit_cuda_rotary_frequencies(const TritRotary *rotary, double *out, size_t cap, double *factor);

/* Turns the pairs of q (rows x q_heads x head_dim) and k (rows x k_heads x
 * head_dim; 0 heads and NULL: no such tensor; at most 65535 heads each) by
 * position * frequency, the exact product of the two 64-bit numbers (positions
 * up to 2^53 either way; a negative one turns back; angles of up to 2^80 radians
 * are right to 2^-24). `positions` has one number a row. q_out and
 * k_out: NULL for in place. Values of a head behind rotary_dim stay as they are.
 * Returns 0, or -1. */
int trit_cuda_rotary_apply(const TritRotary *rotary, const int64_t *positions, size_t rows, const void *q, size_t q_stride,
                           int32_t q_heads, void *q_out, size_t q_out_stride, const void *k, size_t k_stride,
                           int32_t k_heads, void *k_out, size_t k_out_stride, int type, void *cuda_stream);

#ifdef __cplusplus
}
#endif

#endif /* TRIT_CUDA_H */
