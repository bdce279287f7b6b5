/* nutllm_hip.h — C ABI of the MI355X (gfx950) token loop.
 *
 * This is the drop-in boundary under nutllm's C++17 host API: the
 * generate_tokens_cached / prefill_quantized / decode_quantized_token /
 * matvec_quantized_threaded entry points call these functions instead of the
 * reference's CPU kernels. Every function returns a status (never throws);
 * the status names the exception type the reference would have thrown, and
 * nut_last_error() gives its message ("quantized decode: token out of
 * range", ...). Citations are MokiMeow/nutllm path:line.
 *
 * Pointers named d_* are device pointers; all others are host pointers.
 * One host thread drives a handle at a time (the reference serialises calls
 * the same way, src/threading.cpp:50).
 */
#ifndef NUTLLM_HIP_H
#define NUTLLM_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ------------------------------------------------------------ status -- */

enum {
    NUT_OK = 0,
    NUT_EINVAL = 1,      /* std::invalid_argument */
    NUT_EOUTOFRANGE = 2, /* std::out_of_range */
    NUT_ELENGTH = 3,     /* std::length_error */
    NUT_ERANGE = 4,      /* std::range_error */
    NUT_ERUNTIME = 5,    /* std::runtime_error */
    NUT_EDEVICE = 6      /* HIP runtime error or no gfx950 device */
};

/* Message of the last failing call on this thread ("" after success). */
const char *nut_last_error(void);

/* ------------------------------------------------------------- types -- */

/* QuantType (include/quant.hpp:9-12). */
enum { NUT_INT8 = 0, NUT_INT4 = 1 };

/* ModelConfig (include/model.hpp:8-24); kv_heads == 0 means heads. */
typedef struct nut_config {
    size_t layers, heads, dim, head_dim, ffn_dim, vocab_size, max_seq,
        eos_token, kv_heads;
} nut_config;

/* Host view of a QuantizedMatrix's storage (include/quant.hpp:40-49):
 * flattened row-major blocks of block_size weights; INT8 bytes or INT4
 * nibbles (even flattened index in the low nibble), fp16 scale bits. */
typedef struct nut_qmatrix {
    const uint8_t *data;
    const uint16_t *scales;
    size_t rows, cols, block_size;
    int type;
} nut_qmatrix;

/* GenerationStats (include/generate.hpp:19-24). */
typedef struct nut_generation_stats {
    size_t prefill_tokens, generated_tokens;
    double prefill_seconds, decode_seconds;
} nut_generation_stats;

/* ------------------------------------------- host utilities (no GPU) -- */

/* QuantizedMatrix::quantize (src/quant.cpp:154-197), bit-exact: data gets
 * nut_quant_data_bytes bytes, scales nut_quant_scale_count fp16 words.
 * NUT_EINVAL on non-finite weights or bad shape, NUT_ERANGE when a scale
 * exceeds fp16 (src/quant.cpp:24-27,44-45). Runs on host threads. */
int nut_quantize(const float *source, size_t rows, size_t cols, int type,
                 size_t block_size, uint8_t *data, uint16_t *scales);
size_t nut_quant_data_bytes(size_t rows, size_t cols, int type);
size_t nut_quant_scale_count(size_t rows, size_t cols, size_t block_size);
/* QuantizedMatrix::storage_bytes (src/quant.cpp:235-241). */
size_t nut_quant_storage_bytes(size_t rows, size_t cols, int type,
                               size_t block_size);
/* positive_float_to_half / positive_half_to_float (src/quant.cpp:23-56). */
int nut_float_to_half(float value, uint16_t *bits);
float nut_half_to_float(uint16_t bits);
/* ModelConfig::validate (src/attention.cpp:15-27): 1 when valid. */
int nut_config_valid(const nut_config *config);

/* Synthetic workload generator (no reference counterpart: the reference
 * loads checkpoints). N(0, sigma^2) fp32 values from a counter-based
 * splitmix64 + Box-Muller stream keyed by (seed, stream); element i depends
 * only on (seed, stream, i), so any thread count gives the same array. */
int nut_synth_normal(uint64_t seed, uint64_t stream, float sigma, float *out,
                     size_t count);
/* Uniform token ids in [0, vocab) (rejection sampled) from seed. */
int nut_synth_tokens(uint64_t seed, size_t vocab, int *out, size_t count);

/* ------------------------------------------------- device and memory -- */

/* Number of visible gfx950 devices (0 on a host without a GPU). */
int nut_device_count(int *count);
/* Select the device this thread's calls use (default 0). */
int nut_set_device(int device);
int nut_malloc(void **d_ptr, size_t bytes);
int nut_free(void *d_ptr);
/* Device allocations (hipMalloc calls) this library has made since it was
 * loaded, its own and nut_malloc's (no reference counterpart: a
 * diagnostic, for checking that nut_decode_noalloc allocates nothing). */
int nut_device_allocations(unsigned long long *count);
/* Test hook (no reference counterpart): of the calling thread's next device
 * allocations by this library, `skip` succeed and `count` then fail as if the
 * device had no memory left; count = 0 takes it back. */
int nut_fail_allocations(unsigned skip, unsigned count);
int nut_memcpy_h2d(void *d_dst, const void *src, size_t bytes);
int nut_memcpy_d2h(void *dst, const void *d_src, size_t bytes);
/* Device-to-device copy (synchronous); also the known-size copy that
 * calibrates HBM traffic counters. */
int nut_memcpy_d2d(void *d_dst, const void *d_src, size_t bytes);
int nut_memset(void *d_dst, int value, size_t bytes);
int nut_synchronize(void);

/* --------------------------------------------- standalone kernels -- */

/* A QuantizedMatrix uploaded to HBM (weights verbatim, fp16 scales). */
typedef struct nut_qweight nut_qweight;
int nut_qweight_create(const nut_qmatrix *host, nut_qweight **out);
int nut_qweight_destroy(nut_qweight *w);
size_t nut_qweight_device_bytes(const nut_qweight *w);

/* y = W x on the device: matvec_quantized_threaded (src/quant.cpp:262-321).
 * stream may be NULL (the null stream). */
int nut_matvec_q(const nut_qweight *w, const float *d_x, float *d_y,
                 void *stream);
/* fp32 y = W x, W [rows x cols] row-major: matvec_threaded
 * (src/threading.cpp:183-198), the classifier kernel. */
int nut_matvec_f32(const float *d_w, size_t rows, size_t cols,
                   const float *d_x, float *d_y, void *stream);
/* fp32 C = A B, row-major A [m x k], B [k x n]: matmul_threaded
 * (src/threading.cpp:163-181). */
int nut_matmul_f32(const float *d_a, const float *d_b, float *d_c, size_t m,
                   size_t k, size_t n, void *stream);

/* Launch-time of the last nut_matvec_q / nut_matvec_f32 / nut_matmul_f32
 * batch measured with HIP events: call nut_timer_begin(stream), launch,
 * then nut_timer_end(stream, &ms) waits and returns elapsed milliseconds on
 * that stream. (No reference counterpart; the reference times with
 * std::chrono around whole calls.) */
int nut_timer_begin(void *stream);
int nut_timer_end(void *stream, double *milliseconds);

/* ------------------------------------------------------------- model -- */

typedef struct nut_model nut_model;

/* QuantizedModelWeights (include/quant_model.hpp:32-46): validates config,
 * allocates device storage for every layer; tied selects embeddings as the
 * classifier (output_weights(), include/quant_model.hpp:42-44). */
int nut_model_create(const nut_config *config, int type, int tied,
                     nut_model **out);
/* fp32 embeddings [vocab x dim], final_norm [dim], lm_head [vocab x dim]
 * (ignored when tied). */
int nut_model_set_globals(nut_model *m, const float *embeddings,
                          const float *final_norm, const float *lm_head);
/* QuantizedLayerWeights (include/quant_model.hpp:9-30): projections in
 * [out x in] layout: query dim x dim, key/value kv_dim x dim, output
 * dim x dim, gate/up ffn x dim, down dim x ffn. */
int nut_model_set_layer(nut_model *m, size_t layer, const nut_qmatrix *query,
                        const nut_qmatrix *key, const nut_qmatrix *value,
                        const nut_qmatrix *output, const nut_qmatrix *gate,
                        const nut_qmatrix *up, const nut_qmatrix *down,
                        const float *attention_norm, const float *ffn_norm);
/* QuantizedModelWeights::storage_bytes (src/quant_model.cpp:140-156). */
size_t nut_model_storage_bytes(const nut_model *m);
/* load_llama2c_quantized_model (src/llama2.cpp:339-412) straight into a
 * device model: the reference's header and size checks and messages
 * (src/llama2.cpp:199-296, run before the device is touched), pread of one
 * projection at a time, the product quantiser (bit-exact with
 * QuantizedMatrix::quantize) on a worker thread overlapping the upload of
 * the previous layer. A positive vocabulary in the header ties the
 * classifier to the embeddings; eos_token is 1. *load_seconds (may be
 * NULL) gets the load's wall time, the reference CLI's load_s
 * (src/cli.cpp:165-169). */
int nut_model_load_llama2c(const char *path, int type, nut_model **out,
                           double *load_seconds);
/* The configuration, quant type and tied flag a model was created with. */
int nut_model_config(const nut_model *m, nut_config *config, int *type,
                     int *tied);
int nut_model_destroy(nut_model *m);

/* ---------------------------------------------------------- KV cache -- */

/* KVCache (include/kvcache.hpp:8-31, src/kvcache.cpp:173-235): fp32 K and
 * V in HBM, [layer][kv_head][position][head_dim]. */
typedef struct nut_kvcache nut_kvcache;
int nut_kv_create(const nut_config *config, nut_kvcache **out);
int nut_kv_destroy(nut_kvcache *kv);
size_t nut_kv_length(const nut_kvcache *kv);
size_t nut_kv_capacity(const nut_kvcache *kv);
size_t nut_kv_memory_bytes(const nut_kvcache *kv);
int nut_kv_compatible(const nut_kvcache *kv, const nut_config *config);
int nut_kv_reset(nut_kvcache *kv);
int nut_kv_set_length(nut_kvcache *kv, size_t length);
/* KVCache::key / value: copy one [head_dim] row to the host. */
int nut_kv_read(const nut_kvcache *kv, size_t layer, size_t head,
                size_t position, float *key, float *value);
/* KVCache::store: key/value are [kv_heads x head_dim] host vectors. */
int nut_kv_store(nut_kvcache *kv, size_t layer, size_t position,
                 const float *key, const float *value);
/* KVCache::key / value / store over a run of positions at once (one
 * strided copy each way): host arrays [layer][kv_head][end - begin]
 * [head_dim]. Read-back or upload only: the length is not changed. Either
 * output of the read may be NULL. */
int nut_kv_read_positions(const nut_kvcache *kv, size_t begin, size_t end,
                          float *keys, float *values);
int nut_kv_write_positions(nut_kvcache *kv, size_t begin, size_t end,
                           const float *keys, const float *values);

/* ----------------------------------------------------- paged KV cache -- */

/* A cache of one layer's K and V rows for several sequences at once, in
 * pages of page_size rows that the caller hands out (no reference
 * counterpart: KVCache holds one sequence, contiguously). The memory is the
 * caller's; these structs are views of it. Nothing here allocates, every
 * call only launches kernels on `stream` (so it can be captured into a
 * graph), and every workspace is the caller's: calls that may run at the
 * same time, or graphs that may be replayed at the same time, need
 * workspaces of their own. What a call only writes must not overlap what it
 * reads. Device pointers are the device's that nut_set_device selected.
 *
 * Arguments that the host sees are checked (NUT_EINVAL). What only the
 * device sees is checked in the kernels: a page outside [0, pages), or a
 * sequence longer than max_length, is not read or written; it sets a bit of
 * *d_status, which nut_paged_check turns into NUT_EOUTOFRANGE. */
enum { NUT_F32 = 0, NUT_F16 = 1, NUT_BF16 = 2 };

typedef struct nut_paged_kv {
    /* Row `slot` of page p for KV head h starts at element
     * p page_stride + h head_stride + slot slot_stride of both. Strides of 0,
     * 0, 0 mean packed, [pages][kv_heads][page_size][head_dim]. Rows must
     * start at multiples of 16 bytes and must not overlap. */
    void *d_keys, *d_values;
    /* [pages][kv_heads][2][head_dim] of `type`, packed: the smallest, then
     * the largest component of a page's keys. NULL: none are kept, and
     * nut_paged_select refuses the view. */
    void *d_bounds;
    size_t pages, page_size, kv_heads;
    size_t head_dim; /* a multiple of 8, up to 256 */
    size_t page_stride, head_stride, slot_stride;
    int type;      /* NUT_F32, NUT_F16 or NUT_BF16 */
    int *d_status; /* one word, zeroed by the caller once; NULL: none */
} nut_paged_kv;

/* The sequences of a call: sequence b holds d_lengths[b] rows (0 to
 * max_length), row i in page d_pages[b table_stride + i / page_size], slot
 * i % page_size. Sequences may share pages that are only read. */
typedef struct nut_paged_batch {
    const int *d_pages;
    size_t table_stride; /* table_stride page_size >= max_length */
    const int *d_lengths;
    size_t batch, max_length;
} nut_paged_batch;

/* What eviction goes by, [batch][kv_heads][stride] each: the attention
 * weight that a row has gathered, and the position that its token had in
 * the text. stride >= max_length. */
typedef struct nut_paged_history {
    float *d_weights;
    int *d_positions;
    size_t stride;
} nut_paged_history;

/* Puts new rows behind the rows that the sequences hold. d_keys and d_values
 * hold `rows` fp32 rows: row r's head h at element r row_stride +
 * h head_stride (multiples of 4). Each stride of 0 has a default of its own,
 * that of [rows][kv_heads][head_dim]; rows and heads must not overlap.
 * Sequence b gets rows d_starts[b] to d_starts[b + 1] (at most max_new;
 * source rows that no sequence names are left out), or one row, row b, where
 * d_starts is NULL. Rows are rounded to the cache's type (to nearest, ties
 * to even), the page bounds widened, and where history is given the rows'
 * weights set to 0 and their positions to d_first_positions[b] onwards.
 * d_new_lengths (may be NULL; apart from d_lengths, d_starts and
 * d_first_positions) gets the lengths with the new rows; max_length is the
 * most that it may say. A sequence that would pass max_length gets no row and
 * keeps its length. Rows for a page outside [0, pages) are reported and
 * dropped, but counted: new lengths and history are as if they were there. No
 * two sequences may append to one page.
 *
 * d_first_positions NULL stands for d_lengths: right until nut_paged_evict
 * has cut a sequence. From then on its length is not its next token's place in
 * the text: such positions repeat, and lie below those of kept rows, so that
 * the next eviction takes the new rows for old ones. A program that evicts
 * counts each sequence's text and passes the counts. */
int nut_paged_append(const nut_paged_kv *kv, const nut_paged_batch *seqs,
                     const float *d_keys, const float *d_values, size_t rows,
                     size_t row_stride, size_t head_stride,
                     const int *d_starts, size_t max_new,
                     const nut_paged_history *history,
                     const int *d_first_positions, int *d_new_lengths,
                     void *stream);
/* nut_paged_append from a nut_kvcache, such as nut_prefill leaves: its rows
 * [begin, end) of `layer` go behind the one sequence of `seqs`. The source
 * must not change, or be destroyed, before `stream` has come past the call. */
int nut_paged_append_cache(const nut_paged_kv *kv,
                           const nut_paged_batch *seqs,
                           const nut_kvcache *source, size_t layer,
                           size_t begin, size_t end,
                           const nut_paged_history *history,
                           const int *d_first_positions, int *d_new_lengths,
                           void *stream);

/* Attention of one new token a sequence: for every head h of `heads` (a
 * multiple of kv_heads; head h reads KV head h / (heads / kv_heads)),
 * out = softmax(scale q . k) v over the sequence's rows, fp32
 * [batch][heads][head_dim]; query rows of a sequence at d_query +
 * b query_stride (0: packed; a multiple of 4). d_lse (may be NULL) gets the
 * log of each softmax's denominator, [batch][heads]. A sequence without rows,
 * or a head whose scores are all minus infinity, gets zeros and minus
 * infinity. Where a row that weighs something has a value with an infinite
 * component, that component of out is infinite or not a number; where a row of
 * weight 0 beside others has one, or a NaN, it may be not a number.
 *
 * history (may be NULL): every row's weight grows by its attention weight,
 * summed over the heads that share its KV head; the positions are not read.
 *
 * d_selected (may be NULL): [batch][kv_heads][top], only the rows of these
 * pages of the sequence's table are read (indexes into its table row, as
 * nut_paged_select writes them; -1 for none, and one behind the sequence's
 * rows has no row; a page named twice counts twice). Not together with
 * history.
 *
 * The workspace (16-byte aligned) needs nut_paged_attention_workspace bytes,
 * top = 0 standing for no selection; (size_t)-1 for arguments that the call
 * would refuse. */
size_t nut_paged_attention_workspace(const nut_paged_kv *kv,
                                     const nut_paged_batch *seqs,
                                     size_t heads, size_t top, int weighted);
int nut_paged_attention(const nut_paged_kv *kv, const nut_paged_batch *seqs,
                        const float *d_query, size_t query_stride,
                        size_t heads, float scale, const int *d_selected,
                        size_t top, const nut_paged_history *history,
                        float *d_out, float *d_lse, void *d_workspace,
                        size_t workspace_bytes, void *stream);

/* Chooses the pages that a new token's attention reads: for each sequence
 * and KV head the `first` first and the `last` last pages and the best others,
 * `top` in all (first + last <= top), in ascending order, then -1. A page's
 * score is the largest, over the heads that share the KV head, of
 * sum_d max(q_d lo_d, q_d hi_d): no row of the page has a larger q . k. Sums
 * in 64 bits, ties to the lower page; a score that is not a number (of a NaN,
 * of infinite bounds met with both signs, or of one where q_d is 0) ranks
 * first. The workspace (16-byte aligned) needs nut_paged_select_workspace
 * bytes. */
size_t nut_paged_select_workspace(const nut_paged_kv *kv,
                                  const nut_paged_batch *seqs, size_t heads,
                                  size_t top);
int nut_paged_select(const nut_paged_kv *kv, const nut_paged_batch *seqs,
                     const float *d_query, size_t query_stride, size_t heads,
                     size_t top, size_t first, size_t last, int *d_selected,
                     void *d_workspace, size_t workspace_bytes, void *stream);

/* Cuts every sequence down to `budget` rows, each KV head by its own
 * weights: rows at positions below `first` and the rows at the `last` last
 * positions stay (first + last <= budget), and of the others those of the
 * largest weight, ties to the lower row, a weight that is not a number below
 * all others. Rows that stay beyond the budget move, with their weights and
 * positions, into the places of rows that go, both in ascending order;
 * nothing else moves. The bounds of a page that rows move into are widened.
 * d_new_lengths (apart from d_lengths) gets min(length, budget). Positions
 * are distinct and not negative. Pages that hold rows below the budget must
 * not be shared. A row does not move from or to a page outside [0, pages); its
 * weight and position do. The workspace (16-byte aligned) needs
 * nut_paged_evict_workspace bytes.
 *
 * Behind an eviction a sequence's rows do not lie in the order of the text:
 * the newest are where there were holes, and the `last` pages of
 * nut_paged_select are the last by place alone. A page's bounds hold for its
 * rows, and for rows that went too: they become narrower only when an append
 * begins the page anew. Rows that no attention with history has weighed, such
 * as a prompt's from nut_paged_append_cache, all have weight 0, of which the
 * lower ones stay. */
size_t nut_paged_evict_workspace(const nut_paged_kv *kv,
                                 const nut_paged_batch *seqs, size_t budget);
int nut_paged_evict(const nut_paged_kv *kv, const nut_paged_batch *seqs,
                    const nut_paged_history *history, size_t budget,
                    size_t first, size_t last, int *d_new_lengths,
                    void *d_workspace, size_t workspace_bytes, void *stream);

/* Waits for the device, then raises what the view's status word holds
 * (NUT_EOUTOFRANGE: "paged cache: page out of range", "paged cache: length
 * out of range", "paged cache: rows out of range") and clears it. */
int nut_paged_check(const nut_paged_kv *kv);

/* -------------------------------------------------------- token loop -- */

/* decode_quantized_token (src/quant_model.cpp:158-206): one token through
 * every layer at position = length; writes the pre-final-norm hidden state
 * [dim] to hidden (host, may be NULL) and increments the length. */
int nut_decode(nut_model *m, nut_kvcache *kv, int token, float *hidden);
/* nut_decode without allocating (no reference counterpart): for callers
 * that cannot call hipMalloc (tight serving loops, harnesses that forbid
 * it). It allocates nothing, but it is not itself capturable: it runs
 * eagerly on the model's own stream and synchronizes it before returning.
 * Same validation and result as nut_decode on the step kernels
 * (NUT_PATH_STEPS); the split-attention partials and arrival counters live
 * in a per-device 2 MiB scratch array instead of model-owned allocations,
 * and the hidden state goes to the device pointer d_hidden (may be NULL). Limit: heads x splits x
 * (head_dim + 2) words of 8 bytes plus 2 x heads counters must fit 2 MiB,
 * else NUT_EINVAL (TinyLlama needs 0.55 MiB, Llama-2-7B 0.27). Every call
 * on one GPU shares that GPU's array and clears it first: calls that
 * overlap on one GPU (other host threads, other streams) race. */
int nut_decode_noalloc(nut_model *m, nut_kvcache *kv, int token,
                       float *d_hidden);
/* prefill_quantized (src/quant_model.cpp:208-220): resets the cache and
 * runs the prompt; hidden gets the last token's hidden state. */
int nut_prefill(nut_model *m, nut_kvcache *kv, const int *tokens,
                size_t count, float *hidden);
/* Final rmsnorm + fp32 classifier (src/generate.cpp:197-200) on a host
 * hidden state; logits [vocab] to the host. */
int nut_logits(nut_model *m, const float *hidden, float *logits);
/* Greedy generate_tokens_cached (src/generate.cpp:174-216) with its
 * GenerationStats timing; out receives up to max_tokens ids, stopping at
 * eos_token or a full cache. The loop runs on the device: the argmax of
 * each step feeds the next step without a host round trip. */
int nut_generate_greedy(nut_model *m, const int *prompt, size_t prompt_len,
                        size_t max_tokens, int *out, size_t *out_count,
                        nut_generation_stats *stats);

/* generate_tokens_cached with SamplingConfig{max_tokens, temperature,
 * top_p, seed} (src/generate.cpp:31-72,174-216): temperature <= 0 is the
 * greedy loop above; otherwise each step's logits, softmax numerators
 * p = exp((logit - max) / temperature) and their sort (p descending, token
 * ascending) run on the device, and the host walks the sorted prefix with
 * the reference's sequential nucleus sum and draws with std::mt19937(seed)
 * and uniform_real_distribution<double>, as choose_token does. Errors as
 * the reference's: "sampling: invalid temperature or top-p"
 * (NUT_EINVAL), "sampling: non-finite probability" and "sampling: zero
 * probability mass" (NUT_ERUNTIME). */
int nut_generate_sampled(nut_model *m, const int *prompt, size_t prompt_len,
                         size_t max_tokens, float temperature, float top_p,
                         uint32_t seed, int *out, size_t *out_count,
                         nut_generation_stats *stats);

/* ---------------------------------------------------- fp32 model path -- */

/* ModelWeights (include/loader.hpp:46-60) in HBM: fp32 embeddings
 * [vocab x dim], final_norm [dim], lm_head [vocab x dim] (ignored when
 * tied), and per layer the projections in the reference's [in x out]
 * layout (LayerWeights, src/attention.cpp:29-40): query dim x dim, key and
 * value dim x kv_dim, output dim x dim, gate and up dim x ffn, down
 * ffn x dim. The KV cache is the same nut_kvcache. */
typedef struct nut_fmodel nut_fmodel;
int nut_fmodel_create(const nut_config *config, int tied, nut_fmodel **out);
int nut_fmodel_set_globals(nut_fmodel *m, const float *embeddings,
                           const float *final_norm, const float *lm_head);
int nut_fmodel_set_layer(nut_fmodel *m, size_t layer, const float *query,
                         const float *key, const float *value,
                         const float *output, const float *gate,
                         const float *up, const float *down,
                         const float *attention_norm, const float *ffn_norm);
int nut_fmodel_destroy(nut_fmodel *m);
/* decode_token (src/kvcache.cpp:264-284): one token at position = length;
 * hidden (host, may be NULL) gets the hidden state after the last layer. */
int nut_decode_token(nut_fmodel *m, nut_kvcache *kv, int token,
                     float *hidden);
/* prefill_tokens (src/kvcache.cpp:237-262): resets the cache and runs the
 * tokens; rows (host, may be NULL) gets every token's hidden state,
 * [count x dim]. */
int nut_prefill_tokens(nut_fmodel *m, nut_kvcache *kv, const int *tokens,
                       size_t count, float *rows);

/* Execution path of decode / prefill / generate (no reference counterpart;
 * every path computes the same function): NUT_PATH_AUTO picks the
 * cooperative token kernel when the shape has an instantiation and the
 * context fits its attention (fused up to 44-48 positions, split over the
 * grid up to 4,096), else per-phase step kernels; NUT_PATH_STEPS forces the
 * step kernels; NUT_PATH_TOKEN forces the token kernel and fails with
 * NUT_EINVAL where it does not apply. */
enum { NUT_PATH_AUTO = 0, NUT_PATH_STEPS = 1, NUT_PATH_TOKEN = 2 };
int nut_model_set_path(nut_model *m, int path);

/* Phase timeline of the cooperative token kernel, for profiling (no
 * reference counterpart). mode 0 records nothing, 1 workgroup 0, 2 every
 * workgroup of the grid (256): each stamps the device's constant 100 MHz
 * clock at each phase boundary; per decode iteration 4 + 13 * layers
 * entries: iteration start, classifier input staged, classifier pass done,
 * token known (the generate loop; zero in the prefill loop), then per
 * layer the times its QKV
 * input is staged, QKV published, Wo/K/V DMA issued, attention input
 * staged, attention done, Wo published, gate/up DMA issued, FFN input
 * staged, gate/up published, down DMA issued, down input staged, down
 * published and next QKV DMA issued. Entries are
 * [workgroup][max_seq iterations][marks].
 * nut_model_timeline copies up to capacity entries of the last launch's
 * timeline. */
int nut_model_record_timeline(nut_model *m, int mode);
int nut_model_timeline(const nut_model *m, uint64_t *ticks, size_t capacity,
                       size_t *count);

/* Exchange-tag schedule of the cooperative token kernel (no reference
 * counterpart). Every launch polls words tagged with its own base; a base
 * is never 0 and never repeats until the exchange buffer has been zeroed.
 * nut_token_tag_base advances *launch_count and returns the next launch's
 * base, with *clear = 1 when the buffer must be zeroed first (the counter
 * ran out and restarted); it needs no GPU. nut_model_set_launch_count
 * presets a model's counter (a test hook, to cross the restart quickly). */
int nut_token_tag_base(unsigned *launch_count, unsigned *base, int *clear);
int nut_model_set_launch_count(nut_model *m, unsigned launch_count);
/* Test hook of the cooperative token kernel's bounded waits (no reference
 * counterpart): with fault = 1, workgroup 0 of every later launch leaves
 * its words of the first step's h after W2 unpublished, so every wait for
 * them runs into its spin limit; the launch must still end, and the call
 * fail with NUT_EDEVICE ("token kernel: phase exchange timed out").
 * fault = 0 restores normal launches. */
int nut_model_inject_fault(nut_model *m, int fault);

/* Device time (HIP events on the model's stream) of the decode loop of the
 * last nut_generate_greedy call: every classifier, argmax and decode step
 * after the prefill. (No reference counterpart: GenerationStats carries
 * host wall time only.) */
int nut_model_last_decode_ms(const nut_model *m, double *milliseconds);

#ifdef __cplusplus
}
#endif
#endif
