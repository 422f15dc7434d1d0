/* nutllm_cuda.h — C ABI of libnutcuda.so, the B200 (sm_100a) token loop.
 *
 * Plain pointers and sizes only.  Every entry point returns a nut_status;
 * nut_last_error() gives the calling thread's message for the last failure,
 * formatted "component: reason" like the reference's exceptions.  The status
 * codes map one-to-one onto the exception classes the reference throws for
 * the same conditions, so a C++ wrapper can re-throw the same type.
 *
 * Citations are to the reference project (MokiMeow/nutllm) interface each
 * entry point replaces.
 */
#ifndef NUTLLM_CUDA_H
#define NUTLLM_CUDA_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum nut_status {
    NUT_OK = 0,
    NUT_INVALID_ARGUMENT = 1, /* std::invalid_argument */
    NUT_OUT_OF_RANGE = 2,     /* std::out_of_range */
    NUT_LENGTH_ERROR = 3,     /* std::length_error */
    NUT_RUNTIME_ERROR = 4,    /* std::runtime_error, CUDA failures included */
    NUT_RANGE_ERROR = 5,      /* std::range_error */
    NUT_DEVICE_TIMEOUT = 6    /* a bounded device-side wait gave up */
} nut_status;

/* QuantType (include/quant.hpp:9-12). */
enum { NUT_QUANT_INT8 = 0, NUT_QUANT_INT4 = 1 };

/* ModelConfig (include/model.hpp:8-24); kv_heads 0 means kv_heads = heads. */
typedef struct nut_config {
    int64_t layers, heads, dim, head_dim, ffn_dim, vocab_size, max_seq,
        eos_token, kv_heads;
} nut_config;

/* Host view of a QuantizedMatrix's storage (include/quant.hpp:14-50):
 * [rows][cols] row-major, flattened blocks of block_size (must be 32)
 * weights, INT8 one byte per weight or INT4 two's-complement nibbles with
 * the even flattened index in the low nibble, one fp16 scale (bits) per
 * block. */
typedef struct nut_qmatrix_view {
    const uint8_t *data;
    const uint16_t *scales;
    int64_t rows, cols, block_size;
    int32_t type;
} nut_qmatrix_view;

/* QuantizedLayerWeights (include/quant_model.hpp:9-29): projections are
 * [out][in]: query (dim x dim), key/value (kv_dim x dim), output
 * (dim x dim), gate/up (ffn x dim), down (dim x ffn). */
typedef struct nut_layer_view {
    nut_qmatrix_view query, key, value, output, gate, up, down;
    const float *attention_norm, *ffn_norm; /* [dim] each */
} nut_layer_view;

/* QuantizedModelWeights (include/quant_model.hpp:31-46).  lm_head is
 * ignored when tied_embeddings is set (output_weights() == embeddings). */
typedef struct nut_model_view {
    nut_config config;
    int32_t quant_type;
    int32_t tied_embeddings;
    const float *embeddings; /* [vocab][dim] */
    const float *final_norm; /* [dim] */
    const float *lm_head;    /* [vocab][dim] */
    const nut_layer_view *layers;
    int64_t n_layers;
} nut_model_view;

/* fp32 ModelWeights / LayerWeights (include/loader.hpp, include/model.hpp:
 * 26-38) for the `--quant fp32` path: every projection fp32 and [out][in]
 * (the llama2.c storage; the reference's own ModelWeights holds them
 * transposed, [in][out]). */
typedef struct nut_layer_f32_view {
    const float *query, *key, *value, *output, *gate, *up, *down;
    const float *attention_norm, *ffn_norm; /* [dim] each */
} nut_layer_f32_view;

typedef struct nut_model_f32_view {
    nut_config config;
    int32_t tied_embeddings;
    const float *embeddings; /* [vocab][dim] */
    const float *final_norm; /* [dim] */
    const float *lm_head;    /* [vocab][dim], ignored when tied */
    const nut_layer_f32_view *layers;
    int64_t n_layers;
} nut_model_f32_view;

/* GenerationStats (include/generate.hpp:19-24), device-event timed. */
typedef struct nut_generation_stats {
    int64_t prefill_tokens, generated_tokens;
    double prefill_seconds, decode_seconds;
} nut_generation_stats;

typedef struct nut_qmatrix nut_qmatrix;
typedef struct nut_model nut_model;
typedef struct nut_kv nut_kv;

/* Message of the calling thread's last failure ("" if none). */
const char *nut_last_error(void);

/* Number of visible CUDA devices. */
nut_status nut_device_count(int *count);

/* ---- QuantizedMatrix device mirror (src/quant.cpp:154-321) ---------- */

/* Uploads one quantised matrix to `device`. */
nut_status nut_qmatrix_create(const nut_qmatrix_view *view, int device,
                              nut_qmatrix **out);
nut_status nut_qmatrix_destroy(nut_qmatrix *matrix);
/* Reads the device copy back in the reference storage layout. */
nut_status nut_qmatrix_download(const nut_qmatrix *matrix, uint8_t *data,
                                uint16_t *scales);
/* matvec_quantized_threaded (src/quant.cpp:262-321) with HOST buffers:
 * y[rows] = Q x[cols].  Synchronous. */
nut_status nut_qmatvec(nut_qmatrix *matrix, const float *x, float *y);
/* The same product on DEVICE buffers, enqueued on `stream` (a
 * cudaStream_t, NULL = the legacy default stream). */
nut_status nut_qmatvec_async(nut_qmatrix *matrix, const float *x_device,
                             float *y_device, void *stream);

/* Prefill form of the quantised product on DEVICE buffers, enqueued on
 * `stream`: Y[tokens][rows] = X[tokens][cols] Q^T.  Runs on the 5th-gen
 * tensor cores with fp16 operands (Q dequantised once, q * scale rounded to
 * fp16, and cached with the matrix; X rounded to fp16 per call, saturating
 * at +-65504) and fp32 accumulation, so |Y - exact| <= 2^-10 sum_k
 * |x_k q_k s_k| per element (plus fp16's subnormal step below 2^-14).
 * The reference has no batched quantised product: prefill_quantized
 * (src/quant_model.cpp:208-220) runs matvec_quantized_threaded per token;
 * this entry point is that loop over a batch of tokens.  Device-side
 * timeouts are reported by the next nut_qmatrix_error call. */
nut_status nut_qmatrix_gemm(nut_qmatrix *matrix, const float *x_device, int64_t tokens,
                            float *y_device, void *stream);
/* Synchronises the matrix's work and reports a device-side timeout of an
 * earlier asynchronous call (NUT_DEVICE_TIMEOUT), clearing it. */
nut_status nut_qmatrix_error(nut_qmatrix *matrix);

/* ---- fp32 kernels of the reference's benches -------------------------- */

/* matmul_threaded (src/threading.cpp:163-181, include/matmul.hpp:32) on
 * DEVICE buffers: c[m][n] = a[m][k] b[k][n], row-major, every output the
 * k-sequential fused multiply-add chain of the reference build (results
 * are bit-identical).  Enqueued on `stream`. */
nut_status nut_matmul_f32(const float *a, const float *b, float *c, int64_t m, int64_t k,
                          int64_t n, void *stream);
/* matvec_threaded (src/threading.cpp:183-198, include/matmul.hpp:34) on
 * DEVICE buffers: output[r] = sum_c matrix[r][c] vector[c], each row a
 * sequential sum of rounded products (bit-identical to the reference). */
nut_status nut_matvec_f32(const float *matrix, const float *vector, float *output,
                          int64_t rows, int64_t cols, void *stream);

/* ---- Model weights (include/quant_model.hpp:31-46) ------------------- */

/* Copies a QuantizedModelWeights image to `device` (layout private to the
 * library).  Fails with NUT_INVALID_ARGUMENT for an invalid config or a
 * layer whose shape does not match it (src/quant_model.cpp:161-166). */
/* decode_token / prefill_tokens over fp32 weights (src/kvcache.cpp:237-284)
 * as a nut_model: the KV cache, decode, prefill, logits and greedy
 * generation calls below take it like a quantised model (one position per
 * pass; fp32 matvecs with the reference's matvec_threaded order; the fp32
 * reference projects with linear_threaded, so parity is by tolerance). */
nut_status nut_model_create_f32(const nut_model_f32_view *view, int device, nut_model **out);
nut_status nut_model_create(const nut_model_view *view, int device,
                            nut_model **out);
/* The same model built in steps, so a loader can overlap reading and
 * quantising layer l + 1 on the host with the upload of layer l:
 * nut_model_begin takes a view whose `layers` may be NULL (the fp32
 * tensors and the configuration are uploaded and checked), then
 * nut_model_add_layer appends layers 0, 1, ... in order (each packed into
 * tiles and copied to the device before it returns; the host buffers may be
 * reused afterwards), and nut_model_finish completes the model once
 * config.layers layers were added.  A model cannot back a KV cache before
 * it is finished; nut_model_destroy releases it at any step.  nut_model_add_layer
 * may be called from another host thread than nut_model_begin, one call at
 * a time.  Same checks, classes and messages as nut_model_create
 * (reference QuantizedModelWeights construction, include/quant_model.hpp:
 * 31-53, with src/quant_model.cpp:158-172's layer-count check). */
nut_status nut_model_begin(const nut_model_view *view, int device, nut_model **out);
nut_status nut_model_add_layer(nut_model *model, const nut_layer_view *layer);
nut_status nut_model_finish(nut_model *model);
nut_status nut_model_destroy(nut_model *model);
/* QuantizedModelWeights::storage_bytes (src/quant_model.cpp:140-156). */
nut_status nut_model_storage_bytes(const nut_model *model, uint64_t *bytes);

/* The CUDA stream (a cudaStream_t) on which every call with this model
 * enqueues its work, for callers that time or order that work with their
 * own CUDA events.  No counterpart in the reference (its loop is host
 * code). */
nut_status nut_model_stream(const nut_model *model, void **stream);

/* Prompts of at least min_tokens tokens (default 64; 0 = never) are
 * prefilled as one batch: every projection of every layer as one GEMM on
 * the tensor cores with fp16 operands (weights dequantised once, rounded to
 * fp16; fp32 accumulation), instead of the per-token loop of
 * prefill_quantized (src/quant_model.cpp:208-220).  Hidden states and the
 * KV cache then carry fp16 rounding (a looser bound than the per-token
 * path's parity); set 0 to keep every prompt on the per-token path.  The
 * batch's causal attention runs in tiles that share their keys and values;
 * shapes those tiles do not take (head_dim above 128 or not a multiple of
 * 4) keep the per-token path whatever the threshold.  Applies to
 * nut_prefill and nut_generate_greedy.  No counterpart in the reference. */
nut_status nut_model_set_prefill_threshold(nut_model *model, int64_t min_tokens);

/* Total kernels this library has launched in this process (all devices),
 * for callers that account for launches per step.  No counterpart in the
 * reference. */
nut_status nut_launch_count(uint64_t *count);

/* ---- KV cache and decode state (include/kvcache.hpp:8-31) ------------ */

/* KVCache(config) (src/kvcache.cpp:173-177): fp32 keys and values of
 * capacity config.max_seq, resident on the model's device, plus the
 * sequence's decode state (last hidden vector, logits). */
nut_status nut_kv_create(nut_model *model, nut_kv **out);
nut_status nut_kv_destroy(nut_kv *kv);
nut_status nut_kv_reset(nut_kv *kv);                   /* KVCache::reset */
nut_status nut_kv_length(const nut_kv *kv, int64_t *length);
nut_status nut_kv_set_length(nut_kv *kv, int64_t length); /* :231-235 */
nut_status nut_kv_memory_bytes(const nut_kv *kv, uint64_t *bytes);
/* KVCache::store (src/kvcache.cpp:216-229): writes the keys and values of
 * every kv head (kv_heads x head_dim floats each, host) at (layer,
 * position); the length is unchanged. */
nut_status nut_kv_write(nut_kv *kv, int64_t layer, int64_t position, const float *keys,
                        const float *values);
/* KVCache::key / KVCache::value (src/kvcache.cpp:207-214): copies one
 * head_dim vector of each to the host (either pointer may be NULL). */
nut_status nut_kv_read(const nut_kv *kv, int64_t layer, int64_t head,
                       int64_t position, float *key, float *value);

/* ---- Token loop -------------------------------------------------------- */

/* decode_quantized_token (src/quant_model.cpp:158-206): runs one token
 * through every layer at position kv length, appends its keys and values
 * and advances the length.  hidden (dim floats, host) may be NULL; the
 * pre-final-norm hidden vector stays on the device for nut_logits. */
nut_status nut_decode_token(nut_model *model, nut_kv *kv, int32_t token,
                            float *hidden);
/* prefill_quantized (src/quant_model.cpp:208-220): resets the cache and
 * feeds the prompt; hidden (dim floats, host) may be NULL. */
nut_status nut_prefill(nut_model *model, nut_kv *kv, const int32_t *tokens,
                       int64_t n, float *hidden);
/* Final rmsnorm + fp32 lm_head + first-index argmax over the last hidden
 * vector (src/generate.cpp:197-201).  Either output may be NULL. */
nut_status nut_logits(nut_model *model, nut_kv *kv, float *logits,
                      int32_t *argmax);
/* Greedy generate_tokens_cached (src/generate.cpp:174-216): prefill, then
 * up to max_tokens greedy steps, the whole loop on the device.  With
 * stop_at_eos set, a chosen eos_token ends the loop without being emitted
 * (the reference behaviour); with it clear, exactly max_tokens ids are
 * produced (the parity-harness form).  ids has room for max_tokens;
 * logits (max_tokens x vocab, host) and stats may be NULL. */
nut_status nut_generate_greedy(nut_model *model, nut_kv *kv,
                               const int32_t *prompt, int64_t n,
                               int64_t max_tokens, int32_t stop_at_eos,
                               int32_t *ids, int64_t *n_generated,
                               float *logits, nut_generation_stats *stats);

/* ---- Batched decode, tensor parallel ----------------------------------- */

/* B independent sequences generated in lockstep (BASELINE's 7B-shape
 * configuration: batch 64, equal prompt lengths), sharded over `world`
 * ranks, one process per GPU: rank r holds heads [r H/world, (r+1) H/world)
 * of Wq/Wk/Wv and the matching Wo columns, hidden units
 * [r F/world, (r+1) F/world) of Wgate/Wup and the matching Wdown columns,
 * and classifier rows [r V/world, (r+1) V/world); Wo and Wdown partial
 * outputs are summed with one NCCL all-reduce each per layer, the argmax
 * with a 64-bit max all-reduce (first-index tie rule of std::max_element).
 * Heads, kv heads and ffn / 32 must divide by world.  No reference
 * counterpart: the reference generates one sequence at a time on the CPU
 * (src/generate.cpp:174-216); this is that loop for a batch, with the
 * projections as fp16 tensor-core GEMMs (dequantised weights and fp16
 * activations, so logits follow the prefill GEMM's stated bound). */
typedef struct nut_batch nut_batch;

/* ncclGetUniqueId for rank 0 to share with the others (size >= 128). */
nut_status nut_tp_unique_id(uint8_t *id, int64_t size);
/* This rank's shard of a host model (every rank passes the whole view);
 * nccl_id may be NULL when world == 1. */
nut_status nut_batch_create(const nut_model_view *view, int device, int64_t batch, int rank,
                            int world, const uint8_t *nccl_id, nut_batch **out);
/* The same with seeded synthetic weights generated on the device (random
 * INT4 block-32 projections, N(0, 0.02) embeddings and classifier, unit norm
 * gains), for shapes too large to build on the host. */
nut_status nut_batch_create_synthetic(const nut_config *config, uint64_t seed, int device,
                                      int64_t batch, int rank, int world,
                                      const uint8_t *nccl_id, nut_batch **out);
void nut_batch_destroy(nut_batch *batch);
/* info[8] = {batch, heads, kv heads, ffn units, first vocabulary row, vocabulary
 * rows (all of this rank), weight bytes held, world}. */
nut_status nut_batch_info(const nut_batch *batch, int64_t *info);
nut_status nut_batch_stream(nut_batch *batch, void **stream);
/* Peer-memory all-reduce in place of NCCL for the Wo and Wdown sums: each
 * rank exports an IPC handle of its receive area (size >= 64 bytes per
 * handle), the ranks exchange them (e.g. an all-gather on the host), and
 * each opens everyone's handles [world][stride bytes].  Collective, world
 * <= 8, one process per GPU; the argmax still uses NCCL. */
nut_status nut_batch_ipc_handle(nut_batch *batch, uint8_t *handle, int64_t size);
nut_status nut_batch_open_peers(nut_batch *batch, const uint8_t *handles, int64_t stride);
/* Prompts of at least min_tokens tokens (default 16; 0 = never) are
 * prefilled as GEMMs over chunks of whole sequences (causal attention per
 * sequence, in tiles that share their keys and values) instead of one
 * position per pass; shapes the tiles do not take (per-rank head_dim above
 * 128 or not a multiple of 4) keep one position per pass. */
nut_status nut_batch_set_prefill_threshold(nut_batch *batch, int64_t min_tokens);
/* This rank's shard without creating anything (host only): shard[8] =
 * {first head, heads, first kv head, kv heads, first ffn unit, ffn units,
 * first vocabulary row, vocabulary rows}. */
nut_status nut_tp_shard(const nut_config *config, int rank, int world, int64_t *shard);
/* Prompts [batch][n] (host), then `steps` greedy tokens per sequence
 * without an eos stop: ids [batch][steps] (host).  logits [steps][batch]
 * [this rank's vocabulary rows] (host) may be NULL.  Collective: every rank
 * calls it with the same arguments. */
nut_status nut_batch_generate(nut_batch *batch, const int32_t *prompts, int64_t n,
                              int64_t steps, int32_t *ids, float *logits,
                              nut_generation_stats *stats);

/* One call of the peer-memory all-reduce (fp32 sum of n floats, n % 4 ==
 * 0) that the tensor-parallel decoder can use in place of NCCL, on
 * caller-owned buffers: recv[q] / flags[q] are rank q's receive area
 * ([2][world][n] floats) and flag words ([world][NUT_PEER_AR_CHUNKS]), as
 * this process addresses them (its own, or IPC mappings of the peers'),
 * zeroed before the first call; epochs [NUT_PEER_AR_CHUNKS] and error [1]
 * are this rank's, zeroed before the first call.  Every rank makes the same
 * sequence of calls with the same n.  Each wait for a peer's chunk gives up
 * after limit_ns nanoseconds: the call then returns NUT_DEVICE_TIMEOUT (the
 * kernel has ended; the device stays usable) and clears the error word.
 * Synchronises `stream` to read the error word.  The reference has no
 * multi-GPU path; like its RowExecutor, which hands a worker's failure back
 * to the caller (src/threading.cpp:58-74,91-99), a failed wait is reported
 * to the caller instead of hanging. */
#define NUT_PEER_AR_CHUNKS 128
nut_status nut_peer_all_reduce(const float *x, float *out, int64_t n, float *const *recv,
                               unsigned *const *flags, int rank, int world, unsigned *epochs,
                               int *error, int64_t limit_ns, void *stream);

/* ---- Paged KV cache ------------------------------------------------------ */

/* Keys and values of many sequences of unequal length in one pool of
 * fixed-size pages, in the CALLER's device memory, and the operators on it.
 * The reference keeps one contiguous fp32 cache per sequence (include/
 * kvcache.hpp:8-31); KVCache::store, the rotation and attention_step
 * (src/quant_model.cpp:26-105) are what nut_paged_append and
 * nut_paged_attention do for a batch of such caches. */

/* Element types of caches and rows. */
enum { NUT_F32 = 0, NUT_F16 = 1, NUT_BF16 = 2 };

/* The pool and its tables (device pointers).  Slot t of sequence s lies in
 * page table[s][t / page_size] at place t % page_size; element d of kv head
 * h of that slot at
 *   page * page_stride + h * head_stride + place * slot_stride + d
 * of `keys` and of `values`.  All three strides 0 means contiguous
 * [n_pages][kv_heads][page_size][head_dim].  head_dim is a multiple of 8 up
 * to 256; keys, values and the strides are multiples of 16 bytes.  Pages of
 * different sequences must differ.  Table entries behind a sequence's last
 * page are never read.
 *   lengths  slots in use of each sequence, read on the device by every call
 *            (0 is an idle place); the caller advances it before it appends.
 *   bounds, bound_scales  (both or neither; bounds a multiple of 16 bytes) the key bounds of every page and
 *            kv head, for nut_paged_select: greatest and least key of each
 *            dimension over the page's used slots, as int8 in units of
 *            bound_scales (a power of two, the least under which all fit
 *            127), the greatest rounded up and the least down.  Kept by
 *            nut_paged_append and nut_paged_summarise.  NaN keys count as 0
 *            and infinite ones as the largest finite float.
 *   max_rows  most rows of one attention or select call (0: sequences).
 *   track_weights  nut_paged_attention may be asked for attention weights
 *            (costs [sequences][heads][max_pages * page_size] floats). */
typedef struct nut_paged_view {
    void *keys, *values;
    const int32_t *table;   /* [sequences][max_pages] */
    const int32_t *lengths; /* [sequences] */
    int8_t *bounds;         /* [n_pages][kv_heads][2][head_dim], or NULL */
    float *bound_scales;    /* [n_pages][kv_heads], or NULL */
    int64_t page_stride, head_stride, slot_stride; /* in elements */
    int64_t sequences, max_pages, n_pages, page_size;
    int64_t heads, kv_heads, head_dim, max_rows;
    int32_t type; /* of keys and values */
    int32_t track_weights;
} nut_paged_view;

/* A handle on a pool: the view and this library's workspace for it.  The
 * operators enqueue on `stream` (a cudaStream_t, NULL = the legacy default
 * stream) and return without synchronising; none allocates.  The workspace
 * takes 4 bytes for every sequence, kv head and slot of the table (what an
 * eviction moves), with bounds 4 for every row, kv head and page, with
 * track_weights 4 for every sequence, head and slot.  Calls of one
 * handle share its workspace: issue them on one stream or order the streams
 * with events. */
typedef struct nut_paged nut_paged;

nut_status nut_paged_create(const nut_paged_view *view, int device, nut_paged **out);
nut_status nut_paged_destroy(nut_paged *paged);
/* Synchronises `stream` and reports what the device saw wrong in earlier
 * calls' device-resident arguments (NUT_OUT_OF_RANGE: a page number outside
 * the pool, a length outside the table, a row's sequence, a position beyond
 * the rotation table, inconsistent `starts`), clearing it.  The work that
 * met it was skipped: an append stores no row without a slot or a position;
 * an attention leaves out the slots of a bad page, which get no weight, and
 * a row of a bad length or sequence sees nothing; a selection ranks a bad
 * page last; an eviction leaves its sequence as it is.  Nothing outside the
 * caller's buffers is touched.  NUT_DEVICE_TIMEOUT: a copy from the pool did
 * not arrive within seconds; the outputs since are not to be used, and
 * weights_out was not written. */
nut_status nut_paged_error(nut_paged *paged, void *stream);

/* Appends new tokens.  The rows of sequence s are starts[s] ..
 * starts[s + 1] - 1, its newest ones: with n of them they take slots
 * lengths[s] - n .. lengths[s] - 1 and positions seen[s] - n .. seen[s] - 1.
 * Row r of k and v is [kv_heads][head_dim] at r * k_stride / v_stride
 * elements (0: contiguous), likewise q, q_out [heads][head_dim].  Queries
 * and keys are rotated in neighbouring pairs in fp32 with unfused products,
 * as the token loop does (src/quant_model.cpp:26-37), then rounded to the
 * type of q_out / the cache (fp16 saturates at +-65504). */
typedef struct nut_paged_append_args {
    const void *q; /* NULL: keys and values only */
    const void *k, *v;
    void *q_out; /* may be q */
    int64_t q_stride, k_stride, v_stride, q_out_stride;
    const int32_t *starts; /* [sequences + 1], ascending from 0 */
    int64_t rows;    /* starts[sequences] */
    int64_t max_new; /* most rows of one sequence */
    const float *rope_cos, *rope_sin; /* [rope_rows][head_dim / 2]; NULL: no rotation */
    int64_t rope_rows;
    const int32_t *seen; /* [sequences] tokens so far, these included; NULL: lengths */
    /* [sequences][kv_heads][max_pages * page_size], each or NULL: the new
     * slots' positions are recorded, their weights set to 0 */
    int32_t *positions;
    float *weights;
    int32_t type; /* of q, k, v and q_out */
} nut_paged_append_args;
nut_status nut_paged_append(nut_paged *paged, const nut_paged_append_args *args, void *stream);
/* Recomputes the key bounds of every used page of every sequence (after
 * keys were written or moved by other means than nut_paged_append). */
nut_status nut_paged_summarise(nut_paged *paged, void *stream);

/* out[r][h] = sum_t w_t v_t with w = softmax_t(scale q[r][h] . k_t) over the
 * first row_length[r] slots of sequence row_sequence[r], kv head
 * h / (heads / kv_heads).  A row that sees nothing gives zeros and
 * lse = -infinity.  Sums, the softmax and its statistics are fp32.  What
 * multiplies a 16-bit cache is split into 16-bit terms: fp32 queries and
 * their weights keep 22 bits (fp16) or 24 (bf16), the weights of bf16 rows
 * 16; weights below 2^-21 of a row's greatest on an fp16 cache are exact to
 * 2^-43 of it.
 * `selected` restricts row r, kv head g to the pages whose numbers within the
 * sequence are listed, in any order, -1 for none; a page listed twice counts
 * twice.  With weights / weights_out (one row per sequence, no `selected`)
 *   weights_out[s][g][t] = weights[s][g][t] + sum of w_t over the group's heads
 * for the slots in use; the two may be the same buffer.  (A prompt's tokens
 * are ranked by attending its newest rows a second time, one row of every
 * sequence a call, with row_length.) */
typedef struct nut_paged_attention_args {
    const void *q; /* [rows][heads][head_dim] */
    void *out;
    int64_t q_stride, out_stride; /* elements between rows; 0: contiguous */
    float *lse; /* [rows][heads] natural log of the softmax sum, or NULL */
    const int32_t *row_sequence; /* [rows]; NULL: row r is sequence r */
    const int32_t *row_length;   /* [rows]; NULL: the sequence's length */
    const int32_t *selected;     /* [rows][kv_heads][n_selected], or NULL */
    int64_t n_selected;
    const float *weights; /* [sequences][kv_heads][max_pages * page_size], or NULL */
    float *weights_out;
    int64_t rows;
    float scale;  /* 0: 1 / sqrt(head_dim) */
    int32_t type; /* of q and out: NUT_F32 or the cache's */
} nut_paged_attention_args;
nut_status nut_paged_attention(nut_paged *paged, const nut_paged_attention_args *args,
                               void *stream);

/* Chooses pages for each row and kv head by a score that bounds the logits up
 * to the queries' rounding: with each query head in 8 bits, x = rint(q / u), u the least power of two
 * under which |x| <= 127,
 *   score(page) = max over the group's heads of
 *                 u * bound_scale * sum_d max(x_d greatest_d, x_d least_d).
 * Every term is an integer times a power of two, so the score is exact (up
 * to fp32's greatest numbers, which stand for what lies beyond them) and the
 * choice does not depend on the order of any sum.  The first sink_pages
 * and the last recent_pages pages of the row's length come before all
 * others; then the highest scores, ties to the lowest page.  selected[r][g]
 * receives the min(n_selected, pages) chosen ones ascending, then -1. */
typedef struct nut_paged_select_args {
    const void *q;
    int64_t q_stride;
    const int32_t *row_sequence, *row_length; /* as for the attention */
    int32_t *selected; /* [rows][kv_heads][n_selected] */
    int64_t n_selected, sink_pages, recent_pages, rows;
    int32_t type;
} nut_paged_select_args;
nut_status nut_paged_select(nut_paged *paged, const nut_paged_select_args *args, void *stream);

/* Trims each sequence to `budget` slots, for each kv head on its own: kept
 * are the tokens with position < sinks or >= seen - recent, then those with
 * most weight (ties: the lowest slot; a NaN weight is the least, an infinite
 * one ranks with the protected tokens).  The kept
 * tokens in slots from the new length on move into the freed slots below
 * it, both taken in ascending order; keys were rotated when stored, so the
 * order of slots does not matter to the attention.  weights_out and
 * positions_out (which may be weights / positions) receive the moved
 * entries, 0 and -1 in the slots given up, and new_lengths (which may be
 * the view's lengths) min(length, budget).  A sequence with a bad length or,
 * where it has to be trimmed, a bad page number stays as it is in all of
 * these.  Key bounds are not recomputed
 * (nut_paged_summarise). */
typedef struct nut_paged_evict_args {
    const float *weights;     /* [sequences][kv_heads][max_pages * page_size] */
    const int32_t *positions; /* same shape; NULL (with positions_out) if sinks == recent == 0 */
    const int32_t *seen;      /* [sequences]; NULL if recent == 0 */
    int64_t budget, sinks, recent;
    int32_t *new_lengths; /* [sequences] */
    float *weights_out;
    int32_t *positions_out;
} nut_paged_evict_args;
nut_status nut_paged_evict(nut_paged *paged, const nut_paged_evict_args *args, void *stream);

/* ---- Decoding that branches --------------------------------------------- */

/* The reference follows one continuation of one sequence
 * (generate_tokens_cached, src/generate.cpp:174-216).  Here several
 * continuations share a paged cache: trees of drafted tokens that one pass
 * verifies (nut_paged_append_at, nut_paged_tree_attention,
 * nut_paged_compact), and beams (nut_beam_select) whose pages fork
 * (nut_pages_update, nut_paged_copy).  All of it stays on the device and can
 * be captured in a graph. */

/* nut_paged_append with a position of its own for each row (drafted tokens
 * of one depth share one): row_position [rows]; args->seen is not read.  A
 * row whose position is negative or has no rotation is skipped. */
nut_status nut_paged_append_at(nut_paged *paged, const nut_paged_append_args *args,
                               const int32_t *row_position, void *stream);

/* Workspace for nut_paged_tree_attention calls of up to max_new (1 to
 * NUT_TREE_MAX) drafted tokens a sequence: on 148 SMs 592 parts of
 * min(128, max_new * heads / kv_heads) rows of head_dim + 3 floats.
 * Allocates, so not within a capture.  Called again with more it allocates
 * anew; what earlier captures use stays until the handle goes. */
#define NUT_TREE_MAX 1024
nut_status nut_paged_reserve_tree(nut_paged *paged, int64_t max_new);

/* Attention of the drafted tokens of every sequence in one pass over its
 * cache.  The rows of sequence s are starts[s] .. starts[s + 1] - 1; with n
 * of them they are the tokens in its slots P .. P + n - 1, P = lengths[s] - n.
 * Row r sees the slots below P and slot P + j where bit j % 32 of
 * mask[r][j / 32] is set (itself only with its own bit; bits from n on are
 * not read):
 *   out[r][h] = sum_t w_t v_t,  w = softmax_t(scale q[r][h] . k_t)
 * over the slots it sees, kv head h / (heads / kv_heads).  A row that sees
 * nothing gives zeros and lse = -infinity.  Masks need not be those of a
 * tree.  Whatever is stored in slots that a row does not see, infinities and
 * NaN included, has no part in its outputs; an infinity or NaN among the
 * values it sees makes that dimension of its output infinite or NaN, and an
 * infinite key that it sees may make the row NaN.  Sums, the softmax and its
 * statistics are fp32.  Products are formed from 16-bit terms where the cache
 * has 16 bits: fp32 queries and their weights in two (fp16) or three (bf16)
 * of them, rows of the cache's type in one (weights within 2^-8 of themselves
 * on bf16, 2^-11 on fp16; the sum is taken before).
 * Rows behind starts[sequences] are left as they were; out is no part of q.
 * A sequence whose `starts` do not ascend within `rows` is skipped (its rows stay); where its
 * length is bad or n exceeds it or max_new, its rows see nothing; slots of a
 * bad page are not seen.  All of these are reported (nut_paged_error). */
typedef struct nut_paged_tree_args {
    const void *q; /* [rows][heads][head_dim] */
    void *out;
    int64_t q_stride, out_stride; /* elements between rows; 0: contiguous */
    float *lse;            /* [rows][heads] natural log of the softmax sum, or NULL */
    const int32_t *starts; /* [sequences + 1], ascending from 0 */
    const uint32_t *mask;  /* [rows][mask_words] */
    int64_t mask_words;    /* at least max_new / 32, rounded up */
    int64_t rows;          /* rows there are: starts[sequences] or more */
    int64_t max_new;       /* most rows of one sequence, as reserved or fewer */
    float scale;           /* 0: 1 / sqrt(head_dim) */
    int32_t type;          /* of q and out: NUT_F32 or the cache's */
} nut_paged_tree_args;
nut_status nut_paged_tree_attention(nut_paged *paged, const nut_paged_tree_args *args,
                                    void *stream);

/* Keeps the accepted ones of each sequence's drafted tokens next to one
 * another: with n = starts[s + 1] - starts[s] and P = lengths[s] - n, the
 * keys and values of slot P + accepted[s][i] move to slot P + i, and
 * new_lengths[s] = P + the number accepted.  accepted[s] holds ascending
 * numbers below n, then -1.  positions and weights (each or NULL) move with
 * them.  A sequence with a bad length, starts, list or page is left as it is
 * (new_lengths[s] = lengths[s]) and reported.  new_lengths may be the view's
 * lengths where nothing else goes by them.  Handles that share lengths (a
 * model's layers) are all compacted from the lengths as they were, and a book
 * of pages (nut_pages) counts holders by them: there new_lengths is an array
 * of its own, the `keep` of the next nut_pages_update.  Key bounds are not
 * recomputed (nut_paged_summarise). */
typedef struct nut_paged_compact_args {
    const int32_t *starts;   /* [sequences + 1] */
    const int32_t *accepted; /* [sequences][n_accepted] */
    int64_t n_accepted;      /* up to NUT_TREE_MAX */
    int32_t *new_lengths;    /* [sequences] */
    int32_t *positions;      /* [sequences][kv_heads][max_pages * page_size], or NULL */
    float *weights;          /* same shape, or NULL */
} nut_paged_compact_args;
nut_status nut_paged_compact(nut_paged *paged, const nut_paged_compact_args *args, void *stream);

/* Copies pages: keys and values of the first slots[i] slots (NULL: of all)
 * of page source[i] to page target[i], and its key bounds where the pool has
 * them.  Entries with both -1 are passed over, other pages outside the pool
 * are reported and passed over.  No target may be listed twice or be a
 * source. */
typedef struct nut_paged_copy_args {
    const int32_t *source, *target; /* [count] */
    const int32_t *slots;           /* [count], or NULL */
    int64_t count;
} nut_paged_copy_args;
nut_status nut_paged_copy(nut_paged *paged, const nut_paged_copy_args *args, void *stream);

/* The pages of many sequences, in the CALLER's device memory: the table and
 * lengths of one or more nut_paged (a model's layers share them), how many
 * holders each page has, and which pages have none.
 *   refs        entries of the table that hold a page (used pages of every
 *               sequence), plus what the caller holds itself (a prompt kept
 *               for later, say)
 *   free_pages  its first free_count[0] entries are the pages without a
 *               holder; pages are taken from the end of them and given back
 *               there
 * A sequence may write to the slots that its newest update gave it room for:
 * no one else holds their pages.  Others may be shared and are only read
 * (nut_paged_evict, which moves slots anywhere, is not for sequences of a
 * book).  Positions and weights of slots belong to a sequence, not to its
 * pages: they do not follow `parent`. */
typedef struct nut_pages_view {
    int32_t *table;      /* [sequences][max_pages] */
    int32_t *lengths;    /* [sequences] */
    int32_t *refs;       /* [n_pages] */
    int32_t *free_pages; /* [n_pages] */
    int32_t *free_count; /* [1] */
    int64_t sequences, max_pages, n_pages, page_size;
} nut_pages_view;

/* A handle on them with this library's workspace (12 bytes a page, 4 for every
 * entry of the table); as for nut_paged, calls of one handle are
 * ordered by the caller, and none of them allocates. */
typedef struct nut_pages nut_pages;

nut_status nut_pages_create(const nut_pages_view *view, int device, nut_pages **out);
nut_status nut_pages_destroy(nut_pages *pages);
/* Synchronises `stream` and reports what earlier updates met, clearing it:
 * NUT_LENGTH_ERROR (not enough free pages) or NUT_OUT_OF_RANGE (an argument,
 * a table entry or the book out of range). */
nut_status nut_pages_error(nut_pages *pages, void *stream);

/* Every sequence s continues sequence parent[s] (-1: nothing): it keeps the
 * first k = min(keep[s], length of parent[s]) slots and gets room for add[s]
 * more; lengths[s] = k + add[s].  All sequences change at once.
 *   - Pages of kept slots are shared with every other sequence that keeps
 *     them.
 *   - Where add[s] > 0 and the page of slot k - 1 is only partly kept, s
 *     writes to it.  If others hold that page too, s gets a page of its own
 *     instead, and copy_from[s], copy_to[s], copy_slots[s] say what
 *     nut_paged_copy has to copy in each layer (-1, -1, 0: nothing); when all
 *     of its holders are sequences that write to it in this call, the first
 *     of them keeps it.
 *   - New pages are taken from the end of free_pages in order of s, and
 *     within s a copy's page first, then ascending.
 *   - Pages that lost their last holder are then given back, ascending;
 *     they cannot be taken by the same call.
 * Table entries behind a sequence's last page stay as they were.  If a
 * parent, keep, add, length or page is out of range, a sequence outgrows its
 * table, or the free pages do not suffice, nothing changes: the copy lists
 * are all -1 (and 0), and the error is kept for nut_pages_error.  (Lengths are
 * the old ones then: a loop that appends without having asked writes over its
 * sequences' newest slots.  Pages of entries that stay are not looked at.  A
 * book whose refs are fewer than the table shows, or which lists pages in use
 * as free, is reported where an update meets it; what changed is then not
 * undone.) */
typedef struct nut_pages_update_args {
    const int32_t *parent; /* [sequences]; NULL: itself */
    const int32_t *keep;   /* [sequences], not negative; NULL: all */
    const int32_t *add;    /* [sequences], not negative; NULL: none */
    int32_t *copy_from, *copy_to, *copy_slots; /* [sequences] each; NULL, all three, only without `add` */
} nut_pages_update_args;
nut_status nut_pages_update(nut_pages *pages, const nut_pages_update_args *args, void *stream);

/* Beam search's choice for up to `sequences` requests of `beams` beams each
 * over a vocabulary, the n_out best of each request.  n_out up to
 * NUT_BEAM_MAX_OUT.  The handle holds the workspace; calls of one handle
 * are ordered by the caller, and none of them allocates. */
#define NUT_BEAM_MAX_OUT 64
typedef struct nut_beam nut_beam;
nut_status nut_beam_create(int64_t sequences, int64_t beams, int64_t vocab, int64_t n_out,
                           int device, nut_beam **out);
nut_status nut_beam_destroy(nut_beam *beam);

/* Of the candidates (beam b, token t) of request s with
 *   score(b, t) = scores[s][b] + logits[s beams + b][t] - log sum_u exp(logits[..][u])
 * (the sum in fp32 with the parts joined in fp64, scores compared in fp64) the
 * n_out greatest in descending order, ties to the lowest beam, then the lowest
 * token.  A finished beam has one candidate, (b, eos) with score scores[s][b],
 * and its logits are not read.  NaN counts as -infinity in logits and scores,
 * a logit of +infinity as the greatest finite float; candidates of
 * score -infinity rank last.  (Where different logits of a beam round to equal
 * scores in fp64, beside scores of 2^40 and more or because they are next to
 * nothing themselves, which of their tokens go first is not specified.)
 * Where there are fewer candidates than n_out,
 * rows and tokens are -1 and scores -infinity behind them.  The choice does
 * not depend on timing.  out_scores and out_finished may be scores and finished
 * where n_out is beams. */
typedef struct nut_beam_select_args {
    const void *logits;      /* [sequences * beams][vocab] */
    int64_t logits_stride;   /* elements between rows; 0: vocab */
    const float *scores;     /* [sequences][beams] */
    const uint8_t *finished; /* [sequences][beams], or NULL: none */
    float *out_scores;       /* [sequences][n_out], rounded to fp32 */
    int32_t *out_rows;       /* s * beams + b: a row of logits, and a `parent` of nut_pages_update */
    int32_t *out_tokens;
    uint8_t *out_finished;   /* the beam's, or 1 where the token is eos; or NULL */
    int64_t sequences;       /* as created or fewer */
    int32_t eos;             /* -1: none */
    int32_t type;            /* of logits */
} nut_beam_select_args;
nut_status nut_beam_select(nut_beam *beam, const nut_beam_select_args *args, void *stream);

/* ---- Greedy head without allocation ------------------------------------ */

/* Largest batch of nut_greedy_head_static. */
#define NUT_GREEDY_HEAD_MAX_BATCH 64

/* Final rmsnorm + fp32 classifier + first-index argmax of `batch` hidden
 * vectors, with every buffer in caller-provided DEVICE memory and no
 * allocation of any kind.  It is for callers that cannot call cudaMalloc
 * or cudaFree: code whose device memory is handed out by a host runtime's
 * own arena, or that issues GPU work where allocating is not allowed, and
 * which therefore cannot create the nut_model / nut_kv objects whose
 * buffers the rest of this ABI owns.  The kernels' only scratch, one
 * 64-bit argmax accumulator per batch row, is a fixed array of
 * NUT_GREEDY_HEAD_MAX_BATCH entries in this library's device memory, which
 * every GPU that loads the library keeps until the process exits; a larger
 * batch fails with NUT_LENGTH_ERROR.  The first call on a device resolves
 * the array's address (with that device current) and should come before
 * any stream capture.  Every call shares the array and clears the rows it
 * uses: calls whose work overlaps on the GPU race, so the caller must
 * serialise them.  A cudaDeviceReset() after the first call on a device is
 * not supported.
 *   hidden [batch][dim], final_norm [dim], weights [vocab][dim] (fp32),
 *   logits [batch][vocab] (may be NULL), argmax [batch] (int32);
 *   enqueued on `stream` (a cudaStream_t, NULL = legacy default stream).
 * Pointers need only their element's alignment (4 bytes; others fail with
 * NUT_INVALID_ARGUMENT); 16-byte-aligned weights with dim % 4 == 0 are read
 * as float4.  This entry point has no counterpart in the reference;
 * nut_logits is this library's model-handle form of the same head. */
nut_status nut_greedy_head_static(const float *hidden, const float *final_norm,
                                  const float *weights, int64_t batch, int64_t vocab,
                                  int64_t dim, float *logits, int32_t *argmax,
                                  void *stream);

#ifdef __cplusplus
}
#endif
#endif /* NUTLLM_CUDA_H */
