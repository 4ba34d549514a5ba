/*
 * nve_amd_ext.h -- extensions of the MI355X lookup library beyond the
 * reference's C ABI (include/nve_c_api.h).  Same conventions: every call
 * returns nve_status_t, messages go to nve_get_last_error, streams are
 * hipStream_t passed as void*.  Pointers documented as "device" must be
 * GPU-readable (device memory, or pinned host memory for a table).
 */
#ifndef NVE_AMD_EXT_H
#define NVE_AMD_EXT_H

#include "nve_c_api.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Row formats without a reference counterpart (the reference has no int8
 * affine row with fp32 offset and no fp8 row; nve_types.hpp:59-73).  Both
 * dequantize in fp32 and may be emitted as fp16 or fp32:
 *   NVE_DTYPE_X_INT8_AFFINE_F32: int8 q[count], f32 scale, f32 offset;
 *                                value = fma(q, scale, offset)
 *   NVE_DTYPE_X_E4M3_ROWWISE_F32: OCP fp8 e4m3 q[count], f32 scale;
 *                                value = e4m3(q) * scale
 * and the 4-bit format of the key-value cache's pages, OCP MXFP4 (no table
 * stores it, no lookup emits it):
 *   NVE_DTYPE_X_MXFP4: e2m1 codes (0, .5, 1, 1.5, 2, 3, 4, 6 and a sign), value
 *                      2i in the low half of byte i, with an e8m0 scale (the
 *                      exponent byte of a power of two, 255: NaN) for every 32;
 *                      value = e2m1(code) * scale */
enum {
  NVE_DTYPE_X_INT8_AFFINE_F32 = 32,
  NVE_DTYPE_X_E4M3_ROWWISE_F32 = 33,
  NVE_DTYPE_X_MXFP4 = 34,
};

/* Fused find-and-pool over a linear table, keys and outputs in device memory.
 * Restates the reference's kernel-level router find_and_pool
 * (cuda_ops/find_and_pool.cuh:103-132) with a linear table
 * (ECNoCache, load_indices = true): Concatenate emits one dequantized row per
 * key, every other pooling type one fp32-accumulated row per bag.  Keys
 * outside [0, num_rows) read nothing: their Concatenate output rows are left
 * as they are, and a bag counts them as zero rows.
 * output_type: the value type's float precision (either precision for the
 * extension types).  split_hint: 0 lets the library choose how many lane
 * groups share a bag; > 0 forces that many (a power of two); < 0 forces one
 * group per bag (strict key order).  unroll_hint: 0 lets the library choose how
 * many row loads each lane group keeps in flight; 8 or 16 forces it. */
NVE_C_API nve_status_t nve_amd_find_and_pool(
    nve_key_type_t key_type, int64_t num_keys, const void* keys, const void* table,
    int64_t num_rows, int64_t row_size_in_bytes, nve_data_type_t value_dtype,
    nve_pooling_type_t pooling_type, nve_sparse_type_t sparse_type, const void* csr_offsets,
    int64_t num_csr_offsets, int64_t fixed_hotness, const void* weights,
    nve_data_type_t weight_type, nve_data_type_t output_type, void* output,
    int64_t output_stride, int32_t split_hint, int32_t unroll_hint, void* stream);

/* Multi-table jagged pooling in one launch (the reference pools one table per
 * call; this fuses a batch of num_tables tables of equal row format, as a
 * TorchRec KeyedJaggedTensor lays them out).  tables: host array of
 * num_tables device table pointers; table_rows: host array of their row
 * counts (keys outside [0, table_rows[t]) read nothing), or NULL for no bound
 * check.  keys: num_keys keys of the key type,
 * table-major.  offsets: num_tables*batch_size + 1 entries of the key type;
 * bag (t, b) holds keys [offsets[t*batch_size + b], offsets[t*batch_size+b+1]).
 * weights: per key (weighted pooling), f32 or f16.  output: batch_size rows of
 * num_tables*count values of output_type, table t of sample b at
 * output[b][t][:], count = stored values per row.  Sum / Mean / WeightedSum /
 * WeightedMean, fp32 accumulation; an fp16 or fp32 output from any row format. */
NVE_C_API nve_status_t nve_amd_find_and_pool_multi(
    nve_key_type_t key_type, int64_t num_tables, const void* const* tables,
    const int64_t* table_rows, int64_t row_size_in_bytes, nve_data_type_t value_dtype,
    int64_t batch_size, int64_t num_keys,
    const void* keys, const void* offsets, const void* weights, nve_data_type_t weight_type,
    nve_pooling_type_t pooling_type, nve_data_type_t output_type, void* output, void* stream);

/* Key dedup (the reference's Deduper::dedup, cuda_ops/deduper.cuh:136-221),
 * device buffers of the key type, each sized num_keys: unique_out (ascending,
 * signed order), counts_out, inverse_out (original positions ordered by key,
 * stable: inverse_out[offsets_out[u] + j] is the j-th position of unique key
 * u) and offsets_out (exclusive scan of the counts).  *num_unique receives the
 * number of unique keys (the call synchronizes the stream).  workspace: device
 * memory of nve_amd_dedup_workspace_size(num_keys) bytes. */
NVE_C_API nve_status_t nve_amd_dedup_workspace_size(int64_t num_keys, uint64_t* bytes);
NVE_C_API nve_status_t nve_amd_dedup(nve_key_type_t key_type, int64_t num_keys, const void* keys,
                                     void* unique_out, void* counts_out, void* inverse_out,
                                     void* offsets_out, int64_t* num_unique, void* workspace,
                                     uint64_t workspace_bytes, void* stream);

/* Dedup-then-gather over a linear table in device memory: output row i =
 * table row keys[i].  The keys are deduplicated by hashing, each distinct row
 * is read from the table once into the output row of one of its positions,
 * and the other positions copy that row (UnpackDedup).  Keys outside
 * [0, num_rows) leave their output row unchanged.  Asynchronous; workspace as
 * for nve_amd_dedup. */
NVE_C_API nve_status_t nve_amd_dedup_gather(nve_key_type_t key_type, int64_t num_keys,
                                            const void* keys, const void* table, int64_t num_rows,
                                            int64_t row_size_in_bytes, void* output,
                                            int64_t output_stride, void* workspace,
                                            uint64_t workspace_bytes, void* stream);

/* nve_amd_dedup_gather without the workspace argument, for callers that cannot
 * allocate (code under HIP graph capture, tight serving loops, harnesses that
 * forbid hipMalloc); it has no counterpart in the reference.  It allocates
 * nothing: its scratch is a fixed 16 MiB device array, one per GPU, held
 * until the process ends.  num_keys must not exceed 262,144 (larger batches
 * fail with NVE_ERROR_INVALID_ARGUMENT).  Every call on one GPU uses that
 * GPU's array, so the library runs the calls on one GPU one after another, in
 * the order they are issued from any thread or stream: each call's stream
 * waits for the previous call's completion event (one event per GPU, made
 * with the array's address on the GPU's first call).  Under HIP graph capture
 * that ordering is not recorded: a replayed graph must not overlap other
 * calls on its GPU.  Same results as nve_amd_dedup_gather; asynchronous on
 * `stream`. */
NVE_C_API nve_status_t nve_amd_dedup_gather_noalloc(nve_key_type_t key_type, int64_t num_keys,
                                                    const void* keys, const void* table,
                                                    int64_t num_rows, int64_t row_size_in_bytes,
                                                    void* output, int64_t output_stride, void* stream);

/* Random-row read microbenchmark: reads row idx[i] (row_size_in_bytes each, a
 * multiple of 16) of a table for i < n and folds the bytes into sink (one
 * uint32 per 256-thread workgroup, ceil(n/128) words).  The table may be
 * device memory (the HBM random-row ceiling) or pinned host memory from
 * hipHostMalloc (the host link's random-row ceiling, which bounds the reads
 * of missed rows from a LinearUVM backing table). */
NVE_C_API nve_status_t nve_amd_read_ceiling(const void* table, int64_t row_size_in_bytes,
                                            const int64_t* idx, int64_t n, uint32_t* sink,
                                            void* stream);

/* Cache state transfer of a GPU table (checkpoint-style restore, tests):
 * tags = num_sets*8 keys of the table's key type, counters = num_sets*8
 * float, set_ts = num_sets int64; host or device pointers; any may be NULL. */
NVE_C_API nve_status_t nve_amd_gpu_table_num_sets(const nve_table_t table, int64_t* out);
NVE_C_API nve_status_t nve_amd_gpu_table_export_state(nve_table_t table, void* tags,
                                                      float* counters, int64_t* set_ts,
                                                      int64_t* global_ts);
NVE_C_API nve_status_t nve_amd_gpu_table_import_state(nve_table_t table, const void* tags,
                                                      const float* counters,
                                                      const int64_t* set_ts, int64_t global_ts);
/* Device address of the cache rows ((set*8 + way) * row_size_in_bytes). */
NVE_C_API nve_status_t nve_amd_gpu_table_data(nve_table_t table, void** out);

/* GpuTable::insert_from_uvm (include/gpu_table.hpp:160-167, gpu_table.cu:494-576):
 * insert keys whose rows are read from the table's backing (UVM) table at
 * uvm_table + key * row_size_in_bytes.  The reference's C ABI reaches it only
 * through a LinearUVM layer's auto-insert; this entry exposes it directly.
 * Keys may live in host or device memory; keys outside [0, uvm_num_rows) are
 * not inserted. */
NVE_C_API nve_status_t nve_amd_table_insert_from_uvm(nve_table_t table, nve_context_t ctx,
                                                     int64_t n, const void* keys);

/* LinearHostTable (include/linear_host_table.hpp:36-183): a dense table of
 * num_rows rows of config->max_value_size bytes at emb_table (host memory the
 * caller owns and keeps alive), row k at emb_table + k * max_value_size,
 * values of config->value_dtype (FLOAT32, FLOAT16 or a rowwise-quantized
 * type); config->key_size must match key_type.  At most max_threads tasks run
 * per operation (<= 0: no limit beyond the context's thread pool).  The
 * reference builds this table inside its pynve HostEmbedding binding
 * (python/pynve/bindings/binding_layers.hpp:742-756); its C ABI has no
 * constructor for it.  The handle works with nve_table_find / update /
 * update_accumulate (FLOAT32 rows) / insert / erase / clear (the last three
 * have no effect), the getters (device id -1), the lookup counter (keys
 * found) and nve_host_embedding_layer_create.  Nothing it does enters the HIP
 * runtime while its buffers are host memory. */
NVE_C_API nve_status_t nve_amd_linear_host_table_create(nve_table_t* out, nve_key_type_t key_type,
                                                        const nve_host_table_config_t* config,
                                                        void* emb_table, int64_t num_rows,
                                                        int64_t max_threads);

/* Training backprop: the sparse gradient of a lookup with respect to the table
 * (GradientCalculator::compute_gradients, cuda_ops/gradient_calculator.cuh:238-301,
 * which the reference's pynve GPU bindings call as concat_backprop /
 * pooling_backprop, python/pynve/bindings/binding_layers.hpp:131-250).
 * pooling_type NVE_POOL_CONCATENATE: grads_in holds one row per key
 * (num_keys rows); otherwise one row per bag (fixed_hotness, or
 * num_csr_offsets - 1 bags of non-decreasing csr_offsets of the key type).
 * grads_in / grads_out rows: embedding_width values of grad_type (FLOAT32 or
 * FLOAT16); weights (WEIGHTED_*): one per key of weight_type FLOAT32 / FLOAT16.
 * Sum weighs 1, WeightedSum w, Mean 1 / (keys in the bag), WeightedMean
 * w / (the bag's weights added in order).  Outputs: the unique keys ascending
 * (reserve num_keys entries of the key type), one gradient row per unique key
 * (reserve num_keys rows) and *num_unique_out.  Sums are fp32 in a fixed order
 * and rounded once, so the result is deterministic: the positions in dedup
 * order are cut into blocks of 32, each key's positions inside one block are
 * added in position order, and a key's J block sums are added in 8
 * consecutive sub-sequences of ceil(J / 8), then the 8 sub-sums in order.
 * Device buffers and workspace; synchronizes the stream. */
NVE_C_API nve_status_t nve_amd_backprop_workspace_size(int64_t num_keys, int64_t num_bags,
                                                       int64_t embedding_width, uint64_t* bytes);
NVE_C_API nve_status_t nve_amd_pooling_backprop(
    nve_key_type_t key_type, int64_t num_keys, const void* keys, nve_pooling_type_t pooling_type,
    nve_sparse_type_t sparse_type, const void* csr_offsets, int64_t num_csr_offsets,
    int64_t fixed_hotness, const void* weights, nve_data_type_t weight_type, const void* grads_in,
    nve_data_type_t grad_type, int64_t embedding_width, void* unique_keys_out, void* grads_out,
    int64_t* num_unique_out, void* workspace, uint64_t workspace_bytes, void* stream);

/* Paged key-value cache of an attention layer (serving; no counterpart in the
 * reference).  A page holds page_size slots of num_heads key / value heads:
 * k and v are [num_pages, num_heads, page_size, head_dim] of dtype (FLOAT32,
 * FLOAT16, BFLOAT16, E4M3 or X_MXFP4), 16-byte aligned.  E4M3 rows have one f32
 * scale each (value = e4m3(code) * scale) in k_scale and v_scale [num_pages,
 * num_heads, page_size].  X_MXFP4 rows are head_dim / 2 bytes of codes, and
 * k_scale and v_scale point to their head_dim / 32 e8m0 bytes each, [num_pages,
 * num_heads, page_size, head_dim / 32].  NULL for the other types.  weights (f32)
 * and index (int32) are [num_pages, num_heads, page_size]: the attention weight a
 * slot has received so far, and its token's place in its sequence; either may be
 * NULL where a call does not need it.  page_size is a power of two from 8 to
 * 1024, head_dim a multiple of 8 (X_MXFP4: of 32) from 8 to 256.
 * A sequence is a row of block_tables: its slot t lies in page
 * block_tables[s * table_stride + t / page_size], row t % page_size.  Page ids
 * outside [0, num_pages) are neither read nor written: their slots count as
 * absent.  A length below 0 counts as 0, one above max_pages * page_size (or
 * above a call's max_length) as that bound.  All pointers are device memory;
 * strides are in elements, and the last dimension is contiguous. */
typedef struct {
  void* k;
  void* v;
  float* k_scale;
  float* v_scale;
  float* weights;
  int32_t* index;
  int64_t num_pages;
  int32_t num_heads;
  int32_t page_size;
  int32_t head_dim;
  nve_data_type_t dtype;
} nve_amd_kv_pages_t;

/* New tokens enter the cache.  Token t's keys and values (num_heads heads of
 * `dtype`, the pages' type, or FLOAT16 / BFLOAT16 for scaled pages) are written to
 * slot slots[t] = page * page_size + row (a slot outside the cache is skipped;
 * no slot may appear twice), index[t] to the slot's index (with pages->index;
 * index NULL: positions[0][t], or 0 without positions), 0 to its weight (with
 * pages->weights).  E4M3 rows: scale = max(largest magnitude, 1e-30) / 448,
 * code = value / scale rounded to nearest even.  X_MXFP4 rows: the scale of 32
 * values is the least power of two (2^-126 at least) of which no magnitude is
 * over 7 times, code = value / scale rounded to nearest even (6 is the most); 32
 * values with an infinity or a NaN among them have the scale NaN.
 * rot_dim > 0: the first rot_dim values of every key head, and of every head of
 * q, are rotated first.  Pair i (of rot_dim / 2) is values i and i +
 * rot_dim / 2, or 2i and 2i + 1 if interleaved; it belongs to one of num_axes
 * axes, the first sections[0] pairs to axis 0, the next sections[1] to axis 1
 * and so on, and turns by row p = positions[axis * axis_stride + t] of cos_sin
 * [max_position, rot_dim] (f32: the cosines of the pairs, then their sines):
 *   (a, b) -> (a cos - b sin, b cos + a sin)
 * in f32, rounded once.  A position outside [0, max_position) leaves its pairs
 * as they are.  q (may be NULL): [num_tokens, num_q_heads, head_dim] of `dtype`,
 * rotated into q_out, which may be q itself. */
typedef struct {
  int64_t num_tokens;
  const int64_t* slots;
  nve_data_type_t dtype;
  const void* k;
  int64_t k_token_stride, k_head_stride;
  const void* v;
  int64_t v_token_stride, v_head_stride;
  const void* q;
  int64_t q_token_stride, q_head_stride;
  void* q_out;
  int64_t q_out_token_stride, q_out_head_stride;
  int32_t num_q_heads;
  const int32_t* index;
  const int32_t* positions;
  int64_t axis_stride;
  const float* cos_sin;
  int64_t max_position;
  int32_t rot_dim;
  int32_t interleaved;
  int32_t num_axes;
  int32_t sections[4];
} nve_amd_kv_append_t;
NVE_C_API nve_status_t nve_amd_kv_append(const nve_amd_kv_pages_t* pages,
                                         const nve_amd_kv_append_t* call, void* stream);

/* The same with norms of the query and key heads, before the rotation: a head
 * row x of head_dim values becomes (x[d] * r) * weight[d], both products f32,
 * with r = 1 / sqrt(mean of x[d]^2 + eps), the mean and r in 64 bits and r then
 * rounded to f32.  Weights: [head_dim] of the call's dtype; a NULL weight leaves
 * those heads without a norm.  eps is finite and not negative; with 0 a row of
 * zeros becomes NaN. */
typedef struct {
  const void* q_weight;
  const void* k_weight;
  double eps;
} nve_amd_kv_norm_t;
NVE_C_API nve_status_t nve_amd_kv_append_norm(const nve_amd_kv_pages_t* pages,
                                              const nve_amd_kv_append_t* call,
                                              const nve_amd_kv_norm_t* norm, void* stream);

/* Attention of one new token per sequence over its slots t < lengths[s]:
 *   x_t = scale * q . k_t,  p = softmax(x),  out = sum_t p_t v_t
 * q and out: [num_seqs, num_q_heads, head_dim] of `dtype` (the pages' type, or
 * FLOAT16 / BFLOAT16 for scaled pages); query head h reads key head
 * h / (num_q_heads / num_heads).  lse (may be NULL): [num_seqs, num_q_heads],
 * log sum_t exp(x_t).  Where no slot has a score above -infinity (a length of
 * zero, say) out is 0 and lse -infinity.  What lies in a page's rows at or past
 * the length is not used, whatever it is.  Scores, lse, sums and the weights that
 * are added are f32; the p_t that meet FLOAT16 values keep 22 bits and those below
 * 2^-38 of the largest count as 0, the p_t that meet E4M3 and X_MXFP4 values keep 17.  accumulate:
 * p_t, summed over the query heads of a key head, is added to pages->weights;
 * no page may then belong to two sequences of the call.  max_length: the
 * longest length that occurs, if the caller knows it (0: the table's extent);
 * it sizes the launch and the workspace.  workspace: device memory of
 * nve_amd_kv_attend_workspace_size bytes, 16-byte aligned. */
typedef struct {
  int64_t num_seqs;
  int32_t num_q_heads;
  nve_data_type_t dtype;
  const void* q;
  int64_t q_seq_stride, q_head_stride;
  void* out;
  int64_t out_seq_stride, out_head_stride;
  float* lse;
  const int32_t* block_tables;
  int64_t table_stride;
  int64_t max_pages;
  const int32_t* lengths;
  int64_t max_length;
  float scale;
  int32_t accumulate;
} nve_amd_kv_attend_t;
NVE_C_API nve_status_t nve_amd_kv_attend_workspace_size(const nve_amd_kv_pages_t* pages,
                                                        const nve_amd_kv_attend_t* call,
                                                        uint64_t* bytes);
NVE_C_API nve_status_t nve_amd_kv_attend(const nve_amd_kv_pages_t* pages,
                                         const nve_amd_kv_attend_t* call, void* workspace,
                                         uint64_t workspace_bytes, void* stream);

/* Eviction by accumulated attention weight.  Every sequence of more than
 * `budget` slots keeps `budget` of them, chosen for each key head by itself:
 * dropped are the first ones in the order (protected, weight, slot), where a
 * slot is protected if its index is below `sinks` or among the `recent` places
 * up to the head's newest index, a NaN weight is the greatest and slots of
 * absent pages come first.  The j-th dropped slot below `budget` then takes the
 * row (k, v, scales, weight, index) of the j-th kept slot at or past it;
 * nothing else is written, so a row whose gap lies in an absent page is lost
 * (absent pages belong behind a table's others).  new_lengths[s] = min(lengths[s], budget); the two
 * may not overlap.  No page may belong to two sequences of the call.
 * workspace: device memory of nve_amd_kv_evict_workspace_size bytes, 16-byte
 * aligned. */
typedef struct {
  int64_t num_seqs;
  const int32_t* block_tables;
  int64_t table_stride;
  int64_t max_pages;
  const int32_t* lengths;
  int32_t* new_lengths;
  int64_t budget;
  int64_t sinks;
  int64_t recent;
} nve_amd_kv_evict_t;
NVE_C_API nve_status_t nve_amd_kv_evict_workspace_size(const nve_amd_kv_pages_t* pages,
                                                       const nve_amd_kv_evict_t* call,
                                                       uint64_t* bytes);
NVE_C_API nve_status_t nve_amd_kv_evict(const nve_amd_kv_pages_t* pages,
                                        const nve_amd_kv_evict_t* call, void* workspace,
                                        uint64_t workspace_bytes, void* stream);

/* A token for every row of logits [num_rows, vocab_size] (FLOAT32, FLOAT16 or
 * BFLOAT16, rows row_stride elements apart), drawn with u[row] in [0, 1):
 *   w_i = exp((x_i - max x) / temperature)
 * kept are, in the order (x descending, index ascending), the first top_k (0 or
 * at least vocab_size: all), of these the ones whose preceding sum of w is below
 * top_p times the sum over them (1 or more: all; the first one always), and of
 * these the ones with w_i >= min_p.  The token is the first index i, in the
 * vocabulary's order, at which the sum of the kept w_j, j <= i, exceeds u times
 * their sum.  temperature 0: the first of the largest logits.  Exponentials and
 * sums are 64-bit; in the sum over a whole row of 16-bit logits a weight is within
 * 2^-31 of its value.  temperatures, top_ks, top_ps and min_ps (device, [num_rows])
 * hold a limit for each row; NULL: the one value beside it counts for all.  In
 * device memory a temperature that is not above 0 counts as 0, a top_k below 1
 * as 0, a top_p or min_p that is no number as none, one outside [0, 1] as the
 * nearer of 0 and 1.  Logits that are no number count as -infinity; a row of
 * nothing else gives -1.  Where a logit is +infinity the others have no weight.
 * workspace: device memory of nve_amd_sample_workspace_size bytes, 16-byte
 * aligned. */
typedef struct {
  int64_t num_rows;
  int64_t vocab_size;
  nve_data_type_t dtype;
  int32_t top_k;
  const void* logits;
  int64_t row_stride;
  const float* u;
  const float* temperatures;
  const int32_t* top_ks;
  const float* top_ps;
  const float* min_ps;
  float temperature;
  float top_p;
  float min_p;
  int64_t* tokens;
} nve_amd_sample_t;
NVE_C_API nve_status_t nve_amd_sample_workspace_size(const nve_amd_sample_t* call, uint64_t* bytes);
NVE_C_API nve_status_t nve_amd_sample(const nve_amd_sample_t* call, void* workspace,
                                      uint64_t workspace_bytes, void* stream);

/* Log level (include/logging.hpp:34-203): messages at or below the level are
 * written, errors to stderr and the rest to stdout.  Levels: 0 critical,
 * 10 error, 20 warning, 30 perf, 40 info, 100 verbose.  The initial level is
 * NVE_LOG_LEVEL's (CRITICAL, ERROR, WARNING, PERF, INFO or VERBOSE), else
 * warning.  Library calls are also marked as roctx ranges (rocprofv3
 * --marker-trace) unless NVE_ROCTX=0; the reference marks them with NVTX
 * (include/cuda_support.hpp:26-55). */
NVE_C_API nve_status_t nve_amd_set_log_level(int32_t level);
NVE_C_API nve_status_t nve_amd_get_log_level(int32_t* level);
/* Writes one message through the library's logger if `level` is enabled
 * (the bindings log hit rates at the perf level this way, as the reference's
 * binding does with NVE_LOG_PERF_, binding_layers.hpp:370-387). */
NVE_C_API nve_status_t nve_amd_log_message(int32_t level, const char* message);

#ifdef __cplusplus
}
#endif

#endif /* NVE_AMD_EXT_H */
