/*
 * iam.h - C ABI of the MI355X (gfx950) input-adaptive sparse decode library.
 *
 * This is the boundary that replaces the reference's OpenCL runtime
 * (gpu.hpp) and the OpenCL bodies of its operator wrappers.  Every entry
 * point is extern "C", takes plain pointers and sizes, and returns an int
 * status: 0 on success, a negative IAM_E* code on failure, with a message in
 * iam_last_error() (thread-local).  The C++ headers under
 * input-adaptive-matrix-inference-optimization_amd/cpp/ keep the reference's
 * class and method surface on top of these calls and turn non-zero statuses
 * into std::runtime_error, as the reference does.
 *
 * Execution model: one HIP stream per context, in order.  Every call is
 * asynchronous except iam_write / iam_read (blocking, like the reference's
 * writeBuffer/readBuffer) and iam_sync (the reference's eval()).  A context
 * is not thread-safe.  Device pointers come from iam_alloc; "_dev" arguments
 * point to device memory.
 *
 * Citations are to files of the reference repository.
 */
#ifndef IAM_H
#define IAM_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* status codes */
#define IAM_OK 0
#define IAM_E_INVALID (-1)    /* bad argument or shape */
#define IAM_E_HIP (-2)        /* HIP runtime error */
#define IAM_E_NOMEM (-3)      /* allocation failed or over the byte budget */
#define IAM_E_STATE (-4)      /* call out of order (e.g. mul before calc_dispatch) */
#define IAM_E_IO (-5)         /* file missing, truncated or malformed */

#define IAM_PROBES_COUNT 4096 /* bucketMul.cl:18, bucket_mul.hpp:101 */

typedef struct iam_ctx iam_ctx;

/* ------------------------------------------------------------------ runtime */

/* Gpu::Gpu() (gpu.hpp:109-159): one device, one in-order queue. */
int iam_ctx_create(int device, iam_ctx** out);
/* Gpu::~Gpu() (gpu.hpp:161-188); frees everything allocated through the context. */
int iam_ctx_destroy(iam_ctx* ctx);
/* Gpu::eval() (gpu.hpp:399-447): wait for the queue, fold kernel timings. */
int iam_sync(iam_ctx* ctx);
/* Gpu::checkError message (gpu.hpp:581-587), thread-local. */
const char* iam_last_error(void);
/* device name / CU count / global memory (gpu.hpp:123-135, :28-31) */
int iam_device_info(iam_ctx* ctx, char* name, size_t name_len, int* compute_units,
                    size_t* global_mem_bytes);
/* MemoryTracker (gpu.hpp:21-60): byte budget = device memory - margin.
 * allocated counts the prefill buffers the models keep (iam_model_generate);
 * an allocation that finds no room frees those first. */
int iam_mem_status(iam_ctx* ctx, size_t* allocated, size_t* usable);

/* Gpu::createBuffer (gpu.hpp:236-262) */
int iam_alloc(iam_ctx* ctx, size_t bytes, void** out_dev);
/* Gpu::releaseBuffer (gpu.hpp:264-269) */
int iam_free(iam_ctx* ctx, void* dev);
/* BufferWrapper::zero (bucket_mul.hpp:34-38): a fill kernel, safe under graph capture. */
int iam_zero(iam_ctx* ctx, void* dev, size_t offset_bytes, size_t bytes);
/* Gpu::writeBuffer (gpu.hpp:464-469), blocking. */
int iam_write(iam_ctx* ctx, void* dst_dev, size_t dst_offset, const void* src_host, size_t bytes);
/* Gpu::readBuffer (gpu.hpp:457-462), blocking (waits for prior work). */
int iam_read(iam_ctx* ctx, void* dst_host, const void* src_dev, size_t src_offset, size_t bytes);
/* Gpu::copyBuffer (gpu.hpp:449-455), asynchronous device-to-device. */
int iam_copy(iam_ctx* ctx, void* dst_dev, size_t dst_offset, const void* src_dev,
             size_t src_offset, size_t bytes);

/* Measured streaming-read bandwidth of the device (GB/s): reps timed passes
 * of 16-byte loads over a zero-filled buffer of `bytes` (allocated and freed
 * here; 2 GiB keeps it out of the 256 MB Infinity Cache).  Blocking.  No
 * counterpart in the reference: the measured peak the walk's roofline is
 * also reported against. */
int iam_read_bandwidth(iam_ctx* ctx, size_t bytes, int reps, double* gb_per_s);

/* Per-kernel profiling (gpu.hpp:104-106, :275-290, :411-432): when enabled each
 * launch is bracketed by HIP events and iam_sync folds the durations. */
int iam_profiling(iam_ctx* ctx, int enable);
/* Gpu::printKernelStats (gpu.hpp:190-234) into a text buffer. */
int iam_kernel_stats(iam_ctx* ctx, char* buf, size_t len);
int iam_kernel_stats_reset(iam_ctx* ctx);
/* total time (ms) and launch count of one kernel name since the last reset.
 * The model's walk launches are labelled by matrix group ("bucket_walk.qkv",
 * ".o", ".ffn13", ".ffn2", ".lm"); a name without a dot also sums its
 * labelled launches ("bucket_walk" = every walk); "*" sums every kernel. */
int iam_kernel_stat(iam_ctx* ctx, const char* name, double* total_ms, int* calls);

/* --------------------------------------------------------------- bucketMul */

/* One weight matrix in the reference's bucket layout
 * (preprocess_layer_fixed_gpu.py:110-242, binary_loader.hpp:30-37):
 *   buckets  fp16 [n_experts * expert_rows][bucket_cols], packed value|position
 *   stats    fp16, stats_stride values per row; selection reads
 *            stats[row * stats_stride + stats_channel]
 *            (reference files: stride 4, channel 3, bucketMul.cl:372)
 *   probes   fp16, at least (expert_no + 1) * 4096 values (bucketMul.cl:103-109)
 *   expert_rows = 16 * in_dim, bucket_cols = out_dim / 16. */
typedef struct {
    const uint16_t* buckets;
    const uint16_t* stats;
    const uint16_t* probes;
    int expert_rows;
    int bucket_cols;
    int stats_stride;
    int stats_channel;
} iam_bucket_matrix;

/* BucketMul::calcDispatch (bucket_mul.hpp:147-191): cutoff search
 * (findCutoffBinarySearch, bucketMul.cl:68-214) and row selection
 * (prepareDispatch, bucketMul.cl:351-386) for x against stats/probes in the
 * reference's 4-channel stats layout.  The dispatch is kept in the context,
 * like the BucketMul singleton's scratch (bucket_mul.hpp:125-144).
 * expert_size is the row count R of one expert; rows with r/16 >= in_size
 * are skipped, as in the reference.  x must hold at least max(4096, in_size)
 * floats, because the cutoff always reads x[0:4096] (bucketMul.cl:102-110). */
int iam_bucketmul_calc_dispatch(iam_ctx* ctx, const float* x_dev, const uint16_t* stats_dev,
                                const uint16_t* probes_dev, int expert_no, int in_size,
                                int bucket_cols, int expert_size, float effort);
/* BucketMul::mul (bucket_mul.hpp:193-252): walk the rows selected by the last
 * calc_dispatch and write y[16 * bucket_cols] (overwritten). */
int iam_bucketmul_mul(iam_ctx* ctx, const uint16_t* buckets_dev, int bucket_cols, float* y_dev);
/* BucketMul::fullMul (bucket_mul.hpp:254-267) */
int iam_bucketmul_full(iam_ctx* ctx, const float* x_dev, const uint16_t* stats_dev,
                       const uint16_t* probes_dev, const uint16_t* buckets_dev, int expert_no,
                       int in_size, int bucket_cols, int expert_size, float effort, float* y_dev);
/* Up to 3 independent matrices in one launch, like iam_bucketmul_full every
 * walk workgroup running the cutoff search of its matrix itself (the q/k/v and
 * gate/up calls of attention.hpp:160-170 and feedforward.hpp:60-68 share an
 * input).  xs[i] may repeat. */
int iam_bucketmul_multi(iam_ctx* ctx, int n, const iam_bucket_matrix* mats,
                        const float* const* xs_dev, const int* in_sizes, float* const* ys_dev,
                        int expert_no, float effort);
/* One matrix group (1..3 matrices sharing one input) in one launch, as the
 * model's decode step runs it: every walk workgroup computes the input
 * itself -- x_dev as given, or, when h_dev is not null, x = RMSNorm(h) * gain
 * (rmsNorm32fast + mul16x32, aux.cl:156-196, :434-440; written to x_dev) --
 * then the cutoff (the same bisection as calc_dispatch, in every workgroup),
 * selects and walks its input slice into fp64 (or fp32) accumulators; the
 * last workgroup to finish a column tile stores that tile of ys_dev[i].
 * Results equal calc_dispatch + mul.  A norm input of other than
 * 4096 values is normalized by a separate RMSNorm launch first.  No
 * counterpart in the reference, which runs the cutoff as a launch of its
 * own (bucket_mul.hpp:147-176). */
int iam_bucketmul_fused(iam_ctx* ctx, int n, const iam_bucket_matrix* mats, float* x_dev, int in_size,
                        float* const* ys_dev, int expert_no, float effort, const float* h_dev,
                        const uint16_t* gain_dev, float eps);
/* iam_bucketmul_fused without any device allocation at call time.  No
 * counterpart in the reference: it is for callers that cannot allocate
 * (code under HIP graph capture, tight serving loops, harnesses that forbid
 * hipMalloc).  The walk's scratch lives in one fixed device array per GPU
 * (about 1 MiB, held from the first call on that GPU until the process
 * ends): at most IAM_NOALLOC_MAX_OUTPUTS outputs (16 * bucket_cols summed
 * over the matrices), 256 column tiles and 1024 input slices per matrix;
 * larger groups fail with IAM_E_INVALID.  A norm input (h_dev, gain_dev)
 * must be 4096 long.  Results equal iam_bucketmul_fused's.  Every call on a
 * GPU shares that array: calls that overlap on one GPU (other streams,
 * contexts or threads) race.  The call is not recorded in the dispatch
 * slots (dispatch_info / walk_count do not see it) and launches without
 * profiling events. */
#define IAM_NOALLOC_MAX_OUTPUTS 131072
int iam_bucketmul_fused_noalloc(iam_ctx* ctx, int n, const iam_bucket_matrix* mats, float* x_dev,
                                int in_size, float* const* ys_dev, int expert_no, float effort,
                                const float* h_dev, const uint16_t* gain_dev, float eps);
/* Parity outputs of the last calc_dispatch / multi / fused call for matrix slot
 * `slot`: the cutoff (fp32, as written by findCutoffBinarySearch) and the
 * selected-row count S.  The selection is re-run by a separate list kernel
 * that recomputes the cutoff on its own; the call fails with IAM_E_STATE if
 * the two cutoffs differ.  Blocking. */
int iam_bucketmul_dispatch_info(iam_ctx* ctx, int slot, float* cutoff, uint32_t* count);
/* The selected rows (expert-local row ids, ascending) of slot `slot`; writes
 * min(S, cap) ids into rows_host.  Blocking. */
int iam_bucketmul_dispatch_rows(iam_ctx* ctx, int slot, uint32_t* rows_host, size_t cap,
                                uint32_t* count);
/* Rows the last walk (mul / multi / full) of slot `slot` selected, counted
 * inside the walk kernel.  Blocking.  No counterpart in the reference. */
int iam_bucketmul_walk_count(iam_ctx* ctx, int slot, uint32_t* count);
/* effort -> quantile exactly as bucket_mul.hpp:164 */
int iam_effort_quantile(float effort);
/* Device-side counters of the walk: the algorithmic weight bytes streamed
 * (2 * S * bucket_cols summed over every matrix walked), the selected rows
 * S and the matrices walked, since the last reset.  They are updated inside
 * the walk kernel, so graph replays count too.  Blocking. */
int iam_walk_counters(iam_ctx* ctx, uint64_t* weight_bytes, uint64_t* rows, uint64_t* matrices,
                      int reset);
/* The model's walk launches by matrix group: the counters above split by the
 * group that streamed them (IAM_WALK_GROUP_NONE: standalone calls).  Reset
 * with iam_walk_counters.  Blocking.  No counterpart in the reference. */
#define IAM_WALK_GROUP_NONE 0
#define IAM_WALK_GROUP_QKV 1
#define IAM_WALK_GROUP_O 2
#define IAM_WALK_GROUP_FFN13 3
#define IAM_WALK_GROUP_FFN2 4
#define IAM_WALK_GROUP_LM 5
int iam_walk_group_counters(iam_ctx* ctx, int group, uint64_t* weight_bytes, uint64_t* rows,
                            uint64_t* matrices);
/* Of the group's walks since the last reset: the matrices whose cutoff
 * search started from a hint (tries; see iam_set_search_hints) and those
 * whose hinted window held the cutoff's ranks (hits; the others ran the
 * full search).  Counted with the counters above (iam_set_walk_counting).
 * Blocking.  No counterpart in the reference. */
int iam_walk_group_hints(iam_ctx* ctx, int group, uint64_t* tries, uint64_t* hits);
/* Counting of the walk's selected rows (default on): the first column tile
 * of each input slice adds its row count to the counters above (three
 * 64-bit atomics per slice).  Off, the counters are not updated.  The
 * per-slice counts behind iam_bucketmul_walk_count are stored either way.
 * Changing it re-captures the model's decode graph.  Not during capture.
 * No counterpart in the reference. */
int iam_set_walk_counting(iam_ctx* ctx, int on);
/* Hints for the walk's cutoff search (default off for the calls of this
 * context; a model's decode steps always use them, one per matrix of each
 * layer).  On, each iam_bucketmul_fused call starts the search of matrix
 * slot i from the cutoff that slot found in the previous fused call: one
 * pass over the importances counts those above the window [7/8, 8/7] of the
 * hint and bins those inside it, which locates the cutoff's neighbourhood
 * (ranks t-2 .. t+2) without the coarse histogram when the input changes
 * little between calls, as from one decode step to the next; where the
 * window misses those ranks the full search runs.  The cutoff, the selected
 * rows and the outputs are the same either way.  iam_set_search_hint sets
 * slot i's hint; any value is accepted (0, a negative, a non-finite one or
 * one outside [1e-30, 1e30] means no hint).  Not during capture.  No
 * counterpart in the reference. */
int iam_set_search_hints(iam_ctx* ctx, int on);
int iam_set_search_hint(iam_ctx* ctx, int slot, float value);
/* Block-structured selection, the thesis's future work (THESIS p.42-43):
 * with block_inputs B > 1, the inputs are taken in blocks of B consecutive
 * ones, and rank k of every input of a block is selected when rank k of any
 * of them passes the cutoff (the block's largest rank-k importance >= the
 * cutoff); the cutoff itself is the reference's.  It applies to calls whose
 * effort is below below_effort (the hybrid of fine selection at moderate
 * and blocks at aggressive sparsity); B = 1 (the default) is the
 * reference's per-row selection.  B is 1, 2, 4, 8 or 16.  Changing it
 * re-captures a model's decode graph.  Not during capture.  No counterpart
 * in the reference. */
int iam_set_selection_block(iam_ctx* ctx, int block_inputs, float below_effort);
int iam_get_selection_block(iam_ctx* ctx, int* block_inputs, float* below_effort);
/* Accumulation of the bucket walk (and of attention) for this context:
 * IAM_ACC_FP64 (default) adds the exact fp64 products in fp64 and rounds each
 * output once: every output is within an fp64 rounding of the correctly
 * rounded sum, whatever the order of the additions.  IAM_ACC_FP32 forms the
 * products in fp32 as the reference's bucketMul does (bucketMul.cl:430-445)
 * and adds them in fp64; attention runs in fp32.  No counterpart in the
 * reference (its fp32 atomics are order dependent). */
#define IAM_ACC_FP32 0
#define IAM_ACC_FP64 1
int iam_set_accumulation(iam_ctx* ctx, int mode);
int iam_get_accumulation(iam_ctx* ctx, int* mode);
/* Derive a compact copy stats3[r] = stats[r*4 + 3] (device), so the
 * selection reads 2 bytes per row instead of 8.  The file layout is unchanged. */
int iam_stats_compact(iam_ctx* ctx, const uint16_t* stats_dev, size_t rows, int stride,
                      int channel, uint16_t* out_dev);

/* ------------------------------------------------------------ layer ops */

/* rmsNorm32fast (aux.cl:156-196) then the fp16 gain mul16x32 (aux.cl:434-440) /
 * mulVec32by16 (aux.cl:301-306).  n must be a multiple of 1024, at most
 * 16384; vectors 16-byte aligned, the gain 8-byte aligned. */
int iam_rmsnorm_gain(iam_ctx* ctx, const float* in_dev, const uint16_t* gain_dev, int n,
                     float eps, float* out_dev);
/* add32 (bucketMul.cl:517-520) into h, then rmsnorm_gain of the sum
 * (transformer_layer.hpp:108-112 fused).  h_dev is updated in place. */
int iam_add_rmsnorm_gain(iam_ctx* ctx, float* h_dev, const float* delta_dev,
                         const uint16_t* gain_dev, int n, float eps, float* out_dev);
/* add32 (bucketMul.cl:517-520): out = a + b */
int iam_add(iam_ctx* ctx, const float* a_dev, const float* b_dev, int n, float* out_dev);
/* silu32 (matrix.cl:27-32): out = up * gate / (1 + exp(-gate)) */
int iam_silu_mul(iam_ctx* ctx, const float* gate_dev, const float* up_dev, int n,
                 float* out_dev);
/* precompute_rope_cache (attention.hpp:207-235): host table
 * [max_pos][head_dim/2][2] of (cos, sin) in float. */
int iam_rope_table(double theta, int head_dim, int max_pos, float* table_host);
/* rope_mx (aux.cl:227-248) on n_heads heads; table row = *pos_dev. */
int iam_rope(iam_ctx* ctx, const float* in_dev, const float* table_dev, const int* pos_dev,
             int n_heads, int head_dim, float* out_dev);
/* RoPE of q (n_heads) and k (n_kv heads), then the KV append
 * (attention.hpp:172-189 and :281-309) into fp16 caches laid out
 * [max_ctx][n_kv][head_dim] at position *pos_dev (ignored unless
 * 0 <= *pos_dev < max_ctx). */
int iam_rope_kv_append(iam_ctx* ctx, const float* q_dev, const float* k_dev, const float* v_dev,
                       const float* table_dev, const int* pos_dev, int n_heads, int n_kv,
                       int head_dim, int max_ctx, float* q_out_dev, uint16_t* kcache_dev,
                       uint16_t* vcache_dev);
/* Decode attention over positions 0..*pos_dev of an fp16 GQA cache
 * (dotSetScore2 aux.cl:497-540, sum_of_exps32_mx :204-210, softmax_add32_mx
 * :219-225, sumScores32 :370-384; driver attention.hpp:311-404), split over
 * the context.  Query head h reads KV head h*n_kv/n_heads (repeat4x32). */
int iam_attention_decode(iam_ctx* ctx, const float* q_dev, const uint16_t* kcache_dev,
                         const uint16_t* vcache_dev, const int* pos_dev, int n_heads, int n_kv,
                         int head_dim, int max_ctx, float* out_dev);
/* The reference's KV cache layout and fp32 attention, the parity mode of
 * iam_rope_kv_append / iam_attention_decode: the caches hold K (after RoPE)
 * and V repeated to every query head, fp32 [max_ctx][n_heads][head_dim] per
 * layer (model.hpp:97-98).  RoPE of q and k, then K and V of KV head
 * h*n_kv/n_heads stored for every query head h at *pos_dev (repeat4x32
 * aux.cl:266-275, rope_mx :227-248, the copies of attention.hpp:281-309). */
int iam_rope_kv_append_f32(iam_ctx* ctx, const float* q_dev, const float* k_dev, const float* v_dev,
                           const float* table_dev, const int* pos_dev, int n_heads, int n_kv, int head_dim,
                           int max_ctx, float* q_out_dev, float* kcache_dev, float* vcache_dev);
/* Attention over positions 0..*pos_dev of those caches in the reference's
 * fp32 arithmetic (dotSetScore2 aux.cl:497-540 with its work-group tree,
 * sum_of_exps32_mx / softmax_add32_mx :204-225 with no maximum subtracted,
 * sumScores32 :370-384; driver attention.hpp:311-404): one IEEE operation
 * at a time, the sums of exp and of p*v in splits of 64 positions taken in
 * order (the reference's float atomics have no fixed order).  A score above
 * log(FLT_MAX) ~ 88.72 makes that head's outputs NaN, as in the reference. */
int iam_attention_decode_f32(iam_ctx* ctx, const float* q_dev, const float* kcache_dev,
                             const float* vcache_dev, const int* pos_dev, int n_heads, int head_dim,
                             int max_ctx, float* out_dev);
/* matmul16x32 (aux.cl:454-490), the reference's dense LM head (model.hpp:
 * 207-227, 256 work-items per row): out[r] = the fp16 row r of W [rows][cols]
 * times x, each row's products summed per work-item over the columns
 * l, l+256, ... in order and then by the 256-way work-group tree, in fp32
 * without contraction.  cols <= 16384. */
int iam_matmul_f16_dense(iam_ctx* ctx, const uint16_t* w_dev, const float* x_dev, int rows, int cols,
                         float* out_dev);
/* fetchRow16to32 (aux.cl:442-452): out = (float) table[*token_dev][:]; a
 * token outside [0, vocab) yields zeros. */
int iam_embed_gather(iam_ctx* ctx, const uint16_t* table_dev, int cols, int vocab,
                     const int* token_dev, float* out_dev);
/* greedy pick (test_generation.cpp:235, :276): first index of the maximum */
int iam_argmax(iam_ctx* ctx, const float* v_dev, int n, int* out_dev);

/* ---------------------------------------------------- long-context operators
 * No counterpart in the reference, which rotates one token with unscaled
 * angles, keeps its cache in fp32 and answers with the first maximum. */

/* number types of activations */
#define IAM_F32 0
#define IAM_F16 1
#define IAM_BF16 2

/* which values of a head form a pair: (i, i + rot_dim/2), or (2i, 2i + 1) */
#define IAM_ROPE_HALF 0
#define IAM_ROPE_INTERLEAVED 1

/* Scaling of the rotary angles for contexts past the trained one.  With
 * f_i = theta^(-2i/rot_dim), pair i turns by pos * f_i' and is multiplied by
 * `magnitude` (0: 1, or RAMP's own):
 *   NONE    f_i' = f_i
 *   LINEAR  f_i / factor (position interpolation)
 *   BASE    f_i of the base theta * factor^(rot_dim / (rot_dim - 2))
 *   BANDS   with t_i = original_ctx * f_i / 2 pi turns over the trained
 *           context: f_i where t_i >= high, f_i / factor where t_i <= low, in
 *           between the mix of both that is linear in t_i
 *   RAMP    f_i for pairs below the one that turns `high` times over the
 *           trained context, f_i / factor past the one that turns `low`
 *           times, linear in i between them (YaRN; their places
 *           rot_dim * ln(original_ctx / (2 pi turns)) / (2 ln theta) rounded
 *           down and up, kept in [0, rot_dim - 1]); magnitude 0.1 ln(factor) + 1
 * factor is at least 1; original_ctx, low and high (0 < low < high) are read
 * by BANDS and RAMP only. */
#define IAM_ROPE_SCALE_NONE 0
#define IAM_ROPE_SCALE_LINEAR 1
#define IAM_ROPE_SCALE_BASE 2
#define IAM_ROPE_SCALE_BANDS 3
#define IAM_ROPE_SCALE_RAMP 4
typedef struct {
    int kind;
    double factor;
    double original_ctx;
    double low;
    double high;
    double magnitude;
} iam_rope_scaling;

/* The table of iam_rope_tokens, fp32 [max_pos][rot_dim/2][2] of (cos, sin) on
 * the device: angles, cosines and sines in fp64, each value rounded once
 * (iam_rope_table rounds the angle to fp32 first, as the reference does,
 * up to 0.004 radians off at position 100000; its tables have the same form
 * and serve iam_rope_tokens too).  rot_dim is even, 2 .. 1024; scaling may be
 * null (NONE).  table_dev is 8-byte aligned.  Blocking. */
int iam_rope_scaled_table(iam_ctx* ctx, double theta, int rot_dim, int max_pos,
                          const iam_rope_scaling* scaling, float* table_dev);
/* Rotary positions of n_tokens rows of n_heads heads: the first rot_dim of a
 * head's head_dim values are rotated in pairs (layout) by the table's row
 * pos_dev[token], the others pass through.  Arithmetic in fp32 (iam_rope's
 * operations), one rounding to the type.  Rows are x_stride / out_stride
 * values apart (0: n_heads * head_dim), each row's heads contiguous; q and k
 * that lie side by side are one call over their heads together.  out_dev may
 * be x_dev with the same stride; else the two may not overlap.  A token whose
 * position lies outside [0, max_pos) leaves its out row as it was. */
int iam_rope_tokens(iam_ctx* ctx, const void* x_dev, int type, int n_tokens, int n_heads, int head_dim,
                    int rot_dim, int layout, size_t x_stride, const float* table_dev, int max_pos,
                    const int* pos_dev, void* out_dev, size_t out_stride);

/* A KV cache in 8 bits for n_seq sequences of up to max_ctx tokens.  The
 * tokens of a sequence are taken in blocks of IAM_KV8_BLOCK.  A full block
 * holds, for each KV head, 8-bit numbers and one fp32 scale for K and one for
 * V: scale = largest magnitude * fp32(1/127) and round(x / scale) for INT8,
 * largest magnitude * fp32(1/448) and the nearest e4m3 number (3 bits behind
 * the leading one, exponents down to 2^-6, then steps of 2^-9) for E4M3.  The
 * scale is rounded to fp32, the numbers to nearest even of the exact
 * quotient; a number stands for number * scale.  The block
 * that is not full yet is held in fp16, so a token's place in the cache does
 * not depend on how many came with it.  K and V are rounded to fp16 first, as
 * in the fp16 cache.  A block that holds an infinity or a NaN in a head has
 * the scale NaN there once it is full.
 *
 * Device memory, the caller's (iam_kv8_size says how much; every part 16-byte
 * aligned).  b counts blocks (ceil(max_ctx / 64) of them), t tokens in a block,
 * d values in a head:
 *   k, v              bytes [n_seq][b][n_kv][64 * head_dim], INT8 as number + 128
 *   k_scale, v_scale  fp32 [n_seq][b][n_kv]; negative: not full (iam_kv8_reset)
 *   k_open, v_open    fp16 [n_seq][n_kv][64 * head_dim], the open block
 * A block's 64 * head_dim values are in the order in which the matrix
 * instructions of the attention take them (iam_kv8_read gives plain rows):
 *   K: ((t/16 * head_dim/64 + d/64) * 64 + d%64/16 * 16 + t%16) * 16 + d%16
 *   V: (d/16 * 64 + t/4%4 * 16 + d%16) * 16 + t/32 * 8 + t/16%2 * 4 + t%4
 * head_dim is 64, 128 or 256. */
#define IAM_KV8_BLOCK 64
#define IAM_KV8_INT8 0
#define IAM_KV8_E4M3 1
typedef struct {
    uint8_t* k;
    uint8_t* v;
    float* k_scale;
    float* v_scale;
    uint16_t* k_open;
    uint16_t* v_open;
    int n_seq;
    int max_ctx;
    int n_kv;
    int head_dim;
    int format;
} iam_kv8_cache;

/* Bytes of each part: k (and v), k_scale (and v_scale), k_open (and v_open). */
int iam_kv8_size(int n_seq, int max_ctx, int n_kv, int head_dim, size_t* numbers, size_t* scales,
                 size_t* open);
/* Marks every block as not full.  Once, before the first append; a slot whose
 * sequence is over is used again by appending from position 0. */
int iam_kv8_reset(iam_ctx* ctx, const iam_kv8_cache* cache);
/* Writes n_tokens tokens of each sequence, k and v [n_seq][n_tokens] rows of
 * n_kv * head_dim values (of the type), kv_stride values apart (0: n_kv *
 * head_dim), at positions pos_dev[s] and on.  count_dev, if not null, says
 * how many of sequence s's tokens are there (the rest of a padded batch is
 * not read).  Tokens at or past max_ctx are dropped; a negative position
 * skips its sequence.  A sequence is appended to in order; going back (as
 * after rejected draft tokens) is allowed: where the position lies inside a
 * full block, the block's earlier tokens become open again as the values
 * that it stands for, rounded to fp16.  A call's blocks times n_kv stay below
 * 2^23 (here and in iam_kv8_read). */
int iam_kv8_append(iam_ctx* ctx, const iam_kv8_cache* cache, const void* k_dev, const void* v_dev, int type,
                   int n_tokens, size_t kv_stride, const int* pos_dev, const int* count_dev);
/* The values that positions pos_dev[s] .. pos_dev[s] + n_tokens - 1 stand for,
 * as fp32 rows [n_seq][n_tokens][n_kv][head_dim].  Rows of positions outside
 * [0, max_ctx) are left as they were; what a position holds that was never
 * written is undefined. */
int iam_kv8_read(iam_ctx* ctx, const iam_kv8_cache* cache, const int* pos_dev, int n_tokens, float* k_out_dev,
                 float* v_out_dev);
/* Attention of n_tokens consecutive tokens of each sequence over its cache
 * (which holds them already): q and out [n_seq][n_tokens] rows of n_heads *
 * head_dim values (of the type), q_stride / out_stride values apart (0: n_heads
 * * head_dim).  Token t of sequence s is at position p = pos_dev[s] + t (past
 * max_ctx: taken as max_ctx - 1) and sees positions 0 .. p, or the last
 * `window` of them if window > 0.  Query head h reads KV head h * n_kv /
 * n_heads.  The softmax takes scale * q.k (scale 0: 1 / sqrt(head_dim)).
 * Sums and the softmax in fp32 (an fp32 q enters the products to 22 bits, the
 * probabilities to 21), one rounding to the type.  Sequences with a negative
 * position give rows of zeros; rows of tokens from count_dev[s] on (if not
 * null) are left as they were.  An infinity or a NaN in the cache makes the
 * rows that see it NaN or infinite; in a full block, all rows that see any
 * token of the block's head.  In a row of q it makes that row NaN.  out may be
 * q with the same stride.  The rows of a sequence and KV head are taken in
 * groups of 16 to 128: below 2^23 of them a call. */
int iam_attention_kv8(iam_ctx* ctx, const iam_kv8_cache* cache, const void* q_dev, int type, int n_heads,
                      int n_tokens, size_t q_stride, const int* pos_dev, const int* count_dev, int window,
                      float scale, void* out_dev, size_t out_stride);

/* Log probabilities under softmax(row) of n_rows rows of `vocab` logits, `stride`
 * values apart (0: vocab): logprob_dev[r] of token targets_dev[r] (0 for a
 * target outside [0, vocab), the padding of a batch), entropy_dev[r] (may be
 * null) and, for top_k > 0, the top_k most likely tokens, likeliest first,
 * equal logits by the lower token: top_ids_dev and top_logprobs_dev
 * [n_rows][top_k] (top_k at most min(vocab, 64); either may be null).
 * The terms e^(x - max) and their products with x - max are fp32 (exponentials
 * good to 2^-22 of a rounded argument), added up in fp32 for at most 32 at a
 * time and in fp64 from there; one rounding to fp32.
 * A row of nothing but -inf gives -inf and the entropy 0; a row with a NaN or
 * +inf gives NaN for both and for the alternatives' log probabilities (their
 * tokens are ordered with NaN last). */
#define IAM_LOGPROBS_MAX_TOP 64
int iam_token_logprobs(iam_ctx* ctx, const void* logits_dev, int type, int n_rows, int vocab, size_t stride,
                       const int* targets_dev, float* logprob_dev, float* entropy_dev, int top_k,
                       int* top_ids_dev, float* top_logprobs_dev);

/* --------------------------------------- 4-bit weights and drafted tokens
 * No counterpart in the reference, whose weights are fp16 and whose steps
 * give one token each.
 * iam_q4_mul and iam_verify_drafts use scratch of the context's.  The first
 * call of a larger size frees it and allocates and clears more (and waits for
 * the device meanwhile); it is kept until the context is destroyed: at most
 * 2.5 GB, which products of many long fp32 rows reach. */

/* 8-bit number types of rows: signed whole numbers -127 .. 127, and e4m3 (as in
 * IAM_KV8_E4M3, up to 448).  A number stands for number * scale. */
#define IAM_I8 3
#define IAM_E4M3 4

/* A matrix of 4-bit weights, out_dim rows of in_dim.  Each row's inputs are
 * taken in groups of `group` (32, 64 or 128; the last one may be short); weight
 * (o, k) is scale * (n - zero) with n in 0 .. 15 and the scale (fp16) and the
 * zero point (a whole number 0 .. 15; 8 for a matrix without zero points, where
 * `zeros` is null) of row o's group.
 *
 * Device memory, the caller's (iam_q4_size says how much; every part 16-byte
 * aligned), in the order in which the matrix instructions take it.  Rows come
 * in strips of 16, inputs in tiles of 128 and chunks of four tiles:
 *   numbers  [strip][tile][lane 16 g + row][step j] 4-byte words: inputs 32 j +
 *            8 g + e of the tile, e = 0, 2, 4, 6, 1, 3, 5, 7 from the lowest
 *            four bits on, each n xor 8
 *   scales   fp16 [strip][chunk][row / 4][group of the chunk][row % 4]
 *   zeros    bytes [strip][chunk][row][group of the chunk]
 * What lies past the matrix in its last strip or chunk is 0. */
typedef struct {
    uint8_t* numbers;
    uint16_t* scales;
    uint8_t* zeros;
    int out_dim;
    int in_dim;
    int group;
} iam_q4_matrix;

/* Bytes of each part (zeros: if there are any).  out_dim is at most 2^24,
 * in_dim 2^20. */
int iam_q4_size(int out_dim, int in_dim, int group, size_t* numbers, size_t* scales, size_t* zeros);
/* Lays out a matrix once, from n as rows of ceil(in_dim / 2) bytes (input 2 i in
 * the low half of byte i), scales fp16 and zero points (bytes; null if
 * matrix->zeros is) as rows of ceil(in_dim / group).  The sources are not
 * needed afterwards. */
int iam_q4_pack(iam_ctx* ctx, const iam_q4_matrix* matrix, const uint8_t* n_dev, const uint16_t* scale_dev,
                const uint8_t* zero_dev);
/* Rounds the rows of a matrix in a float type (w_stride values apart, 0: in_dim)
 * to 4 bits.  Without zero points scale = fp16(largest magnitude / 7); with them,
 * low and high being the group's smallest and largest weight and 0, scale =
 * fp16((high - low) / 15) and zero = round(-low / scale), at most 15.  n =
 * round(w / scale) + zero, kept in 0 .. 15; quotients in fp32, halves to even.
 * A group whose scale is not finite has the scale NaN; one whose scale is 0
 * stands for zeros. */
int iam_q4_quantize(iam_ctx* ctx, const iam_q4_matrix* matrix, const void* w_dev, int type, size_t w_stride);
/* What rows first_row .. first_row + n_rows - 1 stand for, as fp32 rows of
 * in_dim (exact: 11 bits times 5). */
int iam_q4_read(iam_ctx* ctx, const iam_q4_matrix* matrix, int first_row, int n_rows, float* out_dev);
/* Products of n_rows rows of in_dim values with the matrix: y[r][o] = sum over k
 * of x[r][k] * weight (o, k).  Rows are x_stride / y_stride values apart (0: no
 * gaps).  x is of a float type (x_scale_dev null), or in 8 bits with fp32 scales
 * x_scale_dev [n_rows][1] (x_group 0) or [n_rows][ceil(in_dim / 128)] (x_group
 * 128).  y is of a float type, rounded once.  Products of whole numbers are
 * exact and sums fp32; a float row enters to 22 bits of the largest value of
 * its 128 inputs (or of 2^-102, if that is larger) or better, up to four fp32
 * rows to 30 (of 2^-96).  Matrices that share their input are one matrix of
 * their rows.  A row of x that holds an infinity or a NaN (or a scale that is
 * one) gives infinities and NaN in its own row of y only.  y may not overlap
 * the inputs. */
int iam_q4_mul(iam_ctx* ctx, const iam_q4_matrix* matrix, const void* x_dev, int x_type, size_t x_stride,
               const float* x_scale_dev, int x_group, int n_rows, void* y_dev, int y_type, size_t y_stride);

/* Root-mean-square norm of n_rows rows of dim values, with the residual's
 * addition before it.  h = x + residual (fp32, rounded to residual_type, which
 * is x's type or IAM_F32; h = x where residual_dev is null), kept in sum_dev if
 * that is not null; y = h / sqrt(mean of h^2 + eps) * gain (fp16, null: 1) in
 * fp64, rounded once to out_type: a float type, or IAM_I8 / IAM_E4M3 with
 * scale = fp32(largest magnitude / 127 or 448) of the row (group 0) or of each
 * 128 values (group 128) in scale_dev [n_rows][groups], and the number nearest
 * to y / scale (halves to even; 0 where the scale is 0).  Where y is infinite
 * or NaN the scale of its group is NaN and the group's numbers are 0.  Rows are
 * x_stride, residual_stride (sum_dev too) and out_stride values apart (0: dim).
 * sum_dev may be residual_dev; with a float out_type of x's type out_dev may be
 * x_dev with the same stride.  No other overlaps.  dim is at most 2^20. */
int iam_rmsnorm_rows(iam_ctx* ctx, const void* x_dev, int type, size_t x_stride, const void* residual_dev,
                     int residual_type, size_t residual_stride, void* sum_dev, int n_rows, int dim,
                     const uint16_t* gain_dev, float eps, void* out_dev, int out_type, size_t out_stride,
                     float* scale_dev, int group);
/* The values that 8-bit rows (stride values apart, 0: dim) stand for, as fp32
 * rows of dim: number * scale. */
int iam_rows8_read(iam_ctx* ctx, const void* x_dev, int type, size_t stride, const float* scale_dev, int group,
                   int n_rows, int dim, float* out_dev);

/* Judges drafted tokens.  Sequence s has drafted tokens tokens_dev[s][i], i <
 * n_draft (the first count_dev[s] of them where count_dev is not null), and
 * n_draft + 1 rows of the target's logits, target_stride values apart (0:
 * vocab), row i of the place that token i was drafted for.  With p_i the softmax
 * of row i / temperature and q_i that of the draft's logits for the same place
 * / draft_temperature ([n_seq][n_draft] rows draft_stride apart; draft_dev null:
 * q_i is 1 at token i), token i is accepted if uniform_dev[s][i] * q_i(token) <
 * p_i(token).  Of the a tokens before the first rejected one (all, if none is)
 * out_dev[s][0 .. a-1] are copies; out_dev[s][a] is drawn from max(p_a - q_a, 0)
 * if token a was rejected, else from p_a: the lowest token whose weights up to
 * it add up to more than uniform_dev[s][n_draft] times all of them (or the last
 * one of any weight).  The rest of out_dev [n_seq][n_draft + 1] is -1;
 * accepted_dev[s] = a.  All in fp64 from the logits on.
 * temperature 0: token i is accepted if it is the first largest logit of row i,
 * which also is the one that follows; no random numbers or drafts' logits are
 * read (both pointers may be null).
 * A drafted token outside the vocabulary is rejected (q_i is then taken as 0).
 * A row of the target with a NaN, a +inf or nothing but -inf has no
 * distribution: its token is rejected, and the one that follows is -1.  Where
 * the draft's row has none the token is rejected and the next is drawn from p,
 * as it is where p - q is nowhere positive (where its positive parts add up to
 * less than 1e-12: fp64's rounding).  temperatures are 2^-64 to 2^64 (or 0, as
 * above); n_draft 0 .. 64; random numbers lie in [0, 1). */
#define IAM_VERIFY_MAX_DRAFT 64
int iam_verify_drafts(iam_ctx* ctx, const void* target_dev, int target_type, size_t target_stride,
                      const void* draft_dev, int draft_type, size_t draft_stride, int n_seq, int n_draft, int vocab,
                      double temperature, double draft_temperature, const int* tokens_dev, const int* count_dev,
                      const float* uniform_dev, int* out_dev, int* accepted_dev);

/* -------------------------------------------------------- synthetic data */

/* Counter-based generator shared with the CPU oracle: element n of tensor
 * `tensor_id` = mean + sigma * (sum of 12 uniform uint32 - 6*2^32) / 2^32,
 * rounded to float (and then to fp16 for the f16 variant). */
int iam_gen_f16(iam_ctx* ctx, uint64_t seed, uint64_t tensor_id, size_t count, double mean,
                double sigma, uint16_t* out_dev);
int iam_gen_f32(iam_ctx* ctx, uint64_t seed, uint64_t tensor_id, size_t count, double mean,
                double sigma, float* out_dev);
/* GPU bucketizer, byte-identical to bucketize_fp16_packed
 * (preprocess_layer_fixed_gpu.py:110-242): W fp16 [out_dim][in_dim] ->
 * buckets [16*in][out/16], stats [16*in][4], probes [in]. */
int iam_bucketize(iam_ctx* ctx, const uint16_t* w_dev, int out_dim, int in_dim,
                  uint16_t* buckets_dev, uint16_t* stats_dev, uint16_t* probes_dev);

/* ----------------------------------------------------------------- model */

/* Mistral-shaped decoder (model.hpp:15-30, attention.hpp:21-27): dims,
 * heads, vocabulary, KV capacity and RoPE theta are parameters. */
typedef struct {
    int n_layers;
    int dim;
    int ffn_dim;
    int n_heads;
    int n_kv_heads;
    int head_dim;
    int vocab;
    int max_ctx;
    double rope_theta;
    float norm_eps;
} iam_model_config;

typedef struct iam_model iam_model;

/* MistralModel::MistralModel (model.hpp:84-127): allocates weights (bucket
 * layout, LM head included), fp16 KV caches [n_layers][max_ctx][n_kv][hd],
 * activations and the RoPE table. */
int iam_model_create(iam_ctx* ctx, const iam_model_config* cfg, iam_model** out);
int iam_model_destroy(iam_model* m);
/* Fill every weight from the synthetic generator: matrices N(0, 0.02^2)
 * bucketized on the GPU, gains 1 + N(0, 0.01^2), embedding N(0, 0.02^2). */
int iam_model_synthesize(iam_model* m, uint64_t seed);
/* MistralModel::forward (model.hpp:152-231): one token at position pos;
 * logits (vocab floats, device) are written; the KV cache at pos is filled. */
int iam_model_forward(iam_model* m, int token, int pos, float effort, float* logits_dev);
/* Like forward, but the token and position are read from device memory
 * (token_dev, pos_dev) and the next token (first argmax) is written back to
 * token_dev and pos is advanced, so a captured step replays without host
 * involvement.  hidden_override_dev, if non-NULL, replaces the embedding. */
int iam_model_step_device(iam_model* m, float effort, const float* hidden_override_dev);
/* Greedy decode (test_generation.cpp:197-276): feeds the prompt, then
 * generates n_new tokens with first-max argmax.  With use_graph the per-token
 * step is captured once as a HIP graph and replayed.  The prompt's tokens
 * before the last go through the model in batches where that is faster (fp64
 * accumulation, from 6 to 16 tokens on by shape and effort), in buffers the
 * model keeps until an allocation needs their room (about 2 MB a token, at
 * most 512 tokens', at 4096 wide with FFN 14336; fewer where there is less
 * room).  The KV cache, the picks in "history" and the walk counters' bytes,
 * rows and matrices are as by steps; batched tokens take no search hints, so
 * they count no tries or hits of them (iam_walk_group_hints).  The last
 * token's step leaves the activations and logits.
 * out_tokens receives n_new ids. */
int iam_model_generate(iam_model* m, const int* prompt, int n_prompt, int n_new, float effort,
                       int use_graph, int* out_tokens);
/* Continue greedy decoding from the current device state (the token picked
 * by the previous step at the current position) for n_steps steps, replaying
 * the captured step when use_graph is set.  Asynchronous. */
int iam_model_decode(iam_model* m, int n_steps, float effort, int use_graph);
/* Set the device position the next step computes (0 <= pos <= max_ctx).
 * decode and step_device refuse steps past the KV capacity, counted from
 * this position (or from forward / generate / reset_caches). */
int iam_model_set_position(iam_model* m, int pos);
/* MistralModel::reset_caches (model.hpp:233-237); also rewinds the position. */
int iam_model_reset_caches(iam_model* m);
/* The LM head as the reference's dense fp16 product (matmul16x32 over
 * lm_dense_dev [vocab][dim], a caller-owned device buffer that must outlive
 * its use; model.hpp:207-227) instead of the bucket-layout one; NULL restores
 * the bucket layout.  The step then runs the final norm, the dense product
 * and the first-max pick as launches of their own. */
int iam_model_set_lm_dense(iam_model* m, const uint16_t* lm_dense_dev);
/* Per-channel fp32 factors applied to the gathered embedding before the
 * first layer (NULL restores plain fetchRow16to32).  Used for the skewed-
 * channel decode workload, which scales 1% of hidden channels. */
int iam_model_set_embed_scale(iam_model* m, const float* scale_host);
/* Device pointer and size of a named model tensor, e.g. "layer3.w1.buckets",
 * "layer0.attn_gain", "embed", "final_gain", "lm_head.stats", "kcache",
 * "vcache", "rope", "logits", "token", "pos", "hidden" (the residual stream
 * after the last layer), "hidden_norm" (its final RMSNorm, the LM head input). */
int iam_model_tensor(iam_model* m, const char* name, void** dev, size_t* bytes);
/* The bucket-matrix descriptor of "layer{L}.{wq,wk,wv,wo,w1,w3,w2}" or "lm_head". */
int iam_model_matrix(iam_model* m, const char* name, iam_bucket_matrix* out);

#ifdef __cplusplus
}
#endif
#endif
