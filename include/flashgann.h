/*
 * flashgann.h -- C ABI of the B200 FlashGANN search engine (libflashgann.so).
 *
 * Drop-in boundary for the reference's search path (SophiaSun18/FlashGANN):
 * plain pointers and sizes, no C++ or torch types, every failure returned as
 * a status code instead of the reference's exit()/throw.  Each entry point
 * names the reference interface it replaces (file:line in that project).
 *
 * Threading: an fg_index may be used by one host thread at a time.
 * Devices: every call runs on the device the index was created on and
 * restores the caller's current device before returning.
 */
#ifndef FLASHGANN_H
#define FLASHGANN_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- status codes (the reference exits or throws instead) ---- */
#define FG_OK 0
#define FG_ERR_IO 1          /* file cannot be opened or is short      (qg.hpp:22-23 throws) */
#define FG_ERR_FORMAT 2      /* codebook/vecs content inconsistent     (data_io.hpp:41 asserts) */
#define FG_ERR_ARG 3         /* invalid argument                       */
#define FG_ERR_CUDA 4        /* CUDA runtime error                     (utils.cuh:42-50 exits) */
#define FG_ERR_OOM 5         /* not enough device memory               (gpu_search_adaptive.cu:61-63 throws) */
#define FG_ERR_UNSUPPORTED 6 /* outside this build's supported envelope */
#define FG_ERR_NO_DEVICE 7   /* no CUDA device / product kernels not loadable */

/* ---- metric (include/metric.hpp:9) ---- */
#define FG_METRIC_L2 0
#define FG_METRIC_IP 1

/* ---- device argument of fg_index_load / fg_index_create: the calling
 * thread's current CUDA device, which is where the reference's search runs
 * (gpu_search_adaptive.cu:30-34) ---- */
#define FG_DEVICE_CURRENT (-1)

typedef struct fg_index fg_index;

/* Codebook layout in float words, as QuantizationGraph's getters report it
 * (include/qg.hpp:49-60,66-73). */
typedef struct fg_layout {
    uint64_t num_nodes;
    uint64_t dim;
    uint64_t padded_dim;
    uint64_t code_offset;
    uint64_t factor_offset;
    uint64_t neighbor_offset;
    uint64_t row_offset;
    int32_t degree;
    uint32_t entry_point; /* resolved: the centroid fallback already applied */
    int32_t metric;
    int32_t device;
} fg_layout;

/* Per-query counters written by fg_search_device_ex (all optional). */
typedef struct fg_query_stats {
    uint32_t iterations;  /* loop iterations that merged candidates into the beam */
    uint32_t expansions;  /* parents expanded (neighbour lists read) */
    uint32_t evaluations; /* exact distances computed, entry point included */
    uint32_t estimates;   /* RaBitQ estimates computed */
} fg_query_stats;

const char* fg_status_string(int status);
/* Message of the last failure on the calling thread ("" if none). */
const char* fg_last_error(void);

/* Replaces QuantizationGraph::QuantizationGraph(n, dim, degree, path)
 * (include/qg.hpp:17-42) together with the index upload of
 * QuantizationGraph::gpu_search_adaptive (gpu_search_adaptive.cu:46-77):
 * reads the qg_codebook file, resolves entry point UINT32_MAX to the node
 * nearest the centroid (include/common.hpp:26-47), checks free memory and
 * keeps the codebook resident on `device` (FG_DEVICE_CURRENT: the current
 * device) until fg_index_free. */
int fg_index_load(const char* path, uint64_t num_nodes, uint64_t dim, int32_t degree, int32_t metric,
                  int32_t device, fg_index** out);

/* Same, from a codebook already in host memory: rows[num_nodes*row_offset]
 * and signs[padded_dim] in the qg_codebook layout. */
int fg_index_create(const float* rows, const float* signs, uint32_t entry_point, uint64_t num_nodes,
                    uint64_t dim, int32_t degree, int32_t metric, int32_t device, fg_index** out);

/* Same, from a codebook already in device memory on `device` (d_rows,
 * d_signs: device pointers, copied device to device; the caller keeps or
 * frees its buffers) -- for indexes built on the GPU, such as the shards of
 * a base too large for one host.  entry_point must be a node id (the
 * UINT32_MAX centroid fallback needs the rows on the host). */
int fg_index_create_device(const float* d_rows, const float* d_signs, uint32_t entry_point, uint64_t num_nodes,
                           uint64_t dim, int32_t degree, int32_t metric, int32_t device, fg_index** out);

/* Replaces ~QuantizationGraph (include/qg.hpp:44-47). NULL is accepted. */
int fg_index_free(fg_index* index);

/* Replaces the layout getters (include/qg.hpp:49-60). */
int fg_index_layout(const fg_index* index, fg_layout* out);

/* Replaces QuantizationGraph::set_metric (include/qg.hpp:54). */
int fg_index_set_metric(fg_index* index, int32_t metric);

/* What the kernel planner aims for (fg_index_set_plan_goal). */
#define FG_GOAL_LATENCY 0
#define FG_GOAL_THROUGHPUT 1

/* Sets what the planner optimises an index's searches for; no counterpart in
 * the reference (one kernel shape for every batch).  Every kernel returns the
 * same results, only their speed differs.
 * FG_GOAL_LATENCY (the default): the shortest time for one batch on an
 * otherwise idle GPU -- the CTA kernel for batches of up to 4 queries per SM,
 * the warp kernel's pair mode while the whole batch is resident at once, one
 * warp per query above.
 * FG_GOAL_THROUGHPUT: the most queries per second when the caller keeps
 * batches in flight on two or more streams (fg_search_async, or
 * fg_search_device on several streams), so that each batch shares the GPU
 * with the next: the pair mode while two batches of this size are resident at
 * once, one warp per query above.  FG_KERNEL=cta|pair|warp|staged in the
 * environment overrides either goal. */
int fg_index_set_plan_goal(fg_index* index, int32_t goal);

/* Kernel codes of fg_search_plan. */
#define FG_PLAN_CTA 0    /* one CTA per query */
#define FG_PLAN_WARP 1   /* one warp per query */
#define FG_PLAN_STAGED 2 /* one warp per query, parent blocks staged in shared memory */
#define FG_PLAN_PAIR 3   /* two warps per query */

/* The kernel the planner picks for a batch of nq queries at (K, beam) under
 * the index's goal, and how many queries it holds resident on the device at
 * once (kernel and resident_queries may be NULL).  No counterpart in the
 * reference; launches nothing. */
int fg_search_plan(fg_index* index, int32_t nq, int32_t K, int32_t beam, int32_t* kernel, int32_t* resident_queries);

/* Replaces QuantizationGraph::gpu_search_adaptive(nq, queries, K, result_idx,
 * beam_sz, elapsed) (gpu_search_adaptive.cu:12-114): host buffers in and out,
 * synchronous.  queries[nq*dim] row-major fp32, result_idx[nq*K].
 * elapsed_s (optional) = wall time of the search launch and its
 * synchronisation, excluding the copies, as the reference measures it
 * (gpu_search_adaptive.cu:98-107).  Supported: 1 <= K, 1 <= beam <= 1024,
 * degree <= 32, dim <= 4096. */
int fg_search(fg_index* index, int32_t nq, const float* queries, int32_t K, uint32_t* result_idx, int32_t beam,
              double* elapsed_s);

/* Replicated index on several devices from one host thread: `indexes` holds
 * `count` handles of the same codebook, each loaded on its own device
 * (fg_index_load with device = 0, 1, ...).  The batch is split into
 * contiguous, balanced slices in handle order; every device's copies and
 * launch are issued before any is awaited, so the devices search concurrently;
 * result_idx[nq*K] (and result_dist[nq*K], optional) are gathered in query
 * order.  elapsed_s (optional) = wall time from the first launch to the last
 * device's completion, excluding the copies.  Same arguments and errors as
 * fg_search otherwise; no counterpart in the reference (its search uses the
 * current device only, gpu_search_adaptive.cu:30-34). */
int fg_search_multi(fg_index* const* indexes, int32_t count, int32_t nq, const float* queries, int32_t K,
                    uint32_t* result_idx, float* result_dist, int32_t beam, double* elapsed_s);

/* Number of buffer slots of fg_search_async per index. */
#define FG_ASYNC_SLOTS 4

/* Streamed variant of fg_search for pipelines of query batches (the
 * reference re-uploads its index and synchronises on every call,
 * gpu_search_adaptive.cu:65-113): enqueues on `stream` the upload of
 * queries[nq*dim], the search and the download of the ids into
 * result_idx[nq*K], and returns without waiting.  `slot` (0 ..
 * FG_ASYNC_SLOTS-1) names the index's device buffers the batch uses, so
 * batches in different slots may be in flight at once -- one slot per stream
 * lets batch i+1's upload overlap batch i's search.  Host buffers should be
 * pinned (cudaHostAlloc) for the copies to run asynchronously.  The caller
 * synchronises the stream before reading result_idx and before reusing the
 * slot or the host buffers.  The first use of a slot, or a larger batch than
 * it has held, allocates its buffers. */
int fg_search_async(fg_index* index, int32_t slot, int32_t nq, const float* queries, int32_t K, uint32_t* result_idx,
                    int32_t beam, void* stream);

/* Size of the fixed device scratch used by fg_search_noalloc (8 MiB). */
#define FG_NOALLOC_SCRATCH_BYTES 8388608

/* fg_search without any device allocation; it has no counterpart in the
 * reference.  Same arguments, results and errors as fg_search, but the
 * queries, the result ids and the kernel's work counter are staged in a fixed
 * FG_NOALLOC_SCRATCH_BYTES array of device memory that is part of the
 * library, where fg_search grows buffers with cudaMalloc on demand (and the
 * reference allocates and frees them on every call).  It is for callers that
 * must not allocate during a search: a serving loop that must not stall its
 * other streams on the device-wide synchronisation cudaFree implies, or a
 * process whose device memory is entirely owned by another allocator.
 * Limit: 256 + round_up(nq*dim*4, 256) + nq*K*4 <= FG_NOALLOC_SCRATCH_BYTES
 * (e.g. 14,000 queries of dim 128 with K = 10); a larger batch returns
 * FG_ERR_ARG with a message -- split it or call fg_search.
 * Like fg_search the call is synchronous: it waits for the query upload, the
 * search and the download of the ids before it returns.
 * The first call on each device looks up the scratch's address on that
 * device; make that first call before any stream capture.  All calls on a
 * device share the one scratch array: calls that overlap in time (from
 * several threads, or on several indexes of one device) race on it and must
 * be serialised by the caller. */
int fg_search_noalloc(fg_index* index, int32_t nq, const float* queries, int32_t K, uint32_t* result_idx,
                      int32_t beam, double* elapsed_s);

/* Device-resident variant: d_queries / d_result_idx / d_result_dist (optional)
 * are device pointers on the index's device; the call is asynchronous on
 * `stream` (a cudaStream_t, NULL = default stream).  Searches on different
 * streams may run at the same time (each stream gets its own work counter,
 * allocated on its first search; at most 64 streams per index). */
int fg_search_device(fg_index* index, int32_t nq, const float* d_queries, int32_t K, uint32_t* d_result_idx,
                     float* d_result_dist, int32_t beam, void* stream);

/* Extended device variant: optional per-query counters d_stats[nq] and an
 * optional traversal trace d_trace[nq*trace_cap*8] (expander node ids per
 * iteration, 0xFFFFFFFF when unused) with d_trace_count[nq*trace_cap]. */
int fg_search_device_ex(fg_index* index, int32_t nq, const float* d_queries, int32_t K, uint32_t* d_result_idx,
                        float* d_result_dist, int32_t beam, void* stream, fg_query_stats* d_stats,
                        uint32_t* d_trace, int32_t* d_trace_count, int32_t trace_cap);

/* Query-side rotation and quantisation (include/utils.cuh:790-939) as a
 * standalone kernel: per query the rotated vector d_rotated[nq*D], the 6-bit
 * codes d_quant[nq*D], the 16-entry nibble LUT d_lut[nq*4*D] and
 * d_factors[nq*3] = (low, high, width), d_sum_q[nq].  Any output may be NULL
 * except d_factors. */
int fg_query_prepare_device(const float* d_queries, int32_t nq, int32_t dim, const float* d_signs,
                            float* d_rotated, uint8_t* d_quant, uint8_t* d_lut, float* d_factors,
                            int32_t* d_sum_q, void* stream);

/* Beam merge primitive on device, for verification (include/utils.cuh:1369-1399):
 * ncase independent cases, each [itopk beam entries | cbs candidates] in
 * d_idx/d_dist, merged in place with the reference's tie order. */
int fg_beam_merge_device(uint32_t* d_idx, float* d_dist, int32_t ncase, int32_t itopk, int32_t cbs, int32_t first,
                         void* stream);

/* Global top-K of a sharded index (the base split into
 * `shards` parts, each with its own graph): d_ids / d_dists hold, shard-major,
 * every shard's ascending top-k of the same nq queries ([shards][nq][k],
 * local ids as fg_search_device returns them, e.g. after an all-gather);
 * shard_offsets (host, `shards` entries, NULL = all 0) is the global id of
 * each shard's node 0.  Writes d_out_ids[nq*K] (global ids) and optionally
 * d_out_dists[nq*K]: the lists' stable merge by (distance, shard, position).
 * Asynchronous on `stream`.  Needs shards*k >= K and shards <= 64.  No
 * counterpart in the reference, whose index is one graph on one device
 * (gpu_search_adaptive.cu:65-72). */
int fg_shard_merge_device(const uint32_t* d_ids, const float* d_dists, const uint32_t* shard_offsets, int32_t shards,
                          int32_t nq, int32_t k, int32_t K, uint32_t* d_out_ids, float* d_out_dists, void* stream);

/* ---- key/value cache and attention over it ----
 *
 * What a decoder needs next to a search over its keys (metric
 * FG_METRIC_IP: the base is the keys of one kv head, a query is a query
 * vector, the ids are positions of the context): a paged cache that the
 * positions address, and attention over the first tokens, a sliding window
 * and the retrieved ids.  No counterpart in the reference, which ends at the
 * ids.
 *
 * All calls run on the calling thread's current device and are asynchronous
 * on `stream` (a cudaStream_t, NULL = default stream); they allocate nothing,
 * keep nothing and may be captured in a CUDA graph (make a first call of each
 * kind before a capture: it loads the kernels).  Buffers are device memory and
 * must not overlap, nor rows of one that is written (an output, the cache of an
 * append, a plan's block table): strides by which an axis does not pass what the
 * axes with smaller strides cover are refused.  Lengths, tables, slots and ids
 * are read on the device: values that address nothing (negative or too large
 * pages, slots, ids) are skipped, never followed. */

/* Element types of queries, caches and outputs. */
#define FG_DTYPE_F16 0
#define FG_DTYPE_BF16 1

/* A paged cache: position j of a request lies in page block_table[j /
 * page_size], row j % page_size.  Row (page, t, head) of K starts at element
 * page * page_stride + t * token_stride + head * head_stride of k, and of V
 * likewise of v: any order of the axes, and slices of a larger buffer.
 * k, v and the strides in bytes must be multiples of 16 (that of an axis of one
 * entry, here and in all rows, is not looked at); page_size a power of two; dim
 * 64, 96 or 128, contiguous. */
typedef struct fg_kv_cache {
    void* k;
    void* v;
    int64_t page_stride, token_stride, head_stride; /* elements */
    int32_t pages, page_size, heads, dim, dtype;
} fg_kv_cache;

/* The plan of one step for a batch of requests: request b has d_ctx_len[b]
 * tokens in the cache and gets d_new_len[b] more (negative: 0).
 * d_block_table [requests, table_width] (rows table_stride elements apart)
 * holds the pages of the first and receives those of the rest, taken in
 * request order from d_free_pages[free_count], starting at *d_free_head (NULL:
 * 0).  Outputs: d_query_start[requests+1], the first row of each request in
 * the step's token tensors; d_kv_len[requests] = ctx + new; for each token
 * row d_position[tokens] and d_slot[tokens] (page * page_size + row), -1 past
 * the last request's; d_free_head_out[1], the first page not taken (not
 * d_free_head itself, which other CTAs may still be reading);
 * d_refused[requests], 1 for a request that got nothing because its length
 * passes the table's width or 2^31 - 1, or because it needs pages that are no
 * longer there after the requests before it (one that needs none goes on): its kv_len
 * is 0, its positions and slots -1, its table row as it was.
 * At most 8192 requests. */
int fg_kv_plan_device(const int32_t* d_ctx_len, const int32_t* d_new_len, int32_t requests,
                      const int32_t* d_free_pages, int32_t free_count, const int32_t* d_free_head, int32_t page_size,
                      int32_t* d_block_table, int32_t table_width, int64_t table_stride, int32_t tokens,
                      int32_t* d_query_start, int32_t* d_kv_len, int32_t* d_position, int64_t* d_slot,
                      int32_t* d_free_head_out, int32_t* d_refused, void* stream);

/* Writes the new tokens' rows to the cache: row t of d_k and d_v [tokens,
 * heads, dim] (token and head strides in elements, multiples of 16 bytes) to
 * slot d_slot[t]; slots below 0 or past the cache are skipped.  Slots of one
 * call must differ. */
int fg_kv_append_device(const fg_kv_cache* cache, const void* d_k, int64_t k_token_stride, int64_t k_head_stride,
                        const void* d_v, int64_t v_token_stride, int64_t v_head_stride, const int64_t* d_slot,
                        int32_t tokens, void* stream);

/* Arguments of the attention calls. */
typedef struct fg_attention {
    const void* q;                              /* [tokens, heads, dim] of the cache's dtype */
    int64_t q_token_stride, q_head_stride;      /* elements, multiples of 16 bytes */
    void* out;                                  /* [tokens, heads, dim] */
    int64_t out_token_stride, out_head_stride;
    float* lse;                                 /* [tokens, heads], natural log; NULL: not written */
    const int32_t* block_table;                 /* [requests, table_width] */
    int64_t table_stride;
    const int32_t* query_start;                 /* [requests + 1] */
    const int32_t* kv_len;                      /* [requests], new tokens included */
    const int32_t* ids;                         /* fg_retrieved_attention_device: [tokens, heads, ids_count]
                                                 * fg_block_attention_device: blocks [tokens, kv heads, ids_count] */
    int64_t ids_token_stride, ids_head_stride;
    void* workspace;                            /* fg_attention_workspace_bytes, 256-byte aligned; contents do not matter;
                                                 * NULL where 0 bytes are needed */
    uint64_t workspace_bytes;
    int32_t tokens, heads, requests, table_width;
    int32_t max_new;                            /* most new tokens of a request: picks the kernel, not the result */
    int32_t window;                             /* -1: none */
    int32_t sinks;
    int32_t ids_count;
    float scale;
} fg_attention;

/* Bytes of workspace that a call needs on the current device, for partial
 * results of rows whose keys are split over CTAs (0: none, where no row can
 * have many keys).  retrieved: 1 for fg_retrieved_attention_device, 2 for
 * fg_block_attention_device.  Depends
 * on args' counts (tokens, heads, requests, table_width, max_new, window,
 * sinks, ids_count), the scale's sign and which strides are 0 only. */
int fg_attention_workspace_bytes(const fg_kv_cache* cache, const fg_attention* args, int32_t retrieved,
                                 uint64_t* bytes);

/* Causal attention of a batch's new tokens over the cache.  Token i of
 * request b (row query_start[b] + i) stands at p = kv_len[b] - new_b + i and
 * sees the keys 0 <= j <= p, with a window >= 0 those with p - j < window or
 * j < sinks; query head h reads kv head h / (heads / cache->heads).  out =
 * softmax(scale * q.k) v over the visible keys, lse = log of the sum of
 * exponentials; a row that sees nothing (or only scores of -inf) gets 0 and
 * -inf.  K and V of keys that a row does not see do not touch it, whatever
 * they hold.  Sums are kept in 32 bits; the weights of the second product are
 * rounded to the cache's type (those of float16 scaled so that weights of 2^-32
 * of the largest still count).  Results are the same on every run.  Rows past
 * query_start[requests] are not written.  At most 16384 requests, heads /
 * cache->heads <= 256. */
int fg_paged_attention_device(const fg_kv_cache* cache, const fg_attention* args, void* stream);

/* The same with retrieved keys: row (token, head) also sees the positions in
 * ids[token, head, :] that are in [0, p].  The visible keys are a set: an id
 * that repeats, or that the window or the first tokens hold already, counts
 * once; ids outside [0, p] (such as the search's padding, 0xFFFFFFFF) count
 * nothing.  Needs a window >= 0; at most 1024 ids for each row (more
 * than a search finds). */
int fg_retrieved_attention_device(const fg_kv_cache* cache, const fg_attention* args, void* stream);

/* ---- attention over chosen pages ----
 *
 * For contexts that no index was built over: each page's keys are summed up in
 * 8 bits, a query's bound on its scores with them is computed for every page,
 * and the attention reads the window, the first tokens and the pages of the
 * highest bounds.  The same rules as above hold (device, stream, buffers,
 * capture). */

/* Summaries of a cache's pages, for each kv head: bounds[page, head, 0, d] and
 * [page, head, 1, d] are the least and the largest value of the page's keys in
 * element d, rounded down and up to whole multiples (-127 to 127) of
 * scale[page, head], which is the largest magnitude times the 32-bit number
 * nearest 1 / 127.  scale is inf (and the bounds 0) where a key is not finite.
 * The last two axes are contiguous; bounds and its strides are multiples of 16
 * bytes. */
typedef struct fg_kv_summary {
    int8_t* bounds;
    float* scale;
    int64_t bounds_page_stride, bounds_head_stride; /* bytes */
    int64_t scale_page_stride, scale_head_stride;   /* elements */
    int32_t pages, page_size, heads, dim;
} fg_kv_summary;

/* Writes the summaries of the pages that hold the new tokens of each request,
 * positions kv_len[b] - new_b to kv_len[b] - 1 (new_b = query_start[b + 1] -
 * query_start[b]; a query_start made from kv_len itself gives all pages), from
 * the keys before kv_len[b] alone, whatever lies behind them.  After the append
 * of the step; with a cache whose v may be NULL.  tokens: the most that
 * query_start[requests] can be.  Pages of one call must differ. */
int fg_kv_summarize_device(const fg_kv_cache* cache, const fg_kv_summary* summary, const int32_t* d_block_table,
                           int32_t table_width, int64_t table_stride, const int32_t* d_query_start,
                           const int32_t* d_kv_len, int32_t requests, int32_t tokens, void* stream);

/* Arguments of the selection. */
typedef struct fg_block_selection {
    const void* q;                         /* [tokens, heads, dim] of `dtype` */
    int64_t q_token_stride, q_head_stride; /* elements, multiples of 16 bytes */
    const int32_t* block_table;            /* [requests, table_width] */
    int64_t table_stride;
    const int32_t* query_start;            /* [requests + 1] */
    const int32_t* kv_len;                 /* [requests], new tokens included */
    int32_t* blocks;                       /* [tokens, kv_heads, count] */
    int64_t blocks_token_stride, blocks_head_stride;
    void* workspace;                       /* fg_select_blocks_workspace_bytes, 16-byte aligned; contents do not matter;
                                            * NULL where 0 bytes are needed */
    uint64_t workspace_bytes;
    int32_t tokens, heads, requests, table_width;
    int32_t window, sinks, count, dtype;
} fg_block_selection;

/* Bytes of workspace that a selection needs, for the scores of long contexts
 * (0 where table_width is small).  Depends on tokens, table_width and
 * summary->heads only. */
int fg_select_blocks_workspace_bytes(const fg_kv_summary* summary, const fg_block_selection* args, uint64_t* bytes);

/* For the new token at position p (as in fg_paged_attention_device) and each kv
 * head, the `count` blocks of the highest score, ascending, then -1.  Block x of
 * a request is its positions [x * page_size, (x + 1) * page_size), the page
 * block_table[x].  Blocks that end past the first tokens and begin before the
 * window (x * page_size <= p - window and (x + 1) * page_size > sinks) are
 * chosen from: all with a position that neither shows, and, where window and
 * first tokens meet inside of one block, that block, which adds nothing.  Those
 * without a page in the cache are not.  A block's score is that of all keys that
 * were summed up, later tokens of the same step among them (the attention reads
 * none of those).  The score is in the 8-bit arithmetic of the summary:
 * with top the largest |q_d| of a query head, Q_d = q_d * 127 / top rounded to
 * the nearest whole number and t = top times the 32-bit number nearest 1 / 127,
 *   score = max over the kv head's query heads of
 *           (sum_d Q_d * bounds[Q_d < 0 ? 0 : 1][d]) * t, times scale,
 * the products after the sum in 32 bits.  But for their roundings it bounds the
 * q.k of the page's keys for the query that Q_d * t stands for; that of q itself
 * may pass it by the query's rounding, top / 254 * sum_d |k_d| at most.  (So it
 * is for attention with a positive scale.)  A query head with a value that is not
 * finite counts as 0, a page of scale inf has the score inf.  Of equal scores the lowest block comes
 * first.  The same bits on every run.  Waits inside a kernel are bounded: one
 * that runs out (a second; a sound device has none) leaves -2 in all of its
 * row's places.  The last axis of blocks is contiguous.
 * Rows past query_start[requests] are not written.  Needs a window >= 0 and
 * heads / summary->heads <= 256. */
int fg_select_blocks_device(const fg_kv_summary* summary, const fg_block_selection* args, void* stream);

/* fg_paged_attention_device over window, first tokens and chosen blocks: row
 * (token, head) also sees the positions j <= p of the blocks of page_size
 * positions in ids[token, head's kv head, :].  The visible keys are a set:
 * blocks in any order, a block that repeats counts once, as do its positions
 * that window and first tokens show already; negative blocks and those past the
 * context count nothing.  The weights of the product with V are rounded to the
 * cache's type, as in fg_paged_attention_device.  Needs a window >= 0; at most
 * 1024 blocks for each kv head. */
int fg_block_attention_device(const fg_kv_cache* cache, const fg_attention* args, void* stream);

/* ---- eviction by attention weight ----
 *
 * The other way to bound what a step reads: keep the cache short.  Each key's
 * attention weight is summed up over the steps, and where a request has passed
 * its budget each kv head drops its lightest keys.  The same rules as above
 * hold. */

/* Adds to d_weights (float [pages, heads, page_size], strides in elements, the
 * last axis contiguous; beside the cache, one for each layer) the weights that
 * the step's rows gave to each key: for position j of a request and each kv head
 *   weight = (j < held ? weight : 0) + sum of exp(scale * q.k_j - lse)
 * over its new tokens' rows of the kv head's query heads that see j (mask as in
 * fg_paged_attention_device).  args: q, lse (here read: [tokens, heads], as the
 * step's attention left it), block_table, query_start, kv_len, window, sinks,
 * scale and the counts; out, ids, workspace and max_new are not looked at.
 * d_held [requests]: tokens whose weights are there already (NULL: those before
 * the new ones); weights from there to kv_len[b] start at 0, whatever was there,
 * also of requests without new tokens, and in a call without any.
 * Rows whose lse is not finite add nothing.  Sums are 32 bits, in the order of
 * the rows: the same bits on every run, but where requests share a page, whose
 * sums are added to it in any order (of shared pages none may be new).  Only the last tokens of a prompt may be
 * given: query_start counts them alone.  The cache's v may be NULL. */
int fg_attention_weights_device(const fg_kv_cache* cache, const fg_attention* args, float* d_weights,
                                int64_t weights_page_stride, int64_t weights_head_stride, const int32_t* d_held,
                                void* stream);

/* For each request of more than `budget` positions and each kv head: the first
 * `sinks`, the last `recent` and, of those between, the budget - sinks - recent
 * of the largest weights stay (of equal weights the lowest position; NaN counts
 * as -inf, positions without a page are lighter still) and move, in ascending
 * order, to positions 0 to budget - 1: rows of K and V and their weights, in
 * place.  Lengths count as max(0, min(kv_len, table_width * page_size)): the
 * last positions are those of the table where a length passes it.
 * d_kv_len_out[requests]: the smaller of that and the budget (it may not overlap
 * d_kv_len); d_kept [requests, heads, budget]: the position that each was at, -1
 * past the request's length.  Requests within the budget stay as they are.  Pages of
 * block_table from ceil(budget / page_size) on are free afterwards (where all
 * layers that share the table are done); pages that two requests share must not
 * be evicted from.  sinks + recent <= budget, budget >= 1. */
int fg_kv_evict_device(const fg_kv_cache* cache, float* d_weights, int64_t weights_page_stride,
                       int64_t weights_head_stride, const int32_t* d_block_table, int32_t table_width,
                       int64_t table_stride, const int32_t* d_kv_len, int32_t requests, int32_t budget, int32_t recent,
                       int32_t sinks, int32_t* d_kv_len_out, int32_t* d_kept, void* stream);

/* ---- host helpers of the reference CLI ---- */

/* include/utils.cuh:119-127 */
uint32_t fg_effective_sort_beam_size(uint32_t beam);

/* include/common.hpp:26-47: the entry point a codebook gets when its header
 * holds UINT32_MAX -- the node whose raw vector (the first dim floats of each
 * row of row_floats floats) is nearest the centroid of all raw vectors (largest
 * inner product for FG_METRIC_IP), the first such node on ties.  fg_index_load
 * and fg_index_create apply it.  Returns UINT32_MAX for invalid arguments
 * (NULL rows, num_nodes or dim 0, row_floats < dim). */
uint32_t fg_entry_point_centroid(const float* rows, uint64_t num_nodes, uint64_t dim, uint64_t row_floats,
                                 int32_t metric);

/* include/common.hpp:49-66: recall of predicted[nq*topk] against
 * groundtruth[nq*gt_k]; duplicates in a prediction row are all counted. */
float fg_compute_recall(const uint32_t* predicted, const int32_t* groundtruth, uint64_t nq, int32_t topk,
                        int32_t gt_k);

/* include/common.hpp:68-94: append TopK,Beam_size,Runtime,Latency,Throughput,Recall. */
int fg_append_run_stats_csv(const char* path, int32_t k, int32_t beam, double runtime, double latency,
                            double throughput, double recall);

/* include/metric.hpp:13-28: FG_METRIC_IP iff the path contains "text2image1m". */
int32_t fg_infer_metric_from_path(const char* path);

/* include/data_io.hpp:18-77: count and dim of an fvecs/ivecs file
 * (count = file_size / (4 + 4*dim)), then read it into dst[count*dim]. */
int fg_vecs_info(const char* path, uint64_t* count, int32_t* dim);
int fg_vecs_read(const char* path, void* dst, uint64_t count, int32_t dim);

#ifdef __cplusplus
}
#endif
#endif
