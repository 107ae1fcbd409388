// fg_internal.h -- launch interface between the C ABI (fg_api.cu) and the
// kernels (fg_search.cu, fg_search_warp.cu).  Not installed; the public surface is
// include/flashgann.h.
#pragma once

#include <atomic>
#include <cstddef>
#include <cstdint>

#include <cuda_runtime.h>

#include "../../include/flashgann.h"

namespace fg {

// Everything a search launch needs; sizes in float words like the codebook.
struct SearchArgs {
    const float* rows = nullptr;      // device, n * row floats
    const float* signs = nullptr;     // device, padded_dim floats
    const float* queries = nullptr;   // device, nq * dim
    uint32_t* out_ids = nullptr;      // device, nq * K
    float* out_dists = nullptr;       // device, nq * K (optional)
    fg_query_stats* stats = nullptr;  // device, nq (optional)
    uint32_t* trace = nullptr;        // device, nq * trace_cap * SEARCH_WIDTH (optional)
    int32_t* trace_count = nullptr;   // device, nq * trace_cap (optional)
    int trace_cap = 0;
    uint32_t* work_counter = nullptr; // device scratch, one uint32 (zeroed by the launcher)
    uint64_t n = 0, row = 0, code_off = 0, factor_off = 0, nbr_off = 0;
    int dim = 0, padded_dim = 0, degree = 0;
    uint32_t entry = 0;
    int use_ip = 0;
    int nq = 0, K = 0, beam = 0;
    int goal = 0;  // FG_GOAL_LATENCY or FG_GOAL_THROUGHPUT: what plan_search optimises for
};

// Derived per-launch constants, computed on the host (plan_search).
struct SearchPlan {
    uint32_t padded = 0;       // effective sort beam (include/utils.cuh:119-127)
    uint32_t cbs = 0;          // candidate buffer size (adaptive_search_utils.cuh:231-236)
    uint32_t collect_cap = 0;  // min(BUFFER_BOUND, cbs)
    int hbits = 0;             // visited table bits
    float phase2_rho = 0.0f;   // adaptive_search_utils.cuh:20-23
    int max_iter = 0;          // gpu_search_adaptive.cu:96
    int merge_n2 = 0;          // 1/2/4: register bitonic merge, 0: merge path
    int mp_active = 0;         // merge-path output segments
    int vec_codes = 0;         // codes 16-byte aligned: 128-bit code loads
    int variant = 0;           // CTA kernel variant (warps per query, register budget)
    int kernel = 0;            // 0: one CTA per query (fg_search.cu), 1: one warp per query (fg_search_warp.cu)
    uint32_t slots = 0;        // warp kernel: visited-set slots
    size_t slice_bytes = 0;    // warp kernel: shared memory per query
    int min_ctas = 0;          // warp kernel: CTAs per SM its register budget is compiled for
    uint32_t blk = 0;          // warp kernel, staged variant: bytes of one parent block (0: not staged)
    int warp_mode = 0;         // warp kernel: 0 one warp per query, 1 staged, 2 a pair of warps per query
    int resident_queries = 0;  // warp kernel: queries resident at once on the device
    size_t smem_bytes = 0;
    int grid = 0;
    int threads = 0;
    int blocks_per_sm = 0;
};

int plan_search(const SearchArgs& a, SearchPlan* plan, int device, char* err, size_t errlen);
cudaError_t launch_search(const SearchArgs& a, const SearchPlan& plan, cudaStream_t stream);

// The warp-per-query kernel (fg_search_warp.cu): padded dimensions 32..256.
bool warp_kernel_supports(int padded_dim);
// mode: 0 one warp per query, 1 its staged variant, 2 a pair of warps per query
int plan_search_warp(const SearchArgs& a, SearchPlan* plan, int device, char* err, size_t errlen, int mode);
cudaError_t launch_search_warp(const SearchArgs& a, const SearchPlan& plan, cudaStream_t stream);

cudaError_t launch_query_prepare(const float* queries, int nq, int dim, const float* signs, float* rotated,
                                 uint8_t* quant, uint8_t* lut, float* factors, int32_t* sum_q,
                                 cudaStream_t stream);

cudaError_t launch_beam_merge(uint32_t* idx, float* dist, int ncase, int itopk, int cbs, int first,
                              cudaStream_t stream);

// Per-query merge of a sharded index's top-k lists (fg_shard_merge.cu).
int shard_merge_max_shards();
cudaError_t launch_shard_merge(const uint32_t* ids, const float* dists, const uint32_t* offsets, int shards, int nq,
                               int k, int K, uint32_t* out_ids, float* out_dists, cudaStream_t stream);

// ---- key/value cache and attention (fg_kv.cu, fg_attention_rows.cu, fg_attention_tiles.cu) ----

// A kernel's shared memory limit, raised on a device's first launch of it to the most that any launch takes: threads may
// launch at the same time.
struct SmemOnce {
    std::atomic<uint64_t> devices{0};
    cudaError_t set(const void* kernel, int bytes) {
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess) return e;
        const uint64_t bit = dev < 64 ? uint64_t{1} << dev : 0;
        if (devices.load(std::memory_order_relaxed) & bit) return cudaSuccess;
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e == cudaSuccess) devices.fetch_or(bit, std::memory_order_relaxed);
        return e;
    }
};

struct PlanArgs {
    const int32_t* ctx_len = nullptr;
    const int32_t* new_len = nullptr;
    const int32_t* free_pages = nullptr;
    const int32_t* free_head = nullptr;  // optional
    int32_t* block_table = nullptr;
    int32_t* query_start = nullptr;
    int32_t* kv_len = nullptr;
    int32_t* position = nullptr;
    int64_t* slot = nullptr;
    int32_t* free_head_out = nullptr;
    int32_t* refused = nullptr;
    int64_t table_stride = 0;
    int requests = 0, free_count = 0, page_shift = 0, table_width = 0, tokens = 0;
};
int kv_plan_max_requests();
cudaError_t launch_kv_plan(const PlanArgs& a, cudaStream_t stream);

struct AppendArgs {
    void* k_cache = nullptr;
    void* v_cache = nullptr;
    const void* k = nullptr;
    const void* v = nullptr;
    const int64_t* slot = nullptr;
    int64_t page_stride = 0, token_stride = 0, head_stride = 0;  // of the cache, in 16-byte pieces
    int64_t k_token_stride = 0, k_head_stride = 0, v_token_stride = 0, v_head_stride = 0;  // in 16-byte pieces
    int pages = 0, page_shift = 0, heads = 0, pieces = 0;  // pieces: 16-byte pieces of a row
    int tokens = 0;
};
cudaError_t launch_kv_append(const AppendArgs& a, cudaStream_t stream);

struct AttentionParams {
    const void* k_cache = nullptr;
    const void* v_cache = nullptr;
    int64_t page_stride = 0, token_stride = 0, head_stride = 0;  // elements
    int pages = 0, page_size = 0, page_shift = 0;
    int dim = 0, dtype = 0;
    const void* q = nullptr;
    int64_t q_token_stride = 0, q_head_stride = 0;
    void* out = nullptr;
    int64_t out_token_stride = 0, out_head_stride = 0;
    float* lse = nullptr;  // [tokens, heads], optional
    const int32_t* block_table = nullptr;
    int64_t table_stride = 0;
    int table_width = 0;
    const int32_t* query_start = nullptr;
    const int32_t* kv_len = nullptr;
    int requests = 0, tokens = 0, heads = 0, kv_heads = 0, group = 0;
    uint32_t group_mul = 0;  // n / group = n * group_mul >> group_shift for n < 2^31
    int group_shift = 0;
    int window = -1, sinks = 0;
    float scale_log2 = 0.f;  // scale * log2(e): all exponents are base 2
    const int32_t* ids = nullptr;
    int ids_count = 0;
    int64_t ids_token_stride = 0, ids_head_stride = 0;
    void* workspace = nullptr;
    int ctas = 0;           // CTAs that share the work (to the launchers: SMs)
    int base_align = 16;    // power of two that windows' key chunks start at multiples of
    int unit_shift = 0;     // log2 of the key chunks in a unit of work
    int tile_units = 0;     // what a tile costs beside its chunks, in units
    int tile_rows = 16;     // retrieved form: heads to a tile
    // kernel of many rows: how often a wait inside a CTA looks again before it gives up; block whose K tile never comes
    int wait_tries = 0, lost_block = 0;
};
int attention_max_requests();
int attention_max_ids();
bool attention_rows_splits(const AttentionParams& a);
size_t attention_rows_workspace(const AttentionParams& a, int sms, int dim);  // 0 where nothing is split
cudaError_t launch_attention_rows(const AttentionParams& a, cudaStream_t stream);
bool attention_tiles_counts(const AttentionParams& a);
void set_attention_waits(int lost_block, int tries);  // for tests; below 0: none, and a limit of a second
size_t attention_tiles_workspace(int sms, int dim);
cudaError_t launch_attention_tiles(const AttentionParams& a, cudaStream_t stream);

// Host restatements shared with the CLI and the API.
uint32_t effective_sort_beam(uint32_t beam);
uint32_t candidate_buffer_size(int degree);
int hash_bits(uint32_t padded, uint32_t cbs);

}  // namespace fg
