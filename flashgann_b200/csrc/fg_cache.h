// fg_cache.h -- arguments and launchers of the kernels that choose what a step
// reads from the cache: page summaries, block selection, key weights, eviction.
#pragma once

#include <cstdint>

#include <cuda_runtime.h>

namespace fg {

// K of a paged cache, or of both halves; strides in elements.
struct PagedRows {
    const void* k = nullptr;
    int64_t page_stride = 0, token_stride = 0, head_stride = 0;
    int pages = 0, page_shift = 0, heads = 0, dim = 0, dtype = 0;
};

struct Requests {
    const int32_t* block_table = nullptr;
    int64_t table_stride = 0;
    const int32_t* query_start = nullptr;
    const int32_t* kv_len = nullptr;
    int table_width = 0, requests = 0, tokens = 0;
};

// int8 [pages, heads, 2, dim] (lower bounds, upper bounds) and float [pages, heads]; strides in elements
struct Summary {
    int8_t* bounds = nullptr;
    float* scale = nullptr;
    int64_t bounds_page_stride = 0, bounds_head_stride = 0, scale_page_stride = 0, scale_head_stride = 0;
};

// For tests: the search by which a row's or a page's request is found, where `first` and all after it are past.
int first_past_on_host(int n, int first);

struct SummarizeArgs {
    PagedRows cache;
    Summary summary;
    Requests req;
};
cudaError_t launch_kv_summarize(const SummarizeArgs& a, cudaStream_t stream);

struct SelectArgs {
    Summary summary;
    Requests req;
    const void* q = nullptr;
    int64_t q_token_stride = 0, q_head_stride = 0;
    int32_t* blocks = nullptr;  // [tokens, kv_heads, count]
    int64_t blocks_token_stride = 0, blocks_head_stride = 0;
    int pages = 0, page_shift = 0, kv_heads = 0, group = 0, dim = 0, dtype = 0;
    int window = 0, sinks = 0, count = 0;
    uint32_t* scores = nullptr;  // workspace
    int sms = 0;
};
void set_selection_waits(int lost_item, int tries);  // for tests; below 0: none, and a limit of a second
bool select_counts(int tokens, int kv_heads, int table_width);  // whether a launch can have so many CTAs
size_t select_workspace(int tokens, int kv_heads, int table_width);  // 0 where the scores stay in shared memory
cudaError_t launch_select_blocks(const SelectArgs& a, cudaStream_t stream);

struct AttentionParams;

// float [pages, heads, page_size], the last axis contiguous; strides in elements
struct KeyWeights {
    float* w = nullptr;
    int64_t page_stride = 0, head_stride = 0;
};

struct WeightsArgs {
    KeyWeights weights;
    const float* lse = nullptr;     // [tokens, heads]
    const int32_t* held = nullptr;  // [requests], optional
    float scale = 0.f;
};
void set_key_weights_waits(int lost_block, int tries);  // for tests; below 0: none, and a limit of a second
cudaError_t launch_attention_weights(const AttentionParams& a, const WeightsArgs& w, cudaStream_t stream);

struct EvictArgs {
    PagedRows cache;
    void* v = nullptr;
    KeyWeights weights;
    const int32_t* block_table = nullptr;
    int64_t table_stride = 0;
    const int32_t* kv_len = nullptr;
    int table_width = 0, requests = 0;
    int budget = 0, recent = 0, sinks = 0;
    int32_t* kv_len_out = nullptr;
    int32_t* kept = nullptr;  // [requests, heads, budget]
    int sms = 0;
};
cudaError_t launch_kv_evict(const EvictArgs& a, cudaStream_t stream);

}  // namespace fg
