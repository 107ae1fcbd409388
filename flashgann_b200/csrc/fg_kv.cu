// fg_kv.cu -- the paged key/value cache: a step's plan (block tables and slot
// maps from request lengths) and the append of new rows.
#include <algorithm>
#include <cstdint>

#include <cuda_runtime.h>

#include "fg_internal.h"

namespace fg {
namespace {

// ---- plan ----
//
// Request b has ctx tokens in the cache and gets new ones.  With ps tokens to
// a page and pages(n) = ceil(n / ps) it needs need_b = pages(ctx + new) -
// pages(ctx) fresh pages; those are free_pages[head + first_b ..), first = the
// exclusive sum of need.  Token i of b (row query_start_b + i of the step's
// tensors, query_start = the exclusive sum of new) stands at position ctx + i
// and goes to slot page * ps + position % ps.
//
// A few bytes for each request and 12 for each token: the time is the launch
// and one chain of dependent loads.  So there is one launch and no
// communication between CTAs: every CTA scans all requests (each thread sums a
// run of them, one block scan joins the runs), keeps both prefixes in shared
// memory, and then maps its own share of tokens and pages back to requests by
// bisection.  A fresh page is taken from the free list by index, never read
// back from the table that another thread may be writing.  Measured: 3.5 us for
// 8 requests, 6.4 to 6.9 us for 1000 with 62K tokens, of which 3.1 are the scan
// and 1.0 the token rows.
constexpr int kPlanThreads = 512;

struct Need {
    int64_t pages;  // fresh pages, 0 for a request that is too long for the table
    int64_t had;    // pages in use
    bool wide;
};

__device__ __forceinline__ Need page_need(const PlanArgs& a, int64_t ctx, int64_t add) {
    const int64_t round = (int64_t{1} << a.page_shift) - 1;
    Need n;
    n.had = (ctx + round) >> a.page_shift;
    const int64_t will = (ctx + add + round) >> a.page_shift;
    n.wide = will > a.table_width || ctx + add > INT32_MAX;  // lengths and positions are 32 bits
    n.pages = n.wide ? 0 : will - n.had;
    return n;
}

// first index with end[i] > x, of n ascending values whose last exceeds x
template <typename T>
__device__ __forceinline__ int owner(const T* end, int n, T x) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (end[mid] > x) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

__global__ void __launch_bounds__(kPlanThreads) kv_plan_kernel(const PlanArgs a) {
    extern __shared__ int64_t plan_smem[];
    int64_t* page_end = plan_smem;                // inclusive sum of need
    int64_t* token_end = page_end + a.requests;   // inclusive sum of new
    int32_t* ctx_of = reinterpret_cast<int32_t*>(token_end + a.requests);
    __shared__ int64_t warp_pages[kPlanThreads / 32], warp_tokens[kPlanThreads / 32];
    __shared__ unsigned long long taken;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per = (a.requests + kPlanThreads - 1) / kPlanThreads;
    const int b0 = min(tid * per, a.requests), b1 = min(b0 + per, a.requests);
    if (tid == 0) taken = 0;
    int64_t pages = 0, tokens = 0;
#pragma unroll 4
    for (int b = b0; b < b1; ++b) {
        const int64_t ctx = max(0, __ldg(a.ctx_len + b)), add = max(0, __ldg(a.new_len + b));
        pages += page_need(a, ctx, add).pages;
        tokens += add;
        page_end[b] = pages;
        token_end[b] = tokens;
        ctx_of[b] = static_cast<int32_t>(ctx);
    }
    int64_t sp = pages, st = tokens;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int64_t vp = __shfl_up_sync(0xFFFFFFFFu, sp, d), vt = __shfl_up_sync(0xFFFFFFFFu, st, d);
        if (lane >= d) {
            sp += vp;
            st += vt;
        }
    }
    if (lane == 31) {
        warp_pages[warp] = sp;
        warp_tokens[warp] = st;
    }
    __syncthreads();
    int64_t bp = sp - pages, bt = st - tokens;
    for (int w = 0; w < warp; ++w) {
        bp += warp_pages[w];
        bt += warp_tokens[w];
    }
    const int64_t head = a.free_head ? max(0, *a.free_head) : 0;
    const int64_t room = max(static_cast<int64_t>(0), a.free_count - head);
    const bool writes = blockIdx.x == 0;  // the outputs for each request
    int64_t last = 0, tokens_before = bt;
    for (int b = b0; b < b1; ++b) {
        const int64_t pe = page_end[b] += bp, te = token_end[b] += bt;
        if (!writes) continue;
        const int64_t ctx = ctx_of[b], add = te - tokens_before;
        tokens_before = te;
        const Need n = page_need(a, ctx, add);
        const bool refused = n.wide || (n.pages > 0 && pe > room);
        if (!refused && n.pages > 0) last = pe;  // the admitted ones are a prefix of those that need pages
        a.query_start[b + 1] = static_cast<int32_t>(min(te, static_cast<int64_t>(INT32_MAX)));
        a.kv_len[b] = refused ? 0 : static_cast<int32_t>(ctx + add);
        a.refused[b] = refused;
    }
    if (writes && last) atomicMax(&taken, static_cast<unsigned long long>(last));
    __syncthreads();
    if (writes && tid == 0) {
        a.query_start[0] = 0;
        *a.free_head_out = static_cast<int32_t>(head + static_cast<int64_t>(taken));
    }
    const int64_t threads = static_cast<int64_t>(gridDim.x) * kPlanThreads;
    const int64_t first = static_cast<int64_t>(blockIdx.x) * kPlanThreads + tid;
    const int64_t all_tokens = token_end[a.requests - 1], all_pages = min(page_end[a.requests - 1], room);
    for (int64_t t = first; t < a.tokens; t += threads) {
        int32_t pos = -1;
        int64_t slot = -1;
        if (t < all_tokens) {
            const int b = owner(token_end, a.requests, t);
            const int64_t ctx = ctx_of[b], add = token_end[b] - (b ? token_end[b - 1] : 0);
            const Need n = page_need(a, ctx, add);
            if (!(n.wide || (n.pages > 0 && page_end[b] > room))) {
                const int64_t p = ctx + t - (token_end[b] - add);
                const int64_t page = p >> a.page_shift;
                const int32_t id = page < n.had ? a.block_table[b * a.table_stride + page]
                                                : a.free_pages[head + page_end[b] - n.pages + page - n.had];
                pos = static_cast<int32_t>(p);
                if (id >= 0) slot = (static_cast<int64_t>(id) << a.page_shift) + (p & ((1 << a.page_shift) - 1));
            }
        }
        a.position[t] = pos;
        a.slot[t] = slot;
    }
    for (int64_t x = first; x < all_pages; x += threads) {
        const int b = owner(page_end, a.requests, x);
        if (page_end[b] > room) continue;  // the pool ends inside this request: it is refused whole
        const int64_t ctx = ctx_of[b], add = token_end[b] - (b ? token_end[b - 1] : 0);
        const Need n = page_need(a, ctx, add);
        a.block_table[b * a.table_stride + n.had + x - (page_end[b] - n.pages)] = a.free_pages[head + x];
    }
}

// ---- append ----
//
// A copy of tokens * heads rows of K and of V: 2 * 2 bytes of traffic for each
// element, nothing else.  A thread moves one 16-byte piece of each; consecutive
// threads take consecutive pieces of a row, so that a row is whole 128-byte
// lines on both sides.  (2, 4 and 8 pieces to a thread: 1, 11 and 48 % slower
// for 16001 tokens of 4 x 96; what hides the latency is the number of CTAs.)  Measured: those 49 MB in
// 10.4 to 11.0 us, 4.5 to 4.7 TB/s: start and end weigh in a copy of 7 us (as
// many contiguous bytes through a kernel of one operation: 9.2 to 10.0 us).
constexpr int kAppendThreads = 256;

__global__ void __launch_bounds__(kAppendThreads) kv_append_kernel(const AppendArgs a) {
    const int64_t slots = static_cast<int64_t>(a.pages) << a.page_shift;
    const uint32_t per = static_cast<uint32_t>(a.heads) * a.pieces;  // pieces of a token
    const int64_t total = static_cast<int64_t>(a.tokens) * per;
    const int64_t idx = static_cast<int64_t>(blockIdx.x) * kAppendThreads + threadIdx.x;
    if (idx >= total) return;
    const int64_t t = total <= UINT32_MAX ? static_cast<uint32_t>(idx) / per : idx / per;
    const uint32_t rest = static_cast<uint32_t>(idx - t * per);
    const uint32_t h = rest / a.pieces, p = rest % a.pieces;
    const int64_t slot = __ldg(a.slot + t);
    const uint4 k = __ldg(static_cast<const uint4*>(a.k) + t * a.k_token_stride + h * a.k_head_stride + p);
    const uint4 v = __ldg(static_cast<const uint4*>(a.v) + t * a.v_token_stride + h * a.v_head_stride + p);
    if (slot < 0 || slot >= slots) return;
    const int64_t to = (slot >> a.page_shift) * a.page_stride + (slot & ((1 << a.page_shift) - 1)) * a.token_stride + h * a.head_stride + p;
    static_cast<uint4*>(a.k_cache)[to] = k;
    static_cast<uint4*>(a.v_cache)[to] = v;
}

}  // namespace

constexpr int kPlanRequests = 8192;
constexpr int kPlanBytes = 2 * sizeof(int64_t) + sizeof(int32_t);  // of a request, in one CTA's shared memory
int kv_plan_max_requests() { return kPlanRequests; }

cudaError_t launch_kv_plan(const PlanArgs& a, cudaStream_t stream) {
    const size_t smem = static_cast<size_t>(a.requests) * kPlanBytes;
    if (smem > 40 * 1024) {
        static SmemOnce once;
        const cudaError_t e = once.set(reinterpret_cast<const void*>(kv_plan_kernel), kPlanRequests * kPlanBytes);
        if (e != cudaSuccess) return e;
    }
    const int64_t pages = std::min<int64_t>(a.free_count, static_cast<int64_t>(a.requests) * a.table_width);
    const int64_t items = std::max<int64_t>(a.tokens, pages);
    const int grid = static_cast<int>(std::clamp<int64_t>((items + kPlanThreads - 1) / kPlanThreads, 1, 148));
    kv_plan_kernel<<<grid, kPlanThreads, smem, stream>>>(a);
    return cudaGetLastError();
}

cudaError_t launch_kv_append(const AppendArgs& a, cudaStream_t stream) {
    const int64_t total = static_cast<int64_t>(a.tokens) * a.heads * a.pieces;
    const int64_t grid = (total + kAppendThreads - 1) / kAppendThreads;
    if (grid > INT32_MAX) return cudaErrorInvalidConfiguration;
    kv_append_kernel<<<static_cast<unsigned>(grid), kAppendThreads, 0, stream>>>(a);
    return cudaGetLastError();
}

}  // namespace fg
