// fg_evict.cu -- eviction from the cache by accumulated weight.
//
// Of a request of `len` positions that are more than the budget, each kv head
// keeps the first `sinks`, the last `recent` and, of those between, the heaviest
// budget - sinks - recent (of equal weights the lowest position; NaN counts as
// -inf).  In ascending order they move to positions 0 .. budget - 1: rows of K and
// V and the weights, in place.
//
// A cluster of CTAs has one request and kv head.  Its weights are read once, as
// keys of fg_topk.cuh (those beyond shared memory's room are read again), the kept
// positions go to the result, and then the cluster moves the rows, chunk by chunk
// of consecutive places: all of its CTAs load the chunk's rows into registers, the
// cluster waits, and they store them.  Place i is filled from kept[i] >= i, and the
// sources of later chunks lie behind the chunk, so the next chunk's loads need not
// wait for the stores.
#include <algorithm>
#include <cmath>
#include <cstdint>

#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include "fg_cache.h"
#include "fg_internal.h"
#include "fg_topk.cuh"

namespace fg {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxCluster = 8;
constexpr int kMaxSmem = 100 * 1024;  // two CTAs to an SM
constexpr int kLoads = 8;             // 16-byte pieces of a thread under way

template <int kDim, typename Ctas>
__global__ void __launch_bounds__(kThreads) kv_evict_kernel(const EvictArgs a, int room) {
    extern __shared__ __align__(16) char smem[];
    topk::Shared& s = *reinterpret_cast<topk::Shared*>(smem);
    uint32_t* near = reinterpret_cast<uint32_t*>(smem + sizeof(topk::Shared));  // [room]
    const int tid = threadIdx.x;
    const int ranks = Ctas::ranks(), rank = Ctas::rank();
    const int row = static_cast<int>(blockIdx.x) / ranks;
    const int b = row / a.cache.heads, head = row - b * a.cache.heads;
    const int shift = a.cache.page_shift, in_page = (1 << shift) - 1;
    const int len = static_cast<int>(min(static_cast<int64_t>(max(0, __ldg(a.kv_len + b))), static_cast<int64_t>(a.table_width) << shift));
    int32_t* kept = a.kept + static_cast<int64_t>(row) * a.budget;
    if (head == 0 && rank == 0 && tid == 0) a.kv_len_out[b] = min(len, a.budget);
    if (len <= a.budget) {
        for (int x = rank * kThreads + tid; x < a.budget; x += ranks * kThreads) kept[x] = x < len ? x : -1;
        return;
    }
    const int32_t* table = a.block_table + b * a.table_stride;
    const auto page_of = [&](int j) {
        const int page = __ldg(table + (j >> shift));
        return static_cast<uint32_t>(page) < static_cast<uint32_t>(a.cache.pages) ? page : -1;
    };
    float* weights = a.weights.w + head * a.weights.head_stride;
    const auto weight_at = [&](int page, int j) { return weights + page * a.weights.page_stride + (j & in_page); };

    // this CTA's positions between the first and the recent ones
    const int n = len - a.recent - a.sinks;
    const int per = (n + ranks - 1) / ranks;
    const int c0 = min(n, per * rank), m = min(n, c0 + per) - c0;
    const auto read = [&](int i) -> uint32_t {
        const int j = a.sinks + c0 + i, page = page_of(j);
        if (page < 0) return 1u;  // nothing there: lighter than any
        const float w = *weight_at(page, j);
        return topk::order_key(w == w ? w : -INFINITY);
    };
    topk::clear<kThreads>(s);
    uint32_t least = 0xFFFFFFFFu, most = 0;
    for (int i = tid; i < m; i += kThreads) {
        const uint32_t key = read(i);
        least = min(least, key);
        most = max(most, key);
        if (i < room) near[i] = key;
    }
    __syncthreads();
    topk::range(s, least, most);
    Ctas::sync();
    const auto keys = topk::read_keys<kThreads>([&](int i) { return i < room ? near[i] : read(i); });
    const topk::Threshold thr = topk::threshold<kThreads, Ctas>(s, m, a.budget - a.recent - a.sinks, keys);
    topk::emit<kThreads, Ctas>(s, m, thr, keys, [&](int place, int i) { kept[a.sinks + place] = a.sinks + c0 + i; });
    for (int x = rank * kThreads + tid; x < a.sinks; x += ranks * kThreads) kept[x] = x;
    for (int x = rank * kThreads + tid; x < a.recent; x += ranks * kThreads) kept[a.budget - a.recent + x] = len - a.recent + x;
    __threadfence();
    Ctas::sync();  // the whole list is there, and no weight is read as a key any more

    // a thread has one 16-byte piece of K or V of several rows
    constexpr int kPieces = 2 * kDim / 8, kTogether = kThreads / kPieces;
    const int piece = tid % kPieces, slot = tid / kPieces;
    const bool values = piece >= kPieces / 2;
    char* base = static_cast<char*>(values ? a.v : const_cast<void*>(a.cache.k));
    const int64_t off = head * a.cache.head_stride + (values ? piece - kPieces / 2 : piece) * 8;
    const auto piece_at = [&](int page, int j) {
        return reinterpret_cast<uint4*>(base + 2 * (page * a.cache.page_stride + (j & in_page) * a.cache.token_stride + off));
    };
    for (int i0 = a.sinks; i0 < a.budget; i0 += ranks * kLoads * kTogether) {
        uint4 v[kLoads];
        float w[kLoads];
        uint4* to[kLoads];
        int from[kLoads];
#pragma unroll
        for (int x = 0; x < kLoads; ++x) {
            const int i = i0 + (rank * kLoads + x) * kTogether + slot;
            from[x] = slot < kTogether && i < a.budget ? __ldcg(kept + i) : i;
            if (from[x] == i) from[x] = -1;  // in place already, or none
        }
#pragma unroll
        for (int x = 0; x < kLoads; ++x) {
            const int i = i0 + (rank * kLoads + x) * kTogether + slot;
            to[x] = nullptr;
            if (from[x] < 0) continue;
            const int here = page_of(from[x]), there = page_of(i);
            if (here < 0 || there < 0) continue;
            v[x] = *piece_at(here, from[x]);
            to[x] = piece_at(there, i);
            if (piece == 0) w[x] = *weight_at(here, from[x]);
        }
        Ctas::sync();
#pragma unroll
        for (int x = 0; x < kLoads; ++x) {
            if (!to[x]) continue;
            const int i = i0 + (rank * kLoads + x) * kTogether + slot;
            *to[x] = v[x];
            if (piece == 0) *weight_at(page_of(i), i) = w[x];
        }
    }
}

template <int kDim>
cudaError_t launch_evict(const EvictArgs& a, cudaStream_t stream) {
    const int64_t rows = static_cast<int64_t>(a.requests) * a.cache.heads;
    const int64_t most = std::min<int64_t>(static_cast<int64_t>(a.table_width) << a.cache.page_shift, INT32_MAX);
    int ranks = 1;
    while (ranks < kMaxCluster && rows * ranks < a.sms && most > 2048 * ranks) ranks *= 2;
    constexpr int kRoom = (kMaxSmem - static_cast<int>(sizeof(topk::Shared))) / 4;
    const int room = static_cast<int>(std::min<int64_t>((most + ranks - 1) / ranks, kRoom));
    const int bytes = static_cast<int>(sizeof(topk::Shared)) + room * 4;
    if (ranks == 1) {
        static SmemOnce once;
        const cudaError_t e = once.set(reinterpret_cast<const void*>(kv_evict_kernel<kDim, topk::One>), kMaxSmem);
        if (e != cudaSuccess) return e;
        kv_evict_kernel<kDim, topk::One><<<static_cast<unsigned>(rows), kThreads, bytes, stream>>>(a, room);
        return cudaGetLastError();
    }
    static SmemOnce once;
    const cudaError_t e = once.set(reinterpret_cast<const void*>(kv_evict_kernel<kDim, topk::Cluster>), kMaxSmem);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(rows * ranks));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = bytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(ranks);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kv_evict_kernel<kDim, topk::Cluster>, a, room);
}

}  // namespace

cudaError_t launch_kv_evict(const EvictArgs& a, cudaStream_t stream) {
    return a.cache.dim == 64 ? launch_evict<64>(a, stream) : a.cache.dim == 96 ? launch_evict<96>(a, stream) : launch_evict<128>(a, stream);
}

}  // namespace fg
