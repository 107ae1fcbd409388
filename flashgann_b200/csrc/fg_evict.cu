// fg_evict.cu -- eviction from the cache by accumulated weight.
//
// Of a request of `len` positions that are more than the budget, each kv head
// keeps the first `sinks`, the last `recent` and, of those between, the heaviest
// budget - sinks - recent (of equal weights the lowest position; NaN counts as
// -inf).  In ascending order they move to positions 0 .. budget - 1: rows of K and
// V and the weights, in place.
//
// A CTA, or a cluster where there are few, has one request and kv head.  Its
// weights are read once, as keys of fg_topk.cuh (those beyond shared memory's room
// are read again), the kept positions go to the result, and then the rows move,
// kChunk consecutive places for each CTA at a time: K and V rows come by 16-byte
// cp.async into a ring of kStages chunks, and when all CTAs have a chunk they store
// it.  Place i is filled from kept[i] >= i, and the sources of later chunks lie
// behind the chunk, so loads may run ahead of stores as far as they like.  Where
// rows come from and go to is looked up three chunks before, a step to each, by a
// thread to a row, which moves the row's weight too.
//
// What bounds it: the weights' way and, of the rows that move, there and back.
// 32 requests of 900 to 8000 positions to 1024, 8 kv heads of 128, 94 % of the rows
// move, 258 MB: 74 us from memory, 60 where three sets of inputs take turns in L2,
// of which the selection takes about 10.
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

constexpr int kThreads = 512;
constexpr int kMaxCluster = 8;
constexpr int kMaxSmem = 110 * 1024;  // two CTAs to an SM
constexpr int kChunk = 64;            // rows
constexpr int kStages = 3;            // of chunks (registers instead, a chunk after the other: 93 us for 72)

template <int kDim>
struct Ring {
    static constexpr int kRow = 4 * kDim;  // bytes of K and V
    static constexpr int kBytes = kStages * kChunk * kRow;
};
// Where the rows of chunks begin, from and to (elements of the cache's halves; from below 0: it stays), and their weights.
struct Moves {
    int64_t from[kStages + 1][kChunk], to[kStages + 1][kChunk];
    float w[kStages + 1][kChunk];
    float* w_to[kStages + 1][kChunk];
};

template <int kDim, typename Ctas>
__global__ void __launch_bounds__(kThreads, 2) kv_evict_kernel(const EvictArgs a, int room) {
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
#pragma unroll 8
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

    // the ring and the moves lie where the keys were
    const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(smem));
    Moves& mv = *reinterpret_cast<Moves*>(smem + Ring<kDim>::kBytes);
    // a thread has one 16-byte piece of K or V of several rows
    constexpr int kPieces = 2 * kDim / 8, kTogether = kThreads / kPieces, kEach = (kChunk + kTogether - 1) / kTogether;
    const int piece = tid % kPieces, slot = tid < kTogether * kPieces ? tid / kPieces : kChunk;
    const bool values = piece >= kPieces / 2;
    char* base = static_cast<char*>(values ? a.v : const_cast<void*>(a.cache.k)) +
                 2 * (head * a.cache.head_stride + (values ? piece - kPieces / 2 : piece) * 8);
    const int first = a.sinks, chunks = (a.budget - first + ranks * kChunk - 1) / (ranks * kChunk);
    const auto place = [&](int c) { return first + (c * ranks + rank) * kChunk + tid; };  // of this thread's row of chunk c

    // a row's way: the position it is at (two chunks before its loads), both pages (one before), its offsets and weight
    int from2 = -1, from1 = -1, here1 = -1, there1 = -1;
    const auto step = [&](int c) {  // offsets of chunk c, pages of c + 1, positions of c + 2
        if (tid >= kChunk) return;
        int64_t from = -1, to = 0;
        float w = 0.f;
        float* w_to = nullptr;
        if (from1 >= 0 && here1 >= 0 && there1 >= 0) {
            const int i = place(c);
            from = here1 * a.cache.page_stride + (from1 & in_page) * a.cache.token_stride;
            to = there1 * a.cache.page_stride + (i & in_page) * a.cache.token_stride;
            w = *weight_at(here1, from1);
            w_to = weight_at(there1, i);
        }
        const int at = c & kStages;  // c % (kStages + 1)
        mv.from[at][tid] = from;
        mv.to[at][tid] = to;
        mv.w[at][tid] = w;
        mv.w_to[at][tid] = w_to;
        from1 = from2;
        const int i1 = place(c + 1), i2 = place(c + 2);
        if (from1 == i1) from1 = -1;  // in place already
        here1 = from1 >= 0 ? page_of(from1) : -1;
        there1 = from1 >= 0 ? page_of(i1) : -1;
        from2 = c + 2 < chunks && i2 < a.budget ? __ldcg(kept + i2) : -1;
    };
    static_assert((kStages & (kStages + 1)) == 0, "c & kStages");
    const auto load = [&](int c) {
        if (c < chunks)
#pragma unroll
            for (int x = 0; x < kEach; ++x) {
                const int row = slot + x * kTogether;
                if (row >= kChunk) continue;
                const int64_t at = mv.from[c & kStages][row];
                if (at >= 0)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(ring + (c % kStages * kChunk + row) * Ring<kDim>::kRow + piece * 16),
                                 "l"(base + 2 * at)
                                 : "memory");
            }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    __syncthreads();  // the keys are done with
    step(-2);
    step(-1);
    for (int c = 0; c < kStages; ++c) step(c);
    __syncthreads();
    for (int c = 0; c < kStages - 1; ++c) load(c);
    for (int c = 0; c < chunks; ++c) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
        Ctas::sync();  // all have the chunk; the one before is stored
        load(c + kStages - 1);
#pragma unroll
        for (int x = 0; x < kEach; ++x) {
            const int row = slot + x * kTogether;
            if (row >= kChunk || mv.from[c & kStages][row] < 0) continue;
            uint4 v;
            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                         : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                         : "r"(ring + (c % kStages * kChunk + row) * Ring<kDim>::kRow + piece * 16)
                         : "memory");
            *reinterpret_cast<uint4*>(base + 2 * mv.to[c & kStages][row]) = v;
        }
        if (tid < kChunk && mv.w_to[c & kStages][tid]) *mv.w_to[c & kStages][tid] = mv.w[c & kStages][tid];
        step(c + kStages);  // where chunk c - 1 was
    }
}

// CTAs to a row, by what its table holds at most (a row's length is not known here): one for up to 640 positions, four for up
// to 2048, then as many as there are SMs for.  us with 8 kv heads of 128 of one request, few rows move / all move.  (Over this,
// 2 heads of 64, and four requests of 8 heads of 96, four CTAs take 1.06 of one's time at 480 and 520 positions, 1.01 at 640,
// 0.98 at 670 and 740, 0.93 at 800.)
//     positions    1             4             8
//     480          9.9 / 13.2    10.2 / 13.0   11.4 / 14.5
//     640          11.2 / 15.9   11.2 / 14.8   11.9 / 16.5
//     800          12.2 / 16.1   11.5 / 13.8   12.3 / 17.2
//     1100         15.1 / 21.6   12.3 / 16.0   12.2 / 17.5
//     1800         16.3 / 26.1   13.7 / 19.1   13.2 / 19.4
//     2200         25.3 / 39.2   18.2 / 23.0   17.8 / 20.1
//     16000        42.1 / 69.0   23.8 / 33.7   20.1 / 27.6
// Two CTAs pay for the cluster and gain little: 64 rows, one / two, 800 positions 12.5 / 14.7 (all move 19.3 / 20.5), 1100 15.5
// / 17.4 (26.9 / 27.5), 2200 25.6 / 27.0 (57 / 48), 4000 34.7 / 34.8 (87 / 70).  More CTAs than SMs: 32 rows of 1100 positions
// 18.1 with four CTAs, 34.4 with eight.
constexpr int kOneCta = 640, kFourCtas = 2048;
int row_ctas(int64_t rows, int64_t most, int sms) {
    if (most <= kOneCta) return 1;
    if (most <= kFourCtas) return rows * 4 <= sms ? 4 : 1;
    int ranks = 1;
    while (ranks < kMaxCluster && rows * ranks * 2 <= sms) ranks *= 2;
    return ranks;
}

template <int kDim>
cudaError_t launch_evict(const EvictArgs& a, cudaStream_t stream) {
    const int64_t rows = static_cast<int64_t>(a.requests) * a.cache.heads;
    const int64_t most = std::min<int64_t>(static_cast<int64_t>(a.table_width) << a.cache.page_shift, INT32_MAX);
    const int ranks = row_ctas(rows, most, a.sms);
    constexpr int kRoom = (kMaxSmem - static_cast<int>(sizeof(topk::Shared))) / 4;
    const int room = static_cast<int>(std::min<int64_t>((most + ranks - 1) / ranks, kRoom));
    static_assert(Ring<128>::kBytes + sizeof(Moves) <= kMaxSmem && (kMaxSmem + 1024) * 2 <= 228 * 1024, "two CTAs to an SM");
    const int bytes = std::max(static_cast<int>(sizeof(topk::Shared)) + room * 4, Ring<kDim>::kBytes + static_cast<int>(sizeof(Moves)));
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
