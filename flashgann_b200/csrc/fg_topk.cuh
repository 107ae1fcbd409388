// fg_topk.cuh -- the largest of many keys, by a cluster of CTAs.
//
// The keys of one row (the scores of a context's pages, the weights of a
// context's positions) are spread over the CTAs of a cluster, each of which
// holds a contiguous run of them.  threshold() finds the key of which `want`
// are at least as large, a digit of 8 bits at a time: every CTA counts its
// keys' digits in shared memory, all of them read one another's counts, and
// all come to the same digit.  emit() then walks the keys in order and hands
// out places in the result, so that it is ascending in position and ties go to
// the lowest one.  Counts are whole numbers: the result does not depend on the
// order of the atomics.
#pragma once

#include <cstdint>

#include <cooperative_groups.h>
#include <cuda_runtime.h>

namespace fg {
namespace topk {

namespace cg = cooperative_groups;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr uint32_t kNone = 0;  // the key of what is not there: below that of every number

// Larger for larger numbers; -0 as 0.  NaN has no place of its own: see the callers.
__device__ __forceinline__ uint32_t order_key(float f) {
    const uint32_t u = __float_as_uint(f + 0.f);
    return u ^ (static_cast<int32_t>(u) < 0 ? 0xFFFFFFFFu : 0x80000000u);
}

struct alignas(16) Shared {  // what callers lay behind it is read 16 bytes at a time
    int hist[4][256];
    int warp_a[kWarps], warp_b[kWarps];
    int digit, left, count;
    int above, equal;  // of this CTA, for the others
};

// Taken are the keys above `key` and, in order of position, the first `ties` that equal it.
struct Threshold {
    uint32_t key;
    int ties;
};

// keys(i), 0 <= i < n: this CTA's.  The cluster holds more than `want` >= 0 of them.
template <typename Keys>
__device__ __forceinline__ Threshold threshold(const cg::cluster_group& cluster, Shared& s, int n, int want, Keys keys) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (want == 0) return {0xFFFFFFFFu, 0};
    for (int x = tid; x < 4 * 256; x += kThreads) (&s.hist[0][0])[x] = 0;
    __syncthreads();
    uint32_t prefix = 0, mask = 0;
    int left = want;
    for (int pass = 0; pass < 4; ++pass) {
        const int shift = 24 - 8 * pass;
        for (int i = tid; i < n; i += kThreads) {
            const uint32_t k = keys(i);
            if (((k ^ prefix) & mask) == 0) atomicAdd(&s.hist[pass][(k >> shift) & 255], 1);
        }
        cluster.sync();
        const int bin = 255 - tid;  // largest digit first
        int c = 0;
        for (unsigned r = 0; r < cluster.num_blocks(); ++r) c += cluster.map_shared_rank(&s.hist[pass][0], r)[bin];
        int sum = c;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int v = __shfl_up_sync(0xFFFFFFFFu, sum, d);
            if (lane >= d) sum += v;
        }
        if (lane == 31) s.warp_a[warp] = sum;
        __syncthreads();
        for (int w = 0; w < warp; ++w) sum += s.warp_a[w];
        if (sum >= left && sum - c < left) {
            s.digit = bin;
            s.left = left - (sum - c);
            s.count = c;
        }
        __syncthreads();
        prefix |= static_cast<uint32_t>(s.digit) << shift;
        mask |= 255u << shift;
        left = s.left;
        if (s.count == left) return {prefix ? prefix - 1 : kNone, 0};  // all that begin like this
    }
    return {prefix, prefix == kNone ? 0 : left};
}

// put(place, i) for each key taken, places ascending over the cluster's CTAs and i.  Returns how many the cluster took.
// The caller sees to a cluster.sync() before the CTA ends.
template <typename Keys, typename Put>
__device__ __forceinline__ int emit(const cg::cluster_group& cluster, Shared& s, int n, Threshold thr, Keys keys, Put put) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per = (n + kThreads - 1) / kThreads * 32;  // keys of a warp
    const int i0 = warp * per, i1 = min(n, i0 + per);
    int above = 0, equal = 0;
    for (int i = i0; i < i1; i += 32) {
        const uint32_t k = i + lane < i1 ? keys(i + lane) : kNone;
        above += __popc(__ballot_sync(0xFFFFFFFFu, k > thr.key));
        if (thr.ties) equal += __popc(__ballot_sync(0xFFFFFFFFu, k == thr.key));
    }
    if (lane == 0) {
        s.warp_a[warp] = above;
        s.warp_b[warp] = equal;
    }
    __syncthreads();
    int before_above = 0, before_equal = 0, all_above = 0, all_equal = 0;
    for (int w = 0; w < kWarps; ++w) {
        const int a = s.warp_a[w], e = s.warp_b[w];
        if (w < warp) {
            before_above += a;
            before_equal += e;
        }
        all_above += a;
        all_equal += e;
    }
    if (tid == 0) {
        s.above = all_above;
        s.equal = all_equal;
    }
    cluster.sync();
    all_above = all_equal = 0;
    for (unsigned r = 0; r < cluster.num_blocks(); ++r) {
        const int a = *cluster.map_shared_rank(&s.above, r), e = *cluster.map_shared_rank(&s.equal, r);
        if (r < cluster.block_rank()) {
            before_above += a;
            before_equal += e;
        }
        all_above += a;
        all_equal += e;
    }
    for (int i = i0; i < i1; i += 32) {
        const uint32_t k = i + lane < i1 ? keys(i + lane) : kNone;
        const uint32_t a = __ballot_sync(0xFFFFFFFFu, k > thr.key), e = thr.ties ? __ballot_sync(0xFFFFFFFFu, k == thr.key) : 0u;
        const uint32_t lower = (1u << lane) - 1;
        const int ties_before = before_equal + __popc(e & lower);
        if (k > thr.key || (thr.ties && k == thr.key && ties_before < thr.ties))
            put(before_above + __popc(a & lower) + min(ties_before, thr.ties), i + lane);
        before_above += __popc(a);
        before_equal += __popc(e);
    }
    return all_above + min(all_equal, thr.ties);
}

}  // namespace topk
}  // namespace fg
