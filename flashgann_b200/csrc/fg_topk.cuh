// fg_topk.cuh -- the largest of many keys, by a CTA or a cluster of them.
//
// The keys of one row (the scores of a context's pages, the weights of a
// context's positions) are spread over the CTAs of a cluster, each of which
// holds a contiguous run of them.  threshold() finds the key of which `want`
// are at least as large.  Keys of one row agree in their first bits (scores of
// about the same size have the same exponent), so it begins where the largest
// and the smallest first differ and takes 11 bits from there: every CTA counts
// its keys by those in shared memory, all of them read one another's counts, and
// all come to the same bits.  Of the few keys that begin with them, up to 32
// are compared with one another by a warp; more are counted by the next bits.
// emit() then walks the keys in order and hands out places in the result, so
// that it is ascending in position and ties go to the lowest one.  Counts are
// whole numbers: the result does not depend on the order of the atomics.
//
// (8 bits at a time from the first bit on: four rounds, in the first of which all
// keys fall on a few counts and wait for one another; 64 x 8 rows of 560 keys 28
// us with their scores.)
#pragma once

#include <cstdint>

#include <cooperative_groups.h>
#include <cuda_runtime.h>

namespace fg {
namespace topk {

namespace cg = cooperative_groups;

constexpr uint32_t kNone = 0;  // the key of what is not there: below that of every number

// Larger for larger numbers; -0 as 0.  NaN has no place of its own: see the callers.
__device__ __forceinline__ uint32_t order_key(float f) {
    const uint32_t u = __float_as_uint(f + 0.f);
    return u ^ (static_cast<int32_t>(u) < 0 ? 0xFFFFFFFFu : 0x80000000u);
}

constexpr int kList = 32;
// Bits of a digit: a few thousand keys spread well enough over 256 counts, more want 2048.
constexpr int kMostBins = 2048;
__host__ __device__ constexpr int bits_of(int threads) { return threads >= 512 ? 11 : 8; }

struct alignas(16) Shared {  // what callers lay behind it is read 16 bytes at a time
    int hist[kMostBins];
    uint32_t list[kList];     // keys of the last digit, of this CTA
    int listed;
    int warp_a[32], warp_b[32];
    uint32_t least, most;     // of this CTA's keys
    int digit, left, count;
    uint32_t key;
    int above, equal;         // of this CTA, for the others
};

// Taken are the keys above `key` and, in order of position, the first `ties` that equal it.
struct Threshold {
    uint32_t key;
    int ties;
};

// The CTAs that share a row: one, or a cluster.
struct One {
    static constexpr int kMost = 1;
    __device__ static __forceinline__ int ranks() { return 1; }
    __device__ static __forceinline__ int rank() { return 0; }
    __device__ static __forceinline__ void sync() { __syncthreads(); }
    template <typename X>
    __device__ static __forceinline__ const X* at(const X* p, int) { return p; }
};
struct Cluster {
    static constexpr int kMost = 16;
    __device__ static __forceinline__ int ranks() { return static_cast<int>(cg::this_cluster().num_blocks()); }
    __device__ static __forceinline__ int rank() { return static_cast<int>(cg::this_cluster().block_rank()); }
    __device__ static __forceinline__ void sync() { cg::this_cluster().sync(); }
    template <typename X>
    __device__ static __forceinline__ const X* at(const X* p, int rank) { return cg::this_cluster().map_shared_rank(p, rank); }
};

// kThreads in all of the following: the CTA's.

// Before the first key is made; a barrier of the CTA has to come between this and threshold().
template <int kThreads>
__device__ __forceinline__ void clear(Shared& s) {
    constexpr int kBins = 1 << bits_of(kThreads);
    for (int x = threadIdx.x; x < kBins / 4; x += kThreads) reinterpret_cast<int4*>(s.hist)[x] = make_int4(0, 0, 0, 0);
    if (threadIdx.x == 0) {
        s.least = 0xFFFFFFFFu;
        s.most = 0;
        s.listed = 0;
    }
}
// The keys that a thread made (or none: least 0xFFFFFFFF, most 0).  By all threads, before a barrier of the CTAs and
// threshold().
__device__ __forceinline__ void range(Shared& s, uint32_t least, uint32_t most) {
    least = __reduce_min_sync(0xFFFFFFFFu, least);
    most = __reduce_max_sync(0xFFFFFFFFu, most);
    if ((threadIdx.x & 31) == 0) {
        atomicMin(&s.least, least);
        atomicMax(&s.most, most);
    }
}

// The sum of the counts of the warps before this one, and of all.
template <int kThreads>
__device__ __forceinline__ int lower_warps(const int* counts, int* all = nullptr) {
    const int lane = threadIdx.x & 31, c = lane < kThreads / 32 ? counts[lane] : 0;
    if (all) *all = __reduce_add_sync(0xFFFFFFFFu, c);
    return __reduce_add_sync(0xFFFFFFFFu, lane < static_cast<int>(threadIdx.x >> 5) ? c : 0);
}

// This CTA's keys.  Warp w has the keys [w * per, w * per + per) of the n, 32 at a time, in all passes; held: those in
// registers, of all a warp's turns (the caller sees to n <= kHeld * kThreads), else read(i) is asked each time.
template <int kThreads>
struct Segment {
    int first, last;
    __device__ __forceinline__ explicit Segment(int n) {
        const int per = (n + kThreads - 1) / kThreads * 32;
        first = min(n, static_cast<int>(threadIdx.x >> 5) * per);
        last = min(n, first + per);
    }
};
template <int kThreads, int kHeld>
struct HeldKeys {
    uint32_t k[kHeld];
    // f(key, i) for each turn of the warp, by all its lanes; i below 0 and no key past the end
    template <typename F>
    __device__ __forceinline__ void each(int n, F f) const {
        const Segment<kThreads> g(n);
#pragma unroll
        for (int x = 0; x < kHeld; ++x)
            if (g.first + 32 * x < g.last) {
                const int i = g.first + 32 * x + static_cast<int>(threadIdx.x & 31);
                f(i < g.last ? k[x] : kNone, i < g.last ? i : -1);
            }
    }
};
template <int kThreads, typename Read>
struct ReadKeys {
    Read read;
    template <typename F>
    __device__ __forceinline__ void each(int n, F f) const {
        const Segment<kThreads> g(n);
#pragma unroll 4
        for (int i0 = g.first; i0 < g.last; i0 += 32) {
            const int i = i0 + static_cast<int>(threadIdx.x & 31);
            f(i < g.last ? read(i) : kNone, i < g.last ? i : -1);
        }
    }
};
template <int kThreads, typename Read>
__device__ __forceinline__ ReadKeys<kThreads, Read> read_keys(Read read) {
    return {read};
}

// keys: this CTA's n, of which clear() and range() know, after Ctas::sync().  The CTAs hold more than
// `want` >= 0 of them.
template <int kThreads, typename Ctas, typename Keys>
__device__ __forceinline__ Threshold threshold(Shared& s, int n, int want, const Keys& keys) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, ranks = Ctas::ranks();
    constexpr int kBits = bits_of(kThreads), kBins = 1 << kBits;
    if (want == 0) return {0xFFFFFFFFu, 0};
    // of all CTAs: a lane to each, whose reads of the others' memory are under way together (one after the other they take
    // 0.15 us each)
    uint32_t least = s.least, most = s.most;
    if (ranks > 1) {
        const int r = min(lane, ranks - 1);
        least = __reduce_min_sync(0xFFFFFFFFu, *Ctas::at(&s.least, r));
        most = __reduce_max_sync(0xFFFFFFFFu, *Ctas::at(&s.most, r));
    }
    // bits from `high` on are the same in all keys
    int high = least == most ? 0 : 32 - __clz(least ^ most), left = want;
    if (high == 0) return {most, most == kNone ? 0 : left};
    uint32_t prefix = high == 32 ? 0u : most >> high << high;
    while (true) {
        const int shift = max(0, high - kBits);
        const uint32_t above = high == 32 ? 0u : 0xFFFFFFFFu << high;  // the bits that are known
        keys.each(n, [&](uint32_t k, int i) {
            if (i >= 0 && ((k ^ prefix) & above) == 0) atomicAdd(&s.hist[(k >> shift) & (kBins - 1)], 1);
        });
        Ctas::sync();
        // thread t has the counts of kEach digits, the largest digits first
        constexpr int kEach = kBins / kThreads;
        static_assert(kEach == 1 || kEach == 2 || kEach % 4 == 0, "reads of 4, 8 or 16 bytes");
        int c[kEach] = {}, sum = 0;
        const int base = kBins - kEach * (tid + 1);
        constexpr int kTogether = Ctas::kMost < 4 ? Ctas::kMost : 4;
        for (int r0 = 0; r0 < ranks; r0 += kTogether) {
            int part[kTogether][kEach];
#pragma unroll
            for (int r = 0; r < kTogether; ++r) {
                const int* h = Ctas::at(s.hist + base, min(r0 + r, ranks - 1));
                if constexpr (kEach == 1) {
                    part[r][0] = *h;
                } else if constexpr (kEach == 2) {
                    const int2 v = *reinterpret_cast<const int2*>(h);
                    part[r][0] = v.x, part[r][1] = v.y;
                } else {
#pragma unroll
                    for (int x = 0; x < kEach; x += 4) {
                        const int4 v = *reinterpret_cast<const int4*>(h + x);
                        part[r][x] = v.x, part[r][x + 1] = v.y, part[r][x + 2] = v.z, part[r][x + 3] = v.w;
                    }
                }
            }
#pragma unroll
            for (int r = 0; r < kTogether; ++r)
                if (r0 + r < ranks)
#pragma unroll
                    for (int x = 0; x < kEach; ++x) c[x] += part[r][kEach - 1 - x];
        }
#pragma unroll
        for (int x = 0; x < kEach; ++x) sum += c[x];
        int upto = sum;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int v = __shfl_up_sync(0xFFFFFFFFu, upto, d);
            if (lane >= d) upto += v;
        }
        if (lane == 31) s.warp_a[warp] = upto;
        __syncthreads();
        upto += lower_warps<kThreads>(s.warp_a);
        if (upto >= left && upto - sum < left) {
            int rest = left - (upto - sum);
#pragma unroll
            for (int x = 0; x < kEach; ++x) {
                if (rest > 0 && rest <= c[x]) {
                    s.digit = base + kEach - 1 - x;
                    s.left = rest;
                    s.count = c[x];
                }
                rest -= c[x];
            }
        }
        __syncthreads();
        prefix |= static_cast<uint32_t>(s.digit) << shift;
        left = s.left;
        const int count = s.count;
        if (count == left) return {prefix ? prefix - 1 : kNone, 0};  // all that begin like this
        if (shift == 0) return {prefix, prefix == kNone ? 0 : left};
        high = shift;
        const uint32_t known = 0xFFFFFFFFu << high;
        if (count <= kList) {
            // the keys that are left, compared with one another
            keys.each(n, [&](uint32_t k, int i) {
                if (i >= 0 && ((k ^ prefix) & known) == 0) s.list[atomicAdd(&s.listed, 1)] = k;
            });
            Ctas::sync();
            if (warp == 0) {
                // lane x has the x-th of all CTAs' lists
                const int m = lane < ranks ? *Ctas::at(&s.listed, lane) : 0;
                int from = 0, at = 0;
                for (int r = 0, before = 0; r < ranks; ++r) {
                    const int n_r = __shfl_sync(0xFFFFFFFFu, m, r);
                    if (lane >= before && lane < before + n_r) {
                        from = r;
                        at = lane - before;
                    }
                    before += n_r;
                }
                const uint32_t mine = lane < count ? Ctas::at(s.list, from)[at] : 0;
                int more = 0, as_many = 0;
                for (int x = 0; x < count; ++x) {
                    const uint32_t k = __shfl_sync(0xFFFFFFFFu, mine, x);
                    more += k > mine;
                    as_many += k >= mine;
                }
                if (lane < count && more < left && as_many >= left) {  // all lanes that write have the same key
                    s.key = mine;
                    s.left = left - more;
                }
            }
            __syncthreads();
            return {s.key, s.key == kNone ? 0 : s.left};
        }
        Ctas::sync();  // the counts are read before they are cleared
        for (int x = tid; x < kBins / 4; x += kThreads) reinterpret_cast<int4*>(s.hist)[x] = make_int4(0, 0, 0, 0);
        __syncthreads();
    }
}

// put(place, i) for each key taken, places ascending over the CTAs and i.  Returns how many all CTAs took.  The caller sees
// to a Ctas::sync() before a CTA of a cluster ends.
template <int kThreads, typename Ctas, typename Keys, typename Put>
__device__ __forceinline__ int emit(Shared& s, int n, Threshold thr, const Keys& keys, Put put) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int above = 0, equal = 0;
    keys.each(n, [&](uint32_t k, int) {
        above += __popc(__ballot_sync(0xFFFFFFFFu, k > thr.key));
        if (thr.ties) equal += __popc(__ballot_sync(0xFFFFFFFFu, k == thr.key));
    });
    if (lane == 0) {
        s.warp_a[warp] = above;
        s.warp_b[warp] = equal;
    }
    __syncthreads();
    int all_above = 0, all_equal = 0;
    int before_above = lower_warps<kThreads>(s.warp_a, &all_above), before_equal = lower_warps<kThreads>(s.warp_b, &all_equal);
    if (tid == 0) {
        s.above = all_above;
        s.equal = all_equal;
    }
    Ctas::sync();
    if (Ctas::ranks() > 1) {
        const bool is = lane < Ctas::ranks(), lower = lane < Ctas::rank();
        const int a = is ? *Ctas::at(&s.above, lane) : 0, e = is ? *Ctas::at(&s.equal, lane) : 0;
        all_above = __reduce_add_sync(0xFFFFFFFFu, a);
        all_equal = __reduce_add_sync(0xFFFFFFFFu, e);
        before_above += __reduce_add_sync(0xFFFFFFFFu, lower ? a : 0);
        before_equal += __reduce_add_sync(0xFFFFFFFFu, lower ? e : 0);
    }
    keys.each(n, [&](uint32_t k, int i) {
        const uint32_t a = __ballot_sync(0xFFFFFFFFu, k > thr.key), e = thr.ties ? __ballot_sync(0xFFFFFFFFu, k == thr.key) : 0u;
        const uint32_t lower = (1u << lane) - 1;
        const int ties_before = before_equal + __popc(e & lower);
        if (k > thr.key || (thr.ties && k == thr.key && ties_before < thr.ties))
            put(before_above + __popc(a & lower) + min(ties_before, thr.ties), i);
        before_above += __popc(a);
        before_equal += __popc(e);
    });
    return all_above + min(all_equal, thr.ties);
}

}  // namespace topk
}  // namespace fg
