// fg_blocks.cu -- which pages of a long context a query attends to: a summary
// of each page's keys, and the choice of the pages whose bound on the scores is
// highest.
#include <algorithm>
#include <cmath>
#include <cstdint>

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "fg_cache.h"
#include "fg_internal.h"
#include "fg_tcgen05.cuh"
#include "fg_topk.cuh"

namespace fg {
namespace {

template <typename T>
struct Pair;
template <>
struct Pair<__half> {
    using V = __half2;
    static constexpr uint32_t kInf = 0x7C007C00u;
    __device__ static __forceinline__ float2 floats(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
};
template <>
struct Pair<__nv_bfloat16> {
    using V = __nv_bfloat162;
    static constexpr uint32_t kInf = 0x7F807F80u;
    __device__ static __forceinline__ float2 floats(uint32_t v) {
        return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
    }
};

// The larger and smaller of two pairs; NaN where either is.
template <typename T>
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
    using V = typename Pair<T>::V;
    const V m = __hmax2_nan(*reinterpret_cast<const V*>(&a), *reinterpret_cast<const V*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
}
template <typename T>
__device__ __forceinline__ uint32_t smaller(uint32_t a, uint32_t b) {
    using V = typename Pair<T>::V;
    const V m = __hmin2_nan(*reinterpret_cast<const V*>(&a), *reinterpret_cast<const V*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
}

// x in 127ths of top (|x| <= top, finite, top > 0), before it is rounded to a
// whole number.  The product and top / 128 are exact (16-bit x and top, with
// room down to their subnormals), and the quotient of two numbers of 11 bits is
// either a whole number or half of one, or further from the next than a 32-bit
// quotient is rounded: rounding it up, down or to the nearest gives what the
// exact quotient gives.
__device__ __forceinline__ float in_127ths(float x, float top) { return __fdiv_rn(x * (127.f / 128.f), top * (1.f / 128.f)); }

// in_127ths rounded to the nearest whole number, given scale = 127 / top rounded: a product is off by 2^-15, so that only
// those that come within 2^-13 of the middle between two whole numbers need the quotient itself.
__device__ __forceinline__ int nearest_127th(float x, float top, float scale) {
    const float y = x * scale;
    float n = rintf(y);
    if (!(fabsf(fabsf(y - n) - 0.5f) >= 0x1p-13f)) n = rintf(in_127ths(x, top));
    return static_cast<int>(n);
}

constexpr float k127th = 1.f / 127.f;  // a product, rounded once: what a quotient would give but for its last bit

__device__ __forceinline__ int clamped(const int32_t* p, int most) { return max(0, min(__ldg(p), most)); }

// Places [lo, lo + n), the first of which that is past something is looked for: in 32 runs of them at once.
struct Span {
    int lo, n;
    __host__ __device__ __forceinline__ int run() const { return (n + 31) / 32; }
    // whether run x ends with a place that is past, or with the last place of all or behind it: of such runs the first has
    // places, and if none is past, the last place
    template <typename Past>
    __host__ __device__ __forceinline__ bool ends(int x, const Past& past) const {
        const int at = lo + (x + 1) * run() - 1;
        return at >= lo + n - 1 || past(at);
    }
    __host__ __device__ __forceinline__ void take(int x) {
        const int first = x * run();
        n = n - first < run() ? n - first : run();
        lo += first;
    }
};

// The first of n ascending places that is past something, or the last: 32 at a time, by whole warps.
template <typename Past>
__device__ __forceinline__ int first_past(int n, const Past& past) {
    Span s = {0, n};
    while (s.n > 1) {
        const uint32_t is = __ballot_sync(0xFFFFFFFFu, s.ends(threadIdx.x & 31, past));  // never 0: run 31 ends behind n - 2
        s.take(__ffs(is) - 1);
    }
    return s.lo;
}

// ---- summary ----
//
// Of the keys k_t, 0 <= t < n, of a page and kv head: with hi_d = max_t k_td,
// lo_d = min_t k_td and top = max_d max(|hi_d|, |lo_d|), scale = top / 127 and
// the bounds ceil(hi_d / scale) and floor(lo_d / scale) in 8 bits.  A page with a
// key that is not finite has scale inf.
//
// A warp has one page of one kv head: 16 bytes of a key to a lane, 2 or 4 keys
// at once, minima and maxima in the cache's type (two values to an instruction).
// Pages are found from token rows: those of request b are numbered from
// floor(query_start[b] / page_size) + 2 b on, which leaves room for every page
// that its new tokens can lie in.
constexpr int kSumWarps = 8;

template <typename T, int kDim>
__global__ void __launch_bounds__(kSumWarps * 32) kv_summarize_kernel(const SummarizeArgs a, int64_t items) {
    constexpr int kPieces = kDim / 8, kTogether = 32 / kPieces, kAhead = 8;
    const int lane = threadIdx.x & 31;
    const int64_t w = static_cast<int64_t>(blockIdx.x) * kSumWarps + (threadIdx.x >> 5);
    const int64_t item = w / a.cache.heads;
    const int head = static_cast<int>(w - item * a.cache.heads);
    if (item >= items) return;
    // the last request whose numbers begin at or before this one
    const int shift = a.cache.page_shift;
    const auto first_item = [&](int b) { return static_cast<int64_t>(clamped(a.req.query_start + b, a.req.tokens) >> shift) + 2 * static_cast<int64_t>(b); };
    const int lo = first_past(a.req.requests, [&](int b) { return first_item(b + 1) > item; });
    const int rows = clamped(a.req.query_start + lo + 1, a.req.tokens) - clamped(a.req.query_start + lo, a.req.tokens);
    const int kv_len = max(0, __ldg(a.req.kv_len + lo));
    if (rows <= 0 || kv_len == 0) return;
    const int64_t col = (max(0, kv_len - rows) >> shift) + (item - first_item(lo));
    if (col < 0 || col > ((kv_len - 1) >> shift) || col >= a.req.table_width) return;
    const int page = __ldg(a.req.block_table + lo * a.req.table_stride + col);
    if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(a.cache.pages)) return;
    const int n = static_cast<int>(min(static_cast<int64_t>(1) << shift, kv_len - (col << shift)));

    const int piece = lane % kPieces, part = lane / kPieces;
    const T* src = static_cast<const T*>(a.cache.k) + page * a.cache.page_stride + head * a.cache.head_stride + piece * 8;
    uint32_t up[4], down[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        up[e] = Pair<T>::kInf | 0x80008000u;
        down[e] = Pair<T>::kInf;
    }
    if (part < kTogether) {
        for (int t0 = part; t0 < n; t0 += kTogether * kAhead) {
            uint4 v[kAhead];
#pragma unroll
            for (int x = 0; x < kAhead; ++x) {
                const int t = min(t0 + x * kTogether, n - 1);  // the last key again, past the end
                v[x] = __ldg(reinterpret_cast<const uint4*>(src + t * a.cache.token_stride));
            }
#pragma unroll
            for (int x = 0; x < kAhead; ++x) {
                const uint32_t e4[4] = {v[x].x, v[x].y, v[x].z, v[x].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    up[e] = larger<T>(up[e], e4[e]);
                    down[e] = smaller<T>(down[e], e4[e]);
                }
            }
        }
    }
#pragma unroll
    for (int x = 1; x < kTogether; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            // every lane takes part; only the first kPieces have use for it
            up[e] = larger<T>(up[e], __shfl_sync(0xFFFFFFFFu, up[e], (piece + x * kPieces) & 31));
            down[e] = smaller<T>(down[e], __shfl_sync(0xFFFFFFFFu, down[e], (piece + x * kPieces) & 31));
        }
    float h[8], l[8], top = 0.f;
    bool fine = true;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float2 u = Pair<T>::floats(up[e]), d = Pair<T>::floats(down[e]);
        h[2 * e] = u.x;
        h[2 * e + 1] = u.y;
        l[2 * e] = d.x;
        l[2 * e + 1] = d.y;
    }
    if (part == 0) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            fine = fine && isfinite(h[e]) && isfinite(l[e]);
            top = fmaxf(top, fmaxf(fabsf(h[e]), fabsf(l[e])));
        }
    }
    fine = __all_sync(0xFFFFFFFFu, fine);
#pragma unroll
    for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
    if (part == 0) {
        uint32_t words[4] = {0, 0, 0, 0};  // 8 lower bounds, 8 upper ones
        if (fine && top > 0.f) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                int low = static_cast<int>(floorf(in_127ths(l[e], top))), high = static_cast<int>(ceilf(in_127ths(h[e], top)));
                if (l[e] < 0.f) low = min(low, -1);  // the quotient may be below the least number
                if (h[e] > 0.f) high = max(high, 1);
                words[e / 4] |= static_cast<uint32_t>(low & 255) << (8 * (e % 4));
                words[2 + e / 4] |= static_cast<uint32_t>(high & 255) << (8 * (e % 4));
            }
        }
        int8_t* dst = a.summary.bounds + page * a.summary.bounds_page_stride + head * a.summary.bounds_head_stride + piece * 8;
        *reinterpret_cast<uint2*>(dst) = make_uint2(words[0], words[1]);
        *reinterpret_cast<uint2*>(dst + kDim) = make_uint2(words[2], words[3]);
        if (lane == 0) a.summary.scale[page * a.summary.scale_page_stride + head * a.summary.scale_head_stride] = fine ? top * k127th : INFINITY;
    }
}

// ---- selection ----
//
// A query is rounded to 127ths of its largest value like the bounds: Q_d, and
// t = top / 127.  Its score of a page is an upper bound of Q.k t over the page's
// keys, in 8-bit arithmetic,
//     I = sum_d Q_d * (Q_d < 0 ? lower_d : upper_d),     score = max_h (I_h t_h) * scale
// over the heads h of the group.  I is a product of (min(Q, 0), max(Q, 0)) with
// the page's 2 * dim bounds as they lie in memory, a whole number below 2^21, and
// two 32-bit roundings follow: every order of summation gives the same score, so
// the choice is the same bit for bit.
//
// Three ways, see kShort.  Few rows (a row: a token's kv head) with few pages: a
// CTA to each, which multiplies in its threads (dp4a), keeps the scores in shared
// memory as keys and finds the largest of them (fg_topk.cuh).  Many rows: a CTA to
// each, which multiplies on the tensor cores (tcgen05 in 8 bits; neither dp4a nor
// mma.sync in 8 bits is one instruction of this GPU).  Few rows with many pages:
// two kernels, of which the first has the pages of a row in many CTAs and leaves
// the keys in the workspace, and the second, started beside the first's end, a CTA
// to each row.
//
// What bounds it: 2 * dim + 4 bytes a page and kv head from memory, which many rows
// read at 2.9 TB/s (64 tokens, 286K pages and heads, 71 MB: 24.5 us): a CTA's start,
// the first pages' way and the selection are as long as the pages' way.  One token
// of 131K positions: 14.2 us.
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
static_assert(sizeof(topk::Shared) % 16 == 0, "the queries behind it are read 16 bytes at a time");

// The pages that a token row chooses from.
struct Row {
    int request, first, n;   // blocks [first, first + n) of the request; n below 0: no request's row
    const int32_t* table;    // of the first of them
};
// The request of a row is the first that ends after it.  In a decode step that is the row's own number, which is tried
// first, with all that is read of it under way together; else it is searched for.  By whole warps.
__device__ __forceinline__ Row row_of(const SelectArgs& a, int token) {
    const Requests& q = a.req;
    int lo = min(token, q.requests - 1);
    int start = clamped(q.query_start + lo, q.tokens), end = clamped(q.query_start + lo + 1, q.tokens), len = __ldg(q.kv_len + lo);
    if (token < start || token >= end) {
        lo = first_past(q.requests, [&](int b) { return clamped(q.query_start + b + 1, q.tokens) > token; });
        start = clamped(q.query_start + lo, q.tokens);
        end = clamped(q.query_start + lo + 1, q.tokens);
        len = __ldg(q.kv_len + lo);
    }
    const int p = max(0, len) - (end - token);
    Row r;
    r.request = lo;
    r.first = a.sinks >> a.page_shift;
    const int last = p >= a.window ? min(((p - a.window) >> a.page_shift) + 1, q.table_width) : 0;
    r.n = token < start || token >= end ? -1 : max(0, last - r.first);
    r.table = q.block_table + lo * q.table_stride + r.first;
    return r;
}
// Page i of them, or -1.  It is read beside what r.n comes from.
__device__ __forceinline__ int page_of(const SelectArgs& a, const Row& r, int i) {
    const int page = i < a.req.table_width - r.first ? __ldg(r.table + i) : -1;
    return i < r.n && static_cast<uint32_t>(page) < static_cast<uint32_t>(a.pages) ? page : -1;
}

// Some query heads of a token in 8 bits (a warp to each): 2 * kDim bytes, those below 0 and those above,
// and their t.
template <typename T, int kDim>
struct Queries {
    const SelectArgs& a;
    const T* q;
    int all;
    __device__ __forceinline__ Queries(const SelectArgs& args, int token, int first, int count)
        : a(args), q(static_cast<const T*>(args.q) + token * args.q_token_stride + first * args.q_head_stride), all(count) {}
    __device__ __forceinline__ uint2 load(int x) const {
        const int lane = threadIdx.x & 31;
        if (x >= all || lane >= kDim / 4) return make_uint2(0, 0);
        return __ldg(reinterpret_cast<const uint2*>(q + x * a.q_head_stride) + lane);
    }
    // warp: its number of `warps`; query: load() of it; put(number, the lane's 4 bytes below 0, those above, t) for each head
    template <typename Put>
    __device__ __forceinline__ void round(int warp, int warps, uint2 query, Put put) const {
        for (int x = warp; x < all; x += warps) {
            const float2 lo = Pair<T>::floats(query.x), hi = Pair<T>::floats(query.y);
            const float v[4] = {lo.x, lo.y, hi.x, hi.y};
            query = load(x + warps);
            float top = 0.f;
            bool fine = true;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                fine = fine && isfinite(v[e]);
                top = fmaxf(top, fabsf(v[e]));
            }
            fine = __all_sync(0xFFFFFFFFu, fine);
            top = __uint_as_float(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(top)));  // none is below 0
            uint32_t below = 0, above = 0;
            if (fine && top > 0.f) {
                const float scale = top > 0x1p-100f ? __fdiv_rn(127.f, top) : NAN;  // NaN: the quotients themselves
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int w = nearest_127th(v[e], top, scale);
                    below |= static_cast<uint32_t>(min(w, 0) & 255) << (8 * e);
                    above |= static_cast<uint32_t>(max(w, 0) & 255) << (8 * e);
                }
            }
            put(x, below, above, fine ? top * k127th : 0.f);
        }
    }
};

// 32 pages of a kv head on their way.  Lanes 4 r to 4 r + 3 load pages r + 8 y; this lane ends with the score of the one of
// them that is its own, y = lane % 4.
constexpr int kTogether = 32;
__device__ __forceinline__ int own_page() { return ((threadIdx.x & 31) >> 2) + 8 * (threadIdx.x & 3); }

template <int kDim>
struct Pages {
    static constexpr int kSteps = 2 * kDim / 64;  // 64 bytes of each
    uint4 v[4][kSteps];
    float scale;
    bool there;
    // page: of own_page()
    __device__ __forceinline__ void load(const SelectArgs& a, int page, int head) {
        const int8_t* base = a.summary.bounds + head * a.summary.bounds_head_stride + (threadIdx.x & 3) * 16;
        there = page >= 0;
#pragma unroll
        for (int y = 0; y < 4; ++y) {
            const int pg = __shfl_sync(0xFFFFFFFFu, page, (threadIdx.x & 28) | y);
            const uint4* src = reinterpret_cast<const uint4*>(base + pg * a.summary.bounds_page_stride);
#pragma unroll
            for (int k = 0; k < kSteps; ++k) v[y][k] = pg >= 0 ? __ldg(src + 4 * k) : make_uint4(0, 0, 0, 0);
        }
        scale = there ? __ldg(a.summary.scale + page * a.summary.scale_page_stride + head * a.summary.scale_head_stride) : 0.f;
    }
    // its score as a key; q8, t_of: the kv head's queries
    __device__ __forceinline__ uint32_t score(const SelectArgs& a, const uint32_t* q8, const float* t_of) const {
        const int4* q4 = reinterpret_cast<const int4*>(q8) + (threadIdx.x & 3);
        float best = -INFINITY;
#pragma unroll 2
        for (int g = 0; g < a.group; ++g) {
            int c[4] = {0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                const int4 b = q4[g * (kDim / 8) + 4 * k];
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    c[y] = __dp4a(static_cast<int>(v[y][k].x), b.x, c[y]);
                    c[y] = __dp4a(static_cast<int>(v[y][k].y), b.y, c[y]);
                    c[y] = __dp4a(static_cast<int>(v[y][k].z), b.z, c[y]);
                    c[y] = __dp4a(static_cast<int>(v[y][k].w), b.w, c[y]);
                }
            }
            // the sum over the 4 lanes, to the lane whose page it is
            const bool odd = threadIdx.x & 1, upper = threadIdx.x & 2;
            const int s0 = (odd ? c[1] : c[0]) + __shfl_xor_sync(0xFFFFFFFFu, odd ? c[0] : c[1], 1);
            const int s1 = (odd ? c[3] : c[2]) + __shfl_xor_sync(0xFFFFFFFFu, odd ? c[2] : c[3], 1);
            const int sum = (upper ? s1 : s0) + __shfl_xor_sync(0xFFFFFFFFu, upper ? s0 : s1, 2);
            best = fmaxf(best, __fmul_rn(static_cast<float>(sum), t_of[g]));
        }
        return there ? topk::order_key(scale == INFINITY ? INFINITY : __fmul_rn(best, scale)) : topk::kNone;
    }
};

// A wait for products that runs out leaves its row's pages without scores.  Their keys say so (order_key gives none between
// kNone and that of -inf), and the whole list is -2 then: a shorter one, or another, would look like a choice.
constexpr uint32_t kLostKey = 1;
constexpr int32_t kLostBlock = -2;
struct Limits {
    int tries, lost;  // of waits; item from which on no products are issued (none: INT32_MAX)
};

// The list of a row whose scores are lost, by all threads.
__device__ __forceinline__ void give_up(const SelectArgs& a, int token, int head) {
    int32_t* out = a.blocks + token * a.blocks_token_stride + head * a.blocks_head_stride;
    for (int x = threadIdx.x; x < a.count; x += static_cast<int>(blockDim.x)) out[x] = kLostBlock;
}

// The largest keys of a row to its place in the result.
template <int kRowThreads, typename Keys>
__device__ __forceinline__ void choose(const SelectArgs& a, topk::Shared& s, const Row& r, int token, int head, topk::Threshold thr, const Keys& keys) {
    int32_t* out = a.blocks + token * a.blocks_token_stride + head * a.blocks_head_stride;
    const int taken = topk::emit<kRowThreads, topk::One>(s, r.n, thr, keys, [&](int place, int i) { out[place] = r.first + i; });
    for (int x = taken + static_cast<int>(threadIdx.x); x < a.count; x += kRowThreads) out[x] = -1;
}

template <typename T, int kDim>
__global__ void __launch_bounds__(kThreads, 3) select_blocks_kernel(const SelectArgs a) {
    extern __shared__ __align__(16) char smem[];
    topk::Shared& s = *reinterpret_cast<topk::Shared*>(smem);
    const int token = static_cast<int>(blockIdx.x) / a.kv_heads, head = static_cast<int>(blockIdx.x) - token * a.kv_heads;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const Queries<T, kDim> queries(a, token, head * a.group, a.group);
    float* t_of = reinterpret_cast<float*>(smem + sizeof(topk::Shared));  // [group]
    uint32_t* q8 = reinterpret_cast<uint32_t*>(t_of + ((queries.all + 3) & ~3));  // [group][2 * kDim bytes]
    uint32_t* keys = q8 + queries.all * (kDim / 2);
    const uint2 query = queries.load(warp);  // beside what follows
    topk::clear<kThreads>(s);
    const Row r = row_of(a, token);
    if (r.n < 0) return;
    topk::Threshold thr = {0, 0};
    if (r.n <= a.count) {
        for (int i = threadIdx.x; i < r.n; i += kThreads) keys[i] = page_of(a, r, i) >= 0 ? 1u : topk::kNone;
        __syncthreads();
    } else {
        int next = page_of(a, r, warp * kTogether + own_page());
        queries.round(warp, kWarps, query, [&](int x, uint32_t below, uint32_t above, float t) {
            if (lane < kDim / 4) {
                q8[x * (kDim / 2) + lane] = below;
                q8[x * (kDim / 2) + kDim / 4 + lane] = above;
            }
            if (lane == 0) t_of[x] = t;
        });
        __syncthreads();
        uint32_t least = 0xFFFFFFFFu, most = 0;
        for (int i0 = warp * kTogether; i0 < r.n; i0 += kWarps * kTogether) {
            Pages<kDim> pages;
            pages.load(a, next, head);
            next = page_of(a, r, i0 + kWarps * kTogether + own_page());
            const uint32_t key = pages.score(a, q8, t_of);
            const int i = i0 + own_page();
            if (i < r.n) {
                keys[i] = key;
                least = min(least, key);
                most = max(most, key);
            }
        }
        topk::range(s, least, most);
        __syncthreads();
        thr = topk::threshold<kThreads, topk::One>(s, r.n, a.count, topk::read_keys<kThreads>([&](int i) { return keys[i]; }));
    }
    choose<kThreads>(a, s, r, token, head, thr, topk::read_keys<kThreads>([&](int i) { return keys[i]; }));
}

constexpr int kPart = 128;       // pages to a CTA of the first of two kernels: the rows of a product
constexpr int kPartThreads = 256;  // half of them load, half have a page's scores each
constexpr int kStages = 3;
constexpr int kTries = 1 << 18;  // of a wait for products; a try that finds nothing takes 4 us: a second

template <int kDim>
struct Tile {
    static constexpr int kPanels = (2 * kDim + 127) / 128;  // 128 bytes of each page
    static constexpr int kPanel = kPart * 128;
    static constexpr int kBytes = kPanels * kPanel;
};
struct Scoring {
    int64_t row[kPart];  // where a page's bounds begin (-1: it is not there)
    uint64_t done[2];
    uint64_t drain;
    uint32_t tmem;
    alignas(16) float t[kStages + 1][32];  // of the queries in work, those before and those that come
};
// Heads of a group in a product's columns, kSlice of them at most at a time; their bytes, panel by panel; what is asked of
// TMEM for two products; shared memory.
constexpr int kSlice = 32;
__host__ __device__ __forceinline__ int columns_of(int group) { return (min(group, kSlice) + 15) & ~15; }
template <int kDim>
__host__ __device__ __forceinline__ int queries_of(int group) { return (Tile<kDim>::kPanels * columns_of(group) * 128 + 1023) & ~1023; }
constexpr int kTmem = 2 * kSlice;
template <int kDim>
int scoring_bytes(int group) {
    return 1024 + kStages * (Tile<kDim>::kBytes + queries_of<kDim>(group)) + static_cast<int>(sizeof(Scoring));
}

// Keys of kPart pages and some kv heads of a token.  An item is a kv head (a slice of its queries, where they are many) with
// its pages.  Pages are lanes of TMEM, the queries its columns: a thread of the first four warps has a page's scores to
// itself.  The other four bring the items: pages' bounds by cp.async and rounded queries, into the 128-byte swizzled layout
// and a ring of kStages.  Between two barriers one item's products run, the scores of the one before are read, and its place
// is filled again.  (One warp after the other for all of it: 700 instructions, 2.2 us to an item.)
template <typename T, int kDim>
__global__ void __launch_bounds__(kPartThreads, 2) score_blocks_kernel(const SelectArgs a, int heads_each, const Limits limits) {
    using namespace attn;
    using Tl = Tile<kDim>;
    extern __shared__ char smem[];
    asm volatile("griddepcontrol.launch_dependents;");
    const int parts = (a.req.table_width + kPart - 1) / kPart;
    const int token = static_cast<int>(blockIdx.x) / parts, part = static_cast<int>(blockIdx.x) - token * parts;
    const bool loads = threadIdx.x >= kPart;
    const int tid = threadIdx.x % kPart, lane = tid & 31, warp = tid >> 5;  // of its half
    const Row r = row_of(a, token);
    const int first = part * kPart, n = min(r.n, first + kPart);  // pages [first, n)
    if (r.n <= a.count || first >= n) return;
    const int head0 = static_cast<int>(blockIdx.y) * heads_each, heads = min(heads_each, a.kv_heads - head0);  // kv heads of this CTA
    const int slices = (a.group + kSlice - 1) / kSlice, items = heads * slices;
    const uint32_t tiles = (smem_addr(smem) + 1023) & ~1023u;
    char* base = smem + (tiles - smem_addr(smem));
    const int q_each = queries_of<kDim>(a.group), columns = columns_of(a.group);
    char* q8 = base + kStages * Tl::kBytes;  // [kStages], columns rows of 128 bytes, panel by panel
    Scoring& sh = *reinterpret_cast<Scoring*>(q8 + kStages * q_each);

    const int i = first + tid;
    const int page = page_of(a, r, i);
    if (threadIdx.x == 0) {
        bar_init(&sh.done[0], 1);
        bar_init(&sh.done[1], 1);
        bar_init(&sh.drain, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (threadIdx.x < 32) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&sh.tmem)), "n"(kTmem) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (!loads) sh.row[tid] = page < 0 ? -1 : page * a.summary.bounds_page_stride;
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = sh.tmem;
    bool late = false;
    const auto wait = [&](int item) {  // for its products
        if (late) return;
        for (int k = 0; !bar_try(&sh.done[item & 1], (item >> 1) & 1); ++k)
            if (k >= limits.tries) {
                late = true;
                break;
            }
    };
    if (loads) {
        // a thread has 16 bytes (of each 128) of 8 pages
        const int8_t* from[kPart / 16];
        uint32_t there = 0;
#pragma unroll
        for (int x = 0; x < kPart / 16; ++x) {
            const int64_t at = sh.row[16 * x + (tid >> 3)];
            from[x] = a.summary.bounds + head0 * a.summary.bounds_head_stride + max(at, static_cast<int64_t>(0)) + (tid & 7) * 16;
            there |= static_cast<uint32_t>(at >= 0) << x;
        }
        const uint32_t to = tiles + (tid >> 3) * 128 + (((tid & 7) ^ ((tid >> 3) & 7)) << 4);
        // what comes next: an item, its kv head's first page, its slice, its place, its queries (the warp's first is on its way)
        int item = 0, slice = 0, stage = 0, t_slot = 0, head = head0;
        const auto queries = [&](int h, int sl) {
            return Queries<T, kDim>(a, token, h * a.group + sl * kSlice, h < head0 + heads ? min(kSlice, a.group - sl * kSlice) : 0);
        };
        uint2 query = queries(head, 0).load(warp);
        const auto bring = [&] {
            if (item < items && !late) {
#pragma unroll
                for (int x = 0; x < kPart / 16; ++x)
#pragma unroll
                    for (int b = 0; b < Tl::kPanels; ++b)
                        if (128 * (b + 1) <= 2 * kDim || (tid & 7) < (2 * kDim % 128) / 16) {
                            const int size = (there >> x) & 1 ? 16 : 0;  // 0: filled with zeros and nothing read
                            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + stage * Tl::kBytes + b * Tl::kPanel + x * 2048),
                                         "l"(from[x] + b * 128), "r"(size)
                                         : "memory");
                        }
                const auto now = queries(head, slice);
                const uint2 first_query = query;
                if (++slice == slices) {
                    slice = 0;
                    ++head;
#pragma unroll
                    for (int x = 0; x < kPart / 16; ++x) from[x] += a.summary.bounds_head_stride;
                }
                query = queries(head, slice).load(warp);
                now.round(warp, kPart / 32, first_query, [&](int row, uint32_t below, uint32_t above, float t) {
                    char* dst = q8 + stage * q_each + row * 128;
                    const auto put = [&](int byte, uint32_t v) {  // of the row's 2 * kDim
                        *reinterpret_cast<uint32_t*>(dst + (byte >> 7) * columns * 128 + ((((byte >> 4) & 7) ^ (row & 7)) << 4) + (byte & 15)) = v;
                    };
                    if (lane < kDim / 4) {
                        put(lane * 4, below);
                        put(kDim + lane * 4, above);
                    }
                    if (lane == 0) sh.t[t_slot][row] = t;
                });
                if (++stage == kStages) stage = 0;
                t_slot = (t_slot + 1) % (kStages + 1);
                ++item;
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        for (int s = 0; s < kStages - 1; ++s) bring();
        for (int x = 0; x < items; ++x) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            late = __syncthreads_or(late);
            if (x > 0) wait(x - 1);
            bring();  // where item x - 1 was
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
    } else {
        const uint32_t lanes = tmem + (static_cast<uint32_t>(warp) << 21), idesc = instruction_s8(0) | (static_cast<uint32_t>(columns >> 3) << 17);
        const float* scale_at = a.summary.scale + (page < 0 ? 0 : page * a.summary.scale_page_stride) + head0 * a.summary.scale_head_stride;
        uint32_t* out = a.scores + (static_cast<int64_t>(token) * a.kv_heads + head0) * a.req.table_width + i;
        float scale = page < 0 ? 0.f : __ldg(scale_at), best = -INFINITY;
        int head = 0, rest = a.group, t_slot = 0;  // of the item whose scores are read next; rest: heads of its group from its slice on
        const auto finish = [&](int item) {
            wait(item);
            __syncwarp();
            tmem_fence_after();
            const bool last = rest <= kSlice;
            float next = scale;
            if (last && page >= 0 && head + 1 < heads) next = __ldg(scale_at + (head + 1) * a.summary.scale_head_stride);
            for (int c0 = 0; c0 < columns; c0 += 16) {
                float s[16];
                tmem_load16(lanes + (item & 1) * kSlice + c0, s);
                tmem_load_wait();
#pragma unroll
                for (int c = 0; c < 16; c += 4)
                    if (c0 + c < rest) {
                        const float4 t = *reinterpret_cast<const float4*>(&sh.t[t_slot][c0 + c]);
                        const float x[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (c0 + c + e < rest) best = fmaxf(best, __fmul_rn(static_cast<float>(__float_as_int(s[c + e])), x[e]));
                    }
            }
            tmem_fence_before();
            t_slot = (t_slot + 1) % (kStages + 1);
            if (last) {
                if (i < n) *out = late ? kLostKey : page < 0 ? topk::kNone : topk::order_key(scale == INFINITY ? INFINITY : __fmul_rn(best, scale));
                out += a.req.table_width;
                best = -INFINITY;
                scale = next;
                ++head;
                rest = a.group;
            } else {
                rest -= kSlice;
            }
        };
        int stage = 0;
        // all of a warp's lanes walk along, so that addresses stay in uniform registers; one issues
        const bool issues = warp == 0 && elect_one();
        const uint32_t tm = uniform(tmem), pages_low = uniform(operand_low(tiles, 16)), queries_low = uniform(operand_low(smem_addr(q8), 16));
        const uint32_t desc = uniform(idesc), q_step = uniform(static_cast<uint32_t>(q_each) / 16), q_panel = uniform(static_cast<uint32_t>(columns) * 8);
        for (int x = 0; x < items; ++x) {
            tmem_fence_before();
            late = __syncthreads_or(late);
            tmem_fence_after();
            if (warp == 0 && !late && x < limits.lost) {
                const uint32_t page_low = uniform(pages_low + stage * (Tl::kBytes / 16)), q_low = uniform(queries_low + stage * q_step);
                const uint32_t d = uniform(tm + (x & 1) * kSlice);
                if (issues) {
#pragma unroll
                    for (int k = 0; k < 2 * kDim / 32; ++k)
                        mma_smem_s8(d, page_low + ((k >> 2) * Tl::kPanel + (k & 3) * 32) / 16, q_low + (k >> 2) * q_panel + (k & 3) * 2, desc, k > 0);
                    mma_commit(&sh.done[x & 1]);
                }
                __syncwarp();
            }
            if (++stage == kStages) stage = 0;
            if (x > 0) finish(x - 1);
        }
        finish(items - 1);
        tmem_fence_before();
    }
    // products end before the CTA does, also after a wait that ran out
    late = __syncthreads_or(late);
    if (threadIdx.x == 0 && late) {
        mma_commit(&sh.drain);
        for (int k = 0; k < kTries && !bar_try(&sh.drain, 0); ++k) {
        }
    }
    __syncthreads();
    if (threadIdx.x < 32) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(kTmem) : "memory");
}

// All of a row (a token's kv head) in one CTA: as score_blocks_kernel with the row's pages as items, kPart at a time, and one
// kv head's queries for all of them; the keys stay in shared memory, and the largest are found where the pages were.  One
// place for pages and four CTAs to an SM: what one waits for, the others cover (64 ragged tokens 24.5 us; two places and three
// CTAs 25.4, three and two 27.7).
constexpr int kRowPages = 4096;  // that a row may have
constexpr int kRowGroup = 16;    // and query heads

struct RowScoring {
    alignas(16) float t[kRowGroup];
    uint64_t done[2];
    uint64_t drain;
    uint32_t tmem;
};

template <int kDim>
constexpr int kRowQueries = Tile<kDim>::kPanels * kRowGroup * 128;  // a multiple of 1024
template <int kDim>
constexpr int kRowBytes = 1024 + Tile<kDim>::kBytes + kRowQueries<kDim> + static_cast<int>(sizeof(RowScoring));  // and the keys
static_assert((kRowBytes<128> + kRowPages * 4 + 1024) * 4 <= 228 * 1024, "four CTAs to an SM");

template <typename T, int kDim>
__global__ void __launch_bounds__(kPartThreads, 4) select_rows_kernel(const SelectArgs a, const Limits limits) {
    using namespace attn;
    using Tl = Tile<kDim>;
    extern __shared__ char smem[];
    const int token = static_cast<int>(blockIdx.x) / a.kv_heads, head = static_cast<int>(blockIdx.x) - token * a.kv_heads;
    const bool loads = threadIdx.x >= kPart;
    const int tid = threadIdx.x % kPart, lane = tid & 31, warp = tid >> 5;  // of its half
    const uint32_t tiles = (smem_addr(smem) + 1023) & ~1023u;
    char* base = smem + (tiles - smem_addr(smem));
    const int columns = columns_of(a.group);
    char* q8 = base + Tl::kBytes;  // columns rows of 128 bytes, panel by panel
    RowScoring& sh = *reinterpret_cast<RowScoring*>(q8 + kRowQueries<kDim>);
    uint32_t* keys = reinterpret_cast<uint32_t*>(&sh + 1);  // no more than the table has blocks: what is left is L1's
    topk::Shared& s = *reinterpret_cast<topk::Shared*>(base);
    static_assert(sizeof(topk::Shared) <= Tl::kBytes, "where the pages were");

    const Queries<T, kDim> queries(a, token, head * a.group, a.group);
    const uint2 query = loads ? queries.load(warp) : make_uint2(0, 0);  // beside what follows
    const Row r = row_of(a, token);
    if (r.n < 0) return;
    topk::Threshold thr = {0, 0};
    if (r.n <= a.count) {
        for (int i = threadIdx.x; i < r.n; i += kPartThreads) keys[i] = page_of(a, r, i) >= 0 ? 1u : topk::kNone;
        __syncthreads();
    } else {
        if (threadIdx.x == 0) {
            bar_init(&sh.done[0], 1);
            bar_init(&sh.done[1], 1);
            bar_init(&sh.drain, 1);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        if (threadIdx.x < 32) {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&sh.tmem)), "n"(kTmem) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
        tmem_fence_before();
        __syncthreads();
        tmem_fence_after();
        const uint32_t tmem = sh.tmem;
        const int items = (r.n + kPart - 1) / kPart;
        bool late = false;
        const auto wait = [&](int item) {  // for its products
            if (late) return;
            for (int k = 0; !bar_try(&sh.done[item & 1], (item >> 1) & 1); ++k)
                if (k >= limits.tries) {
                    late = true;
                    break;
                }
        };
        uint32_t least = 0xFFFFFFFFu, most = 0;
        if (loads) {
            // a thread has 16 bytes (of each 128) of 8 pages, whose numbers are looked up an item ahead
            const int8_t* from = a.summary.bounds + head * a.summary.bounds_head_stride + (tid & 7) * 16;
            const uint32_t to = tiles + (tid >> 3) * 128 + (((tid & 7) ^ ((tid >> 3) & 7)) << 4);
            int page[kPart / 16], item = 0;
            const auto look = [&] {
#pragma unroll
                for (int x = 0; x < kPart / 16; ++x) page[x] = page_of(a, r, item * kPart + 16 * x + (tid >> 3));
            };
            const auto bring = [&] {
                if (item < items && !late) {
#pragma unroll
                    for (int x = 0; x < kPart / 16; ++x) {
                        const int8_t* src = from + max(page[x], 0) * a.summary.bounds_page_stride;
                        const int size = page[x] >= 0 ? 16 : 0;  // 0: filled with zeros and nothing read
#pragma unroll
                        for (int b = 0; b < Tl::kPanels; ++b)
                            if (128 * (b + 1) <= 2 * kDim || (tid & 7) < (2 * kDim % 128) / 16)
                                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + b * Tl::kPanel + x * 2048),
                                             "l"(src + b * 128), "r"(size)
                                             : "memory");
                    }
                    ++item;
                    look();
                }
            };
            look();
            bring();
            queries.round(warp, kPart / 32, query, [&](int row, uint32_t below, uint32_t above, float t) {
                const auto put = [&](int byte, uint32_t v) {  // of the row's 2 * kDim
                    *reinterpret_cast<uint32_t*>(q8 + row * 128 + (byte >> 7) * columns * 128 + ((((byte >> 4) & 7) ^ (row & 7)) << 4) + (byte & 15)) = v;
                };
                if (lane < kDim / 4) {
                    put(lane * 4, below);
                    put(kDim + lane * 4, above);
                }
                if (lane == 0) sh.t[row] = t;
            });
            for (int x = 0; x < items; ++x) {
                asm volatile("cp.async.wait_all;" ::: "memory");
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                late = __syncthreads_or(late);
                wait(x);
                bring();  // where item x was
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
        } else {
            const uint32_t lanes = tmem + (static_cast<uint32_t>(warp) << 21);
            const float* scales = a.summary.scale + head * a.summary.scale_head_stride;
            const auto scale_of = [&](int page) { return page >= 0 ? __ldg(scales + page * a.summary.scale_page_stride) : 0.f; };
            int page = page_of(a, r, tid), next = page_of(a, r, kPart + tid);
            float scale = scale_of(page);
            const auto finish = [&](int item) {
                wait(item);
                __syncwarp();
                tmem_fence_after();
                const int now = page, i = item * kPart + tid;
                const float by = scale;
                page = next;
                scale = scale_of(page);
                next = page_of(a, r, i + 2 * kPart);
                float v[16], best = -INFINITY;
                tmem_load16(lanes + (item & 1) * kSlice, v);
                tmem_load_wait();
#pragma unroll
                for (int c = 0; c < 16; c += 4)
                    if (c < a.group) {
                        const float4 t = *reinterpret_cast<const float4*>(&sh.t[c]);
                        const float x[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (c + e < a.group) best = fmaxf(best, __fmul_rn(static_cast<float>(__float_as_int(v[c + e])), x[e]));
                    }
                tmem_fence_before();
                if (i < r.n) {
                    const uint32_t key = now < 0 ? topk::kNone : topk::order_key(by == INFINITY ? INFINITY : __fmul_rn(best, by));
                    keys[i] = key;
                    least = min(least, key);
                    most = max(most, key);
                }
            };
            // all of a warp's lanes walk along, so that addresses stay in uniform registers; one issues
            const bool issues = warp == 0 && elect_one();
            const uint32_t tm = uniform(tmem), pages_low = uniform(operand_low(tiles, 16)), q_low = uniform(operand_low(smem_addr(q8), 16));
            const uint32_t desc = uniform(instruction_s8(0) | (static_cast<uint32_t>(columns >> 3) << 17)), q_panel = uniform(static_cast<uint32_t>(columns) * 8);
            for (int x = 0; x < items; ++x) {
                tmem_fence_before();
                late = __syncthreads_or(late);
                tmem_fence_after();
                if (warp == 0 && !late && x < limits.lost) {
                    const uint32_t d = uniform(tm + (x & 1) * kSlice);
                    if (issues) {
#pragma unroll
                        for (int k = 0; k < 2 * kDim / 32; ++k)
                            mma_smem_s8(d, pages_low + ((k >> 2) * Tl::kPanel + (k & 3) * 32) / 16, q_low + (k >> 2) * q_panel + (k & 3) * 2, desc, k > 0);
                        mma_commit(&sh.done[x & 1]);
                    }
                    __syncwarp();
                }
                finish(x);
            }
            tmem_fence_before();
        }
        // products end before their place is used for something else and the CTA ends, also after a wait that ran out
        late = __syncthreads_or(late);
        if (threadIdx.x == 0 && late) {
            mma_commit(&sh.drain);
            for (int k = 0; k < kTries && !bar_try(&sh.drain, 0); ++k) {
            }
        }
        topk::clear<kPartThreads>(s);
        __syncthreads();
        if (threadIdx.x < 32) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(kTmem) : "memory");
        if (late) return give_up(a, token, head);
        topk::range(s, least, most);
        __syncthreads();
        thr = topk::threshold<kPartThreads, topk::One>(s, r.n, a.count, topk::read_keys<kPartThreads>([&](int i) { return keys[i]; }));
    }
    choose<kPartThreads>(a, s, r, token, head, thr, topk::read_keys<kPartThreads>([&](int i) { return keys[i]; }));
}

// kHeld: a thread's keys are in registers, so many at most; 0: in shared memory, or, behind the first `room`, read again in
// each pass
template <int kRowThreads, int kHeld>
__global__ void __launch_bounds__(kRowThreads) choose_blocks_kernel(const SelectArgs a, int room) {
    extern __shared__ __align__(16) char smem[];
    topk::Shared& s = *reinterpret_cast<topk::Shared*>(smem);
    const int token = static_cast<int>(blockIdx.x) / a.kv_heads, head = static_cast<int>(blockIdx.x) - token * a.kv_heads;
    topk::clear<kRowThreads>(s);
    const Row r = row_of(a, token);
    const bool scored = r.n > a.count;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (r.n < 0) return;
    const uint32_t* scores = a.scores + (static_cast<int64_t>(token) * a.kv_heads + head) * a.req.table_width;
    const auto read = [&](int i) { return scored ? __ldcg(scores + i) : page_of(a, r, i) >= 0 ? 1u : topk::kNone; };
    uint32_t least = 0xFFFFFFFFu, most = 0;
    bool lost = false;
    const auto all = [&](const auto& keys) {
        if (__syncthreads_or(lost && scored)) return give_up(a, token, head);
        topk::Threshold thr = {0, 0};
        if (scored) {
            topk::range(s, least, most);
            __syncthreads();
            thr = topk::threshold<kRowThreads, topk::One>(s, r.n, a.count, keys);
        }
        choose<kRowThreads>(a, s, r, token, head, thr, keys);
    };
    if constexpr (kHeld > 0) {
        topk::HeldKeys<kRowThreads, kHeld> keys;
        const topk::Segment<kRowThreads> g(r.n);
#pragma unroll
        for (int x = 0; x < kHeld; ++x) {
            const int i = g.first + 32 * x + static_cast<int>(threadIdx.x & 31);
            keys.k[x] = i < g.last ? read(i) : topk::kNone;
        }
#pragma unroll
        for (int x = 0; x < kHeld; ++x)
            if (g.first + 32 * x + static_cast<int>(threadIdx.x & 31) < g.last) {
                least = min(least, keys.k[x]);
                most = max(most, keys.k[x]);
                lost = lost || keys.k[x] == kLostKey;
            }
        all(keys);
    } else {
        uint32_t* near = reinterpret_cast<uint32_t*>(smem + sizeof(topk::Shared));
        for (int i = threadIdx.x; i < r.n; i += kRowThreads) {
            const uint32_t key = read(i);
            if (i < room) near[i] = key;
            least = min(least, key);
            most = max(most, key);
            lost = lost || key == kLostKey;
        }
        all(topk::read_keys<kRowThreads>([&](int i) { return i < room ? near[i] : read(i); }));
    }
}

Limits g_limits = {kTries, INT32_MAX};

constexpr int kMaxSmem = 224 * 1024;
// Which kernels take a call, measured with 32 heads on 8 of dim 128, us: as many rows as SMs and up to kRowPages blocks of
// the table, a CTA of the tensor cores to each (64 tokens of 62 / 243 / 937 blocks 9 / 12 / 28; in threads 11 / 18 / 54).
// Fewer rows and up to kShort blocks, a CTA of threads to each (16 tokens 5.7 / 6.9, one 5.3 / 6.2; two kernels 6.9 / 8.8
// and 6.4 / 6.6).  Else two kernels (16 tokens of 937 16, in threads 20; one 8.1, in threads 15).
constexpr int kShort = 256;

int query_bytes(const SelectArgs& a) { return ((a.group + 3) & ~3) * 4 + a.group * 2 * a.dim; }

template <int kRowThreads, int kHeld>
cudaError_t launch_choose(const SelectArgs& a, unsigned rows, cudaStream_t stream) {
    static SmemOnce once;
    const cudaError_t e = once.set(reinterpret_cast<const void*>(choose_blocks_kernel<kRowThreads, kHeld>), kMaxSmem);
    if (e != cudaSuccess) return e;
    const int room = kHeld > 0 ? 0 : std::min<int>(a.req.table_width, (kMaxSmem - static_cast<int>(sizeof(topk::Shared))) / 4);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(rows);
    cfg.blockDim = dim3(kRowThreads);
    cfg.dynamicSmemBytes = sizeof(topk::Shared) + static_cast<size_t>(room) * 4;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, choose_blocks_kernel<kRowThreads, kHeld>, a, room);
}

template <typename T, int kDim>
cudaError_t launch_select(const SelectArgs& a, cudaStream_t stream) {
    const unsigned rows = static_cast<unsigned>(a.req.tokens) * a.kv_heads;
    if (a.group <= kRowGroup && a.req.table_width <= kRowPages && rows >= static_cast<unsigned>(a.sms)) {
        static SmemOnce once;
        const cudaError_t e = once.set(reinterpret_cast<const void*>(select_rows_kernel<T, kDim>), kMaxSmem);
        if (e != cudaSuccess) return e;
        select_rows_kernel<T, kDim><<<rows, kPartThreads, kRowBytes<kDim> + a.req.table_width * 4, stream>>>(a, g_limits);
        return cudaGetLastError();
    }
    if (!a.scores) {
        static SmemOnce once;
        static_assert(sizeof(topk::Shared) + 256 * (4 + 2 * 128) + kShort * 4 <= kMaxSmem, "256 heads of 128 to a kv head");
        const cudaError_t e = once.set(reinterpret_cast<const void*>(select_blocks_kernel<T, kDim>), kMaxSmem);
        if (e != cudaSuccess) return e;
        const int bytes = static_cast<int>(sizeof(topk::Shared)) + query_bytes(a) + a.req.table_width * 4;
        select_blocks_kernel<T, kDim><<<rows, kThreads, bytes, stream>>>(a);
        return cudaGetLastError();
    }
    static SmemOnce scoring;
    const cudaError_t e = scoring.set(reinterpret_cast<const void*>(score_blocks_kernel<T, kDim>), kMaxSmem);
    if (e != cudaSuccess) return e;
    const unsigned parts = (static_cast<unsigned>(a.req.table_width) + kPart - 1) / kPart;
    // kv heads to a CTA: all, or fewer as long as there are places for all CTAs at once, two to an SM (with more than 16 heads of
    // 128 to a kv head, 123 KB of shared memory, one: they may take two rounds then)
    int each = a.kv_heads;
    while (each > 1 && static_cast<int64_t>(a.req.tokens) * parts * ((a.kv_heads + (each + 1) / 2 - 1) / ((each + 1) / 2)) <= 2 * a.sms) each = (each + 1) / 2;
    const dim3 grid(a.req.tokens * parts, static_cast<unsigned>((a.kv_heads + each - 1) / each));
    score_blocks_kernel<T, kDim><<<grid, kPartThreads, scoring_bytes<kDim>(a.group), stream>>>(a, each, g_limits);
    const cudaError_t started = cudaGetLastError();
    if (started != cudaSuccess) return started;
    if (a.req.table_width <= 1024) return launch_choose<256, 4>(a, rows, stream);
    if (a.req.table_width <= 2048) return launch_choose<256, 8>(a, rows, stream);
    if (a.req.table_width <= 8192) return launch_choose<1024, 8>(a, rows, stream);
    return launch_choose<1024, 0>(a, rows, stream);
}

template <typename T>
cudaError_t select_by_dim(const SelectArgs& a, cudaStream_t s) {
    return a.dim == 64 ? launch_select<T, 64>(a, s) : a.dim == 96 ? launch_select<T, 96>(a, s) : launch_select<T, 128>(a, s);
}

template <typename T, int kDim>
cudaError_t launch_summarize(const SummarizeArgs& a, cudaStream_t stream) {
    const int64_t items = (static_cast<int64_t>(a.req.tokens) >> a.cache.page_shift) + 2 * static_cast<int64_t>(a.req.requests);
    const int64_t grid = (items * a.cache.heads + kSumWarps - 1) / kSumWarps;
    if (grid > INT32_MAX) return cudaErrorInvalidConfiguration;
    kv_summarize_kernel<T, kDim><<<static_cast<unsigned>(grid), kSumWarps * 32, 0, stream>>>(a, items);
    return cudaGetLastError();
}
template <typename T>
cudaError_t summarize_by_dim(const SummarizeArgs& a, cudaStream_t s) {
    return a.cache.dim == 64 ? launch_summarize<T, 64>(a, s) : a.cache.dim == 96 ? launch_summarize<T, 96>(a, s) : launch_summarize<T, 128>(a, s);
}

}  // namespace

void set_selection_waits(int lost, int tries) { g_limits = {tries < 0 ? kTries : tries, lost < 0 ? INT32_MAX : lost}; }

int first_past_on_host(int n, int first) {
    struct Past {
        int first;
        __host__ __device__ bool operator()(int x) const { return x >= first; }
    };
    Span s = {0, n};
    while (s.n > 1) {
        int x = 0;
        while (!s.ends(x, Past{first})) ++x;
        s.take(x);
    }
    return s.lo;
}

bool select_counts(int tokens, int kv_heads, int table_width) {
    return static_cast<int64_t>(tokens) * kv_heads <= INT32_MAX && static_cast<int64_t>(tokens) * (table_width / kPart + 1) <= INT32_MAX &&
           kv_heads <= 65535;
}

size_t select_workspace(int tokens, int kv_heads, int table_width) {
    return table_width <= kShort ? 0 : static_cast<size_t>(tokens) * kv_heads * table_width * sizeof(uint32_t);
}

cudaError_t launch_kv_summarize(const SummarizeArgs& a, cudaStream_t stream) {
    return a.cache.dtype == FG_DTYPE_BF16 ? summarize_by_dim<__nv_bfloat16>(a, stream) : summarize_by_dim<__half>(a, stream);
}

cudaError_t launch_select_blocks(const SelectArgs& a, cudaStream_t stream) {
    return a.dtype == FG_DTYPE_BF16 ? select_by_dim<__nv_bfloat16>(a, stream) : select_by_dim<__half>(a, stream);
}

}  // namespace fg
