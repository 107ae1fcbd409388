// fg_blocks.cu -- which pages of a long context a query attends to: a summary
// of each page's keys, and the choice of the pages whose bound on the scores is
// highest.
#include <algorithm>
#include <cmath>
#include <cstdint>

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "fg_cache.h"
#include "fg_internal.h"
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

constexpr float k127th = 1.f / 127.f;  // a product, rounded once: what a quotient would give but for its last bit

__device__ __forceinline__ int clamped(const int32_t* p, int most) { return max(0, min(__ldg(p), most)); }

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
    int lo = 0, hi = a.req.requests - 1;
    const auto first_item = [&](int b) { return static_cast<int64_t>(clamped(a.req.query_start + b, a.req.tokens) >> shift) + 2 * static_cast<int64_t>(b); };
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (first_item(mid) <= item) lo = mid;
        else hi = mid - 1;
    }
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
// t = top / 127.  Its score of a page is an upper bound of q.k over the page's
// keys, in 8-bit arithmetic,
//     I = sum_d Q_d * (Q_d < 0 ? lower_d : upper_d),     score = max_h (I_h t_h) * scale
// over the heads h of the group.  I is a product of (min(Q, 0), max(Q, 0)) with
// the page's 2 * dim bounds as they lie in memory, a whole number below 2^21, and
// two 32-bit roundings follow: every order of summation gives the same score, so
// the choice is the same bit for bit.
//
// A cluster of CTAs has one token and kv head: its pages' summaries are read
// once, by the fragment of an m16n8k32 product straight from memory (16 pages x
// 64 bytes to a load, 4 lanes to a page; the order of a product's 64 summands is
// free, so each lane keeps the 16 bytes that it loads), the scores stay in shared
// memory as keys, and fg_topk.cuh finds the largest.
using topk::kThreads;
using topk::kWarps;

struct SelectShared {
    topk::Shared top;
};
static_assert(sizeof(SelectShared) % 16 == 0, "the queries behind it and 8 floats for each column are read 16 bytes at a time");

__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <typename T, int kDim>
__global__ void __launch_bounds__(kThreads) select_blocks_kernel(const SelectArgs a) {
    namespace cg = cooperative_groups;
    const cg::cluster_group cluster = cg::this_cluster();
    extern __shared__ __align__(16) char smem[];
    SelectShared& s = *reinterpret_cast<SelectShared*>(smem);
    const int columns = (a.group + 7) & ~7;
    float* t_of = reinterpret_cast<float*>(smem + sizeof(SelectShared));         // [columns]
    uint32_t* q8 = reinterpret_cast<uint32_t*>(t_of + columns);                   // [columns][2 * kDim bytes]
    uint32_t* keys = q8 + columns * (kDim / 2);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const unsigned ranks = cluster.num_blocks(), rank = cluster.block_rank();
    const int64_t row = blockIdx.x / ranks;
    const int token = static_cast<int>(row / a.kv_heads), head = static_cast<int>(row - static_cast<int64_t>(token) * a.kv_heads);

    // the request of this row: the first that ends after it
    int lo = 0, hi = a.req.requests - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (clamped(a.req.query_start + mid + 1, a.req.tokens) > token) hi = mid;
        else lo = mid + 1;
    }
    const int start = clamped(a.req.query_start + lo, a.req.tokens), end = clamped(a.req.query_start + lo + 1, a.req.tokens);
    if (token < start || token >= end) return;  // no request's: the whole cluster leaves
    const int p = max(0, __ldg(a.req.kv_len + lo)) - (end - token);
    const int b0 = a.sinks >> a.page_shift;
    const int b1 = p >= a.window ? min(((p - a.window) >> a.page_shift) + 1, a.req.table_width) : 0;
    const int n = max(0, b1 - b0);
    // this CTA's pages: [c0, c0 + m) of the n
    const int per = (n + static_cast<int>(ranks) - 1) / static_cast<int>(ranks);
    const int c0 = min(n, per * static_cast<int>(rank)), m = min(n, c0 + per) - c0;
    const int32_t* table = a.req.block_table + lo * a.req.table_stride + b0 + c0;
    const auto page_of = [&](int i) { return i < m ? __ldg(table + i) : -1; };
    const auto there = [&](int page) { return static_cast<uint32_t>(page) < static_cast<uint32_t>(a.pages); };

    topk::Threshold thr = {0, 0};
    if (n <= a.count) {
        for (int i = tid; i < m; i += kThreads) keys[i] = there(page_of(i)) ? 1u : topk::kNone;
        __syncthreads();
    } else {
        // the group's queries in 8 bits, a warp to each
        for (int g = warp; g < columns; g += kWarps) {
            float v[4] = {0.f, 0.f, 0.f, 0.f}, top = 0.f;
            if (g < a.group && lane < kDim / 4) {
                const uint2 w = __ldg(reinterpret_cast<const uint2*>(static_cast<const T*>(a.q) + token * a.q_token_stride +
                                                                     (static_cast<int64_t>(head) * a.group + g) * a.q_head_stride) + lane);
                const float2 x = Pair<T>::floats(w.x), y = Pair<T>::floats(w.y);
                v[0] = x.x;
                v[1] = x.y;
                v[2] = y.x;
                v[3] = y.y;
            }
            bool fine = true;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                fine = fine && isfinite(v[e]);
                top = fmaxf(top, fabsf(v[e]));
            }
            fine = __all_sync(0xFFFFFFFFu, fine);
#pragma unroll
            for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
            uint32_t below = 0, above = 0;
            if (fine && top > 0.f) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int x = static_cast<int>(rintf(in_127ths(v[e], top)));
                    below |= static_cast<uint32_t>(min(x, 0) & 255) << (8 * e);
                    above |= static_cast<uint32_t>(max(x, 0) & 255) << (8 * e);
                }
            }
            if (lane < kDim / 4) {
                q8[g * (kDim / 2) + lane] = below;
                q8[g * (kDim / 2) + kDim / 4 + lane] = above;
            }
            if (lane == 0) t_of[g] = fine ? top * k127th : 0.f;
        }
        __syncthreads();
        constexpr int kSteps = 2 * kDim / 64;  // 64 bytes of 16 pages
        const int4* q4 = reinterpret_cast<const int4*>(q8);
        for (int i0 = warp * 16; i0 < m; i0 += kWarps * 16) {
            int page[2];
            uint4 v[2][kSteps];
            float scale[2] = {0.f, 0.f};
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                page[y] = page_of(i0 + (lane >> 2) + 8 * y);
                const bool ok = there(page[y]);
                const int8_t* src = a.summary.bounds + page[y] * a.summary.bounds_page_stride + head * a.summary.bounds_head_stride + (lane & 3) * 16;
#pragma unroll
                for (int k = 0; k < kSteps; ++k) v[y][k] = ok ? __ldg(reinterpret_cast<const uint4*>(src) + 4 * k) : make_uint4(0, 0, 0, 0);
                if (ok) scale[y] = __ldg(a.summary.scale + page[y] * a.summary.scale_page_stride + head * a.summary.scale_head_stride);
            }
            float best[2] = {-INFINITY, -INFINITY};
            for (int g0 = 0; g0 < a.group; g0 += 8) {
                int c[4] = {0, 0, 0, 0};
#pragma unroll
                for (int k = 0; k < kSteps; ++k) {
                    const int4 b = q4[(g0 + (lane >> 2)) * (kDim / 8) + 4 * k + (lane & 3)];
                    mma_s8(c, v[0][k].x, v[1][k].x, v[0][k].y, v[1][k].y, b.x, b.y);
                    mma_s8(c, v[0][k].z, v[1][k].z, v[0][k].w, v[1][k].w, b.z, b.w);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int g = g0 + (lane & 3) * 2 + (e & 1);
                    if (g < a.group) best[e >> 1] = fmaxf(best[e >> 1], __fmul_rn(static_cast<float>(c[e]), t_of[g]));
                }
            }
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                best[y] = fmaxf(best[y], __shfl_xor_sync(0xFFFFFFFFu, best[y], 1));
                best[y] = fmaxf(best[y], __shfl_xor_sync(0xFFFFFFFFu, best[y], 2));
                const int i = i0 + (lane >> 2) + 8 * y;
                if ((lane & 3) == 0 && i < m)
                    keys[i] = there(page[y]) ? topk::order_key(scale[y] == INFINITY ? INFINITY : __fmul_rn(best[y], scale[y])) : topk::kNone;
            }
        }
        __syncthreads();
        thr = topk::threshold(cluster, s.top, m, a.count, [&](int i) { return keys[i]; });
    }
    int32_t* out = a.blocks + token * a.blocks_token_stride + head * a.blocks_head_stride;
    const int taken = topk::emit(cluster, s.top, m, thr, [&](int i) { return keys[i]; }, [&](int place, int i) { out[place] = b0 + c0 + i; });
    if (rank == 0)
        for (int x = taken + tid; x < a.count; x += kThreads) out[x] = -1;
    cluster.sync();  // no CTA ends while another may read its counts
}

constexpr int kMaxCluster = 8;
constexpr int kMaxSmem = 200 * 1024;

int select_bytes(const SelectArgs& a, int ranks) {
    const int columns = (a.group + 7) & ~7;
    return static_cast<int>(sizeof(SelectShared)) + columns * (4 + 2 * a.dim) + (a.req.table_width + ranks - 1) / ranks * 4;
}

template <typename T, int kDim>
cudaError_t launch_select(const SelectArgs& a, cudaStream_t stream) {
    // CTAs to a row: as many as fill the SMs once, each with 512 pages at least
    const int64_t rows = static_cast<int64_t>(a.req.tokens) * a.kv_heads;
    int ranks = 1;
    while (ranks < kMaxCluster && ((rows * ranks < a.sms && a.req.table_width > 512 * ranks) || select_bytes(a, ranks) > kMaxSmem)) ranks *= 2;
    static SmemOnce once;
    const cudaError_t e = once.set(reinterpret_cast<const void*>(select_blocks_kernel<T, kDim>), kMaxSmem);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(rows * ranks));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = select_bytes(a, ranks);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(ranks);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, select_blocks_kernel<T, kDim>, a);
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

constexpr int kMaxWidth = 1 << 18;
static_assert(sizeof(SelectShared) + 256 * (4 + 2 * 128) + kMaxWidth / kMaxCluster * 4 <= kMaxSmem, "256 heads of 128 to a kv head");
int select_max_width() { return kMaxWidth; }

cudaError_t launch_kv_summarize(const SummarizeArgs& a, cudaStream_t stream) {
    return a.cache.dtype == FG_DTYPE_BF16 ? summarize_by_dim<__nv_bfloat16>(a, stream) : summarize_by_dim<__half>(a, stream);
}

cudaError_t launch_select_blocks(const SelectArgs& a, cudaStream_t stream) {
    return a.dtype == FG_DTYPE_BF16 ? select_by_dim<__nv_bfloat16>(a, stream) : select_by_dim<__half>(a, stream);
}

}  // namespace fg
