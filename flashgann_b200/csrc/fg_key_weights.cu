// fg_key_weights.cu -- the attention weight that each key of the cache was given.
//
// For the rows r of a step (its new tokens' query heads of one kv head), whose
// log-sum-exp the attention left,
//     w[j] = (j < held ? w[j] : 0) + sum over the rows r that see j of e^(scale q_r.k_j - lse_r).
//
// Every key of a request and kv head is one warp's, which walks all of its rows:
// no atomics, and the sum's order depends on the row's number alone.  A chunk is
// 32 keys, two m16n8k16 products with the keys as their rows and 8 query rows as
// their columns, so that the sum over rows is a sum within a thread and over 4
// lanes.  Keys go from memory straight to the registers of the product: the order
// of its 16 summands is free, so a lane keeps the 16 bytes that it loads (4 lanes
// to 64 bytes of a key), and takes the same elements of the queries.
//
// Few rows are bound by the keys' way from memory, 2 * dim bytes each; 8 KB to a
// warp under way at once.  Many rows (the last tokens of a prompt) are bound by
// the products.  The chunks are split over the CTAs as in fg_attention.cuh.
#include <algorithm>

#include "fg_attention.cuh"
#include "fg_cache.h"

namespace fg {
namespace attn {
namespace {

constexpr int kRows = 16;    // not looked at: a tile is a request
constexpr int kChunk = 32;
constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kCtasPerSm = 2;

template <typename T>
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma<__half>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma<__nv_bfloat16>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 8 query rows as the columns of a product; this lane's two of them for masks and weights.
template <int kDim>
struct Columns {
    uint4 q[kDim / 32];
    float lse[2];
    int p[2];  // positions; -1: no such row, or one whose sum is not finite, which gives nothing
};

template <typename T, int kDim>
__device__ __forceinline__ Columns<kDim> load_columns(const AttentionParams& a, const WeightsArgs& w, const Request& r, int head, int c0) {
    Columns<kDim> c;
    const int lane = threadIdx.x & 31, rows = r.rows * a.group;
    {
        const int R = c0 + (lane >> 2);
        const int i = div_group(a, min(R, rows - 1)), g = min(R, rows - 1) - i * a.group;
        const T* src = static_cast<const T*>(a.q) + static_cast<int64_t>(r.start + i) * a.q_token_stride +
                       static_cast<int64_t>(head * a.group + g) * a.q_head_stride + (lane & 3) * 8;
#pragma unroll
        for (int k = 0; k < kDim / 32; ++k) c.q[k] = __ldg(reinterpret_cast<const uint4*>(src + 32 * k));
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const int R = c0 + (lane & 3) * 2 + e;
        const int i = div_group(a, min(R, rows - 1)), g = min(R, rows - 1) - i * a.group;
        c.lse[e] = __ldg(w.lse + static_cast<int64_t>(r.start + i) * a.heads + head * a.group + g);
        c.p[e] = R < rows && isfinite(c.lse[e]) ? r.kv_len - r.rows + i : -1;
    }
    return c;
}

template <typename T, int kDim>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) attention_weights_kernel(const AttentionParams a, const WeightsArgs w) {
    extern __shared__ __align__(16) int scratch[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Place pl = locate<kRows, kWhole, kChunk, kThreads, 1>(a, scratch, blockIdx.x, a.ctas);
    if (pl.unit >= pl.end) return;
    int head = pl.head, request = pl.request, tile = pl.tile;
    int64_t unit = pl.unit, tile_first = pl.unit - pl.offset;
    Request r = load_request(a, request);
    while (true) {
        const TileKeys keys = tile_keys<kRows, kWhole, kChunk>(a, r, 0);
        const int64_t tile_last = tile_first + keys.units;
        const int cost = whole_cost(a, r);
        // a chunk belongs to the CTA whose range holds its first unit
        const auto chunk_at = [&](int64_t u) {
            return static_cast<int>(min(((u - tile_first + cost - 1) / cost) << a.unit_shift, static_cast<int64_t>(keys.chunks)));
        };
        const int c0 = chunk_at(unit), c1 = chunk_at(min(tile_last, pl.end));
        const int32_t* table = a.block_table + request * a.table_stride;
        const int rows = r.rows * a.group, p0 = r.kv_len - r.rows, p1 = r.kv_len - 1;
        const int held = a.held ? max(0, __ldg(a.held + request)) : max(0, p0);
        // keys of chunk c: from the first one on, those in [from, to) or below `sinks`
        const auto key_of = [&](int c, int x) {
            if (c < keys.sink_chunks) {
                const int j = c * kChunk + x;
                return j < keys.sink_hi ? j : -1;
            }
            const int j = keys.base + (c - keys.sink_chunks) * kChunk + x;
            return j < keys.hi && (j >= keys.lo || j < a.sinks) ? j : -1;
        };
        const auto page_of = [&](int j) {
            if (j < 0) return -1;
            const int at = j >> a.page_shift;
            const int page = at < a.table_width ? __ldg(table + at) : -1;
            return static_cast<uint32_t>(page) < static_cast<uint32_t>(a.pages) ? page : -1;
        };
        const bool few = rows <= 8;
        Columns<kDim> col;
        if (few && c0 + warp < c1) col = load_columns<T, kDim>(a, w, r, head, 0);
        int next[4];
#pragma unroll
        for (int y = 0; y < 4; ++y) next[y] = c0 + warp < c1 ? page_of(key_of(c0 + warp, (lane >> 2) + 8 * y)) : -1;
        for (int c = c0 + warp; c < c1; c += kWarps) {
            // keys (lane / 4) + 8 y
            int j[4], page[4];
            uint4 k[4][kDim / 32];
            float* at[4];
            float before[4], sum[4];
            bool all = true;
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                page[y] = next[y];
                j[y] = key_of(c, (lane >> 2) + 8 * y);
                const T* src = static_cast<const T*>(a.k_cache) + page[y] * a.page_stride + (j[y] & (a.page_size - 1)) * a.token_stride +
                               head * a.head_stride + (lane & 3) * 8;
#pragma unroll
                for (int x = 0; x < kDim / 32; ++x)
                    k[y][x] = page[y] >= 0 ? __ldg(reinterpret_cast<const uint4*>(src + 32 * x)) : make_uint4(0, 0, 0, 0);
                at[y] = w.weights.w + page[y] * w.weights.page_stride + head * w.weights.head_stride + (j[y] & (a.page_size - 1));
                before[y] = page[y] >= 0 && j[y] < held && (lane & 3) == 0 ? *at[y] : 0.f;
                sum[y] = 0.f;
                all = all && page[y] >= 0 && j[y] <= p0 && (a.window < 0 || p1 - j[y] < a.window || j[y] < a.sinks);
            }
#pragma unroll
            for (int y = 0; y < 4; ++y) next[y] = c + kWarps < c1 ? page_of(key_of(c + kWarps, (lane >> 2) + 8 * y)) : -1;
            all = __all_sync(0xFFFFFFFFu, all);
            for (int n0 = 0; n0 < rows; n0 += 8) {
                if (!few) col = load_columns<T, kDim>(a, w, r, head, n0);
                float s[2][4];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    s[h][0] = s[h][1] = s[h][2] = s[h][3] = 0.f;
#pragma unroll
                    for (int x = 0; x < kDim / 32; ++x) {
                        mma<T>(s[h], k[2 * h][x].x, k[2 * h + 1][x].x, k[2 * h][x].y, k[2 * h + 1][x].y, col.q[x].x, col.q[x].y);
                        mma<T>(s[h], k[2 * h][x].z, k[2 * h + 1][x].z, k[2 * h][x].w, k[2 * h + 1][x].w, col.q[x].z, col.q[x].w);
                    }
                }
#pragma unroll
                for (int y = 0; y < 4; ++y)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        // the difference first: scores and lse may be large, it is not where the weight counts
                        const float x = exp2_fast(fmaf(s[y >> 1][(y & 1) * 2 + e], w.scale, -col.lse[e]) * kLog2e);
                        const int p = col.p[e];
                        const bool sees = all ? p >= 0 : j[y] >= 0 && j[y] <= p && (a.window < 0 || p - j[y] < a.window || j[y] < a.sinks);
                        sum[y] += sees ? x : 0.f;
                    }
            }
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                sum[y] += __shfl_xor_sync(0xFFFFFFFFu, sum[y], 1);
                sum[y] += __shfl_xor_sync(0xFFFFFFFFu, sum[y], 2);
                if ((lane & 3) == 0 && page[y] >= 0) *at[y] = before[y] + sum[y];
            }
        }
        if (tile_last >= pl.end || !next_tile<kRows, kWhole>(a, &r, &head, &request, &tile)) break;
        unit = tile_first = tile_last;
    }
}

template <typename T, int kDim>
cudaError_t launch(AttentionParams a, const WeightsArgs& w, cudaStream_t stream) {
    a.base_align = kChunk;
    a.tile_units = 0;
    a.ctas *= kCtasPerSm;
    a.held = w.held;
    // the units of a kv head are summed in 32 bits
    const int64_t keys = std::min<int64_t>(static_cast<int64_t>(a.table_width) * a.page_size, INT32_MAX);
    const int64_t costs = a.requests + ((static_cast<int64_t>(a.tokens) * a.group) >> 6);
    a.unit_shift = 0;
    while (a.unit_shift < 24 && costs * (((keys / kChunk + 3) >> a.unit_shift) + 1) > INT32_MAX) ++a.unit_shift;
    const int bytes = locate_bytes(a.requests);
    static SmemOnce once;
    const cudaError_t e = once.set(reinterpret_cast<const void*>(attention_weights_kernel<T, kDim>), locate_bytes(kMaxRequests));
    if (e != cudaSuccess) return e;
    attention_weights_kernel<T, kDim><<<a.ctas, kThreads, bytes, stream>>>(a, w);
    return cudaGetLastError();
}

template <typename T>
cudaError_t by_dim(const AttentionParams& a, const WeightsArgs& w, cudaStream_t s) {
    return a.dim == 64 ? launch<T, 64>(a, w, s) : a.dim == 96 ? launch<T, 96>(a, w, s) : launch<T, 128>(a, w, s);
}

}  // namespace
}  // namespace attn

cudaError_t launch_attention_weights(const AttentionParams& a, const WeightsArgs& w, cudaStream_t stream) {
    return a.dtype == FG_DTYPE_BF16 ? attn::by_dim<__nv_bfloat16>(a, w, stream) : attn::by_dim<__half>(a, w, stream);
}

}  // namespace fg
