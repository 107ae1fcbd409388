// fg_attention.cuh -- what the attention kernels share: their arguments, the
// mask, the list of key chunks a tile of query rows has to visit, and the
// split of all tiles' chunks over a fixed number of CTAs.
//
// Mathematics.  Query row (token i of a request, head h) stands at position
// p = kv_len - new + i and sees the keys
//     V(p) = { j : 0 <= j <= p, and (no window, or p - j < window, or j < sinks) }
// plus, for the retrieved form, those of its head's ids that are in [0, p].
// With s_j = scale * q.k_j it returns o = sum_j e^(s_j) v_j / sum_j e^(s_j)
// and lse = log sum_j e^(s_j) over j in V(p); 0 and -inf where V(p) is empty.
// All kernels walk the keys once with a running maximum m, sum l and
// unnormalised o (base 2 exponents), so that two disjoint sets of keys join as
//     m = max(m1, m2), l = l1 2^(m1-m) + l2 2^(m2-m), o likewise.
//
// Work split.  Tiles (kv head, request, row tile) differ in length by orders
// of magnitude (one short decode beside a chunk over a long context), so the
// unit of work is not the tile but 2^unit_shift chunks of keys of one tile.
// All units are numbered in tile order and CTA c of P takes the contiguous
// range [c*W/P, (c+1)*W/P) of the W units.  A tile begins with `tile_units`
// units without chunks, for what a CTA spends on any tile (queries, join,
// output); a range that ends in them ends before the tile.  So every CTA gets the same amount of
// key traffic to within one unit whatever the lengths, and at most its first
// and its last tile are shared with a neighbour.  Those go to the workspace as
// partial (o, m, l), which attention_combine_kernel joins in unit order: no
// atomics, no waiting between CTAs, and the same bits on every run.
#pragma once

#include <cfloat>
#include <cstdint>

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "fg_internal.h"

namespace fg {
namespace attn {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// The workspace: a record for each CTA, then its partials.  A CTA whose range
// starts inside a tile that the CTA before it began has the tile to be joined.
struct alignas(16) TileRecord {
    int32_t parts;   // CTAs that share the tile, 0: nothing to join here
    int32_t before;  // number of the first one's partial; the others' are 2c, 2c + 2, ...
    int32_t head, tile;
    int32_t start, rows;  // the request's first query row and its new tokens
    int32_t pad[2];
};

__host__ __device__ inline size_t workspace_records_bytes(int ctas) {
    return (static_cast<size_t>(ctas) * sizeof(TileRecord) + 255) & ~static_cast<size_t>(255);
}
// one partial: rows x dim sums, then rows maxima and rows sums
__host__ __device__ inline size_t partial_floats(int rows, int dim) { return static_cast<size_t>(rows) * (dim + 2); }

// Shared memory that locate takes at its start: the block's warp sums and one
// sum for each request.  A launch of more requests than its kernel's other
// uses have room for asks for this much instead.
constexpr int kMaxRequests = 16384;
__host__ __device__ constexpr int locate_bytes(int requests) { return (64 + requests) * static_cast<int>(sizeof(int)); }

// One request as every kernel reads it, clamped to the buffers the launch was given.
struct Request {
    int start, rows, kv_len;  // first query token, new tokens, keys
};

__device__ __forceinline__ Request load_request(const AttentionParams& a, int b) {
    Request r;
    const int s = max(0, min(a.query_start[b], a.tokens)), e = max(0, min(a.query_start[b + 1], a.tokens));
    r.start = s;
    r.rows = max(0, e - s);
    r.kv_len = max(0, a.kv_len[b]);
    return r;
}

// The chunks of kChunk keys that one tile visits: those of the first tokens
// that lie before the window, those of the window (from `base`, up to `hi`),
// then the retrieved ones.
struct TileKeys {
    int lo, hi, base;            // window part: keys [lo, hi), chunks start at base = lo rounded down to base_align
    int sink_hi;                 // first-token part: keys [0, sink_hi)
    int sink_chunks, near_chunks, id_chunks, chunks;
    int units;
};

// n / group for 0 <= n < 2^31 (the host sees to it): 64-bit divisions of every
// row's number cost more than the copy of the row.
__device__ __forceinline__ int div_group(const AttentionParams& a, int n) {
    return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(n)) * a.group_mul) >> a.group_shift);
}

// The query rows of a tile of one kv head.
//   kPacked  kRows consecutive (token, head of the group) pairs of a request
//   kTokens  the group's heads of as many tokens as fit kRows rows
//   kToken   one token, tile_rows heads of the group (what each head retrieved is its own)
enum Layout { kPacked, kTokens, kToken };

template <int kRows, Layout kLayout>
struct Tiles {
    // tokens of a tile, or tiles of a token
    __device__ static __forceinline__ int per(const AttentionParams& a) {
        return kLayout == kTokens ? div_group(a, kRows) : (a.group + a.tile_rows - 1) / a.tile_rows;
    }
    __device__ static __forceinline__ int count(const AttentionParams& a, const Request& r) {
        if (kLayout == kToken) return r.rows * per(a);
        if (kLayout == kTokens) return (r.rows + per(a) - 1) / per(a);
        return (r.rows * a.group + kRows - 1) / kRows;
    }
    __device__ static __forceinline__ void tokens(const AttentionParams& a, const Request& r, int t, int* i0, int* i1) {
        if (kLayout == kToken) {
            *i0 = *i1 = t / per(a);
        } else if (kLayout == kTokens) {
            *i0 = t * per(a);
            *i1 = min(r.rows, *i0 + per(a)) - 1;
        } else {
            *i0 = div_group(a, t * kRows);
            *i1 = min(r.rows - 1, div_group(a, t * kRows + kRows - 1));
        }
    }
    // row -> (token of the request, head of the group); false past the tile's end
    __device__ static __forceinline__ bool row(const AttentionParams& a, const Request& r, int t, int row, int* i, int* g) {
        if (kLayout == kToken) {
            const int n = per(a);
            *i = t / n;
            *g = (t - *i * n) * a.tile_rows + row;
            return row < a.tile_rows && *g < a.group;
        }
        const int R = kLayout == kTokens ? row : t * kRows + row;
        const int x = div_group(a, R);
        *g = R - x * a.group;
        *i = kLayout == kTokens ? t * per(a) + x : x;
        return *i < r.rows && (kLayout == kPacked || x < per(a));
    }
};

template <int kRows, Layout kLayout, int kChunk>
__device__ __forceinline__ TileKeys tile_keys(const AttentionParams& a, const Request& r, int t) {
    TileKeys k;
    int i0, i1;
    Tiles<kRows, kLayout>::tokens(a, r, t, &i0, &i1);
    const int p0 = r.kv_len - r.rows + i0, p1 = r.kv_len - r.rows + i1;
    // keys that the table can address, and that chunk numbers in 32 bits can
    const int64_t room = min(static_cast<int64_t>(a.table_width) * a.page_size, static_cast<int64_t>(INT32_MAX - 1023));
    k.hi = p1 < 0 ? 0 : static_cast<int>(min(static_cast<int64_t>(p1) + 1, room));
    k.lo = (a.window < 0 || p0 < a.window) ? 0 : min(p0 - a.window + 1, k.hi);
    k.base = k.lo & -a.base_align;
    k.sink_hi = min(a.sinks, k.base);
    k.sink_chunks = (k.sink_hi + kChunk - 1) / kChunk;
    k.near_chunks = (k.hi - k.base + kChunk - 1) / kChunk;
    k.id_chunks = 0;
    if (kLayout == kToken && a.ids_count > 0 && k.lo > 0) {
        const int heads = min(a.tile_rows, a.group - (t % Tiles<kRows, kLayout>::per(a)) * a.tile_rows);
        k.id_chunks = heads * ((a.ids_count + kChunk - 1) / kChunk);
    }
    k.chunks = k.sink_chunks + k.near_chunks + k.id_chunks;
    // a tile that sees nothing still writes its rows
    k.units = a.tile_units + max(1, (k.chunks + (1 << a.unit_shift) - 1) >> a.unit_shift);
    return k;
}

// Where a CTA's range begins, and the range.
struct Place {
    int64_t unit, end;   // this CTA's units [unit, end)
    int64_t total;       // W
    int ctas;            // CTAs with a non-empty range: min(P, W)
    int head, request, tile, offset;  // the first unit: its tile and its place in it
};

// a / b, without a 64-bit division where 32 bits will do
__device__ __forceinline__ int64_t divide(int64_t a, uint32_t b) {
    if ((a >> 32) == 0) return static_cast<uint32_t>(a) / b;
    return a / b;
}
// total * c / ctas
__device__ __forceinline__ int64_t share(int64_t total, int c, int ctas) {
    const int64_t each = divide(total, ctas);
    const uint32_t rest = static_cast<uint32_t>(total - each * ctas);
    return each * c + rest * static_cast<uint32_t>(c) / static_cast<uint32_t>(ctas);  // both below 2^16
}

// Called by all kThreads threads; scratch holds locate_bytes(requests).  The
// units of a kv head are summed in 32 bits: the host sees to it, from the counts
// and the table's width, that there are fewer than 2^31 (64-bit sums cost every
// call 0.2 to 0.3 us, and 1 % in the kernel of many rows).  kLanes
// threads count the tiles of a request: 1 where requests are short, 8 where
// they have many tiles.
template <int kRows, Layout kLayout, int kChunk, int kThreads, int kLanes>
__device__ __forceinline__ Place locate(const AttentionParams& a, int* scratch, int cta, int ctas) {
    int* pre = scratch + 64;  // inclusive prefix of the requests' units
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int kWarps = kThreads / 32;
    int carry = 0, few = 0;
    if (a.requests <= 32 / kLanes) {  // every warp on its own, without a barrier
        if (lane / kLanes < a.requests) {
            const Request r = load_request(a, lane / kLanes);
            const int n = Tiles<kRows, kLayout>::count(a, r);
            for (int t = lane % kLanes; t < n; t += kLanes) few += tile_keys<kRows, kLayout, kChunk>(a, r, t).units;
        }
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int v = __shfl_up_sync(0xFFFFFFFFu, few, d);
            if (lane >= d) few += v;
        }
        carry = __shfl_sync(0xFFFFFFFFu, few, 31);
    } else {
        for (int b0 = 0; b0 < a.requests; b0 += kThreads / kLanes) {
            const int b = b0 + tid / kLanes;
            int s = 0;
            if (b < a.requests) {
                const Request r = load_request(a, b);
                const int n = Tiles<kRows, kLayout>::count(a, r);
                for (int t = tid % kLanes; t < n; t += kLanes) s += tile_keys<kRows, kLayout, kChunk>(a, r, t).units;
            }
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int v = __shfl_up_sync(0xFFFFFFFFu, s, d);
                if (lane >= d) s += v;
            }
            if (lane == 31) scratch[warp] = s;
            __syncthreads();
            int before = carry, sum = 0;
            for (int w = 0; w < kWarps; ++w) {
                const int v = scratch[w];
                if (w < warp) before += v;
                sum += v;
            }
            if (b < a.requests && tid % kLanes == kLanes - 1) pre[b] = before + s;
            carry += sum;
            __syncthreads();
        }
    }
    Place x;
    const int64_t per_head = carry;
    x.total = per_head * a.kv_heads;
    x.ctas = static_cast<int>(min(static_cast<int64_t>(ctas), x.total));
    if (cta >= x.ctas) {
        x.unit = x.end = 0;
        return x;
    }
    x.unit = share(x.total, cta, x.ctas);
    x.end = share(x.total, cta + 1, x.ctas);
    x.head = static_cast<int>(divide(x.unit, static_cast<uint32_t>(per_head)));
    int rest = static_cast<int>(x.unit - x.head * per_head);  // units before the range, of this head
    int lo = 0, hi = a.requests - 1;  // first request whose inclusive prefix exceeds rest
    if (a.requests <= 32 / kLanes) {
        lo = max(0, __ffs(__ballot_sync(0xFFFFFFFFu, few > rest)) - 1) / kLanes;  // none only where sums wrapped, see below
        const int before = __shfl_sync(0xFFFFFFFFu, few, max(lo * kLanes - 1, 0));
        if (lo > 0) rest -= before;
    } else {
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (pre[mid] > rest) hi = mid;
            else lo = mid + 1;
        }
        if (lo > 0) rest -= pre[lo - 1];
    }
    x.request = lo;
    const Request r = load_request(a, lo);
    // the tile that holds unit `rest` of the request, 32 tiles at a time, in every warp
    const int tiles = Tiles<kRows, kLayout>::count(a, r);
    int t = 0;
    bool found = false;
    for (int t0 = 0; t0 < tiles; t0 += 32) {
        const int mine = t0 + lane;
        const int u = mine < tiles ? tile_keys<kRows, kLayout, kChunk>(a, r, mine).units : 0;
        int s = u;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int v = __shfl_up_sync(0xFFFFFFFFu, s, d);
            if (lane >= d) s += v;
        }
        const uint32_t past = __ballot_sync(0xFFFFFFFFu, s > rest);
        if (past) {
            const int first = __ffs(past) - 1;
            t = t0 + first;
            rest -= __shfl_sync(0xFFFFFFFFu, s - u, first);
            found = true;
            break;
        }
        t = min(t0 + 32, tiles) - 1;
        rest -= __shfl_sync(0xFFFFFFFFu, s, 31);
    }
    x.tile = t;
    x.offset = found && rest > 0 ? rest : 0;  // always found, unless query_start is not ascending and sums wrapped
    return x;
}

// The record of CTA c, whose range starts in tile units [first, last) of the given request.
__device__ __forceinline__ TileRecord tile_record(const AttentionParams& a, const Place& x, int c, const Request& r, int units) {
    TileRecord rec = {};
    const int64_t first = x.unit - x.offset, last = first + units;
    if (c == 0 || x.unit >= x.end || x.offset <= a.tile_units) return rec;
    const int64_t before = share(x.total, c - 1, x.ctas);  // where the CTA before starts
    if (before > first + a.tile_units) return rec;      // an earlier CTA's range starts inside the tile too
    // the CTA whose range holds the tile's last unit
    const int end = static_cast<int>(min((last * x.ctas - 1) / x.total, static_cast<int64_t>(x.ctas - 1)));
    rec.parts = end - c + 2;
    rec.before = 2 * (c - 1) + (before >= first ? 0 : 1);  // its second segment unless its range starts with this tile
    rec.head = x.head;
    rec.tile = x.tile;
    rec.start = r.start;
    rec.rows = r.rows;
    return rec;
}

// The next tile in the numbering after (head, request, tile); false after the last.
template <int kRows, Layout kLayout>
__device__ __forceinline__ bool next_tile(const AttentionParams& a, Request* r, int* head, int* request, int* tile) {
    if (++*tile < Tiles<kRows, kLayout>::count(a, *r)) return true;
    *tile = 0;
    do {
        if (++*request == a.requests) {
            *request = 0;
            if (++*head == a.kv_heads) return false;
        }
        *r = load_request(a, *request);
    } while (r->rows == 0);
    return true;
}

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <typename T>
struct Half2;
template <>
struct Half2<__half> {
    static constexpr uint32_t kExpMask = 0x7C00u;
    static constexpr uint32_t kFormat = 0;  // as an operand of tcgen05.mma
    static constexpr bool kNarrow = true;   // ends at 2^-24 and 65504: weights are given room below, see the kernels
    __device__ static __forceinline__ uint32_t pack(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    __device__ static __forceinline__ float low(uint32_t v) { return __low2float(*reinterpret_cast<const __half2*>(&v)); }
    __device__ static __forceinline__ float high(uint32_t v) { return __high2float(*reinterpret_cast<const __half2*>(&v)); }
};
template <>
struct Half2<__nv_bfloat16> {
    static constexpr uint32_t kExpMask = 0x7F80u;
    static constexpr uint32_t kFormat = 1;
    static constexpr bool kNarrow = false;
    __device__ static __forceinline__ uint32_t pack(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    __device__ static __forceinline__ float low(uint32_t v) { return __uint_as_float(v << 16); }
    __device__ static __forceinline__ float high(uint32_t v) { return __uint_as_float(v & 0xFFFF0000u); }
};

// Joins the partials of every tile that two or more CTAs of the main kernel
// shared, by the records that those left; a warp joins kJoin rows, a lane 4
// columns of them.  The maxima first, then the sums, with the loads of 8 rows
// of partials under way together.  Launched as a dependent of the main kernel
// so that its start overlaps the main kernel's tail.
template <typename T, int kRows, int kDim, Layout kLayout, int kJoin>
__global__ void __launch_bounds__(256) attention_combine_kernel(const AttentionParams a) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    constexpr int kBlocks = kRows / (8 * kJoin);
    constexpr int kAhead = 8 / kJoin;  // partials under way
    const char* ws = static_cast<const char*>(a.workspace);
    const int c = blockIdx.x / kBlocks + 1;
    const TileRecord rec = reinterpret_cast<const TileRecord*>(ws)[c];
    if (rec.parts == 0) return;
    const float* partials = reinterpret_cast<const float*>(ws + workspace_records_bytes(a.ctas));
    constexpr size_t kPartial = static_cast<size_t>(kRows) * (kDim + 2);
    const auto partial = [&](int x) { return partials + (x == 0 ? rec.before : 2 * (c - 1 + x)) * kPartial; };
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d = lane * 4;
    const int row = ((blockIdx.x % kBlocks) * 8 + warp) * kJoin;
    const Request r = {rec.start, rec.rows, 0};
    int i[kJoin], g[kJoin];
    bool valid[kJoin];
    float m[kJoin], ref[kJoin], l[kJoin];
    float4 o[kJoin];
#pragma unroll
    for (int y = 0; y < kJoin; ++y) {
        valid[y] = Tiles<kRows, kLayout>::row(a, r, rec.tile, row + y, &i[y], &g[y]);
        m[y] = -INFINITY;
        l[y] = 0.f;
        o[y] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    if (!valid[0]) return;  // rows past the tile's end come last
    bool nan[kJoin] = {};   // a row that holds NaN, or left by a main kernel that gave up
    for (int x = lane; x < rec.parts; x += 32)
#pragma unroll
        for (int y = 0; y < kJoin; ++y) {
            const float v = valid[y] ? partial(x)[kRows * kDim + row + y] : 0.f;
            m[y] = fmaxf(m[y], v);
            nan[y] = nan[y] || v != v;
        }
#pragma unroll
    for (int y = 0; y < kJoin; ++y) {
#pragma unroll
        for (int b = 16; b; b >>= 1) m[y] = fmaxf(m[y], __shfl_xor_sync(0xFFFFFFFFu, m[y], b));
        ref[y] = __any_sync(0xFFFFFFFFu, nan[y]) ? NAN : m[y] == -INFINITY ? 0.f : m[y];
    }
    for (int x0 = 0; x0 < rec.parts; x0 += kAhead) {
        float pm[8], pl[8];
        float4 q[8];
#pragma unroll
        for (int z = 0; z < 8; ++z) {
            const int x = x0 + z / kJoin, y = z % kJoin;
            pm[z] = -INFINITY;
            pl[z] = 0.f;
            q[z] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (x < rec.parts && valid[y]) {
                const float* p = partial(x);
                pm[z] = p[kRows * kDim + row + y];
                pl[z] = p[kRows * kDim + kRows + row + y];
                if (d < kDim) q[z] = *reinterpret_cast<const float4*>(p + (row + y) * kDim + d);
            }
        }
#pragma unroll
        for (int z = 0; z < 8; ++z) {
            const int y = z % kJoin;
            const float f = exp2_fast(pm[z] - ref[y]);
            l[y] += pl[z] * f;
            o[y].x += q[z].x * f;
            o[y].y += q[z].y * f;
            o[y].z += q[z].z * f;
            o[y].w += q[z].w * f;
        }
    }
#pragma unroll
    for (int y = 0; y < kJoin; ++y) {
        if (!valid[y]) continue;
        const float inv = l[y] == 0.f ? 1.f : 1.f / l[y];
        const int64_t token = r.start + i[y];
        const int head = rec.head * a.group + g[y];
        if (d < kDim) {
            T* out = static_cast<T*>(a.out) + token * a.out_token_stride + head * a.out_head_stride + d;
            *reinterpret_cast<uint2*>(out) =
                make_uint2(Half2<T>::pack(o[y].x * inv, o[y].y * inv), Half2<T>::pack(o[y].z * inv, o[y].w * inv));
        }
        if (lane == 0 && a.lse) a.lse[token * a.heads + head] = l[y] == 0.f ? -INFINITY : (ref[y] + log2f(l[y])) * kLn2;
    }
}

// After a main kernel that may have left partials; the main kernel lets it start early.
template <typename T, int kRows, int kDim, Layout kLayout, int kJoin>
cudaError_t launch_combine(const AttentionParams& a, cudaStream_t stream) {
    if (a.ctas < 2) return cudaSuccess;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>((a.ctas - 1) * (kRows / (8 * kJoin))));
    cfg.blockDim = dim3(256);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, attention_combine_kernel<T, kRows, kDim, kLayout, kJoin>, a);
}

}  // namespace attn
}  // namespace fg
