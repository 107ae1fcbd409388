// fg_key_weights.cu -- the attention weight that each key of the cache was given.
//
// For the rows r of a step (its new tokens' query heads of one kv head), whose
// log-sum-exp the attention left,
//     w[j] = (j < held ? w[j] : 0) + sum over the rows r that see j of e^(scale q_r.k_j - lse_r).
//
// A block is 128 keys of one request and kv head.  The tensor cores compute
// S = K Q^T (tcgen05.mma, 128 keys x up to 256 query rows x dim) into TMEM, where a
// key is a lane: a thread reads its key's scores and adds up their exponentials by
// itself.  Every key is one CTA's, which walks all of its rows: an order that
// depends on the row alone.
//
// Few rows (a decode step) are bound by the keys' way from memory, 2 * dim bytes
// each: two CTAs to an SM, whose rings hold three blocks each.  Keys come by
// 16-byte cp.async, which gathers rows of any pages and strides into the 128-byte
// swizzled layout that tcgen05 reads.  64 ragged decodes, 557 MB: 107 us.  Many
// rows (the last tokens of a prompt) are bound by the special-function units, 16
// exponentials a clock and SM, and by the way of queries and keys before the first
// of them: up to 256 rows are gone through at once, by two threads to a key.
// (mma.sync does a sixteenth of tcgen05's operations here, 8 clocks for m16n8k16:
// 256 rows on 8192 keys took 38 us; with 128 rows at a time and a thread to a key
// 20.)  Blocks are split over the CTAs as in fg_attention.cuh.
//
// A request without rows has its keys from `held` on set to 0 by one walk over them,
// in which no row adds anything (its queries are zeros).
//
// Waits for products are bounded: one that runs out ends the CTA's work, with NaN
// in the keys that are left.
#include <algorithm>

#include "fg_attention.cuh"
#include "fg_cache.h"
#include "fg_tcgen05.cuh"

namespace fg {
namespace attn {
namespace {

constexpr int kRows = 16;    // not looked at: a tile is a request
constexpr int kBlock = 128;  // keys
constexpr int kThreads = 2 * kBlock;
constexpr int kCtasPerSm = 2;
constexpr int kFew = 16;     // rows at a time where there are few
constexpr int kMany = 256;   // and where there are many
constexpr int kColumns = kMany;      // of TMEM, a block's scores
constexpr int kTries = 1 << 18;      // a try that finds nothing takes 4 us: a second

template <int kDim>
struct Ring {
    static constexpr int kPanels = (kDim + 63) / 64;  // 64 columns (128 bytes) each
    static constexpr int kPanel = kBlock * 128;
    static constexpr int kTile = kPanels * kPanel;
    static constexpr int kBytes = kTile + kPanels * kMany * 128;  // a block of keys, the queries
};

template <int kDim>
struct Shared {
    alignas(16) float lse[kMany];  // of the rows in work; inf where a row adds nothing,
    alignas(16) int p[kMany];      // and their positions; -1 there
    int64_t row[2][kBlock];  // where keys' rows begin, in elements, of the block that is loaded next and the one behind it; -1: not there
    float part[kBlock];      // sums over the second half of the rows
    uint64_t done;           // products of a block
    uint64_t drain;
    uint32_t tmem;
};

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool ok) {
    const int n = ok ? 16 : 0;  // 0: the destination is filled with zeros and nothing is read
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// What a block's rows gave to a key.  A request adds to a key once for each group of rows, one after the other, by one thread;
// an addition by the memory system is not waited for, and counts those of requests that share a page too.
__device__ __forceinline__ void add_weight(float* to, float x, bool first) {
    if (first) *to = x;
    else asm volatile("red.relaxed.gpu.global.add.f32 [%0], %1;" ::"l"(to), "f"(x) : "memory");
}

struct Limits {
    int tries, lost;  // of waits; block from which on no products are issued (none: INT32_MAX)
};

template <typename T, int kDim>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) attention_weights_kernel(const AttentionParams a, const WeightsArgs w, const Limits limits) {
    using R = Ring<kDim>;
    extern __shared__ char smem[];
    const int tid = threadIdx.x, warp = tid >> 5;
    const Place pl = locate<kRows, kWhole, kBlock, kThreads, 1>(a, reinterpret_cast<int*>(smem), blockIdx.x, a.ctas);
    if (pl.unit >= pl.end) return;
    __syncthreads();  // what follows overlays the scan
    const uint32_t tiles = (smem_addr(smem) + 1023) & ~1023u;  // the ring, on 1024 bytes
    Shared<kDim>& sh = *reinterpret_cast<Shared<kDim>*>(smem + (tiles - smem_addr(smem)) + R::kBytes);
    if (tid == 0) {
        bar_init(&sh.done, 1);
        bar_init(&sh.drain, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&sh.tmem)), "n"(kColumns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = sh.tmem, mine = tmem + (static_cast<uint32_t>(warp & 3) << 21);  // lanes 32 * (warp % 4) on
    const int key = tid % kBlock, half = tid / kBlock;  // two threads to a key, 128 rows each
    // all of a warp's lanes walk along, so that addresses stay in uniform registers; one issues
    const bool issues = warp == 0 && elect_one();
    const uint32_t tm = uniform(tmem), k_low = uniform(operand_low(tiles, 16)), q_low = uniform(operand_low(tiles + R::kTile, 16));

    int head = pl.head, request = pl.request, tile = pl.tile;
    int64_t unit = pl.unit, tile_first = pl.unit - pl.offset;
    Request r = load_request(a, request);
    uint32_t blocks = 0;  // in the CTA so far
    bool late = false;    // a wait ran out
    while (true) {
        const TileKeys keys = tile_keys<kRows, kWhole, kBlock>(a, r, 0);
        const int64_t tile_last = tile_first + keys.units;
        const int cost = whole_cost(a, r);
        // a block belongs to the CTA whose range holds its first unit
        const auto block_at = [&](int64_t u) {
            return static_cast<int>(min(((u - tile_first + cost - 1) / cost) << a.unit_shift, static_cast<int64_t>(keys.chunks)));
        };
        const int c0 = block_at(unit), c1 = block_at(min(tile_last, pl.end));
        const int32_t* table = a.block_table + request * a.table_stride;
        const int rows = r.rows * a.group, p0 = r.kv_len - r.rows, p1 = r.kv_len - 1;
        const int held = a.held ? max(0, __ldg(a.held + request)) : max(0, p0);
        const T* k_head = static_cast<const T*>(a.k_cache) + head * a.head_stride;
        float* w_head = w.weights.w + head * w.weights.head_stride;
        const auto first_key = [&](int c) { return c < keys.sink_chunks ? c * kBlock : keys.base + (c - keys.sink_chunks) * kBlock; };
        for (int g0 = 0; c0 < c1 && g0 < max(rows, 1); g0 += kMany) {
            const int n = min(rows - g0, kMany), columns = n <= 16 ? 16 : (n + 31) & ~31;
            constexpr int panel = kMany * 128;  // of the queries
            const uint32_t queries = tiles + R::kTile, desc = uniform(instruction<T>(0, false) | (static_cast<uint32_t>(columns >> 3) << 17));
            // the page of key `key` of block c, which the first half of the threads look up for all
            const auto find = [&](int c) {
                const int j = first_key(c) + key, at = j >> a.page_shift;
                if (half || c >= c1 || !(c < keys.sink_chunks ? j < keys.sink_hi : j < keys.hi && (j >= keys.lo || j < a.sinks)) || at >= a.table_width)
                    return -1;
                const int page = __ldg(table + at);
                return static_cast<uint32_t>(page) < static_cast<uint32_t>(a.pages) ? page : -1;
            };
            const auto tell = [&](int c, int page) {
                if (!half) sh.row[c & 1][key] = page < 0 ? -1 : page * a.page_stride + ((first_key(c) + key) & (a.page_size - 1)) * a.token_stride;
            };
            const auto load = [&](int c) {
                const uint32_t to = tiles + (tid >> 3) * 128 + (((tid & 7) ^ ((tid >> 3) & 7)) << 4);
                const T* from = k_head + (tid & 7) * 8;
#pragma unroll
                for (int x = 0; x < kBlock / 32; ++x) {  // key 32 x + tid / 8
                    const int64_t row = sh.row[c & 1][32 * x + (tid >> 3)];
                    const T* src = from + max(row, static_cast<int64_t>(0));
#pragma unroll
                    for (int b = 0; b < R::kPanels; ++b)
                        if (kDim % 64 == 0 || b == 0 || (tid & 7) < 4) copy16(to + b * R::kPanel + x * 4096, src + b * 64, row >= 0);
                }
            };
            __syncthreads();  // the blocks before are done with
            int page = find(c0), next = find(c0 + 1);
            for (int x = tid; x < columns * (kDim / 8); x += kThreads) {
                const int at = x / (kDim / 8), piece = x % (kDim / 8), i = div_group(a, g0 + max(0, min(at, n - 1)));
                const T* src = static_cast<const T*>(a.q) + static_cast<int64_t>(r.start + i) * a.q_token_stride +
                               static_cast<int64_t>(head * a.group + g0 + min(at, n - 1) - i * a.group) * a.q_head_stride + piece * 8;
                copy16(queries + (piece >> 3) * panel + at * 128 + (((piece & 7) ^ (at & 7)) << 4), n > 0 ? src : k_head, n > 0);
            }
            for (int x = tid; x < columns; x += kThreads) {
                const int i = div_group(a, g0 + max(0, min(x, n - 1)));
                const float l =
                    n > 0 ? __ldg(w.lse + static_cast<int64_t>(r.start + i) * a.heads + head * a.group + g0 + min(x, n - 1) - i * a.group) : INFINITY;
                const bool adds = x < n && isfinite(l);
                sh.lse[x] = adds ? l : INFINITY;
                sh.p[x] = adds ? p0 + i : -1;
            }
            tell(c0, page);
            tell(c0 + 1, next);
            __syncthreads();
            load(c0);
            copy_commit();
            for (int c = c0; c < c1; ++c) {
                const int first = first_key(c), last = first + kBlock - 1, j = first + key, here = page;
                copy_wait<0>();
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                tmem_fence_before();
                late = __syncthreads_or(late);
                tmem_fence_after();
                if (warp == 0 && !late && c < limits.lost) {
                    if (issues) {
#pragma unroll
                        for (int k = 0; k < kDim / 16; ++k)
                            mma_smem(tm, k_low + ((k >> 2) * R::kPanel + (k & 3) * 32) / 16, q_low + ((k >> 2) * panel + (k & 3) * 32) / 16, desc, k > 0);
                        mma_commit(&sh.done);
                    }
                    __syncwarp();
                }
                page = next;
                next = find(c + 2);
                if (!late)
                    for (int i = 0; !bar_try(&sh.done, blocks & 1); ++i)
                        if (i >= limits.tries) {
                            late = true;
                            break;
                        }
                ++blocks;
                __syncwarp();
                tmem_fence_after();
                // its keys' place is free: the next ones come while its scores are read
                if (c + 1 < c1 && !late) load(c + 1);
                copy_commit();
                tell(c + 2, next);
                const bool all = last <= p0 && last < (c < keys.sink_chunks ? keys.sink_hi : keys.hi) &&
                                 (a.window < 0 || last < a.sinks || (first >= keys.lo && p1 - first < a.window));
                float sum[4] = {0.f, 0.f, 0.f, 0.f};
                __syncwarp();
                const auto add = [&](const float* s, int x0, int count, bool check) {
#pragma unroll
                    for (int x = 0; x < count; x += 4) {
                        const float4 l4 = *reinterpret_cast<const float4*>(&sh.lse[x0 + x]);
                        const float l[4] = {l4.x, l4.y, l4.z, l4.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            // the difference first: scores and lse may be large, it is not where the weight counts
                            const float v = exp2_fast(fmaf(s[x + e], w.scale, -l[e]) * kLog2e);
                            bool sees = l[e] < INFINITY;
                            if (check) {
                                const int p = sh.p[x0 + x + e];
                                sees = j <= p && (a.window < 0 || p - j < a.window || j < a.sinks);
                            }
                            sum[e] += sees ? v : 0.f;
                        }
                    }
                };
                // 32 columns at a time, the last ones perhaps of nobody's
                for (int x0 = half * 128; x0 < min(columns, half * 128 + 128); x0 += 32) {
                    float s[32];
                    if (columns == 16) tmem_load16(mine, s);
                    else tmem_load32(mine + x0, s);
                    tmem_load_wait();
                    if (columns == 16) add(s, 0, 16, !all);
                    else if (all) add(s, x0, 32, false);
                    else add(s, x0, 32, true);
                }
                tmem_fence_before();
                float total = (sum[0] + sum[1]) + (sum[2] + sum[3]);
                if (columns > 128) {
                    if (half) sh.part[key] = total;
                    __syncthreads();
                    if (!half) total += sh.part[key];
                }
                if (here >= 0) add_weight(w_head + here * w.weights.page_stride + (j & (a.page_size - 1)), late ? NAN : total, g0 == 0 && j >= held);
            }
            copy_wait<0>();
        }
        if (tile_last >= pl.end || !next_tile<kRows, kWhole>(a, &r, &head, &request, &tile)) break;
        unit = tile_first = tile_last;
    }
    // products end before the CTA does, also after a wait that ran out
    tmem_fence_before();
    __syncthreads();
    if (tid == 0) {
        mma_commit(&sh.drain);
        for (int i = 0; i < kTries && !bar_try(&sh.drain, 0); ++i) {
        }
    }
    __syncthreads();
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(kColumns) : "memory");
}

// ---- few rows ----

// The blocks of a CTA's range, one after the other; a tile of more than kFew rows is gone through once for each kFew.  A
// segment is the blocks of one tile and such rows.
struct Walk {
    const AttentionParams& a;
    Request r;
    TileKeys keys;
    int head, request, tile, c, c0, c1, g0, rows;
    int64_t tile_first, end;
    bool more;  // there is a block
    bool opens; // and it is the first of its segment
    __device__ __forceinline__ Walk(const AttentionParams& args, const Place& pl)
        : a(args), head(pl.head), request(pl.request), tile(pl.tile), tile_first(pl.unit - pl.offset), end(pl.end), more(true) {
        r = load_request(a, request);
        set(pl.unit);
    }
    __device__ __forceinline__ void set(int64_t unit) {
        while (true) {
            keys = tile_keys<kRows, kWhole, kBlock>(a, r, 0);
            rows = r.rows * a.group;
            const int cost = whole_cost(a, r);
            const int64_t tile_last = tile_first + keys.units;
            // a block belongs to the CTA whose range holds its first unit
            const auto block_at = [&](int64_t u) {
                return static_cast<int>(min(((u - tile_first + cost - 1) / cost) << a.unit_shift, static_cast<int64_t>(keys.chunks)));
            };
            c = c0 = block_at(unit);
            c1 = block_at(min(tile_last, end));
            g0 = 0;
            opens = true;
            if (c0 < c1) return;
            if (tile_last >= end || !next_tile<kRows, kWhole>(a, &r, &head, &request, &tile)) break;
            unit = tile_first = tile_last;
        }
        more = false;
    }
    __device__ __forceinline__ void next() {
        opens = false;
        if (++c < c1) return;
        opens = true;
        c = c0;
        g0 += kFew;
        if (g0 < rows) return;
        const int64_t tile_last = tile_first + keys.units;
        if (tile_last >= end || !next_tile<kRows, kWhole>(a, &r, &head, &request, &tile)) {
            more = false;
            return;
        }
        tile_first = tile_last;
        set(tile_last);
    }
    __device__ __forceinline__ int first() const { return c < keys.sink_chunks ? c * kBlock : keys.base + (c - keys.sink_chunks) * kBlock; }
    // page of key x of the block, or -1
    __device__ __forceinline__ int page(int x) const {
        if (!more) return -1;
        const int j = first() + x, at = j >> a.page_shift;
        if (!(c < keys.sink_chunks ? j < keys.sink_hi : j < keys.hi && (j >= keys.lo || j < a.sinks)) || at >= a.table_width) return -1;
        const int page = __ldg(a.block_table + request * a.table_stride + at);
        return static_cast<uint32_t>(page) < static_cast<uint32_t>(a.pages) ? page : -1;
    }
};

template <int kDim>
struct FewRing {
    static constexpr int kPanels = Ring<kDim>::kPanels, kPanel = Ring<kDim>::kPanel, kTile = Ring<kDim>::kTile;
    static constexpr int kStages = kDim == 64 ? 5 : 3;
    static constexpr int kQuery = kPanels * kFew * 128;  // of a segment; a multiple of 1024
    static constexpr int kBytes = kStages * (kTile + kQuery);  // as many segments as blocks may be in work
};
template <int kDim>
struct FewShared {
    static constexpr int kStages = FewRing<kDim>::kStages;
    // of the segments that are told of: those in the ring, the one before and the one behind it
    alignas(16) float lse[kStages + 2][kFew];  // inf where a row adds nothing,
    alignas(16) int p[kStages + 2][kFew];      // and their positions; -1 there
    // of the block that is brought next and the one behind it; in elements
    int64_t row[2][kBlock];     // where a key's row begins; -1: it is not there
    int64_t query[2][kFew];     // and a query's, where the block is the first of its segment; -1: there is none
    int opens[2];
    uint64_t done[2];
    uint64_t drain;
    uint32_t tmem;
};

// As the kernel of many rows, with kFew rows at a time and without a pause between tiles: half of the warps bring blocks and
// their tiles' queries kStages - 1 blocks ahead, over the ends of tiles, the other half have a key's scores to a thread.  Between
// two barriers one block's products run, the scores of the one before are read, and its place is filled again.
template <typename T, int kDim>
__global__ void __launch_bounds__(2 * kBlock, kCtasPerSm) attention_weights_few_kernel(const AttentionParams a, const WeightsArgs w, const Limits limits) {
    using R = FewRing<kDim>;
    extern __shared__ char smem[];
    const Place pl = locate<kRows, kWhole, kBlock, 2 * kBlock, 1>(a, reinterpret_cast<int*>(smem), blockIdx.x, a.ctas);
    if (pl.unit >= pl.end) return;
    const bool loads = threadIdx.x >= kBlock;
    const int tid = threadIdx.x % kBlock, warp = tid >> 5;  // of its half
    __syncthreads();  // what follows overlays the scan
    const uint32_t tiles = (smem_addr(smem) + 1023) & ~1023u, queries = tiles + R::kStages * R::kTile;  // on 1024 bytes
    FewShared<kDim>& sh = *reinterpret_cast<FewShared<kDim>*>(smem + (tiles - smem_addr(smem)) + R::kBytes);
    if (threadIdx.x == 0) {
        bar_init(&sh.done[0], 1);
        bar_init(&sh.done[1], 1);
        bar_init(&sh.drain, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (threadIdx.x < 32) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&sh.tmem)), "n"(2 * kFew) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = sh.tmem;
    bool late = false;  // a wait ran out
    const auto wait = [&](int block) {  // for its products
        if (late) return;
        for (int i = 0; !bar_try(&sh.done[block & 1], (block >> 1) & 1); ++i)
            if (i >= limits.tries) {
                late = true;
                break;
            }
    };
    Walk at(a, pl);
    if (loads) {
        using Sh = FewShared<kDim>;
        // A block is told of, a key to a thread, one round before it is brought, 16 bytes (of each 128) of 8 keys to a thread;
        // its page is read another round before.
        const uint32_t to = tiles + (tid >> 3) * 128 + (((tid & 7) ^ ((tid >> 3) & 7)) << 4);
        const T* from = static_cast<const T*>(a.k_cache) + (tid & 7) * 8;
        int page = at.page(tid), segment = -1, told = 0, brought = 0, stage = 0, q_slot = -1;
        const auto tell = [&] {
            if (!at.more) return;
            sh.row[told & 1][tid] =
                page < 0 ? -1 : page * a.page_stride + ((at.first() + tid) & (a.page_size - 1)) * a.token_stride + at.head * a.head_stride;
            if (tid == 0) sh.opens[told & 1] = at.opens;
            if (at.opens && ++segment == Sh::kStages + 2) segment = 0;
            if (at.opens && tid < kFew) {
                // the last row again past the end
                const int n = max(0, at.g0 + min(tid, min(kFew, at.rows - at.g0) - 1)), i = div_group(a, n), g = n - i * a.group;
                const float l = at.rows > 0 ? __ldg(w.lse + static_cast<int64_t>(at.r.start + i) * a.heads + at.head * a.group + g) : INFINITY;
                const bool adds = at.g0 + tid < at.rows && isfinite(l);
                sh.query[told & 1][tid] =
                    at.rows > 0 ? static_cast<int64_t>(at.r.start + i) * a.q_token_stride + static_cast<int64_t>(at.head * a.group + g) * a.q_head_stride : -1;
                sh.lse[segment][tid] = adds ? l : INFINITY;
                sh.p[segment][tid] = adds ? at.r.kv_len - at.r.rows + i : -1;
            }
            ++told;
            at.next();
            page = at.page(tid);
        };
        const auto bring = [&] {
            if (brought < told) {
                if (sh.opens[brought & 1]) {
                    if (++q_slot == R::kStages) q_slot = 0;
#pragma unroll
                    for (int x = tid; x < kFew * (kDim / 8); x += kBlock) {
                        const int row = x / (kDim / 8), piece = x % (kDim / 8);
                        const int64_t query = sh.query[brought & 1][row];
                        copy16(queries + q_slot * R::kQuery + (piece >> 3) * (kFew * 128) + row * 128 + (((piece & 7) ^ (row & 7)) << 4),
                               query >= 0 ? static_cast<const T*>(a.q) + query + piece * 8 : from, query >= 0 && !late);
                    }
                }
#pragma unroll
                for (int x = 0; x < kBlock / 16; ++x) {
                    const int64_t row = sh.row[brought & 1][16 * x + (tid >> 3)];
                    const T* src = from + max(row, static_cast<int64_t>(0));
#pragma unroll
                    for (int b = 0; b < R::kPanels; ++b)
                        if (kDim % 64 == 0 || b == 0 || (tid & 7) < 4) copy16(to + stage * R::kTile + b * R::kPanel + x * 2048, src + b * 64, row >= 0 && !late);
                }
                if (++stage == R::kStages) stage = 0;
                ++brought;
            }
            copy_commit();
        };
        const auto half_sync = [] { asm volatile("bar.sync 1, %0;" ::"n"(kBlock) : "memory"); };
        tell();
        for (int x = 0; x < R::kStages - 1; ++x) {
            half_sync();
            bring();
            tell();
        }
        for (int x = 0; x < brought; ++x) {
            copy_wait<R::kStages - 2>();
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            late = __syncthreads_or(late);
            if (x > 0) wait(x - 1);
            bring();  // where block x - 1 was
            tell();
        }
        copy_wait<0>();
    } else {
        const uint32_t lanes = tmem + (static_cast<uint32_t>(warp) << 21);  // lanes 32 * warp on
        int page = at.page(tid), segment = -1;
        // what is read of the walk after it has gone on: the block whose scores are read next
        int head = 0, first = 0, here = -1, p0 = 0, p1 = 0, rows = 0;
        bool all = false, fresh = false;
        const auto take = [&] {
            if (at.opens && ++segment == R::kStages + 2) segment = 0;
            head = at.head;
            first = at.first();
            here = page;
            p0 = at.r.kv_len - at.r.rows;
            p1 = at.r.kv_len - 1;
            rows = min(kFew, at.rows - at.g0);
            const int last = first + kBlock - 1, held = a.held ? max(0, __ldg(a.held + at.request)) : max(0, p0);
            all = last <= p0 && last < (at.c < at.keys.sink_chunks ? at.keys.sink_hi : at.keys.hi) &&
                  (a.window < 0 || last < a.sinks || (first >= at.keys.lo && p1 - first < a.window));
            fresh = at.g0 == 0 && first + tid >= held;
            at.next();
            page = at.page(tid);
        };
        const auto finish = [&](int block) {
            wait(block);
            __syncwarp();
            tmem_fence_after();
            float s[kFew], sum[4] = {0.f, 0.f, 0.f, 0.f};
            tmem_load16(lanes + (block & 1) * kFew, s);
            tmem_load_wait();
            const int j = first + tid;
#pragma unroll
            for (int x = 0; x < kFew; x += 4)
                if (x < rows) {
                    const float4 l4 = *reinterpret_cast<const float4*>(&sh.lse[segment][x]);
                    const float l[4] = {l4.x, l4.y, l4.z, l4.w};
                    int p[4] = {0, 0, 0, 0};
                    if (!all) {
                        const int4 p4 = *reinterpret_cast<const int4*>(&sh.p[segment][x]);
                        p[0] = p4.x, p[1] = p4.y, p[2] = p4.z, p[3] = p4.w;
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        // the difference first: scores and lse may be large, it is not where the weight counts
                        const float v = exp2_fast(fmaf(s[x + e], w.scale, -l[e]) * kLog2e);
                        const bool sees = all ? l[e] < INFINITY : j <= p[e] && (a.window < 0 || p[e] - j < a.window || j < a.sinks);
                        sum[e] += sees ? v : 0.f;
                    }
                }
            tmem_fence_before();
            if (here >= 0)
                add_weight(w.weights.w + head * w.weights.head_stride + here * w.weights.page_stride + (j & (a.page_size - 1)),
                           late ? NAN : (sum[0] + sum[1]) + (sum[2] + sum[3]), fresh);
        };
        // all of a warp's lanes walk along, so that addresses stay in uniform registers; one issues
        const bool issues = warp == 0 && elect_one();
        const uint32_t tm = uniform(tmem), k_low = uniform(operand_low(tiles, 16)), q_low = uniform(operand_low(queries, 16));
        constexpr uint32_t kDesc = instruction<T>(kFew, false);
        int stage = 0, q_slot = -1;
        for (int x = 0; at.more; ++x) {
            tmem_fence_before();
            late = __syncthreads_or(late);
            tmem_fence_after();
            if (at.opens && ++q_slot == R::kStages) q_slot = 0;
            if (warp == 0 && !late && x < limits.lost) {
                const uint32_t kb = uniform(k_low + stage * (R::kTile / 16)), qb = uniform(q_low + q_slot * (R::kQuery / 16)), d = uniform(tm + (x & 1) * kFew);
                if (issues) {
#pragma unroll
                    for (int k = 0; k < kDim / 16; ++k)
                        mma_smem(d, kb + ((k >> 2) * R::kPanel + (k & 3) * 32) / 16, qb + ((k >> 2) * kFew * 128 + (k & 3) * 32) / 16, kDesc, k > 0);
                    mma_commit(&sh.done[x & 1]);
                }
                __syncwarp();
            }
            if (++stage == R::kStages) stage = 0;
            if (x > 0) finish(x - 1);
            take();
            if (!at.more) finish(x);
        }
        tmem_fence_before();
    }
    // products end before the CTA does, also after a wait that ran out
    late = __syncthreads_or(late);
    if (threadIdx.x == 0 && late) {
        mma_commit(&sh.drain);
        for (int i = 0; i < kTries && !bar_try(&sh.drain, 0); ++i) {
        }
    }
    __syncthreads();
    if (threadIdx.x < 32) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(2 * kFew) : "memory");
}

Limits g_limits = {kTries, INT32_MAX};

template <typename T, int kDim, bool kFewRows>
cudaError_t launch(AttentionParams a, const WeightsArgs& w, cudaStream_t stream) {
    a.base_align = kBlock;
    a.tile_units = 0;
    a.tile_rows = kFewRows ? kFew : kMany;
    a.ctas *= kCtasPerSm;
    a.held = w.held;
    // the units of a kv head are summed in 32 bits
    const int64_t keys = std::min<int64_t>(static_cast<int64_t>(a.table_width) * a.page_size, INT32_MAX);
    const int64_t costs = a.requests + static_cast<int64_t>(a.tokens) * a.group / a.tile_rows;
    a.unit_shift = 0;
    while (a.unit_shift < 24 && costs * (((keys / kBlock + 3) >> a.unit_shift) + 1) > INT32_MAX) ++a.unit_shift;
    constexpr int kBytes = 1024 + (kFewRows ? FewRing<kDim>::kBytes + static_cast<int>(sizeof(FewShared<kDim>))
                                            : Ring<kDim>::kBytes + static_cast<int>(sizeof(Shared<kDim>)));
    static_assert((kBytes + 1024) * kCtasPerSm <= 228 * 1024, "two CTAs' shared memory");
    constexpr int most = std::max(kBytes, locate_bytes(kMaxRequests));
    const int bytes = std::max(kBytes, locate_bytes(a.requests));
    const auto kernel = kFewRows ? attention_weights_few_kernel<T, kDim> : attention_weights_kernel<T, kDim>;
    static SmemOnce once;
    const cudaError_t e = once.set(reinterpret_cast<const void*>(kernel), most);
    if (e != cudaSuccess) return e;
    kernel<<<a.ctas, kFewRows ? 2 * kBlock : kThreads, bytes, stream>>>(a, w, g_limits);
    return cudaGetLastError();
}

// Where requests have more than 16 rows on average, up to 256 rows are gone through at once.  us, few / many, 4 heads to a kv
// head of 128:
//     rows    1 request, 8000 keys    8 of 4000        64 of 2000
//     8       10.7 / 10.4             22.2 / 23.7      58.9 / 63.9
//     16      11.5 / 10.5             23.7 / 23.8      60.8 / 63.7
//     20      14.7 / 10.9             32.0 / 24.3      97.9 / 64.6
//     64      20.9 / 12.0             57.1 / 26.2      191 / 70
//     256     57 / 18                 192 / 42         771 / 137
// It is the average because lengths are not known here: a prompt's 256 rows beside 63 decodes go through their keys 16 times.
template <typename T, int kDim>
cudaError_t by_rows(const AttentionParams& a, const WeightsArgs& w, cudaStream_t s) {
    return static_cast<int64_t>(a.tokens) * a.group > static_cast<int64_t>(a.requests) * kFew ? launch<T, kDim, false>(a, w, s) : launch<T, kDim, true>(a, w, s);
}

template <typename T>
cudaError_t by_dim(const AttentionParams& a, const WeightsArgs& w, cudaStream_t s) {
    return a.dim == 64 ? by_rows<T, 64>(a, w, s) : a.dim == 96 ? by_rows<T, 96>(a, w, s) : by_rows<T, 128>(a, w, s);
}

}  // namespace
}  // namespace attn

void set_key_weights_waits(int lost, int tries) {
    attn::g_limits = {tries < 0 ? attn::kTries : tries, lost < 0 ? INT32_MAX : lost};
}

cudaError_t launch_attention_weights(const AttentionParams& a, const WeightsArgs& w, cudaStream_t stream) {
    return a.dtype == FG_DTYPE_BF16 ? attn::by_dim<__nv_bfloat16>(a, w, stream) : attn::by_dim<__half>(a, w, stream);
}

}  // namespace fg
