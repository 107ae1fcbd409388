// fg_key_weights.cu -- the attention weight that each key of the cache was given.
//
// For the rows r of a step (its new tokens' query heads of one kv head), whose
// log-sum-exp the attention left,
//     w[j] = (j < held ? w[j] : 0) + sum over the rows r that see j of e^(scale q_r.k_j - lse_r).
//
// A block is 128 keys of one request and kv head.  The tensor cores compute
// S = K Q^T (tcgen05.mma, 128 keys x up to 128 query rows x dim) into TMEM, where a
// key is a lane: each of the CTA's 128 threads reads its key's scores and adds up
// their exponentials by itself.  Every key is one CTA's, which walks all of its
// rows, 128 at a time: no atomics, and an order that depends on the row alone.
//
// Few rows (a decode step) are bound by the keys' way from memory, 2 * dim bytes
// each: two CTAs to an SM, whose rings hold up to three blocks each.  Keys come by
// 16-byte cp.async, which gathers rows of any pages and strides into the 128-byte
// swizzled layout that tcgen05 reads; pages are looked up a block ahead of the
// copies.  Many rows (the last tokens of a prompt) are bound by the special-function
// units, 16 exponentials a clock and SM: the products of the next block run beside
// them.  (mma.sync does a sixteenth of tcgen05's operations here, 8 clocks for
// m16n8k16: 256 rows on 8192 keys took 38 us.)  Blocks are split over the CTAs as
// in fg_attention.cuh.
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
constexpr int kThreads = 128;
constexpr int kCtasPerSm = 2;
constexpr int kFew = 32;     // up to so many rows' queries lie behind the whole ring,
constexpr int kMany = 128;   // more, up to so many at a time, in its last places
constexpr int kColumns = 2 * kMany;  // of TMEM: two blocks' scores
constexpr int kTries = 1 << 18;      // a try that finds nothing takes 4 us: a second

template <int kDim>
struct Ring {
    static constexpr int kPanels = (kDim + 63) / 64;  // 64 columns (128 bytes) each
    static constexpr int kPanel = kBlock * 128;
    static constexpr int kTile = kPanels * kPanel;
    static constexpr int kStages = kDim == 64 ? 6 : 3;
    static constexpr int kStagesMany = kDim == 64 ? 4 : 2;
    static constexpr int kLook = kStages + 1;         // blocks whose rows are known
    static constexpr int kQueriesFew = kStages * kTile, kQueriesMany = kStagesMany * kTile;
    static constexpr int kBytes = kQueriesFew + kPanels * kFew * 128;
    static_assert(kBytes - kQueriesMany >= kPanels * kMany * 128, "the queries' room");
};

template <int kDim>
struct Shared {
    alignas(16) float lse[kMany];  // of the rows in work; inf where a row adds nothing,
    alignas(16) int p[kMany];      // and their positions; -1 there
    int64_t row[Ring<kDim>::kLook][kBlock];  // where a key's row begins, in elements; -1: it is not there
    uint64_t done[2];              // products of a block
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
// until all but the last n groups have arrived
__device__ __forceinline__ void copy_wait_but(int n) {
    if (n >= 4) copy_wait<4>();
    else if (n == 3) copy_wait<3>();
    else if (n == 2) copy_wait<2>();
    else if (n == 1) copy_wait<1>();
    else copy_wait<0>();
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
        bar_init(&sh.done[0], 1);
        bar_init(&sh.done[1], 1);
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
    const uint32_t tmem = sh.tmem, mine = tmem + (static_cast<uint32_t>(warp) << 21);  // lanes 32 * warp on

    int head = pl.head, request = pl.request, tile = pl.tile;
    int64_t unit = pl.unit, tile_first = pl.unit - pl.offset;
    Request r = load_request(a, request);
    uint32_t issued = 0;  // blocks in the CTA so far: the number of a block says which scores and barrier are its own
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
        for (int g0 = 0; c0 < c1 && g0 < rows; g0 += kMany) {
            const int n = min(rows - g0, kMany), columns = n <= 16 ? 16 : (n + 31) & ~31;
            const int stages = rows <= kFew ? R::kStages : R::kStagesMany;
            const uint32_t queries = tiles + (rows <= kFew ? R::kQueriesFew : R::kQueriesMany);
            const int panel = (rows <= kFew ? kFew : kMany) * 128;  // of the queries
            // the page of this thread's key of block c, which all look up for one another
            const auto find = [&](int c) {
                if (c >= c1) return -1;
                const int j = first_key(c) + tid, at = j >> a.page_shift;
                if (!(c < keys.sink_chunks ? j < keys.sink_hi : j < keys.hi && (j >= keys.lo || j < a.sinks)) || at >= a.table_width) return -1;
                return __ldg(table + at);
            };
            const auto row_of = [&](int c, int page) -> int64_t {
                if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(a.pages)) return -1;
                return page * a.page_stride + ((first_key(c) + tid) & (a.page_size - 1)) * a.token_stride;
            };
            // its weight; beyond the first rows, with what they gave it
            const auto weight = [&](int c, int page) -> float* {
                if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(a.pages)) return nullptr;
                return w_head + page * w.weights.page_stride + ((first_key(c) + tid) & (a.page_size - 1));
            };
            const auto so_far = [&](int c, const float* x) { return x && (g0 > 0 || first_key(c) + tid < held) ? *x : 0.f; };
            const auto load = [&](const int64_t* row, uint32_t to) {
                to += (tid >> 3) * 128 + (((tid & 7) ^ ((tid >> 3) & 7)) << 4);
                const T* from = k_head + (tid & 7) * 8;
#pragma unroll
                for (int x = 0; x < kBlock / 16; ++x) {  // key 16 x + tid / 8
                    const int64_t at = row[16 * x + (tid >> 3)];
                    const T* src = from + max(at, static_cast<int64_t>(0));
#pragma unroll
                    for (int b = 0; b < R::kPanels; ++b)
                        if (kDim % 64 == 0 || b == 0 || (tid & 7) < 4) copy16(to + b * R::kPanel + x * 2048, src + b * 64, at >= 0);
                }
            };
            __syncthreads();  // the blocks before are done with
            // pages of the blocks ahead: looked up kLook blocks before they are read, told kLook - 1 before
            int look[R::kLook + 1];
#pragma unroll
            for (int x = 0; x <= R::kLook; ++x) look[x] = find(c0 + x);
            for (int x = tid; x < columns * (kDim / 8); x += kThreads) {
                const int at = x / (kDim / 8), piece = x % (kDim / 8), i = div_group(a, g0 + min(at, n - 1));
                const T* src = static_cast<const T*>(a.q) + static_cast<int64_t>(r.start + i) * a.q_token_stride +
                               static_cast<int64_t>(head * a.group + g0 + min(at, n - 1) - i * a.group) * a.q_head_stride + piece * 8;
                copy16(queries + (piece >> 3) * panel + at * 128 + (((piece & 7) ^ (at & 7)) << 4), src, true);
            }
            for (int x = tid; x < columns; x += kThreads) {
                const int i = div_group(a, g0 + min(x, n - 1));
                const float l = __ldg(w.lse + static_cast<int64_t>(r.start + i) * a.heads + head * a.group + g0 + min(x, n - 1) - i * a.group);
                const bool adds = x < n && isfinite(l);
                sh.lse[x] = adds ? l : INFINITY;
                sh.p[x] = adds ? p0 + i : -1;
            }
#pragma unroll
            for (int x = 0; x < R::kLook; ++x) sh.row[x][tid] = row_of(c0 + x, look[x]);
            __syncthreads();
            for (int x = 0; x < stages; ++x) {
                if (c0 + x < c1) load(sh.row[x], tiles + x * R::kTile);
                copy_commit();
            }
            float* to = weight(c0, look[0]);
            float before = so_far(c0, to);
            // in turn: where rows are told (of block c in finish(c)), where those of block c + stages are, its keys' place
            int told = 0, next = stages, stage = 0;
            const auto finish = [&](int c, uint32_t number) {
                const int first = first_key(c), last = first + kBlock - 1, j = first + tid;
                if (!late)
                    for (int i = 0; !bar_try(&sh.done[number & 1], (number >> 1) & 1); ++i)
                        if (i >= limits.tries) {
                            late = true;
                            break;
                        }
                __syncwarp();
                tmem_fence_after();
                // its keys' place is free
                if (c + stages < c1 && !late) load(sh.row[next], tiles + stage * R::kTile);
                copy_commit();
                sh.row[told][tid] = row_of(c + R::kLook, look[R::kLook]);
                if (++told == R::kLook) told = 0;
                if (++next == R::kLook) next = 0;
                if (++stage == stages) stage = 0;
#pragma unroll
                for (int x = 0; x < R::kLook; ++x) look[x] = look[x + 1];
                look[R::kLook] = find(c + R::kLook + 1);
                const float old = before;
                float* const here = to;
                to = weight(c + 1, look[0]);
                before = so_far(c + 1, to);
                const bool all = last <= p0 && last < (c < keys.sink_chunks ? keys.sink_hi : keys.hi) &&
                                 (a.window < 0 || last < a.sinks || (first >= keys.lo && p1 - first < a.window));
                float sum[4] = {0.f, 0.f, 0.f, 0.f};
                __syncwarp();
                const uint32_t scores = mine + (number & 1) * kMany;
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
                if (columns <= 16) {
                    float s[16];
                    tmem_load16(scores, s);
                    tmem_load_wait();
#pragma unroll
                    for (int x0 = 0; x0 < 16; x0 += 4)
                        if (x0 < n) {
                            if (all) add(s + x0, x0, 4, false);
                            else add(s + x0, x0, 4, true);
                        }
                } else {
                    // 32 columns at a time, the last ones perhaps of nobody's
                    for (int x0 = 0; x0 < columns; x0 += 32) {
                        float s[32];
                        tmem_load32(scores + x0, s);
                        tmem_load_wait();
                        if (all) add(s, x0, 32, false);
                        else add(s, x0, 32, true);
                    }
                }
                tmem_fence_before();
                if (here) *here = late ? NAN : old + ((sum[0] + sum[1]) + (sum[2] + sum[3]));
            };
            int at = 0;
            for (int c = c0; c < c1; ++c) {
                copy_wait_but(c == c0 ? stages - 1 : stages - 2);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                tmem_fence_before();
                late = __syncthreads_or(late);
                tmem_fence_after();
                if (tid == 0 && !late && c < limits.lost) {
                    const uint32_t d = tmem + (issued & 1) * kMany, q_low = operand_low(queries, 16);
                    const uint32_t k_low = operand_low(tiles + at * R::kTile, 16);
                    const uint32_t idesc = instruction<T>(0, false) | (static_cast<uint32_t>(columns >> 3) << 17);
#pragma unroll
                    for (int k = 0; k < kDim / 16; ++k)
                        mma_smem(d, k_low + ((k >> 2) * R::kPanel + (k & 3) * 32) / 16, q_low + ((k >> 2) * panel + (k & 3) * 32) / 16, idesc, k > 0);
                    mma_commit(&sh.done[issued & 1]);
                }
                ++issued;
                if (++at == stages) at = 0;
                if (c > c0) finish(c - 1, issued - 2);
            }
            finish(c1 - 1, issued - 1);
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

Limits g_limits = {kTries, INT32_MAX};

template <typename T, int kDim>
cudaError_t launch(AttentionParams a, const WeightsArgs& w, cudaStream_t stream) {
    a.base_align = kBlock;
    a.tile_units = 0;
    a.ctas *= kCtasPerSm;
    a.held = w.held;
    // the units of a kv head are summed in 32 bits
    const int64_t keys = std::min<int64_t>(static_cast<int64_t>(a.table_width) * a.page_size, INT32_MAX);
    const int64_t costs = a.requests + ((static_cast<int64_t>(a.tokens) * a.group) >> kWholeRows);
    a.unit_shift = 0;
    while (a.unit_shift < 24 && costs * (((keys / kBlock + 3) >> a.unit_shift) + 1) > INT32_MAX) ++a.unit_shift;
    constexpr int kBytes = Ring<kDim>::kBytes + 1024 + static_cast<int>(sizeof(Shared<kDim>));
    static_assert((kBytes + 1024) * kCtasPerSm <= 228 * 1024, "two CTAs' shared memory");
    constexpr int most = std::max(kBytes, locate_bytes(kMaxRequests));
    const int bytes = std::max(kBytes, locate_bytes(a.requests));
    static SmemOnce once;
    const cudaError_t e = once.set(reinterpret_cast<const void*>(attention_weights_kernel<T, kDim>), most);
    if (e != cudaSuccess) return e;
    attention_weights_kernel<T, kDim><<<a.ctas, kThreads, bytes, stream>>>(a, w, g_limits);
    return cudaGetLastError();
}

template <typename T>
cudaError_t by_dim(const AttentionParams& a, const WeightsArgs& w, cudaStream_t s) {
    return a.dim == 64 ? launch<T, 64>(a, w, s) : a.dim == 96 ? launch<T, 96>(a, w, s) : launch<T, 128>(a, w, s);
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
