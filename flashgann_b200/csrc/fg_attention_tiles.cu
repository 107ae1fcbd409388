// fg_attention_tiles.cu -- attention of many query rows over the paged cache:
// prompts' chunks, and decodes that share a call with them.
//
// A tile is 256 query rows of one kv head (tokens x heads of the group), two
// halves of 128; a block is 128 keys.  For each block and half the tensor
// cores compute S = Q K^T into TMEM (tcgen05.mma, 128 x 128 x dim), the half's
// warpgroup turns S into weights P = 2^(scale S - m) in place, one row to a
// thread, and the tensor cores add P V to the output in TMEM with P as their
// TMEM operand.  TMEM holds exactly S/P and O of both halves: 4 x 128 columns.
//
// Warp roles (16 warps, one CTA per SM):
//   0-3, 4-7   softmax of half 0 and 1 (200 registers a thread)
//   8-11       look through the V tiles that not all rows see whole, see clear_masked
//   12         issues the products
//   13, 14     load K and V with TMA, one copy for each page (or 64 rows of it) and
//              64 columns, into a ring of tiles in the 128-byte swizzled layout
//              that tcgen05 reads; a page that is not there is a coordinate out
//              of range, which TMA fills with zeros
//   15         loads the tile's query rows, one copy for each 64 columns: a tile
//              is the group's heads of consecutive tokens, a box of the queries
// The two halves run in antiphase: while half 0's weights are computed the
// tensor cores work on half 1.
//
// What bounds it: per block and half 4 * 128 * 128 * dim operations, 1024
// cycles of the tensor pipe at dim 128, and 128 * 128 exponentials, 1024
// cycles of the SM's special-function units.  (A polynomial for some of them
// was slower: the special-function units are not what is short, issue slots and
// latencies are.)
//
// Measured: 2048 tokens on 8192 keys, 32 heads on 8, dim 128, bf16: 276 to 281
// us, 1100 to 1120 TFLOP/s on the device.  A block takes 3650 cycles, of which the tensor
// pipe is busy for 2048: each half waits for its own weights.
//
// The base that the weights are relative to is raised only when the running
// maximum is more than 2^8 above what it was then: O and the sum are scaled,
// which costs a round trip of O through registers.  Weights up to 2^8 keep
// their relative precision in both 16-bit types, and the 32-bit sums have room.
// float16 ends at 2^-24: a weight below 2^-25 would be zero in the product
// while the sum counts it, and many keys far below the maximum would be lost.
// Its base is 2^7 below the maximum, so that weights reach 2^15 and those of
// 2^-32 of the maximum still count.  It costs nothing: sums, partials and lse
// are relative to the base in any case.
//
// Every wait is bounded: one that runs out marks the CTA, which ends the other
// roles' waits too.  Nothing is loaded or issued from then on, and the warps that
// did leave once their copies and products have ended; the softmax warps walk on
// to the end of the CTA's range without waiting and write NaN for all of its rows
// that were not stored before.
#include <algorithm>

#include <cuda.h>

#include "fg_attention.cuh"

namespace fg {
namespace attn {
namespace {

constexpr int kRows = 256;
constexpr int kHalf = 128;
constexpr int kBlock = 128;  // keys
constexpr int kThreads = 512;
constexpr int kSlots = 5;    // see Loader::block; K and V tiles in the ring: two blocks and a half
constexpr int kTileBlocks = 3;  // a tile costs about as much as that many blocks beside its own (1 to 4 measured)
constexpr float kRaise = 8.f;
template <typename T>
constexpr float kLift = Half2<T>::kNarrow ? 7.f : 0.f;  // log2 of a float16 weight at the maximum

template <int kDim>
struct Smem {
    static constexpr int kPanels = (kDim + 63) / 64;      // 64 columns (128 bytes) each
    static constexpr int kPanelRows = kBlock * 128;       // bytes of a panel of a K or V tile
    static constexpr int kTile = kPanels * kPanelRows;
    static constexpr int kQPanel = kRows * 128;
    static constexpr int kQ = kPanels * kQPanel;
    static constexpr int kRing = kSlots * kTile;
    static constexpr int kBytes = kQ + kRing + 1024;      // + 1024: the tiles start on 1024 bytes
};

struct Shared {
    uint64_t full[kSlots];
    uint64_t used[4];       // of block n % 4: its V tile, the next block's K tile and, of a segment's first block, its K tile are free
    uint64_t raw[kSlots];   // a V tile that is to be looked through has arrived; `full` follows when that is done
    uint64_t q_full, q_empty;
    uint64_t s_full[2], p_full[2][2], pv_done[2];  // p_full: of each half, the weights of keys 0-63 and 64-127
    uint64_t drain;
    uint32_t tmem;
    int stalled;            // a wait ran out
    int missing[4];         // 1 + number of the block that has keys in range without a page
    uint32_t boxes[4];      // of block n % 4: bit i, copy i found its page
    int nonfinite[kSlots];  // 1 + number of the ring item whose V tile infinities or NaN were taken out of
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void bar_init(uint64_t* b, int count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(b)), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t* b) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(b)) : "memory");
}
__device__ __forceinline__ void bar_arrive3(uint64_t* b) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], 3;" ::"r"(smem_addr(b)) : "memory");
}
__device__ __forceinline__ bool bar_try(uint64_t* b, int parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_addr(b)), "r"(parity)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ void bar_expect(uint64_t* b, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_addr(b)), "r"(bytes) : "memory");
}
// A try that finds nothing takes 4 us (measured), so that the usual limit is a
// second; a wait between two blocks lasts microseconds.
constexpr int kWaitTries = 1 << 18;
__device__ __forceinline__ volatile int* stalled(Shared* sh) { return &sh->stalled; }
// For the softmax warps.  A lane whose wait runs out, or that finds that
// another's did, is late and goes on without waiting any more: no vote, and the
// warp's lanes stay together.
__device__ __forceinline__ void bar_wait(const AttentionParams& a, uint64_t* b, int parity, Shared* sh, bool* late) {
    if (*late) return;
    for (int i = 0; !bar_try(b, parity); ++i)
        if (i >= a.wait_tries || *stalled(sh)) {
            *stalled(sh) = 1;
            *late = true;
            return;
        }
}
// For the issuing warp.  false in all lanes: the wait ran out, or another's did.
__device__ __forceinline__ bool bar_wait_all(const AttentionParams& a, uint64_t* b, int parity, Shared* sh) {
    for (int i = 0; !__all_sync(0xFFFFFFFFu, bar_try(b, parity)); ++i)
        if (__any_sync(0xFFFFFFFFu, i >= a.wait_tries || *stalled(sh))) {
            *stalled(sh) = 1;
            return false;
        }
    return true;
}
// For waits that nothing hurries: leaves the issue slots to the other warps.
// They may last as long as a tile (a V tile to be looked through comes after all
// others: 16 ms in a context of a million keys); where one does not end, one of
// the other kind does not either, which runs out first.
__device__ __forceinline__ bool bar_wait_idle(const AttentionParams& a, uint64_t* b, int parity, Shared* sh) {
    for (int i = 0; !__all_sync(0xFFFFFFFFu, bar_try(b, parity)); ++i) {
        if (__any_sync(0xFFFFFFFFu, i >= a.wait_tries * 256 || *stalled(sh))) {
            *stalled(sh) = 1;
            return false;
        }
        __nanosleep(50);
    }
    return true;
}
// Before a warp leaves: what it started itself, and what ends by itself.
__device__ __forceinline__ void bar_wait_own(uint64_t* b, int parity) {
    for (int i = 0; i < kWaitTries && !bar_try(b, parity); ++i) {
    }
}

// ---- tcgen05 ----

__device__ __forceinline__ void tmem_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }

// 32 columns of this warp's 32 lanes, one row to a thread
__device__ __forceinline__ void tmem_load32(uint32_t addr, float* r) {
    uint32_t* u = reinterpret_cast<uint32_t*>(r);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
          "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]),
          "=r"(u[17]), "=r"(u[18]), "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]),
          "=r"(u[25]), "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_store32(uint32_t addr, const uint32_t* u) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::"r"(
            u[0]),
        "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]), "r"(u[10]),
        "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15]), "r"(u[16]), "r"(u[17]), "r"(u[18]), "r"(u[19]),
        "r"(u[20]), "r"(u[21]), "r"(u[22]), "r"(u[23]), "r"(u[24]), "r"(u[25]), "r"(u[26]), "r"(u[27]), "r"(u[28]),
        "r"(u[29]), "r"(u[30]), "r"(u[31]), "r"(addr)
        : "memory");
}
__device__ __forceinline__ void tmem_load16(uint32_t addr, float* r) {
    uint32_t* u = reinterpret_cast<uint32_t*>(r);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
          "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_store16(uint32_t addr, const uint32_t* u) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(u[0]),
        "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]), "r"(u[10]),
        "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15]), "r"(addr)
        : "memory");
}
__device__ __forceinline__ void tmem_load_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Shared-memory operand descriptor, 128-byte swizzle: start address and strides
// in 16-byte units.  K-major (Q, K): groups of 8 rows 1024 bytes apart.
// MN-major (V): 64-column panels `panel` bytes apart, groups of 8 keys 1024
// bytes apart.  The upper word is the same for all; advancing the start address
// adds to the lower.
constexpr uint32_t kOperandHigh = (1024 >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t operand_low(uint32_t addr, uint32_t panel) { return (addr >> 4) | ((panel >> 4) << 16); }

template <typename T>
__host__ __device__ constexpr uint32_t instruction(int n, bool b_mn_major) {
    const uint32_t f = Half2<T>::kFormat;
    return (1u << 4) | (f << 7) | (f << 10) | (b_mn_major ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) |
           (static_cast<uint32_t>(kHalf >> 4) << 24);
}

__device__ __forceinline__ void mma_smem(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.u32 p, %4, 0;\n\tmov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(add), "r"(kOperandHigh)
        : "memory");
}
__device__ __forceinline__ void mma_tmem(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tsetp.ne.u32 p, %4, 0;\n\tmov.b64 b, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(add), "r"(kOperandHigh)
        : "memory");
}
__device__ __forceinline__ bool elect_one() {
    uint32_t is;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(is));
    return is != 0;
}
// a value that all lanes share, in a form that the compiler knows to be shared
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __shfl_sync(0xFFFFFFFFu, x, 0); }
// arrives on b when all products issued so far are done
__device__ __forceinline__ void mma_commit(uint64_t* b) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(b)) : "memory");
}

// TMEM columns
__device__ __forceinline__ constexpr uint32_t score_column(int half) { return half * 128; }
__device__ __forceinline__ constexpr uint32_t output_column(int half) { return 256 + half * 128; }

// ---- the walk over a CTA's range, the same in every role ----

// Blocks [0, sinks) and [begin, end) of a tile.
struct Span {
    int sinks, begin, end;
    __device__ __forceinline__ bool has(int u) const { return u < sinks || (u >= begin && u < end); }
};

struct Walk {
    const AttentionParams& a;
    Request req;
    TileKeys keys;
    int head, request, tile;
    int64_t unit, end, first;  // units left [unit, end); the tile's first unit
    int u0, u1;                // blocks of the tile in this segment
    int p0, p1;                // positions of the tile's first and last row
    int rows, token;           // rows in the tile; its first token's row of the queries
    bool whole, opening;       // the segment is the whole tile; it is the CTA's first
    Span all;                  // blocks that all rows see; the V tiles of the others are looked through before their use

    __device__ __forceinline__ Walk(const AttentionParams& args, const Place& pl)
        : a(args), head(pl.head), request(pl.request), tile(pl.tile), unit(pl.unit), end(pl.end), first(pl.unit - pl.offset),
          opening(true) {
        req = load_request(a, request);
        set();
    }
    __device__ __forceinline__ void set() {
        keys = tile_keys<kRows, kTokens, kBlock>(a, req, tile);
        int i0, i1;
        Tiles<kRows, kTokens>::tokens(a, req, tile, &i0, &i1);
        p0 = req.kv_len - req.rows + i0;
        p1 = req.kv_len - req.rows + i1;
        rows = (i1 - i0 + 1) * a.group;
        token = req.start + i0;
        const int64_t last = first + keys.units;
        u0 = max(0, static_cast<int>(unit - first) - a.tile_units);
        u1 = static_cast<int>(min(last, end) - first) - a.tile_units;
        whole = u0 == 0 && u1 == keys.units - a.tile_units;
        all = seen(p0, p1);
    }
    __device__ __forceinline__ bool next() {
        first += keys.units;
        unit = first;
        if (end - first <= a.tile_units) return false;
        if (!next_tile<kRows, kTokens>(a, &req, &head, &request, &tile)) return false;
        opening = false;
        set();
        return true;
    }
    // first key of block u; `limit`: keys from it on are not loaded
    __device__ __forceinline__ int block(int u, int* limit) const {
        if (u < keys.sink_chunks) {
            *limit = keys.sink_hi;
            return u * kBlock;
        }
        *limit = keys.hi;
        return keys.base + (u - keys.sink_chunks) * kBlock;
    }
    // The blocks that every row between positions `from` and `to` sees whole.
    __device__ __forceinline__ Span seen(int from, int to) const {
        Span s;
        s.sinks = keys.sink_hi / kBlock;
        const int last = min(from, keys.hi - 1) - (kBlock - 1) - keys.base;  // blocks that start here or before end in time
        const int near = a.window < 0 ? -1 : to - a.window - keys.base;      // blocks that start here or before are too far back
        s.begin = keys.sink_chunks + (near < 0 ? 0 : near / kBlock + 1);
        s.end = keys.sink_chunks + (last < 0 ? 0 : last / kBlock + 1);
        return s;
    }
};

// ---- loads ----

// Copies a box of the cache: 64 columns (from x on) of consecutive rows of one page and head.
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x, int row, int head, int page) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
        "l"(map), "r"(smem_addr(bar)), "r"(x), "r"(row), "r"(head), "r"(page)
        : "memory");
}

// The TMA warps: K (half 0) or V (half 1) of every block.
template <int kDim>
struct Loader {
    using S = Smem<kDim>;
    const AttentionParams& a;
    Shared* sh;
    const uint32_t ring;
    const int lane, box_shift;
    const int box, panel;  // this lane's copy
    const int half;
    const CUtensorMap* const map;
    uint32_t raws = 0;    // bit s: parity of the number of copies that sh->raw[s] told of
    uint32_t flight = 0;  // the last copies, a byte each: 0x80, 0x40 raw, 0x20 parity, slot

    __device__ __forceinline__ Loader(const AttentionParams& args, Shared* s, uint32_t ring_addr, int shift, int h, const CUtensorMap* m)
        : a(args), sh(s), ring(ring_addr), lane(threadIdx.x & 31), box_shift(shift), box((threadIdx.x & 31) / S::kPanels),
          panel((threadIdx.x & 31) % S::kPanels), half(h), map(m) {}

    // the page of this lane's copy in the block at j0, `pages` (out of range) where there is none
    __device__ __forceinline__ int page(const Walk& w, int j0, int limit) const {
        const int j = j0 + (box << box_shift);
        if ((box << box_shift) >= kBlock || j >= limit) return a.pages;
        const int id = __ldg(a.block_table + w.request * a.table_stride + (j >> a.page_shift));  // j < hi: in the table
        return static_cast<uint32_t>(id) < static_cast<uint32_t>(a.pages) ? id : a.pages;
    }

    // before: whether block n - 2 was the first of its segment
    __device__ __forceinline__ bool block(const Walk& w, int u, int j0, int limit, int pg, int n, bool before) {
        const bool checked = !w.all.has(u);
        const int j = j0 + (box << box_shift);
        const bool mine = (box << box_shift) < kBlock;
        const uint32_t found = __ballot_sync(0xFFFFFFFFu, mine && pg < a.pages);
        const uint32_t wanted = __ballot_sync(0xFFFFFFFFu, mine && j < limit);
        const int f = 2 * n + half, slot = f % kSlots;
        // the slot's last content: V of block n - 3 (for K), K of block n - 2 (for V)
        const int e = half == 1 && before ? n - 2 : n - 3;
        if (e >= 0 && !bar_wait_idle(a, &sh->used[e & 3], (e >> 2) & 1, sh)) return false;
        const bool to_raw = half == 1 && checked;
        uint64_t* bar = to_raw ? &sh->raw[slot] : &sh->full[slot];
        const uint32_t parity = (to_raw ? raws >> slot : f / kSlots) & 1;
        if (to_raw) raws ^= 1u << slot;
        flight = flight << 8 | 0x80u | (to_raw ? 0x40u : 0u) | parity << 5 | slot;
        if (lane == 0) {
            if (half == 0 && found != wanted) {
                uint32_t bits = 0;
                for (int b = 0; b < 32 / S::kPanels; ++b) bits |= ((found >> (b * S::kPanels)) & 1u) << b;
                sh->boxes[n & 3] = bits;
                sh->missing[n & 3] = 1 + n;
            }
            if (!to_raw) bar_arrive3(bar);
            bar_expect(bar, S::kTile);
        }
        __syncwarp();
        if (mine) load_box(ring + slot * S::kTile + panel * S::kPanelRows + (box << box_shift) * 128, map, bar, panel * 64, j & (a.page_size - 1), w.head, pg);
        return true;
    }
    // The copies that may be under way: K of the last two blocks, V of the last three (block() waits for the use of those
    // before).  They are done when all went well.
    __device__ __forceinline__ void finish() const {
        for (int i = 0; i < 2 + half; ++i) {
            const uint32_t code = flight >> (8 * i);
            if (code & 0x80u) bar_wait_own(code & 0x40u ? &sh->raw[code & 7u] : &sh->full[code & 7u], (code >> 5) & 1);
        }
    }
};

// Warps 8-11.
template <typename T, int kDim>
struct Helper {
    using S = Smem<kDim>;
    static constexpr int kPieces = kDim / 8;
    const AttentionParams& a;
    Shared* sh;
    const uint32_t ring;
    const int tid;        // 0 .. 127
    uint32_t looked = 0;  // bit s: parity of the number of tiles looked through in slot s

    __device__ __forceinline__ Helper(const AttentionParams& args, Shared* s, uint32_t ring_addr)
        : a(args), sh(s), ring(ring_addr), tid(threadIdx.x & 127) {}

    // A V tile that not all rows see whole: 0 * inf and 0 * NaN must not reach
    // the rows that do not see the key.  Infinities and NaN are
    // taken out; the softmax warps give those of keys in range back to the rows
    // that see them.  j0: the tile's first key, f: its number
    // in the ring.
    __device__ __forceinline__ bool clear_masked(const Walk& w, int j0, int limit, int f) {
        const int slot = f % kSlots;
        if (!bar_wait_idle(a, &sh->raw[slot], (looked >> slot) & 1, sh)) return false;
        looked ^= 1u << slot;
        const uint32_t base = ring + slot * S::kTile;
        const int p = tid & 15;
        bool bad = false;
        if (p < kPieces) {
#pragma unroll 4
            for (int r = tid >> 4; r < kBlock; r += 8) {
                const int j = j0 + r;
                const bool seen = j < limit && (j >= w.keys.lo || j < a.sinks);
                const uint32_t at = base + (p >> 3) * S::kPanelRows + r * 128 + (((p & 7) ^ (r & 7)) << 4);
                uint32_t v[4];
                asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                             : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                             : "r"(at)
                             : "memory");
                // a half word whose exponent bits are all set is zero in x; the usual test for a zero among the two
                constexpr uint32_t kE = Half2<T>::kExpMask | (Half2<T>::kExpMask << 16);
                bool here = false;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t x = ~v[e] & kE;
                    here |= ((x - 0x00010001u) & ~x & 0x80008000u) != 0;
                }
                if (here) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t x = ~v[e] & kE;
                        if (!(x & 0xFFFFu)) v[e] &= 0xFFFF0000u;
                        if (!(x >> 16)) v[e] &= 0x0000FFFFu;
                    }
                }
                if (here) {
                    bad |= seen;
                    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3])
                                 : "memory");
                }
            }
        }
        if (bad) sh->nonfinite[slot] = 1 + f;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if ((tid & 31) == 0) bar_arrive(&sh->full[slot]);
        return true;
    }
};

// ---- weights ----

struct Pair {
    float x, y;
};
__device__ __forceinline__ uint64_t bits(Pair v) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(v.x), "f"(v.y));
    return r;
}
__device__ __forceinline__ Pair pair(uint64_t r) {
    Pair v;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(r));
    return v;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)), "l"(bits(c)));
    return pair(r);
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)));
    return pair(r);
}
// bits 0 .. n - 1
__device__ __forceinline__ uint32_t below(int n) { return n <= 0 ? 0u : n >= 32 ? 0xFFFFFFFFu : (1u << n) - 1u; }
// NaN if any is
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

template <typename T, int kDim>
struct Softmax {
    const AttentionParams& a;
    Shared* sh;
    const int half;       // 0, 1
    const uint32_t score, output;  // TMEM addresses of this warp's lanes
    const int row;        // of the tile
    float m, l;           // base of the weights, their sum
    bool late = false;    // see bar_wait
    int done = 0;         // blocks of this half so far, over all tiles
    int settled = 0;      // of them, those whose products pv_done tells of: a segment's last, and with a V tile looked through
    const int box_shift;

    __device__ __forceinline__ Softmax(const AttentionParams& args, Shared* s, uint32_t tmem, int shift)
        : a(args), sh(s), half(threadIdx.x >> 7), score(tmem + (((threadIdx.x >> 5) & 3) << 21) + score_column(threadIdx.x >> 7)),
          output(tmem + (((threadIdx.x >> 5) & 3) << 21) + output_column(threadIdx.x >> 7)), row(threadIdx.x & 255),
          box_shift(shift) {}

    // The weights of 64 keys from their scores, into place from column `to` on.
    __device__ __forceinline__ void weights(const float* s, float base, Pair (&sum)[2], uint32_t to) {
        const Pair scale{a.scale_log2, a.scale_log2}, shift{base, base};
#pragma unroll
        for (int c0 = 0; c0 < 64; c0 += 32) {
            uint32_t pk[16];
#pragma unroll
            for (int c = 0; c < 32; c += 2) {
                const Pair x = fma2(Pair{s[c0 + c], s[c0 + c + 1]}, scale, shift);
                const Pair e{exp2_fast(x.x), exp2_fast(x.y)};
                sum[(c / 2) & 1] = add2(sum[(c / 2) & 1], e);
                // weights go to the product in the cache's 16-bit type, as the tensor cores take them; the sum keeps 32 bits
                pk[c / 2] = Half2<T>::pack(e.x, e.y);
            }
            tmem_store16(to + c0 / 2, pk);
        }
    }
    __device__ __forceinline__ float row_max(const float (&s)[kBlock]) {
        float top[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int c = 4; c < kBlock - 4; c += 8)
#pragma unroll
            for (int x = 0; x < 4; ++x) top[x] = max3(top[x], s[c + 2 * x], s[c + 2 * x + 1]);
        top[0] = max3(top[0], s[kBlock - 4], s[kBlock - 3]);
        top[1] = max3(top[1], s[kBlock - 2], s[kBlock - 1]);
        return max3(max3(top[0], top[1], top[2]), top[3], top[3]) * a.scale_log2;
    }
    // the products of these 64 keys need not wait for the others
    __device__ __forceinline__ void hand_over(int part) {
        tmem_store_wait();
        tmem_fence_before();
        __syncwarp();
        if ((threadIdx.x & 31) == 0) bar_arrive(&sh->p_full[half][part]);
    }

    // block u of the walk's tile, number n in the CTA
    __device__ __forceinline__ void block(const Walk& w, int u, int n, int p, const Span& mine) {
        // the scores are there, and with them the products of the block before have reached O
        bar_wait(a, &sh->s_full[half], done & 1, sh, &late);
        tmem_fence_after();
        float s[kBlock];
#pragma unroll
        for (int c = 0; c < kBlock; c += 32) tmem_load32(score + c, s + c);
        const bool lost = sh->missing[n & 3] == 1 + n;
        const bool whole = !lost && mine.has(u), checked = !w.all.has(u);
        bool poison = false;
        tmem_load_wait();
        if (!whole) {
            // visible: c <= last and (c >= near or c < sink)
            int limit;
            const int j0 = w.block(u, &limit);
            const int last = min(p - j0, limit - 1 - j0);
            const int near = (a.window < 0 || p < a.window) ? 0 : p - a.window + 1 - j0;
            const int sink = a.sinks - j0;
#pragma unroll
            for (int c0 = 0; c0 < kBlock; c0 += 32) {  // 32 columns at a time as bits
                uint32_t see = below(last + 1 - c0) & (~below(near - c0) | below(sink - c0));
                if (lost) {
                    const uint32_t found = sh->boxes[n & 3];
#pragma unroll 1
                    for (int c = 0; c < 32; c += 8)  // a box is 8 keys or more
                        if (!((found >> ((c0 + c) >> box_shift)) & 1u)) see &= ~(0xFFu << c);
                }
#pragma unroll
                for (int c = 0; c < 32; ++c)
                    if (!((see >> c) & 1u)) s[c0 + c] = -INFINITY;
            }
        }
        if (checked) {  // the V tile was looked through
            const int f = 2 * n + 1;
            bar_wait(a, &sh->full[f % kSlots], (f / kSlots) & 1, sh, &late);
            poison = sh->nonfinite[f % kSlots] == 1 + f;
        }
        const float mx = row_max(s);
        // where the base's own rounding is no longer small beside that room, nothing above the maximum is let pass
        const float room = kLift<T> + (kLift<T> == 0.f || fabsf(m) < 0x1p20f ? kRaise : 0.f);
        if (__any_sync(0xFFFFFFFFu, !(mx <= m + room) && m == m)) {  // also where mx is NaN: so becomes the row, once
            const float mn = max3(m, mx - kLift<T>, mx - kLift<T>);
            if (u != w.u0) {  // the segment's first products write O, all others add to it
                const float f = mn == -INFINITY ? 1.f : exp2_fast(m - mn);
                l *= f;
#pragma unroll 1
                for (int d = 0; d < kDim; d += 16) {
                    float o[16];
                    tmem_load16(output + d, o);
                    tmem_load_wait();
#pragma unroll
                    for (int x = 0; x < 16; ++x) o[x] *= f;
                    tmem_store16(output + d, reinterpret_cast<const uint32_t*>(o));
                }
            }
            m = mn;
        }
        // a row without a visible key yet has no base; one with a score of +inf is NaN, as inf - inf
        const float base = m == -INFINITY ? 0.f : m == INFINITY ? NAN : -m;
        Pair sum[2] = {{0.f, 0.f}, {0.f, 0.f}};
#pragma unroll
        for (int part = 0; part < 2; ++part) {
            weights(s + part * 64, base, sum, score + part * 32);
            hand_over(part);
        }
        const Pair both = add2(sum[0], sum[1]);
        l += both.x + both.y;
        ++done;
        if (checked || u + 1 == w.u1) ++settled;
        if (poison) {
            bar_wait(a, &sh->pv_done[half], (settled - 1) & 1, sh, &late);
            tmem_fence_after();
            add_nonfinite(w, u, n, p);
            tmem_store_wait();
            tmem_fence_before();
        }
    }

    // Infinities and NaN that the loader took out of V, for the rows that see them.
    __device__ __forceinline__ void add_nonfinite(const Walk& w, int u, int n, int p) {
        int limit;
        const int j0 = w.block(u, &limit);
        const int32_t* table = a.block_table + w.request * a.table_stride;
#pragma unroll 1
        for (int d = 0; d < kDim; d += 32) {
            float o[32];
            tmem_load32(output + d, o);
            tmem_load_wait();
#pragma unroll 1
            for (int c = 0; c < kBlock; ++c) {
                const int j = j0 + c;
                if (j >= limit || j > p || !(a.window < 0 || p - j < a.window || j < a.sinks)) continue;
                const int id = __ldg(table + (j >> a.page_shift));
                if (static_cast<uint32_t>(id) >= static_cast<uint32_t>(a.pages)) continue;
                const T* v = static_cast<const T*>(a.v_cache) + id * a.page_stride + (j & (a.page_size - 1)) * a.token_stride +
                             w.head * a.head_stride + d;
#pragma unroll
                for (int x = 0; x < 32; x += 2) {
                    const uint32_t word = *reinterpret_cast<const uint32_t*>(v + x);
                    const float v0 = Half2<T>::low(word), v1 = Half2<T>::high(word);
                    if (!isfinite(v0)) o[x] += v0;
                    if (!isfinite(v1)) o[x + 1] += v1;
                }
            }
            tmem_store32(output + d, reinterpret_cast<const uint32_t*>(o));
        }
    }

    // Piece k of quad thread j becomes piece j of thread k.
    __device__ static __forceinline__ void exchange(uint4 (&v)[4], int mate) {
#pragma unroll
        for (int bit = 1; bit < 4; bit <<= 1)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (k & bit) continue;
                const bool high = mate & bit;  // gives the lower of the two pieces and keeps the upper
                uint4 give = high ? v[k] : v[k + bit];
                give.x = __shfl_xor_sync(0xFFFFFFFFu, give.x, bit);
                give.y = __shfl_xor_sync(0xFFFFFFFFu, give.y, bit);
                give.z = __shfl_xor_sync(0xFFFFFFFFu, give.z, bit);
                give.w = __shfl_xor_sync(0xFFFFFFFFu, give.w, bit);
                if (high) v[k] = give;
                else v[k + bit] = give;
            }
    }

    // The segment's end: this thread's row of O to the output or, for part of a tile, to the workspace.
    __device__ __forceinline__ void store(const Walk& w) {
        bar_wait(a, &sh->pv_done[half], (settled - 1) & 1, sh, &late);
        tmem_fence_after();
        // after another warp of the half was late, products may have been issued before this one's weights were there
        const bool ok = !__any_sync(0xFFFFFFFFu, late || *stalled(sh));
        int i = 0, g = 0;
        const bool valid = Tiles<kRows, kTokens>::row(a, w.req, w.tile, row, &i, &g);
        const int64_t token = w.req.start + i;
        const int head = w.head * a.group + g;
        char* ws = static_cast<char*>(a.workspace);
        float* part = reinterpret_cast<float*>(ws + workspace_records_bytes(a.ctas)) +
                      (2 * static_cast<size_t>(blockIdx.x) + (w.opening ? 0 : 1)) * partial_floats(kRows, kDim);
        const float inv = !ok ? NAN : l == 0.f ? 1.f : 1.f / l;
        // A row lies in one thread; the four threads of a quad exchange 16-byte pieces, so that each of them writes
        // every fourth piece of each other's rows and a store is 64 contiguous bytes of 8 rows, not 16 of 32.
        const int lane = threadIdx.x & 31, mate = lane & 3;
        char* to[4];  // the quad's rows, null where there is none
        {
            char* mine = nullptr;
            if (valid)
                mine = w.whole ? reinterpret_cast<char*>(static_cast<T*>(a.out) + token * a.out_token_stride + head * a.out_head_stride)
                               : reinterpret_cast<char*>(part + row * kDim);
#pragma unroll
            for (int k = 0; k < 4; ++k)
                to[k] = reinterpret_cast<char*>(__shfl_sync(0xFFFFFFFFu, reinterpret_cast<unsigned long long>(mine), (lane & ~3) + k));
        }
#pragma unroll 1
        for (int d = 0; d < kDim; d += 32) {
            float o[32];
            tmem_load32(output + d, o);
            tmem_load_wait();
            if (w.whole) {
                uint4 v[4];
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    v[x] = make_uint4(Half2<T>::pack(o[8 * x] * inv, o[8 * x + 1] * inv), Half2<T>::pack(o[8 * x + 2] * inv, o[8 * x + 3] * inv),
                                      Half2<T>::pack(o[8 * x + 4] * inv, o[8 * x + 5] * inv),
                                      Half2<T>::pack(o[8 * x + 6] * inv, o[8 * x + 7] * inv));
                exchange(v, mate);
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (to[k]) *reinterpret_cast<uint4*>(to[k] + d * 2 + mate * 16) = v[k];
            } else {
#pragma unroll
                for (int y = 0; y < 32; y += 16) {
                    uint4 v[4];
#pragma unroll
                    for (int x = 0; x < 4; ++x)
                        v[x] = make_uint4(__float_as_uint(o[y + 4 * x]), __float_as_uint(o[y + 4 * x + 1]), __float_as_uint(o[y + 4 * x + 2]),
                                          __float_as_uint(o[y + 4 * x + 3]));
                    exchange(v, mate);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (to[k]) *reinterpret_cast<uint4*>(to[k] + (d + y) * 4 + mate * 16) = v[k];
                }
            }
        }
        if (valid && w.whole) {
            if (a.lse) a.lse[token * a.heads + head] = !ok ? NAN : l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
        } else if (valid) {
            part[kRows * kDim + row] = ok ? m : NAN;
            part[kRows * kDim + kRows + row] = ok ? l : NAN;
        }
        tmem_fence_before();
    }
};

template <typename T, int kDim>
__global__ void __launch_bounds__(kThreads, 1)
attention_tiles_kernel(const AttentionParams a, const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                       const __grid_constant__ CUtensorMap v_map, const int box_shift) {
    using S = Smem<kDim>;
    extern __shared__ __align__(16) char dynamic[];
    __shared__ Shared shared;
    Shared* sh = &shared;
    const uint32_t raw = smem_addr(dynamic);
    const uint32_t q = (raw + 1023) & ~1023u, ring = q + S::kQ;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    char* ws = static_cast<char*>(a.workspace);

    asm volatile("griddepcontrol.launch_dependents;");
    const Place pl = locate<kRows, kTokens, kBlock, kThreads, 8>(a, reinterpret_cast<int*>(dynamic), blockIdx.x, a.ctas);
    if (pl.unit >= pl.end) {
        if (threadIdx.x == 0) reinterpret_cast<TileRecord*>(ws)[blockIdx.x] = TileRecord{};
        return;
    }
    Walk w(a, pl);
    if (threadIdx.x == 0) reinterpret_cast<TileRecord*>(ws)[blockIdx.x] = tile_record(a, pl, blockIdx.x, w.req, w.keys.units);
    if (w.u1 <= 0) return;  // the range ends before the tile's first block
    if (threadIdx.x == 0) {
        for (int i = 0; i < kSlots; ++i) {
            bar_init(&sh->full[i], 4);  // the four helper warps, or four times the loader
            bar_init(&sh->raw[i], 1);
            sh->nonfinite[i] = 0;
        }
        bar_init(&sh->q_full, 1);
        bar_init(&sh->q_empty, 1);
        for (int i = 0; i < 2; ++i) {
            bar_init(&sh->s_full[i], 1);
            bar_init(&sh->p_full[i][0], 4);
            bar_init(&sh->p_full[i][1], 4);
            bar_init(&sh->pv_done[i], 1);
        }
        bar_init(&sh->drain, 1);
        for (int i = 0; i < 4; ++i) {
            bar_init(&sh->used[i], 1);
            sh->missing[i] = 0;
        }
        sh->stalled = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&sh->tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // locate's sums lie where the copies go
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = sh->tmem;
    if (warp < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
        Softmax<T, kDim> sm(a, sh, tmem, box_shift);
        int n = 0;
        do {
            if (sm.half * kHalf >= w.rows) {  // nothing in this half
                n += w.u1 - w.u0;
                continue;
            }
            int i = 0, g = 0;
            const bool valid = Tiles<kRows, kTokens>::row(a, w.req, w.tile, sm.row, &i, &g);
            const int p = valid ? w.req.kv_len - w.req.rows + i : -1;
            // positions of the half's first and last row
            const int from = w.p0 + div_group(a, sm.half * kHalf);
            const int to = min(w.p1, w.p0 + div_group(a, sm.half * kHalf + kHalf - 1));
            const Span mine = w.seen(from, to);
            sm.m = -INFINITY;
            sm.l = 0.f;
            for (int u = w.u0; u < w.u1; ++u, ++n) sm.block(w, u, n, p, mine);
            sm.store(w);
        } while (w.next());
    } else if (warp < 12) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        Helper<T, kDim> hp(a, sh, ring);
        int n = 0;
        bool ok = true;
        do {
            for (int u = w.u0; ok && u < w.u1; ++u, ++n) {
                if (w.all.has(u)) continue;
                int limit;
                const int j0 = w.block(u, &limit);
                ok = hp.clear_masked(w, j0, limit, 2 * n + 1);
            }
        } while (ok && w.next());
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == 12) {
            // all lanes walk along, so that addresses stay in uniform registers; one issues
            const bool lead = elect_one();
            constexpr uint32_t kQk = instruction<T>(kBlock, false), kPv = instruction<T>(kDim, true);
            const uint32_t tm = uniform(tmem), q_low = uniform(operand_low(q, 16)), k_low = uniform(operand_low(ring, 16)),
                           v_low = uniform(operand_low(ring, S::kPanelRows));
            const auto commit = [&](uint64_t* b) {
                if (lead) mma_commit(b);
            };
            const auto scores = [&](int half, uint32_t slot) {
                const uint32_t qa = q_low + half * (kHalf * 128 / 16), kb = k_low + slot * (S::kTile / 16);
                if (lead) {
#pragma unroll
                    for (int k = 0; k < kDim / 16; ++k)
                        mma_smem(tm + score_column(half), qa + ((k >> 2) * S::kQPanel + (k & 3) * 32) / 16,
                                 kb + ((k >> 2) * S::kPanelRows + (k & 3) * 32) / 16, kQk, k > 0);
                    mma_commit(&sh->s_full[half]);
                }
            };
            // keys 64 part .. 64 part + 63
            const auto output = [&](int half, uint32_t slot, int part, bool add) {
                const uint32_t vb = v_low + slot * (S::kTile / 16);
                if (lead) {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        mma_tmem(tm + output_column(half), tm + score_column(half) + (part * 4 + k) * 8, vb + (part * 4 + k) * (2048 / 16),
                                 kPv, add || k > 0);
                }
            };
            struct Turn {  // a place in the ring, and the parity of its use
                uint32_t slot;
                int parity;
                __device__ __forceinline__ void advance() {
                    if (++slot == kSlots) {
                        slot = 0;
                        parity ^= 1;
                    }
                }
            } at{0, 0};  // the next tile to be used
            const auto filled = [&](const Turn& t) { return bar_wait_all(a, &sh->full[t.slot], t.parity, sh); };
            int n = 0, segment = 0, done[2] = {0, 0};
            bool ok = true;
            do {
                const int halves = w.rows > kHalf ? 2 : 1, blocks = w.u1 - w.u0;
                ok = bar_wait_all(a, &sh->q_full, segment & 1, sh) && filled(at);
                if (!ok) break;
                scores(0, at.slot);
                if (halves == 2) scores(1, at.slot);
                if (blocks == 1) commit(&sh->q_empty);
                at.advance();
                // V of the block in work and K of the next one; waited for a half block before they are used, so that
                // nothing but the weights is waited for between two halves' products
                Turn v = at, k = at;
                k.advance();
                ok = filled(v) && (blocks == 1 || filled(k));
                bool tell = blocks == 1 || !w.all.has(w.u0);
                for (int b = 0; ok && b < blocks; ++b, ++n) {
                    const bool more = b + 1 < blocks;
                    const auto turn = [&](int h) {
                        ok = bar_wait_all(a, &sh->p_full[h][0], done[h] & 1, sh);
                        if (!ok) return;
                        tmem_fence_after();
                        output(h, v.slot, 0, b > 0);
                        // the block before, told late: a commit takes its time, and here the tensor cores have work
                        if (h == 0 && b > 0) commit(&sh->used[(n - 1) & 3]);
                        ok = bar_wait_all(a, &sh->p_full[h][1], done[h] & 1, sh);
                        if (!ok) return;
                        tmem_fence_after();
                        output(h, v.slot, 1, true);
                        if (tell) commit(&sh->pv_done[h]);
                        ++done[h];
                        if (more) scores(h, k.slot);
                    };
                    turn(0);
                    if (!ok) break;
                    Turn next_v = k, next_k = k;
                    next_v.advance();
                    next_k = next_v;
                    next_k.advance();
                    if (more) ok = filled(next_v) && (b + 2 >= blocks || filled(next_k));
                    const bool next_tell = b + 2 >= blocks || !w.all.has(w.u0 + b + 1);
                    if (ok && halves == 2) turn(1);
                    if (!ok) break;
                    if (b + 2 == blocks) commit(&sh->q_empty);
                    if (!more) commit(&sh->used[n & 3]);
                    at = more ? next_v : k;
                    v = next_v;
                    k = next_k;
                    tell = next_tell;
                }
                ++segment;
            } while (ok && w.next());
            // all products end before the block does, also after a stall
            commit(&sh->drain);
            bar_wait_own(&sh->drain, 0);
        } else if (warp == 15) {
            int segment = 0;
            bool ok = true;
            do {
                ok = bar_wait_idle(a, &sh->q_empty, (segment & 1) ^ 1, sh);
                if (!ok) break;
                if (lane == 0) {
                    const int rows = Tiles<kRows, kTokens>::per(a) * a.group;
                    bar_expect(&sh->q_full, S::kPanels * rows * 128);
                    for (int i = 0; i < S::kPanels; ++i) load_box(q + i * S::kQPanel, &q_map, &sh->q_full, i * 64, w.head * a.group, w.token, 0);
                }
                __syncwarp();
                ++segment;
            } while (w.next());
            if (segment > 0) bar_wait_own(&sh->q_full, (segment - 1) & 1);
        } else {
            Loader<kDim> ld(a, sh, ring, box_shift, warp - 13, warp == 13 ? &k_map : &v_map);
            int n = 0;
            uint32_t firsts = 0;  // bit i: block n - 1 - i was the first of its segment
            bool ok = true;
            do {
                int limit, j0 = w.block(w.u0, &limit);
                int pg = ld.page(w, j0, limit);
                for (int u = w.u0; ok && u < w.u1; ++u, ++n) {
                    int next_limit = 0, next_j0 = 0, next_pg = 0;
                    if (u + 1 < w.u1) {  // looked up one block ahead
                        next_j0 = w.block(u + 1, &next_limit);
                        next_pg = ld.page(w, next_j0, next_limit);
                    }
                    if (warp == 13 && n >= a.lost_block) ok = false;
                    else ok = ld.block(w, u, j0, limit, pg, n, (firsts >> 1) & 1);
                    firsts = firsts << 1 | (u == w.u0);
                    j0 = next_j0;
                    limit = next_limit;
                    pg = next_pg;
                }
            } while (ok && w.next());
            ld.finish();
        }
        __syncwarp();
    }
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    if (warp == 12) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

std::atomic<int> g_wait_tries{kWaitTries}, g_lost_block{INT32_MAX};

using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                            const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                            CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

Encode find_encode() {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &r) != cudaSuccess ||
        r != cudaDriverEntryPointSuccess)
        return nullptr;
    return reinterpret_cast<Encode>(f);
}

// A tensor of 16-bit elements, dim contiguous and three outer axes; boxes of 64 columns, box1 and box2 of the next two axes.
bool encode(CUtensorMap* map, const AttentionParams& a, const void* data, const int64_t (&size)[3], const int64_t (&stride)[3], int box1,
            int box2) {
    static const Encode f = find_encode();
    if (!f) return false;
    cuuint64_t dims[4] = {static_cast<cuuint64_t>(a.dim)}, strides[3];
    for (int i = 0; i < 3; ++i) {
        dims[i + 1] = static_cast<cuuint64_t>(size[i]);
        strides[i] = static_cast<cuuint64_t>(size[i] > 1 ? stride[i] : a.dim) * 2;  // that of an axis of one entry is never used
    }
    const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(box1), static_cast<cuuint32_t>(box2), 1}, step[4] = {1, 1, 1, 1};
    return f(map, a.dtype == FG_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
             const_cast<void*>(data), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int kDim>
cudaError_t launch(AttentionParams a, cudaStream_t stream) {
    constexpr int bytes = Smem<kDim>::kBytes;
    static_assert(bytes >= locate_bytes(kMaxRequests), "the scan over the requests fits the tiles' room");
    static SmemOnce once;
    cudaError_t e = once.set(reinterpret_cast<const void*>(attention_tiles_kernel<T, kDim>), bytes);
    if (e != cudaSuccess) return e;
    // A box is as much of a page as a block takes, so that the copies are few; with a window 64 rows at most, because
    // blocks then start at multiples of it and begin with that many keys less one that no row sees.  (16 rows always:
    // 2048 tokens on 8192 20 % slower with pages of 64.)
    const int box_shift = min(a.page_shift, a.window < 0 ? 7 : 6);
    a.base_align = 1 << box_shift;
    a.unit_shift = 0;
    a.tile_units = kTileBlocks;
    a.wait_tries = g_wait_tries.load(std::memory_order_relaxed);
    a.lost_block = g_lost_block.load(std::memory_order_relaxed);
    const int64_t cache_size[3] = {a.page_size, a.kv_heads, a.pages}, cache_stride[3] = {a.token_stride, a.head_stride, a.page_stride};
    const int64_t q_size[3] = {a.heads, a.tokens, 1}, q_stride[3] = {a.q_head_stride, a.q_token_stride, 0};
    CUtensorMap q_map, k_map, v_map;
    if (!encode(&q_map, a, a.q, q_size, q_stride, a.group, kRows / a.group) ||
        !encode(&k_map, a, a.k_cache, cache_size, cache_stride, 1 << box_shift, 1) ||
        !encode(&v_map, a, a.v_cache, cache_size, cache_stride, 1 << box_shift, 1))
        return cudaErrorInvalidValue;
    attention_tiles_kernel<T, kDim><<<a.ctas, kThreads, bytes, stream>>>(a, q_map, k_map, v_map, box_shift);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
    return launch_combine<T, kRows, kDim, kTokens, 4>(a, stream);
}

template <typename T>
cudaError_t by_dim(const AttentionParams& a, cudaStream_t s) {
    switch (a.dim) {
        case 64: return launch<T, 64>(a, s);
        case 96: return launch<T, 96>(a, s);
        default: return launch<T, 128>(a, s);
    }
}

}  // namespace
}  // namespace attn

// Whether the 32-bit sums of blocks hold a call: 2^31 blocks would take the kernel ten seconds, but the table's width and
// the counts do not exclude them.
bool attention_tiles_counts(const AttentionParams& a) {
    const int64_t keys = std::min<int64_t>(static_cast<int64_t>(a.table_width) * a.page_size, INT32_MAX);
    const int64_t tiles = static_cast<int64_t>(a.tokens) / (attn::kRows / a.group) + a.requests;
    return tiles * (keys / attn::kBlock + 4 + attn::kTileBlocks) <= INT32_MAX;
}

void set_attention_waits(int lost_block, int tries) {
    attn::g_lost_block.store(lost_block < 0 ? INT32_MAX : lost_block, std::memory_order_relaxed);
    attn::g_wait_tries.store(tries < 0 ? attn::kWaitTries : tries, std::memory_order_relaxed);
}

size_t attention_tiles_workspace(int sms, int dim) {
    const int ctas = sms;
    return attn::workspace_records_bytes(ctas) + 2 * static_cast<size_t>(ctas) * attn::partial_floats(attn::kRows, dim) * sizeof(float);
}

cudaError_t launch_attention_tiles(const AttentionParams& a, cudaStream_t stream) {
    return a.dtype == FG_DTYPE_BF16 ? attn::by_dim<__nv_bfloat16>(a, stream) : attn::by_dim<__half>(a, stream);
}

}  // namespace fg
