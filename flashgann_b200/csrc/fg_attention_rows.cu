// fg_attention_rows.cu -- attention of few query rows over the paged cache:
// decode steps, a few drafted tokens, and the retrieved form.
//
// A tile is 16 query rows of one kv head (the heads that share it, times the
// request's tokens), the height of one m16n8k16 product.  With so few rows a
// key costs 4*dim bytes of traffic and 16 * 4 * dim multiply-adds on the
// matrix pipe, a quarter of what that pipe does in the time HBM needs for the
// bytes: the kernel is bound by bandwidth, and everything serves keeping loads
// in flight.
//
// Layout.  Two CTAs of 4 warps per SM, so that one's start, list of ids and join
// pass beside the other's loads.  A chunk is 16 keys; warp w of a CTA takes
// chunks w, w+4, ... of the CTA's range and is on its own until the tile
// ends: it looks the keys' pages up, copies their K and V rows to its own ring
// of shared memory with 16-byte cp.async (kStages - 1 chunks ahead, the pages
// one more), and keeps
// its own running maximum, sum and 16 x dim output in registers, so no barrier
// sits between a load and its use.  Gathering by row costs nothing extra over
// a tile copy here, and makes pages of any size, any strides, windows that
// start inside a page and retrieved ids the same code.  At a tile's end the
// warps join through shared memory.
//
// Retrieved ids are chunks like the others: 16 ids of one head, whose scores
// count in that head's row alone.  The other rows' share of the product is
// waste on a pipe that idles anyway.  At a tile's start the warps read the
// heads' lists once, drop the ids that do not count (out of range, in the window,
// repeated) and leave the rest in shared memory, see stage_ids.
//
// Measured (device time, 32 or 64 query heads on 8, dim 128, bf16): 64 ragged
// decodes, 1.1 GB of keys and values, 174 to 180 us, 6.1 to 6.3 TB/s; one of
// 131K keys at most, 80 to 83 us; one of a few hundred keys of dim 64 7.6 to 8.3
// us.  With 64 requests x 100 ids 57 to 58 us for 175 MB: there 8 warps per SM, as many as their registers allow,
// do not cover the latency of short tiles.
//
// Tiles that are short whatever the lengths are (a narrow table, or a window and
// a few ids) are not split where that leaves the CTAs evenly filled, see
// attention_rows_splits.
#include <algorithm>

#include "fg_attention.cuh"

namespace fg {

namespace {
constexpr int kRows = 16;
constexpr int kChunk = 16;
constexpr int kCtasPerSm = 2;
constexpr int kMaxIds = 1024;  // ids of a tile's heads, in shared memory

// Places of a list of ids in shared memory: whole groups of 128.
__host__ __device__ __forceinline__ int staged_pitch(int count) { return (count + 127) & ~127; }

// Heads to a tile: with ids as many as have room for theirs.
int tile_rows(const AttentionParams& a) { return a.ids_count > 0 ? std::min(kRows, kMaxIds / staged_pitch(a.ids_count)) : kRows; }
}  // namespace

// Whether tiles are split over CTAs (a.ctas: SMs).  The host knows how many
// chunks no tile has more of (from the table's width, or from the window, the
// first tokens and the ids) and about how many tiles there are.  Not split: no
// partials, no second kernel, and every tile's ids are read once; but the CTAs
// are as unevenly filled as the tiles fall.  So tiles longer than 64 chunks are
// always split, and shorter ones by how the CTAs (296) would be filled.
// Measured, us a call, whole / split, 4 heads of 128:
//   an eighth of the CTAs or less: 1 tile of 15 chunks 8.2 / 9.5, of 21
//     10.3 / 9.4, of 40 14.5 / 9.5; 32 of 21 10.4 / 10.8, of 27 12.3 / 10.9;
//     with ids 32 tiles of 12 12.7 / 14.4, of 24 16.4 / 16.1, of 36 20.5 / 16.4
//   up to 80 % of them: 96 of 33 14.4 / 15.2, of 40 16.4 / 15.4; 160 of 33
//     17.6 / 18.5, of 40 20.3 / 18.9; with ids, whose table every part makes
//     again, 96 of 60 28.7 / 31.9, 160 of 36 22.6 / 26.7
//   a last round below 80 %: 320 of 15 18.5 / 18.5, of 21 22.6 / 20.5, of 40
//     34.7 / 28.8; with ids 320 of 12 26.5 / 26.3, of 24 33.7 / 30.8
//   fuller: 296 of 40 21.5 / 22.6, 512 of 40 41.5 / 42.9, with ids 47.3 / 51.5
bool attention_rows_splits(const AttentionParams& a) {
    int64_t keys = static_cast<int64_t>(a.table_width) * a.page_size;
    if (a.window >= 0) keys = std::min<int64_t>(keys, static_cast<int64_t>(a.window) + kRows + a.sinks);
    int64_t chunks = keys / kChunk + 3;
    int64_t tiles = static_cast<int64_t>(a.requests) * a.kv_heads;
    if (a.ids_count > 0) {
        const int rows = tile_rows(a);
        chunks += static_cast<int64_t>(std::min(a.group, rows)) * ((a.ids_count + kChunk - 1) / kChunk);
        tiles = static_cast<int64_t>(a.tokens) * a.kv_heads * ((a.group + rows - 1) / rows);
    }
    const int64_t ctas = static_cast<int64_t>(a.ctas) * kCtasPerSm;
    if (chunks > 64) return true;
    if (tiles * 8 <= ctas) return chunks > 20;
    if (tiles * 10 >= (tiles + ctas - 1) / ctas * ctas * 8) return false;
    return tiles <= ctas ? chunks > 36 && a.ids_count == 0 : chunks > 18;
}

namespace attn {
namespace {

constexpr int kWarps = 4;
constexpr int kTileUnits = 2;  // a tile's start and end take about as long as two chunks of each warp
constexpr int kThreads = kWarps * 32;
static_assert(kThreads == 128, "lists of ids lie in groups of 128");
constexpr int kTable = 8192;     // places of the hash table over them: with 2048 or 4096 staging takes twice or 1.3 times as long

template <int kDim, bool kIds>
struct Smem {
    // ldmatrix reads 8 rows without bank conflicts: rows of 128 or 256 bytes with their 16-byte pieces exchanged by the
    // row's number, rows of 192 bytes padded to an odd multiple of 16
    static constexpr bool kExchange = kDim % 64 == 0;
    static constexpr int kPitch = kExchange ? kDim * 2 : kDim * 2 + 16;
    __device__ static __forceinline__ uint32_t at(int row, int piece) {
        return row * kPitch + (kExchange ? piece ^ (row & 7) : piece) * 16;
    }
    static constexpr int kTile = kChunk * kPitch;
    static constexpr int kStages = kIds ? 2 : 3;  // of the ring; with ids the third one's room is the table's (3 % for decodes)
    static constexpr int kRing = kStages * 2 * kTile;  // K and V of each stage
    static constexpr int kWarpBytes = kRing;
    static constexpr int kIdsAt = kWarps * kWarpBytes;  // retrieved form: the tile's ids and the table
    static constexpr int kBytes = kIdsAt + (kIds ? kMaxIds * 4 + kTable * 4 : 0);
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool ok) {
    const int n = ok ? 16 : 0;  // 0: the destination is filled with zeros and nothing is read
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

template <typename T>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The element offset of key j's row in the cache (either half) given its page, or -1 where there is no such page.
__device__ __forceinline__ int64_t key_offset(const AttentionParams& a, int page, int j, int64_t head_off) {
    if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(a.pages)) return -1;
    return page * a.page_stride + (j & (a.page_size - 1)) * a.token_stride + head_off;
}
__device__ __forceinline__ int key_page(const AttentionParams& a, const int32_t* table, int j) {
    const int at = j >> a.page_shift;
    return at < a.table_width ? __ldg(table + at) : -1;
}

// A chunk whose keys' pages are being looked up.  A lane has two keys, number
// lane / 4 and that + 8, and copies every fourth 16-byte piece of their rows:
// 64 contiguous bytes to each 4 lanes, and addresses that differ by constants.
struct Found {
    int key, row;          // as in Chunk
    int j[2], page[2];     // this lane's keys (-1: none) and, when they arrive, their pages
};

// One chunk in flight.
struct Chunk {
    int key;         // first key (contiguous chunks)
    int row;         // row that alone sees it (retrieved ids), or -1
    uint32_t ok[2];  // bits 4 i .. 4 i + 3: key i (and 8 + i) is loaded and may be visible
    __device__ __forceinline__ bool has(int col) const { return (ok[col >> 3] >> ((col & 7) * 4)) & 1u; }
};

template <typename T, int kDim, bool kIds>
struct Warp {
    using S = Smem<kDim, kIds>;
    static constexpr int kPieces = kDim / 8;              // 16-byte pieces of a row
    // A float16 weight below 2^-25 would be zero in the product while the sum l counts it: many keys far below the
    // maximum would be lost.  Weights and o are 2^15 times as large there, exactly, until the warps join, so that those
    // down to 2^-29 keep their relative precision and those down to 2^-40 count.
    static constexpr float kLift = Half2<T>::kNarrow ? 32768.f : 1.f;

    const AttentionParams& a;
    const int lane;
    const uint32_t ring;
    // the tile
    Request req;
    TileKeys keys;
    const int32_t* table;
    int64_t head_off;
    int p0, p1;        // positions of the tile's first and last row
    int prow[2];       // positions of this lane's two rows (-1: no row)
    const int32_t* ids;  // the tile's lists of retrieved ids
    const int* staged;   // those of all its rows that count, in shared memory
    // running state
    uint32_t q[kDim / 16][4];
    float o[kDim / 8][4];
    float m[2], l[2];
    bool safe;

    __device__ __forceinline__ Warp(const AttentionParams& args, uint32_t ring_addr)
        : a(args), lane(threadIdx.x & 31), ring(ring_addr) {}

    __device__ __forceinline__ void begin(int head, int request, int tile) {
        table = a.block_table + request * a.table_stride;
        head_off = head * a.head_stride;
        int i0, i1;
        Tiles<kRows, kIds ? kToken : kPacked>::tokens(a, req, tile, &i0, &i1);
        p0 = req.kv_len - req.rows + i0;
        p1 = req.kv_len - req.rows + i1;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            int i, g;
            const bool ok = Tiles<kRows, kIds ? kToken : kPacked>::row(a, req, tile, (lane >> 2) + 8 * x, &i, &g);
            prow[x] = ok ? req.kv_len - req.rows + i : -1;
            const T* src = static_cast<const T*>(a.q) + static_cast<int64_t>(req.start + i) * a.q_token_stride +
                           static_cast<int64_t>(head * a.group + g) * a.q_head_stride + (lane & 3) * 2;
#pragma unroll
            for (int k = 0; k < kDim / 16; ++k) {
                q[k][x] = ok ? *reinterpret_cast<const uint32_t*>(src + k * 16) : 0u;
                q[k][x + 2] = ok ? *reinterpret_cast<const uint32_t*>(src + k * 16 + 8) : 0u;
            }
        }
        safe = false;
        clear();
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int n = 0; n < kDim / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
        m[0] = m[1] = -INFINITY;
        l[0] = l[1] = 0.f;
    }

    // The lists of a tile's heads.
    __device__ __forceinline__ const int32_t* lists(const Request& r, int head, int tile) const {
        int i, g;
        Tiles<kRows, kIds ? kToken : kPacked>::row(a, r, tile, 0, &i, &g);
        return a.ids + static_cast<int64_t>(r.start + i) * a.ids_token_stride + static_cast<int64_t>(head * a.group + g) * a.ids_head_stride;
    }
    // The lists lie in shared memory in groups of kThreads places, each of one head; group `at` and the three after it.
    __device__ __forceinline__ void read_groups(const int32_t* from, int at, int groups, int (&id)[4]) const {
        const int per = staged_pitch(a.ids_count) / kThreads;
#pragma unroll
        for (int y = 0; y < 4; ++y) {
            const int h = (at + y) / per, n = (at + y - h * per) * kThreads + threadIdx.x;
            id[y] = at + y < groups && n < a.ids_count ? __ldg(from + h * a.ids_head_stride + n) : -1;
        }
    }
    __device__ __forceinline__ int list_heads(int tile) const {
        return min(a.tile_rows, a.group - (tile % Tiles<kRows, kToken>::per(a)) * a.tile_rows);
    }
    // The first ids of a tile that comes next, into registers.
    __device__ __forceinline__ void read_ids(const Request& r, int head, int tile) {
        ids = lists(r, head, tile);
        read_groups(ids, 0, list_heads(tile) * (staged_pitch(a.ids_count) / kThreads), early);
    }
    int early[4];

    // Starts looking chunk c's keys up.
    __device__ __forceinline__ Found find(int c) const {
        Found f;
        f.row = -1;
        f.key = 0;
        f.j[0] = f.j[1] = f.page[0] = f.page[1] = -1;
        const int x = lane >> 2;
        if (c < keys.sink_chunks) {
            f.key = c * kChunk;
#pragma unroll
            for (int y = 0; y < 2; ++y)
                if (f.key + x + 8 * y < keys.sink_hi) f.j[y] = f.key + x + 8 * y;
        } else if (c < keys.sink_chunks + keys.near_chunks) {
            f.key = keys.base + (c - keys.sink_chunks) * kChunk;
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                const int j = f.key + x + 8 * y;
                if (j < keys.hi && (j >= keys.lo || j < a.sinks)) f.j[y] = j;
            }
        } else if (kIds) {
            const int per = (a.ids_count + kChunk - 1) / kChunk;
            const int at = c - keys.sink_chunks - keys.near_chunks;
            f.row = at / per;
            const int n = (at - f.row * per) * kChunk + x;  // the list is padded to whole chunks
            const int* list = staged + f.row * staged_pitch(a.ids_count);
            f.j[0] = list[n];
            f.j[1] = list[n + 8];
        }
#pragma unroll
        for (int y = 0; y < 2; ++y)
            if (f.j[y] >= 0) f.page[y] = key_page(a, table, f.j[y]);
        return f;
    }

    // Whether a retrieved id counts, repeats aside: in range, and not visible by the mask already.
    __device__ __forceinline__ bool counts(int id) const { return id >= a.sinks && id <= p0 && p0 - id >= a.window; }

    // Reads the lists of the tile's heads into shared memory, with -1 in the
    // place of ids that do not count.  Of equal ids in a list the first stays: a
    // hash table (open addressing, an eighth full at most) holds for each id of each
    // head the least of its places in the lists; an id whose place is another's
    // goes.  The result does not depend on the order of the atomics.  Called by
    // the whole CTA.
    __device__ __forceinline__ void stage_ids(int* list, int* table, int heads) const {
        constexpr int kFree = -1;  // (16-bit places would do, but their atomics are ten times as slow)
        const int pitch = staged_pitch(a.ids_count), per = pitch / kThreads, groups = heads * per;
        for (int x = threadIdx.x; x < kTable / 4; x += kThreads) reinterpret_cast<int4*>(table)[x] = make_int4(kFree, kFree, kFree, kFree);
        int id4[4] = {early[0], early[1], early[2], early[3]};
        for (int at = 0; at < groups; at += 4) {
            if (at > 0) read_groups(ids, at, groups, id4);
#pragma unroll
            for (int y = 0; y < 4; ++y)
                if (at + y < groups) list[(at + y) * kThreads + threadIdx.x] = counts(id4[y]) ? id4[y] : -1;
        }
        __syncthreads();
        const auto first_place = [&](int id, int h) {
            return ((static_cast<uint32_t>(id) + static_cast<uint32_t>(h) * 0x9E3779B9u) * 2654435761u) >> 19;  // of 8192
        };
        const auto same = [&](int x, int id, int h) { return list[x] == id && static_cast<uint32_t>(x - h * pitch) < static_cast<uint32_t>(pitch); };
        for (int at = 0; at < groups; ++at) {
            const int x = at * kThreads + threadIdx.x, id = list[x], h = at / per;
            if (id < 0) continue;
            for (uint32_t place = first_place(id, h);; place = (place + 1) % kTable) {
                const int old = atomicCAS(table + place, kFree, x);
                if (old == kFree) break;
                if (!same(old, id, h)) continue;  // another id's place
                atomicMin(table + place, x);
                break;
            }
        }
        __syncthreads();
        for (int at = 0; at < groups; ++at) {
            const int x = at * kThreads + threadIdx.x, id = list[x], h = at / per;
            if (id < 0) continue;
            uint32_t place = first_place(id, h);
            while (!same(table[place], id, h)) place = (place + 1) % kTable;
            if (table[place] != x) list[x] = -1;  // no place that the table holds
        }
        __syncthreads();
    }

    // Starts the copies of a chunk into stage s.
    __device__ __forceinline__ Chunk load(const Found& f, int s) const {
        Chunk ch;
        ch.key = f.key;
        ch.row = f.row;
        const uint32_t dst = ring + s * 2 * S::kTile;
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            const int64_t off = f.j[y] >= 0 ? key_offset(a, f.page[y], f.j[y], head_off) : -1;
            const bool ok = off >= 0;
            ch.ok[y] = __ballot_sync(0xFFFFFFFFu, ok);
            const T* k = static_cast<const T*>(a.k_cache) + (ok ? off + (lane & 3) * 8 : 0);
            const T* v = static_cast<const T*>(a.v_cache) + (ok ? off + (lane & 3) * 8 : 0);
#pragma unroll
            for (int i = 0; i < kPieces / 4; ++i) {
                const uint32_t to = dst + S::at((lane >> 2) + 8 * y, 4 * i + (lane & 3));
                copy16(to, k + i * 32, ok);
                copy16(to + S::kTile, v + i * 32, ok);
            }
        }
        return ch;
    }

    __device__ __forceinline__ bool sees(const Chunk& ch, int x, int col) const {
        if (!ch.has(col)) return false;
        if (kIds) return ch.row < 0 || (lane >> 2) + 8 * x == ch.row;  // one token: what is loaded is visible
        const int j = ch.key + col, p = prow[x];
        return j <= p && (a.window < 0 || p - j < a.window || j < a.sinks);
    }

    // V rows that some rows of the tile see and others do not: 0 * inf and
    // 0 * NaN must not reach the ones that do not.  That is rare, and shows in
    // the sums: only where a tile's sums are not finite (or the values that
    // belong there are not) its chunks are done once more with `safe` set.  Then
    // each lane clears such values from the pieces that it copied itself,
    __device__ __forceinline__ bool clear_nonfinite(int s) {
        bool bad = false;
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int i = 0; i < kPieces / 4; ++i) {
                const uint32_t at = ring + s * 2 * S::kTile + S::kTile + S::at((lane >> 2) + 8 * y, 4 * i + (lane & 3));
                uint32_t w[4];
                asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                             : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                             : "r"(at)
                             : "memory");
                bool here = false;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    constexpr uint32_t kE = Half2<T>::kExpMask;
                    if ((w[e] & kE) == kE) {
                        w[e] &= 0xFFFF0000u;
                        here = true;
                    }
                    if ((w[e] & (kE << 16)) == (kE << 16)) {
                        w[e] &= 0x0000FFFFu;
                        here = true;
                    }
                }
                if (here) {
                    bad = true;
                    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
                                 : "memory");
                }
            }
        return __any_sync(0xFFFFFFFFu, bad);
    }

    // and the rows that do see them get them back.  id_chunk: number of the chunk among the retrieved ones.
    __device__ __forceinline__ void add_nonfinite(const Chunk ch, int id_chunk) {
        const T* vc = static_cast<const T*>(a.v_cache);
#pragma unroll 1
        for (int col = 0; col < kChunk; ++col) {
            if (!ch.has(col)) continue;
            const bool see0 = sees(ch, 0, col), see1 = sees(ch, 1, col);
            int j = ch.key + col;
            if (kIds && ch.row >= 0) {
                const int per = (a.ids_count + kChunk - 1) / kChunk;
                j = staged[ch.row * staged_pitch(a.ids_count) + (id_chunk % per) * kChunk + col];
            }
            const T* src = vc + key_offset(a, key_page(a, table, j), j, head_off) + (lane & 3) * 2;
#pragma unroll
            for (int n = 0; n < kDim / 8; ++n) {
                const uint32_t w = *reinterpret_cast<const uint32_t*>(src + n * 8);
                const float v0 = Half2<T>::low(w), v1 = Half2<T>::high(w);
                if (!isfinite(v0)) {
                    if (see0) o[n][0] += v0;
                    if (see1) o[n][2] += v0;
                }
                if (!isfinite(v1)) {
                    if (see0) o[n][1] += v1;
                    if (see1) o[n][3] += v1;
                }
            }
        }
    }

    // Rows of the tile differ in what they see, and a sum is not finite.
    __device__ __forceinline__ bool tainted() const {
        if (!kIds && p0 == p1) return false;
        float t = 0.f;
#pragma unroll
        for (int n = 0; n < kDim / 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) t = fmaf(o[n][e], 0.f, t);
        return __any_sync(0xFFFFFFFFu, t != 0.f);
    }

    __device__ __forceinline__ void compute(const Chunk& ch, int s, int id_chunk) {
        const uint32_t kt = ring + s * 2 * S::kTile, vt = kt + S::kTile;
        float sc[2][4];
#pragma unroll
        for (int n = 0; n < 2; ++n) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
        // keys (lane & 7) + 8 * (lane >= 16), k offset 8 * ((lane >> 3) & 1)
        const int krow = (lane & 7) + ((lane >> 4) << 3), kpiece = (lane >> 3) & 1;
#pragma unroll
        for (int k = 0; k < kDim / 16; ++k) {
            uint32_t b[4];
            ldmatrix4(kt + S::at(krow, 2 * k + kpiece), b);
            mma<T>(sc[0], q[k], b[0], b[1]);
            mma<T>(sc[1], q[k], b[2], b[3]);
        }
        const bool whole = (ch.ok[0] & ch.ok[1]) == 0xFFFFFFFFu && ch.row < 0 &&
                           (kIds || p0 == p1 || (ch.key + kChunk - 1 <= p0 && (a.window < 0 || p1 - ch.key < a.window ||
                                                                              ch.key + kChunk - 1 < a.sinks)));
        bool poison = false;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[n][e] *= a.scale_log2;
        if (!whole) {
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (!sees(ch, e >> 1, n * 8 + (lane & 3) * 2 + (e & 1))) sc[n][e] = -INFINITY;
            if (safe) {
                poison = clear_nonfinite(s);
                __syncwarp();
            }
        }
        uint32_t pa[4];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            float mx = fmaxf(fmaxf(sc[0][2 * x], sc[0][2 * x + 1]), fmaxf(sc[1][2 * x], sc[1][2 * x + 1]));
            mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 2));
            const float mn = fmaxf(m[x], mx), ref = mn == -INFINITY ? 0.f : mn;
            if (__any_sync(0xFFFFFFFFu, mn > m[x])) {
                const float f = exp2_fast(m[x] - ref);
                l[x] *= f;
#pragma unroll
                for (int n = 0; n < kDim / 8; ++n) {
                    o[n][2 * x] *= f;
                    o[n][2 * x + 1] *= f;
                }
                m[x] = mn;
            }
            float e0 = exp2_fast(sc[0][2 * x] - ref), e1 = exp2_fast(sc[0][2 * x + 1] - ref);
            float e2 = exp2_fast(sc[1][2 * x] - ref), e3 = exp2_fast(sc[1][2 * x + 1] - ref);
            l[x] += (e0 + e1) + (e2 + e3);  // this lane's columns; joined over the 4 lanes of a row at the end
            // weights go to the product in the cache's 16-bit type, as the matrix pipe takes them: at most 1, relative
            // rounding 2^-8 (bf16) or 2^-11, in size that of the result's own rounding; the sum l keeps 32 bits
            pa[x] = Half2<T>::pack(e0 * kLift, e1 * kLift);
            pa[x + 2] = Half2<T>::pack(e2 * kLift, e3 * kLift);
        }
        // keys (lane & 15), dims 8 * (lane >= 16)
        const int vrow = lane & 15, vpiece = lane >> 4;
#pragma unroll
        for (int n = 0; n < kDim / 16; ++n) {
            uint32_t b[4];
            ldmatrix4_trans(vt + S::at(vrow, 2 * n + vpiece), b);
            mma<T>(o[2 * n], pa, b[0], b[1]);
            mma<T>(o[2 * n + 1], pa, b[2], b[3]);
        }
        if (poison) add_nonfinite(ch, id_chunk);
    }
};

template <typename T, int kDim, bool kIds>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) attention_rows_kernel(const AttentionParams a) {
    using S = Smem<kDim, kIds>;
    extern __shared__ __align__(128) char smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    char* ws = static_cast<char*>(a.workspace);

    asm volatile("griddepcontrol.launch_dependents;");
    const Place pl = locate<kRows, kIds ? kToken : kPacked, kChunk, kThreads, 1>(a, reinterpret_cast<int*>(smem), blockIdx.x, a.ctas);
    __syncthreads();  // the rings overlay the scan
    if (pl.unit >= pl.end) {
        if (threadIdx.x == 0 && ws) reinterpret_cast<TileRecord*>(ws)[blockIdx.x] = TileRecord{};
        return;
    }

    Warp<T, kDim, kIds> w(a, smem_addr(smem) + warp * S::kWarpBytes);
    int head = pl.head, request = pl.request, tile = pl.tile;
    int64_t unit = pl.unit, tile_first = pl.unit - pl.offset;
    w.req = load_request(a, request);
    w.keys = tile_keys<kRows, kIds ? kToken : kPacked, kChunk>(a, w.req, tile);
    if (threadIdx.x == 0 && ws) reinterpret_cast<TileRecord*>(ws)[blockIdx.x] = tile_record(a, pl, blockIdx.x, w.req, w.keys.units);
    if (kIds) w.read_ids(w.req, head, tile);
    bool first_segment = true;
    while (true) {
        const int64_t tile_last = tile_first + w.keys.units;
        const int u0 = max(0, static_cast<int>(unit - tile_first) - a.tile_units);
        const int u1 = static_cast<int>(min(tile_last, pl.end) - tile_first) - a.tile_units;
        if (u1 <= 0) break;  // the range ends before the tile's first chunk
        const int c1 = min(u1 << a.unit_shift, w.keys.chunks);
        w.begin(head, request, tile);
        const int window_end = w.keys.sink_chunks + w.keys.near_chunks;  // chunks from here on need the tile's ids
        const int c0 = u0 << a.unit_shift;
        while (true) {
            int c = c0 + warp;
            // the chunks in flight: a shift register of kStages - 1 descriptors, and one chunk whose pages are looked up
            Chunk flight[S::kStages - 1];
            Found found[S::kStages];
            const auto begin_stages = [&](int from, int to) {
#pragma unroll
                for (int s = 0; s < S::kStages; ++s)
                    if (s >= from && s < to && c + s * kWarps < c1) found[s] = w.find(c + s * kWarps);
#pragma unroll
                for (int s = 0; s < S::kStages - 1; ++s)
                    if (s >= from && s < to) {
                        if (c + s * kWarps < c1) flight[s] = w.load(found[s], s);
                        copy_commit();
                    }
            };
            int ready = S::kStages;
            if (kIds && !w.safe && c1 > window_end) {
                // those of the first chunks that need no ids, so that their copies are under way while the ids are read
                ready = max(0, min(ready, (window_end - c0) / kWarps));
                begin_stages(0, ready);
                int* list = reinterpret_cast<int*>(smem + S::kIdsAt);
                w.stage_ids(list, list + kMaxIds, w.list_heads(tile));
                w.staged = list;
                begin_stages(ready, S::kStages);
            } else {
                begin_stages(0, S::kStages);
            }
            Found next_up = found[S::kStages - 1];
            int stage = 0;
            for (; c < c1; c += kWarps) {
                copy_wait<S::kStages - 2>();
                __syncwarp();
                const Chunk now = flight[0];
#pragma unroll
                for (int s = 0; s + 1 < S::kStages - 1; ++s) flight[s] = flight[s + 1];
                const int ahead = c + (S::kStages - 1) * kWarps;
                int next = stage + S::kStages - 1;
                if (next >= S::kStages) next -= S::kStages;
                if (ahead < c1) {
                    flight[S::kStages - 2] = w.load(next_up, next);
                    if (ahead + kWarps < c1) next_up = w.find(ahead + kWarps);
                }
                copy_commit();
                w.compute(now, stage, c - window_end);
                if (++stage == S::kStages) stage = 0;
                __syncwarp();
            }
            copy_wait<0>();
            if (w.safe || !w.tainted()) break;
            w.safe = true;
            w.clear();
            __syncwarp();
        }

        // the next tile's request and ids are read beside the join
        Request next_req = w.req;
        int next_head = head, next_request = request, next_number = tile;
        const bool more = pl.end - tile_last > a.tile_units && next_tile<kRows, kIds ? kToken : kPacked>(a, &next_req, &next_head, &next_request, &next_number);
        if (kIds && more) w.read_ids(next_req, next_head, next_number);

        // join the warps: rows of (m, l) and sums, over the rings
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            w.l[x] += __shfl_xor_sync(0xFFFFFFFFu, w.l[x], 1);
            w.l[x] += __shfl_xor_sync(0xFFFFFFFFu, w.l[x], 2);
        }
        __syncthreads();
        constexpr float kUnlift = 1.f / Warp<T, kDim, kIds>::kLift;
        constexpr int kSumPitch = kDim + 4;
        float* sums = reinterpret_cast<float*>(smem);                       // [warp][row][kSumPitch]
        float* stat = sums + kWarps * kRows * kSumPitch;                    // [warp][row][2]
        static_assert((kWarps * kRows * (kSumPitch + 2)) * 4 <= S::kBytes, "the join fits the rings");
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int row = (lane >> 2) + 8 * x;
            float* dst = sums + (warp * kRows + row) * kSumPitch + (lane & 3) * 2;
#pragma unroll
            for (int n = 0; n < kDim / 8; ++n)
                *reinterpret_cast<float2*>(dst + n * 8) = make_float2(w.o[n][2 * x] * kUnlift, w.o[n][2 * x + 1] * kUnlift);
            if ((lane & 3) == 0) {
                stat[(warp * kRows + row) * 2] = w.m[x];
                stat[(warp * kRows + row) * 2 + 1] = w.l[x];
            }
        }
        __syncthreads();
        const bool whole_tile = u0 == 0 && u1 == w.keys.units - a.tile_units;
        float* part = nullptr;
        if (!whole_tile) {
            const size_t slot = 2 * static_cast<size_t>(blockIdx.x) + (first_segment ? 0 : 1);
            part = reinterpret_cast<float*>(ws + workspace_records_bytes(a.ctas)) + slot * partial_floats(kRows, kDim);
        }
        for (int idx = threadIdx.x; idx < kRows * (kDim / 4); idx += kThreads) {
            const int row = idx / (kDim / 4), d = (idx % (kDim / 4)) * 4;
            float mm = -INFINITY;
#pragma unroll
            for (int y = 0; y < kWarps; ++y) mm = fmaxf(mm, stat[(y * kRows + row) * 2]);
            const float ref = mm == -INFINITY ? 0.f : mm;
            float ll = 0.f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int y = 0; y < kWarps; ++y) {
                const float f = exp2_fast(stat[(y * kRows + row) * 2] - ref);
                ll += stat[(y * kRows + row) * 2 + 1] * f;
                const float4 v = *reinterpret_cast<const float4*>(sums + (y * kRows + row) * kSumPitch + d);
                acc.x += v.x * f;
                acc.y += v.y * f;
                acc.z += v.z * f;
                acc.w += v.w * f;
            }
            if (whole_tile) {
                int i, g;
                if (Tiles<kRows, kIds ? kToken : kPacked>::row(a, w.req, tile, row, &i, &g)) {
                    const float inv = ll == 0.f ? 1.f : 1.f / ll;
                    const int64_t token = w.req.start + i;
                    const int h = head * a.group + g;
                    T* out = static_cast<T*>(a.out) + token * a.out_token_stride + h * a.out_head_stride + d;
                    *reinterpret_cast<uint2*>(out) = make_uint2(Half2<T>::pack(acc.x * inv, acc.y * inv),
                                                                Half2<T>::pack(acc.z * inv, acc.w * inv));
                    if (d == 0 && a.lse) a.lse[token * a.heads + h] = ll == 0.f ? -INFINITY : (mm + log2f(ll)) * kLn2;
                }
            } else {
                *reinterpret_cast<float4*>(part + row * kDim + d) = acc;
                if (d == 0) {
                    part[kRows * kDim + row] = mm;
                    part[kRows * kDim + kRows + row] = ll;
                }
            }
        }
        if (!more) break;
        unit = tile_first = tile_last;
        w.req = next_req;
        head = next_head;
        request = next_request;
        tile = next_number;
        w.keys = tile_keys<kRows, kIds ? kToken : kPacked, kChunk>(a, w.req, tile);
        first_segment = false;
        __syncthreads();  // the join's reads end before the next tile's copies
    }
}

// log2 of the chunks in a unit where tiles are split: one for each warp, more only where the table's width and the counts
// do not exclude 2^31 units of a kv head (thousands of requests that share a context of millions of keys, a prompt of 2^19
// tiles).
int unit_shift(const AttentionParams& a) {
    const int64_t keys = std::min<int64_t>(static_cast<int64_t>(a.table_width) * a.page_size, INT32_MAX);
    const int64_t heads = a.ids_count > 0 ? std::min(a.group, a.tile_rows) : 0;
    const int64_t chunks = keys / kChunk + 4 + heads * ((a.ids_count + kChunk - 1) / kChunk);
    const int64_t tiles = a.ids_count > 0 ? static_cast<int64_t>(a.tokens) * ((a.group + a.tile_rows - 1) / a.tile_rows)
                                          : static_cast<int64_t>(a.tokens) * a.group / kRows + a.requests;
    int shift = 2;
    while (shift < 24 && tiles * ((chunks >> shift) + 1 + kTileUnits) > INT32_MAX) ++shift;
    return shift;
}

template <typename T, int kDim, bool kIds>
cudaError_t launch(AttentionParams a, cudaStream_t stream) {
    using S = Smem<kDim, kIds>;
    static_assert((S::kBytes + 1024) * kCtasPerSm <= 228 * 1024, "two CTAs' shared memory");
    constexpr int most = std::max(S::kBytes, locate_bytes(kMaxRequests));
    static_assert(most <= 227 * 1024, "a CTA's shared memory");
    const int bytes = std::max(S::kBytes, locate_bytes(a.requests));
    a.base_align = kChunk;
    a.tile_rows = tile_rows(a);
    const bool split = attention_rows_splits(a);
    a.ctas *= kCtasPerSm;
    a.unit_shift = split ? unit_shift(a) : 24;  // a unit: one chunk for each warp (or more, see there), or a tile
    a.tile_units = split ? kTileUnits : 0;
    static SmemOnce once;
    cudaError_t e = once.set(reinterpret_cast<const void*>(attention_rows_kernel<T, kDim, kIds>), most);
    if (e != cudaSuccess) return e;
    attention_rows_kernel<T, kDim, kIds><<<a.ctas, kThreads, bytes, stream>>>(a);
    if ((e = cudaGetLastError()) != cudaSuccess || !split) return e;
    return launch_combine<T, kRows, kDim, kIds ? kToken : kPacked, 1>(a, stream);
}

template <typename T, int kDim>
cudaError_t by_ids(const AttentionParams& a, cudaStream_t s) {
    return a.ids ? launch<T, kDim, true>(a, s) : launch<T, kDim, false>(a, s);
}
template <typename T>
cudaError_t by_dim(const AttentionParams& a, cudaStream_t s) {
    switch (a.dim) {
        case 64: return by_ids<T, 64>(a, s);
        case 96: return by_ids<T, 96>(a, s);
        default: return by_ids<T, 128>(a, s);
    }
}

}  // namespace
}  // namespace attn

size_t attention_rows_workspace(const AttentionParams& a, int sms, int dim) {
    if (!attention_rows_splits(a)) return 0;
    const int ctas = sms * kCtasPerSm;
    return attn::workspace_records_bytes(ctas) + 2 * static_cast<size_t>(ctas) * attn::partial_floats(kRows, dim) * sizeof(float);
}
int attention_max_requests() { return attn::kMaxRequests; }
int attention_max_ids() { return kMaxIds; }

cudaError_t launch_attention_rows(const AttentionParams& a, cudaStream_t stream) {
    return a.dtype == FG_DTYPE_BF16 ? attn::by_dim<__nv_bfloat16>(a, stream) : attn::by_dim<__half>(a, stream);
}

}  // namespace fg
