// Attention of one or a few new tokens per sequence over a paged cache: HBM-bound streaming of K and V.
//
// The group x tokens (at most 16) query rows that share a kv head are the M = 16 rows of one mma.sync tile, so every K
// and V byte is read once.  16 FLOP per byte with 4x row padding is far below what mma.sync gives; a 128-row tcgen05
// tile would be seven eighths empty and its TMEM round trip longer than the tile's loads.
//
// A persistent CTA per SM takes its part of all tiles (128 positions of one item; paged_attn.cuh says how they are
// shared out), whatever items these belong to, and its ring of tiles never drains between items.
//   warps 8-10  loads, K, V and an 8-bit cache's exponent bytes: page numbers of the next tile are on their way while
//               this one waits for its slot; a TMA box per page; what the consumers have to know of the tile
//   warps 0-7   16 keys of every tile each: S = Q K^T, online softmax in registers, O += P V with P straight from the
//               accumulators; at the end of an item the eight states are merged through shared memory
//
// 8-bit rows become fp16, not the query's type: e4m3 -> fp16 is one exact instruction, and the rows' 2^e (exact in
// fp16) are multiplied into S for K, into the fragments for V.  bf16 queries are brought to fp16 scaled by a power of
// two per row, so that only elements below 2^-14 of the row's largest lose bits (2^-25 of it at most).  P is rounded to
// the 16-bit type that multiplies V, as in the dense kernels; maxima, sums and accumulators are fp32.
//
// Measured (32 query heads over 8 kv heads of 128).  64 single tokens over 512 .. 16384 positions, bf16: 340 to 346 us with
// pages of 64 or 16, 6.5 TB/s, what a copy gets; 256 over 200 .. 1000 120 us (5.3 TB/s), 128 over 100 .. 300 45 to 47 us, where items'
// starts and ends count.  One token over 1000 positions: 12 us with the join, all latency.
// 48 x 4 tokens over up to 8192 positions of an 8-bit cache: 124 us, 3.5 TB/s (a 16-bit one 149): there the consumers'
// instructions bound it, not the memory.  A warp's part of a tile takes 1440 cycles, at 442 instructions and two warps on a
// scheduler, and about 300 go by around it, where the loads alone would allow 1350.  Twelve consumer warps do not fit (128
// registers a thread: 173 us), e4m3 by shifts instead of conversions costs more instructions than it saves (157 us; half and
// half 142), 32 keys a warp on every other tile brought nothing.
#include <cmath>
#include <type_traits>

#include "paged_attn.cuh"
#include "tc_prims.cuh"
#include "tma_host.cuh"

namespace pb {
namespace {

using namespace tc;

constexpr int kConsumers = 8;
constexpr int threads_of(bool e8) { return (kConsumers + (e8 ? 3 : 2)) * 32; }
constexpr int kRows = 16;
constexpr int kMaxStages = 8;
constexpr int kMetaBytes = 48;

// What a stage of the ring holds: K tile, V tile, the query rows (first tile of an item), exponents.
template <bool E8, int HD> struct Ring {
    static constexpr int kRow = E8 ? HD : 128;                    // bytes of a swizzled row
    static constexpr int kSlabs = E8 ? 1 : HD / 64;
    static constexpr int kSlab = kTileKeys * kRow;
    static constexpr int kTile = kSlabs * kSlab;
    static constexpr int kQ = 2 * kTile;                           // offset of the query rows
    static constexpr int kExp = kQ + (HD / 64) * kRows * 128;      // K's exponent bytes, then V's
    static constexpr int kBytes = kExp + (E8 ? 1024 : 0);          // a multiple of 1024
    // Columns of the outputs that are merged at a time: 64, in 32 KB, or half that where three whole stages leave no more.
    static constexpr int kMergeCols = E8 || HD == 64 ? 64 : 32;
    static constexpr int kMergeBytes = kConsumers * kRows * kMergeCols * 4;
    static constexpr int kFit = (224 * 1024 - kMergeBytes) / kBytes;
    static constexpr int kStages = kFit < kMaxStages ? kFit : kMaxStages;
    static constexpr int kMerge = kStages * kBytes;
    static constexpr int kMl = kMerge + kMergeBytes;               // [8][16] maxima, [8][16] sums, of this item and the last
    static constexpr int kMeta = kMl + 4 * kConsumers * kRows * 4;
    static constexpr int kSums = kMeta + kMaxStages * kMetaBytes;
    static constexpr int kThreads = threads_of(E8);
    static constexpr int kBars = kSums + (kThreads / 32 + 3) * 8;
    static constexpr int kMisc = kBars + (2 * kMaxStages + 1) * 8 + 8;
    static constexpr int kLaunch = kMisc + 16 + 1024;
    static_assert(kLaunch <= 227 * 1024, "shared memory of a CTA");
    static_assert(kBytes % 1024 == 0 && kMeta % 16 == 0 && kSums % 8 == 0, "alignment");
};

struct alignas(16) TileMeta {        // kMetaBytes, one per stage
    int key0;
    int flags;           // 1 first tile of the item here, 2 last, 4 the item is not whole here, 8 keys are to be masked
    uint32_t pages;      // bit i: page i of the tile is there
    int kend;            // positions the item attends: keys from here on are not
    // with an item's first and last tile only
    int row0, nq, hk, slot;
    int pos0;
    int pad[3];
};
static_assert(sizeof(TileMeta) == kMetaBytes, "");

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
// Two 16 x 16 matrices of bytes, transposed: lane l of a row group g = l / 4, t = l % 4 gets, of the first, bytes
// (row 4t .. 4t+3, column g) and (.., column g + 8), then the same of the second.  Lanes 0-15 and 16-31 name their rows.
__device__ __forceinline__ void ldsm2_t8(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
template <bool BF16>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (BF16) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    } else {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
    const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
    uint32_t r;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(r) : "r"(a));
    return r;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
    uint2 r;
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "r"(a));
    return r;
}

// 5-D tiled load global -> shared, completion on an mbarrier.
__device__ __forceinline__ void tma_load_5d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2, int c3, int c4) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4)
        : "memory");
}

// Byte offset of 16-byte unit c of row r in a tile that TMA wrote with the 128- or 64-byte swizzle.
template <int ROW>
__device__ __forceinline__ uint32_t swz(int r, int c) {
    if constexpr (ROW == 128) return uint32_t(r * 128 + ((c ^ (r & 7)) << 4));
    else return uint32_t(r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
}

// Tiles of a sequence's items: one item per kv head.  A sequence with new tokens and nothing to attend has one empty tile
// per item (its rows are zeros), one without new tokens none.
__device__ __forceinline__ int seq_keys(const PagedParams& p, const PagedSeq& s) { return paged_keys(p, s, s.nq - 1); }
__device__ __forceinline__ int seq_tiles(const PagedParams& p, const PagedSeq& s) {
    return s.nq <= 0 ? 0 : max(1, (seq_keys(p, s) + kTileKeys - 1) / kTileKeys);
}

template <bool BF16, bool E8, int HD>
__global__ void __launch_bounds__(Ring<E8, HD>::kThreads, 1)
paged_decode_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                    const __grid_constant__ CUtensorMap map_v, const PagedParams p, const PagedWorkspace ws) {
    using R = Ring<E8, HD>;
    constexpr bool kBfOps = BF16 && !E8;     // type of the MMA operands
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
    auto full = [&](int s) { return base + R::kBars + 8u * s; };
    auto empty = [&](int s) { return base + R::kBars + 8u * (kMaxStages + s); };
    const uint32_t merge_bar = base + R::kBars + 8u * (2 * kMaxStages);
    TileMeta* meta = reinterpret_cast<TileMeta*>(gen + R::kMeta);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(gen + R::kMisc);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < R::kStages; ++s) {
            mbar_init(full(s), E8 ? 2 + 32 : 2);      // K's and V's producers, a lane each of the exponents'
            mbar_init(empty(s), kConsumers);
        }
        mbar_init(merge_bar, kConsumers);
        *abort_flag = 0;
        mbar_fence_init();
        fence_proxy_async_smem();
    }
    if (!p.wait_late) asm volatile("griddepcontrol.wait;" ::: "memory");
    int b0;
    int64_t base0;
    const PagedRange range = paged_range(p.B, reinterpret_cast<int64_t*>(gen + R::kSums),
                                         [&](int b) { return int64_t(p.Hkv) * seq_tiles(p, paged_seq(p, b)); }, &b0, &base0);
    const int ntiles = int(range.end - range.begin);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    if (warp >= kConsumers) {
        // ------------------------------ producers ------------------------------
        // Each walks the same tiles: warp 8 issues K's boxes (and the queries') and describes the tile, warp 9 V's, warp 10
        // brings the exponents of an 8-bit cache.
        if (lane == 0) {
            tma_prefetch_desc(&map_q);
            tma_prefetch_desc(&map_k);
            tma_prefetch_desc(&map_v);
        }
        const int role = warp - kConsumers;
        PagedJoin join{};
        join.first_slot = -1;
        const bool exp4 = E8 && p.eks[2] == 1 && p.evs[2] == 1 && ((p.eks[0] | p.eks[1] | p.evs[0] | p.evs[1]) & 3) == 0 &&
                          ((reinterpret_cast<uintptr_t>(p.ek) | reinterpret_cast<uintptr_t>(p.ev)) & 3) == 0;
        // where the tile to be asked for next stands
        PagedSeq sq{};
        int b = b0, hk = 0, tile = 0, nt = 0, kend = 0;
        int64_t item0 = 0;       // place of the item's first tile
        auto enter = [&]() {     // the first sequence from b on that has tiles
            for (; b < p.B; ++b) {
                sq = paged_seq(p, b);
                nt = seq_tiles(p, sq);
                if (nt > 0) break;
            }
            kend = nt > 0 ? seq_keys(p, sq) : 0;
        };
        if (ntiles > 0) {
            enter();
            const int64_t in = range.begin - base0;
            hk = int(in / nt);
            tile = int(in - int64_t(hk) * nt);
            item0 = base0 + int64_t(hk) * nt;
        }
        // Page numbers come 32 at a time, the next 32 on their way while these are used: with the ring full of loads a
        // further one takes microseconds.  The walk over the batches runs ahead of the walk over the tiles.
        auto entry_of = [&](int t) { return p.tpp > 1 ? t / p.tpp : t * p.npg; };    // of the tile's first box in the table
        int lb = b, lhk = hk, lbatch = 0, lnb = 0;
        auto load_batch = [&]() -> int {
            const int e = lbatch * 32 + lane;
            return lb < p.B && e < p.max_pages ? __ldg(p.table + int64_t(lb) * p.table_stride + e) : -1;
        };
        auto next_batch = [&]() {
            if (lb < p.B && ++lbatch == lnb) {
                lbatch = 0;
                if (++lhk == p.Hkv) {
                    lhk = 0;
                    int n = 0;
                    while (n == 0 && ++lb < p.B) n = seq_tiles(p, paged_seq(p, lb));
                    lnb = n > 0 ? (entry_of(n - 1) >> 5) + 1 : 0;
                }
            }
        };
        int batch = 0, cur = -1, nxt = -1;
        if (ntiles > 0) {
            lbatch = batch = entry_of(tile) >> 5;
            lnb = (entry_of(nt - 1) >> 5) + 1;
            cur = load_batch();
            next_batch();
            nxt = load_batch();
        }
        // lane i: page number of box i of the tile, -1 when it is not there or not to be read
        auto page_of = [&]() -> int {
            const int pg = __shfl_sync(0xffffffffu, cur, (entry_of(tile) & 31) + lane);
            return lane < p.npg && tile * kTileKeys + (lane << p.box_shift) < kend && uint32_t(pg) < uint32_t(p.pages) ? pg : -1;
        };
        // on to the next tile, and to its batch of page numbers
        auto advance = [&]() {
            bool item = false;
            if (++tile == nt) {
                item = true;
                tile = 0;
                item0 += nt;
                if (++hk == p.Hkv) {
                    hk = 0;
                    ++b;
                    enter();
                }
            }
            const int now = entry_of(tile) >> 5;
            if (item || now != batch) {
                batch = now;
                cur = nxt;
                next_batch();
                nxt = load_batch();
            }
        };
        auto row_of = [&]() { return p.tpp > 1 ? (tile % p.tpp) * kTileKeys : 0; };     // the tile's first row in its page
        if (role == 2) {
            // Exponent bytes: lane l brings those of the keys 4l .. 4l+3, as copies that the stage's barrier waits for; 127
            // where no page is.
            for (int i = 0; i < ntiles; ++i) {
                const int s = i % R::kStages;
                if (!__all_sync(0xffffffffu, mbar_wait(empty(s), ((i / R::kStages) & 1) ^ 1u, abort_flag, 2))) break;
                const uint32_t dst = base + s * R::kBytes + R::kExp + lane * 4;
                const int key = 4 * lane, pg = page_of();
                const int mine = __shfl_sync(0xffffffffu, pg, key >> p.box_shift);
                const int off = row_of() + (key & ((1 << p.box_shift) - 1));
                const int64_t page = max(mine, 0);
                const uint8_t* k = p.ek + page * p.eks[0] + int64_t(hk) * p.eks[1] + int64_t(off) * p.eks[2];
                const uint8_t* v = p.ev + page * p.evs[0] + int64_t(hk) * p.evs[1] + int64_t(off) * p.evs[2];
                if (mine >= 0 && exp4) {
                    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(k) : "memory");
                    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst + 128), "l"(v) : "memory");
                    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(full(s)) : "memory");
                } else {      // (ordinary stores, which an ordinary arrival releases)
                    uint32_t ek = 0x7f7f7f7fu, ev = 0x7f7f7f7fu;
                    if (mine >= 0) {
                        ek = ev = 0;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            ek |= uint32_t(k[e * p.eks[2]]) << (8 * e);
                            ev |= uint32_t(v[e * p.evs[2]]) << (8 * e);
                        }
                    }
                    asm volatile("st.shared.b32 [%0], %1;" ::"r"(dst), "r"(ek) : "memory");
                    asm volatile("st.shared.b32 [%0], %1;" ::"r"(dst + 128), "r"(ev) : "memory");
                    mbar_arrive(full(s));
                }
                if (i + 1 < ntiles) advance();
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
        }
        bool first = true;
        for (int i = 0; role != 2 && i < ntiles; ++i) {
            const int pg = page_of(), row = row_of();
            const int s = i % R::kStages;
            if (!__all_sync(0xffffffffu, mbar_wait(empty(s), ((i / R::kStages) & 1) ^ 1u, abort_flag, 2))) break;
            const uint32_t dst = base + s * R::kBytes;
            const bool last = tile + 1 == nt || i + 1 == ntiles;
            // (pages outside the tensor read as zeros)
            const bool has = pg >= 0;
            const int page = has ? pg : p.pages;
            if (role == 0) {
                const uint32_t there = __ballot_sync(0xffffffffu, has);
                if (lane == 0) {
                    TileMeta& m = meta[s];
                    const int key0 = tile * kTileKeys;
                    // every row attends every key of the tile, and all of it is there
                    const int all = p.causal ? min(kend, sq.pos0 + 1) : kend;
                    const bool full_tile = key0 + kTileKeys <= all && there == (1u << p.npg) - 1u;
                    int flags = (first ? 1 : 0) | (last ? 2 : 0) | (full_tile ? 0 : 8);
                    if (first || last) {
                        const bool whole = item0 >= range.begin && item0 + nt <= range.end;
                        flags |= whole ? 0 : 4;
                        // the item the range begins with leaves its part in slot 2c, a later one that goes on in 2c+1
                        const int slot = 2 * int(blockIdx.x) + (item0 > range.begin ? 1 : 0);
                        m.row0 = sq.row0;
                        m.nq = sq.nq;
                        m.hk = hk;
                        m.slot = slot;
                        m.pos0 = sq.pos0;
                        if (!whole && item0 >= range.begin) {
                            join.first_slot = slot;
                            join.last_cta = range.owner(item0 + nt - 1);
                            join.row0 = sq.row0;
                            join.nq = sq.nq;
                            join.hk = hk;
                        }
                    }
                    m.key0 = key0;
                    m.flags = flags;
                    m.pages = there;
                    m.kend = kend;
                }
            }
            const CUtensorMap* map = role ? &map_v : &map_k;
            const uint32_t at = dst + (role ? R::kTile : 0);
            if (lane == 0)
                mbar_arrive_expect_tx(full(s), R::kTile + (role == 0 && first ? (HD / 64) * p.qbox * p.group * 128 : 0));
            __syncwarp();
            // one lane issues: a box per lane would be issued one after the other too, with a loop around it
            for (int x = 0; x < p.npg; ++x) {
                const int pgx = __shfl_sync(0xffffffffu, page, x);
                if (lane == 0) tma_load_5d(at + (x << p.box_shift) * R::kSlabs * R::kRow, map, full(s), 0, row, 0, hk, pgx);
            }
            if (role == 0 && first && lane == 0) {
#pragma unroll
                for (int c = 0; c < HD / 64; ++c)
                    tma_load_4d(dst + R::kQ + c * kRows * 128, &map_q, full(s), 64 * c, 0, hk, sq.row0);
            }
            first = last;
            if (i + 1 < ntiles) advance();
        }
        if (role == 0 && lane == 0) ws.join[blockIdx.x] = join;
    } else {
        // ------------------------------ consumers ------------------------------
        const int r0 = lane >> 2, t = lane & 3;
        const int krow = warp * 16;             // this warp's keys in a tile
        // A tile is boxes of 2^box_shift keys, each with its slabs of 128-byte rows one after the other: where row r's
        // first slab begins, and how far the next one is.
        auto row_at = [&](int r) {
            return uint32_t(((r >> p.box_shift) << p.box_shift) * R::kSlabs + (r & ((1 << p.box_shift) - 1))) * uint32_t(R::kRow);
        };
        const uint32_t slab_step = uint32_t(R::kRow) << p.box_shift;
        // of K, column n of an n-tile is any key: key n of 8, or, where four keys of V share a register, the one that leaves a
        // thread with keys 4t, 4t+1 of the first n-tile and 4t+2, 4t+3 of the second
        int krows[2];
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) krows[nt] = krow + (E8 ? 4 * ((lane & 7) >> 1) + 2 * nt + (lane & 1) : nt * 8 + (lane & 7));
        const uint32_t k_at[2] = {row_at(krows[0]), row_at(krows[1])}, v_at = row_at(krow + (lane & 15));
        // 16-byte unit c of row r of a slab, swizzled
        auto unit = [](int r, int c) { return swz<R::kRow>(r, c) - uint32_t(r * R::kRow); };
        float* merge = reinterpret_cast<float*>(gen + R::kMerge);
        float* m_sm = reinterpret_cast<float*>(gen + R::kMl);
        float* l_sm = m_sm + kConsumers * kRows;
        int other = 2 * kConsumers * kRows;     // to the next item's maxima and sums
        // row / group without a division for every item (rows below 16, groups up to 16); kept for this thread's rows where
        // registers are short
        const int by_group = E8 ? (65536 + p.group - 1) / p.group : 0;
        const int toks[2] = {E8 ? 0 : r0 / p.group, E8 ? 0 : (r0 + 8) / p.group};
        uint32_t qf[HD / 16][4];
        float acc[HD / 8][4];
        float m_run[2], l_run[2];       // reference (in units of S) and sum of a row
        float c2[2], lag[2];            // S * c2 is the exponent of 2; 2^8 in units of S
        const float lag0 = 8.f / p.scale_log2;
        int lim[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            m_run[h] = -INFINITY;
            l_run[h] = 0.f;
            c2[h] = p.scale_log2;
            lag[h] = lag0;
            lim[h] = 0;
        }
#pragma unroll
        for (int i = 0; i < HD / 8; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][e] = 0.f;
#pragma unroll
        for (int i = 0; i < HD / 16; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) qf[i][e] = 0u;
        // a barrier of the consumer warps, bounded like every other wait (a hardware barrier would not be)
        bool ok = true;
        uint32_t merge_phase = 0;
        auto merge_sync = [&]() {
            __syncwarp();
            if (lane == 0) mbar_arrive(merge_bar);
            ok = __all_sync(0xffffffffu, ok && mbar_wait(merge_bar, merge_phase & 1u, abort_flag, 4));
            ++merge_phase;
        };
        for (int i = 0; ok && i < ntiles; ++i) {
            const int s = i % R::kStages;
            if (!__all_sync(0xffffffffu, mbar_wait(full(s), (i / R::kStages) & 1, abort_flag, 3))) break;
            const uint32_t kt = base + s * R::kBytes, vt = kt + R::kTile;
            const TileMeta& md = meta[s];
            const int4 head = *reinterpret_cast<const int4*>(&md);       // key0, flags, pages, kend
            const int flags = head.y, key0 = head.x, kend = head.w;
            if (flags & 1) {
                // ---- a new item: query fragments, limits, empty state ----
                const uint32_t qt = kt + R::kQ;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int r = r0 + 8 * h;
                    m_run[h] = -INFINITY;
                    l_run[h] = 0.f;
                    lim[h] = p.causal ? min(kend, md.pos0 + (E8 ? (r * by_group) >> 16 : toks[h]) + 1) : kend;
                    if constexpr (!E8) {
                        // a0/a1: d = 16 ks + 2t (+1); a2/a3: d + 8
#pragma unroll
                        for (int ks = 0; ks < HD / 16; ++ks) {
                            const uint32_t a = qt + (ks >> 2) * kRows * 128 + t * 4;
                            qf[ks][h] = lds32(a + swz<128>(r, (ks & 3) * 2));
                            qf[ks][2 + h] = lds32(a + swz<128>(r, (ks & 3) * 2 + 1));
                        }
                    } else {
                        // the contraction index is free to choose: k = 2t, 2t+1 stand for d = 16 ks + 4t, +1 and
                        // k + 8 for d + 2, +3, which is how four e4m3 bytes of a fragment lie
                        float amax = 0.f;
#pragma unroll
                        for (int ks = 0; ks < HD / 16; ++ks) {
                            const uint32_t a = qt + (ks >> 2) * kRows * 128 + swz<128>(r, (ks & 3) * 2 + (t >> 1)) + (t & 1) * 8;
                            const uint2 w = lds64(a);
                            qf[ks][h] = w.x;
                            qf[ks][2 + h] = w.y;
                            if constexpr (BF16) {
                                const float2 x = pair16_to_f32<true>(w.x), y = pair16_to_f32<true>(w.y);
                                amax = fmaxf(fmaxf(amax, fmaxf(fabsf(x.x), fabsf(x.y))), fmaxf(fabsf(y.x), fabsf(y.y)));
                            }
                        }
                        if constexpr (BF16) {
                            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
                            // largest magnitude to [1, 2)
                            const int ex = max(-120, min(120, int(__float_as_uint(amax) >> 23) - 127));
                            const float f = pow2f(-ex);
                            c2[h] = fmaxf(p.scale_log2 * pow2f(ex), kLeastC2);
                            lag[h] = fminf(lag0 * f, 1e37f);       // (8 / c2)
#pragma unroll
                            for (int ks = 0; ks < HD / 16; ++ks) {
                                const float2 x = pair16_to_f32<true>(qf[ks][h]), y = pair16_to_f32<true>(qf[ks][2 + h]);
                                qf[ks][h] = pack16<false>(x.x * f, x.y * f);
                                qf[ks][2 + h] = pack16<false>(y.x * f, y.y * f);
                            }
                        }
                    }
                }
#pragma unroll
                for (int x = 0; x < HD / 8; ++x)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[x][e] = 0.f;
            }
            // All fragments of a product are asked for before its first MMA, and V's before the softmax: with two warps
            // on a scheduler nothing else would hide the loads.
            constexpr int kLd = R::kTile / 4096;     // ldmatrix.x4 of 16 rows
            uint32_t kf[kLd][4], vf[kLd][4];
#pragma unroll
            for (int x = 0; x < kLd; ++x) {
                const int c = (x >> 1) * 4 + (lane >> 3);   // 16-byte unit of the row
                ldsm4(kt + k_at[x & 1] + (E8 ? unit(krows[x & 1], c) : (c >> 3) * slab_step + unit(krows[x & 1], c & 7)), kf[x]);
            }
            // ---- S = Q K^T: two n-tiles of 8 keys ----
            float sc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
            for (int x = 0; x < kLd; ++x) {
                const int nt = x & 1, k = x >> 1;
                if constexpr (!E8) {
                    mma<kBfOps>(sc[nt], qf[2 * k], kf[x][0], kf[x][1]);
                    mma<kBfOps>(sc[nt], qf[2 * k + 1], kf[x][2], kf[x][3]);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        uint32_t lo, hi;
                        e4m3x4_to_f16x4(kf[x][e], &lo, &hi);
                        mma<false>(sc[nt], qf[4 * k + e], lo, hi);
                    }
                }
            }
#pragma unroll
            for (int x = 0; x < kLd; ++x) {
                const int row = krow + (lane & 15), c = x * 2 + (lane >> 4);
                if constexpr (E8) ldsm2_t8(vt + v_at + unit(row, c), vf[x]);
                else ldsm4_t(vt + v_at + (c >> 3) * slab_step + unit(row, c & 7), vf[x]);
            }
            // this thread's columns of n-tile nt: keys first + step * nt, + 1
            const int first = krow + (E8 ? 4 : 2) * t;
            constexpr int kStep = E8 ? 2 : 8;
            uint32_t ek = E8 ? lds32(kt + R::kExp + first) : 0u;
            uint32_t ev = E8 ? lds32(kt + R::kExp + 128 + first) : 0u;
            // 2^(byte - 127) of byte i (zero for a byte of 0, which no cache holds)
            auto scale_of = [](uint32_t w, int i) { return __uint_as_float(((w >> (8 * i)) & 0xffu) << 23); };
            if constexpr (E8) {
#pragma unroll
                for (int nt = 0; nt < 2; ++nt) {
                    const float k0 = scale_of(ek, 2 * nt), k1 = scale_of(ek, 2 * nt + 1);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        sc[nt][2 * h] *= k0;
                        sc[nt][2 * h + 1] *= k1;
                    }
                }
            }
            // ---- mask, online softmax ----
            const int kb = key0 + first;
            if (flags & 8) {
                // (a page holds whole groups of 8 keys, so both of an n-tile's)
                const uint32_t here0 = (md.pages >> (first >> p.box_shift)) & 1u;
                const uint32_t here1 = (md.pages >> ((first + kStep) >> p.box_shift)) & 1u;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            if (kb + nt * kStep + e >= lim[h] || !(nt ? here1 : here0)) sc[nt][2 * h + e] = -INFINITY;
            }
            // The reference m of a row lags behind its maximum: it moves when a score of the row has outgrown it by 2^8 (P stays far
            // inside 16 bits), which after an item's first tiles is rare, so that a tile usually needs no exchange between lanes.
            float mx[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) mx[h] = fmaxf(fmaxf(sc[0][2 * h], sc[0][2 * h + 1]), fmaxf(sc[1][2 * h], sc[1][2 * h + 1]));
            const bool over[2] = {mx[0] > m_run[0] + lag[0], mx[1] > m_run[1] + lag[1]};
            if (__any_sync(0xffffffffu, over[0] || over[1])) {
                float alpha[2];
                uint32_t up = (over[0] ? 1u : 0u) | (over[1] ? 2u : 0u);
                up |= __shfl_xor_sync(0xffffffffu, up, 1);
                up |= __shfl_xor_sync(0xffffffffu, up, 2);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
                    mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
                    // a row goes by its own scores: its bits depend neither on its neighbours nor on the rows of the tile of
                    // queries that no token fills, which hold anything
                    const float m_new = (up >> h) & 1u ? mx[h] : m_run[h];
                    alpha[h] = m_new == m_run[h] ? 1.f : ex2_approx((m_run[h] - m_new) * c2[h]);
                    l_run[h] *= alpha[h];
                    m_run[h] = m_new;
                }
#pragma unroll
                for (int x = 0; x < HD / 8; ++x) {
                    acc[x][0] *= alpha[0];
                    acc[x][1] *= alpha[0];
                    acc[x][2] *= alpha[1];
                    acc[x][3] *= alpha[1];
                }
            }
            float pr[2][4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float neg = m_run[h] == -INFINITY ? 0.f : -m_run[h] * c2[h];     // (no key yet: every P is 0)
#pragma unroll
                for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float pv = ex2_approx(fmaf(sc[nt][2 * h + e], c2[h], neg));
                        pr[nt][2 * h + e] = pv;
                        l_run[h] += pv;      // of this thread's keys; the quad is added up at the end of the item
                    }
            }
            // ---- O += P V ----
            if (key0 + kTileKeys > kend) {
                // past the end of the sequence the page holds anything, NaN too: 0 * NaN must not reach the sum
                if constexpr (E8) {
                    const int live = kend - kb;      // of the four keys of a register
                    const uint32_t keep = live >= 4 ? 0xffffffffu : live <= 0 ? 0u : (1u << (8 * live)) - 1u;
#pragma unroll
                    for (int x = 0; x < kLd; ++x)
#pragma unroll
                        for (int e = 0; e < 4; ++e) vf[x][e] &= keep;
                    ev = (ev & keep) | (0x7f7f7f7fu & ~keep);      // (an infinite 2^e would make NaN of the zeros)
                } else {
                    const uint32_t keep0 = (kb < kend ? 0xffffu : 0u) | (kb + 1 < kend ? 0xffff0000u : 0u);
                    const uint32_t keep1 = (kb + 8 < kend ? 0xffffu : 0u) | (kb + 9 < kend ? 0xffff0000u : 0u);
#pragma unroll
                    for (int x = 0; x < kLd; ++x)
#pragma unroll
                        for (int e = 0; e < 4; ++e) vf[x][e] &= (e & 1) ? keep1 : keep0;
                }
            }
            uint32_t pa[4];
            pa[0] = pack16<kBfOps>(pr[0][0], pr[0][1]);
            pa[1] = pack16<kBfOps>(pr[0][2], pr[0][3]);
            pa[2] = pack16<kBfOps>(pr[1][0], pr[1][1]);
            pa[3] = pack16<kBfOps>(pr[1][2], pr[1][3]);
            // (2^-15 is subnormal in fp16, which the conversion knows)
            const uint32_t sv01 = E8 ? pack16<false>(scale_of(ev, 0), scale_of(ev, 1)) : 0u;
            const uint32_t sv23 = E8 ? pack16<false>(scale_of(ev, 2), scale_of(ev, 3)) : 0u;
#pragma unroll
            for (int x = 0; x < kLd; ++x) {
                if constexpr (!E8) {
                    mma<kBfOps>(acc[2 * x], pa, vf[x][0], vf[x][1]);
                    mma<kBfOps>(acc[2 * x + 1], pa, vf[x][2], vf[x][3]);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        uint32_t lo, hi;
                        e4m3x4_to_f16x4(vf[x][e], &lo, &hi);
                        mma<false>(acc[4 * x + e], pa, hmul2(lo, sv01), hmul2(hi, sv23));
                    }
                }
            }
            int nq = 0, row_tok = 0, hk = 0, slot = 0;
            if (flags & 2) {
                nq = md.nq;
                row_tok = md.row0;
                hk = md.hk;
                slot = md.slot;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(empty(s));
            if (flags & 2) {
                // ---- the item ends here: the eight warps' states become one ----
                const int rows = nq * p.group;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 1);
                    l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 2);
                }
                // (the previous item's maxima and sums lie elsewhere, so that only the barrier behind these is needed: who passes
                // it has read all of the previous merge)
                if (t == 0) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        // (exponents of 2 from here on; scores of nothing but NaN leave no maximum, but their sum has to count)
                        m_sm[warp * kRows + r0 + 8 * h] = m_run[h] == -INFINITY && l_run[h] != l_run[h] ? 0.f : m_run[h] * c2[h];
                        l_sm[warp * kRows + r0 + 8 * h] = l_run[h];
                    }
                }
                merge_sync();
                float f[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float M = -INFINITY;
#pragma unroll
                    for (int w = 0; w < kConsumers; ++w) M = fmaxf(M, m_sm[w * kRows + r0 + 8 * h]);
                    f[h] = m_run[h] == -INFINITY ? 0.f : ex2_approx(m_run[h] * c2[h] - M);
                }
                // The outputs of RC rows, kCols columns at a time, through [warp][RC][kCols] fp32 in shared memory; 256 / RC threads
                // finish a row, whose maximum and sum they find once.  All columns at once where the rows are few: 128 single
                // tokens over 100 .. 300 positions 60 us with 32 columns a pass, 49 in one.
                const float *m_in = m_sm, *l_in = l_sm;
                auto finish = [&](auto rows_c, auto cols_c) {
                    constexpr int RC = decltype(rows_c)::value, kCols = decltype(cols_c)::value;
                    constexpr int kPerRow = kConsumers * 32 / RC, kMine = kCols / kPerRow;
                    static_assert(kMine >= 2 && kConsumers * RC * kCols * 4 <= R::kMergeBytes, "");
                    const int r = threadIdx.x / kPerRow, cp = threadIdx.x % kPerRow;
                    float M = -INFINITY, l = 0.f;
#pragma unroll
                    for (int w = 0; w < kConsumers; ++w) M = fmaxf(M, m_in[w * kRows + r]);
#pragma unroll
                    for (int w = 0; w < kConsumers; ++w) {
                        const float mw = m_in[w * kRows + r];
                        if (mw != -INFINITY) l = fmaf(l_in[w * kRows + r], ex2_approx(mw - M), l);
                    }
                    const float inv = M == -INFINITY ? 0.f : 1.0f / l;
                    const int rt = E8 ? (r * by_group) >> 16 : r / p.group, tok = row_tok + rt, hq = hk * p.group + (r - rt * p.group);
                    const size_t at = size_t(slot) * kRows + r;
                    uint16_t* out = static_cast<uint16_t*>(p.out) + int64_t(tok) * p.os[0] + int64_t(hq) * p.os[1];
                    if (r < rows && cp == 0) {
                        if (flags & 4) ws.ml[at] = make_float2(M, l);
                        else if (p.lse) p.lse[int64_t(tok) * p.Hq + hq] = M == -INFINITY ? -INFINITY : M * 0.6931471805599453f + logf(l);
                    }
                    // groups of 8 columns are exchanged by row so that the rows lie on different banks
#pragma unroll
                    for (int c = 0; c < HD / kCols; ++c) {
                        if (c > 0) merge_sync();
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int rr = r0 + 8 * h;
                            if (rr < rows && rr < RC) {
                                float* dst = merge + (warp * RC + rr) * kCols;
#pragma unroll
                                for (int x = 0; x < kCols / 8; ++x)
                                    *reinterpret_cast<float2*>(dst + 8 * (x ^ (rr & (kCols / 8 - 1))) + 2 * t) =
                                        make_float2(acc[c * (kCols / 8) + x][2 * h] * f[h], acc[c * (kCols / 8) + x][2 * h + 1] * f[h]);
                            }
                        }
                        merge_sync();
                        if (r < rows) {
                            float o[kMine];
#pragma unroll
                            for (int e = 0; e < kMine; ++e) o[e] = 0.f;
                            const int col = kMine * cp;
                            const float* src = merge + r * kCols + 8 * ((col >> 3) ^ (r & (kCols / 8 - 1))) + (col & 7);
#pragma unroll
                            for (int w = 0; w < kConsumers; ++w)
#pragma unroll
                                for (int e = 0; e < kMine; e += 2) {
                                    const float2 v = *reinterpret_cast<const float2*>(src + w * RC * kCols + e);
                                    o[e] += v.x;
                                    o[e + 1] += v.y;
                                }
#pragma unroll
                            for (int e = 0; e < kMine; e += 2) {
                                const int d = c * kCols + col + e;
                                if (flags & 4) {
                                    *reinterpret_cast<float2*>(ws.o + at * HD + d) = make_float2(o[e], o[e + 1]);
                                } else {
                                    const uint32_t w = pack16<BF16>(o[e] * inv, o[e + 1] * inv);
                                    out[d] = uint16_t(w);
                                    out[d + 1] = uint16_t(w >> 16);
                                }
                            }
                        }
                    }
                };
                m_sm += other;
                l_sm += other;
                other = -other;
                constexpr int kWhole = R::kMergeBytes / (kConsumers * HD * 4);     // rows that all columns are there for at once
                if (kWhole < kRows && rows <= kWhole) finish(std::integral_constant<int, kWhole < kRows ? kWhole : kRows>(), std::integral_constant<int, HD>());
                else finish(std::integral_constant<int, kRows>(), std::integral_constant<int, R::kMergeCols>());
            }
        }
    }
    // (launched beside the kernel for chunks, whose inputs are complete: only what follows must find both done)
    if (p.wait_late) asm volatile("griddepcontrol.wait;" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0 && *abort_flag) {
        drain_after_abort();
        *p.status = *abort_flag;
        __threadfence_system();
    }
}

template <bool BF16, bool E8, int HD>
int launch(int gpu, int G, cudaStream_t s, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const PagedParams& p,
           const PagedWorkspace& ws) {
    constexpr int bytes = Ring<E8, HD>::kLaunch;
    PB_CUDA((paged_allow_smem<paged_decode_kernel<BF16, E8, HD>>(gpu, bytes)));
    PB_CUDA(paged_launch(paged_decode_kernel<BF16, E8, HD>, dim3(unsigned(G)), Ring<E8, HD>::kThreads, bytes, s, mq, mk, mv, p, ws));
    return PARAS_OK;
}

}  // namespace

int paged_decode_rows() { return kRows; }

bool paged_decode_supported(const Gpu* g, const paras_paged_attn_args& a) {
    return g->cc_major >= 9 && a.dtype != PARAS_F32 && paged_tma_ok(a.cache) && paged_q_tma_ok(a) &&
           a.Hq / a.cache.Hkv <= kRows && paged_scale_ok(a) && g->smem_optin >= 227 * 1024;
}

int paged_decode_launch(Gpu* g, const paras_paged_attn_args& a, const PagedParams& p, const PagedWorkspace& ws, int G, cudaStream_t s) {
    int st = check_status_word(g);
    if (st != PARAS_OK) return st;
    CUtensorMap mq, mk, mv;
    if ((st = paged_q_map(&mq, a, p.qbox)) != PARAS_OK) return st;
    if ((st = paged_cache_map(&mk, a.cache, 0, true)) != PARAS_OK) return st;
    if ((st = paged_cache_map(&mv, a.cache, 1, true)) != PARAS_OK) return st;
    const bool bf = a.dtype == PARAS_BF16, e8 = a.cache.cache_dtype == PARAS_E4M3;
#define PB_GO(B, E, H) launch<B, E, H>(g->ordinal, G, s, mq, mk, mv, p, ws)
    if (p.D == 128) st = bf ? (e8 ? PB_GO(true, true, 128) : PB_GO(true, false, 128)) : (e8 ? PB_GO(false, true, 128) : PB_GO(false, false, 128));
    else st = bf ? (e8 ? PB_GO(true, true, 64) : PB_GO(true, false, 64)) : (e8 ? PB_GO(false, true, 64) : PB_GO(false, false, 64));
#undef PB_GO
    return st;
}

}  // namespace pb
