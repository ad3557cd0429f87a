// Attention of chunks of new tokens over a paged cache on the tensor cores (tcgen05, accumulators in TMEM).
//
// Per 128-position tile j and 128-row query tile t:  S_t = Q_t K_j^T,  P_t = exp2(c S_t - c m_t),  O_t += P_t V_j.
// Compute-bound from a few hundred query rows per kv head on; below that (a step that mixes single tokens with a chunk)
// the same kernel streams the cache.  The roles are the dense kernel's (sdpa_tc.cu), whose measurements chose them:
//   warps 0-3, 4-7  softmax of query tile 0 / 1, a thread per row, the whole S row in registers
//   warp  8         one lane issues every tcgen05.mma
//   warp  9         finds the items, loads Q (TMA), and K / V of a 16-bit cache: a TMA box per page
//   warps 10-11     16-bit cache: zero what a page holds past the end of its sequence (0 * NaN must not reach O)
//   warps 10-13     8-bit cache: bring e4m3 rows to fp16 (cp.async into a staging tile, exact conversion, 2^e of the row
//                   multiplied in), a tile ahead of the MMAs; with two warps for this, 2 x 2048 tokens over 6000-8192
//                   positions took 594 us, with four 553 (430 and 361 with heads of 64), and 330 (306) from a 16-bit cache:
//                   the conversion shares the issue slots with the softmax.  (14 and 15 only fill their warpgroup.)
// What differs: the query heads of a GQA group always share a tile (rows = (token, head), floor(128 / group) tokens of a
// tile, by a 4-D box on q), so that K and V are read once per group whatever the lengths; tiles are shared out over the
// CTAs as paged_attn.cuh describes, cut items leaving fp32 partial outputs; the lengths are read on the device, and the
// loading warp hands the items to the others through a ring of descriptors.
//
// m_t is a reference that lags behind the row's maximum, as in the dense kernel: the first tile (and any tile before
// which a row has seen no key at all) looks for its maximum, later ones only check their row sum: above 2^8 the
// reference moves before the next tile, above 2^15 the tile is redone against its maximum before P is stored.
// P is rounded to the operands' 16-bit type; S, O, sums and references are fp32.  bf16 queries over an 8-bit cache are
// brought to fp16 in shared memory, scaled by a power of two per row (see paged_decode.cu).
//
// Measured (32 query heads over 8 kv heads of 128, causal, bf16): 2 x 2048 tokens at the end of 6000 .. 8192 positions 330 us
// (1100 TFLOP/s; 380 when run back to back for long, under the power cap), 2 x 128 over 16384 84 us, 64 over 1024 19 us.
// As in the dense kernel the chain S -> softmax -> P -> O of the two query tiles bounds it.  Ranges in several rounds, so
// that all CTAs read the same few kv heads at a time, cost more in cut items than the L2 gave back up to 134 MB of keys and
// values (64 heads, 2 x 1024 over 8192: 466 for 435 us) and won 10 % at 268 MB: not kept.
#include <cmath>

#include "paged_attn.cuh"
#include "tc_prims.cuh"
#include "tma_host.cuh"

namespace pb {
namespace {

using namespace tc;

constexpr int BM = 128, BN = kTileKeys;
constexpr int kChunkBytes = 64 * 2 * 128;    // 64 elements x 128 rows
constexpr int kMmaWarp = 8, kLoadWarp = 9, kHelpWarp = 10;
constexpr int kItems = 4;                     // descriptors in flight
constexpr float kRescaleSum = 256.0f, kRedoSum = 32768.0f;
constexpr int kColS = 0, kColO = 256;

constexpr int kSmemQ = 0;
constexpr int kMaxPairs = 4;
constexpr int kBarQFull = 0, kBarQEmpty = 2, kBarSFull = 4, kBarPFull = 6, kBarOFull = 8, kBarQConv = 10, kBarKVFull = 12,
              kBarKVEmpty = kBarKVFull + kMaxPairs, kBarVLand = kBarKVEmpty + kMaxPairs, kBarItemFull = kBarVLand + kMaxPairs,
              kBarItemEmpty = kBarItemFull + kItems, kNumBars = kBarItemEmpty + kItems;

template <bool E8, int HD> struct Layout {
    static constexpr int kTileBytes = HD / 64 * kChunkBytes;           // of Q, K or V, fp16 or bf16
    static constexpr int kPairBytes = 2 * kTileBytes;                  // V_j, then K_j+1
    static constexpr int kPairLog = HD == 64 ? 2 : 1, kPairs = 1 << kPairLog;      // as many as there is room for
    // (heads of 64 with two: 4 x 16 tokens over 16384 positions 66 us, with four 59)
    static constexpr int kSmemKV = 2 * kTileBytes;
    static constexpr int kSmemO = kSmemKV + kPairs * kPairBytes;       // per softmax warp: staging of finished rows
    static constexpr int kConv = E8 ? 4 : 0;                           // warps that convert, a quarter of a tile's rows each
    static constexpr int kThreads = E8 ? 512 : 384;
    static constexpr int kAtLaunch = E8 ? 128 : 168;                   // registers per thread
    static constexpr int kORow = E8 ? 64 : 128;                        // bytes a row of the output staging holds
    static constexpr int kOStage = 32 * kORow;
    static constexpr int kRaw = kSmemO + 8 * kOStage;                  // 8-bit: a tile of e4m3 rows
    static constexpr int kScale = kRaw + (E8 ? 16 * 1024 : 0);         // 8-bit: 2^e of the rows, fp16 twice
    static constexpr int kItem = kScale + (E8 ? 512 : 0);
    static constexpr int kBits = kItem + kItems * 64;                  // pages that are there, of the last 2 * kPairs tiles
    static constexpr int kSums = kBits + 2 * kPairs * 4;
    static constexpr int kBars = kSums + (kThreads / 32 + 3) * 8 + 8;
    static constexpr int kMisc = kBars + kNumBars * 8;
    static constexpr int kLaunch = kMisc + 16 + 1024;
    // Registers per thread after setmaxnreg, which come to no more than what the CTA was launched with: 256 * 200 + 128 * 96
    // = 63488 of 384 * 168 = 64512; 8-bit: 256 * 200 + 256 * 56 = 65536 of 512 * 128.  (A softmax thread with 192 spills a
    // third of its row.)
    static constexpr int kRegsSoftmax = 200, kRegsOther = E8 ? 56 : 96;
    static_assert(256 * kRegsSoftmax + (kThreads - 256) * kRegsOther <= kThreads * kAtLaunch, "register split");
    static_assert(kLaunch <= 227 * 1024, "shared memory of a CTA");
    static_assert(kItem % 16 == 0 && kSums % 8 == 0 && kBars % 8 == 0, "alignment");
};

// A piece of work: a range of kv tiles for up to 256 query rows of one kv head.
struct Item {            // 64 bytes
    int b, hk;
    int row0, nq;         // first token row, tokens (at most 2 * tokens per tile)
    int pos;              // position of the first token
    int kv;               // positions of the sequence
    int kfin;             // positions that its computed tokens attend; what lies behind may be anything
    int kv0;              // first kv tile
    int n;                // kv tiles; 0: no more items
    int ntile[2];         // of them, tiles that query tile t visits
    int partial;          // results go to the workspace's slot
    int slot;
    int edge;             // the last tile's page goes on past kfin
    int pad[2];
};
static_assert(sizeof(Item) == 64, "");

__device__ __forceinline__ int keys_at(const PagedParams& p, int kv, int pos) { return p.causal ? max(0, min(kv, pos + 1)) : kv; }

__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 x;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(a));
    return x;
}

template <bool BF16, bool E8, int HD>
__global__ void __launch_bounds__(Layout<E8, HD>::kThreads, 1)
paged_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                const __grid_constant__ CUtensorMap map_v, const PagedParams p, const PagedWorkspace ws) {
    using L = Layout<E8, HD>;
    constexpr int kTileBytes = L::kTileBytes, kPairBytes = L::kPairBytes, kSmemKV = L::kSmemKV, kSmemO = L::kSmemO;
    constexpr bool kBfOps = BF16 && !E8;
    constexpr int kChunks = HD / 64;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
    auto bar = [&](int i) { return base + L::kBars + 8u * i; };
    auto slot_of = [](int g) { return g & (L::kPairs - 1); };               // of pair g, and the parity of its turn there
    auto turn_of = [](int g) { return uint32_t(g >> L::kPairLog) & 1u; };
    constexpr int kBitsMask = 2 * L::kPairs - 1;
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gen + L::kMisc);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(gen + L::kMisc + 4);
    // kv tiles the MMA warp has issued: waits that last a whole item (for its end, or for the next one) take their limit by it
    volatile uint32_t* progress = reinterpret_cast<volatile uint32_t*>(gen + L::kMisc + 8);
    Item* items = reinterpret_cast<Item*>(gen + L::kItem);
    volatile uint32_t* bits = reinterpret_cast<volatile uint32_t*>(gen + L::kBits);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int pt = BM / p.group;      // tokens of a query tile

    if (threadIdx.x == 0) {
        for (int i = 0; i < kNumBars; ++i) {
            int n = 1;                                                                   // a commit, a TMA, the loading warp
            if (i >= kBarKVFull && i < kBarKVFull + kMaxPairs) n = E8 ? 2 * L::kConv : 2;        // entries of a pair (by four warps)
            else if ((i >= kBarPFull && i < kBarPFull + 2) || i == kBarQConv || i == kBarQConv + 1) n = 4;   // softmax warps
            else if (i >= kBarItemEmpty) n = 1 + 8 + (E8 ? L::kConv : 2);                // MMA, softmax, converting or helping warps
            mbar_init(bar(i), n);
        }
        *abort_flag = 0;
        *progress = 0;
        mbar_fence_init();
    }
    // rows that no token fills (128 is not a multiple of the group) stay zero
    for (int i = threadIdx.x; i < 2 * kTileBytes / 16; i += L::kThreads) st_shared_v4(base + kSmemQ + i * 16, make_uint4(0, 0, 0, 0));
    fence_proxy_async_smem();
    if (warp == kMmaWarp) {
        tmem_alloc(base + L::kMisc, 512);
        tmem_relinquish();
    }
    if (warp == kLoadWarp && lane == 0) {
        tma_prefetch_desc(&map_q);
        tma_prefetch_desc(&map_k);
        tma_prefetch_desc(&map_v);
    }
    tc_fence_before_sync();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    int b0;
    int64_t base0;
    const PagedRange range = paged_range(p.B, reinterpret_cast<int64_t*>(gen + L::kSums),
                                         [&](int b) { return p.Hkv * head_tiles(p, paged_seq(p, b), pt); }, &b0, &base0);
    tc_fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    const int npg = p.npg;              // pages (or, of larger pages, pieces) in a tile
    // Item i of this CTA for the warps that wait for it, false at the end; its descriptor stays until they let it go.
    auto wait_item = [&](uint32_t i, int tag) -> bool {
        if (!__all_sync(0xffffffffu, mbar_wait_progress(bar(kBarItemFull + i % kItems), (i / kItems) & 1, abort_flag, tag, progress))) return false;
        if (items[i % kItems].n > 0) return true;
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(kBarItemEmpty + i % kItems));
        return false;
    };
    auto drop_item = [&](uint32_t i) {
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(kBarItemEmpty + i % kItems));
    };
    auto get_item = [&](uint32_t i, Item* it, int tag) -> bool {
        if (!wait_item(i, tag)) return false;
        *it = items[i % kItems];
        drop_item(i);
        return true;
    };

    if (warp >= kMmaWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::kRegsOther));
        if (warp == kLoadWarp) {
            // ------------------------------ items, Q, and K / V of a 16-bit cache ------------------------------
            PagedJoin join{};
            join.first_slot = -1;
            PagedSeq sq{};
            int b = b0, hk = 0, qi = 0, tile = 0, nt = 0, nitems = 0;
            int64_t at = range.begin;        // the next tile's place
            auto enter = [&]() {             // the first sequence from b on that has tiles
                nitems = 0;
                for (; b < p.B; ++b) {
                    sq = paged_seq(p, b);
                    nitems = (sq.nq + 2 * pt - 1) / (2 * pt);
                    if (nitems > 0) break;
                }
                nt = nitems > 0 ? item_tiles(p, sq, 0, pt) : 0;
            };
            if (at < range.end) {
                enter();
                const int64_t per = head_tiles(p, sq, pt);
                int64_t in = at - base0;
                hk = int(in / per);
                in -= int64_t(hk) * per;
                while (in >= nt) {
                    in -= nt;
                    nt = item_tiles(p, sq, ++qi, pt);
                }
                tile = int(in);
            }
            int r = 0;               // entries so far: K0 | V0 K1 | V1 K2 | ...  entry r belongs to pair (r + 1) / 2
            uint32_t qcnt[2] = {0, 0};
            bool ok = true;
            // lane i: page of box i of kv tile `t`, -1 where nothing is to be read
            auto page_of = [&](const Item& it, int t) -> int {
                if (lane >= npg || t * BN + (lane << p.box_shift) >= it.kfin) return -1;
                const int entry = p.tpp > 1 ? t / p.tpp : t * npg + lane;
                const int pg = __ldg(p.table + int64_t(it.b) * p.table_stride + entry);
                return uint32_t(pg) < uint32_t(p.pages) ? pg : -1;
            };
            // entry: K (which = 0) or V of kv tile t, whose pages are pg
            auto load_entry = [&](const Item& it, int which, int t, int pg, bool edge) -> bool {
                const int g = (r + 1) >> 1, slot = slot_of(g);
                if ((r & 1) || r == 0) {      // the pair's first entry: its slot must have been released
                    if (!__all_sync(0xffffffffu, mbar_wait(bar(kBarKVEmpty + slot), turn_of(g) ^ 1u, abort_flag, 2))) return false;
                    if (r == 0 && lane == 0) mbar_arrive(bar(kBarKVFull + slot));
                }
                const uint32_t full = bar(edge ? kBarVLand + slot : kBarKVFull + slot);
                if (!which) {
                    const uint32_t there = __ballot_sync(0xffffffffu, pg >= 0);
                    if (lane == 0) bits[g & kBitsMask] = there;
                }
                if (lane == 0) mbar_arrive_expect_tx(full, kChunks * kChunkBytes);
                __syncwarp();
                if (lane < npg) {
                    const uint32_t dst = base + kSmemKV + slot * kPairBytes + (which ? 0 : kTileBytes) + (lane << p.box_shift) * 128;
                    const int page = pg >= 0 ? pg : p.pages, row = p.tpp > 1 ? (t % p.tpp) * BN : 0;   // (outside: zeros)
#pragma unroll
                    for (int c = 0; c < kChunks; ++c) tma_load_4d(dst + c * kChunkBytes, which ? &map_v : &map_k, full, 64 * c, row, it.hk, page);
                }
                ++r;
                return true;
            };
            uint32_t seq = 0;
            auto put = [&](const Item& it) -> bool {
                if (!__all_sync(0xffffffffu, mbar_wait_progress(bar(kBarItemEmpty + seq % kItems), ((seq / kItems) & 1) ^ 1u, abort_flag, 12, progress)))
                    return false;
                if (lane == 0) {
                    items[seq % kItems] = it;
                    mbar_arrive(bar(kBarItemFull + seq % kItems));
                }
                __syncwarp();
                ++seq;
                return true;
            };
            while (ok && at < range.end) {
                // ---- describe the item ----
                Item it{};
                it.b = b;
                it.hk = hk;
                const int tok0 = qi * 2 * pt;
                it.row0 = sq.row0 + tok0;
                it.nq = min(2 * pt, sq.nq - tok0);
                it.pos = sq.pos0 + tok0;
                it.kv = sq.kv;
                it.kfin = paged_keys(p, sq, sq.nq - 1);
                it.kv0 = tile;
                it.n = int(min(int64_t(nt - tile), range.end - at));
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const int live = min(pt, it.nq - t * pt);
                    it.ntile[t] = live > 0 ? max(0, min(it.n, tiles_for(keys_at(p, sq.kv, it.pos + t * pt + live - 1)) - tile)) : 0;
                }
                it.partial = it.n < nt;
                // the item the range begins with leaves its part in slot 2c, a later one that goes on in 2c + 1
                it.slot = 2 * int(blockIdx.x) + (at > range.begin ? 1 : 0);
                const int end_key = (tile + it.n) * BN;
                it.edge = !E8 && end_key > it.kfin && it.kfin > end_key - BN && (it.kfin & ((1 << p.box_shift) - 1)) != 0;
                if (it.partial && tile == 0) {
                    join.first_slot = it.slot;
                    join.last_cta = range.owner(at + nt - 1);
                    join.row0 = it.row0;
                    join.nq = it.nq;
                    join.hk = hk;
                }
                ok = put(it);
                // ---- its loads ----
                if (ok) {
                    int pg = -1, pg_next = -1;
                    if constexpr (!E8) {
                        pg = page_of(it, it.kv0);
                        ok = load_entry(it, 0, it.kv0, pg, false);
                    }
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        if (ok && it.ntile[t] > 0) {
                            ok = __all_sync(0xffffffffu, mbar_wait_progress(bar(kBarQEmpty + t), (qcnt[t] & 1u) ^ 1u, abort_flag, 0 + t, progress));
                            if (!ok) break;
                            ++qcnt[t];
                            if (lane == 0) {
                                mbar_arrive_expect_tx(bar(kBarQFull + t), uint32_t(kChunks * pt * p.group * 128));
#pragma unroll
                                for (int c = 0; c < kChunks; ++c)
                                    tma_load_4d(base + kSmemQ + t * kTileBytes + c * kChunkBytes, &map_q, bar(kBarQFull + t), 64 * c, 0, it.hk,
                                                it.row0 + t * pt);
                            }
                        }
                    }
                    if constexpr (!E8) {
                        for (int j = 0; ok && j < it.n; ++j) {
                            if (j + 1 < it.n) pg_next = page_of(it, it.kv0 + j + 1);
                            const bool edge = it.edge && j + 1 == it.n;
                            ok = load_entry(it, 1, it.kv0 + j, pg, edge);
                            if (ok && j + 1 < it.n) ok = load_entry(it, 0, it.kv0 + j + 1, pg_next, false);
                            pg = pg_next;
                        }
                    }
                }
                // ---- on to the next one ----
                at += it.n;
                tile = 0;
                if (++qi == nitems) {
                    qi = 0;
                    if (++hk == p.Hkv) {
                        hk = 0;
                        ++b;
                        if (at < range.end) enter();
                    }
                }
                if (at < range.end) nt = item_tiles(p, sq, qi, pt);
            }
            if (ok) {
                if (!E8 && r > 0 && lane == 0) mbar_arrive(bar(kBarKVFull + slot_of(r >> 1)));   // the last pair has no K
                Item end{};
                put(end);
            }
            if (lane == 0) ws.join[blockIdx.x] = join;
        } else if (warp == kMmaWarp) {
            // ------------------------------ MMA issuer ------------------------------
            constexpr uint32_t idesc_qk = instr_desc_f16(kBfOps ? 1 : 0, BM, BN, false, false);
            constexpr uint32_t idesc_pv = instr_desc_f16(kBfOps ? 1 : 0, BM, HD, false, true);
            auto issue_qk = [&](int t, int pair) {
                const uint32_t qa = base + kSmemQ + t * kTileBytes;
                const uint32_t ka = base + kSmemKV + slot_of(pair) * kPairBytes + kTileBytes;
#pragma unroll
                for (int c = 0; c < kChunks; ++c)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t off = c * kChunkBytes + i * 32;
                        mma_ss(tmem + kColS + t * 128, smem_desc_sw128(qa + off, 16, 1024), smem_desc_sw128(ka + off, 16, 1024), idesc_qk,
                               (c | i) ? 1u : 0u);
                    }
            };
            auto issue_pv = [&](int t, int pair, bool acc) {
                const uint32_t va = base + kSmemKV + slot_of(pair) * kPairBytes;
#pragma unroll
                for (int ks = 0; ks < BN / 16; ++ks)
                    mma_ts(tmem + kColO + t * 128, tmem + kColS + t * 128 + ks * 8, smem_desc_sw128(va + ks * 16 * 128, kChunkBytes, 1024),
                           idesc_pv, (acc || ks) ? 1u : 0u);
            };
            if (lane == 0) {
                bool ok = true, have = false;
                int G = 0;                    // pair that holds the item's K0 (and the previous item's last V)
                uint32_t qcnt[2] = {0, 0}, pcnt[2] = {0, 0};
                for (uint32_t seq = 0; ok; ++seq) {
                    ok = mbar_wait(bar(kBarItemFull + seq % kItems), (seq / kItems) & 1, abort_flag, 13);
                    if (!ok) break;
                    const int n = items[seq % kItems].n;
                    const int nt[2] = {items[seq % kItems].ntile[0], items[seq % kItems].ntile[1]};
                    mbar_arrive(bar(kBarItemEmpty + seq % kItems));
                    if (n == 0) break;
                    if (!have) ok = mbar_wait(bar(kBarKVFull + slot_of(G)), turn_of(G), abort_flag, 3);
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        if (ok && nt[t] > 0) {
                            ok = mbar_wait(bar((E8 && BF16 ? kBarQConv : kBarQFull) + t), qcnt[t] & 1u, abort_flag, 4 + t);
                            if (ok) {
                                tc_fence_after_sync();
                                issue_qk(t, G);
                                tc_commit(bar(kBarSFull + t));
                                if (nt[t] == 1) tc_commit(bar(kBarQEmpty + t));
                            }
                        }
                    }
                    if (!ok) break;
                    tc_commit(bar(kBarKVEmpty + slot_of(G)));
                    for (int j = 0; ok && j < n; ++j) {
                        const int g = G + j + 1;          // (V_j, K_j+1)
                        *progress = uint32_t(g);
                        ok = mbar_wait(bar(kBarKVFull + slot_of(g)), turn_of(g), abort_flag, 3);
                        if (!ok) break;
#pragma unroll
                        for (int t = 0; t < 2; ++t) {
                            if (ok && j < nt[t]) {
                                ok = mbar_wait(bar(kBarPFull + t), pcnt[t] & 1u, abort_flag, 6 + t);
                                if (!ok) break;
                                ++pcnt[t];
                                tc_fence_after_sync();
                                issue_pv(t, g, j > 0);
                                if (j + 1 < nt[t]) {
                                    issue_qk(t, g);
                                    tc_commit(bar(kBarSFull + t));
                                    if (j + 2 == nt[t]) tc_commit(bar(kBarQEmpty + t));
                                } else {
                                    tc_commit(bar(kBarOFull + t));
                                }
                            }
                        }
                        if (!ok) break;
                        if (j + 1 < n) tc_commit(bar(kBarKVEmpty + slot_of(g)));   // the last one also holds the next item's K0
                    }
#pragma unroll
                    for (int t = 0; t < 2; ++t)
                        if (nt[t] > 0) ++qcnt[t];
                    G += n;
                    have = true;
                }
            }
            __syncwarp();
        } else if constexpr (!E8) {
            // ------------------------------ zeros past the end of a sequence (V) ------------------------------
            Item it;
            int G = 0;
            uint32_t turns = 0;                 // bit per slot: parity of its next edge
            for (uint32_t seq = 0; get_item(seq, &it, 14); ++seq) {
                G += it.n;                              // the last tile's V is in pair G (after this)
                if (warp != kHelpWarp || !it.edge) continue;
                const int slot = slot_of(G);
                if (!__all_sync(0xffffffffu, mbar_wait_progress(bar(kBarVLand + slot), (turns >> slot) & 1u, abort_flag, 15, progress))) break;
                turns ^= 1u << slot;
                const int r0 = it.kfin - (it.kv0 + it.n - 1) * BN, r1 = (r0 + (1 << p.box_shift) - 1) >> p.box_shift << p.box_shift;   // the page's rest
                for (int i = lane; i < (r1 - r0) * kChunks * 8; i += 32) {
                    const int row = r0 + i / (kChunks * 8), u = i % (kChunks * 8);
                    st_shared_v4(base + kSmemKV + slot * kPairBytes + (u >> 3) * kChunkBytes + row * 128 + (u & 7) * 16, make_uint4(0, 0, 0, 0));
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(kBarKVFull + slot));
            }
        } else if (warp < kHelpWarp + L::kConv) {
            // ------------------------------ e4m3 rows to fp16 ------------------------------
            // Each of the four warps brings 32 of a tile's rows; HD / 16 lanes take a row, 16 bytes each.  The rows of the
            // next entry are on their way into the staging tile while this one is converted, unit by unit in the same place.
            constexpr int kPer = HD / 16, kUnits = kPer;              // lanes of a row, units of a lane (32 / kPer rows each)
            const int w = warp - kHelpWarp;
            const uint32_t raw = base + L::kRaw + w * 4096, scales = base + L::kScale + w * 128;
            int r = 0;
            // Entry x of an item: K_0, then V_j (odd x), K_j+1 (even x): kv tile x / 2.
            struct Part { int b, hk, kv0, n, kfin; };      // what this role needs of an item
            auto get_part = [&](uint32_t i, Part* it) -> bool {
                it->n = 0;
                if (!wait_item(i, 14)) return false;
                const Item& src = items[i % kItems];
                *it = Part{src.b, src.hk, src.kv0, src.n, src.kfin};
                drop_item(i);
                return true;
            };
            // lane l looks after the warp's row l: its page, ...
            auto page_for = [&](const Part& it, int x) -> int {
                const int t = it.kv0 + (x >> 1), key = w * 32 + lane;
                if (t * BN + key >= it.kfin) return -1;
                const int pg = __ldg(p.table + int64_t(it.b) * p.table_stride + (p.tpp > 1 ? t / p.tpp : t * npg + (key >> p.box_shift)));
                return uint32_t(pg) < uint32_t(p.pages) ? pg : -1;
            };
            auto row_in_page = [&](const Part& it, int x) -> int {
                const int t = it.kv0 + (x >> 1), key = w * 32 + lane;
                return (p.tpp > 1 ? (t % p.tpp) * BN : 0) + (key & ((1 << p.box_shift) - 1));
            };
            // ... its exponent byte (127 where there is no row), ...
            auto exps_for = [&](const Part& it, int x, int pg) -> uint32_t {
                if (pg < 0) return 127u;
                const bool v = x & 1;      // (selected one by one: a pointer into the parameters would copy them to local memory)
                return __ldg((v ? p.ev : p.ek) + int64_t(pg) * (v ? p.evs[0] : p.eks[0]) + int64_t(it.hk) * (v ? p.evs[1] : p.eks[1]) +
                             int64_t(row_in_page(it, x)) * (v ? p.evs[2] : p.eks[2]));
            };
            // ... and where it lies; the low bit says that there is such a row
            auto rows_for = [&](const Part& it, int x, int pg) -> uint64_t {
                const bool v = x & 1;
                const char* src = v ? p.cv : p.ck;
                if (pg < 0) return reinterpret_cast<uint64_t>(src);
                return reinterpret_cast<uint64_t>(src + int64_t(pg) * (v ? p.cvs[0] : p.cks[0]) + int64_t(it.hk) * (v ? p.cvs[1] : p.cks[1]) +
                                                  int64_t(row_in_page(it, x)) * (v ? p.cvs[2] : p.cks[2])) | 1u;
            };
            const int my_row = lane / kPer, my_c = lane % kPer;       // of a unit's 32 / kPer rows
            // asks for unit u (rows u * 32 / kPer ..): `rows` as rows_for gave it
            auto fetch = [&](uint64_t rows, int u) {
                const uint64_t at = __shfl_sync(0xffffffffu, rows, u * (32 / kPer) + my_row);
                const bool live = at & 1u;
                const uint64_t src = (at & ~uint64_t(15)) + (live ? my_c * 16 : 0);
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(raw + u * 512 + lane * 16), "l"(src), "r"(live ? 16 : 0)
                             : "memory");
            };
            Part it, nx;
            bool more = get_part(0, &it), ok = true;
            uint32_t seq = 0;
            int pg = -1;
            uint32_t ex = 127u;
            if (more) {
                pg = page_for(it, 0);
                ex = exps_for(it, 0, pg);
                const uint64_t rows = rows_for(it, 0, pg);
                for (int u = 0; u < kUnits; ++u) fetch(rows, u);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            while (ok && more) {
                nx = it;
                bool next_more = false, have_next = false;
                for (int x = 0; ok && x < 2 * it.n; ++x) {
                    // what comes after this entry
                    int nxx = x + 1;
                    if (nxx == 2 * it.n) {
                        next_more = get_part(++seq, &nx);
                        have_next = true;
                        nxx = 0;
                    }
                    const bool go = !have_next || next_more;
                    int pg2 = -1;
                    uint32_t ex2 = 127u;
                    uint64_t rows2 = 0;
                    if (go) {
                        pg2 = (nxx & 1) ? pg : page_for(nx, nxx);      // V_j lies where K_j does
                        rows2 = rows_for(nx, nxx, pg2);
                        ex2 = exps_for(nx, nxx, pg2);
                    }
                    const int g = (r + 1) >> 1, slot = slot_of(g);
                    if ((r & 1) || r == 0) {
                        ok = __all_sync(0xffffffffu, mbar_wait(bar(kBarKVEmpty + slot), turn_of(g) ^ 1u, abort_flag, 2));
                        if (!ok) break;
                        if (r == 0 && lane == 0) mbar_arrive(bar(kBarKVFull + slot));
                    }
                    if (!(x & 1)) {
                        // bit i: page i of the tile is there, from the warp that has its first row
                        const int key = lane << p.box_shift, mine = __shfl_sync(0xffffffffu, pg, key & 31);
                        const uint32_t there = __ballot_sync(0xffffffffu, lane < npg && key >> 5 == w && mine >= 0);
                        if (lane == 0) reinterpret_cast<volatile uint8_t*>(gen + L::kBits)[4 * (g & kBitsMask) + w] = uint8_t(there >> ((w * 32) >> p.box_shift));
                    }
                    // 2^e of this lane's row, fp16 twice
                    {
                        const int e = max(kExpLo, min(kExpHi, int(ex) - 127));
                        const uint32_t f = e >= -14 ? uint32_t(e + 15) << 10 : 0x200u;
                        asm volatile("st.shared.b32 [%0], %1;" ::"r"(scales + lane * 4), "r"(f | (f << 16)) : "memory");
                    }
                    asm volatile("cp.async.wait_group 0;" ::: "memory");
                    __syncwarp();
                    const uint32_t dst = base + kSmemKV + slot * kPairBytes + ((x & 1) ? 0 : kTileBytes);
                    // two units at a time: their loads side by side, then their conversions
#pragma unroll 1
                    for (int u2 = 0; u2 < kUnits; u2 += 2) {
                        uint4 v[2];
                        uint32_t sc[2];
#pragma unroll
                        for (int y = 0; y < 2; ++y) {
                            v[y] = lds128(raw + (u2 + y) * 512 + lane * 16);
                            asm volatile("ld.shared.b32 %0, [%1];" : "=r"(sc[y]) : "r"(scales + ((u2 + y) * (32 / kPer) + my_row) * 4));
                        }
#pragma unroll
                        for (int y = 0; y < 2; ++y) {
                            const __half2 s2 = *reinterpret_cast<const __half2*>(&sc[y]);
                            const uint32_t in[4] = {v[y].x, v[y].y, v[y].z, v[y].w};
                            uint32_t o[8];
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                uint32_t lo, hi;
                                e4m3x4_to_f16x4(in[i], &lo, &hi);
                                const __half2 a = __hmul2(*reinterpret_cast<__half2*>(&lo), s2), bb = __hmul2(*reinterpret_cast<__half2*>(&hi), s2);
                                o[2 * i] = *reinterpret_cast<const uint32_t*>(&a);
                                o[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&bb);
                            }
                            // 16 elements are two 16-byte units of a 64-element slab; odd slabs write theirs in the other
                            // order, which keeps the eight lanes of a row on different banks
                            const int R = w * 32 + (u2 + y) * (32 / kPer) + my_row, odd = (my_c >> 2) & 1, un = (my_c & 3) * 2;
                            const uint32_t rowa = dst + (my_c >> 2) * kChunkBytes + R * 128;
                            const uint4 A = make_uint4(o[0], o[1], o[2], o[3]), B = make_uint4(o[4], o[5], o[6], o[7]);
                            st_shared_v4(rowa + uint32_t(((un + odd) ^ (R & 7)) << 4), odd ? B : A);
                            st_shared_v4(rowa + uint32_t(((un + 1 - odd) ^ (R & 7)) << 4), odd ? A : B);
                        }
                        if (go) {      // (what they will overwrite has been read)
#pragma unroll
                            for (int y = 0; y < 2; ++y) fetch(rows2, u2 + y);
                        }
                    }
                    asm volatile("cp.async.commit_group;" ::: "memory");
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar(kBarKVFull + slot));
                    ++r;
                    pg = pg2;
                    ex = ex2;
                }
                it = nx;
                more = next_more;
            }
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            if (ok && r > 0 && lane == 0) mbar_arrive(bar(kBarKVFull + slot_of(r >> 1)));   // the last pair has no K
        }
    } else {
        // ------------------------------ softmax and results ------------------------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(L::kRegsSoftmax));
        const int t = warp >> 2, wq = warp & 3;
        const uint32_t lane_base = uint32_t(wq * 32) << 16;
        const uint32_t s_addr = tmem + lane_base + kColS + t * 128, o_addr = tmem + lane_base + kColO + t * 128;
        const uint32_t stage = base + kSmemO + warp * L::kOStage;
        const int row = wq * 32 + lane;                   // of the tile
        const uint32_t all_pages = (1u << npg) - 1u;
        bool ok = true;
        uint32_t scnt = 0, ocnt = 0, G = 0;
        for (uint32_t seq = 0; ok && wait_item(seq, 14); ++seq, drop_item(seq - 1)) {
            const Item& it = items[seq % kItems];
            const int nt = it.ntile[t];
            uint32_t g = G;                                  // pair of K_j
            G += uint32_t(it.n);
            if (nt == 0) {
                // a cut item's range that lies beyond this query tile's keys
                if (it.partial && row < min(pt, it.nq - t * pt) * p.group)
                    ws.ml[size_t(it.slot) * 256 + t * pt * p.group + row] = make_float2(-INFINITY, 0.f);
                continue;
            }
            int col0 = it.kv0 * BN;
            const int my_keys = keys_at(p, it.kv, it.pos + t * pt + row / p.group);
            const int min_keys = keys_at(p, it.kv, it.pos + t * pt);      // of the tile's first token
            float c2 = p.scale_log2;
            if constexpr (E8 && BF16) {
                // this thread's row of the new Q tile, brought to fp16 with its largest magnitude in [1, 2)
                ok = __all_sync(0xffffffffu, mbar_wait(bar(kBarQFull + t), ocnt & 1u, abort_flag, 18 + t));
                if (!ok) break;
                const uint32_t qrow = base + kSmemQ + t * kTileBytes + row * 128;
                float amax = 0.f;
#pragma unroll
                for (int u = 0; u < HD / 8; ++u) {
                    const uint4 v = lds128(qrow + (u >> 3) * kChunkBytes + uint32_t(((u & 7) ^ (row & 7)) << 4));
                    const uint32_t vv[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float2 f = pair16_to_f32<true>(vv[i]);
                        amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
                    }
                }
                const int ex = max(-120, min(120, int(__float_as_uint(amax) >> 23) - 127));
                const float f = pow2f(-ex);
                c2 = fmaxf(c2 * pow2f(ex), kLeastC2);
#pragma unroll
                for (int u = 0; u < HD / 8; ++u) {
                    const uint32_t a = qrow + (u >> 3) * kChunkBytes + uint32_t(((u & 7) ^ (row & 7)) << 4);
                    const uint4 v = lds128(a);
                    const uint32_t vv[4] = {v.x, v.y, v.z, v.w};
                    uint32_t o[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float2 x = pair16_to_f32<true>(vv[i]);
                        o[i] = pack16<false>(x.x * f, x.y * f);
                    }
                    st_shared_v4(a, make_uint4(o[0], o[1], o[2], o[3]));
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(kBarQConv + t));
            }
            const float inv_c2 = 1.0f / c2;
            float m = -INFINITY, m_next = -INFINITY, l = 0.f;     // m: reference in units of S, -inf: no key seen yet
            bool move_ref = false, unseen = true;
            for (int j = 0; j < nt; ++j, ++g, col0 += BN) {
                ok = __all_sync(0xffffffffu, mbar_wait(bar(kBarSFull + t), scnt & 1u, abort_flag, 10 + t));
                if (!ok) break;
                ++scnt;
                tc_fence_after_sync();
                // (O_t is at rest: PV_t(j-1) has completed, PV_t(j) waits for this tile's P)
                auto rescale_o = [&](float alpha) {
#pragma unroll 1
                    for (int c = 0; c < HD / 16; ++c) {
                        uint32_t o[16];
                        tmem_ld16(o_addr + 16 * c, o);
                        tmem_wait_ld();
                        tmem_ld_fence16(o);
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                        tmem_st16(o_addr + 16 * c, o);
                    }
                    tmem_wait_st();      // (a second rescaling in the same tile loads these columns again)
                };
                if (j > 0 && move_ref) {
                    const float alpha = m_next == m ? 1.f : ex2_approx((m - m_next) * c2);
                    l *= alpha;
                    rescale_o(alpha);
                    m = m_next;
                }
                uint32_t there = bits[g & kBitsMask];
                if constexpr (E8) {                              // (a byte per converting warp)
                    const uint32_t of = there;
                    there = 0u;
#pragma unroll
                    for (int w = 0; w < L::kConv; ++w) there |= ((of >> (8 * w)) & 0xffu) << ((w * 32) >> p.box_shift);
                }
                uint32_t pk[BN / 2];
                float l_tile;
                bool bad = false;
#pragma unroll 1
                for (int attempt = 0;; ++attempt) {
                    uint32_t s[BN];
#pragma unroll
                    for (int c = 0; c < 4; ++c) tmem_ld32(s_addr + 32 * c, reinterpret_cast<uint32_t(&)[32]>(s[32 * c]));
                    tmem_wait_ld();
#pragma unroll
                    for (int c = 0; c < 4; ++c) tmem_ld_fence32(reinterpret_cast<uint32_t(&)[32]>(s[32 * c]));
                    if (col0 + BN > min_keys) {
                        const int limit = my_keys - 1 - col0;
#pragma unroll
                        for (int i = 0; i < BN; ++i)
                            if (i > limit) s[i] = 0xff800000u;
                    }
                    if (there != all_pages) {
#pragma unroll
                        for (int i = 0; i < BN; ++i)
                            if (!((there >> (i >> p.box_shift)) & 1u)) s[i] = 0xff800000u;
                    }
                    const bool look = unseen || attempt == 1;        // (the same for the whole warp)
                    if (look) {
                        float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
                        for (int i = 0; i < BN; i += 4) {
                            mx0 = fmax3(mx0, __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
                            mx1 = fmax3(mx1, __uint_as_float(s[i + 2]), __uint_as_float(s[i + 3]));
                        }
                        const float mx = fmaxf(mx0, mx1);
                        const float m_new = (m == -INFINITY || bad) ? mx : m;
                        if (j > 0) {
                            const float alpha = (m == -INFINITY || m_new == m) ? 1.f : ex2_approx((m - m_new) * c2);   // (nothing to scale yet: O is 0)
                            l *= alpha;
                            rescale_o(alpha);
                        }
                        m = m_new;
                    }
                    const float ref = m == -INFINITY ? 0.f : m;       // no key yet: every P is 0
                    const float neg_m = -ref * c2;
                    const float2 c22 = make_float2(c2, c2), nm2 = make_float2(neg_m, neg_m);
                    float2 ls0 = make_float2(0.f, 0.f), ls1 = make_float2(0.f, 0.f);
#pragma unroll
                    for (int i = 0; i < BN / 2; ++i) {
                        const float2 x = ffma2(make_float2(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), c22, nm2);
                        const float p0 = ex2_approx(x.x), p1 = ex2_approx(x.y);
                        if (i & 1) ls1 = fadd2(ls1, make_float2(p0, p1));
                        else ls0 = fadd2(ls0, make_float2(p0, p1));
                        pk[i] = pack16<kBfOps>(p0, p1);
                    }
                    l_tile = (ls0.x + ls0.y) + (ls1.x + ls1.y);
                    if (j == 0 || attempt == 1) break;
                    bad = !(l_tile <= kRedoSum);
                    if (!__any_sync(0xffffffffu, bad)) break;
                }
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_st16(s_addr + 16 * c, reinterpret_cast<uint32_t(&)[16]>(pk[16 * c]));
                l += l_tile;
                tmem_wait_st();
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(kBarPFull + t));
                m_next = l_tile > kRescaleSum ? m + lg2_approx(l_tile) * inv_c2 : m;
                move_ref = __any_sync(0xffffffffu, m_next != m);
                unseen = __any_sync(0xffffffffu, m == -INFINITY);
            }
            if (!ok) break;
            ok = __all_sync(0xffffffffu, mbar_wait(bar(kBarOFull + t), ocnt & 1u, abort_flag, 16 + t));
            if (!ok) break;
            ++ocnt;
            tc_fence_after_sync();
            // (scores of nothing but NaN leave no maximum either, but a sum that is NaN: the row's results are)
            const bool none = m == -INFINITY && l == l;
            const float m2 = m == -INFINITY ? 0.f : m * c2;
            const int live = min(pt, it.nq - t * pt) * p.group;            // rows of this tile that are tokens
            const int crow = t * pt * p.group;                             // its first row in the item
            // Rows leave through the warp's staging buffer, so that a store writes whole pieces of kORow bytes of
            // neighbouring rows: 16-byte unit u of row r sits at u ^ (r mod units).
            constexpr int kUnitsRow = L::kORow / 16;        // 8 or 4 lanes take a row
            constexpr int kRowsAt = 32 / kUnitsRow;
            const int u0 = lane % kUnitsRow, rr0 = lane / kUnitsRow;
            if (it.partial) {
                constexpr int kCols = L::kORow / 4;
#pragma unroll 1
                for (int c = 0; c < HD / kCols; ++c) {
                    uint32_t o[kCols];
                    if constexpr (kCols == 32) {
                        tmem_ld32(o_addr + kCols * c, reinterpret_cast<uint32_t(&)[32]>(o));
                        tmem_wait_ld();
                        tmem_ld_fence32(reinterpret_cast<uint32_t(&)[32]>(o));
                    } else {
                        tmem_ld16(o_addr + kCols * c, reinterpret_cast<uint32_t(&)[16]>(o));
                        tmem_wait_ld();
                        tmem_ld_fence16(reinterpret_cast<uint32_t(&)[16]>(o));
                    }
                    __syncwarp();
#pragma unroll
                    for (int u = 0; u < kUnitsRow; ++u)
                        st_shared_v4(stage + lane * L::kORow + ((u ^ (lane % kUnitsRow)) << 4), make_uint4(o[4 * u], o[4 * u + 1], o[4 * u + 2], o[4 * u + 3]));
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 32 / kRowsAt; ++i) {
                        const int rr = i * kRowsAt + rr0, tr = wq * 32 + rr;
                        const uint4 v = lds128(stage + rr * L::kORow + ((u0 ^ (rr % kUnitsRow)) << 4));
                        if (tr < live)
                            *reinterpret_cast<uint4*>(ws.o + (size_t(it.slot) * 256 + crow + tr) * HD + kCols * c + 4 * u0) = v;
                    }
                }
                if (row < live) ws.ml[size_t(it.slot) * 256 + crow + row] = make_float2(none ? -INFINITY : m2, l);
            } else {
                constexpr int kCols = L::kORow / 2;
                const float inv = none ? 0.f : 1.0f / l;
#pragma unroll 1
                for (int c = 0; c < HD / kCols; ++c) {
                    __syncwarp();
#pragma unroll
                    for (int h = 0; h < kCols / 32; ++h) {
                        uint32_t o[32];
                        tmem_ld32(o_addr + kCols * c + 32 * h, o);
                        tmem_wait_ld();
                        tmem_ld_fence32(o);
#pragma unroll
                        for (int v = 0; v < 4; ++v) {
                            uint4 w;
                            w.x = pack16<BF16>(__uint_as_float(o[8 * v + 0]) * inv, __uint_as_float(o[8 * v + 1]) * inv);
                            w.y = pack16<BF16>(__uint_as_float(o[8 * v + 2]) * inv, __uint_as_float(o[8 * v + 3]) * inv);
                            w.z = pack16<BF16>(__uint_as_float(o[8 * v + 4]) * inv, __uint_as_float(o[8 * v + 5]) * inv);
                            w.w = pack16<BF16>(__uint_as_float(o[8 * v + 6]) * inv, __uint_as_float(o[8 * v + 7]) * inv);
                            st_shared_v4(stage + lane * L::kORow + (((4 * h + v) ^ (lane % kUnitsRow)) << 4), w);
                        }
                    }
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 32 / kRowsAt; ++i) {
                        const int rr = i * kRowsAt + rr0, tr = wq * 32 + rr;
                        const uint4 v = lds128(stage + rr * L::kORow + ((u0 ^ (rr % kUnitsRow)) << 4));
                        if (tr < live) {
                            const int tok = it.row0 + t * pt + tr / p.group, h = it.hk * p.group + tr % p.group;
                            uint16_t* out = static_cast<uint16_t*>(p.out) + int64_t(tok) * p.os[0] + int64_t(h) * p.os[1] + kCols * c + 8 * u0;
                            *reinterpret_cast<uint4*>(out) = v;
                        }
                    }
                }
                if (p.lse && row < live) {
                    const int tok = it.row0 + t * pt + row / p.group, h = it.hk * p.group + row % p.group;
                    p.lse[int64_t(tok) * p.Hq + h] = none ? -INFINITY : m2 * 0.6931471805599453f + logf(l);
                }
            }
            // (the next item's S_t, and with it the next write to O_t, waits for these warps' next P)
            tc_fence_before_sync();
        }
    }

    // ------------------------------ common exit ------------------------------
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    if (warp == kMmaWarp) {
        if (*abort_flag) drain_after_abort();
        tmem_dealloc(tmem, 512);
    }
    if (threadIdx.x == 0 && *abort_flag) {
        *p.status = *abort_flag;
        __threadfence_system();
    }
}

template <bool BF16, bool E8, int HD>
int launch(int gpu, int G, cudaStream_t s, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const PagedParams& p,
           const PagedWorkspace& ws) {
    constexpr int bytes = Layout<E8, HD>::kLaunch;
    PB_CUDA((paged_allow_smem<paged_tc_kernel<BF16, E8, HD>>(gpu, bytes, Layout<E8, HD>::kAtLaunch)));
    PB_CUDA(paged_launch(paged_tc_kernel<BF16, E8, HD>, dim3(unsigned(G)), Layout<E8, HD>::kThreads, bytes, s, mq, mk, mv, p, ws));
    return PARAS_OK;
}

}  // namespace

int paged_tc_rows() { return 256; }

bool paged_tc_supported(const Gpu* g, const paras_paged_attn_args& a) {
    if (g->cc_major != 10 || a.dtype == PARAS_F32 || !paged_tma_ok(a.cache) || !paged_q_tma_ok(a)) return false;
    if (a.Hq / a.cache.Hkv > BM || !paged_scale_ok(a) || g->smem_optin < 227 * 1024) return false;
    // finished rows leave in 16-byte pieces
    return (reinterpret_cast<uintptr_t>(a.out) & 15u) == 0 && a.o_strides[0] % 8 == 0 && a.o_strides[1] % 8 == 0;
}

int paged_tc_launch(Gpu* g, const paras_paged_attn_args& a, const PagedParams& p, const PagedWorkspace& ws, int G, cudaStream_t s) {
    int st = check_status_word(g);
    if (st != PARAS_OK) return st;
    CUtensorMap mq, mk, mv;
    if ((st = paged_q_map(&mq, a, BM / p.group)) != PARAS_OK) return st;
    if ((st = paged_cache_map(&mk, a.cache, 0, false)) != PARAS_OK) return st;
    if ((st = paged_cache_map(&mv, a.cache, 1, false)) != PARAS_OK) return st;
    const bool bf = a.dtype == PARAS_BF16, e8 = a.cache.cache_dtype == PARAS_E4M3;
#define PB_GO(B, E, H) launch<B, E, H>(g->ordinal, G, s, mq, mk, mv, p, ws)
    if (p.D == 128) st = bf ? (e8 ? PB_GO(true, true, 128) : PB_GO(true, false, 128)) : (e8 ? PB_GO(false, true, 128) : PB_GO(false, false, 128));
    else st = bf ? (e8 ? PB_GO(true, true, 64) : PB_GO(true, false, 64)) : (e8 ? PB_GO(false, true, 64) : PB_GO(false, false, 64));
#undef PB_GO
    return st;
}

}  // namespace pb
