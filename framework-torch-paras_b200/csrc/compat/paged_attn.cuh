// Internal interfaces of the attention kernels over a paged cache.
#pragma once

#include <atomic>

#include "paged_common.cuh"

struct CUtensorMap_st;

namespace pb {

// What every route needs of the call.
struct PagedParams {
    const void* q;
    void* out;
    float* lse;
    const char *ck, *cv;
    const uint8_t *ek, *ev;
    const int32_t *table, *kv_lens, *cu;
    int64_t table_stride;
    int64_t qs[2], os[2];
    int64_t cks[3], cvs[3], eks[3], evs[3];
    int T, Hq, Hkv, group, D, B, max_pages, pages, page, max_q;
    // A launch takes the sequences of q_min to q_max new tokens (a call that mixes single tokens with chunks makes one
    // launch for each); qbox: tokens that a TMA box on q covers in the launch for few.
    int q_min, q_max, qbox;
    int wait_late;       // the launch depends on the one before it only for the order of what comes after
    int cap;             // positions the page table can name
    int causal;
    float scale, scale_log2;
    int* status;
    // Pages as the TMA routes see them: a tile of 128 positions is `npg` boxes of 2^box_shift positions, one per page, or
    // one box of a page that holds `tpp` tiles.
    int box_shift, npg, tpp;
};

// The new tokens of sequence b: first row, count (at most max_q), positions in the cache.  Whatever the device arrays
// hold, rows stay within [0, T).
struct PagedSeq {
    int row0, nq;
    int kv;       // positions 0 .. kv-1, kv <= cap
    int pos0;     // position of the first new token (may be negative or past kv); pos0 + nq is at most kv_lens[b]
};
// From cu[b], cu[b+1] and kv_lens[b].  A row's position is kv_lens[b] - cu[b+1] + row, also of a sequence that goes on past the last
// row there is; below -2^31 any negative position is as good.
__host__ __device__ __forceinline__ PagedSeq paged_place(const PagedParams& p, int c0, int c1, int kv) {
    PagedSeq s;
    s.row0 = c0 < 0 ? 0 : c0 < p.T ? c0 : p.T;
    const int end = c1 < s.row0 ? s.row0 : c1 < p.T ? c1 : p.T;
    const int count = end - s.row0;
    s.nq = count < p.max_q ? count : p.max_q;
    if (s.nq < p.q_min || s.nq > p.q_max) s.nq = 0;
    s.kv = kv < 0 ? 0 : kv < p.cap ? kv : p.cap;
    const int64_t pos0 = int64_t(kv) - c1 + s.row0, least = -(int64_t(1) << 31);
    s.pos0 = int(pos0 < least ? least : pos0);
    return s;
}
__device__ __forceinline__ PagedSeq paged_seq(const PagedParams& p, int b) {
    return paged_place(p, __ldg(p.cu + b), __ldg(p.cu + b + 1), __ldg(p.kv_lens + b));
}
// Keys that new token i of the sequence attends: positions 0 .. n-1.
__host__ __device__ __forceinline__ int paged_keys(const PagedParams& p, const PagedSeq& s, int i) {
    const int n = s.pos0 + i + 1;
    return !p.causal ? s.kv : n < 0 ? 0 : n < s.kv ? n : s.kv;
}

// The streaming kernels move their reference by products with c2 = scale * log2(e) (times a row's power of two) and its
// inverse, which have to stay finite: scales below 2^-100 go to the CUDA cores, a row's c2 stays above 2^-120 (rows of q
// below 2^-126 of an ordinary one, whose scores are all the same to fp32).
constexpr float kLeastC2 = 7.5231638452626401e-37f;      // 2^-120
inline bool paged_scale_ok(const paras_paged_attn_args& a) { return a.scale >= 7.888609052210118e-31; }   // 2^-100

int paged_simt_launch(const PagedParams& p, int dtype, bool cache8, cudaStream_t s);

// ---- the streaming kernels' shared-out work ------------------------------------------------------
// Their unit of work is a tile: 128 positions of the cache for one item (the query rows that share a pass over a kv
// head's keys).  All W tiles of a call stand in one row, sequence by sequence, and CTA c of G takes those from c*W/G to
// (c+1)*W/G (with fewer tiles than CTAs, G = W of them take one each): every CTA streams the same amount whatever the
// lengths are, and the host need not know them.  An item cut by such a border leaves partial results in the workspace, at
// most two per CTA (slot 2c for the item that the CTA starts in the middle of or at its first tile, 2c+1 for a later one
// that goes on in the next CTA), and a second kernel joins the parts of each such item in the order of the CTAs.
constexpr int kTileKeys = 128;

// Tiles of the kernel for chunks: an item is up to 2 * pt tokens of a sequence (two query tiles) and one kv head, and an item
// with nothing to attend has one empty tile.  A head's tiles are counted in 64 bits: many items of long sequences pass 2^31.
__host__ __device__ __forceinline__ int tiles_for(int keys) { return keys <= kTileKeys ? 1 : (keys + kTileKeys - 1) / kTileKeys; }
__host__ __device__ __forceinline__ int item_tiles(const PagedParams& p, const PagedSeq& s, int i, int pt) {
    const int end = (i + 1) * 2 * pt;
    return tiles_for(paged_keys(p, s, (end < s.nq ? end : s.nq) - 1));
}
__host__ __device__ __forceinline__ int64_t head_tiles(const PagedParams& p, const PagedSeq& s, int pt) {
    const int items = (s.nq + 2 * pt - 1) / (2 * pt);
    if (!p.causal) return items > 0 ? int64_t(items) * tiles_for(s.kv) : 0;
    int64_t n = 0;
    for (int i = 0; i < items; ++i) n += item_tiles(p, s, i, pt);
    return n;
}

struct PagedRange {
    int64_t total, ctas;    // W, G
    int64_t begin, end;
    // the CTA that has tile x: the largest c with c * W / G <= x
    __device__ __forceinline__ int owner(int64_t x) const { return int(((x + 1) * ctas - 1) / total); }
};

// What the joining kernel has to know of the item that starts in CTA c and goes on; written by that CTA.
struct PagedJoin {
    int first_slot;   // -1: nothing to join
    int last_cta;     // parts: first_slot, then slot 2*k for the CTAs up to this one
    int row0;         // first token row, tokens and kv head of the item
    int nq, hk;
    int pad[3];
};
static_assert(sizeof(PagedJoin) == 32, "joins are laid out as 32-byte records");

// Workspace of G CTAs with items of `rows` query rows: joins, {max, sum} pairs, partial outputs (fp32, unnormalised).
struct PagedWorkspace {
    PagedJoin* join;
    float2* ml;       // [2G][rows]   maximum of the scores * scale * log2(e), sum of the exponentials
    float* o;         // [2G][rows][D]
};
inline size_t paged_workspace_bytes(int G, int rows, int D) {
    return size_t(G) * sizeof(PagedJoin) + size_t(2 * G) * rows * (sizeof(float2) + size_t(D) * sizeof(float));
}
inline PagedWorkspace paged_carve(void* base, int G, int rows) {
    PagedWorkspace w;
    w.join = static_cast<PagedJoin*>(base);
    w.ml = reinterpret_cast<float2*>(w.join + G);
    w.o = reinterpret_cast<float*>(w.ml + size_t(2 * G) * rows);   // (G*32 + 2G*rows*8 bytes: a multiple of 16)
    return w;
}

// Inclusive sum over a warp.
__device__ __forceinline__ int64_t warp_scan(int64_t v) {
    const int lane = int(threadIdx.x) & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    return v;
}

// Finds this CTA's range and the sequence in which it begins; every thread of the block calls it.  tiles(b) is the number
// of tiles of sequence b.  `sums` has a place per warp and three more.  Returns the range; *b0 / *base0: that sequence
// and the place of its first tile in the row (only where begin < end).
template <typename Tiles>
__device__ __forceinline__ PagedRange paged_range(int B, int64_t* sums, Tiles tiles, int* b0, int64_t* base0) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = int(blockDim.x) >> 5;
    int64_t* total = sums + nw;   // total, found sequence, its base
    int64_t W = 0;
    for (int chunk = 0; chunk < B; chunk += int(blockDim.x)) {
        const int b = chunk + tid;
        W += b < B ? tiles(b) : 0;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) W += __shfl_xor_sync(0xffffffffu, W, o);
    if (lane == 0) sums[warp] = W;
    __syncthreads();
    W = 0;
    for (int i = 0; i < nw; ++i) W += sums[i];
    PagedRange r;
    r.total = W;
    r.ctas = min(W, int64_t(gridDim.x));
    r.begin = r.end = 0;
    if (int64_t(blockIdx.x) < r.ctas) {
        r.begin = int64_t(blockIdx.x) * W / r.ctas;
        r.end = (int64_t(blockIdx.x) + 1) * W / r.ctas;
    }
    if (tid == 0) {
        total[1] = 0;
        total[2] = 0;
    }
    if (r.begin < r.end) {        // (the same for the whole block)
        int64_t base = 0;
        for (int chunk = 0; chunk < B && base <= r.begin; chunk += int(blockDim.x)) {
            const int b = chunk + tid;
            const int64_t n = b < B ? tiles(b) : 0;
            const int64_t incl = warp_scan(n);
            __syncthreads();      // sums is free
            if (lane == 31) sums[warp] = incl;
            __syncthreads();
            int64_t before = base, all = base;
            for (int i = 0; i < nw; ++i) {
                if (i < warp) before += sums[i];
                all += sums[i];
            }
            const int64_t at = before + incl - n;
            if (n > 0 && at <= r.begin && r.begin < at + n) {
                total[1] = b;
                total[2] = at;
            }
            base = all;
        }
    }
    __syncthreads();
    *b0 = int(total[1]);
    *base0 = total[2];
    return r;
}

// Lets `Kernel` use `bytes` of dynamic shared memory on the current device `gpu`; asked of the driver once per device.  A kernel
// that moves registers between its warps counts on `regs` a thread at launch: with fewer it would wait for them for ever.
template <auto Kernel>
cudaError_t paged_allow_smem(int gpu, int bytes, int regs = 0) {
    static std::atomic<uint64_t> done{0};
    const uint64_t bit = uint64_t(1) << (gpu & 63);
    if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
    cudaError_t e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && regs > 0) {
        cudaFuncAttributes at;
        e = cudaFuncGetAttributes(&at, Kernel);
        if (e == cudaSuccess && at.numRegs < regs) e = cudaErrorLaunchOutOfResources;
    }
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    return e;
}

// Joins the partial results that up to two streaming launches (of G CTAs, items of rows[i] query rows) left of their cut
// items: one launch after them on the same stream.
int paged_join_launch(const Gpu* g, const PagedParams& p, const PagedWorkspace* ws, const int* rows, int count, int G, int dtype,
                      cudaStream_t s);

// Launches `kernel` so that its start may overlap the end of the kernel before it, for whose memory it waits itself
// (griddepcontrol.wait).
template <typename... Params, typename... Args>
cudaError_t paged_launch(void (*kernel)(Params...), dim3 grid, int threads, size_t smem, cudaStream_t s, const Args&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(unsigned(threads), 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, Params(args)...);
}

bool paged_decode_supported(const Gpu* g, const paras_paged_attn_args& a);
int paged_decode_rows();     // query rows of an item in the workspace
int paged_decode_launch(Gpu* g, const paras_paged_attn_args& a, const PagedParams& p, const PagedWorkspace& ws, int G, cudaStream_t s);

bool paged_tc_supported(const Gpu* g, const paras_paged_attn_args& a);
int paged_tc_rows();
int paged_tc_launch(Gpu* g, const paras_paged_attn_args& a, const PagedParams& p, const PagedWorkspace& ws, int G, cudaStream_t s);

// Can the cache be read by TMA in tiles of 128 positions (page size, alignment, strides)?
bool paged_tma_ok(const paras_paged_cache& c);
// Map of the cache's K (which = 0) or V, a box of one page's (at most 128) rows by 128 bytes (the row, where it is
// shorter): {D, position, head, page}, 16-bit rows in slabs of 64 elements that are loaded one by one; or, with `whole`,
// {64, position, slab, head, page} and all slabs in one box, slab after slab.
int paged_cache_map(CUtensorMap_st* map, const paras_paged_cache& c, int which, bool whole);
// Map of q seen as {D, group, kv head, token}: box {64, group, 1, tokens}.
bool paged_q_tma_ok(const paras_paged_attn_args& a);
int paged_q_map(CUtensorMap_st* map, const paras_paged_attn_args& a, int tokens);

}  // namespace pb
