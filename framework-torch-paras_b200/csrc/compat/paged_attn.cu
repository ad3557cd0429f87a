// Attention of new tokens over a paged cache (include/paras_b200.h, "paged key / value cache"): entry point, and the
// CUDA-core kernel that takes every type, head dim, page size and alignment.
//
//   out_t = sum_j softmax_j(scale * q_t . k_j) v_j     over the positions j that token t attends
//
// paged_simt_kernel: a warp per (token, query head).  Keys in blocks of 32: lane j forms the whole score of key j
// (q comes from shared memory), the block's maximum and sum join the running ones, then the warp adds p_j v_j with
// the head dim over its lanes.  Keys and values that are not attended are never touched.
#include "paged_attn.cuh"

#include <cmath>

namespace pb {
namespace {

thread_local const char* tl_paged_kernel = "";

constexpr int kWarps = 4;

// element d of a cache row
template <typename T, bool CACHE8>
__device__ __forceinline__ float cache_at(const char* base, int64_t at) {
    if constexpr (CACHE8) return e4m3_to_f32(reinterpret_cast<const uint8_t*>(base)[at]);
    else return to_f32<T>(reinterpret_cast<const T*>(base)[at]);
}

template <typename T, bool CACHE8>
__global__ void __launch_bounds__(kWarps * 32)
paged_simt_kernel(const PagedParams p) {
    __shared__ float q_sm[kWarps][256];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t unit = int64_t(blockIdx.x) * kWarps + warp;
    if (unit >= int64_t(p.T) * p.Hq) return;
    const int t = int(unit / p.Hq), h = int(unit - int64_t(t) * p.Hq), hk = h / p.group;
    const int b = warp_count_le(p.cu + 1, p.B, t);
    if (b >= p.B) return;
    const PagedSeq sq = paged_seq(p, b);
    const int i = t - sq.row0;
    if (i < 0 || i >= sq.nq) return;
    const T* qrow = static_cast<const T*>(p.q) + int64_t(t) * p.qs[0] + int64_t(h) * p.qs[1];
    for (int d = lane; d < p.D; d += 32) q_sm[warp][d] = to_f32<T>(qrow[d]);
    __syncwarp();
    const int n = paged_keys(p, sq, i);
    float m = -INFINITY, l = 0.f, acc[8];
    bool nan = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = 0.f;
    for (int j0 = 0; j0 < n; j0 += 32) {
        const int j = j0 + lane;
        float s = -INFINITY, vscale = 1.f;
        int64_t vrow = -1;
        if (j < n) {
            const int page = __ldg(p.table + int64_t(b) * p.table_stride + j / p.page), off = j % p.page;
            if (uint32_t(page) < uint32_t(p.pages)) {
                const int64_t krow = int64_t(page) * p.cks[0] + int64_t(hk) * p.cks[1] + int64_t(off) * p.cks[2];
                vrow = int64_t(page) * p.cvs[0] + int64_t(hk) * p.cvs[1] + int64_t(off) * p.cvs[2];
                float dot = 0.f;
                for (int d = 0; d < p.D; ++d) dot = fmaf(q_sm[warp][d], cache_at<T, CACHE8>(p.ck, krow + d), dot);
                if constexpr (CACHE8) {
                    dot *= exp_byte(p.ek[int64_t(page) * p.eks[0] + int64_t(hk) * p.eks[1] + int64_t(off) * p.eks[2]]);
                    vscale = exp_byte(p.ev[int64_t(page) * p.evs[0] + int64_t(hk) * p.evs[1] + int64_t(off) * p.evs[2]]);
                }
                s = dot * p.scale;
            }
        }
        nan = nan || __any_sync(0xffffffffu, s != s);      // (maxima skip it)
        const float m_new = fmaxf(m, warp_max(s));
        if (m_new == -INFINITY) continue;     // nothing attended so far
        const float alpha = expf(m - m_new);
        const float pj = vrow >= 0 ? expf(s - m_new) : 0.f;
        l = l * alpha + warp_sum(pj);
        m = m_new;
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] *= alpha;
        const float w = pj * vscale;
        const int cnt = min(32, n - j0);
        for (int k = 0; k < cnt; ++k) {
            const int64_t at = __shfl_sync(0xffffffffu, vrow, k);
            const float wk = __shfl_sync(0xffffffffu, w, k);
            if (at < 0) continue;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (lane + 32 * e < p.D) acc[e] = fmaf(wk, cache_at<T, CACHE8>(p.cv, at + lane + 32 * e), acc[e]);
        }
    }
    T* orow = static_cast<T*>(p.out) + int64_t(t) * p.os[0] + int64_t(h) * p.os[1];
    const float inv = nan ? NAN : m == -INFINITY ? 0.f : 1.0f / l;
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (lane + 32 * e < p.D) orow[lane + 32 * e] = from_f32<T>(acc[e] * inv);
    if (p.lse && lane == 0) p.lse[unit] = nan ? NAN : m == -INFINITY ? -INFINITY : m + logf(l);
}

int check(const paras_paged_attn_args* args, const char* what) {
    if (!args) return fail(PARAS_E_INVALID, "%s: null args", what);
    const paras_paged_attn_args& a = *args;
    const int st = check_paged_cache(a.cache, a.dtype, what);
    if (st != PARAS_OK) return st;
    if (a.T < 0 || a.max_q < 0) return fail(PARAS_E_INVALID, "%s: negative size", what);
    if (a.Hq < 1 || a.Hq % a.cache.Hkv)
        return fail(PARAS_E_INVALID, "%s: query heads (%d) must be a multiple of key/value heads (%d)", what, a.Hq, a.cache.Hkv);
    if (int64_t(a.T) * a.Hq > (int64_t(1) << 32)) return fail(PARAS_E_UNSUPPORTED, "%s: more than 2^32 query rows", what);
    if (!std::isfinite(float(a.scale))) return fail(PARAS_E_INVALID, "%s: scale is not finite", what);
    return PARAS_OK;
}

// At most 16 query rows per kv head stream through mma.sync tiles (64 single tokens over 512 .. 16384 positions: 340 us, in
// 128-row tiles 441; 48 x 4 tokens: 144 and 199, from an 8-bit cache 122 and 320; one token over 1000: 12.0 and 14.3), more go
// to the tensor-core tiles of 128 rows; fp32, other head dims than 64 and 128, pages that no tile of 128 positions is made of,
// and unaligned tensors to CUDA cores.
// A call for chunks whose sequences besides the longest average less than twice 16 rows is taken to mix both, and makes a
// launch for each where the others may have enough tiles to make up for the second launch (about 12 us): 80 for each
// multiprocessor, or 14 of an 8-bit cache, whose bytes the 128-row kernel converts at half the rate.  In one launch and in
// two, one sequence of 700 tokens and n of one over up to L positions, 8 kv heads of 128: 16-bit n = 15, L = 4096: 97 and
// 108 us; 47, 4096: 157 and 160; 95, 4096: 255 and 235; 31, 16384: 419 and 379; 8-bit n = 3, L = 4096: 105 and 109 us;
// 7, 4096: 120 and 117; 31, 4096: 210 and 154; 15, 16384: 495 and 367.
// The rule goes by counts the host knows, of lengths the page table's reach; where it is wrong, the second launch costs that.
struct Routes {
    bool decode, tc;
    int small;      // tokens a sequence may have for the first of the two
};
Routes pick_routes(const Gpu* g, const paras_paged_attn_args& a) {
    Routes r{};
    const int group = a.Hq / a.cache.Hkv;
    r.small = 16 / group;
    const bool dec = paged_decode_supported(g, a);
    if (dec && a.max_q <= r.small) {
        r.decode = true;
    } else if (paged_tc_supported(g, a)) {
        r.tc = true;
        const int64_t others = a.cache.B - 1, left = int64_t(a.T) - a.max_q;
        const int64_t tiles = others * a.cache.Hkv * ((int64_t(a.cache.max_pages) * a.cache.page + kTileKeys - 1) / kTileKeys);
        const int64_t least = a.cache.cache_dtype == PARAS_E4M3 ? 14 : 80;
        r.decode = dec && others > 0 && left < others * 2 * r.small && tiles >= least * g->sm_count;
    }
    return r;
}
size_t round16(size_t n) { return (n + 15) & ~size_t(15); }
int stream_ctas(const Gpu* g) { return g->sm_count > 0 ? g->sm_count : 148; }   // persistent, one per SM

PagedParams make_params(const Gpu* g, const paras_paged_attn_args& a) {
    const paras_paged_cache& c = a.cache;
    PagedParams p{};
    p.q = a.q; p.out = a.out; p.lse = a.lse;
    p.ck = static_cast<const char*>(c.k); p.cv = static_cast<const char*>(c.v);
    p.ek = c.k_exp; p.ev = c.v_exp;
    p.table = c.page_table; p.kv_lens = a.kv_lens; p.cu = a.cu; p.table_stride = c.table_stride;
    for (int i = 0; i < 2; ++i) { p.qs[i] = a.q_strides[i]; p.os[i] = a.o_strides[i]; }
    for (int i = 0; i < 3; ++i) {
        p.cks[i] = c.k_strides[i]; p.cvs[i] = c.v_strides[i];
        p.eks[i] = c.k_exp_strides[i]; p.evs[i] = c.v_exp_strides[i];
    }
    p.T = a.T; p.Hq = a.Hq; p.Hkv = c.Hkv; p.group = a.Hq / c.Hkv; p.D = c.D; p.B = c.B;
    p.max_pages = c.max_pages; p.pages = c.pages; p.page = c.page; p.max_q = a.max_q;
    p.cap = c.max_pages * c.page;
    p.causal = a.causal;
    p.scale = float(a.scale);
    p.scale_log2 = p.scale * 1.4426950408889634f;
    p.q_min = 1;
    p.q_max = p.qbox = p.max_q;
    p.status = g->status_dev;
    const int box = c.page < kTileKeys ? c.page : kTileKeys;
    p.box_shift = 0;
    while ((2 << p.box_shift) <= box) ++p.box_shift;
    p.npg = kTileKeys >> p.box_shift;
    p.tpp = c.page > kTileKeys ? c.page / kTileKeys : 1;
    return p;
}

}  // namespace

int paged_simt_launch(const PagedParams& p, int dtype, bool cache8, cudaStream_t s) {
    const unsigned blocks = unsigned((int64_t(p.T) * p.Hq + kWarps - 1) / kWarps);
    auto go = [&](auto kernel) { kernel<<<blocks, kWarps * 32, 0, s>>>(p); };
    switch (dtype) {
        case PARAS_F32: cache8 ? go(paged_simt_kernel<float, true>) : go(paged_simt_kernel<float, false>); break;
        case PARAS_BF16: cache8 ? go(paged_simt_kernel<__nv_bfloat16, true>) : go(paged_simt_kernel<__nv_bfloat16, false>); break;
        default: cache8 ? go(paged_simt_kernel<__half, true>) : go(paged_simt_kernel<__half, false>); break;
    }
    PB_LAUNCH_CHECK("paged_simt_kernel");
    tl_paged_kernel = "paged_simt";
    return PARAS_OK;
}

}  // namespace pb

using pb::fail;

extern "C" {

int paras_b200_paged_attn(const paras_paged_attn_args* args) {
    pb::NvtxRange range("paras_b200_paged_attn");
    const char* what = "paras paged_attention";
    int st = pb::check(args, what);
    if (st != PARAS_OK) return st;
    const paras_paged_attn_args& a = *args;
    pb::DeviceRestore restore;
    pb::Gpu* g = pb::use_gpu(a.gpu, &st);
    if (!g) return st;
    if (a.T == 0 || a.cache.B == 0 || a.max_q == 0) return PARAS_OK;
    if (!a.q || !a.out || !a.kv_lens || !a.cu) return fail(PARAS_E_INVALID, "%s: null pointer", what);
    const pb::PagedParams p = pb::make_params(g, a);
    cudaStream_t s = pb::pick_stream(g, a.stream);
    const pb::Routes r = pb::pick_routes(g, a);
    if (!r.decode && !r.tc) return pb::paged_simt_launch(p, a.dtype, a.cache.cache_dtype == PARAS_E4M3, s);
    const int G = pb::stream_ctas(g);
    const size_t dec_bytes = r.decode ? pb::round16(pb::paged_workspace_bytes(G, pb::paged_decode_rows(), p.D)) : 0;
    const size_t need = dec_bytes + (r.tc ? pb::paged_workspace_bytes(G, pb::paged_tc_rows(), p.D) : 0);
    void* scratch = a.workspace;
    if (scratch) {
        if (a.workspace_bytes < need)
            return fail(PARAS_E_INVALID, "%s: workspace of %zu bytes is too small, %zu are needed", what, a.workspace_bytes, need);
        if (reinterpret_cast<uintptr_t>(scratch) & 15u) return fail(PARAS_E_INVALID, "%s: workspace is not 16-byte aligned", what);
    } else if ((st = paras_b200_malloc_async(a.gpu, need, s, &scratch)) != PARAS_OK) {
        return st;
    }
    pb::PagedWorkspace ws[2];
    int rows[2], count = 0;
    if (r.tc) {
        pb::PagedParams pt = p;
        if (r.decode) pt.q_min = r.small + 1;
        rows[count] = pb::paged_tc_rows();
        ws[count] = pb::paged_carve(static_cast<char*>(scratch) + dec_bytes, G, rows[count]);
        st = pb::paged_tc_launch(g, a, pt, ws[count++], G, s);
    }
    if (st == PARAS_OK && r.decode) {
        pb::PagedParams pd = p;
        pd.q_max = r.small < p.max_q ? r.small : p.max_q;
        pd.qbox = pd.q_max;
        pd.wait_late = r.tc;
        rows[count] = pb::paged_decode_rows();
        ws[count] = pb::paged_carve(scratch, G, rows[count]);
        st = pb::paged_decode_launch(g, a, pd, ws[count++], G, s);
    }
    if (st == PARAS_OK) st = pb::paged_join_launch(g, p, ws, rows, count, G, a.dtype, s);
    if (st == PARAS_OK) pb::tl_paged_kernel = r.tc ? (r.decode ? "paged_tcgen05+paged_decode" : "paged_tcgen05") : "paged_decode";
    if (!a.workspace) {
        const int st2 = paras_b200_free_async(a.gpu, scratch, s);
        if (st == PARAS_OK) st = st2;
    }
    return st;
}

int paras_b200_paged_attn_workspace_bytes(const paras_paged_attn_args* args, size_t* bytes) {
    int st = pb::check(args, "paras paged_attention");
    if (st != PARAS_OK) return st;
    if (!bytes) return fail(PARAS_E_INVALID, "paras paged_attention: null pointer");
    *bytes = 0;
    pb::DeviceRestore restore;
    pb::Gpu* g = pb::use_gpu(args->gpu, &st);
    if (!g) return st;
    const pb::Routes r = pb::pick_routes(g, *args);
    const int G = pb::stream_ctas(g), D = args->cache.D;
    if (r.decode) *bytes += pb::round16(pb::paged_workspace_bytes(G, pb::paged_decode_rows(), D));
    if (r.tc) *bytes += pb::paged_workspace_bytes(G, pb::paged_tc_rows(), D);
    return PARAS_OK;
}

const char* paras_b200_paged_attn_last_kernel(void) { return pb::tl_paged_kernel; }

}  // extern "C"
