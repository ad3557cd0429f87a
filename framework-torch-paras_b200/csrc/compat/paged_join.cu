// What the streaming attention kernels over a paged cache share beside their loops: the TMA maps of cache and queries,
// and the kernel that joins the partial results of items cut between CTAs.
#include "paged_attn.cuh"
#include "tc_prims.cuh"
#include "tma_host.cuh"

namespace pb {
namespace {

constexpr int kJoinThreads = 256;

struct JoinSet {
    PagedWorkspace ws[2];
    int rows[2];
    int count, G;
};
constexpr int kMostRecords = 512;         // of both sets, on a GPU of up to 256 SMs

// out = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s over the parts s of an item, in the order of the CTAs.  A warp
// takes a row, the head dim over its lanes; the rows of all cut items stand in one row and are shared out evenly, which
// every block finds from the CTAs' records.  The parts were written a moment ago and lie in L2; with few of them
// latency is all of the cost: the launch is early and waits for the streaming kernel's memory, and four parts' outputs are
// asked for together with the maxima that weigh them.  Measured by itself: 5.9 us for one token over 1000 positions (7.2
// with a block per cut item and row, which had to look its record up first), 6.9 us for 64 tokens over 1024 (15.5),
// 10.7 us for 2 x 128 tokens over 16384 (16.0).
template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads)
paged_join_kernel(const PagedParams p, const __grid_constant__ JoinSet set) {
    __shared__ int ends[kMostRecords];          // rows up to and with record i
    __shared__ int4 recs[kMostRecords];         // first_slot, last_cta, row0, hk
    __shared__ int sums[kJoinThreads / 32];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int records = set.count * set.G;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    int total = 0;
    for (int i0 = 0; i0 < records; i0 += kJoinThreads) {
        const int i = i0 + tid;
        int n = 0;
        if (i < records) {
            const PagedJoin* j = i < set.G ? set.ws[0].join + i : set.ws[1].join + (i - set.G);
            const int4 a = __ldcg(reinterpret_cast<const int4*>(j));      // first_slot, last_cta, row0, nq
            const int hk = __ldcg(&j->hk);
            n = a.x >= 0 ? a.w * p.group : 0;
            recs[i] = make_int4(a.x, a.y, a.z, hk);
        }
        int incl = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        if (lane == 31) sums[warp] = incl;
        __syncthreads();
        int before = total;
        for (int w = 0; w < kJoinThreads / 32; ++w) {
            if (w < warp) before += sums[w];
            total += sums[w];
        }
        if (i < records) ends[i] = before + incl;
        __syncthreads();
    }
    constexpr int E = D / 32, kAhead = 4;
    for (int idx = int(blockIdx.x) * (kJoinThreads / 32) + warp; idx < total; idx += int(gridDim.x) * (kJoinThreads / 32)) {
        int lo = 0, hi = records - 1;        // the first record whose rows end after idx
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (ends[mid] > idx) hi = mid;
            else lo = mid + 1;
        }
        const int which = lo >= set.G, cta = which ? lo - set.G : lo;
        const PagedWorkspace ws = which ? set.ws[1] : set.ws[0];
        const int slot_rows = which ? set.rows[1] : set.rows[0], r = idx - (lo > 0 ? ends[lo - 1] : 0);
        const int4 rec = recs[lo];
        const int parts = rec.y - cta + 1;
        auto slot = [&](int i) { return i == 0 ? rec.x : 2 * (cta + i); };
        auto outputs = [&](int i, float (&o)[E]) {
            const float* src = ws.o + (size_t(slot(i)) * slot_rows + r) * D + lane * E;
#pragma unroll
            for (int e = 0; e < E; e += 2) {
                const float2 v = __ldcg(reinterpret_cast<const float2*>(src + e));
                o[e] = v.x;
                o[e + 1] = v.y;
            }
        };
        float M = -INFINITY, l = 0.f, acc[E];
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = 0.f;
        // 32 parts at a time (there are hardly ever more), four at once
        for (int i0 = 0; i0 < parts; i0 += 32) {
            const int n = min(32, parts - i0);
            float ahead[kAhead][E];
#pragma unroll
            for (int k = 0; k < kAhead; ++k)
                if (k < n) outputs(i0 + k, ahead[k]);
            float2 ml = make_float2(-INFINITY, 0.f);
            if (lane < n) ml = __ldcg(&ws.ml[size_t(slot(i0 + lane)) * slot_rows + r]);
            const float m_new = fmaxf(M, warp_max(ml.x));
            if (m_new == -INFINITY) continue;
            const float alpha = M == -INFINITY ? 0.f : tc::ex2_approx(M - m_new);
            // a part that saw no key weighs nothing, and its outputs may not have been written
            const float w = ml.x == -INFINITY ? 0.f : tc::ex2_approx(ml.x - m_new);
            l = l * alpha + warp_sum(w * ml.y);
            M = m_new;
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] *= alpha;
            for (int k0 = 0; k0 < n; k0 += kAhead) {
                if (k0 > 0) {
#pragma unroll
                    for (int k = 0; k < kAhead; ++k)
                        if (k0 + k < n) outputs(i0 + k0 + k, ahead[k]);
                }
#pragma unroll
                for (int k = 0; k < kAhead; ++k) {
                    const float wk = __shfl_sync(0xffffffffu, w, (k0 + k) & 31);
                    if (k0 + k < n && wk != 0.f) {
#pragma unroll
                        for (int e = 0; e < E; ++e) acc[e] = fmaf(wk, ahead[k][e], acc[e]);
                    }
                }
            }
        }
        const int tok = rec.z + r / p.group, h = rec.w * p.group + r % p.group;
        const float inv = M == -INFINITY ? 0.f : 1.0f / l;
        T* out = static_cast<T*>(p.out) + int64_t(tok) * p.os[0] + int64_t(h) * p.os[1];
#pragma unroll
        for (int e = 0; e < E; ++e) out[lane * E + e] = from_f32<T>(acc[e] * inv);
        if (p.lse && lane == 0)
            p.lse[int64_t(tok) * p.Hq + h] = M == -INFINITY ? -INFINITY : M * 0.6931471805599453f + logf(l);
    }
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace

int paged_join_launch(const Gpu* g, const PagedParams& p, const PagedWorkspace* ws, const int* rows, int count, int G, int dtype,
                      cudaStream_t s) {
    JoinSet set{};
    int most = 0;
    for (int i = 0; i < count; ++i) {
        set.ws[i] = ws[i];
        set.rows[i] = rows[i];
        most += G * rows[i];
    }
    set.count = count;
    set.G = G;
    if (count * G > kMostRecords) return fail(PARAS_E_UNSUPPORTED, "paras paged_attention: a GPU of more than 256 SMs");
    // up to four blocks an SM, as many as the most rows that can be cut give work to
    const int per_sm = (most + 8 * g->sm_count - 1) / (8 * g->sm_count);
    const dim3 grid(unsigned(g->sm_count * (per_sm < 4 ? per_sm : 4)));
    cudaError_t e;
    if (dtype == PARAS_BF16)
        e = p.D == 128 ? paged_launch(paged_join_kernel<__nv_bfloat16, 128>, grid, kJoinThreads, 0, s, p, set)
                       : paged_launch(paged_join_kernel<__nv_bfloat16, 64>, grid, kJoinThreads, 0, s, p, set);
    else
        e = p.D == 128 ? paged_launch(paged_join_kernel<__half, 128>, grid, kJoinThreads, 0, s, p, set)
                       : paged_launch(paged_join_kernel<__half, 64>, grid, kJoinThreads, 0, s, p, set);
    if (e != cudaSuccess) return fail(PARAS_E_CUDA, "paras paged_attention: launch of paged_join_kernel failed: %s", cudaGetErrorString(e));
    return PARAS_OK;
}

bool paged_tma_ok(const paras_paged_cache& c) {
    // a tile of 128 positions is one piece of a page, or whole pages of whole 8-row swizzle groups
    const bool page_ok = c.page % kTileKeys == 0 || (c.page >= 8 && kTileKeys % c.page == 0);
    if (!page_ok || c.pages < 1 || c.max_pages < 1 || (c.D != 128 && c.D != 64)) return false;
    const int64_t es = c.cache_dtype == PARAS_E4M3 ? 1 : 2;
    for (int which = 0; which < 2; ++which) {
        const int64_t* st = which ? c.v_strides : c.k_strides;
        const int64_t n[3] = {c.pages, c.Hkv, c.page};
        if (!al16(which ? c.v : c.k)) return false;
        for (int i = 0; i < 3; ++i)
            if (n[i] > 1 && (st[i] <= 0 || (st[i] * es) % 16 || st[i] * es >= (int64_t(1) << 40))) return false;
    }
    return true;
}

int paged_cache_map(CUtensorMap* map, const paras_paged_cache& c, int which, bool whole) {
    TensorMapEncodeFn fn = tensor_map_encode_fn();
    if (!fn) return fail(PARAS_E_CUDA, "paras_b200: cuTensorMapEncodeTiled is unavailable");
    const bool e8 = c.cache_dtype == PARAS_E4M3;
    const int64_t es = e8 ? 1 : 2;
    const int64_t* st = which ? c.v_strides : c.k_strides;
    // the stride of a size-1 dim is never used for addressing; keep it a legal multiple of 16 bytes
    const int64_t s2 = c.page > 1 ? st[2] : c.D, s1 = c.Hkv > 1 ? st[1] : s2 * c.page, s0 = c.pages > 1 ? st[0] : s1 * c.Hkv;
    const cuuint32_t rows = cuuint32_t(c.page < kTileKeys ? c.page : kTileKeys), inner = cuuint32_t(e8 ? c.D : 64), slabs = cuuint32_t(c.D) / inner;
    const cuuint32_t estr[5] = {1, 1, 1, 1, 1};
    const CUtensorMapDataType dt = e8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                      : c.cache_dtype == PARAS_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const CUtensorMapSwizzle swizzle = e8 && c.D == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B;
    void* base = which ? c.v : c.k;
    CUresult r;
    if (whole) {
        const cuuint64_t dims[5] = {inner, cuuint64_t(c.page), slabs, cuuint64_t(c.Hkv), cuuint64_t(c.pages)};
        const cuuint64_t strides[4] = {cuuint64_t(s2 * es), 128, cuuint64_t(s1 * es), cuuint64_t(s0 * es)};
        const cuuint32_t box[5] = {inner, rows, slabs, 1, 1};
        r = fn(map, dt, 5, base, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    } else {
        const cuuint64_t dims[4] = {cuuint64_t(c.D), cuuint64_t(c.page), cuuint64_t(c.Hkv), cuuint64_t(c.pages)};
        const cuuint64_t strides[3] = {cuuint64_t(s2 * es), cuuint64_t(s1 * es), cuuint64_t(s0 * es)};
        const cuuint32_t box[4] = {inner, rows, 1, 1};
        r = fn(map, dt, 4, base, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    }
    if (r != CUDA_SUCCESS) return fail(PARAS_E_CUDA, "paras_b200: cuTensorMapEncodeTiled failed with code %d", int(r));
    return PARAS_OK;
}

bool paged_q_tma_ok(const paras_paged_attn_args& a) {
    if (!al16(a.q)) return false;
    if (a.T > 1 && (a.q_strides[0] <= 0 || a.q_strides[0] % 8)) return false;
    if (a.Hq > 1 && (a.q_strides[1] <= 0 || a.q_strides[1] % 8)) return false;
    return true;
}

int paged_q_map(CUtensorMap* map, const paras_paged_attn_args& a, int tokens) {
    TensorMapEncodeFn fn = tensor_map_encode_fn();
    if (!fn) return fail(PARAS_E_CUDA, "paras_b200: cuTensorMapEncodeTiled is unavailable");
    const int64_t g = a.Hq / a.cache.Hkv, D = a.cache.D;
    const cuuint64_t dims[4] = {cuuint64_t(D), cuuint64_t(g), cuuint64_t(a.cache.Hkv), cuuint64_t(a.T)};
    const int64_t sh = a.Hq > 1 ? a.q_strides[1] : D, st = a.T > 1 ? a.q_strides[0] : sh * a.Hq;
    const cuuint64_t strides[3] = {cuuint64_t(sh * 2), cuuint64_t(sh * g * 2), cuuint64_t(st * 2)};
    const cuuint32_t box[4] = {64, cuuint32_t(g), 1, cuuint32_t(tokens)};
    const cuuint32_t estr[4] = {1, 1, 1, 1};
    const CUresult r = fn(map, a.dtype == PARAS_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                          const_cast<void*>(a.q), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(PARAS_E_CUDA, "paras_b200: cuTensorMapEncodeTiled failed with code %d", int(r));
    return PARAS_OK;
}

}  // namespace pb
