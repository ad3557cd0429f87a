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
};

// out = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s over the parts s of an item, in the order of the CTAs: a warp per
// row, the head dim over its lanes.  The parts were written a moment ago and lie in L2, and few items are cut, so latency
// is all of its cost: it is launched early and waits for the streaming kernel's memory, and the first four parts' outputs
// are asked for together with the maxima that weigh them.
template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads)
paged_join_kernel(const PagedParams p, const JoinSet set) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const PagedWorkspace& ws = set.ws[blockIdx.z];
    const int slot_rows = set.rows[blockIdx.z];
    const PagedJoin j = ws.join[blockIdx.x];
    if (j.first_slot < 0) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rows = j.nq * p.group, parts = j.last_cta - int(blockIdx.x) + 1;
    constexpr int E = D / 32, kAhead = 4;
    auto slot = [&](int i) { return i == 0 ? j.first_slot : 2 * (int(blockIdx.x) + i); };
    for (int r = blockIdx.y * (kJoinThreads / 32) + warp; r < rows; r += gridDim.y * (kJoinThreads / 32)) {
        auto outputs = [&](int i, float (&o)[E]) {
            const float* src = ws.o + (size_t(slot(i)) * slot_rows + r) * D + lane * E;
#pragma unroll
            for (int e = 0; e < E; e += 2) {
                const float2 v = __ldcg(reinterpret_cast<const float2*>(src + e));
                o[e] = v.x;
                o[e + 1] = v.y;
            }
        };
        float ahead[kAhead][E];
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
            if (i < parts) outputs(i, ahead[i]);
        // lane i looks at parts i, i + 32, ...
        float M = -INFINITY;
        float2 ml = make_float2(-INFINITY, 0.f);
        if (lane < parts) ml = __ldcg(&ws.ml[size_t(slot(lane)) * slot_rows + r]);
        M = ml.x;
        for (int i = lane + 32; i < parts; i += 32) M = fmaxf(M, __ldcg(&ws.ml[size_t(slot(i)) * slot_rows + r]).x);
        M = warp_max(M);
        float l = 0.f, acc[E];
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = 0.f;
        if (M != -INFINITY) {
            float w = 0.f;      // of part i0 + lane; 0 for one that saw no key, whose outputs may not have been written
            for (int i = 0; i < parts; ++i) {
                if ((i & 31) == 0) {
                    if (i > 0) ml = i + lane < parts ? __ldcg(&ws.ml[size_t(slot(i + lane)) * slot_rows + r]) : make_float2(-INFINITY, 0.f);
                    w = ml.x == -INFINITY ? 0.f : tc::ex2_approx(ml.x - M);
                    l += warp_sum(w * ml.y);
                }
                const float wi = __shfl_sync(0xffffffffu, w, i & 31);
                float o[E];
                if (i < kAhead) {
#pragma unroll
                    for (int k = 0; k < kAhead; ++k)
                        if (k == i) {
#pragma unroll
                            for (int e = 0; e < E; ++e) o[e] = ahead[k][e];
                        }
                } else {
                    outputs(i, o);
                }
                if (wi != 0.f) {
#pragma unroll
                    for (int e = 0; e < E; ++e) acc[e] = fmaf(wi, o[e], acc[e]);
                }
            }
        }
        const int tok = j.row0 + r / p.group, h = j.hk * p.group + r % p.group;
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

int paged_join_launch(const PagedParams& p, const PagedWorkspace* ws, const int* rows, int count, int G, int dtype, cudaStream_t s) {
    JoinSet set{};
    int most = 0;
    for (int i = 0; i < count; ++i) {
        set.ws[i] = ws[i];
        set.rows[i] = rows[i];
        most = rows[i] > most ? rows[i] : most;
    }
    // an item of many rows is shared by several blocks
    const dim3 grid(unsigned(G), unsigned(most > 16 ? 16 : 2), unsigned(count));
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
