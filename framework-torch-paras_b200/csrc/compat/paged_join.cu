// What the streaming attention kernels over a paged cache share beside their loops: the TMA maps of cache and queries,
// and the kernel that joins the partial results of items cut between CTAs.
#include "paged_attn.cuh"
#include "tc_prims.cuh"
#include "tma_host.cuh"

namespace pb {
namespace {

constexpr int kJoinThreads = 256;

// out = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s over the parts s of an item, in the order of the CTAs: a warp per
// row, the head dim over its lanes.  The parts were written a moment ago and lie in L2; few items are cut, so the
// launch itself is most of its cost: it is launched early and waits for the streaming kernel's memory.
template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads)
paged_join_kernel(const PagedParams p, const PagedWorkspace ws, int rows_per_slot) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const PagedJoin j = ws.join[blockIdx.x];
    if (j.first_slot < 0) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rows = j.nq * p.group, parts = j.last_cta - int(blockIdx.x) + 1;
    constexpr int E = D / 32;
    auto slot = [&](int i) { return i == 0 ? j.first_slot : 2 * (int(blockIdx.x) + i); };
    for (int r = blockIdx.y * (kJoinThreads / 32) + warp; r < rows; r += gridDim.y * (kJoinThreads / 32)) {
        float M = -INFINITY;
        for (int i = lane; i < parts; i += 32) M = fmaxf(M, __ldcg(&ws.ml[size_t(slot(i)) * rows_per_slot + r]).x);
        M = warp_max(M);
        float l = 0.f, acc[E];
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = 0.f;
        if (M != -INFINITY) {
#pragma unroll 4
            for (int i = 0; i < parts; ++i) {
                const size_t at = size_t(slot(i)) * rows_per_slot + r;
                const float2 ml = __ldcg(&ws.ml[at]);
                if (ml.x == -INFINITY) continue;      // a part that saw no key: its outputs may not have been written
                const float w = tc::ex2_approx(ml.x - M);
                l = fmaf(w, ml.y, l);
#pragma unroll
                for (int e = 0; e < E; e += 2) {
                    const float2 o = __ldcg(reinterpret_cast<const float2*>(ws.o + at * D + lane * E + e));
                    acc[e] = fmaf(w, o.x, acc[e]);
                    acc[e + 1] = fmaf(w, o.y, acc[e + 1]);
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

int paged_join_launch(const PagedParams& p, const PagedWorkspace& ws, int G, int rows, int dtype, cudaStream_t s) {
    cudaLaunchConfig_t cfg{};
    // an item of many rows is shared by several blocks
    cfg.gridDim = dim3(unsigned(G), unsigned(rows > 16 ? 8 : 1), 1);
    cfg.blockDim = dim3(kJoinThreads, 1, 1);
    cfg.stream = s;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    cudaError_t e;
    if (dtype == PARAS_BF16)
        e = p.D == 128 ? cudaLaunchKernelEx(&cfg, paged_join_kernel<__nv_bfloat16, 128>, p, ws, rows)
                       : cudaLaunchKernelEx(&cfg, paged_join_kernel<__nv_bfloat16, 64>, p, ws, rows);
    else
        e = p.D == 128 ? cudaLaunchKernelEx(&cfg, paged_join_kernel<__half, 128>, p, ws, rows)
                       : cudaLaunchKernelEx(&cfg, paged_join_kernel<__half, 64>, p, ws, rows);
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

int paged_cache_map(CUtensorMap* map, const paras_paged_cache& c, int which) {
    TensorMapEncodeFn fn = tensor_map_encode_fn();
    if (!fn) return fail(PARAS_E_CUDA, "paras_b200: cuTensorMapEncodeTiled is unavailable");
    const bool e8 = c.cache_dtype == PARAS_E4M3;
    const int64_t es = e8 ? 1 : 2;
    const int64_t* st = which ? c.v_strides : c.k_strides;
    const cuuint64_t dims[4] = {cuuint64_t(c.D), cuuint64_t(c.page), cuuint64_t(c.Hkv), cuuint64_t(c.pages)};
    // the stride of a size-1 dim is never used for addressing; keep it a legal multiple of 16 bytes
    const int64_t s2 = c.page > 1 ? st[2] : c.D, s1 = c.Hkv > 1 ? st[1] : s2 * c.page, s0 = c.pages > 1 ? st[0] : s1 * c.Hkv;
    const cuuint64_t strides[3] = {cuuint64_t(s2 * es), cuuint64_t(s1 * es), cuuint64_t(s0 * es)};
    const cuuint32_t box[4] = {cuuint32_t(e8 ? c.D : 64), cuuint32_t(c.page < kTileKeys ? c.page : kTileKeys), 1, 1};
    const cuuint32_t estr[4] = {1, 1, 1, 1};
    const CUtensorMapDataType dt = e8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                      : c.cache_dtype == PARAS_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const CUresult r = fn(map, dt, 4, which ? c.v : c.k, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          e8 && c.D == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
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
