// The paged cache's writer and reader (include/paras_b200.h, "paged key / value cache"): HBM-bound copies of rows of D
// elements between ragged token tensors and pages, with the 8-bit rows' rounding in the same pass.
//
//   write   e = smallest exponent with max|x| * 2^-e <= 448 (clamped), bytes = e4m3(x * 2^-e): the scaling is by a
//           power of two, so the only rounding is the one to e4m3.
//   read    e4m3 * 2^e, exact in every row type.
//
// Sixteen lanes take a row, eight elements each at a time (16 bytes of a 16-bit row), the other half of the warp the
// matching row of V: a 128-element head is one load a lane, the row's maximum four shuffles.  Which sequence a token
// belongs to is found by the warp (warp_count_le) while the row's loads are in flight.
#include "paged_common.cuh"

namespace pb {
namespace {

struct KvParams {
    char *k, *v;                 // token rows
    char *ck, *cv;               // cache
    uint8_t *ek, *ev;
    int64_t ks[2], vs[2], cks[3], cvs[3], eks[3], evs[3];
    const int32_t *table, *kv_lens, *cu;
    int64_t table_stride;
    int pages, page, Hkv, D, B, max_pages, T;
};

constexpr int kWarps = 4;

// Position of token t in its sequence, and the page that holds it; false when the token has none.
template <bool WRITE>
__device__ __forceinline__ bool locate(const KvParams& p, int t, int* page, int* off) {
    const int b = warp_count_le(p.cu + 1, p.B, t);
    if (b >= p.B) return false;
    const int c0 = __ldg(p.cu + b);
    if (t < c0) return false;
    int64_t pos = int64_t(t) - c0;
    if (WRITE) pos += int64_t(__ldg(p.kv_lens + b)) - (int64_t(__ldg(p.cu + b + 1)) - c0);
    if (pos < 0 || pos >= int64_t(p.max_pages) * p.page) return false;
    const int i = int(pos) / p.page;
    *off = int(pos) - i * p.page;
    *page = __ldg(p.table + int64_t(b) * p.table_stride + i);
    return true;
}

// N consecutive elements as fp32
template <typename T, int N>
__device__ __forceinline__ void load_row(const T* p, float (&f)[N]) {
    if constexpr (N == 1) {
        f[0] = to_f32<T>(*p);
    } else {
#pragma unroll
        for (int i = 0; i < N / Vec16<T>::N; ++i) {
            const Vec16<T> v = ld16_stream(p + i * Vec16<T>::N);
#pragma unroll
            for (int e = 0; e < Vec16<T>::N; ++e) f[i * Vec16<T>::N + e] = to_f32<T>(v.v[e]);
        }
    }
}

// N = 8 (rows whole and aligned in 16-byte units, 8 in an 8-bit cache) or 1 (anything).
template <typename T, bool CACHE8, int N>
__global__ void __launch_bounds__(kWarps * 32)
paged_kv_write_kernel(const KvParams p) {
    const int lane = threadIdx.x & 31, half = lane >> 4, l16 = lane & 15;
    const int64_t unit = int64_t(blockIdx.x) * kWarps + (threadIdx.x >> 5);
    if (unit >= int64_t(p.T) * p.Hkv) return;
    const int t = int(unit / p.Hkv), h = int(unit - int64_t(t) * p.Hkv);
    const T* row = half ? reinterpret_cast<const T*>(p.v) + int64_t(t) * p.vs[0] + int64_t(h) * p.vs[1]
                        : reinterpret_cast<const T*>(p.k) + int64_t(t) * p.ks[0] + int64_t(h) * p.ks[1];
    float f[N];
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] = 0.f;
    if (l16 * N < p.D) load_row<T, N>(row + l16 * N, f);
    int page = 0, off = 0;
    if (!locate<true>(p, t, &page, &off) || uint32_t(page) >= uint32_t(p.pages)) return;
    // (strides are selected one by one: a pointer into the parameters would copy them to local memory)
    const int64_t at = int64_t(page) * (half ? p.cvs[0] : p.cks[0]) + int64_t(h) * (half ? p.cvs[1] : p.cks[1]) +
                       int64_t(off) * (half ? p.cvs[2] : p.cks[2]);
    if constexpr (CACHE8) {
        float amax = 0.f;   // (fmaxf skips NaN)
#pragma unroll
        for (int e = 0; e < N; ++e) amax = fmaxf(amax, fabsf(f[e]));
        for (int d = (l16 + 16) * N; d < p.D; d += 16 * N) {
            float g[N];
            load_row<T, N>(row + d, g);
#pragma unroll
            for (int e = 0; e < N; ++e) amax = fmaxf(amax, fabsf(g[e]));
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        const int ex = row_exponent(amax);
        const float s = pow2f(-ex);
        uint8_t* out = reinterpret_cast<uint8_t*>(half ? p.cv : p.ck) + at;
        for (int d = l16 * N; d < p.D; d += 16 * N) {
            if (d >= 16 * N) load_row<T, N>(row + d, f);
            if constexpr (N == 8) {
                uint2 w;
                w.x = pack_e4m3(f[0] * s, f[1] * s) | (pack_e4m3(f[2] * s, f[3] * s) << 16);
                w.y = pack_e4m3(f[4] * s, f[5] * s) | (pack_e4m3(f[6] * s, f[7] * s) << 16);
                *reinterpret_cast<uint2*>(out + d) = w;
            } else {
                out[d] = uint8_t(pack_e4m3(f[0] * s, 0.f));
            }
        }
        if (l16 == 0) {
            (half ? p.ev : p.ek)[int64_t(page) * (half ? p.evs[0] : p.eks[0]) + int64_t(h) * (half ? p.evs[1] : p.eks[1]) +
                                 int64_t(off) * (half ? p.evs[2] : p.eks[2])] = uint8_t(ex + 127);
        }
    } else {
        T* out = reinterpret_cast<T*>(half ? p.cv : p.ck) + at;
        for (int d = l16 * N; d < p.D; d += 16 * N) {
            if (d >= 16 * N) load_row<T, N>(row + d, f);
            if constexpr (N == 8) {
#pragma unroll
                for (int i = 0; i < 8 / Vec16<T>::N; ++i) {
                    Vec16<T> w;
#pragma unroll
                    for (int e = 0; e < Vec16<T>::N; ++e) w.v[e] = from_f32<T>(f[i * Vec16<T>::N + e]);
                    st16(out + d + i * Vec16<T>::N, w);
                }
            } else {
                out[d] = from_f32<T>(f[0]);
            }
        }
    }
}

template <typename T, bool CACHE8, int N>
__global__ void __launch_bounds__(kWarps * 32)
paged_kv_read_kernel(const KvParams p) {
    const int lane = threadIdx.x & 31, half = lane >> 4, l16 = lane & 15;
    const int64_t unit = int64_t(blockIdx.x) * kWarps + (threadIdx.x >> 5);
    if (unit >= int64_t(p.T) * p.Hkv) return;
    const int t = int(unit / p.Hkv), h = int(unit - int64_t(t) * p.Hkv);
    int page = 0, off = 0;
    const int b = warp_count_le(p.cu + 1, p.B, t);
    if (b >= p.B || t < __ldg(p.cu + b)) return;   // a row of no sequence
    const bool have = locate<false>(p, t, &page, &off) && uint32_t(page) < uint32_t(p.pages);
    const int64_t at = have ? int64_t(page) * (half ? p.cvs[0] : p.cks[0]) + int64_t(h) * (half ? p.cvs[1] : p.cks[1]) +
                                  int64_t(off) * (half ? p.cvs[2] : p.cks[2]) : 0;
    T* row = half ? reinterpret_cast<T*>(p.v) + int64_t(t) * p.vs[0] + int64_t(h) * p.vs[1]
                  : reinterpret_cast<T*>(p.k) + int64_t(t) * p.ks[0] + int64_t(h) * p.ks[1];
    float s = 0.f;
    if (CACHE8 && have) {
        s = exp_byte((half ? p.ev : p.ek)[int64_t(page) * (half ? p.evs[0] : p.eks[0]) + int64_t(h) * (half ? p.evs[1] : p.eks[1]) +
                                          int64_t(off) * (half ? p.evs[2] : p.eks[2])]);
    }
    for (int d = l16 * N; d < p.D; d += 16 * N) {
        float f[N];
#pragma unroll
        for (int e = 0; e < N; ++e) f[e] = 0.f;
        if (have) {
            if constexpr (CACHE8) {
                const uint8_t* src = reinterpret_cast<const uint8_t*>(half ? p.cv : p.ck) + at + d;
                if constexpr (N == 8) {
                    const uint2 w = __ldcs(reinterpret_cast<const uint2*>(src));
                    const uint32_t ww[2] = {w.x, w.y};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float2 v = e4m3x2_to_f32((ww[i >> 1] >> (16 * (i & 1))) & 0xffffu);
                        f[2 * i] = v.x * s;
                        f[2 * i + 1] = v.y * s;
                    }
                } else {
                    f[0] = e4m3_to_f32(*src) * s;
                }
            } else {
                load_row<T, N>(reinterpret_cast<const T*>(half ? p.cv : p.ck) + at + d, f);
            }
        }
        if constexpr (N == 8) {
#pragma unroll
            for (int i = 0; i < 8 / Vec16<T>::N; ++i) {
                Vec16<T> w;
#pragma unroll
                for (int e = 0; e < Vec16<T>::N; ++e) w.v[e] = from_f32<T>(f[i * Vec16<T>::N + e]);
                st16_stream(row + d + i * Vec16<T>::N, w);
            }
        } else {
            row[d] = from_f32<T>(f[0]);
        }
    }
}

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
bool multiples(const int64_t* s, int n, int64_t of) {
    for (int i = 0; i < n; ++i)
        if (s[i] % of) return false;
    return true;
}

template <bool WRITE, typename T>
void launch(const KvParams& p, bool cache8, bool vec, int blocks, cudaStream_t s) {
    auto go = [&](auto kernel) { kernel<<<blocks, kWarps * 32, 0, s>>>(p); };
    if constexpr (WRITE) {
        if (cache8) vec ? go(paged_kv_write_kernel<T, true, 8>) : go(paged_kv_write_kernel<T, true, 1>);
        else vec ? go(paged_kv_write_kernel<T, false, 8>) : go(paged_kv_write_kernel<T, false, 1>);
    } else {
        if (cache8) vec ? go(paged_kv_read_kernel<T, true, 8>) : go(paged_kv_read_kernel<T, true, 1>);
        else vec ? go(paged_kv_read_kernel<T, false, 8>) : go(paged_kv_read_kernel<T, false, 1>);
    }
}

template <bool WRITE>
int run(const paras_paged_kv_args* args, const char* what) {
    if (!args) return fail(PARAS_E_INVALID, "%s: null args", what);
    const paras_paged_kv_args& a = *args;
    const paras_paged_cache& c = a.cache;
    int st = check_paged_cache(c, a.dtype, what);
    if (st != PARAS_OK) return st;
    if (a.T < 0) return fail(PARAS_E_INVALID, "%s: negative number of rows", what);
    if (int64_t(a.T) * c.Hkv > (int64_t(1) << 32)) return fail(PARAS_E_UNSUPPORTED, "%s: more than 2^32 rows", what);
    DeviceRestore restore;
    Gpu* g = use_gpu(a.gpu, &st);
    if (!g) return st;
    if (a.T == 0 || c.B == 0) return PARAS_OK;
    if (!a.k || !a.v || !a.cu || (WRITE && !a.kv_lens)) return fail(PARAS_E_INVALID, "%s: null pointer", what);
    KvParams p{};
    p.k = static_cast<char*>(a.k); p.v = static_cast<char*>(a.v);
    p.ck = static_cast<char*>(c.k); p.cv = static_cast<char*>(c.v);
    p.ek = c.k_exp; p.ev = c.v_exp;
    for (int i = 0; i < 2; ++i) { p.ks[i] = a.k_strides[i]; p.vs[i] = a.v_strides[i]; }
    for (int i = 0; i < 3; ++i) {
        p.cks[i] = c.k_strides[i]; p.cvs[i] = c.v_strides[i];
        p.eks[i] = c.k_exp_strides[i]; p.evs[i] = c.v_exp_strides[i];
    }
    p.table = c.page_table; p.table_stride = c.table_stride; p.kv_lens = a.kv_lens; p.cu = a.cu;
    p.pages = c.pages; p.page = c.page; p.Hkv = c.Hkv; p.D = c.D; p.B = c.B; p.max_pages = c.max_pages; p.T = a.T;
    const bool cache8 = c.cache_dtype == PARAS_E4M3;
    const int64_t unit = 16 / int64_t(dtype_size(a.dtype));         // elements in 16 bytes of a token row
    const int64_t cunit = cache8 ? 8 : unit;                         // elements in the cache's aligned unit
    const bool vec = c.D % 8 == 0 && aligned(a.k, 16) && aligned(a.v, 16) && aligned(c.k, cache8 ? 8 : 16) &&
                     aligned(c.v, cache8 ? 8 : 16) && multiples(a.k_strides, 2, unit) && multiples(a.v_strides, 2, unit) &&
                     multiples(c.k_strides, 3, cunit) && multiples(c.v_strides, 3, cunit);
    const int blocks = int((int64_t(a.T) * c.Hkv + kWarps - 1) / kWarps);
    cudaStream_t s = pick_stream(g, a.stream);
    switch (a.dtype) {
        case PARAS_F32: launch<WRITE, float>(p, cache8, vec, blocks, s); break;
        case PARAS_BF16: launch<WRITE, __nv_bfloat16>(p, cache8, vec, blocks, s); break;
        default: launch<WRITE, __half>(p, cache8, vec, blocks, s); break;
    }
    PB_LAUNCH_CHECK(what);
    return PARAS_OK;
}

}  // namespace

int check_paged_cache(const paras_paged_cache& c, int dtype, const char* what) {
    if (dtype != PARAS_F32 && dtype != PARAS_BF16 && dtype != PARAS_F16)
        return fail(PARAS_E_UNSUPPORTED, "%s: unsupported dtype %d", what, dtype);
    if (c.cache_dtype != dtype && c.cache_dtype != PARAS_E4M3)
        return fail(PARAS_E_INVALID, "%s: the cache has to have the rows' type or be 8-bit (e4m3)", what);
    if (c.pages < 0 || c.Hkv < 0 || c.B < 0 || c.max_pages < 0)
        return fail(PARAS_E_INVALID, "%s: negative size", what);
    if (c.page < 1 || c.page > 65536) return fail(PARAS_E_INVALID, "%s: a page holds 1 to 65536 positions", what);
    if (c.D < 1 || c.D > 256) return fail(PARAS_E_UNSUPPORTED, "%s: head dim %d is not within 1..256", what, c.D);
    if (c.Hkv < 1) return fail(PARAS_E_INVALID, "%s: no kv heads", what);
    if (int64_t(c.max_pages) * c.page > INT32_MAX)
        return fail(PARAS_E_INVALID, "%s: max_pages * page exceeds 2^31 - 1 positions", what);
    if (c.B > 0 && c.max_pages > 0 && !c.page_table) return fail(PARAS_E_INVALID, "%s: null page table", what);
    if (c.pages > 0 && (!c.k || !c.v)) return fail(PARAS_E_INVALID, "%s: null cache", what);
    if (c.cache_dtype == PARAS_E4M3 && c.pages > 0 && (!c.k_exp || !c.v_exp))
        return fail(PARAS_E_INVALID, "%s: an 8-bit cache needs its exponent bytes", what);
    return PARAS_OK;
}

}  // namespace pb

extern "C" {

int paras_b200_paged_kv_write(const paras_paged_kv_args* args) {
    pb::NvtxRange range("paras_b200_paged_kv_write");
    return pb::run<true>(args, "paras paged_kv_write");
}

int paras_b200_paged_kv_read(const paras_paged_kv_args* args) {
    pb::NvtxRange range("paras_b200_paged_kv_read");
    return pb::run<false>(args, "paras paged_kv_read");
}

}  // extern "C"
