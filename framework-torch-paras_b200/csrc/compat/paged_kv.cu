// The paged cache's writer and reader (include/paras_b200.h, "paged key / value cache"): HBM-bound copies of rows of D
// elements between ragged token tensors and pages, with the 8-bit rows' rounding in the same pass.
//
//   write   e = smallest exponent with max|x| * 2^-e <= 448 (clamped), bytes = e4m3(x * 2^-e): the scaling is by a
//           power of two, so the only rounding is the one to e4m3.
//   read    e4m3 * 2^e, exact in every row type.
//
// Sixteen lanes take a row, eight elements each (16 bytes of a 16-bit row), the other half of the warp the matching row
// of V: a 128-element head is one load a lane, the row's maximum four shuffles.  Which sequence a token belongs to is
// found by the warp (warp_count_le) while the row's loads are in flight.
//
// Measured (8 kv heads of 128, pages of 64): write of 4 x 4096 tokens 21.1 us as bf16 (5.9 TB/s), 19.1 us into 8 bits
// (4.9 TB/s; bound by instruction issue, DRAM at 42 % and SM at 64 %; 25.3 us before the rows stayed in pairs of 16 bits); one token for each of 64
// sequences 2.6 us; read of 16 sequences of up to 8192 from 8 bits 61.4 us (5.8 TB/s), of one of 1500 as bf16 3.8 us.
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

// Place of token t in the cache: sequence (-1: none), page and row in it; false when the token has no place there.
template <bool WRITE>
__device__ __forceinline__ bool locate(const KvParams& p, int t, int* page, int* off, int* seq) {
    const int b = warp_count_le(p.cu + 1, p.B, t);
    *seq = -1;
    if (b >= p.B) return false;
    const int c0 = __ldg(p.cu + b);
    if (t < c0) return false;
    *seq = b;
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

// Eight elements of an 8-bit row and its 2^e as fp32.
__device__ __forceinline__ void unpack8(uint2 w, float s, float (&f)[8]) {
    const uint32_t ww[2] = {w.x, w.y};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        uint32_t lo, hi;
        e4m3x4_to_f16x4(ww[i], &lo, &hi);
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo)), b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
        f[4 * i] = a.x * s;
        f[4 * i + 1] = a.y * s;
        f[4 * i + 2] = b.x * s;
        f[4 * i + 3] = b.y * s;
    }
}
// Eight elements of a row as the writer holds them: their largest magnitude and their 8-bit form.  16-bit elements stay in
// pairs: magnitudes and maxima are taken two at a time, and the product by a power of two is exact there too (an fp16 value
// that becomes subnormal is far below half of e4m3's smallest and rounds to zero by either way).
template <typename T>
struct Lane8 {
    uint32_t w[4];
    __device__ __forceinline__ void load(const T* p) { *reinterpret_cast<uint4*>(w) = __ldcs(reinterpret_cast<const uint4*>(p)); }
    __device__ __forceinline__ void clear() { w[0] = w[1] = w[2] = w[3] = 0u; }
    __device__ __forceinline__ void store(T* p) const { __stcs(reinterpret_cast<uint4*>(p), *reinterpret_cast<const uint4*>(w)); }
};
template <>
struct Lane8<float> {
    float f[8];
    __device__ __forceinline__ void load(const float* p) { load_row<float, 8>(p, f); }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = 0.f;
    }
    __device__ __forceinline__ void store(float* p) const {
#pragma unroll
        for (int i = 0; i < 2; ++i) __stcs(reinterpret_cast<float4*>(p) + i, make_float4(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]));
    }
};
template <typename T> struct Pair;
template <> struct Pair<__half> {
    using V = __half2;
    static __device__ __forceinline__ float value(uint32_t h) { return __half2float(__ushort_as_half(uint16_t(h))); }
    static __device__ __forceinline__ uint32_t scaled(uint32_t w, int e) {       // two e4m3 of w * 2^e, -7 <= e <= 15
        const uint32_t s = uint32_t(e + 15) * 0x04000400u;
        const __half2 v = __hmul2(*reinterpret_cast<const __half2*>(&w), *reinterpret_cast<const __half2*>(&s));
        uint16_t r;
        asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(r) : "r"(*reinterpret_cast<const uint32_t*>(&v)));
        return r;
    }
};
template <> struct Pair<__nv_bfloat16> {
    using V = __nv_bfloat162;
    static __device__ __forceinline__ float value(uint32_t h) { return __uint_as_float(h << 16); }
    static __device__ __forceinline__ uint32_t scaled(uint32_t w, int e) {
        const uint32_t s = uint32_t(e + 127) * 0x00800080u;
        const __nv_bfloat162 v = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&w), *reinterpret_cast<const __nv_bfloat162*>(&s));
        const uint32_t b = *reinterpret_cast<const uint32_t*>(&v);
        return pack_e4m3(__uint_as_float(b << 16), __uint_as_float(b & 0xffff0000u));
    }
};
template <typename T>
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    using V = typename Pair<T>::V;
    const V r = __hmax2(*reinterpret_cast<const V*>(&a), *reinterpret_cast<const V*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}
template <typename T>
__device__ __forceinline__ uint2 pack8(const Lane8<T>& v, int e) {
    uint2 r;
    if constexpr (sizeof(T) == 4) {
        const float s = pow2f(e);
        r.x = pack_e4m3(v.f[0] * s, v.f[1] * s) | (pack_e4m3(v.f[2] * s, v.f[3] * s) << 16);
        r.y = pack_e4m3(v.f[4] * s, v.f[5] * s) | (pack_e4m3(v.f[6] * s, v.f[7] * s) << 16);
    } else {
        r.x = __byte_perm(Pair<T>::scaled(v.w[0], e), Pair<T>::scaled(v.w[1], e), 0x5410);
        r.y = __byte_perm(Pair<T>::scaled(v.w[2], e), Pair<T>::scaled(v.w[3], e), 0x5410);
    }
    return r;
}
// The exponent of row (lane mod ROWS) of the half-warp's ROWS rows.  Maxima skip NaN.
template <typename T, int ROWS>
__device__ __forceinline__ int row_exponents(const Lane8<T> (&v)[ROWS]) {
    const int lane = int(threadIdx.x) & 31;
    float mine = 0.f;
    if constexpr (sizeof(T) == 4) {
        float amax[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            amax[r] = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) amax[r] = fmaxf(amax[r], fabsf(v[r].f[e]));
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1)
#pragma unroll
            for (int r = 0; r < ROWS; ++r) amax[r] = fmaxf(amax[r], __shfl_xor_sync(0xffffffffu, amax[r], o));
#pragma unroll
        for (int r = 0; r < ROWS; ++r) mine = (lane & (ROWS - 1)) == r ? amax[r] : mine;
    } else {
        constexpr int kPairs = (ROWS + 1) / 2;
        constexpr uint32_t kAbs = 0x7fff7fffu;
        uint32_t m[2 * kPairs], both[kPairs];        // two rows' maxima in a word
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
            m[r] = max2<T>(max2<T>(v[r].w[0] & kAbs, v[r].w[1] & kAbs), max2<T>(v[r].w[2] & kAbs, v[r].w[3] & kAbs));
        if constexpr (ROWS & 1) m[ROWS] = m[ROWS - 1];
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
            both[i] = max2<T>(__byte_perm(m[2 * i], m[2 * i + 1], 0x5410), __byte_perm(m[2 * i], m[2 * i + 1], 0x7632));
            both[i] = max2<T>(both[i], 0u);          // nothing but NaN counts as zeros
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1)
#pragma unroll
            for (int i = 0; i < kPairs; ++i) both[i] = max2<T>(both[i], __shfl_xor_sync(0xffffffffu, both[i], o));
        uint32_t w = both[0];
#pragma unroll
        for (int i = 1; i < kPairs; ++i) w = (lane & (ROWS - 1)) >> 1 == i ? both[i] : w;
        mine = Pair<T>::value(lane & 1 ? w >> 16 : w & 0xffffu);
    }
    return row_exponent(mine);
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 8 / Vec16<T>::N; ++i) {
        Vec16<T> w;
#pragma unroll
        for (int e = 0; e < Vec16<T>::N; ++e) w.v[e] = from_f32<T>(f[i * Vec16<T>::N + e]);
        st16_stream(p + i * Vec16<T>::N, w);
    }
}

// Which rows a half-warp looks after: `half` 0 is K, 1 is V; strides are selected one by one (a pointer into the
// parameters would copy them to local memory).
template <typename T>
struct RowMap {
    T* row;                  // the token's row of head 0
    int64_t row_head;
    char* cache;
    int64_t cache_page, cache_head, cache_off;
    uint8_t* exps;
    int64_t exp_page, exp_head, exp_off;
    __device__ __forceinline__ RowMap(const KvParams& p, int half, int t) {
        row = reinterpret_cast<T*>(half ? p.v : p.k) + int64_t(t) * (half ? p.vs[0] : p.ks[0]);
        row_head = half ? p.vs[1] : p.ks[1];
        cache = half ? p.cv : p.ck;
        cache_page = half ? p.cvs[0] : p.cks[0];
        cache_head = half ? p.cvs[1] : p.cks[1];
        cache_off = half ? p.cvs[2] : p.cks[2];
        exps = half ? p.ev : p.ek;
        exp_page = half ? p.evs[0] : p.eks[0];
        exp_head = half ? p.evs[1] : p.eks[1];
        exp_off = half ? p.evs[2] : p.eks[2];
    }
};

// Rows of at most 128 elements, whole and aligned in 16-byte units (8 in an 8-bit cache): a lane holds its eight elements
// of ROWS heads, all loaded before the token's place is looked up.
template <typename T, bool CACHE8, int ROWS>
__global__ void __launch_bounds__(kWarps * 32)
paged_kv_write_kernel(const KvParams p) {
    const int lane = threadIdx.x & 31, half = lane >> 4, d = (lane & 15) * 8;
    const int64_t unit = int64_t(blockIdx.x) * kWarps + (threadIdx.x >> 5);
    const int groups = (p.Hkv + ROWS - 1) / ROWS;
    if (unit >= int64_t(p.T) * groups) return;
    const int t = int(unit / groups), h0 = int(unit - int64_t(t) * groups) * ROWS;
    const RowMap<T> m(p, half, t);
    const int heads = min(ROWS, p.Hkv - h0);
    Lane8<T> v[ROWS];
    const T* row = m.row + int64_t(h0) * m.row_head + d;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        v[r].clear();
        if (d < p.D && r < heads) v[r].load(row);
        row += m.row_head;
    }
    int page = 0, off = 0, b = 0;
    if (!locate<true>(p, t, &page, &off, &b) || uint32_t(page) >= uint32_t(p.pages)) return;
    const int64_t at = int64_t(page) * m.cache_page + int64_t(off) * m.cache_off + int64_t(h0) * m.cache_head + d;
    if constexpr (CACHE8) {
        static_assert((ROWS & (ROWS - 1)) == 0 && ROWS <= 16, "a lane per row's exponent");
        const int ex = row_exponents<T, ROWS>(v), r = lane & 15;
        if (r < ROWS && r < heads)
            m.exps[int64_t(page) * m.exp_page + int64_t(h0 + r) * m.exp_head + int64_t(off) * m.exp_off] = uint8_t(ex + 127);
        char* to = m.cache + at;
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            const int e = __shfl_sync(0xffffffffu, ex, i, 16);
            if (d < p.D && i < heads) *reinterpret_cast<uint2*>(to) = pack8<T>(v[i], -e);
            to += m.cache_head;
        }
    } else {
        T* to = reinterpret_cast<T*>(m.cache) + at;
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            if (d < p.D && r < heads) v[r].store(to);
            to += m.cache_head;
        }
    }
}

template <typename T, bool CACHE8, int ROWS>
__global__ void __launch_bounds__(kWarps * 32)
paged_kv_read_kernel(const KvParams p) {
    const int lane = threadIdx.x & 31, half = lane >> 4, d = (lane & 15) * 8;
    const int64_t unit = int64_t(blockIdx.x) * kWarps + (threadIdx.x >> 5);
    const int groups = (p.Hkv + ROWS - 1) / ROWS;
    if (unit >= int64_t(p.T) * groups) return;
    const int t = int(unit / groups), h0 = int(unit - int64_t(t) * groups) * ROWS;
    int page = 0, off = 0, b = 0;
    const bool have = locate<false>(p, t, &page, &off, &b) && uint32_t(page) < uint32_t(p.pages);
    if (b < 0 || d >= p.D) return;      // a row of no sequence
    const RowMap<T> m(p, half, t);
    const int64_t at = int64_t(page) * m.cache_page + int64_t(off) * m.cache_off + d;
    const int64_t eat = int64_t(page) * m.exp_page + int64_t(off) * m.exp_off;
    uint2 w[CACHE8 ? ROWS : 1];
    float s[CACHE8 ? ROWS : 1], f[CACHE8 ? 1 : ROWS][8];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        const bool live = have && h0 + r < p.Hkv;
        if constexpr (CACHE8) {
            w[r] = make_uint2(0, 0);
            s[r] = 0.f;
            if (live) {
                w[r] = __ldcs(reinterpret_cast<const uint2*>(m.cache + at + int64_t(h0 + r) * m.cache_head));
                s[r] = exp_byte(m.exps[eat + int64_t(h0 + r) * m.exp_head]);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) f[r][e] = 0.f;
            if (live) load_row<T, 8>(reinterpret_cast<const T*>(m.cache) + at + int64_t(h0 + r) * m.cache_head, f[r]);
        }
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        if (h0 + r >= p.Hkv) break;
        T* out = m.row + int64_t(h0 + r) * m.row_head + d;
        if constexpr (CACHE8) {
            unpack8(w[r], s[r], f[0]);
            store8(out, f[0]);
        } else {
            store8(out, f[r]);
        }
    }
}

// Any row length and alignment, an element at a time: 16 lanes a row as above.
template <typename T, bool CACHE8, bool WRITE>
__global__ void __launch_bounds__(kWarps * 32)
paged_kv_any_kernel(const KvParams p) {
    const int lane = threadIdx.x & 31, half = lane >> 4, l16 = lane & 15;
    const int64_t unit = int64_t(blockIdx.x) * kWarps + (threadIdx.x >> 5);
    if (unit >= int64_t(p.T) * p.Hkv) return;
    const int t = int(unit / p.Hkv), h = int(unit - int64_t(t) * p.Hkv);
    int page = 0, off = 0, b = 0;
    const bool have = locate<WRITE>(p, t, &page, &off, &b) && uint32_t(page) < uint32_t(p.pages);
    if (b < 0 || (WRITE && !have)) return;
    const RowMap<T> m(p, half, t);
    T* row = m.row + int64_t(h) * m.row_head;
    const int64_t at = have ? int64_t(page) * m.cache_page + int64_t(h) * m.cache_head + int64_t(off) * m.cache_off : 0;
    const int64_t eat = have && CACHE8 ? int64_t(page) * m.exp_page + int64_t(h) * m.exp_head + int64_t(off) * m.exp_off : 0;
    if constexpr (WRITE) {
        float s = 1.f;
        if constexpr (CACHE8) {
            float amax = 0.f;
            for (int d = l16; d < p.D; d += 16) amax = fmaxf(amax, fabsf(to_f32<T>(row[d])));
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
            const int ex = row_exponent(amax);
            s = pow2f(-ex);
            if (l16 == 0) m.exps[eat] = uint8_t(ex + 127);
        }
        for (int d = l16; d < p.D; d += 16) {
            if constexpr (CACHE8) reinterpret_cast<uint8_t*>(m.cache)[at + d] = uint8_t(pack_e4m3(to_f32<T>(row[d]) * s, 0.f));
            else reinterpret_cast<T*>(m.cache)[at + d] = row[d];
        }
    } else {
        const float s = CACHE8 && have ? exp_byte(m.exps[eat]) : 0.f;
        for (int d = l16; d < p.D; d += 16) {
            float f = 0.f;
            if (have) {
                if constexpr (CACHE8) f = e4m3_to_f32(reinterpret_cast<const uint8_t*>(m.cache)[at + d]) * s;
                else f = to_f32<T>(reinterpret_cast<const T*>(m.cache)[at + d]);
            }
            row[d] = from_f32<T>(f);
        }
    }
}

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
bool multiples(const int64_t* s, int n, int64_t of) {
    for (int i = 0; i < n; ++i)
        if (s[i] % of) return false;
    return true;
}

template <bool WRITE, typename T, bool CACHE8>
void launch(const KvParams& p, bool vec, int sms, cudaStream_t s) {
    const int64_t rows = int64_t(p.T) * p.Hkv;
    auto go = [&](auto kernel, int64_t warps) { kernel<<<unsigned((warps + kWarps - 1) / kWarps), kWarps * 32, 0, s>>>(p); };
    if (!vec) return go(paged_kv_any_kernel<T, CACHE8, WRITE>, rows);
    // Several heads a warp: the look-up of the token's place is shared and more loads are in flight.  4 x 4096 bf16 tokens of
    // 8 heads into an 8-bit cache: 19.1 us with four heads a warp, 26.0 with two, 19.0 with eight (which costs short rows
    // more: 4 x 2048 of 4 heads of 64 take 6.0, 8.0, 7.2 us), 46.2 with one; 256 rows 2.6 us either way.  A reader waits for
    // page numbers before its loads and is slower at few rows: 256 rows 2.4 us with one head a warp, 3.3 with eight; 2048
    // rows 2.9 and 3.3; 8192 rows 4.8 and 3.8; 16000 rows 7.2 and 4.4 (16-bit: 2.4 / 2.9, 2.7 / 2.9, 3.9 / 3.4, 6.2 / 4.3).
    constexpr int kMany = WRITE ? 4 : 8;
    const bool many = p.Hkv > 1 && (WRITE || rows >= int64_t(sms) * 32);
    const int64_t warps = many ? int64_t(p.T) * ((p.Hkv + kMany - 1) / kMany) : rows;
    if constexpr (WRITE) many ? go(paged_kv_write_kernel<T, CACHE8, kMany>, warps) : go(paged_kv_write_kernel<T, CACHE8, 1>, warps);
    else many ? go(paged_kv_read_kernel<T, CACHE8, kMany>, warps) : go(paged_kv_read_kernel<T, CACHE8, 1>, warps);
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
    const bool vec = c.D % 8 == 0 && c.D <= 128 && aligned(a.k, 16) && aligned(a.v, 16) && aligned(c.k, cache8 ? 8 : 16) &&
                     aligned(c.v, cache8 ? 8 : 16) && multiples(a.k_strides, 2, unit) && multiples(a.v_strides, 2, unit) &&
                     multiples(c.k_strides, 3, cunit) && multiples(c.v_strides, 3, cunit);
    cudaStream_t s = pick_stream(g, a.stream);
    auto go = [&](auto row) {
        using T = decltype(row);
        cache8 ? launch<WRITE, T, true>(p, vec, g->sm_count, s) : launch<WRITE, T, false>(p, vec, g->sm_count, s);
    };
    switch (a.dtype) {
        case PARAS_F32: go(float()); break;
        case PARAS_BF16: go(__nv_bfloat16()); break;
        default: go(__half()); break;
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
    if (int64_t(c.max_pages) * c.page > kMostPositions)
        return fail(PARAS_E_INVALID, "%s: max_pages * page exceeds 2^31 - 256 positions", what);
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
