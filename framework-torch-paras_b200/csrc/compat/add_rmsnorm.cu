// Residual addition and RMSNorm in one pass, with a 16-bit / fp32 or an 8-bit output, and its gradient
// (include/paras_b200.h, "residual addition and RMSNorm in one pass").  HBM-bound: x and residual are read once, h
// and y written once; composed of add, rms_norm and a quantising pass the same work moves h three times more.
//
//   h = T(x + r)      the sum every later layer sees, so the statistics are taken of the rounded value and the
//                     backward pass needs h alone
//   rstd = 1 / sqrt(mean(h^2) + eps)          sums in fp32 per thread (at most 32 squares each), in double across them;
//                                             a row too large or too small for fp32 squares again, in double
//   y = h * rstd * w                          fp32, rounded once: to T, or to e4m3 of y / scale
//   scale = max(max|y| / 448, 2^-126)         over a row or over 32 / 64 / 128 columns
//
// Backward, with n = h * rstd and a = grad_y * w:
//   grad_x = rstd * (a - n * mean(a * n)) + grad_h          grad_w = sum over rows of grad_y * n
// evaluated in this order, in which everything but the result is near grad_y's size whatever h's is.
//
// Measured, bf16: 16384 x 4096 forward 81 us (6.65 TB/s), with 8-bit output by 128 columns 72 us (6.6 TB/s), backward 88 us
// (6.1 TB/s); 64 x 4096 with 8-bit output 2.9 us; 8192 x 5000 forward 51 us and backward 63 us with grad_w; rows that are summed again
// in double only where they occur.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "paged_common.cuh"
#include "tc_prims.cuh"

namespace pb {
namespace {

struct NormParams {
    const void *x, *r, *w;
    void *h, *y;        // y: T, or e4m3 bytes
    float *rstd, *scales;
    int64_t rows, H;
    int64_t groups;     // scales per row
    int group;          // columns per scale, 0 = the row
    double eps;
};

// A row in 32-bit words of E elements: conversions and roundings work on whole words (element by element they, not the
// memory, bound the 16-bit kernels: 4.6 of 6.5 TB/s).
template <typename T> struct Word;
template <> struct Word<float> {
    static constexpr int E = 1;
    static __device__ __forceinline__ void get(uint32_t w, float (&f)[1]) { f[0] = __uint_as_float(w); }
    static __device__ __forceinline__ uint32_t put(const float (&f)[1]) { return __float_as_uint(f[0]); }
    static __device__ __forceinline__ uint32_t add(uint32_t a, uint32_t b) { return __float_as_uint(__uint_as_float(a) + __uint_as_float(b)); }
    static constexpr uint32_t kOnes = 0x3f800000u;
};
template <> struct Word<__nv_bfloat16> {
    static constexpr int E = 2;
    static __device__ __forceinline__ void get(uint32_t w, float (&f)[2]) {
        f[0] = __uint_as_float(w << 16);
        f[1] = __uint_as_float(w & 0xffff0000u);
    }
    static __device__ __forceinline__ uint32_t put(const float (&f)[2]) { return tc::pack16<true>(f[0], f[1]); }
    static __device__ __forceinline__ uint32_t add(uint32_t a, uint32_t b) {
        const __nv_bfloat162 r = __hadd2_rn(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
    static constexpr uint32_t kOnes = 0x3f803f80u;
};
template <> struct Word<__half> {
    static constexpr int E = 2;
    static __device__ __forceinline__ void get(uint32_t w, float (&f)[2]) {
        const float2 r = __half22float2(*reinterpret_cast<const __half2*>(&w));
        f[0] = r.x;
        f[1] = r.y;
    }
    static __device__ __forceinline__ uint32_t put(const float (&f)[2]) { return tc::pack16<false>(f[0], f[1]); }
    static __device__ __forceinline__ uint32_t add(uint32_t a, uint32_t b) {
        const __half2 r = __hadd2_rn(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
    static constexpr uint32_t kOnes = 0x3c003c00u;
};
struct Quad { uint32_t w[4]; };     // 16 bytes of a row
__device__ __forceinline__ Quad load_quad(const void* p, int64_t i) {
    Quad q;
    *reinterpret_cast<uint4*>(&q) = __ldcs(static_cast<const uint4*>(p) + i);
    return q;
}
__device__ __forceinline__ Quad load_quad_kept(const void* p, int64_t i) {
    Quad q;
    *reinterpret_cast<uint4*>(&q) = __ldg(static_cast<const uint4*>(p) + i);
    return q;
}
__device__ __forceinline__ void store_quad(void* p, int64_t i, const Quad& q) {
    __stcs(static_cast<uint4*>(p) + i, *reinterpret_cast<const uint4*>(&q));
}

// The 8-bit form multiplies by reciprocals, each rounded once: a y within 2^-23 of the border between two e4m3 steps may fall on the
// other one.
constexpr float kScaleMin = 1.1754943508222875e-38f;   // 2^-126
__device__ __forceinline__ float scale_of(float amax) { return fmaxf(amax * (1.0f / 448.0f), kScaleMin); }

// Squares are summed in fp32 first, which is right unless magnitudes reach 2^63 (infinite squares, rstd = 0) or the mean square
// with eps lies below 2^-100 (a square is off by up to 2^-150).  Such a row is told by its rstd and summed again in double.
__device__ __forceinline__ bool fp32_squares_fail(float rstd) { return !(rstd > 0.f && rstd <= 1125899906842624.f); }      // 2^50

// The squares of a thread's pieces of `N` consecutive elements of a row; not inlined, so that the usual path keeps its registers.
template <typename T, int N>
__device__ __noinline__ double squares_in_double(const T* row, int H, int tid, int threads) {
    double sum = 0.0;
#pragma unroll 1
    for (int j = tid * N; j < H; j += threads * N)
#pragma unroll 1
        for (int e = 0; e < N; ++e) {
            const double f = to_f32<T>(row[j + e]);
            sum += f * f;
        }
    return sum;
}

// TPR threads hold a row in registers, V vectors of 16 bytes each (rows whole and aligned in such vectors).
// (blocks an SM: as many as the registers that a row of V vectors takes leave room for; with two registers more a thread rows of 200
// bf16 columns take 33.7 us for 30.8)
constexpr int rows_blocks(int tpr, int v, bool quant) {
    return tpr > 128 ? 1024 / tpr : tpr == 32 && v == 1 ? (quant ? 10 : 12) : v <= 2 && !quant ? 10 : 8;
}
template <typename T, int TPR, int V, bool QUANT>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR, rows_blocks(TPR, V, QUANT))
add_rmsnorm_rows_kernel(const NormParams p) {
    using W = Word<T>;
    constexpr int E = W::E, N = 4 * E;
    constexpr int kRows = TPR < 128 ? 128 / TPR : 1;
    constexpr int kW = TPR / 32;
    static_assert(TPR % 32 == 0, "a row takes whole warps");
    __shared__ double red[kW > 1 ? kW : 1];
    __shared__ float redm[kW > 1 ? kW : 1];
    const int tid = threadIdx.x % TPR, lane = threadIdx.x & 31, warp = tid >> 5;
    const int64_t row = int64_t(blockIdx.x) * kRows + threadIdx.x / TPR;
    if (row >= p.rows) return;      // (whole warps leave: with several rows a block, a row is one warp)
    const int nvec = int(p.H / N);
    const int64_t at = row * nvec + tid;
    Quad hv[V], wv[V];
    {
        Quad rv[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (i * TPR + tid < nvec) {
                hv[i] = load_quad(p.x, at + i * TPR);
                if (p.r) rv[i] = load_quad(p.r, at + i * TPR);
            }
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int c = i * TPR + tid;
            if (p.w && c < nvec) wv[i] = load_quad_kept(p.w, c);
            else wv[i] = Quad{{W::kOnes, W::kOnes, W::kOnes, W::kOnes}};
        }
        if (p.r) {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (i * TPR + tid < nvec) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) hv[i].w[k] = W::add(hv[i].w[k], rv[i].w[k]);
                    store_quad(p.h, at + i * TPR, hv[i]);
                }
        }
    }
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (i * TPR + tid < nvec) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float f[E];
                W::get(hv[i].w[k], f);
#pragma unroll
                for (int e = 0; e < E; ++e) ss = fmaf(f[e], f[e], ss);
            }
        }
    auto rstd_of = [&](double part) {
        part = warp_sum(part);
        if constexpr (kW > 1) {
            if (lane == 0) red[warp] = part;
            __syncthreads();
            part = 0.0;
#pragma unroll
            for (int i = 0; i < kW; ++i) part += red[i];
        }
        return float(1.0 / sqrt(part / double(p.H) + p.eps));
    };
    float rstd = rstd_of(double(ss));
    if (fp32_squares_fail(rstd)) {       // (the same for the whole row, which each thread reads as it wrote it)
        if constexpr (kW > 1) __syncthreads();
        rstd = rstd_of(squares_in_double<T, N>(static_cast<const T*>(p.r ? p.h : p.x) + row * p.H, int(p.H), tid, TPR));
    }
    if (p.rstd && tid == 0) p.rstd[row] = rstd;
    // y of word k of vector i.  (The 8-bit form needs it twice, for the maxima and for the result: keeping it would cost 32
    // registers and with them loads in flight.)
    auto yv = [&](int i, int k, float (&y)[E]) {
        float f[E], w[E];
        W::get(hv[i].w[k], f);
        W::get(wv[i].w[k], w);
#pragma unroll
        for (int e = 0; e < E; ++e) y[e] = f[e] * rstd * w[e];
    };
    if constexpr (!QUANT) {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i * TPR + tid < nvec) {
                Quad o;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float y[E];
                    yv(i, k, y);
                    o.w[k] = W::put(y);
                }
                store_quad(p.y, at + i * TPR, o);
            }
    } else {
        float amax[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            amax[i] = 0.f;
            if (i * TPR + tid < nvec) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float y[E];
                    yv(i, k, y);
#pragma unroll
                    for (int e = 0; e < E; ++e) amax[i] = fmaxf(amax[i], fabsf(y[e]));
                }
            }
        }
        if (p.group == 0) {
            float m = 0.f;
#pragma unroll
            for (int i = 0; i < V; ++i) m = fmaxf(m, amax[i]);
            m = warp_max(m);
            if constexpr (kW > 1) {
                if (lane == 0) redm[warp] = m;
                __syncthreads();
                m = 0.f;
#pragma unroll
                for (int i = 0; i < kW; ++i) m = fmaxf(m, redm[i]);
            }
#pragma unroll
            for (int i = 0; i < V; ++i) amax[i] = m;
            if (tid == 0) p.scales[row] = scale_of(m);
        } else {
            const int gl = p.group / N;    // lanes of a group: 4 .. 32, a power of two
            const int sh = 31 - __clz(gl);
            for (int o = gl >> 1; o > 0; o >>= 1) {
#pragma unroll
                for (int i = 0; i < V; ++i) amax[i] = fmaxf(amax[i], __shfl_xor_sync(0xffffffffu, amax[i], o));
            }
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int c = i * TPR + tid;
                if (c < nvec && (c & (gl - 1)) == 0) p.scales[row * p.groups + (c >> sh)] = scale_of(amax[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (i * TPR + tid >= nvec) continue;
            const float inv = 1.0f / scale_of(amax[i]);
            uint32_t b[E];
#pragma unroll
            for (int x = 0; x < E; ++x) {       // four elements: 4 / E words
                float f[4];
#pragma unroll
                for (int k = 0; k < 4 / E; ++k) {
                    float y[E];
                    yv(i, x * (4 / E) + k, y);
#pragma unroll
                    for (int e = 0; e < E; ++e) f[k * E + e] = y[e] * inv;
                }
                b[x] = pack_e4m3(f[0], f[1]) | (pack_e4m3(f[2], f[3]) << 16);
            }
            if constexpr (E == 2) __stcs(static_cast<uint2*>(p.y) + at + i * TPR, make_uint2(b[0], b[1]));
            else __stcs(static_cast<uint32_t*>(p.y) + at + i * TPR, b[0]);
        }
    }
}

// Rows that are not whole 16-byte vectors, or not aligned: TPR threads hold a row in registers as single columns, thread t
// columns t, t + TPR, ...  Loads and stores of two bytes a lane, 64 a warp, are half as fast as vectors; rows need not
// start anywhere in particular.
// (48 registers for the rows of up to 256 columns, as without the second sum; 0: left to the compiler)
template <typename T, int TPR, int V, bool QUANT>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR, TPR == 32 && V == 8 ? 10 : 0)
add_rmsnorm_cols_kernel(const NormParams p) {
    constexpr int kW = TPR / 32, kRows = TPR < 128 ? 128 / TPR : 1;
    static_assert(kRows == 1 || kW == 1, "several rows a block: a warp each");
    __shared__ double red[kW];
    __shared__ float redm[QUANT ? kRows : 1][QUANT ? V : 1][kW], inv[QUANT ? kRows : 1][QUANT ? V : 1][kW];
    const int sub = threadIdx.x / TPR, tid = threadIdx.x % TPR, lane = tid & 31, warp = tid >> 5, H = int(p.H);
    const int64_t row = int64_t(blockIdx.x) * kRows + sub, at = row * p.H;
    if (row >= p.rows) return;      // (whole warps, that no barrier waits for)
    auto sync = [] {
        if constexpr (kW == 1) __syncwarp();
        else __syncthreads();
    };
    const T *x = static_cast<const T*>(p.x) + at, *r = static_cast<const T*>(p.r) + at, *w = static_cast<const T*>(p.w);
    T hv[V], rv[V], wv[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int j = i * TPR + tid;
        if (j < H) {
            hv[i] = x[j];
            if (p.r) rv[i] = r[j];
            wv[i] = w ? w[j] : from_f32<T>(1.0f);
        } else {
            hv[i] = wv[i] = from_f32<T>(0.0f);
        }
    }
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int j = i * TPR + tid;
        if (p.r && j < H) {
            hv[i] = from_f32<T>(to_f32<T>(hv[i]) + to_f32<T>(rv[i]));
            static_cast<T*>(p.h)[at + j] = hv[i];
        }
        const float f = to_f32<T>(hv[i]);
        ss = fmaf(f, f, ss);
    }
    auto rstd_of = [&](double part) {
        part = warp_sum(part);
        if constexpr (kW > 1) {
            if (lane == 0) red[warp] = part;
            __syncthreads();
            part = 0.0;
#pragma unroll
            for (int i = 0; i < kW; ++i) part += red[i];
        }
        return float(1.0 / sqrt(part / double(p.H) + p.eps));
    };
    float rstd = rstd_of(double(ss));
    if (fp32_squares_fail(rstd)) {
        if constexpr (kW > 1) __syncthreads();
        double sd = 0.0;
        if constexpr (kW == 1) {      // (a call costs the narrowest rows a tenth; so does this code the others)
#pragma unroll
            for (int i = 0; i < V; ++i) sd += double(to_f32<T>(hv[i])) * double(to_f32<T>(hv[i]));
        } else {
            sd = squares_in_double<T, 1>(static_cast<const T*>(p.r ? p.h : p.x) + at, H, tid, TPR);
        }
        rstd = rstd_of(sd);
    }
    if (p.rstd && tid == 0) p.rstd[row] = rstd;
    auto yv = [&](int i) { return to_f32<T>(hv[i]) * rstd * to_f32<T>(wv[i]); };
    if constexpr (!QUANT) {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i * TPR + tid < H) static_cast<T*>(p.y)[at + i * TPR + tid] = from_f32<T>(yv(i));
    } else {
        float row_inv = 0.f;
        if (p.group == 0) {
            float m = 0.f;
#pragma unroll
            for (int i = 0; i < V; ++i) m = fmaxf(m, fabsf(yv(i)));
            m = warp_max(m);
            if constexpr (kW > 1) {
                if (lane == 0) redm[0][0][warp] = m;
                __syncthreads();
#pragma unroll
                for (int i = 0; i < kW; ++i) m = fmaxf(m, redm[0][0][i]);
            }
            if (tid == 0) p.scales[row] = scale_of(m);
            row_inv = 1.0f / scale_of(m);
        } else {
            // A warp's 32 columns of step i are a group of 32 or a piece of a larger one, whose other pieces are the
            // neighbouring warps', or, where a warp has the row, its neighbouring steps.  A scale is formed once per piece.
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float m = warp_max(fabsf(yv(i)));
                if (lane == 0) redm[sub][i][warp] = m;
            }
            sync();
            const int per = p.group / 32;
            for (int e = tid; e < V * kW; e += TPR) {
                const int first = e & ~(per - 1);
                float m = 0.f;
                for (int k = first; k < min(first + per, V * kW); ++k) m = fmaxf(m, redm[sub][k / kW][k % kW]);
                inv[sub][e / kW][e % kW] = 1.0f / scale_of(m);
                if (e == first && int64_t(e) * 32 < p.H) p.scales[row * p.groups + e / per] = scale_of(m);
            }
            sync();
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int j = i * TPR + tid;
            const float f = p.group ? inv[sub][i][warp] : row_inv;
            if (j < H) static_cast<uint8_t*>(p.y)[at + j] = uint8_t(pack_e4m3(yv(i) * f, 0.f));
        }
    }
}

// Rows too long for registers: a CTA per row, h kept in memory between the passes (L2 holds it).
template <typename T, bool QUANT>
__global__ void __launch_bounds__(256)
add_rmsnorm_any_kernel(const NormParams p) {
    __shared__ double red[8];
    __shared__ float redm[8];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* x = static_cast<const T*>(p.x) + row * p.H;
        const T* r = p.r ? static_cast<const T*>(p.r) + row * p.H : nullptr;
        const T* w = static_cast<const T*>(p.w);
        T* hrow = p.r ? static_cast<T*>(p.h) + row * p.H : nullptr;
        // each thread writes and later re-reads the same columns of h: no barrier between
        auto at = [&](int64_t j) { return to_f32<T>(hrow ? hrow[j] : x[j]); };
        double acc = 0.0;
        for (int64_t j = tid; j < p.H; j += 256) {
            T v = x[j];
            if (r) {
                v = from_f32<T>(to_f32<T>(v) + to_f32<T>(r[j]));
                hrow[j] = v;
            }
            const float f = to_f32<T>(v);
            acc += double(f) * double(f);
        }
        acc = warp_sum(acc);
        if (lane == 0) red[warp] = acc;
        __syncthreads();
        double total = 0.0;
        for (int i = 0; i < 8; ++i) total += red[i];
        const float rstd = float(1.0 / sqrt(total / double(p.H) + p.eps));
        if (p.rstd && tid == 0) p.rstd[row] = rstd;
        auto yv = [&](int64_t j) { return at(j) * rstd * (w ? to_f32<T>(w[j]) : 1.0f); };
        if constexpr (!QUANT) {
            T* y = static_cast<T*>(p.y) + row * p.H;
            for (int64_t j = tid; j < p.H; j += 256) y[j] = from_f32<T>(yv(j));
        } else {
            uint8_t* q = static_cast<uint8_t*>(p.y) + row * p.H;
            if (p.group == 0) {
                float m = 0.f;
                for (int64_t j = tid; j < p.H; j += 256) m = fmaxf(m, fabsf(yv(j)));
                m = warp_max(m);
                if (lane == 0) redm[warp] = m;
                __syncthreads();
                m = 0.f;
                for (int i = 0; i < 8; ++i) m = fmaxf(m, redm[i]);
                if (tid == 0) p.scales[row] = scale_of(m);
                const float inv = 1.0f / scale_of(m);
                for (int64_t j = tid; j < p.H; j += 256) q[j] = uint8_t(pack_e4m3(yv(j) * inv, 0.f));
            } else {
                // a group spans one to four warps: its maximum goes through the warps' own (a column's thread is
                // j mod 256, so the groups of 256 / group different 32-column pieces are side by side)
                for (int64_t j0 = 0; j0 < p.H; j0 += 256) {
                    const int64_t j = j0 + tid;
                    const float f = j < p.H ? yv(j) : 0.f;
                    float m = warp_max(fabsf(f));
                    __syncthreads();
                    if (lane == 0) redm[warp] = m;
                    __syncthreads();
                    const int per = p.group / 32, first = warp / per * per;
                    m = 0.f;
                    for (int i = 0; i < per; ++i) m = fmaxf(m, redm[first + i]);
                    if (j < p.H) {
                        q[j] = uint8_t(pack_e4m3(f * (1.0f / scale_of(m)), 0.f));
                        if (j % p.group == 0) p.scales[row * p.groups + j / p.group] = scale_of(m);
                    }
                }
            }
        }
        __syncthreads();
    }
}

template <typename T, bool QUANT>
void launch_fwd(const NormParams& p, bool vec, cudaStream_t s) {
    constexpr int N = Vec16<T>::N;
    const int64_t nvec = p.H / N;
    // A row stays in registers up to 4 vectors a thread.  Few threads a row leave more rows in flight on an SM; past
    // 32 * 4 vectors a warp would have to hold more than that.  bf16, 67 million elements, 8-bit output by the row: 512 columns
    // 74 us with a warp a row, 139 with four; 1024: 71 and 88; 2048: 75 with four warps, 94 with eight; 4096: 71 and 82;
    // 8192: 71 with eight, 90 with sixteen.  (64 rows gain 0.3 to 0.6 us of 2.9 by twice the threads.)
    auto go = [&](auto kernel, int tpr) {
        const int64_t per = tpr < 128 ? 128 / tpr : 1;
        kernel<<<unsigned((p.rows + per - 1) / per), tpr < 128 ? 128 : tpr, 0, s>>>(p);
    };
    if (vec && nvec <= 32 * 4) {
        if (nvec <= 32) go(add_rmsnorm_rows_kernel<T, 32, 1, QUANT>, 32);
        else if (nvec <= 64) go(add_rmsnorm_rows_kernel<T, 32, 2, QUANT>, 32);
        else go(add_rmsnorm_rows_kernel<T, 32, 4, QUANT>, 32);
    } else if (vec && nvec <= 128 * 4) {
        if (nvec <= 256) go(add_rmsnorm_rows_kernel<T, 128, 2, QUANT>, 128);
        else go(add_rmsnorm_rows_kernel<T, 128, 4, QUANT>, 128);
    } else if (vec && nvec <= 256 * 4) {
        if (nvec <= 768) go(add_rmsnorm_rows_kernel<T, 256, 3, QUANT>, 256);
        else go(add_rmsnorm_rows_kernel<T, 256, 4, QUANT>, 256);
    } else if (vec && nvec <= 1024 * 4) {
        if (nvec <= 2048) go(add_rmsnorm_rows_kernel<T, 512, 4, QUANT>, 512);
        else go(add_rmsnorm_rows_kernel<T, 1024, 4, QUANT>, 1024);
    } else if (p.H <= 256 * 4) {
        // (a warp to 256 columns, 128 threads to 1024)
        if (p.H <= 128) go(add_rmsnorm_cols_kernel<T, 32, 4, QUANT>, 32);
        else if (p.H <= 256) go(add_rmsnorm_cols_kernel<T, 32, 8, QUANT>, 32);
        else if (p.H <= 512) add_rmsnorm_cols_kernel<T, 128, 4, QUANT><<<unsigned(p.rows), 128, 0, s>>>(p);
        else add_rmsnorm_cols_kernel<T, 128, 8, QUANT><<<unsigned(p.rows), 128, 0, s>>>(p);
    } else if (p.H <= 1024 * 16) {
        if (p.H <= 256 * 8) add_rmsnorm_cols_kernel<T, 256, 8, QUANT><<<unsigned(p.rows), 256, 0, s>>>(p);
        else if (p.H <= 256 * 16) add_rmsnorm_cols_kernel<T, 256, 16, QUANT><<<unsigned(p.rows), 256, 0, s>>>(p);
        else if (p.H <= 512 * 16) add_rmsnorm_cols_kernel<T, 512, 16, QUANT><<<unsigned(p.rows), 512, 0, s>>>(p);
        else add_rmsnorm_cols_kernel<T, 1024, 16, QUANT><<<unsigned(p.rows), 1024, 0, s>>>(p);
    } else {
        const int64_t blocks = std::min<int64_t>(p.rows, 148 * 8);
        add_rmsnorm_any_kernel<T, QUANT><<<int(blocks), 256, 0, s>>>(p);
    }
}

// ---- backward --------------------------------------------------------------------------------
// A CTA walks rows of its own; every thread owns the same columns of all of them, so grad_weight is summed in its
// registers and leaves once per CTA (fp32 [parts, H], summed in double by the second kernel: no atomics, one order).
// The three inputs of the next two rows are in flight (cp.async, each thread copying what it will read itself) while
// a row is reduced and written; one row for the longest rows, of which no third stage fits into shared memory.
__host__ __device__ constexpr int bwd_stages(int threads, int v) { return 3 * 3 * threads * v * 16 <= 224 * 1024 ? 3 : 2; }

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT> __device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}

// mean(a * n) is summed as rstd times a sum of a * h, which stays in fp32's range while rstd is within 2^-40 .. 2^40; other rows are
// summed as the definition has it, a product more an element (8192 x 5000 bf16: 62 us this way, 70 with that product for all).
__device__ __forceinline__ bool far_from_one(float rstd) { return !(rstd >= 9.094947017729282e-13f && rstd <= 1099511627776.f); }

// a * n over a thread's pieces of `N` consecutive elements of a row.
template <typename T, int N>
__device__ __forceinline__ float normed_dot(const T* gy, const T* h, const T* w, float rstd, int H, int tid, int threads) {
    float sum = 0.f;
#pragma unroll 1
    for (int j = tid * N; j < H; j += threads * N)
#pragma unroll 1
        for (int e = j; e < j + N; ++e) sum = fmaf(to_f32<T>(gy[e]) * (w ? to_f32<T>(w[e]) : 1.0f), to_f32<T>(h[e]) * rstd, sum);
    return sum;
}
template <typename T, int N>
__device__ __noinline__ float normed_dot_call(const T* gy, const T* h, const T* w, float rstd, int H, int tid, int threads) {
    return normed_dot<T, N>(gy, h, w, rstd, H, tid, threads);
}

struct BwdParams {
    const void *gy, *gh, *h, *w;
    const float* rstd;
    void* gx;
    float* part;       // [gridDim.x, H], null: no grad_weight wanted
    int64_t rows, H;
};

template <typename T, int THREADS, int V>
__global__ void __launch_bounds__(THREADS, 512 / THREADS)
add_rmsnorm_bwd_rows_kernel(const BwdParams p) {
    using W = Word<T>;
    constexpr int E = W::E, N = 4 * E;
    constexpr int kStages = bwd_stages(THREADS, V);
    constexpr uint32_t kOne = THREADS * V * 16, kStage = 3 * kOne;
    extern __shared__ __align__(16) unsigned char ring_raw[];
    __shared__ float red[2][THREADS / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(ring_raw));
    const int nvec = int(p.H / N);
    const uint4 *gy = static_cast<const uint4*>(p.gy), *gh = static_cast<const uint4*>(p.gh), *h = static_cast<const uint4*>(p.h);
    auto issue = [&](int64_t row, int stage) {
        if (row < p.rows) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int c = i * THREADS + tid;
                if (c < nvec) {
                    const uint32_t dst = ring + stage * kStage + uint32_t(c) * 16;
                    const int64_t at = row * nvec + c;
                    copy16(dst, gy + at);
                    copy16(dst + kOne, h + at);
                    if (gh) copy16(dst + 2 * kOne, gh + at);
                }
            }
        }
        copy_commit();
    };
    Quad wv[V];
    float dw[V * N];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int c = i * THREADS + tid;
        if (p.w && c < nvec) wv[i] = load_quad_kept(p.w, c);
        else wv[i] = Quad{{W::kOnes, W::kOnes, W::kOnes, W::kOnes}};
    }
#pragma unroll
    for (int i = 0; i < V * N; ++i) dw[i] = 0.f;
    const float inv_h = 1.0f / float(p.H);
#pragma unroll
    for (int st = 0; st < kStages - 1; ++st) issue(int64_t(blockIdx.x) + int64_t(st) * gridDim.x, st);
    int stage = 0, flip = 0;
    float rr_next = p.rstd[blockIdx.x];
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, flip ^= 1) {
        issue(row + int64_t(kStages - 1) * gridDim.x, stage == 0 ? kStages - 1 : stage - 1);
        const float rr = rr_next;
        rr_next = p.rstd[min(row + int64_t(gridDim.x), p.rows - 1)];
        copy_wait<kStages - 1>();
        const uint4* buf = reinterpret_cast<const uint4*>(ring_raw + stage * kStage);
        stage = stage + 1 == kStages ? 0 : stage + 1;
        Quad g[V], x[V];
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int c = i * THREADS + tid;
            if (c < nvec) {
                *reinterpret_cast<uint4*>(&g[i]) = buf[c];
                *reinterpret_cast<uint4*>(&x[i]) = buf[kOne / 16 + c];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float ge[E], xe[E], we[E];
                    W::get(g[i].w[k], ge);
                    W::get(x[i].w[k], xe);
                    W::get(wv[i].w[k], we);
#pragma unroll
                    for (int e = 0; e < E; ++e) dot = fmaf(ge[e] * we[e], xe[e], dot);
                }
            }
        }
        dot *= rr;
        if (far_from_one(rr)) {
            const T *g0 = reinterpret_cast<const T*>(buf), *x0 = reinterpret_cast<const T*>(buf + kOne / 16), *w0 = static_cast<const T*>(p.w);
            // (4 vectors a thread: a call leaves them in registers, 8192 x 8192 bf16 97 us for 103; fewer are held up by it, 8192 x 5000 71 for 63)
            dot = V == 4 ? normed_dot_call<T, N>(g0, x0, w0, rr, int(p.H), tid, THREADS) : normed_dot<T, N>(g0, x0, w0, rr, int(p.H), tid, THREADS);
        }
        dot = warp_sum(dot);
        if (lane == 0) red[flip][warp] = dot;
        __syncthreads();      // (two buffers in turn: the next row's writes cannot overtake these reads)
        dot = 0.f;
#pragma unroll
        for (int i = 0; i < THREADS / 32; ++i) dot += red[flip][i];
        const float mean = inv_h * dot;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int c = i * THREADS + tid;
            if (c < nvec) {
                Quad o, a{};
                if (gh) *reinterpret_cast<uint4*>(&a) = buf[2 * (kOne / 16) + c];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float ge[E], xe[E], we[E], ae[E], oe[E];
                    W::get(g[i].w[k], ge);
                    W::get(x[i].w[k], xe);
                    W::get(wv[i].w[k], we);
                    W::get(a.w[k], ae);
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const float n = xe[e] * rr;
                        oe[e] = fmaf(fmaf(-n, mean, ge[e] * we[e]), rr, ae[e]);
                        dw[i * N + k * E + e] = fmaf(ge[e], n, dw[i * N + k * E + e]);
                    }
                    o.w[k] = W::put(oe);
                }
                store_quad(p.gx, row * nvec + c, o);
            }
        }
    }
    copy_wait<0>();
    if (p.part) {
        float* part = p.part + int64_t(blockIdx.x) * p.H;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int c = i * THREADS + tid;
            if (c < nvec)
#pragma unroll
                for (int e = 0; e < N; e += 4)
                    *reinterpret_cast<float4*>(part + int64_t(c) * N + e) =
                        make_float4(dw[i * N + e], dw[i * N + e + 1], dw[i * N + e + 2], dw[i * N + e + 3]);
        }
    }
}

// The same for rows that are not whole aligned vectors, a column at a time as in the forward: the next row's values are in
// flight, in registers, while a row is reduced and written.
template <typename T, int THREADS, int V>
__global__ void __launch_bounds__(THREADS < 128 ? 128 : THREADS)
add_rmsnorm_bwd_cols_kernel(const BwdParams p) {
    // below 128 threads a block is several walkers, a warp each, that share nothing
    constexpr int kSubs = THREADS < 128 ? 128 / THREADS : 1;
    static_assert(kSubs == 1 || THREADS == 32, "a walker is a warp or the block");
    __shared__ float red[2][THREADS / 32];
    const int64_t walker = int64_t(blockIdx.x) * kSubs + threadIdx.x / THREADS, walkers = int64_t(gridDim.x) * kSubs;
    const int tid = threadIdx.x % THREADS, lane = tid & 31, warp = tid >> 5, H = int(p.H);
    const T *gy = static_cast<const T*>(p.gy), *gh = static_cast<const T*>(p.gh), *h = static_cast<const T*>(p.h), *w = static_cast<const T*>(p.w);
    const T zero = from_f32<T>(0.f);
    T wv[V], g[V], x[V], a[V], g2[V], x2[V], a2[V];
    float dw[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int j = i * THREADS + tid;
        wv[i] = w && j < H ? w[j] : from_f32<T>(1.0f);
        dw[i] = 0.f;
        g[i] = x[i] = a[i] = zero;
    }
    auto fetch = [&](int64_t row, T (&fg)[V], T (&fx)[V], T (&fa)[V]) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int j = i * THREADS + tid;
            const bool live = j < H && row < p.rows;
            const int64_t at = row * p.H + j;
            fg[i] = live ? gy[at] : zero;
            fx[i] = live ? h[at] : zero;
            fa[i] = live && gh ? gh[at] : zero;
        }
    };
    const float inv_h = 1.0f / float(p.H);
    int flip = 0;
    auto step = [&](int64_t row, const T (&fg)[V], const T (&fx)[V], const T (&fa)[V]) {
        const float rr = p.rstd[row];
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) dot = fmaf(to_f32<T>(fg[i]) * to_f32<T>(wv[i]), to_f32<T>(fx[i]), dot);
        dot *= rr;
        if (far_from_one(rr)) {
            dot = 0.f;
#pragma unroll
            for (int i = 0; i < V; ++i) dot = fmaf(to_f32<T>(fg[i]) * to_f32<T>(wv[i]), to_f32<T>(fx[i]) * rr, dot);
        }
        dot = warp_sum(dot);
        if constexpr (kSubs == 1) {
            if (lane == 0) red[flip][warp] = dot;
            __syncthreads();
            dot = 0.f;
#pragma unroll
            for (int i = 0; i < THREADS / 32; ++i) dot += red[flip][i];
            flip ^= 1;
        }
        const float mean = inv_h * dot;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int j = i * THREADS + tid;
            const float ge = to_f32<T>(fg[i]), n = to_f32<T>(fx[i]) * rr;
            if (j < H) static_cast<T*>(p.gx)[row * p.H + j] = from_f32<T>(fmaf(fmaf(-n, mean, ge * to_f32<T>(wv[i])), rr, to_f32<T>(fa[i])));
            dw[i] = fmaf(ge, n, dw[i]);
        }
    };
    fetch(walker, g, x, a);
    for (int64_t row = walker; row < p.rows; row += 2 * walkers) {
        const int64_t next = row + walkers;
        fetch(next, g2, x2, a2);
        step(row, g, x, a);
        if (next >= p.rows) break;       // (the same for the whole walker)
        fetch(next + walkers, g, x, a);
        step(next, g2, x2, a2);
    }
    if (p.part) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int j = i * THREADS + tid;
            if (j < H) p.part[walker * p.H + j] = dw[i];
        }
    }
}

// Rows too long for registers: grad_x, a CTA per row.
template <typename T>
__global__ void __launch_bounds__(256)
add_rmsnorm_bwd_dx_kernel(const BwdParams p) {
    __shared__ double red[8];
    const int tid = threadIdx.x;
    const T* w = static_cast<const T*>(p.w);
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* gy = static_cast<const T*>(p.gy) + row * p.H;
        const T* h = static_cast<const T*>(p.h) + row * p.H;
        const T* gh = p.gh ? static_cast<const T*>(p.gh) + row * p.H : nullptr;
        double dot = 0.0;
        for (int64_t j = tid; j < p.H; j += 256)
            dot += double(to_f32<T>(gy[j]) * (w ? to_f32<T>(w[j]) : 1.0f)) * double(to_f32<T>(h[j]));
        dot = warp_sum(dot);
        if ((tid & 31) == 0) red[tid >> 5] = dot;
        __syncthreads();
        dot = 0.0;
        for (int i = 0; i < 8; ++i) dot += red[i];
        const float rr = p.rstd[row], mean = float(dot * double(rr) / double(p.H));
        T* out = static_cast<T*>(p.gx) + row * p.H;
        for (int64_t j = tid; j < p.H; j += 256) {
            const float a = to_f32<T>(gy[j]) * (w ? to_f32<T>(w[j]) : 1.0f);
            out[j] = from_f32<T>(fmaf(fmaf(-(to_f32<T>(h[j]) * rr), mean, a), rr, gh ? to_f32<T>(gh[j]) : 0.f));
        }
        __syncthreads();
    }
}
// ... and grad_weight: 32 columns a CTA, the rows over its other 32 threads.
template <typename T>
__global__ void __launch_bounds__(1024)
add_rmsnorm_bwd_dw_kernel(const BwdParams p, T* __restrict__ gw) {
    __shared__ double part[32][33];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int64_t col = int64_t(blockIdx.x) * 32 + tx;
    double acc = 0.0;
    if (col < p.H)
        for (int64_t r = ty; r < p.rows; r += 32)
            acc += double(to_f32<T>(static_cast<const T*>(p.gy)[r * p.H + col])) *
                   double(to_f32<T>(static_cast<const T*>(p.h)[r * p.H + col])) * double(p.rstd[r]);
    part[ty][tx] = acc;
    __syncthreads();
    if (ty == 0 && col < p.H) {
        double t = 0.0;
        for (int i = 0; i < 32; ++i) t += part[i][tx];
        gw[col] = from_f32<T>(float(t));
    }
}
template <typename T>
__global__ void __launch_bounds__(1024)
add_rmsnorm_bwd_dw_sum_kernel(const float* __restrict__ parts, T* __restrict__ gw, int count, int64_t H) {
    __shared__ double sh[32][33];
    const int cx = threadIdx.x & 31, py = threadIdx.x >> 5;
    const int64_t col = int64_t(blockIdx.x) * 32 + cx;
    double acc = 0.0;
    if (col < H) {
#pragma unroll 4
        for (int i = py; i < count; i += 32) acc += double(__ldcs(parts + int64_t(i) * H + col));
    }
    sh[py][cx] = acc;
    __syncthreads();
    if (py == 0 && col < H) {
        double t = 0.0;
#pragma unroll
        for (int i = 0; i < 32; ++i) t += sh[i][cx];
        gw[col] = from_f32<T>(float(t));
    }
}

template <typename T>
int launch_bwd(Gpu* g, BwdParams p, void* gw, bool vec, cudaStream_t s) {
    constexpr int N = Vec16<T>::N;
    const int64_t nvec = p.H / N;
    const int sms = g->sm_count > 0 ? g->sm_count : 148;
    const unsigned dwblocks = unsigned((p.H + 31) / 32);
    const bool cols = !(vec && nvec <= 512 * 4) && p.H <= 1024 * 8;
    if (cols || (vec && nvec <= 512 * 4)) {
        // 32 threads a row to 64 vectors, 64 to 128, then 128, 256 or 512, at most 4 vectors each; the ring (2 or 3 stages of 3
        // inputs) takes at most 9 / 18 / 72 / 144 / 216 KB a CTA; 16 / 8 / 4 / 2 / 1 CTAs share an SM as registers and shared
        // memory allow.  131072 x 512 bf16: 99 us with 32 threads, 114 with 64, 138 with 128; 65536 x 1024: 103, 94, 104.
        // (columns: 32 to 1024 threads, at most 8 columns each)
        const int threads = cols ? (p.H <= 256 ? 32 : p.H <= 1024 ? 128 : p.H <= 2048 ? 256 : p.H <= 4096 ? 512 : 1024) : nvec <= 64 ? 32 : nvec <= 128 ? 64 : nvec <= 128 * 4 ? 128 : nvec <= 256 * 4 ? 256 : 512;
        const int v = cols ? 8 : int((nvec + threads - 1) / threads);
        const size_t ring = cols ? 0 : size_t(bwd_stages(threads, v)) * 3 * threads * v * 16;
        int per_sm = std::max(1, (cols ? 1024 : 512) / threads);
        while (per_sm > 1 && (ring + 1024) * per_sm > 220 * 1024) --per_sm;
        // (few rows: a CTA for four of them rather than more parts of grad_weight)
        const int64_t most = !cols && threads < 128 ? std::min<int64_t>(int64_t(sms) * per_sm, std::max<int64_t>(int64_t(sms) * 4, p.rows / 4))
                                                    : int64_t(sms) * per_sm;
        const int parts = cols && threads == 32 ? int((std::min<int64_t>(p.rows, int64_t(sms) * 32) + 3) / 4 * 4)
                                                : int(std::min<int64_t>(p.rows, most));
        void* scratch = nullptr;
        if (gw) {
            const int st = paras_b200_malloc_async(g->ordinal, size_t(parts) * size_t(p.H) * sizeof(float), s, &scratch);
            if (st != PARAS_OK) return st;
        }
        p.part = static_cast<float*>(scratch);
        cudaError_t err = cudaSuccess;
        auto go = [&](auto kernel) {
            err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(ring));
            if (err == cudaSuccess) kernel<<<parts, threads, ring, s>>>(p);
        };
        auto by_v = [&](auto th) {
            constexpr int TH = decltype(th)::value;
            if (v == 1) go(add_rmsnorm_bwd_rows_kernel<T, TH, 1>);
            else if (v == 2) go(add_rmsnorm_bwd_rows_kernel<T, TH, 2>);
            else if (v == 3) go(add_rmsnorm_bwd_rows_kernel<T, TH, 3>);
            else go(add_rmsnorm_bwd_rows_kernel<T, TH, 4>);
        };
        auto plain = [&](auto kernel) { kernel<<<parts, threads, 0, s>>>(p); };
        if (cols) {
            if (threads == 32) add_rmsnorm_bwd_cols_kernel<T, 32, 8><<<parts / 4, 128, 0, s>>>(p);
            else if (threads == 128) plain(add_rmsnorm_bwd_cols_kernel<T, 128, 8>);
            else if (threads == 256) plain(add_rmsnorm_bwd_cols_kernel<T, 256, 8>);
            else if (threads == 512) plain(add_rmsnorm_bwd_cols_kernel<T, 512, 8>);
            else plain(add_rmsnorm_bwd_cols_kernel<T, 1024, 8>);
        } else if (threads == 32) v == 1 ? go(add_rmsnorm_bwd_rows_kernel<T, 32, 1>) : go(add_rmsnorm_bwd_rows_kernel<T, 32, 2>);
        else if (threads == 64) go(add_rmsnorm_bwd_rows_kernel<T, 64, 2>);
        else if (threads == 128) by_v(std::integral_constant<int, 128>());
        else if (threads == 256) by_v(std::integral_constant<int, 256>());
        else by_v(std::integral_constant<int, 512>());
        if (err == cudaSuccess && gw)
            add_rmsnorm_bwd_dw_sum_kernel<T><<<dwblocks, 1024, 0, s>>>(p.part, static_cast<T*>(gw), parts, p.H);
        if (err == cudaSuccess) err = cudaGetLastError();
        const int st2 = scratch ? paras_b200_free_async(g->ordinal, scratch, s) : PARAS_OK;
        if (err != cudaSuccess) return fail(PARAS_E_CUDA, "paras add_rms_norm_backward: launch failed: %s", cudaGetErrorString(err));
        return st2;
    }
    add_rmsnorm_bwd_dx_kernel<T><<<int(std::min<int64_t>(p.rows, int64_t(sms) * 8)), 256, 0, s>>>(p);
    if (gw) add_rmsnorm_bwd_dw_kernel<T><<<dwblocks, 1024, 0, s>>>(p, static_cast<T*>(gw));
    PB_LAUNCH_CHECK("add_rmsnorm_bwd kernels");
    return PARAS_OK;
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int check_sizes(int64_t rows, int64_t H, int dtype, const char* what) {
    if (rows < 0 || H < 0) return fail(PARAS_E_INVALID, "%s: negative size", what);
    if (rows >= (int64_t(1) << 31) || H >= (int64_t(1) << 31)) return fail(PARAS_E_UNSUPPORTED, "%s: a size exceeds 2^31 - 1", what);
    if (dtype != PARAS_F32 && dtype != PARAS_BF16 && dtype != PARAS_F16)
        return fail(PARAS_E_UNSUPPORTED, "%s: unsupported dtype %d", what, dtype);
    return PARAS_OK;
}

template <bool QUANT>
int forward(int gpu, const void* x, const void* residual, const void* weight, void* h, void* y, float* rstd, float* scales,
            int64_t rows, int64_t H, double eps, int group, int dtype, void* stream, const char* what) {
    int st = check_sizes(rows, H, dtype, what);
    if (st != PARAS_OK) return st;
    if (QUANT && group != 0 && group != 32 && group != 64 && group != 128)
        return fail(PARAS_E_INVALID, "%s: group is %d columns, not 0 (a row), 32, 64 or 128", what, group);
    DeviceRestore restore;
    Gpu* g = use_gpu(gpu, &st);
    if (!g) return st;
    if (rows == 0 || H == 0) return PARAS_OK;
    if (!x || !y || (residual && !h) || (QUANT && !scales)) return fail(PARAS_E_INVALID, "%s: null pointer", what);
    NormParams p{};
    p.x = x; p.r = residual; p.w = weight; p.h = h; p.y = y; p.rstd = rstd; p.scales = scales;
    p.rows = rows; p.H = H; p.eps = eps; p.group = group;
    p.groups = group ? (H + group - 1) / group : 1;
    const int64_t n = 16 / int64_t(dtype_size(dtype));
    const bool vec = H % n == 0 && al16(x) && (!residual || (al16(residual) && al16(h))) && (!weight || al16(weight)) &&
                     (QUANT ? reinterpret_cast<uintptr_t>(y) % 8 == 0 : al16(y));
    cudaStream_t s = pick_stream(g, stream);
    switch (dtype) {
        case PARAS_F32: launch_fwd<float, QUANT>(p, vec, s); break;
        case PARAS_BF16: launch_fwd<__nv_bfloat16, QUANT>(p, vec, s); break;
        default: launch_fwd<__half, QUANT>(p, vec, s); break;
    }
    PB_LAUNCH_CHECK(what);
    return PARAS_OK;
}

}  // namespace
}  // namespace pb

using pb::fail;

extern "C" {

int paras_b200_add_rmsnorm_fwd(int gpu, const void* x, const void* residual, const void* weight, void* h, void* y,
                               float* rstd, int64_t rows, int64_t H, double eps, int dtype, void* stream) {
    pb::NvtxRange range("paras_b200_add_rmsnorm_fwd");
    return pb::forward<false>(gpu, x, residual, weight, h, y, rstd, nullptr, rows, H, eps, 0, dtype, stream, "paras add_rms_norm");
}

int paras_b200_add_rmsnorm_quant_fwd(int gpu, const void* x, const void* residual, const void* weight, void* h,
                                     void* q, float* scales, int64_t rows, int64_t H, double eps, int group, int dtype,
                                     void* stream) {
    pb::NvtxRange range("paras_b200_add_rmsnorm_quant_fwd");
    return pb::forward<true>(gpu, x, residual, weight, h, q, nullptr, scales, rows, H, eps, group, dtype, stream,
                             "paras add_rms_norm_quant");
}

int paras_b200_add_rmsnorm_bwd(int gpu, const void* grad_y, const void* grad_h, const void* h, const void* weight,
                               const float* rstd, void* grad_x, void* grad_weight, int64_t rows, int64_t H, int dtype,
                               void* stream) {
    pb::NvtxRange range("paras_b200_add_rmsnorm_bwd");
    const char* what = "paras add_rms_norm_backward";
    int st = pb::check_sizes(rows, H, dtype, what);
    if (st != PARAS_OK) return st;
    pb::DeviceRestore restore;
    pb::Gpu* g = pb::use_gpu(gpu, &st);
    if (!g) return st;
    if (H == 0) return PARAS_OK;
    if (weight && !grad_weight) return fail(PARAS_E_INVALID, "%s: null pointer", what);
    cudaStream_t s = pb::pick_stream(g, stream);
    if (rows == 0) {
        if (grad_weight) PB_CUDA(cudaMemsetAsync(grad_weight, 0, size_t(H) * pb::dtype_size(dtype), s));
        return PARAS_OK;
    }
    if (!grad_y || !h || !rstd || !grad_x) return fail(PARAS_E_INVALID, "%s: null pointer", what);
    pb::BwdParams p{};
    p.gy = grad_y; p.gh = grad_h; p.h = h; p.w = weight; p.rstd = rstd; p.gx = grad_x; p.rows = rows; p.H = H;
    const int64_t n = 16 / int64_t(pb::dtype_size(dtype));
    const bool vec = H % n == 0 && pb::al16(grad_y) && pb::al16(grad_h) && pb::al16(h) && pb::al16(weight) && pb::al16(grad_x);
    void* gw = weight ? grad_weight : nullptr;
    switch (dtype) {
        case PARAS_F32: return pb::launch_bwd<float>(g, p, gw, vec, s);
        case PARAS_BF16: return pb::launch_bwd<__nv_bfloat16>(g, p, gw, vec, s);
        default: return pb::launch_bwd<__half>(g, p, gw, vec, s);
    }
}

}  // extern "C"
