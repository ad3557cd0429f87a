// What the kernels over a paged key / value cache share: the ragged rows' search, the 8-bit row format, argument checks.
#pragma once

#include "common.cuh"

namespace pb {

// The number of entries of a[0..n) that are <= t, a non-decreasing, found by a whole warp: every round probes 32 places
// and leaves a 33rd part of the range, so 1000 sequences cost two dependent loads.
__device__ __forceinline__ int warp_count_le(const int32_t* __restrict__ a, int n, int t) {
    const int lane = int(threadIdx.x) & 31;
    int lo = 0, hi = n;
    while (lo < hi) {
        const int step = (hi - lo + 31) / 32;
        const int64_t idx = int64_t(lo) + int64_t(lane + 1) * step - 1;
        const bool le = idx < hi && __ldg(a + idx) <= t;
        lo += __popc(__ballot_sync(0xffffffffu, le)) * step;
        hi = min(hi, lo + step - 1);
    }
    return lo;
}

// ---- rows of e4m3 with one exponent byte ----------------------------------------------------
constexpr int kExpLo = -15, kExpHi = 7;   // e4m3 * 2^e: multiples of 2^-24 below 57345, exact in fp16 and bf16

// Smallest e with amax * 2^-e <= 448 = 1.75 * 2^8, within [kExpLo, kExpHi]; 0 for an empty row.
__device__ __forceinline__ int row_exponent(float amax) {
    const uint32_t bits = __float_as_uint(amax);
    const int e = int(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return amax == 0.f ? 0 : max(kExpLo, min(kExpHi, e));
}
__device__ __forceinline__ float pow2f(int e) { return __uint_as_float(uint32_t(e + 127) << 23); }   // -126 <= e <= 127
// 2^(byte - 127) for any byte: 0 stands for 2^-127 (a subnormal), 255 for 2^128 (infinity in fp32)
__device__ __forceinline__ float exp_byte(uint32_t byte) {
    return byte == 0 ? __uint_as_float(0x00400000u) : __uint_as_float(byte << 23);
}
// Two fp32 -> two e4m3 bytes, nearest even, magnitudes above 448 to 448, NaN to NaN; `lo` in the low byte.
__device__ __forceinline__ uint32_t pack_e4m3(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
// Two e4m3 bytes -> a pair of fp16 (exact).
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t two) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(uint16_t(two)));
    return r;
}
// Four bytes -> two pairs, low bytes first.
__device__ __forceinline__ void e4m3x4_to_f16x4(uint32_t four, uint32_t* lo, uint32_t* hi) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(*lo), "=r"(*hi) : "r"(four));
}
__device__ __forceinline__ float2 e4m3x2_to_f32(uint32_t two) {
    const uint32_t h = e4m3x2_to_f16x2(two);
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
__device__ __forceinline__ float e4m3_to_f32(uint8_t b) { return e4m3x2_to_f32(b).x; }

// Positions that a page table may reach: the kernels count them in 32 bits and step or round up by as many as 128 beyond.
constexpr int64_t kMostPositions = (int64_t(1) << 31) - 256;

// Checks shared by the entry points; `what` names the caller in the message.
int check_paged_cache(const paras_paged_cache& c, int dtype, const char* what);

// Restores the caller's current device when a call ends.
struct DeviceRestore {
    int old = -1;
    DeviceRestore() {
        if (cudaGetDevice(&old) != cudaSuccess) { cudaGetLastError(); old = -1; }
    }
    ~DeviceRestore() {
        if (old >= 0) cudaSetDevice(old);
    }
};

}  // namespace pb
