// Internal interfaces of the attention kernels over a paged cache.
#pragma once

#include "paged_common.cuh"

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
    int cap;             // positions the page table can name
    int causal;
    float scale, scale_log2;
    int* status;
};

// The new tokens of sequence b: first row, count (at most max_q), positions in the cache.  Whatever the device arrays
// hold, rows stay within [0, T).
struct PagedSeq {
    int row0, nq;
    int kv;       // positions 0 .. kv-1, kv <= cap
    int pos0;     // position of the first new token (may be negative or past kv)
};
__device__ __forceinline__ PagedSeq paged_seq(const PagedParams& p, int b) {
    PagedSeq s;
    const int c0 = __ldg(p.cu + b), c1 = __ldg(p.cu + b + 1), kv = __ldg(p.kv_lens + b);
    s.row0 = max(0, min(c0, p.T));
    const int end = max(s.row0, min(c1, p.T));
    const int count = end - s.row0;
    s.nq = min(count, p.max_q);
    s.kv = max(0, min(kv, p.cap));
    s.pos0 = int(max(int64_t(-(1 << 30)), min(int64_t(kv) - count, int64_t(1 << 30))));
    return s;
}
// Keys that new token i of the sequence attends: positions 0 .. n-1.
__device__ __forceinline__ int paged_keys(const PagedParams& p, const PagedSeq& s, int i) {
    return p.causal ? max(0, min(s.kv, s.pos0 + i + 1)) : s.kv;
}

int paged_simt_launch(const PagedParams& p, int dtype, bool cache8, cudaStream_t s);

}  // namespace pb
