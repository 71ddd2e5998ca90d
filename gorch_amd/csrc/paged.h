// paged.h — what the paged KV cache's kernels share: the batch and the pools
// as kernels see them, the sequence a token row belongs to, the address of a
// position.
#pragma once
#include "common.h"

namespace gh {

// Division of 0 <= n < 2^31 by a fixed d: with l = ceil(log2 d) and m =
// ceil(2^(31 + l) / d) (which fits 32 bits), n / d = n * m >> (31 + l): the
// excess m d - 2^(31 + l) is below 2^l, so n times it stays below 2^(31 + l).
struct FastDiv {
    uint32_t d, m, sh;
    __host__ void set(uint32_t div) {
        d = div;
        uint32_t l = 0;
        while ((1ull << l) < div) l++;
        sh = 31 + l;
        m = (uint32_t)(((1ull << sh) + div - 1) / div);
    }
    __device__ __forceinline__ uint32_t div(uint32_t n) const { return (uint32_t)(((uint64_t)n * m) >> sh); }
};

struct PagedArgs {
    void* k;
    void* v;
    float* ks;
    float* vs;
    const int* cu;
    const int* lens;
    const int* table;
    int tokens, seqs, max_pages;
    int num_pages, num_kv, hd;
    int limit;  // positions at or past it are not looked at
    FastDiv page;
};

// First row of sequence s, kept in range whatever the array holds.
__device__ __forceinline__ int seq_begin(const PagedArgs& a, int s) { return min(max(a.cu[s], 0), a.tokens); }

// The last s with key(s) <= x among 0 .. n - 1 (key not decreasing), -1 if
// none; every lane of the wave calls it with the same x and gets the answer.
// 64 candidates a step, so 64 sequences take one load and 4096 two.
template <typename Key>
__device__ __forceinline__ int wave_find(int n, int x, Key key) {
    const int lane = threadIdx.x & 63;
    int lo = 0;
    bool first = true;
    while (n > 1 || first) {
        const int step = (n + 63) / 64, at = lane * step;
        const bool le = at < n && key(lo + at) <= x;
        const int c = __popcll(__ballot(le));
        if (c == 0) return -1;
        lo += (c - 1) * step;
        n = min(step, n - (c - 1) * step);
        first = false;
    }
    return lo;
}

// Pool row of position p of sequence s for KV head h (in rows of hd elements;
// also the scale's index), or -1 where there is none.
__device__ __forceinline__ long long pool_row(const PagedArgs& a, int s, int p, int h) {
    if ((unsigned)p >= (unsigned)a.limit) return -1;
    const uint32_t i = a.page.div((uint32_t)p);
    const int page = a.table[(size_t)s * a.max_pages + i];
    if ((unsigned)page >= (unsigned)a.num_pages) return -1;
    return ((long long)page * a.num_kv + h) * a.page.d + (p - (int)(i * a.page.d));
}

// Checks a cache and a batch and fills the kernels' view of them.
int paged_args(const char* who, const gorch_hip_paged_kv* kv, const gorch_hip_paged_batch* b, PagedArgs& a);

// e4m3 code -> f32, exact (NaN for the codes 0x7f and 0xff).
template <int BYTE>
__device__ __forceinline__ float e4m3_f32(uint32_t w) {
    return __builtin_amdgcn_cvt_f32_fp8((int)w, BYTE);
}

}  // namespace gh
