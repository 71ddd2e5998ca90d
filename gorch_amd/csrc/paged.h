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

// The sequence of a batch that x belongs to: the last s with key(s, first row
// of s) <= x (key not decreasing), its rows and its length; false if there is
// none. Every lane of the wave calls it with the same x and gets the answer.
// 64 candidates a step, and the last step fetches everything at once: up to
// 64 sequences take one round trip to memory, up to 4096 two.
struct SeqAt {
    int s, begin, end, len;
};
template <typename Key>
__device__ __forceinline__ bool wave_seq(const PagedArgs& a, int x, Key key, SeqAt& r) {
    const int lane = threadIdx.x & 63;
    int lo = 0, n = a.seqs;
    while (n > 64) {
        const int step = (n + 63) / 64, at = lane * step;
        const int c = __popcll(__ballot(at < n && key(lo + at, seq_begin(a, lo + at)) <= x));
        if (c == 0) return false;
        lo += (c - 1) * step;
        n = min(step, n - (c - 1) * step);
    }
    const int i = lo + min(lane, n - 1);
    const int b = seq_begin(a, i), e = max(b, seq_begin(a, i + 1)), len = a.lens[i];
    const int c = __popcll(__ballot(lane < n && key(i, b) <= x));
    if (c == 0) return false;
    r.s = lo + c - 1;
    r.begin = __builtin_amdgcn_readlane(b, c - 1);
    r.end = __builtin_amdgcn_readlane(e, c - 1);
    r.len = __builtin_amdgcn_readlane(len, c - 1);
    return true;
}
// The sequence that token row t belongs to.
__device__ __forceinline__ bool token_seq(const PagedArgs& a, int t, SeqAt& r) {
    return wave_seq(a, t, [](int, int begin) { return begin; }, r) && t < r.end;
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
