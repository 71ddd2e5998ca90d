// paged_attention.hip — attention of ragged new tokens over a KV cache in
// pages (gorch_hip_gqa_attention_cached's mathematics, GQA.forwardCached
// nn/gqa.go:308-352): over the positions j that a token sees,
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(s_j - m),  s_j = log2(e) q . k_j / sqrt(hd),
// with the running maximum m and sum of one pass over the keys.
#include <algorithm>
#include <cmath>

#include "paged_attention.h"

namespace gh {

// Few rows: a block takes CW rows of a sequence (with their KV head) and a
// range of its keys, its four waves 32 keys each in turn. K goes from memory
// to the operand registers, V through a wave's own LDS; NB tiles of rows are
// on their way while one is weighed (a fetch is unconditional: a branch around
// loads would make the next use wait for all of them; one tile where two would
// leave the registers, bf16 of 128 columns and either type of 256). Bound by
// the loads that a CU keeps in flight: 64 conversations of up to 8,192 tokens,
// 8 x 128 in e4m3 (397 MB), 96 us with the join, 4.1 TB/s (in bf16 170 us, 4.5),
// where plain reads reach 7.1; waves wait a quarter of their cycles, the matrix
// cores are busy 5%, and a block's first loads and the last ranges' ends are
// not covered by others. One token over 777 keys 6.7 us and 3.4 for the join,
// three dependent round trips (page, key, key of the next step).
template <bool F8, int HD, bool PART, int CW>
struct FewBlock {
    static constexpr int NW = 4, NB = Tile<F8, HD>::NT <= 2 ? 2 : 1, OROW = HD + 4;
    static constexpr int STAGE = NW * (Tile<F8, HD>::BYTES + 256), JOIN = NW * 16 * (OROW + 2) * 4;
    char lds[STAGE > JOIN ? STAGE : JOIN];
    OddBits<CW, HD> odd;
};
template <bool F8, int HD, bool PART, int CW>
__device__ __forceinline__ void few_tile(const PagedAttnArgs& a, const SeqAt& s, int r0, int kvh, int split,
                                         const int (&page)[FewBlock<F8, HD, PART, CW>::NB + 1],
                                         FewBlock<F8, HD, PART, CW>& sh) {
    using T = Tile<F8, HD>;
    using R = FewRows<F8, HD, CW>;
    using Sh = FewBlock<F8, HD, PART, CW>;
    constexpr int NW = Sh::NW, STEP = 32 * NW, NB = Sh::NB, OROW = Sh::OROW;
    char* const lds = sh.lds;
    auto& odd = sh.odd;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4;
    const int G = a.group.d, n = s.end - s.begin;
    const int end_tok = (int)a.group.div((uint32_t)(min(r0 + CW, n * G) - 1));
    const int T1 = min((a.causal ? s.len - n + end_tok : s.len - 1) + 1, a.p.limit);
    const int k0 = split * a.chunk, k1 = a.splits == 1 ? T1 : min(T1, k0 + a.chunk);
    if (k0 >= k1) {
        if (split == 0) put_nothing<CW>(a, split, s, r0, kvh);
        return;
    }

    char* vt = lds + wave * (T::BYTES + 256);
    float* sc = reinterpret_cast<float*>(vt + T::BYTES);  // K scales of the 32 keys, then V's
    struct Buf {
        u32x4 k[2][T::NT], v[2][T::NT];
        float scale;
        uint32_t seen;
    } buf[NB];
    // row: the pool row of key lane % 32 of the tile
    auto fetch = [&](long long row, Buf& b) {
        const auto lo = __builtin_amdgcn_permlane16_swap((uint32_t)row, (uint32_t)row, false, false);
        const auto hi = __builtin_amdgcn_permlane16_swap((uint32_t)(row >> 32), (uint32_t)(row >> 32), false, false);
        b.seen = (uint32_t)__ballot(row >= 0);
#pragma unroll
        for (int j = 0; j < 2; j++)
            fetch_row<F8, HD, PART>(a.p.k, (long long)(((uint64_t)hi[j] << 32) | lo[j]), a.p.hd, g, b.k[j]);
        if constexpr (F8) {
            const float* from = lane < 32 ? a.p.ks : a.p.vs;
            b.scale = *(row >= 0 ? from + row : reinterpret_cast<const float*>(kZeros));
        }
#pragma unroll
        for (int j = 0; j < 2; j++)
            fetch_row<F8, HD, PART>(a.p.v, (long long)(((uint64_t)hi[j] << 32) | lo[j]), a.p.hd, g, b.v[j]);
    };
    R rows;
    int key0 = k0 + 32 * wave;
    int next;  // the page of the next tile to fetch
    {
        next = page[NB];
        float4 x[T::NU][2];
        rows.template fetch<PART>(a, s, r0, kvh, x);
#pragma unroll
        for (int i = 0; i < NB; i++) fetch(key_row(a.p, page[i], key0 + i * STEP + (lane & 31), k1, kvh), buf[i]);
        for (int i = threadIdx.x; i < (int)(sizeof(odd) / 4); i += 64 * NW) reinterpret_cast<uint32_t*>(&odd)[i] = 0;
        rows.begin(a, x);
    }
    __syncthreads();
    // (what is fetched does not depend on whether a tile is past the end, so
    // the loads in flight are the same on every way to the next tile)
    auto step = [&](Buf& b, int key) {
        const bool on = key < k1;
        const uint32_t here = b.seen;
        floatx4 scores[2];
        if (on) {
            scores[0] = rows.score(b.k[0]);
            scores[1] = rows.score(b.k[1]);
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int t = 0; t < T::NT; t++)
                    *reinterpret_cast<u32x4*>(vt + j * T::GROUP + t * 1024 + lane * 16) = b.v[j][t];
            if (__any(any_nonfinite<F8>(b.v[0]) | any_nonfinite<F8>(b.v[1])))
#pragma unroll 1
                for (int i = 0; i < 2 * T::NT; i++) {
                    const int j = i & 1, t = i >> 1;
                    clean_odd<F8, CW, HD>(odd, a, s, r0, key + 16 * j + (lane & 15), (4 * t + g) * (16 / T::ES),
                                          vt + j * T::GROUP + t * 1024 + lane * 16);
                }
            if constexpr (F8) sc[lane] = b.scale;
        }
        // (the page of the tile after goes out first: loads are waited for in
        // order, and the next fetch waits for it)
        const int after = key_page(a.p, s.s, key + (NB + 1) * STEP + (lane & 31));
        __builtin_amdgcn_sched_barrier(0);
        fetch(key_row(a.p, next, key + NB * STEP + (lane & 31), k1, kvh), b);
        next = after;
        if (on) rows.take(scores, key, here, sc, sc + 32, vt);
    };
    for (; key0 < k1; key0 += NB * STEP) {
        step(buf[0], key0);
        if constexpr (NB == 2) step(buf[1], key0 + STEP);
    }
    // the waves' sums, joined in wave order
    __syncthreads();
    float* jo = reinterpret_cast<float*>(lds);
    float* jm = jo + NW * 16 * OROW;
    float* jl = jm + NW * 16;
    const float l = col_sum(rows.l);
#pragma unroll
    for (int d = 0; d < HD / 16; d++)
        *reinterpret_cast<floatx4*>(jo + (wave * 16 + (lane & 15)) * OROW + 16 * d + 4 * g) = rows.o[d];
    if (g == 0) {
        jm[wave * 16 + lane] = rows.m;
        jl[wave * 16 + lane] = l;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < CW * (HD / 4); i += 64 * NW) {
        const int r = i / (HD / 4), c = 4 * (i % (HD / 4));
        if (r0 + r >= n * G || (PART && c >= a.p.hd)) continue;
        float M = jm[r];
#pragma unroll
        for (int w = 1; w < NW; w++) M = fmaxf(M, jm[w * 16 + r]);
        const float use = M == -INFINITY ? 0.f : M;
        floatx4 o = {0.f, 0.f, 0.f, 0.f};
        float L = 0.f;
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const float f = __builtin_amdgcn_exp2f(jm[w * 16 + r] - use);
            L += f * jl[w * 16 + r];
#pragma unroll
            for (int t = 0; t < 3 && t < R::TP; t++) {
                const floatx4 x = *reinterpret_cast<const floatx4*>(jo + (w * 16 + t * CW + r) * OROW + c);
#pragma unroll
                for (int e = 0; e < 4; e++) o[e] += f * x[e];
            }
        }
        if (odd.any) o = add_odd(odd, r, c, o);
        const RowAt at = row_at(a, s, r0 + r, kvh);
        put(a, split, at, c, o, L);
        if (a.splits > 1 && c == 0) a.part_ml[(size_t)split * a.part_rows + at.part] = make_float2(M, L);
    }
}
// Block `block` of a grid that has `per` tiles for every sequence (enough for
// max_new).
template <bool F8, int HD, bool PART, int CW>
__device__ __forceinline__ void few_block(const PagedAttnArgs& a, int block, FewBlock<F8, HD, PART, CW>& sh) {
    const int kvh = block % a.p.num_kv, rest = block / a.p.num_kv;
    const int tile = rest % a.tiles, split = a.last_first ? a.splits - 1 - rest / a.tiles : rest / a.tiles;
    SeqAt s;
    s.s = tile / a.per;
    // the first tiles' pages, beside the sequence's place (the range's start is
    // known without it)
    using Sh = FewBlock<F8, HD, PART, CW>;
    int page[Sh::NB + 1];
#pragma unroll
    for (int i = 0; i <= Sh::NB; i++)
        page[i] = key_page(a.p, s.s, split * a.chunk + 32 * (int)(threadIdx.x >> 6) + i * 32 * Sh::NW + (int)(threadIdx.x & 31));
    const int b = seq_begin(a.p, s.s), e = seq_begin(a.p, s.s + 1), len = a.p.lens[s.s];
    s.begin = __builtin_amdgcn_readfirstlane(b);
    s.end = __builtin_amdgcn_readfirstlane(max(b, e));
    s.len = __builtin_amdgcn_readfirstlane(len);
    const int rows = (s.end - s.begin) * (int)a.group.d;
    if (rows < a.lo_rows || rows > a.hi_rows) return;
    const int r0 = (tile - s.s * a.per) * CW;
    if (r0 < rows) few_tile<F8, HD, PART, CW>(a, s, r0, kvh, split, page, sh);
}
template <bool F8, int HD, bool PART, int CW>
__global__ __launch_bounds__(256, HD > 128 ? 1 : (HD == 64 && CW == 4 ? 3 : 2)) void k_paged_attn_few(PagedAttnArgs a) {
    __shared__ __align__(16) FewBlock<F8, HD, PART, CW> sh;
    few_block<F8, HD, PART, CW>(a, (int)blockIdx.x, sh);
}

// Many rows: a block takes 128 rows of a sequence, 16 NR a wave, and its keys
// (or a range of them) in tiles of 32 that all NW waves read from LDS. Loads
// go straight to LDS, two tiles ahead of the one that is weighed: one on its
// way, one landed, in which the waves look for infinities in V. 2,048 rows of 16
// heads of 128 over 16,384 keys (257 GFLOP, 771 in three terms) 641-662 us (e4m3,
// which every wave widens for itself, 728): 1.2 PFLOP/s of matrix instructions,
// the rate of a large bf16 product here, of the 2.05 that a plain loop of them
// reaches. The matrix cores are busy 53%; a wave's exponentials, splits and LDS
// reads stand between its products, and the block meets every 32 keys with all
// its loads landed. (No faster: a ring of four or five tiles, operands read two
// or three steps ahead, priorities by wave.)
template <bool F8, int HD>
struct ManyBlock {
    alignas(16) char kt[3][Tile<F8, HD>::BYTES], vt[3][Tile<F8, HD>::BYTES];
    alignas(16) float sc[3][4][F8 ? 64 : 1];  // e4m3 scales: K's two groups, V's two (16 each)
    uint32_t seen_of[3][2];
    OddBits<kManyRows, HD> odd;
};
template <bool F8, int HD, bool PART, int NR>
__device__ __forceinline__ void many_block(const PagedAttnArgs& a, int block, ManyBlock<F8, HD>& sh) {
    using T = Tile<F8, HD>;
    constexpr int BM = kManyRows, NW = BM / (16 * NR);
    auto& kt = sh.kt;
    auto& vt = sh.vt;
    auto& sc = sh.sc;
    auto& seen_of = sh.seen_of;
    auto& odd = sh.odd;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4;
    const int kvh = block % a.p.num_kv, rest = block / a.p.num_kv;
    // the last rows of a sequence see the most keys: they go first
    const int tile = a.tiles - 1 - rest % a.tiles, split = rest / a.tiles;
    SeqAt s;
    int r0;
    if (!find_tile<BM>(a, tile, s, r0)) return;
    const int G = a.group.d, n = s.end - s.begin;
    // the last position that any of the block's rows sees
    const int end_tok = (int)a.group.div((uint32_t)(min(r0 + BM, n * G) - 1));
    const int T1 = min((a.causal ? s.len - n + end_tok : s.len - 1) + 1, a.p.limit);
    const int k0 = split * a.chunk, k1 = a.splits == 1 ? T1 : min(T1, k0 + a.chunk);
    if (k0 >= k1) {
        if (split == 0) put_nothing<BM>(a, split, s, r0, kvh);
        return;
    }

    // of four waves, 0 and 1 fetch K's two groups of a tile, 2 and 3 V's
    const int j = wave & 1;
    const bool isv = (wave & 2) != 0;
    auto page_of = [&](int key0) { return key_page(a.p, s.s, key0 + 16 * j + (lane & 15)); };
    auto fetch = [&](int page, int key0, int b) {
        const long long row = key_row(a.p, page, key0 + 16 * j + (lane & 15), k1, kvh);
        typedef __attribute__((address_space(1))) const uint32_t* global_ptr;
        typedef GH_LDS uint32_t* lds_ptr;
        const char* zero = reinterpret_cast<const char*>(kZeros);
        const char* p = row >= 0 ? static_cast<const char*>(isv ? a.p.v : a.p.k) + row * (a.p.hd * T::ES) : zero;
        char* to = (isv ? vt[b] : kt[b]) + j * T::GROUP;
#pragma unroll
        for (int t0 = 0; t0 < T::NT; t0 += NW / 4) {
            const int t = t0 + (wave >> 2), o = (4 * t + g) * 16;
            __builtin_amdgcn_global_load_lds((global_ptr)(PART && o >= a.p.hd * T::ES ? zero : p + o),
                                             (lds_ptr)(to + t * 1024), 16, 0, 0);
        }
        if (F8 && wave < 4) {
            const float* f = row >= 0 ? (isv ? a.p.vs : a.p.ks) + row : reinterpret_cast<const float*>(kZeros);
            __builtin_amdgcn_global_load_lds((global_ptr)f, (lds_ptr)sc[b][wave], 4, 0, 0);
        }
        const uint32_t here = (uint32_t)__ballot(row >= 0) & 0xffffu;
        if (lane == 0 && wave < 2) seen_of[b][j] = here;
    };
    // a wave's share of a landed tile's V
    auto check = [&](int key0, int b) {
        int any = 0;
#pragma unroll
        for (int i0 = 0; i0 < 2 * T::NT; i0 += NW) {
            const int i = i0 + wave;
            if (2 * T::NT % NW != 0 && i >= 2 * T::NT) break;
            u32x4 c[1] = {*reinterpret_cast<const u32x4*>(vt[b] + (i & 1) * T::GROUP + (i >> 1) * 1024 + lane * 16)};
            any |= any_nonfinite<F8>(c);
        }
        if (__any(any))
#pragma unroll 1
            for (int i = wave; i < 2 * T::NT; i += NW)
                clean_odd<F8, BM, HD>(odd, a, s, r0, key0 + 16 * (i & 1) + (lane & 15),
                                           (4 * (i >> 1) + g) * (16 / T::ES),
                                           vt[b] + (i & 1) * T::GROUP + (i >> 1) * 1024 + lane * 16);
    };
    Rows<F8, HD, NR> rows;
    int next = page_of(k0 + 32);
    fetch(page_of(k0), k0, 0);
    {
        float4 x[NR][T::NU][2];
        rows.template fetch<PART>(a, s, r0 + 16 * NR * wave, kvh, x);
        fetch(next, k0 + 32, 1);
        next = page_of(k0 + 64);
        for (int i = threadIdx.x; i < (int)(sizeof(odd) / 4); i += 64 * NW) reinterpret_cast<uint32_t*>(&odd)[i] = 0;
        rows.begin(a, x);
    }
    block_sync_dma();
    check(k0, 0);
    block_sync_dma();
    for (int key0 = k0, b = 0; key0 < k1; key0 += 32) {
        const int b1 = b == 2 ? 0 : b + 1, b2 = b1 == 2 ? 0 : b1 + 1;
        const int after = page_of(key0 + 96);
        fetch(next, key0 + 64, b2);
        next = after;
        if (key0 <= rows.last) {
            floatx4 scores[2][NR];
            rows.score(kt[b], scores);
            rows.take(scores, key0, seen_of[b][0] | (seen_of[b][1] << 16), sc[b][0], sc[b][2], vt[b]);
        }
        check(key0 + 32, b1);
        block_sync_dma();
        b = b1;
    }
#pragma unroll
    for (int i = 0; i < NR; i++) {
        const float l = col_sum(rows.l[i]);
        const int r = r0 + 16 * (NR * wave + i) + (lane & 15);
        if (r >= n * G) continue;
        const RowAt at = row_at(a, s, r, kvh);
#pragma unroll
        for (int d = 0; d < HD / 16; d++)
            if (!PART || 16 * d < a.p.hd) {
                const int c = 16 * d + 4 * g;
                put(a, split, at, c, odd.any ? add_odd(odd, r - r0, c, rows.o[i][d]) : rows.o[i][d], l);
            }
        if (a.splits > 1 && g == 0) a.part_ml[(size_t)split * a.part_rows + at.part] = make_float2(rows.m[i], l);
    }
}
template <bool F8, int HD, bool PART, int NR>
__global__ __launch_bounds__(kManyRows / NR * 4, HD == 64 ? 3 : 2) void k_paged_attn_many(PagedAttnArgs a) {
    __shared__ __align__(16) ManyBlock<F8, HD> sh;
    many_block<F8, HD, PART, NR>(a, (int)blockIdx.x, sh);
}
// Both in one launch, for up to 128 columns, where their blocks are of one
// size: the blocks of few rows, which wait for memory, run beside those of
// many, which keep the matrix cores busy.
template <bool F8, int HD, bool PART, int CW>
__global__ __launch_bounds__(256, HD == 64 ? 3 : 2) void k_paged_attn_both(PagedAttnArgs many, PagedAttnArgs few,
                                                                                     int many_blocks) {
    __shared__ __align__(16) union {
        ManyBlock<F8, HD> many;
        FewBlock<F8, HD, PART, CW> few;
    } sh;
    if ((int)blockIdx.x < many_blocks) many_block<F8, HD, PART, 2>(many, (int)blockIdx.x, sh.many);
    else few_block<F8, HD, PART, CW>(few, (int)blockIdx.x - many_blocks, sh.few);
}

// A row's splits joined, each weighted by 2^(its maximum - the largest): WPR
// waves per (token, query head), 16 bytes of a split's columns a lane, the
// splits dealt to SLOTS groups of lanes (sums in a fixed order: a slot's
// splits, then the slots). The first loads go out before the sequence is
// known, as if it were no exception (few_cap); splits past the row's last are
// then left out.
constexpr int kMaxSplits = 64;
template <int NL, int WPR>
__global__ __launch_bounds__(256) void k_paged_attn_join(PagedAttnArgs a) {
    constexpr int SLOTS = WPR * 64 / NL, RPB = 4 / WPR;
    __shared__ floatx4 so[RPB][SLOTS][NL];
    const int lane = threadIdx.x & 63, sub = threadIdx.x / (64 * WPR), tid = threadIdx.x % (64 * WPR);
    const long long total = (long long)a.p.tokens * a.hq;
    const long long row = min(__builtin_amdgcn_readfirstlane(blockIdx.x * RPB + sub), (int)total - 1);
    const bool mine = (long long)blockIdx.x * RPB + sub < total;
    const int c = tid % NL, slot = tid / NL, col = min(4 * c, a.p.hd - 4);
    const float* po = a.part_o;
    long long stride = a.part_rows, at = min(row, a.part_rows - 1);
    int last = (a.few_cap && a.splits2 > 1 ? a.splits2 : max(a.splits, a.splits2)) - 1;
    float2 ml = a.part_ml[min(lane, last) * stride + at];
    auto part = [&](int j) {
        return *reinterpret_cast<const floatx4*>(po + (min(j, last) * stride + at) * a.p.hd + col);
    };
    floatx4 x = part(slot);
    const int t = (int)(row / a.hq);
    SeqAt s;
    int nc = 0;
    if (token_seq(a.p, t, s)) {
        const bool few = (s.end - s.begin) * (int)a.group.d <= a.hi_rows;
        const int chunk = few ? a.chunk : a.chunk2, splits = few ? a.splits : a.splits2;
        const int T = min(a.causal ? s.len - s.end + t + 1 : s.len, a.p.limit);
        nc = splits == 1 ? 0 : min(max((T + chunk - 1) / chunk, 1), splits);  // (one split: out is written)
        if (few && a.few_cap && nc > 0) {
            const int G = a.group.d, h = (int)(row - (long long)t * a.hq), kvh = h / G;
            po = a.few_o;
            stride = a.few_rows;
            at = ((long long)s.s * a.few_cap + (t - s.begin) * G + (h - kvh * G)) * a.p.num_kv + kvh;
            last = splits - 1;
            ml = a.few_ml[min(lane, last) * stride + at];
            x = part(slot);
        }
    }
    if (lane >= nc) ml = make_float2(-INFINITY, 0.f);
    const float M = wave_max(ml.x), use = M == -INFINITY ? 0.f : M;
    const float w = __builtin_amdgcn_exp2f(ml.x - use);
    const float L = wave_sum(w * ml.y);
    floatx4 o = {0.f, 0.f, 0.f, 0.f};
    for (int j = slot; j - slot < nc; j += SLOTS) {
        const floatx4 y = part(j + SLOTS);
        const float f = __shfl(w, j & 63);
        // (an infinity is a value's, noted: it stays where its range's weight, f, is 0)
        if (j < nc)
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] += __builtin_isinf(x[e]) ? x[e] : f * x[e];
        x = y;
    }
    so[sub][slot][c] = o;
    __syncthreads();
    if (tid >= NL || nc == 0 || !mine || 4 * c >= a.p.hd) return;
#pragma unroll
    for (int j = 1; j < SLOTS; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] += so[sub][j][c][e];
    const float r = L == 0.f ? 0.f : 1.0f / L;
    *reinterpret_cast<floatx4*>(a.out + row * a.p.hd + col) = floatx4{o[0] * r, o[1] * r, o[2] * r, o[3] * r};
}

// ---------------------------------------------------------------- launch

// Rows (tokens x heads of a group) up to which a batch whose sequences have no
// more goes to the kernel for few rows alone.
constexpr int kFewRows = 32;

static AttnPlan attn_plan(const PagedArgs& p, int hq, int max_new) {
    AttnPlan r{};
    const auto over = [](long long a, long long b) { return (a + b - 1) / b; };
    const long long G = hq / p.num_kv;
    const long long most = std::min<long long>(max_new > 0 ? max_new : p.tokens, p.tokens) * G;
    r.many = most > kFewRows;
    // beside prompts, the kernel for few rows takes the single tokens
    const long long rows = r.many ? G : most;
    r.few_width = rows <= 4 ? 4 : 16;
    r.few_rows = !r.many ? 0x7fffffff : (int)over(rows, r.few_width) * r.few_width;
    r.few = !r.many || (p.seqs > 1 && rows <= kFewRows);
    const int bm = kManyRows;
    r.few_per = (int)over(r.many ? std::min<long long>(r.few_rows, most) : most, r.few_width);
    r.few_tiles = r.few_per * p.seqs;
    r.many_tiles = (int)(p.tokens * G / bm) + p.seqs;
    // how `keys` keys are split into at most n ranges of whole units
    const auto split = [&](long long n, int unit, int& chunk) {
        const long long units = std::max(1ll, ((long long)p.limit + unit - 1) / unit);
        n = std::max(1ll, std::min({n, units, (long long)kMaxSplits}));
        const long long per = (units + n - 1) / n;
        chunk = (int)std::min<long long>(per * unit, 0x7fffff00);
        return (int)((units + per - 1) / per);
    };
    // blocks that are expected to have work, unsplit
    const long long few = std::max(1ll, p.seqs * over(rows, r.few_width)) * p.num_kv;
    const long long many = std::min<long long>(over(p.tokens * G, bm) + (over(p.tokens * G, most) - 1) / 2,
                                                   p.seqs * over(most, bm)) * p.num_kv;
    r.few_splits = r.many_splits = 1;
    // (past 2^25 rows a join would leave a launch's range)
    const bool joins = (long long)p.tokens * hq < 1 << 25;
    if (r.few) {
        // 1024 blocks, four for each CU (which holds two to four at once), whose
        // ends even out over ragged lengths; of up to 32 tiles, or where a CU
        // holds one block (more than 128 columns), one a CU: 3 tokens over up to
        // 32,749 keys 16.5 -> 13.8 us, 4 of 32/8 x 128 over 10,000 32 -> 26, 64 of
        // 8/1 x 256 over 8,192 91 -> 70; but 64 of 14/2 x 64 over 4,096 15.8 -> 21.
        // Ranges of at most 2048 keys, so that the longest sequence's end is not
        // waited for alone; not from 2048 tiles on, where it costs a batch of one
        // long sequence: one of 32,768 keys (16/8 x 128, bf16) and others of 500,
        // 154 us for 255 sequences, 500 for 256
        const long long blocks = few <= 32 || p.hd > 128 ? 256 : 1024;
        const long long n = std::max(over(blocks, few), few < 2048 ? over(p.limit, 2048) : 1);
        const int unit = few * over(p.limit, 256) < 128 ? 128 : 256;
        r.few_splits = split(joins ? n : 1, unit, r.few_chunk);
        // more blocks than most kernels run at once (256 to 1024 by type, columns
        // and tile): the last splits first, which are the long sequences' (64
        // conversations in e4m3 97.5 -> 93.8 us; where all run at once it costs: 3
        // x 32,749 keys 17.4 -> 21 us)
        r.few_last_first = few * r.few_splits > 768;
    }
    // (two blocks a CU, three with up to 64 columns, all at once; with more than
    // 128, whose 512 threads have a CU alone, two rounds)
    if (r.many) r.many_splits = split(joins ? over(p.hd <= 64 ? 768 : 512, many) : 1, 128, r.many_chunk);
    // (single tokens beside prompts have rows of their own: as part of the
    // prompts' they would take hundreds of times the memory)
    r.few_cap = r.few && r.many ? r.few_per * r.few_width : 0;
    r.many_part = r.many_splits > 1 ? p.tokens * (long long)hq : 0;
    r.few_part = r.few_splits == 1 ? 0 : (r.few_cap ? (long long)p.seqs * r.few_cap * p.num_kv : p.tokens * (long long)hq);
    r.bytes = (size_t)(r.few_splits * r.few_part + r.many_splits * r.many_part) * (p.hd * 4 + 8);
    return r;
}

const char* paged_attn_choice_name(int tokens, int seqs, int hq, int hkv, int hd, int max_new, int positions) {
    PagedArgs p{};
    p.tokens = tokens;
    p.seqs = seqs;
    p.num_kv = hkv;
    p.hd = hd;
    p.limit = positions;
    const AttnPlan pl = attn_plan(p, hq, max_new);
    static const char* const few[2][2] = {{"few4", "few4 split"}, {"few16", "few16 split"}};
    static const char* const both[2][2] = {{"few4+many", "few4+many split"}, {"few16+many", "few16+many split"}};
    const int w = pl.few_width == 4 ? 0 : 1, split = pl.bytes > 0;
    if (!pl.few) return split ? "many split" : "many";
    return pl.many ? both[w][split] : few[w][split];
}

static int attn_args(const gorch_hip_paged_kv* kv, const gorch_hip_paged_batch* b, int num_q, PagedAttnArgs& a) {
    GH_TRY(paged_args("gorch_hip_paged_attention", kv, b, a.p));
    GH_REQUIRE(num_q > 0 && num_q % kv->num_kv == 0, "gorch/nn: GQA NumQ must be divisible by NumKV");
    GH_SUPPORTED((long long)b->tokens * num_q < (1ll << 28) && (long long)b->seqs < (1ll << 28) / kv->num_kv,
                 "gorch_hip_paged_attention: tokens * num_q must be below 2^28");
    // (no position at all: the kernels' reads of a page go elsewhere)
    if (a.p.limit == 0) {
        a.p.table = a.p.cu;
        a.p.max_pages = 0;
    }
    a.hq = num_q;
    a.scale = (float)(1.4426950408889634 / std::sqrt((double)kv->head_dim));
    a.group.set((uint32_t)(num_q / kv->num_kv));
    return GORCH_HIP_OK;
}

// The arguments of the kernel for few rows and of that for many.
static void split_args(const PagedAttnArgs& base, const AttnPlan& pl, PagedAttnArgs& few, PagedAttnArgs& many) {
    few = many = base;
    few.part_o = base.few_o;
    few.part_ml = base.few_ml;
    few.part_rows = pl.few_part;
    few.few_cap = pl.few_cap;
    many.part_rows = pl.many_part;
    few.tiles = pl.few_tiles;
    few.per = pl.few_per;
    few.lo_rows = 0;
    few.hi_rows = pl.few_rows;
    few.chunk = pl.few_chunk;
    few.splits = pl.few_splits;
    few.last_first = pl.few_last_first;
    many.tiles = pl.many_tiles;
    many.lo_rows = pl.few ? pl.few_rows + 1 : 0;
    many.hi_rows = 0x7fffffff;
    many.chunk = pl.many_chunk;
    many.splits = pl.many_splits;
}

template <bool F8, int HD, bool PART>
static void launch_attn(hipStream_t s, const PagedAttnArgs& few, const PagedAttnArgs& many, const AttnPlan& pl) {
    constexpr int NR = HD <= 128 ? 2 : 1, NT = kManyRows / NR * 4;
    const int few_blocks = few.tiles * few.p.num_kv * few.splits, many_blocks = many.tiles * many.p.num_kv * many.splits;
    const auto width = [&](auto go) {
        if (pl.few_width == 4) go(std::integral_constant<int, 4>{});
        else go(std::integral_constant<int, 16>{});
    };
    if constexpr (HD <= 128)
        if (pl.few && pl.many) {
            width([&](auto w) {
                hipLaunchKernelGGL((k_paged_attn_both<F8, HD, PART, decltype(w)::value>), dim3((unsigned)(many_blocks + few_blocks)),
                                   dim3(256), 0, s, many, few, many_blocks);
            });
            return;
        }
    if (pl.few)
        width([&](auto w) {
            hipLaunchKernelGGL((k_paged_attn_few<F8, HD, PART, decltype(w)::value>), dim3((unsigned)few_blocks), dim3(256), 0, s, few);
        });
    if (pl.many) hipLaunchKernelGGL((k_paged_attn_many<F8, HD, PART, NR>), dim3((unsigned)many_blocks), dim3(NT), 0, s, many);
}

template <bool F8>
static void launch_attn_hd(hipStream_t s, const PagedAttnArgs& few, const PagedAttnArgs& many, const AttnPlan& pl) {
    const int hd = few.p.hd;
    if (hd == 64) launch_attn<F8, 64, false>(s, few, many, pl);
    else if (hd < 64) launch_attn<F8, 64, true>(s, few, many, pl);
    else if (hd == 128) launch_attn<F8, 128, false>(s, few, many, pl);
    else if (hd < 128) launch_attn<F8, 128, true>(s, few, many, pl);
    else if (hd == 256) launch_attn<F8, 256, false>(s, few, many, pl);
    else launch_attn<F8, 256, true>(s, few, many, pl);
}

// A wave per row; a block for many splits where rows are few (single tokens
// beside prompts: 30 sequences of 14 heads, 4 chunks of up to 400 rows over
// 2,500 keys 57 -> 47 us; 3 tokens over 32,749 keys, 64 ranges, 17 us against 21).
static void launch_join(hipStream_t s, const PagedAttnArgs& a, int splits) {
    const long long rows = (long long)a.p.tokens * a.hq;
    const auto go = [&](auto kernel, int per) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)((rows + per - 1) / per)), dim3(256), 0, s, a);
    };
    const bool wide = splits > 8 && rows <= 2048;
    if (a.p.hd <= 64) wide ? go(k_paged_attn_join<16, 4>, 1) : go(k_paged_attn_join<16, 1>, 4);
    else if (a.p.hd <= 128) wide ? go(k_paged_attn_join<32, 4>, 1) : go(k_paged_attn_join<32, 1>, 4);
    else wide ? go(k_paged_attn_join<64, 4>, 1) : go(k_paged_attn_join<64, 1>, 4);
}

}  // namespace gh

using namespace gh;

extern "C" size_t gorch_hip_paged_attention_workspace_size(const gorch_hip_paged_kv* kv, const gorch_hip_paged_batch* b,
                                                           int num_q) {
    PagedAttnArgs a{};
    if (attn_args(kv, b, num_q, a) != GORCH_HIP_OK || b->tokens == 0 || b->seqs == 0) return 0;
    return attn_plan(a.p, num_q, b->max_new).bytes;
}

extern "C" int gorch_hip_paged_attention(void* stream, const gorch_hip_paged_kv* kv, const gorch_hip_paged_batch* b,
                                         const float* q, int num_q, float* out, int causal, void* workspace,
                                         size_t workspace_bytes) {
    PagedAttnArgs a{};
    GH_TRY(attn_args(kv, b, num_q, a));
    if (b->tokens == 0 || b->seqs == 0) return GORCH_HIP_OK;
    GH_REQUIRE(q && out, "gorch_hip_paged_attention: null q or out");
    const AttnPlan pl = attn_plan(a.p, num_q, b->max_new);
    // (a launch has less than 2^32 threads)
    GH_SUPPORTED((!pl.few || (long long)pl.few_tiles * kv->num_kv * pl.few_splits < 1 << 23) &&
                     (!pl.many || (long long)pl.many_tiles * kv->num_kv * pl.many_splits < 1 << 23),
                 "gorch_hip_paged_attention: too many sequences or tokens for one call");
    GH_REQUIRE(workspace_bytes >= pl.bytes && (workspace || pl.bytes == 0),
               "gorch_hip_paged_attention: workspace too small");
    GH_SUPPORTED(reinterpret_cast<uintptr_t>(q) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0 &&
                     reinterpret_cast<uintptr_t>(workspace) % 16 == 0,
                 "gorch_hip_paged_attention: q, out and the workspace must be 16-byte aligned");
    hipStream_t s = stream_of(stream);
    GH_TRY(bf16_gate(s));
    a.q = q;
    a.out = out;
    a.causal = causal != 0;
    const int splits = std::max(pl.few_splits, pl.many_splits);
    const size_t few_part = (size_t)pl.few_splits * pl.few_part, many_part = (size_t)pl.many_splits * pl.many_part;
    a.few_o = static_cast<float*>(workspace);
    a.part_o = a.few_o + few_part * a.p.hd;
    a.few_ml = reinterpret_cast<float2*>(a.part_o + many_part * a.p.hd);
    a.part_ml = a.few_ml + few_part;
    PagedAttnArgs few_args, many_args;
    split_args(a, pl, few_args, many_args);
    if (kv->dtype == GORCH_HIP_KV_MXFP4) launch_attn_mx(s, few_args, many_args, pl);
    else if (kv->dtype == GORCH_HIP_KV_E4M3) launch_attn_hd<true>(s, few_args, many_args, pl);
    else launch_attn_hd<false>(s, few_args, many_args, pl);
    GH_TRY(check_launch("paged_attention"));
    if (splits > 1) {
        a.hi_rows = pl.few ? pl.few_rows : -1;
        a.chunk = pl.few_chunk;
        a.splits = pl.few_splits;
        a.chunk2 = pl.many_chunk;
        a.splits2 = pl.many_splits;
        a.few_cap = pl.few_cap;
        a.few_rows = pl.few_part;
        a.part_rows = pl.many_part;
        if (pl.many_part == 0) {  // (of few rows alone, or read for nothing)
            a.part_o = a.few_o;
            a.part_ml = a.few_ml;
            a.part_rows = pl.few_part;
        }
        launch_join(s, a, splits);
        GH_TRY(check_launch("paged_attention join"));
    }
    count(CNT_ATTENTION);
    return finish(stream, GORCH_HIP_OK);
}
