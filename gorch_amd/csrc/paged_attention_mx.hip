// paged_attention_mx.hip — attention over a paged cache in MXFP4: the running
// softmax of paged_attention.h over keys and values of four bits.
//
// Scores: a key's codes are an operand of the scaled matrix instructions as
// they lie in memory (lane l: key l % 16, 32 columns with their scale byte),
// against q's five 6-bit terms (mx.h): two or five instructions for 16 keys of
// 128 columns, where widened codes and three bf16 terms would take twelve.
// Values: their scales differ from key to key, along the sum, so codes are
// widened (exactly) to bf16 on their way to LDS, a lane's 32 columns under one
// scale, and multiplied as a bf16 cache's are. A value with scale byte 0 (below
// 2^-124) counts as zero.
#include "mx.h"
#include "paged_attention.h"

namespace gh {

// A lane's pieces of one key's row: 16 bytes of codes and a scale byte for each
// step of 128 columns; zeros where there is no row or no column.
template <int HD>
struct MxTile {
    static constexpr int NU = (HD + 127) / 128;
    static constexpr int GROUP = Tile<false, HD>::GROUP;  // bytes of 16 widened rows in LDS
};
template <int HD>
struct MxRow {
    u32x4 c[MxTile<HD>::NU];
    uint32_t s[MxTile<HD>::NU];
};
template <int HD, bool PART>
__device__ __forceinline__ void mx_fetch(const void* pool, const float* scales, long long row, int hd, int g, MxRow<HD>& r) {
    const char* zero = reinterpret_cast<const char*>(kZeros);
    const int gpr = PART ? (hd + 31) / 32 : HD / 32;
    const char* p = row >= 0 ? static_cast<const char*>(pool) + row * (PART ? hd / 2 : HD / 2) : zero;
    const uint8_t* s = row >= 0 ? reinterpret_cast<const uint8_t*>(scales) + row * gpr : reinterpret_cast<const uint8_t*>(kZeros);
#pragma unroll
    for (int u = 0; u < MxTile<HD>::NU; u++) {
        const int at = 4 * u + g;
        if constexpr (PART) {
            // (heads are multiples of 16 columns, 8 bytes)
            const u32x2 lo = *reinterpret_cast<const u32x2*>(32 * at < hd ? p + 16 * at : zero);
            const u32x2 hi = *reinterpret_cast<const u32x2*>(32 * at + 16 < hd ? p + 16 * at + 8 : zero);
            r.c[u] = u32x4{lo[0], lo[1], hi[0], hi[1]};
        } else {
            r.c[u] = *reinterpret_cast<const u32x4*>(at < gpr ? p + 16 * at : zero);
        }
        r.s[u] = *(at < gpr ? s + at : reinterpret_cast<const uint8_t*>(zero));
    }
}
// A value's pieces to a tile in LDS (16-key group j) as bf16; true where its
// scale is NaN (zeros are written).
template <int HD>
__device__ __forceinline__ bool mx_put(const MxRow<HD>& r, char* vt, int j, int lane) {
    const int g = lane >> 4, key = lane & 15;
    bool odd = false;
#pragma unroll
    for (int u = 0; u < MxTile<HD>::NU; u++) {
        if (HD < 128 && g >= HD / 32) continue;
        const bool nan = r.s[u] == kMxNaN, none = nan || r.s[u] == 0;
        odd |= nan;
        const float s = __uint_as_float(none ? 0x3f800000u : r.s[u] << 23);
        char* to = vt + j * MxTile<HD>::GROUP + (4 * u + g) * 1024 + key * 16;
#pragma unroll
        for (int i = 0; i < 4; i++) *reinterpret_cast<u32x4*>(to + i * 256) = mx_widen8(none ? 0u : r.c[u][i], s);
    }
    return odd;
}
// NaN groups of a value (key `key`) noted for every row that sees it.
template <int BM, int HD>
__device__ __forceinline__ void mx_note(OddBits<BM, HD>& odd, const PagedAttnArgs& a, const SeqAt& s, int r0, int key,
                                        const MxRow<HD>& v, int g) {
    const int G = a.group.d, n = s.end - s.begin;
#pragma unroll
    for (int u = 0; u < MxTile<HD>::NU; u++) {
        if (v.s[u] != kMxNaN || 4 * u + g >= HD / 32) continue;
        odd.any = 1;
#pragma unroll 1
        for (int r = 0; r < BM && r0 + r < n * G; r++) {
            const int pos = a.causal ? s.len - n + (int)a.group.div((uint32_t)(r0 + r)) : s.len - 1;
            if (key > pos) continue;
            atomicOr(&odd.bits[0][r][4 * u + g], ~0u);
            atomicOr(&odd.bits[1][r][4 * u + g], ~0u);
        }
    }
}

// The 32 columns from 128 u + 32 g on of row r of a sequence, scaled.
template <bool PART, int NU>
__device__ __forceinline__ void mx_fetch_q(const PagedAttnArgs& a, const SeqAt& s, int r, int kvh, int g, int hd, floatx4 (&x)[NU][8]) {
    const int G = a.group.d, n = s.end - s.begin;
    const int tok = (int)a.group.div((uint32_t)r), h = kvh * G + r - tok * G;
    const float* zero = reinterpret_cast<const float*>(kZeros);
    const float* src = a.q + ((size_t)(s.begin + tok) * a.hq + h) * a.p.hd;
#pragma unroll
    for (int u = 0; u < NU; u++)
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int c = 128 * u + 32 * g + 4 * i;
            x[u][i] = *reinterpret_cast<const floatx4*>(r < n * G && c < hd ? src + c : zero);
        }
}
__device__ __forceinline__ void mx_terms(const floatx4 (&x)[8], float scale, MxTerms& t) {
    floatx32 f;
#pragma unroll
    for (int i = 0; i < 32; i++) f[i] = x[i >> 2][i & 3] * scale;
    mx_split(f, t);
}

// FewRows over keys of four bits. CW = 4: a row in four columns, which hold its
// first four terms for one instruction; the fifth is the first column's of
// another.
template <int HD, int CW>
struct MxFewRows : FewRows<false, HD, CW> {
    static constexpr int NU = MxTile<HD>::NU, NQ = CW == 4 ? 2 : kMxTerms;
    u32x6 q6[NU][NQ];
    uint32_t sq[NU][2];

    template <bool PART>
    __device__ __forceinline__ void fetch(const PagedAttnArgs& a, const SeqAt& s, int r0, int kvh, floatx4 (&x)[NU][8]) {
        const int lane = threadIdx.x & 63, G = a.group.d, n = s.end - s.begin;
        const int r = r0 + (lane & (CW - 1));
        const int tok = (int)a.group.div((uint32_t)r);
        this->pos = r < n * G ? (a.causal ? s.len - n + tok : s.len - 1) : -1;
        this->first = a.causal ? s.len - n + (int)a.group.div((uint32_t)r0) : s.len - 1;
        mx_fetch_q<PART, NU>(a, s, r, kvh, lane >> 4, PART ? a.p.hd : HD, x);
    }
    __device__ __forceinline__ void begin(const PagedAttnArgs& a, const floatx4 (&x)[NU][8]) {
        const int k = (int)(threadIdx.x & 15) / CW;
#pragma unroll
        for (int u = 0; u < NU; u++) {
            MxTerms t;
            mx_terms(x[u], a.scale, t);
            if constexpr (CW == 4) {
#pragma unroll
                for (int e = 0; e < 6; e++) {
                    q6[u][0][e] = k == 0 ? t.t[0][e] : (k == 1 ? t.t[1][e] : (k == 2 ? t.t[2][e] : t.t[3][e]));
                    q6[u][1][e] = k == 0 ? t.t[4][e] : 0;
                }
                sq[u][0] = t.scale >> (8 * k);
            } else {
#pragma unroll
                for (int e = 0; e < kMxTerms; e++) q6[u][e] = t.t[e];
                sq[u][0] = t.scale;
            }
            sq[u][1] = t.last;
        }
        this->clear();
    }
    // scores of a group's 16 keys: lane group g holds keys 4 g .. 4 g + 3
    __device__ __forceinline__ floatx4 score(const MxRow<HD>& key) {
        floatx4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < NU; u++) {
            const i32x8 k = mx_op4(key.c[u]);
            s = mx_mfma_t<0, 0>(k, key.s[u], mx_op6(q6[u][NQ - 1]), sq[u][1], s);
            if constexpr (CW == 16) {
                s = mx_mfma_t<0, 3>(k, key.s[u], mx_op6(q6[u][3]), sq[u][0], s);
                s = mx_mfma_t<0, 2>(k, key.s[u], mx_op6(q6[u][2]), sq[u][0], s);
                s = mx_mfma_t<0, 1>(k, key.s[u], mx_op6(q6[u][1]), sq[u][0], s);
            }
            s = mx_mfma_t<0, 0>(k, key.s[u], mx_op6(q6[u][0]), sq[u][0], s);
        }
        if constexpr (CW == 4)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                s[e] += dpp_f<0x128>(s[e]);  // 16 lanes rotated by 8
                s[e] += dpp_f<0x124>(s[e]);  // and by 4
            }
        return s;
    }
};

// Few rows: as k_paged_attn_few, the values widened on their way to LDS.
template <int HD, bool PART, int CW>
struct MxFewBlock {
    static constexpr int NW = 4, NB = 2, OROW = HD + 4;
    static constexpr int STAGE = NW * Tile<false, HD>::BYTES, JOIN = NW * 16 * (OROW + 2) * 4;
    char lds[STAGE > JOIN ? STAGE : JOIN];
    OddBits<CW, HD> odd;
};
template <int HD, bool PART, int CW>
__device__ __forceinline__ void mx_few_tile(const PagedAttnArgs& a, const SeqAt& s, int r0, int kvh, int split,
                                            const int (&page)[MxFewBlock<HD, PART, CW>::NB + 1],
                                            MxFewBlock<HD, PART, CW>& sh) {
    using R = MxFewRows<HD, CW>;
    using Sh = MxFewBlock<HD, PART, CW>;
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
    char* vt = lds + wave * Tile<false, HD>::BYTES;
    struct Buf {
        MxRow<HD> k[2], v[2];
        uint32_t seen;
    } buf[NB];
    // row: the pool row of key lane % 32 of the tile
    auto fetch = [&](long long row, Buf& b) {
        const auto lo = __builtin_amdgcn_permlane16_swap((uint32_t)row, (uint32_t)row, false, false);
        const auto hi = __builtin_amdgcn_permlane16_swap((uint32_t)(row >> 32), (uint32_t)(row >> 32), false, false);
        b.seen = (uint32_t)__ballot(row >= 0);
#pragma unroll
        for (int j = 0; j < 2; j++) mx_fetch<HD, PART>(a.p.k, a.p.ks, (long long)(((uint64_t)hi[j] << 32) | lo[j]), a.p.hd, g, b.k[j]);
#pragma unroll
        for (int j = 0; j < 2; j++) mx_fetch<HD, PART>(a.p.v, a.p.vs, (long long)(((uint64_t)hi[j] << 32) | lo[j]), a.p.hd, g, b.v[j]);
    };
    R rows;
    int key0 = k0 + 32 * wave;
    int next = page[NB];  // the page of the next tile to fetch
    {
        floatx4 x[R::NU][8];
        rows.template fetch<PART>(a, s, r0, kvh, x);
#pragma unroll
        for (int i = 0; i < NB; i++) fetch(key_row(a.p, page[i], key0 + i * STEP + (lane & 31), k1, kvh), buf[i]);
        for (int i = threadIdx.x; i < (int)(sizeof(odd) / 4); i += 64 * NW) reinterpret_cast<uint32_t*>(&odd)[i] = 0;
        rows.begin(a, x);
    }
    __syncthreads();
    auto step = [&](Buf& b, int key) {
        const bool on = key < k1;
        const uint32_t here = b.seen;
        floatx4 scores[2];
        if (on) {
#pragma unroll
            for (int j = 0; j < 2; j++) scores[j] = rows.score(b.k[j]);
            bool nan = false;
#pragma unroll
            for (int j = 0; j < 2; j++) nan |= mx_put<HD>(b.v[j], vt, j, lane);
            if (__any(nan))
#pragma unroll 1
                for (int j = 0; j < 2; j++) mx_note<CW, HD>(odd, a, s, r0, key + 16 * j + (lane & 15), j ? b.v[1] : b.v[0], g);
        }
        const int after = key_page(a.p, s.s, key + (NB + 1) * STEP + (lane & 31));
        __builtin_amdgcn_sched_barrier(0);
        fetch(key_row(a.p, next, key + NB * STEP + (lane & 31), k1, kvh), b);
        next = after;
        if (on) rows.take(scores, key, here, nullptr, nullptr, vt);
    };
    for (; key0 < k1; key0 += NB * STEP)
#pragma unroll
        for (int i = 0; i < NB; i++) step(buf[i], key0 + i * STEP);
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
template <int HD, bool PART, int CW>
__device__ __forceinline__ void mx_few_block(const PagedAttnArgs& a, int block, MxFewBlock<HD, PART, CW>& sh) {
    using Sh = MxFewBlock<HD, PART, CW>;
    const int kvh = block % a.p.num_kv, rest = block / a.p.num_kv;
    const int tile = rest % a.tiles, split = a.last_first ? a.splits - 1 - rest / a.tiles : rest / a.tiles;
    SeqAt s;
    s.s = tile / a.per;
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
    if (r0 < rows) mx_few_tile<HD, PART, CW>(a, s, r0, kvh, split, page, sh);
}
template <int HD, bool PART, int CW>
__global__ __launch_bounds__(256, HD > 128 ? 1 : 2) void k_paged_attn_mx_few(PagedAttnArgs a) {
    __shared__ __align__(16) MxFewBlock<HD, PART, CW> sh;
    mx_few_block<HD, PART, CW>(a, (int)blockIdx.x, sh);
}

// Rows over keys of four bits.
template <int HD, int NR>
struct MxRowsOf : Rows<false, HD, NR> {
    static constexpr int NU = MxTile<HD>::NU;
    u32x6 q6[NR][NU][kMxTerms];
    uint32_t sq[NR][NU][2];

    template <bool PART>
    __device__ __forceinline__ void fetch(const PagedAttnArgs& a, const SeqAt& s, int r0, int kvh, floatx4 (&x)[NR][NU][8]) {
        const int lane = threadIdx.x & 63, G = a.group.d, n = s.end - s.begin;
#pragma unroll
        for (int i = 0; i < NR; i++) {
            const int r = r0 + 16 * i + (lane & 15), tok = (int)a.group.div((uint32_t)r);
            this->pos[i] = r < n * G ? (a.causal ? s.len - n + tok : s.len - 1) : -1;
            mx_fetch_q<PART, NU>(a, s, r, kvh, lane >> 4, PART ? a.p.hd : HD, x[i]);
        }
        const int at = r0 < n * G ? (int)a.group.div((uint32_t)r0) : 0;
        const int to = (int)a.group.div((uint32_t)(min(r0 + 16 * NR, n * G) - 1));
        this->first = r0 < n * G ? (a.causal ? s.len - n + at : s.len - 1) : 0x7fffffff;
        this->last = r0 < n * G ? (a.causal ? s.len - n + to : s.len - 1) : -1;
    }
    __device__ __forceinline__ void begin(const PagedAttnArgs& a, const floatx4 (&x)[NR][NU][8]) {
#pragma unroll
        for (int i = 0; i < NR; i++) {
#pragma unroll
            for (int u = 0; u < NU; u++) {
                MxTerms t;
                mx_terms(x[i][u], a.scale, t);
#pragma unroll
                for (int e = 0; e < kMxTerms; e++) q6[i][u][e] = t.t[e];
                sq[i][u][0] = t.scale;
                sq[i][u][1] = t.last;
            }
            this->m[i] = -INFINITY;
            this->l[i] = 0.f;
#pragma unroll
            for (int d = 0; d < HD / 16; d++) this->o[i][d] = floatx4{0.f, 0.f, 0.f, 0.f};
        }
    }
    // kt: a tile's codes, [group][step] KB in lane order; ks: their scale bytes
    __device__ __forceinline__ void score(const char* kt, const uint8_t* ks, floatx4 (&sc)[2][NR]) {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int j = 0; j < 2; j++) {
#pragma unroll
            for (int i = 0; i < NR; i++) sc[j][i] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int u = 0; u < NU; u++) {
                const i32x8 k = mx_op4(*reinterpret_cast<const u32x4*>(kt + ((j * NU + u) * 64 + lane) * 16));
                const uint32_t s = ks[(j * NU + u) * 64 + lane];
#pragma unroll
                for (int i = 0; i < NR; i++) sc[j][i] = mx_mfma_t<0, 0>(k, s, mx_op6(q6[i][u][4]), sq[i][u][1], sc[j][i]);
#pragma unroll
                for (int i = 0; i < NR; i++) sc[j][i] = mx_mfma_t<0, 3>(k, s, mx_op6(q6[i][u][3]), sq[i][u][0], sc[j][i]);
#pragma unroll
                for (int i = 0; i < NR; i++) sc[j][i] = mx_mfma_t<0, 2>(k, s, mx_op6(q6[i][u][2]), sq[i][u][0], sc[j][i]);
#pragma unroll
                for (int i = 0; i < NR; i++) sc[j][i] = mx_mfma_t<0, 1>(k, s, mx_op6(q6[i][u][1]), sq[i][u][0], sc[j][i]);
#pragma unroll
                for (int i = 0; i < NR; i++) sc[j][i] = mx_mfma_t<0, 0>(k, s, mx_op6(q6[i][u][0]), sq[i][u][0], sc[j][i]);
            }
        }
    }
};

// Many rows: 128 rows of a sequence a block, 16 NR a wave, tiles of 32 keys
// that all waves read from LDS. Waves 0 and 1 (of each step of 128 columns)
// fetch the keys' two groups, 2 and 3 the values', into registers a tile ahead
// and from there to the other of two stages, the values widened.
template <int HD>
struct MxManyBlock {
    alignas(16) char kt[2][2 * MxTile<HD>::NU * 1024], vt[2][Tile<false, HD>::BYTES];
    uint8_t ks[2][2 * MxTile<HD>::NU * 64];
    uint32_t seen_of[2][2];
    OddBits<kManyRows, HD> odd;
};
template <int HD, bool PART, int NR>
__device__ __forceinline__ void mx_many_block(const PagedAttnArgs& a, int block, MxManyBlock<HD>& sh) {
    constexpr int BM = kManyRows, NW = BM / (16 * NR), NU = MxTile<HD>::NU;
    static_assert(NW == 4 * NU);
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
    const int j = wave & 1, u = wave >> 2;
    const bool isv = (wave & 2) != 0;
    auto page_of = [&](int key0) { return key_page(a.p, s.s, key0 + 16 * j + (lane & 15)); };
    MxRow<64> raw;  // this wave's step
    uint32_t here;
    auto fetch = [&](int page, int key0) {
        const long long row = key_row(a.p, page, key0 + 16 * j + (lane & 15), k1, kvh);
        const char* zero = reinterpret_cast<const char*>(kZeros);
        const int hd = PART ? a.p.hd : HD, gpr = (hd + 31) / 32, at = 4 * u + g;
        const char* p = static_cast<const char*>(isv ? a.p.v : a.p.k) + row * (hd / 2) + 16 * at;
        const uint8_t* sp = reinterpret_cast<const uint8_t*>(isv ? a.p.vs : a.p.ks) + row * gpr + at;
        if constexpr (PART) {
            const u32x2 lo = *reinterpret_cast<const u32x2*>(row >= 0 && 32 * at < hd ? p : zero);
            const u32x2 hi = *reinterpret_cast<const u32x2*>(row >= 0 && 32 * at + 16 < hd ? p + 8 : zero);
            raw.c[0] = u32x4{lo[0], lo[1], hi[0], hi[1]};
        } else {
            raw.c[0] = *reinterpret_cast<const u32x4*>(row >= 0 && at < gpr ? p : zero);
        }
        raw.s[0] = *(row >= 0 && at < gpr ? sp : reinterpret_cast<const uint8_t*>(zero));
        here = (uint32_t)__ballot(row >= 0) & 0xffffu;
    };
    auto stage = [&](int key0, int b) {
        if (!isv) {
            *reinterpret_cast<u32x4*>(sh.kt[b] + ((j * NU + u) * 64 + lane) * 16) = raw.c[0];
            sh.ks[b][(j * NU + u) * 64 + lane] = (uint8_t)raw.s[0];
            if (lane == 0 && u == 0) sh.seen_of[b][j] = here;
        } else if (HD >= 128 || g < HD / 32) {
            const bool nan = raw.s[0] == kMxNaN, none = nan || raw.s[0] == 0;
            const float f = __uint_as_float(none ? 0x3f800000u : raw.s[0] << 23);
            char* to = sh.vt[b] + j * MxTile<HD>::GROUP + (4 * u + g) * 1024 + (lane & 15) * 16;
#pragma unroll
            for (int i = 0; i < 4; i++) *reinterpret_cast<u32x4*>(to + i * 256) = mx_widen8(none ? 0u : raw.c[0][i], f);
            if (nan) {
                sh.odd.any = 1;
#pragma unroll 1
                for (int r = 0; r < BM && r0 + r < n * G; r++) {
                    const int pos = a.causal ? s.len - n + (int)a.group.div((uint32_t)(r0 + r)) : s.len - 1;
                    if (key0 + 16 * j + (lane & 15) > pos) continue;
                    atomicOr(&sh.odd.bits[0][r][4 * u + g], ~0u);
                    atomicOr(&sh.odd.bits[1][r][4 * u + g], ~0u);
                }
            }
        }
    };
    MxRowsOf<HD, NR> rows;
    int next = page_of(k0 + 32);
    fetch(page_of(k0), k0);
    for (int i = threadIdx.x; i < (int)(sizeof(sh.odd) / 4); i += 64 * NW) reinterpret_cast<uint32_t*>(&sh.odd)[i] = 0;
    {
        floatx4 x[NR][NU][8];
        rows.template fetch<PART>(a, s, r0 + 16 * NR * wave, kvh, x);
        rows.begin(a, x);
    }
    __syncthreads();
    stage(k0, 0);
    fetch(next, k0 + 32);
    next = page_of(k0 + 64);
    __syncthreads();
    for (int key0 = k0, b = 0; key0 < k1; key0 += 32, b ^= 1) {
        stage(key0 + 32, b ^ 1);
        const int after = page_of(key0 + 96);
        fetch(next, key0 + 64);
        next = after;
        if (key0 <= rows.last) {
            floatx4 scores[2][NR];
            rows.score(sh.kt[b], sh.ks[b], scores);
            rows.take(scores, key0, sh.seen_of[b][0] | (sh.seen_of[b][1] << 16), nullptr, nullptr, sh.vt[b]);
        }
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0xc07f);  // LDS alone: the next tile's loads stay in flight
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
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
                put(a, split, at, c, sh.odd.any ? add_odd(sh.odd, r - r0, c, rows.o[i][d]) : rows.o[i][d], l);
            }
        if (a.splits > 1 && g == 0) a.part_ml[(size_t)split * a.part_rows + at.part] = make_float2(rows.m[i], l);
    }
}
template <int HD, bool PART, int NR>
__global__ __launch_bounds__(kManyRows / NR * 4, 2) void k_paged_attn_mx_many(PagedAttnArgs a) {
    __shared__ __align__(16) MxManyBlock<HD> sh;
    mx_many_block<HD, PART, NR>(a, (int)blockIdx.x, sh);
}
template <int HD, bool PART, int CW>
__global__ __launch_bounds__(256, 2) void k_paged_attn_mx_both(PagedAttnArgs many, PagedAttnArgs few, int many_blocks) {
    __shared__ __align__(16) union {
        MxManyBlock<HD> many;
        MxFewBlock<HD, PART, CW> few;
    } sh;
    if ((int)blockIdx.x < many_blocks) mx_many_block<HD, PART, 2>(many, (int)blockIdx.x, sh.many);
    else mx_few_block<HD, PART, CW>(few, (int)blockIdx.x - many_blocks, sh.few);
}

template <int HD, bool PART>
static void launch_mx(hipStream_t s, const PagedAttnArgs& few, const PagedAttnArgs& many, const AttnPlan& pl) {
    constexpr int NR = HD <= 128 ? 2 : 1;
    const unsigned few_blocks = (unsigned)(few.tiles * few.p.num_kv * few.splits);
    const unsigned many_blocks = (unsigned)(many.tiles * many.p.num_kv * many.splits);
    const auto width = [&](auto go) {
        if (pl.few_width == 4) go(std::integral_constant<int, 4>{});
        else go(std::integral_constant<int, 16>{});
    };
    if constexpr (HD <= 128)
        if (pl.few && pl.many) {
            width([&](auto w) {
                hipLaunchKernelGGL((k_paged_attn_mx_both<HD, PART, decltype(w)::value>), dim3(many_blocks + few_blocks), dim3(256), 0,
                                   s, many, few, (int)many_blocks);
            });
            return;
        }
    if (pl.few)
        width([&](auto w) {
            hipLaunchKernelGGL((k_paged_attn_mx_few<HD, PART, decltype(w)::value>), dim3(few_blocks), dim3(256), 0, s, few);
        });
    if (pl.many) hipLaunchKernelGGL((k_paged_attn_mx_many<HD, PART, NR>), dim3(many_blocks), dim3(kManyRows / NR * 4), 0, s, many);
}

void launch_attn_mx(hipStream_t s, const PagedAttnArgs& few, const PagedAttnArgs& many, const AttnPlan& pl) {
    const int hd = few.p.hd;
    if (hd == 64) launch_mx<64, false>(s, few, many, pl);
    else if (hd < 64) launch_mx<64, true>(s, few, many, pl);
    else if (hd == 128) launch_mx<128, false>(s, few, many, pl);
    else if (hd < 128) launch_mx<128, true>(s, few, many, pl);
    else if (hd == 256) launch_mx<256, false>(s, few, many, pl);
    else launch_mx<256, true>(s, few, many, pl);
}

}  // namespace gh
