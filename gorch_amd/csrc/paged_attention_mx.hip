// paged_attention_mx.hip — attention over a paged cache in MXFP4: the running
// softmax of paged_attention.h over keys and values of four bits.
//
// Scores: a key's codes are an operand of the scaled matrix instructions as
// they lie in memory (lane l: key l % 16, 32 columns with their scale byte),
// against q's five 6-bit terms (mx.h): two or five instructions for 16 keys of
// 128 columns, where widened codes and three bf16 terms would take twelve.
// Values: their scales differ from key to key, along the sum, so codes are
// widened (exactly) to bf16 on their way to LDS, a lane's 32 columns under one
// scale, and multiplied as a bf16 cache's are.
#include "mx.h"
#include "paged_attention.h"

namespace gh {

// What weights are relative to (m below) is set this much past the largest score,
// so that few tiles rescale the sums and no weight is above 1: sums leave f32's
// range where those of the other caches do. Weights stay normal numbers down to
// 2^-118 of the largest at least, in place of 2^-126.
constexpr float kSlack = 8.0f;

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
__device__ __forceinline__ void mx_fetch(const void* pool, long long row, int hd, int g, MxRow<HD>& r) {
    const char* zero = reinterpret_cast<const char*>(kZeros);
    const char* p = static_cast<const char*>(pool) + row * (PART ? hd / 2 : HD / 2);
#pragma unroll
    for (int u = 0; u < MxTile<HD>::NU; u++) {
        const int at = 4 * u + g;
        if constexpr (PART) {
            // (heads are multiples of 16 columns, 8 bytes)
            const u32x2 lo = *reinterpret_cast<const u32x2*>(32 * at < hd ? p + 16 * at : zero);
            const u32x2 hi = *reinterpret_cast<const u32x2*>(32 * at + 16 < hd ? p + 16 * at + 8 : zero);
            r.c[u] = u32x4{lo[0], lo[1], hi[0], hi[1]};
        } else {
            r.c[u] = *reinterpret_cast<const u32x4*>(HD >= 128 || g < HD / 32 ? p + 16 * at : zero);
        }
    }
}
// The scale bytes of a tile's K and V rows: as they are fetched, and dealt to
// the lanes when they have come. row: that of this lane's key (of 32); lo, hi:
// those of its key in each 16-key group. Heads of whole words of scales: lanes
// 0 .. 31 fetch their key's K words, the others V's.
template <int HD, bool PART>
struct MxScales {
    static constexpr int NU = MxTile<HD>::NU;
    static constexpr bool WORDS = !PART;
    uint32_t w[WORDS ? NU : 4 * NU];

    template <typename Pair>
    __device__ __forceinline__ void fetch(const PagedArgs& p, long long row, Pair lo, Pair hi, int g) {
        if constexpr (WORDS) {
            const uint8_t* from = reinterpret_cast<const uint8_t*>((threadIdx.x & 32) ? p.vs : p.ks) + row * (HD / 32);
#pragma unroll
            for (int u = 0; u < NU; u++) {
                if constexpr (HD == 64) w[u] = *reinterpret_cast<const uint16_t*>(from);
                else w[u] = *reinterpret_cast<const uint32_t*>(from + 4 * u);
            }
        } else {
            const int gpr = (p.hd + 31) / 32;
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const long long at = (long long)(((uint64_t)hi[j] << 32) | lo[j]) * gpr;
#pragma unroll
                for (int u = 0; u < NU; u++) {
                    const uint8_t* zero = reinterpret_cast<const uint8_t*>(kZeros);
                    const int i = 4 * u + g;
                    w[4 * u + j] = *(i < gpr ? reinterpret_cast<const uint8_t*>(p.ks) + at + i : zero);
                    w[4 * u + 2 + j] = *(i < gpr ? reinterpret_cast<const uint8_t*>(p.vs) + at + i : zero);
                }
            }
        }
    }
    __device__ __forceinline__ void deal(int g, MxRow<HD> (&k)[2], MxRow<HD> (&v)[2]) const {
#pragma unroll
        for (int u = 0; u < NU; u++) {
            if constexpr (WORDS) {
                const auto h = __builtin_amdgcn_permlane16_swap(w[u], w[u], false, false);
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const auto kv = __builtin_amdgcn_permlane32_swap(h[j], h[j], false, false);
                    // (of 64 columns the lanes of groups 2 and 3 have none: byte 0)
                    k[j].s[u] = kv[0] >> (8 * g) & 0xff;
                    v[j].s[u] = kv[1] >> (8 * g) & 0xff;
                }
            } else {
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    k[j].s[u] = w[4 * u + j];
                    v[j].s[u] = w[4 * u + 2 + j];
                }
            }
        }
    }
};
// The nibbles of codes that scale byte s takes past f32: 4 and 6 of 253, 2 to 6
// of 254, all of 255.
__device__ __forceinline__ uint32_t mx_past(uint32_t w, uint32_t s) {
    const uint32_t m = s == 253 ? w >> 2 & w >> 1 : (s == 254 ? w >> 2 : (s == kMxNaN ? ~0u : 0u));
    return (m & 0x11111111u) * 15u;
}
// A lane's codes as a tile of values holds them, and true where some are
// infinite or NaN (zeros are left, since a weight of 0 would make them NaN).
__device__ __forceinline__ bool mx_finite(u32x4& c, uint32_t s) {
    if (!__any(s >= 253)) return false;
    uint32_t past = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t p = mx_past(c[i], s);
        past |= p;
        c[i] &= ~p;
    }
    return past != 0;
}
// A value's pieces to its place (key `key`) of a tile in LDS as bf16; true
// where some are not finite.
template <int HD>
__device__ __forceinline__ bool mx_put(const MxRow<HD>& r, char* vt, int key, int lane) {
    const int g = lane >> 4;
    bool odd = false;
#pragma unroll
    for (int u = 0; u < MxTile<HD>::NU; u++) {
        if (HD < 128 && g >= HD / 32) continue;
        u32x4 codes = r.c[u];
        odd |= mx_finite(codes, r.s[u]);
        const bool none = r.s[u] == kMxNaN;
        const float s = mx_power(none ? 127 : r.s[u]);
        const uint32_t keep = none ? 0u : ~0u;  // (a mask: a choice per word becomes a branch)
        char* to = vt + (key >> 4) * MxTile<HD>::GROUP + (4 * u + g) * 1024 + (key & 15) * 16;
#pragma unroll
        for (int i = 0; i < 4; i++) *reinterpret_cast<u32x4*>(to + i * 256) = mx_widen8(codes[i] & keep, s);
    }
    return odd;
}
// The values that are not finite of a group of 32 (the word-th; of key `key`,
// codes c, scale byte s) noted for every row that sees them.
template <int BM, int HD>
__device__ __forceinline__ void mx_note(OddBits<BM, HD>& odd, const PagedAttnArgs& a, const SeqAt& s, int r0, int key,
                                        u32x4 c, uint32_t scale, int word) {
    if (scale < 253 || word >= HD / 32) return;
    const int G = a.group.d, n = s.end - s.begin;
    uint32_t up = 0, down = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t past = mx_past(c[i], scale);
#pragma unroll 1
        for (int e = 0; e < 8; e++) {
            const uint32_t bit = (past >> 4 * e & 1u) << (8 * i + e);
            const bool neg = (c[i] >> (4 * e + 3) & 1u) != 0;
            up |= neg && scale != kMxNaN ? 0u : bit;
            down |= neg || scale == kMxNaN ? bit : 0u;
        }
    }
    odd.any = 1;
#pragma unroll 1
    for (int r = 0; r < BM && r0 + r < n * G; r++) {
        const int pos = a.causal ? s.len - n + (int)a.group.div((uint32_t)(r0 + r)) : s.len - 1;
        if (key > pos) continue;
        atomicOr(&odd.bits[0][r][word], up);
        atomicOr(&odd.bits[1][r][word], down);
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

// FewRows over keys of four bits.
template <int HD>
struct MxFewRows : FewRows<false, HD, 16> {
    static constexpr int NU = MxTile<HD>::NU;
    u32x6 q6[NU][kMxTerms];
    uint32_t sq[NU][2];

    template <bool PART, typename Block>
    __device__ __forceinline__ void begin(const PagedAttnArgs& a, const SeqAt& s, int r0, int kvh, Block&) {
        const int lane = threadIdx.x & 63, G = a.group.d, n = s.end - s.begin;
        const int r = r0 + (lane & 15);
        const int tok = (int)a.group.div((uint32_t)r);
        this->pos = r < n * G ? (a.causal ? s.len - n + tok : s.len - 1) : -1;
        this->first = a.causal ? s.len - n + (int)a.group.div((uint32_t)r0) : s.len - 1;
        floatx4 x[NU][8];
        mx_fetch_q<PART, NU>(a, s, r, kvh, lane >> 4, PART ? a.p.hd : HD, x);
#pragma unroll
        for (int u = 0; u < NU; u++) {
            MxTerms t;
            mx_terms(x[u], a.scale, t);
#pragma unroll
            for (int e = 0; e < kMxTerms; e++) q6[u][e] = t.t[e];
            sq[u][0] = t.scale;
            sq[u][1] = t.last;
        }
        this->clear();
    }
    template <typename Block>
    __device__ __forceinline__ void ready(Block&) {}
    // scores of a group's 16 keys: lane group g holds keys 4 g .. 4 g + 3
    __device__ __forceinline__ floatx4 score(const MxRow<HD>& key) {
        floatx4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < NU; u++) {
            const i32x8 k = mx_op4(key.c[u]);
            s = mx_mfma_t<0, 0>(k, key.s[u], mx_op6(q6[u][4]), sq[u][1], s);
            s = mx_mfma_t<0, 3>(k, key.s[u], mx_op6(q6[u][3]), sq[u][0], s);
            s = mx_mfma_t<0, 2>(k, key.s[u], mx_op6(q6[u][2]), sq[u][0], s);
            s = mx_mfma_t<0, 1>(k, key.s[u], mx_op6(q6[u][1]), sq[u][0], s);
            s = mx_mfma_t<0, 0>(k, key.s[u], mx_op6(q6[u][0]), sq[u][0], s);
        }
        return s;
    }
    __device__ __forceinline__ void weigh(floatx4 (&sc)[2], int key0, uint32_t seen, const char* vt, char*) {
        this->take(sc, key0, seen, nullptr, nullptr, vt);
    }
    // a row's maximum and sum of weights, in the lanes of group 0
    __device__ __forceinline__ void totals(float& m, float& l, int& r) const {
        m = this->m;
        l = col_sum(this->l);
        r = (threadIdx.x & 63) < 16 ? (int)(threadIdx.x & 15) : -1;
    }
};

// Up to four rows: S = Q K^T, the first four terms of row g as rows 4 g .. 4 g
// + 3 of one operand and its fifth as row 4 g of another, so that a lane (g, c)
// adds up the score of row g and key c itself and a tile's 32 keys are two
// scores a lane (as columns of the other form they would be eight, each four
// times over: 57 -> 42 us for 64 conversations of up to 8,192 tokens). The
// weights' three bf16 terms then go through LDS to their places in P^T: column
// 4 t + g of the operand holds term t of row g; lanes c and c + 1 first trade
// one of their two weights, so that each has two neighbours there. (A numbering
// of the keys that made a lane's own two neighbours read every second row of a
// cache line: 74 us.) A block's first waves split q for all.
template <int HD>
struct MxFour {
    static constexpr int NU = MxTile<HD>::NU, TP = 4;
    u32x6 q6[NU][2];
    uint32_t sq[NU][2];
    floatx4 o[HD / 16];
    float m, l;
    int pos, first;

    template <bool PART, typename Block>
    __device__ __forceinline__ void begin(const PagedAttnArgs& a, const SeqAt& s, int r0, int kvh, Block& sh) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, c = lane & 15;
        const int G = a.group.d, n = s.end - s.begin, r = r0 + g;
        pos = r < n * G ? (a.causal ? s.len - n + (int)a.group.div((uint32_t)r) : s.len - 1) : -1;
        first = a.causal ? s.len - n + (int)a.group.div((uint32_t)r0) : s.len - 1;
        if (wave < 2 * NU) {
            // wave 2 u: terms 0 .. 3 of columns 128 u .., wave 2 u + 1: term 4
            const int u = wave >> 1, fifth = wave & 1, t = fifth ? 4 : (c & 3);
            floatx4 x[1][8];
            mx_fetch_q<PART, 1>(a, s, r0 + (c >> 2), kvh, 4 * u + g, PART ? a.p.hd : HD, x);
            floatx32 f;
#pragma unroll
            for (int i = 0; i < 32; i++) f[i] = x[0][i >> 2][i & 3] * a.scale;
            uint32_t sc;
            u32x6 six = mx_term(f, t, sc);
            if (fifth && (c & 3) != 0) six = u32x6{0, 0, 0, 0, 0, 0}, sc = sc == kMxNaN ? sc : 0;
            sh.q[wave].lo[lane] = u32x4{six[0], six[1], six[2], six[3]};
            sh.q[wave].hi[lane] = u32x2{six[4], six[5]};
            sh.q[wave].s[lane] = sc;
        }
        m = -INFINITY;
        l = 0.f;
#pragma unroll
        for (int d = 0; d < HD / 16; d++) o[d] = floatx4{0.f, 0.f, 0.f, 0.f};
    }
    template <typename Block>
    __device__ __forceinline__ void ready(Block& sh) {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int u = 0; u < NU; u++)
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const u32x4 lo = sh.q[2 * u + k].lo[lane];
                const u32x2 hi = sh.q[2 * u + k].hi[lane];
                q6[u][k] = u32x6{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1]};
                sq[u][k] = sh.q[2 * u + k].s[lane];
            }
    }
    // the score of row g and the group's key c
    __device__ __forceinline__ float score(const MxRow<HD>& key) {
        floatx4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < NU; u++) {
            const i32x8 k = mx_op4(key.c[u]);
            s = mx_mfma<0, 0>(mx_op6(q6[u][1]), sq[u][1], k, key.s[u], s);
            s = mx_mfma<0, 0>(mx_op6(q6[u][0]), sq[u][0], k, key.s[u], s);
        }
        return ((s[3] + s[2]) + s[1]) + s[0];
    }
    // pt: a KB of LDS of the wave's own
    __device__ __forceinline__ void weigh(float (&sc)[2], int key0, uint32_t seen, const char* vt, char* pt) {
        using T = Tile<false, HD>;
        const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
        if (key0 + 31 > first || seen != 0xffffffffu) {
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int sees = (int)(seen >> (16 * j + c) & 1u) & (key0 + 16 * j + c <= pos ? 1 : 0);
                sc[j] = sees ? sc[j] : -INFINITY;
            }
        }
        float top = fmaxf(sc[0], sc[1]);
        if (__any(top > m)) {
            top = fmaxf(top, dpp_f<kDppQuadSwap1>(top));
            top = fmaxf(top, dpp_f<kDppQuadSwap2>(top));
            top = fmaxf(top, dpp_f<kDppRowHalfMirror>(top));
            top = fmaxf(top, dpp_f<kDppRowMirror>(top));
            const float mn = fmaxf(m, top + kSlack), al = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.f : mn));
            m = mn;
            l *= al;
            // a column's row is its number's last two bits
            const float a0 = readlane_f(al, 0), a1 = readlane_f(al, 16), a2 = readlane_f(al, 32), a3 = readlane_f(al, 48);
            const float f = c & 2 ? (c & 1 ? a3 : a2) : (c & 1 ? a1 : a0);
#pragma unroll
            for (int d = 0; d < HD / 16; d++) o[d] *= f;
        }
        const float use = m == -INFINITY ? 0.f : m;
        // of keys c, c + 1 of group 0 (c even), or c - 1, c of group 1
        const float x0 = __builtin_amdgcn_exp2f(sc[0] - use), x1 = __builtin_amdgcn_exp2f(sc[1] - use);
        l += x0 + x1;
        const bool odd = (c & 1) != 0;
        const float other = dpp_f<kDppQuadSwap1>(odd ? x0 : x1);
        const float x[2] = {odd ? other : x0, odd ? x1 : other};
        uint32_t w[2][3];
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const float r1 = x[j] - __uint_as_float(__float_as_uint(x[j]) & 0xffff0000u);
            w[j][0] = __float_as_uint(x[j]);
            w[j][1] = __float_as_uint(r1);
            w[j][2] = __float_as_uint(r1 - __uint_as_float(__float_as_uint(r1) & 0xffff0000u));
        }
        char* to = pt + g * 64 + 16 * (c >> 2) + (odd ? 8 : 0) + 2 * (c & 2);
#pragma unroll
        for (int t = 0; t < 3; t++)
            *reinterpret_cast<uint32_t*>(to + t * 256) = __builtin_amdgcn_perm(w[1][t], w[0][t], 0x07060302u);
        const bf16x8 p = *reinterpret_cast<const bf16x8*>(pt + c * 64 + g * 16);
#pragma unroll
        for (int d = 0; d < HD / 16; d++) o[d] = mfma16x16x32(T::vfrag(vt, d, lane), p, o[d]);
    }
    __device__ __forceinline__ void totals(float& mt, float& lt, int& r) const {
        mt = m;
        lt = seg_sum<16>(l);
        r = (threadIdx.x & 15) == 0 ? (int)(threadIdx.x & 63) >> 4 : -1;
    }
};

// Few rows: as k_paged_attn_few, the values widened on their way to LDS. The
// floor is the codes: 64 tokens over 179,769 keys of 8 x 128 42 to 43 us (4.6 TB/s
// of 196 MB), with the join 46.6, where e4m3's 371 MB take 87. Two tiles are on
// their way; three and four were no faster (48.6, 48.1 us with the join against
// 46.3). One token over 777 keys 6.0 us, a chain of loads (page, keys, join).
template <int HD, bool PART, int CW>
struct MxFewBlock {
    static constexpr int NW = 4, NB = 2, OROW = HD + 4, PT = CW == 4 ? 1024 : 0;
    static constexpr int STAGE = NW * (Tile<false, HD>::BYTES + PT), JOIN = NW * 16 * (OROW + 2) * 4;
    char lds[STAGE > JOIN ? STAGE : JOIN];
    struct Operand {
        u32x4 lo[64];
        u32x2 hi[64];
        uint32_t s[64];
    };
    Operand q[CW == 4 ? 2 * MxTile<HD>::NU : 1];
    OddBits<CW, HD> odd;
};
template <int HD, bool PART, int CW>
__device__ __forceinline__ void mx_few_tile(const PagedAttnArgs& a, const SeqAt& s, int r0, int kvh, int split,
                                            const int (&page)[MxFewBlock<HD, PART, CW>::NB + 1],
                                            MxFewBlock<HD, PART, CW>& sh) {
    using R = typename std::conditional<CW == 4, MxFour<HD>, MxFewRows<HD>>::type;
    using Sh = MxFewBlock<HD, PART, CW>;
    constexpr int NW = Sh::NW, STEP = 32 * NW, NB = Sh::NB, OROW = Sh::OROW;
    char* const lds = sh.lds;
    auto& odd = sh.odd;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4;
    const int G = a.group.d, n = s.end - s.begin, mine = lane & 31;
    const int end_tok = (int)a.group.div((uint32_t)(min(r0 + CW, n * G) - 1));
    const int T1 = min((a.causal ? s.len - n + end_tok : s.len - 1) + 1, a.p.limit);
    const int k0 = split * a.chunk, k1 = a.splits == 1 ? T1 : min(T1, k0 + a.chunk);
    if (k0 >= k1) {
        if (split == 0) put_nothing<CW>(a, split, s, r0, kvh);
        return;
    }
    char* vt = lds + wave * (Tile<false, HD>::BYTES + Sh::PT);
    char* pt = vt + Tile<false, HD>::BYTES;
    struct Buf {
        MxRow<HD> k[2], v[2];
        MxScales<HD, PART> s;
        uint32_t seen;
    } buf[NB];
    // row: the pool row of this lane's key of the tile (-1: none; what row 0
    // holds is read then, and not looked at)
    auto fetch = [&](long long row, Buf& b) {
        b.seen = (uint32_t)__ballot(row >= 0);
        row = row < 0 ? 0 : row;
        const auto lo = __builtin_amdgcn_permlane16_swap((uint32_t)row, (uint32_t)row, false, false);
        const auto hi = __builtin_amdgcn_permlane16_swap((uint32_t)(row >> 32), (uint32_t)(row >> 32), false, false);
#pragma unroll
        for (int j = 0; j < 2; j++) mx_fetch<HD, PART>(a.p.k, (long long)(((uint64_t)hi[j] << 32) | lo[j]), a.p.hd, g, b.k[j]);
        b.s.fetch(a.p, row, lo, hi, g);
#pragma unroll
        for (int j = 0; j < 2; j++) mx_fetch<HD, PART>(a.p.v, (long long)(((uint64_t)hi[j] << 32) | lo[j]), a.p.hd, g, b.v[j]);
    };
    R rows;
    int key0 = k0 + 32 * wave;
    int next = page[NB];  // the page of the next tile to fetch
#pragma unroll
    for (int i = 0; i < NB; i++) fetch(key_row(a.p, page[i], key0 + i * STEP + mine, k1, kvh), buf[i]);
    for (int i = threadIdx.x; i < (int)(sizeof(odd) / 4); i += 64 * NW) reinterpret_cast<uint32_t*>(&odd)[i] = 0;
    rows.template begin<PART>(a, s, r0, kvh, sh);
    __syncthreads();
    rows.ready(sh);
    auto step = [&](Buf& b, int key) {
        const bool on = key < k1;
        const uint32_t here = b.seen;
        decltype(rows.score(b.k[0])) scores[2];
        if (on) {
            b.s.deal(g, b.k, b.v);
#pragma unroll
            for (int j = 0; j < 2; j++) scores[j] = rows.score(b.k[j]);
            bool nan = false;
#pragma unroll
            for (int j = 0; j < 2; j++) nan |= mx_put<HD>(b.v[j], vt, 16 * j + (lane & 15), lane);
            if (__any(nan)) {
                // (a dynamic choice of the rows themselves would put them into scratch memory)
#pragma unroll
                for (int u = 0; u < MxTile<HD>::NU; u++) {
                    const int w = 4 * u + g, c = lane & 15;
                    if (here >> c & 1u) mx_note<CW, HD>(odd, a, s, r0, key + c, b.v[0].c[u], b.v[0].s[u], w);
                    if (here >> (16 + c) & 1u) mx_note<CW, HD>(odd, a, s, r0, key + 16 + c, b.v[1].c[u], b.v[1].s[u], w);
                }
            }
        }
        const int after = key_page(a.p, s.s, key + (NB + 1) * STEP + mine);
        __builtin_amdgcn_sched_barrier(0);
        fetch(key_row(a.p, next, key + NB * STEP + mine, k1, kvh), b);
        next = after;
        if (on) rows.weigh(scores, key, here, vt, pt);
    };
    for (; key0 < k1; key0 += NB * STEP)
#pragma unroll
        for (int i = 0; i < NB; i++) step(buf[i], key0 + i * STEP);
    // the waves' sums, joined in wave order
    __syncthreads();
    float* jo = reinterpret_cast<float*>(lds);
    float* jm = jo + NW * 16 * OROW;
    float* jl = jm + NW * 16;
    {
        float m, l;
        int r;
        rows.totals(m, l, r);
        if (r >= 0) {
            jm[wave * 16 + r] = m;
            jl[wave * 16 + r] = l;
        }
    }
#pragma unroll
    for (int d = 0; d < HD / 16; d++)
        *reinterpret_cast<floatx4*>(jo + (wave * 16 + (lane & 15)) * OROW + 16 * d + 4 * g) = rows.o[d];
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
        page[i] = key_page(a.p, s.s, split * a.chunk + 32 * (int)(threadIdx.x >> 6) + i * 32 * Sh::NW +
                                         (int)(threadIdx.x & 31));
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
    floatx4 less[NR];
    float limit[NR];  // less: -m; limit: what a score less m must pass to move it, 0 (of m -infinity: 0, -infinity)
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
            this->m[i] = limit[i] = -INFINITY;
            this->l[i] = 0.f;
            less[i] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int d = 0; d < HD / 16; d++) this->o[i][d] = floatx4{0.f, 0.f, 0.f, 0.f};
        }
    }
    // kt: a tile's codes, [group][step] KB in lane order; ks: their scale bytes.
    // Scores less what weights are relative to: the first products take it as the
    // sum to add to, and what the smaller terms are added to is then small.
    __device__ __forceinline__ void score(const char* kt, const uint8_t* ks, floatx4 (&sc)[2][NR]) {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int j = 0; j < 2; j++) {
            i32x8 k[NU];
            uint32_t s[NU];
#pragma unroll
            for (int u = 0; u < NU; u++) {
                k[u] = mx_op4(*reinterpret_cast<const u32x4*>(kt + ((j * NU + u) * 64 + lane) * 16));
                s[u] = ks[(j * NU + u) * 64 + lane];
            }
#pragma unroll
            for (int i = 0; i < NR; i++) sc[j][i] = less[i];
            const auto term = [&](auto tc) {
                constexpr int t = decltype(tc)::value;
#pragma unroll
                for (int u = 0; u < NU; u++)
#pragma unroll
                    for (int i = 0; i < NR; i++)
                        sc[j][i] = mx_mfma_t<0, t & 3>(k[u], s[u], mx_op6(q6[i][u][t]), sq[i][u][t / 4], sc[j][i]);
            };
            term(std::integral_constant<int, 0>{});
            term(std::integral_constant<int, 1>{});
            term(std::integral_constant<int, 2>{});
            term(std::integral_constant<int, 3>{});
            term(std::integral_constant<int, 4>{});
        }
    }
    // A tile's 32 keys from key0 on, as Rows::take.
    __device__ __forceinline__ void take(floatx4 (&sc)[2][NR], int key0, uint32_t seen, const char* vt) {
        using T = Tile<false, HD>;
        const int lane = threadIdx.x & 63, g = lane >> 4;
        if (key0 + 31 > this->first || seen != 0xffffffffu) {
#pragma unroll
            for (int i = 0; i < NR; i++)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int k = 16 * (e >> 2) + 4 * g + (e & 3);
                    const int sees = (int)(seen >> k & 1u) & (key0 + k <= this->pos[i] ? 1 : 0);
                    sc[e >> 2][i][e & 3] = sees ? sc[e >> 2][i][e & 3] : -INFINITY;
                }
        }
        float top[NR];
        bool grew = false;
#pragma unroll
        for (int i = 0; i < NR; i++) {
            top[i] = sc[0][i][0];
#pragma unroll
            for (int e = 1; e < 8; e++) top[i] = fmaxf(top[i], sc[e >> 2][i][e & 3]);
            grew |= top[i] > limit[i];
        }
        if (__any(grew)) {
#pragma unroll
            for (int i = 0; i < NR; i++) {
                const float mn = fmaxf(this->m[i], col_max(top[i]) - less[i][0] + kSlack), use = mn == -INFINITY ? 0.f : mn;
                const float al = __builtin_amdgcn_exp2f(this->m[i] - use), by = use + less[i][0];
                this->m[i] = mn;
                less[i] = floatx4{-use, -use, -use, -use};
                limit[i] = mn == -INFINITY ? mn : 0.f;
                this->l[i] *= al;
#pragma unroll
                for (int e = 0; e < 8; e++) sc[e >> 2][i][e & 3] -= by;
#pragma unroll
                for (int d = 0; d < HD / 16; d++) this->o[i][d] *= al;
            }
        }
        bf16x8 p[NR][3];
#pragma unroll
        for (int i = 0; i < NR; i++) {
            float w[8], sum = 0.f;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                w[e] = __builtin_amdgcn_exp2f(sc[e >> 2][i][e & 3]);
                sum += w[e];
            }
            this->l[i] += sum;
            split3(w, p[i]);
        }
        bf16x8 v = T::vfrag(vt, 0, lane);
#pragma unroll
        for (int d = 0; d < HD / 16; d++) {
            const bf16x8 ahead = d + 1 < HD / 16 ? T::vfrag(vt, d + 1, lane) : v;
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int t = 2; t >= 0; t--)
#pragma unroll
                for (int i = 0; i < NR; i++) this->o[i][d] = mfma16x16x32(v, p[i][t], this->o[i][d]);
            v = ahead;
        }
    }
};

// Many rows: 128 rows of a sequence a block, 16 NR a wave, tiles of 32 keys
// that all waves read from LDS. Waves 0 and 1 (of each step of 128 columns)
// fetch the keys' two groups, 2 and 3 the values', into registers a tile ahead
// and from there to the other of two stages, the values widened. Bound by issue: for
// 2,048 tokens over 16,384 keys of 8 x 128 (16 query heads) 480 us with the join,
// 0.54 PFLOP/s of the product; vector instructions (exponentials, the weights'
// three terms) and matrix instructions take about half of the cycles each and
// overlap little. A reference that is moved by 8 at once took off 3%, and
// scores that come out less that reference 4% (of 525). No faster: the next
// tile's scores ahead in a third stage (543 against 540), a row tile's weights
// between the other's products (500 against 484; values are then read twice),
// K and V staged by all waves alike (490).
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
            u32x4 codes = raw.c[0];
            const bool far = mx_finite(codes, raw.s[0]), none = raw.s[0] == kMxNaN;
            const float f = mx_power(none ? 127 : raw.s[0]);
            const uint32_t keep = none ? 0u : ~0u;
            char* to = sh.vt[b] + j * MxTile<HD>::GROUP + (4 * u + g) * 1024 + (lane & 15) * 16;
#pragma unroll
            for (int i = 0; i < 4; i++) *reinterpret_cast<u32x4*>(to + i * 256) = mx_widen8(codes[i] & keep, f);
            if (far) mx_note<BM, HD>(sh.odd, a, s, r0, key0 + 16 * j + (lane & 15), raw.c[0], raw.s[0], 4 * u + g);
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
            rows.take(scores, key0, sh.seen_of[b][0] | (sh.seen_of[b][1] << 16), sh.vt[b]);
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
