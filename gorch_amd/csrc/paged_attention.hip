// paged_attention.hip — attention of ragged new tokens over a KV cache in
// pages (gorch_hip_gqa_attention_cached's mathematics, GQA.forwardCached
// nn/gqa.go:308-352): over the positions j that a token sees,
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(s_j - m),  s_j = log2(e) q . k_j / sqrt(hd),
// with the running maximum m and sum of one pass over the keys.
//
// Accuracy: the cache's values (bf16, or e4m3 codes widened to bf16) are exact
// matrix operands. q (scaled, f32) is split into three bf16 terms by
// truncation, which together hold its 24 bits, and so is every p: three
// v_mfma_f32_16x16x32_bf16 per product give f32 products summed in f32. Two
// terms would save a third of the matrix time and leave errors of 2^-16 of each
// q and p, 30 times those of f32 sums. An e4m3 row's scale
// multiplies the scores of its key (K) or its weight (V), never a rounded
// operand.
//
// Layout: S^T = K Q^T and O^T = V^T P^T, so a lane's column is one query row
// in both: a score's weight, and its row's maximum and rescaling, stay in the
// lane that needs them. A key's row is fetched in 16-byte chunks, lane l of a
// wave taking key l % 16, chunk 4 t + l / 16: that is the operand layout of K
// (in LDS, a fragment is 1 KB in lane order, free of bank conflicts), and V's
// fragments come out of the same layout by the LDS transpose reads, 16 columns
// at once. The keys of a 32-key tile are numbered so that a lane's scores (4
// keys of each 16) are its operand's 8 keys: the sum over keys has no order to
// keep.
#include <algorithm>
#include <cmath>

#include "paged.h"

namespace gh {

struct PagedAttnArgs {
    PagedArgs p;
    const float* q;
    float* out;
    float* part_o;   // [splits][part_rows][hd] unnormalised sums of a key range
    float2* part_ml; // [splits][part_rows] its maximum (log2) and weight sum
    long long part_rows;  // tokens * hq, row (token, head); or, of a few_cap > 0,
    int few_cap;          // seqs * few_cap * num_kv, row (sequence, row there, KV head)
    int hq, causal;
    float scale;     // log2(e) / sqrt(hd)
    FastDiv group;   // query heads per KV head
    int tiles;       // row tiles of this kernel's grid
    int per;         // of them, of each sequence (the kernel for few rows)
    int lo_rows, hi_rows;  // this kernel takes sequences of lo_rows <= rows <= hi_rows
    int chunk, splits;     // keys of a split; splits == 1: no partial results
    int last_first;        // the blocks of the last splits go first
    // the joining kernel: chunk and splits of sequences of more than hi_rows
    // rows, and with few_cap the partial sums of the others
    int chunk2, splits2;
    float* few_o;
    float2* few_ml;
    long long few_rows;
};

typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
#define GH_LDS __attribute__((address_space(3)))

// What rows and chunks that do not exist are read from.
__device__ __align__(16) uint32_t kZeros[128];

// f = t0 + t1 + t2 exactly (24 bits in 8 + 8 + 8; below 2^-110 the last ones
// fall away): each term f's leading bits, cut off.
__device__ __forceinline__ void split3(const float (&f)[8], bf16x8 (&t)[3]) {
    uint32_t w[3][4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint32_t u[3][2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const float x = f[2 * i + e];
            u[0][e] = __float_as_uint(x) & 0xffff0000u;
            const float r = x - __uint_as_float(u[0][e]);
            u[1][e] = __float_as_uint(r) & 0xffff0000u;
            u[2][e] = __float_as_uint(r - __uint_as_float(u[1][e]));
        }
#pragma unroll
        for (int k = 0; k < 3; k++) w[k][i] = __builtin_amdgcn_perm(u[k][1], u[k][0], 0x07060302u);
    }
#pragma unroll
    for (int k = 0; k < 3; k++) t[k] = __builtin_bit_cast(bf16x8, w[k]);
}

// Eight e4m3 codes as bf16 (exact).
__device__ __forceinline__ bf16x8 widen8(uint32_t a, uint32_t b) {
    bf16x2 w[4];
    w[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, false);
    w[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, true);
    w[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, false);
    w[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, true);
    return __builtin_bit_cast(bf16x8, w);
}

// Maximum and sum over the four lanes that hold one query row's scores (l, l
// + 16, l + 32, l + 48).
__device__ __forceinline__ float col_max(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float col_sum(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Sizes of a 32-key tile of K or V: NT 16-byte chunks of each lane for each of
// its two 16-key groups.
template <bool F8, int HD>
struct Tile {
    static constexpr int ES = F8 ? 1 : 2;
    static constexpr int NT = HD * ES / 64;
    static constexpr int NU = HD / 32;      // matrix steps along the head
    static constexpr int BYTES = 32 * HD * ES;
    static constexpr int GROUP = NT * 1024; // bytes of a 16-key group in LDS
    // first head column of lane group g in step u (8 columns)
    __device__ static __forceinline__ int col(int u, int g) {
        return F8 ? 64 * (u >> 1) + 16 * g + 8 * (u & 1) : 32 * u + 8 * g;
    }
    // step u's operand out of a lane's chunks
    __device__ static __forceinline__ bf16x8 frag(const u32x4 (&c)[NT], int u) {
        if constexpr (F8) return (u & 1) ? widen8(c[u >> 1][2], c[u >> 1][3]) : widen8(c[u >> 1][0], c[u >> 1][1]);
        else return __builtin_bit_cast(bf16x8, c[u]);
    }
    // V^T's operand for columns 16 dt .. 16 dt + 15 from a tile in LDS: slot
    // 4 j + i of lane group g is key 16 j + 4 g + i
    __device__ static __forceinline__ bf16x8 vfrag(const char* tile, int dt, int lane) {
        const int g = lane >> 4;
        if constexpr (F8) {
            const int r = (lane & 15) >> 1, c = lane & 1;
            const char* p = tile + (r >> 2) * GROUP + (dt >> 2) * 1024 + ((dt & 3) * 16 + 4 * g + (r & 3)) * 16 + 8 * c;
            const i32x2 w = __builtin_amdgcn_ds_read_tr8_b64_v2i32((GH_LDS i32x2*)p);
            return widen8((uint32_t)w[0], (uint32_t)w[1]);
        } else {
            const int r = (lane & 15) >> 2, c = lane & 3, ch = 2 * dt + (c >> 1);
            const char* p = tile + (ch >> 2) * 1024 + ((ch & 3) * 16 + 4 * g + r) * 16 + 8 * (c & 1);
            s16x4 w[2];
            w[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((GH_LDS s16x4*)p);
            w[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((GH_LDS s16x4*)(p + GROUP));
            return __builtin_bit_cast(bf16x8, w);
        }
    }
};

// Infinities and NaN in V. Their product with the weight 0 of a key that a row
// does not see is NaN, so a lane that finds some in its chunks of a tile turns
// them into zeros and notes, for every row that sees the key, +inf and -inf
// (NaN: both) for the column: bits [0 / 1][row][column] in LDS, added to the
// sums at the end. All that an ordinary tile pays is the test.
template <bool F8, int N>
__device__ __forceinline__ int any_nonfinite(const u32x4 (&c)[N]) {
    if constexpr (F8) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < N; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) m |= (c[i][e] & 0x7f7f7f7fu) + 0x01010101u;
        return (m & 0x80808080u) != 0;
    } else {
        u16x2 m = {0, 0};
#pragma unroll
        for (int i = 0; i < N; i++)
#pragma unroll
            for (int e = 0; e < 4; e++)
                m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, c[i][e] & 0x7fff7fffu));
        return m[0] >= 0x7f80 || m[1] >= 0x7f80;
    }
}
template <int BM, int HD>
struct OddBits {
    uint32_t any, bits[2][BM][HD / 32];
};
// One chunk of key `key` in LDS, columns col0 on; the block's rows are r0 .. r0
// + BM - 1 of sequence s.
template <bool F8, int BM, int HD>
__device__ __forceinline__ void clean_odd(OddBits<BM, HD>& odd, const PagedAttnArgs& a, const SeqAt& s, int r0, int key,
                                          int col0, char* chunk) {
    const int G = a.group.d, n = s.end - s.begin;
#pragma unroll 1
    for (int e = 0; e < (F8 ? 16 : 8); e++) {
        const int col = col0 + e;
        bool up, down;
        if constexpr (F8) {  // no infinities, NaN is 0x7f
            uint8_t* x = reinterpret_cast<uint8_t*>(chunk) + e;
            up = down = (*x & 0x7f) == 0x7f;
            if (up) *x = 0;
        } else {
            uint16_t* x = reinterpret_cast<uint16_t*>(chunk) + e;
            const int v = *x, m = v & 0x7fff;
            up = m > 0x7f80 || v == 0x7f80;
            down = m > 0x7f80 || v == 0xff80;
            if (up || down) *x = 0;
        }
        if (!up && !down) continue;
        odd.any = 1;
#pragma unroll 1
        for (int r = 0; r < BM && r0 + r < n * G; r++) {
            const int pos = a.causal ? s.len - n + (int)a.group.div((uint32_t)(r0 + r)) : s.len - 1;
            if (key > pos) continue;
            if (up) atomicOr(&odd.bits[0][r][col / 32], 1u << (col % 32));
            if (down) atomicOr(&odd.bits[1][r][col / 32], 1u << (col % 32));
        }
    }
}
template <int BM, int HD>
__device__ __forceinline__ floatx4 add_odd(const OddBits<BM, HD>& odd, int r, int c, floatx4 o) {
    for (int e = 0; e < 4; e++) {
        if (odd.bits[0][r][c / 32] >> (c % 32 + e) & 1u) o[e] += INFINITY;
        if (odd.bits[1][r][c / 32] >> (c % 32 + e) & 1u) o[e] -= INFINITY;
    }
    return o;
}

// A lane's fetch of one key row: its chunks, zeros where there is no row or
// (PART: hd < HD) no column.
template <bool F8, int HD, bool PART>
__device__ __forceinline__ void fetch_row(const void* pool, long long row, int hd, int g, u32x4 (&c)[Tile<F8, HD>::NT]) {
    constexpr int ES = Tile<F8, HD>::ES;
    const char* zero = reinterpret_cast<const char*>(kZeros);
    const char* p = row >= 0 ? static_cast<const char*>(pool) + row * (hd * ES) : zero;
#pragma unroll
    for (int t = 0; t < Tile<F8, HD>::NT; t++) {
        const int o = (4 * t + g) * 16;
        c[t] = *reinterpret_cast<const u32x4*>(PART && o >= hd * ES ? zero : p + o);
    }
}

// One wave's query rows (NR tiles of 16) and their running state.
template <bool F8, int HD, int NR>
struct Rows {
    using T = Tile<F8, HD>;
    bf16x8 q[NR][T::NU][3];
    floatx4 o[NR][HD / 16];
    float m[NR], l[NR];
    int pos[NR];   // the position of a lane's row (what it sees ends there), -1: none
    int first, last;  // smallest and largest of the wave's rows that exist

    // Rows r0 + 16 i + lane % 16 of a sequence: where they stand, and their q on
    // the way.
    template <bool PART>
    __device__ __forceinline__ void fetch(const PagedAttnArgs& a, const SeqAt& s, int r0, int kvh, float4 (&x)[NR][T::NU][2]) {
        const int lane = threadIdx.x & 63, g = lane >> 4, G = a.group.d, n = s.end - s.begin;
#pragma unroll
        for (int i = 0; i < NR; i++) {
            const int r = r0 + 16 * i + (lane & 15);
            const int tok = (int)a.group.div((uint32_t)r), h = kvh * G + r - tok * G;
            const bool live = r < n * G;
            pos[i] = live ? (a.causal ? s.len - n + tok : s.len - 1) : -1;
            const float* src = live ? a.q + ((size_t)(s.begin + tok) * a.hq + h) * a.p.hd : reinterpret_cast<const float*>(kZeros);
#pragma unroll
            for (int u = 0; u < T::NU; u++) {
                const int c = T::col(u, g);
                const float* p = live && (!PART || c < a.p.hd) ? src + c : reinterpret_cast<const float*>(kZeros);
                x[i][u][0] = *reinterpret_cast<const float4*>(p);
                x[i][u][1] = *reinterpret_cast<const float4*>(p + 4);
            }
        }
        const int at = r0 < n * G ? (int)a.group.div((uint32_t)r0) : 0;
        const int to = (int)a.group.div((uint32_t)(min(r0 + 16 * NR, n * G) - 1));
        first = r0 < n * G ? (a.causal ? s.len - n + at : s.len - 1) : 0x7fffffff;
        last = r0 < n * G ? (a.causal ? s.len - n + to : s.len - 1) : -1;
    }
    __device__ __forceinline__ void begin(const PagedAttnArgs& a, const float4 (&x)[NR][T::NU][2]) {
#pragma unroll
        for (int i = 0; i < NR; i++) {
#pragma unroll
            for (int u = 0; u < T::NU; u++) {
                const float4 y = x[i][u][0], z = x[i][u][1];
                const float f[8] = {y.x * a.scale, y.y * a.scale, y.z * a.scale, y.w * a.scale,
                                    z.x * a.scale, z.y * a.scale, z.z * a.scale, z.w * a.scale};
                split3(f, q[i][u]);
            }
            m[i] = -INFINITY;
            l[i] = 0.f;
#pragma unroll
            for (int d = 0; d < HD / 16; d++) o[i][d] = floatx4{0.f, 0.f, 0.f, 0.f};
        }
    }

    // Scores of a tile's two 16-key groups, K in LDS: sc[j][i] of row tile i holds
    // keys 16 j + 4 g .. + 3. A chunk is read while the one before is multiplied.
    __device__ __forceinline__ void score(const char* kt, floatx4 (&sc)[2][NR]) {
        const char* mine = kt + (threadIdx.x & 63) * 16;
        constexpr int PER = F8 ? 2 : 1;  // matrix steps of a chunk
        u32x4 c[1] = {*reinterpret_cast<const u32x4*>(mine)};
#pragma unroll
        for (int n = 0; n < 2 * T::NT; n++) {
            u32x4 ahead = c[0];
            if (n + 1 < 2 * T::NT) ahead = *reinterpret_cast<const u32x4*>(mine + (n + 1) * 1024);
            __builtin_amdgcn_sched_barrier(0);
            const int j = n / T::NT;
            if (n % T::NT == 0)
#pragma unroll
                for (int i = 0; i < NR; i++) sc[j][i] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int h = 0; h < PER; h++) {
                const bf16x8 k = F8 ? widen8(c[0][2 * h], c[0][2 * h + 1]) : __builtin_bit_cast(bf16x8, c[0]);
#pragma unroll
                for (int t = 2; t >= 0; t--)
#pragma unroll
                    for (int i = 0; i < NR; i++) sc[j][i] = mfma16x16x32(k, q[i][n % T::NT * PER + h][t], sc[j][i]);
            }
            c[0] = ahead;
        }
    }

    // A tile's 32 keys from key0 on, scores in sc[j][i], V in LDS. seen: bit k
    // for key k there; ksc / vsc: e4m3 scales of its keys (LDS).
    __device__ __forceinline__ void take(floatx4 (&sc)[2][NR], int key0, uint32_t seen, const float* ksc, const float* vsc,
                                         const char* vt) {
        const int lane = threadIdx.x & 63, g = lane >> 4;
        floatx4 ks[2], vs[2];
        if constexpr (F8) {
#pragma unroll
            for (int j = 0; j < 2; j++) {
                ks[j] = *reinterpret_cast<const floatx4*>(ksc + 64 * j + 4 * g);
                vs[j] = *reinterpret_cast<const floatx4*>(vsc + 64 * j + 4 * g);
            }
        }
        const bool edge = key0 + 31 > first || seen != 0xffffffffu;  // some row does not see some key
        if constexpr (F8)
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int i = 0; i < NR; i++) sc[j][i] *= ks[j];
        if (edge) {
#pragma unroll
            for (int i = 0; i < NR; i++)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int k = 16 * (e >> 2) + 4 * g + (e & 3);
                    const int sees = (int)(seen >> k & 1u) & (key0 + k <= pos[i] ? 1 : 0);
                    sc[e >> 2][i][e & 3] = sees ? sc[e >> 2][i][e & 3] : -INFINITY;
                }
        }
        bf16x8 p[NR][3];
        float al[NR];
        bool grew = false;
#pragma unroll
        for (int i = 0; i < NR; i++) {
            float top = sc[0][i][0];
#pragma unroll
            for (int e = 1; e < 8; e++) top = fmaxf(top, sc[e >> 2][i][e & 3]);
            const float mn = fmaxf(m[i], col_max(top)), use = mn == -INFINITY ? 0.f : mn;
            al[i] = __builtin_amdgcn_exp2f(m[i] - use);
            grew |= mn != m[i];
            m[i] = mn;
            float w[8], sum = 0.f;
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    float x = __builtin_amdgcn_exp2f(sc[j][i][e] - use);
                    sum += x;
                    if constexpr (F8) {
                        x *= vs[j][e];
                        // (a scale that is not finite, of a key that is not seen)
                        if (edge) x = sc[j][i][e] == -INFINITY ? 0.f : x;
                    }
                    w[4 * j + e] = x;
                }
            l[i] = l[i] * al[i] + sum;
            split3(w, p[i]);
        }
        if (__any(grew)) {
#pragma unroll
            for (int i = 0; i < NR; i++)
#pragma unroll
                for (int d = 0; d < HD / 16; d++) o[i][d] *= al[i];
        }
        // the next columns' operands are read while these are multiplied
        bf16x8 v = T::vfrag(vt, 0, lane);
#pragma unroll
        for (int d = 0; d < HD / 16; d++) {
            const bf16x8 ahead = d + 1 < HD / 16 ? T::vfrag(vt, d + 1, lane) : v;
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int t = 2; t >= 0; t--)
#pragma unroll
                for (int i = 0; i < NR; i++) o[i][d] = mfma16x16x32(v, p[i][t], o[i][d]);
            v = ahead;
        }
    }
};

// Where tile `tile` of BM flattened rows (token, head of the
// group) stands: the sequence and its first row. Tiles are numbered from
// floor(first row * G / BM) + s for sequence s, which leaves room for a part
// tile each.
template <int BM>
__device__ __forceinline__ bool find_tile(const PagedAttnArgs& a, int tile, SeqAt& s, int& r0) {
    const int G = a.group.d;
    if (!wave_seq(a.p, tile, [&](int i, int begin) { return begin * G / BM + i; }, s)) return false;
    r0 = (tile - (s.begin * G / BM + s.s)) * BM;
    const int rows = (s.end - s.begin) * G;
    return r0 >= 0 && r0 < rows && rows >= a.lo_rows && rows <= a.hi_rows;
}

// Row r of sequence s for KV head kvh among (token, head) rows, and among those
// of partial sums.
struct RowAt {
    size_t row, part;
};
__device__ __forceinline__ RowAt row_at(const PagedAttnArgs& a, const SeqAt& s, int r, int kvh) {
    const int G = a.group.d, tok = (int)a.group.div((uint32_t)r);
    RowAt at;
    at.row = (size_t)(s.begin + tok) * a.hq + kvh * G + (r - tok * G);
    at.part = a.few_cap ? ((size_t)s.s * a.few_cap + r) * a.p.num_kv + kvh : at.row;
    return at;
}

// Finished (or, of a split, partial) sums of four columns of a row.
__device__ __forceinline__ void put(const PagedAttnArgs& a, int split, const RowAt& at, int c, floatx4 o, float l) {
    if (a.splits == 1) {
        const float r = l == 0.f ? 0.f : 1.0f / l;  // a row that sees nothing: zeros
        *reinterpret_cast<floatx4*>(a.out + at.row * a.p.hd + c) = floatx4{o[0] * r, o[1] * r, o[2] * r, o[3] * r};
    } else {
        *reinterpret_cast<floatx4*>(a.part_o + ((size_t)split * a.part_rows + at.part) * a.p.hd + c) = o;
    }
}

// The page that holds key `key` of a sequence (of the last position for those
// past it), read without knowing the sequence's length and with no branch
// around the load; and the pool row of the key there, -1 if it is not below k1
// or on no page.
__device__ __forceinline__ int key_page(const PagedArgs& a, int s, int key) {
    return a.table[(size_t)s * a.max_pages + a.page.div((uint32_t)min(key, max(a.limit, 1) - 1))];
}
__device__ __forceinline__ long long key_row(const PagedArgs& a, int page, int key, int k1, int kvh) {
    const int p = min(key, max(a.limit, 1) - 1);
    const long long row = ((long long)page * a.num_kv + kvh) * a.page.d + (p - (int)(a.page.div((uint32_t)p) * a.page.d));
    const int there = (key < k1 ? 1 : 0) & ((unsigned)page < (unsigned)a.num_pages ? 1 : 0);
    return there ? row : -1;
}

// A block's rows of which none sees a key: zeros (or an empty partial result).
// (A path of its own: joined with the others before the loop over keys, it
// makes the compiler wait there for every load in flight.)
template <int BM>
__device__ __forceinline__ void put_nothing(const PagedAttnArgs& a, int split, const SeqAt& s, int r0, int kvh) {
    const int G = a.group.d, rows = min(BM, (s.end - s.begin) * G - r0), hd4 = a.p.hd / 4;
    for (int i = threadIdx.x; i < rows * hd4; i += blockDim.x) {
        const int r = r0 + i / hd4, c = 4 * (i % hd4);
        const RowAt at = row_at(a, s, r, kvh);
        put(a, split, at, c, floatx4{0.f, 0.f, 0.f, 0.f}, 0.f);
        if (a.splits > 1 && c == 0) a.part_ml[(size_t)split * a.part_rows + at.part] = make_float2(-INFINITY, 0.f);
    }
}

// The rows of a wave that has few: CW query rows of one sequence. CW = 16: a
// row a column of the operand and an instruction a term, as for many rows.
// CW = 4: a row in four columns, which hold its terms, so that one matrix
// instruction makes all three terms' products; a score is the sum of its row's
// columns, a lane's weights are the terms of its own columns, and the columns
// of O are added at the end. (24 single tokens of 12 heads beside 3 prompts
// 49 us with 16, 42 with 4; 64 of 2 rows per KV head 95.8 and 95.)
template <bool F8, int HD, int CW>
struct FewRows {
    using T = Tile<F8, HD>;
    static_assert(CW == 4 || CW == 16);
    static constexpr int TP = 16 / CW;  // columns of a row
    static constexpr int NP = CW == 4 ? 1 : 3;
    bf16x8 q[T::NU][NP];
    floatx4 o[HD / 16];
    float m, l;
    int pos, first;

    // a lane's operand p of the terms t
    __device__ __forceinline__ static bf16x8 pick(const bf16x8 (&t)[3], int p) {
        if constexpr (CW == 16) return t[p];
        const int k = (int)(threadIdx.x & 15) / CW;
        const uint32_t is[3] = {k == 0 ? ~0u : 0u, k == 1 ? ~0u : 0u, k == 2 ? ~0u : 0u};
        u32x4 r = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 3; i++) r |= __builtin_bit_cast(u32x4, t[i]) & is[i];
        return __builtin_bit_cast(bf16x8, r);
    }
    template <bool PART>
    __device__ __forceinline__ void fetch(const PagedAttnArgs& a, const SeqAt& s, int r0, int kvh, float4 (&x)[T::NU][2]) {
        const int lane = threadIdx.x & 63, g = lane >> 4, G = a.group.d, n = s.end - s.begin;
        const int r = r0 + (lane & (CW - 1));
        const int tok = (int)a.group.div((uint32_t)r), h = kvh * G + r - tok * G;
        const bool live = r < n * G;
        pos = live ? (a.causal ? s.len - n + tok : s.len - 1) : -1;
        const float* zero = reinterpret_cast<const float*>(kZeros);
        const float* src = a.q + ((size_t)(s.begin + tok) * a.hq + h) * a.p.hd;
#pragma unroll
        for (int u = 0; u < T::NU; u++) {
            const int c = T::col(u, g);
            const float* p = live && (!PART || c < a.p.hd) ? src + c : zero;
            x[u][0] = *reinterpret_cast<const float4*>(p);
            x[u][1] = *reinterpret_cast<const float4*>(p + 4);
        }
        first = a.causal ? s.len - n + (int)a.group.div((uint32_t)r0) : s.len - 1;
    }
    __device__ __forceinline__ void begin(const PagedAttnArgs& a, const float4 (&x)[T::NU][2]) {
#pragma unroll
        for (int u = 0; u < T::NU; u++) {
            const float4 y = x[u][0], z = x[u][1];
            const float f[8] = {y.x * a.scale, y.y * a.scale, y.z * a.scale, y.w * a.scale,
                                z.x * a.scale, z.y * a.scale, z.z * a.scale, z.w * a.scale};
            bf16x8 t[3];
            split3(f, t);
#pragma unroll
            for (int p = 0; p < NP; p++) q[u][p] = pick(t, p);
        }
        clear();
    }
    __device__ __forceinline__ void clear() {
        m = -INFINITY;
        l = 0.f;
#pragma unroll
        for (int d = 0; d < HD / 16; d++) o[d] = floatx4{0.f, 0.f, 0.f, 0.f};
    }
    // scores of a group's 16 keys: lane group g holds keys 4 g .. 4 g + 3
    __device__ __forceinline__ floatx4 score(const u32x4 (&c)[T::NT]) {
        floatx4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < T::NU; u++) {
            const bf16x8 k = T::frag(c, u);
#pragma unroll
            for (int p = NP - 1; p >= 0; p--) s = mfma16x16x32(k, q[u][p], s);
        }
        if constexpr (CW == 4)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                s[e] += dpp_f<0x128>(s[e]);  // 16 lanes rotated by 8
                s[e] += dpp_f<0x124>(s[e]);  // and by 4
            }
        return s;
    }
    // a tile's 32 keys from key0 on (as Rows::take)
    __device__ __forceinline__ void take(floatx4 (&sc)[2], int key0, uint32_t seen, const float* ksc, const float* vsc,
                                         const char* vt) {
        const int lane = threadIdx.x & 63, g = lane >> 4, k = (lane & 15) / CW;
        floatx4 vs[2];
        if constexpr (F8) {
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const floatx4 ks = *reinterpret_cast<const floatx4*>(ksc + 16 * j + 4 * g);
                vs[j] = *reinterpret_cast<const floatx4*>(vsc + 16 * j + 4 * g);
#pragma unroll
                for (int e = 0; e < 4; e++) sc[j][e] *= ks[e];
            }
        }
        const bool edge = key0 + 31 > first || seen != 0xffffffffu;
        if (edge) {
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int at = 16 * j + 4 * g + e;
                    const int sees = (int)(seen >> at & 1u) & (key0 + at <= pos ? 1 : 0);
                    sc[j][e] = sees ? sc[j][e] : -INFINITY;
                }
        }
        float top = sc[0][0];
#pragma unroll
        for (int e = 1; e < 8; e++) top = fmaxf(top, sc[e >> 2][e & 3]);
        const float mn = fmaxf(m, col_max(top)), use = mn == -INFINITY ? 0.f : mn;
        const float al = __builtin_amdgcn_exp2f(m - use);
        const bool grew = mn != m;
        m = mn;
        float w[8], sum = 0.f;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            float x = __builtin_amdgcn_exp2f(sc[e >> 2][e & 3] - use);
            sum += x;
            if constexpr (F8) {
                x *= vs[e >> 2][e & 3];
                if (edge) x = sc[e >> 2][e & 3] == -INFINITY ? 0.f : x;
            }
            w[e] = x;
        }
        l = l * al + sum;
        bf16x8 p[NP];
        if constexpr (CW == 4) {
            // a term's leading bits are cut off by the packing: term k of x is
            // x, what its first term leaves, or what both leave (the fourth
            // column's sum is never looked at)
            uint32_t u[8];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float r1 = w[e] - __uint_as_float(__float_as_uint(w[e]) & 0xffff0000u);
                const float r2 = r1 - __uint_as_float(__float_as_uint(r1) & 0xffff0000u);
                u[e] = __float_as_uint(k == 0 ? w[e] : (k == 1 ? r1 : r2));
            }
            uint32_t x[4];
#pragma unroll
            for (int e = 0; e < 4; e++) x[e] = __builtin_amdgcn_perm(u[2 * e + 1], u[2 * e], 0x07060302u);
            p[0] = __builtin_bit_cast(bf16x8, x);
        } else {
            bf16x8 t[3];
            split3(w, t);
#pragma unroll
            for (int i = 0; i < NP; i++) p[i] = t[i];
        }
        if (__any(grew)) {
#pragma unroll
            for (int d = 0; d < HD / 16; d++) o[d] *= al;
        }
#pragma unroll
        for (int d = 0; d < HD / 16; d++) {
            const bf16x8 v = T::vfrag(vt, d, lane);
#pragma unroll
            for (int i = NP - 1; i >= 0; i--) o[d] = mfma16x16x32(v, p[i], o[d]);
        }
    }
};

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
constexpr int kManyRows = 128;
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

struct AttnPlan {
    bool few, many;
    int few_width;  // rows of a tile of the kernel for few rows: 4 or 16
    int few_rows;   // sequences of up to so many rows go to it
    int few_per, few_tiles, many_tiles;
    int few_chunk, few_splits, many_chunk, many_splits;
    bool few_last_first;
    int few_cap;
    long long few_part, many_part;  // rows of partial sums
    size_t bytes;
};

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

template <bool F8, int HD, bool PART>
static void launch_attn(hipStream_t s, const PagedAttnArgs& base, const AttnPlan& pl) {
    constexpr int NR = HD <= 128 ? 2 : 1, NT = kManyRows / NR * 4;
    PagedAttnArgs few = base, many = base;
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
static void launch_attn_hd(hipStream_t s, const PagedAttnArgs& a, const AttnPlan& pl) {
    const int hd = a.p.hd;
    if (hd == 64) launch_attn<F8, 64, false>(s, a, pl);
    else if (hd < 64) launch_attn<F8, 64, true>(s, a, pl);
    else if (hd == 128) launch_attn<F8, 128, false>(s, a, pl);
    else if (hd < 128) launch_attn<F8, 128, true>(s, a, pl);
    else if (hd == 256) launch_attn<F8, 256, false>(s, a, pl);
    else launch_attn<F8, 256, true>(s, a, pl);
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
    if (kv->dtype == GORCH_HIP_KV_E4M3) launch_attn_hd<true>(s, a, pl);
    else launch_attn_hd<false>(s, a, pl);
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
