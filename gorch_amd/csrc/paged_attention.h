// paged_attention.h — what the kernels of attention over a paged cache share:
// the running softmax of a wave's query rows, where rows and keys stand, and
// how sums are put down. Values of bf16 (and of four bits, widened to bf16) take
// F8 = false, e4m3 codes F8 = true.
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
#pragma once
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
static __device__ __align__(16) uint32_t kZeros[128];

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

constexpr int kManyRows = 128;  // rows of a block of the kernel for many

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
// Over a cache in MXFP4 (paged_attention_mx.hip), whose codes are two a byte
// and whose scales are bytes.
void launch_attn_mx(hipStream_t s, const PagedAttnArgs& few, const PagedAttnArgs& many, const AttnPlan& pl);

}  // namespace gh
