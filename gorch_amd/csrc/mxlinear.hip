// mxlinear.hip — Linear over MXFP4 weights (nn/module.go:61-88 with the
// weight's values rounded to four bits): y = residual + epi(x W^T + bias). The
// codes go to the matrix cores as they are; x goes there as the five 6-bit
// terms of mx.h, which hold it to 2^-24 of the largest of each 32 columns.
#include <algorithm>
#include <atomic>
#include <chrono>
#include <iterator>

#include "mx.h"
#include "stage_lds.h"

namespace gh {

struct MxLinearArgs {
    const float* x;
    const u32x4* wp;      // codes, gorch_hip_pack_mxfp4's layout
    const uint32_t* wsc;  // its scale words
    const float* bias;
    const float* residual;
    float* y;
    int M, N, K, epi;
    int nt, nk, nq;  // 16-row tiles of W, 128-column tiles, words of four of those
    char* terms;     // of more than 16 rows: x's operands (k_mx_terms)
    // of up to 16 rows: K in `slices` ranges of `chunks` * T column tiles, W's
    // row tiles `per` to a block; of several slices, partial sums [row
    // tile][slice][lane][4] and a counter for each block of row tiles, which
    // counts from `mark` on
    int slices, chunks, per, blocks;
    float* part;
    uint64_t* done;
    uint64_t mark;
};

// Barrier for LDS alone: loads into registers stay in flight.
__device__ __forceinline__ void lds_sync() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(kWaitLgkm0);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// The 32 values of row m, columns k .. k + 31 (zeros past K or without a row;
// no load stands under a branch, where each would be waited for by itself).
__device__ __forceinline__ floatx32 load_group(const float* x, int m, int M, int k, int K) {
    const float* row = x + (size_t)min(m, M - 1) * K;
    floatx4 f[8];
#pragma unroll
    for (int i = 0; i < 8; i++) f[i] = *reinterpret_cast<const floatx4*>(row + min(k + 4 * i, K - 4));
    floatx32 v;
#pragma unroll
    for (int i = 0; i < 8; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) v[4 * i + e] = m < M && k + 4 * i < K ? f[i][e] : 0.f;
    return v;
}

__device__ __forceinline__ void mx_store(const MxLinearArgs& a, int m, int n, float v) {
    if (a.bias) v += a.bias[n];
    if (a.epi == GORCH_HIP_EPI_GELU) v = gelu_gemm(v);
    const size_t at = (size_t)m * a.N + n;
    if (a.residual) v += a.residual[at];
    a.y[at] = v;
}

// x's operands made once for all blocks, 8 KB for each 16 rows and 128 columns:
// the terms' first 16 bytes, then their last 8, then the scale words, each in
// lane order; in row tile, column tile order.
constexpr int kTermBytes = 8192, kTerm8 = kMxTerms * 1024, kTermScale = kTerm8 + kMxTerms * 512;
// (Rows go through LDS: a lane's 128 bytes straight from memory would take 64
// lines a load, eight times.) Bound by memory: 2,000 x 4,096 12.2 us, 64 MB at
// the rate of a large copy (blocks that multiply would each split the same rows
// again).
__global__ __launch_bounds__(256) void k_mx_terms(MxLinearArgs a) {
    constexpr int ROW = 132;
    __shared__ __align__(16) float xs[4][16 * ROW];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = blockIdx.y, j = blockIdx.x * 4 + wave;
    if (j >= a.nk) return;
    {
        const int col = 128 * j + 4 * (lane & 31), from = min(col, a.K - 4);
        floatx4 f[8];
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const int m = 16 * i + 2 * k + (lane >> 5);
            f[k] = *reinterpret_cast<const floatx4*>(a.x + (size_t)min(m, a.M - 1) * a.K + from);
        }
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const int r = 2 * k + (lane >> 5);
            if (16 * i + r >= a.M || col >= a.K) f[k] = floatx4{0.f, 0.f, 0.f, 0.f};
            *reinterpret_cast<floatx4*>(xs[wave] + r * ROW + 4 * (lane & 31)) = f[k];
        }
    }
    floatx32 v;
#pragma unroll
    for (int k = 0; k < 8; k++) {
        const floatx4 f = *reinterpret_cast<const floatx4*>(xs[wave] + (lane & 15) * ROW + 32 * (lane >> 4) + 4 * k);
#pragma unroll
        for (int e = 0; e < 4; e++) v[4 * k + e] = f[e];
    }
    MxTerms r;
    mx_split(v, r);
    char* to = a.terms + ((size_t)i * a.nk + j) * kTermBytes;
#pragma unroll
    for (int q = 0; q < kMxTerms; q++) {
        *reinterpret_cast<u32x4*>(to + q * 1024 + lane * 16) = u32x4{r.t[q][0], r.t[q][1], r.t[q][2], r.t[q][3]};
        *reinterpret_cast<u32x2*>(to + kTerm8 + q * 512 + lane * 8) = u32x2{r.t[q][4], r.t[q][5]};
    }
    *reinterpret_cast<u32x2*>(to + kTermScale + lane * 8) = u32x2{r.scale, r.last};
}
// The same for up to 16 rows, where it is waited for: a wave a term. 16 x 1,600
// 3.6 us, of which a launch's latency is the most.
__global__ __launch_bounds__(64 * kMxTerms) void k_mx_terms16(MxLinearArgs a) {
    const int lane = threadIdx.x & 63, q = threadIdx.x >> 6, j = blockIdx.x;
    uint32_t s;
    const u32x6 t = mx_term(load_group(a.x, lane & 15, a.M, 128 * j + 32 * (lane >> 4), a.K), q, s);
    char* to = a.terms + (size_t)j * kTermBytes;
    *reinterpret_cast<u32x4*>(to + q * 1024 + lane * 16) = u32x4{t[0], t[1], t[2], t[3]};
    *reinterpret_cast<u32x2*>(to + kTerm8 + q * 512 + lane * 8) = u32x2{t[4], t[5]};
    reinterpret_cast<uint8_t*>(to + kTermScale + lane * 8)[q] = (uint8_t)s;
}

// Up to 16 rows of x. A block takes a slice of K and some row tiles of W: it
// splits its columns of x into terms in LDS once, and its 8 waves, WK along the
// columns and 8 / WK along the row tiles, stream 1 KB of codes a step into one
// instruction (kRow1: up to 3 rows, whose terms are rows of one operand) or
// five. For many columns of more rows another kernel has made the terms
// (kMade), which are loaded. The last of a row tile's blocks to finish adds up
// the slices, in their order. The floor is the weight's bytes: 1 x 1,024 x
// 151,936 16.2 us (5.1 TB/s of 83 MB); of small weights it is a chain of loads
// and a split: 1 x 1,024 x 4,096 4.5 us; 16 x 1,600 x 6,400 5.8 us after 3.6 for
// the terms (34 us when each block split all of x).
constexpr int kGemvWaves = 8;
constexpr int kGemvSlices = 16;
constexpr uint64_t kMarkStep = 32;  // a mark is a multiple of it, more than a counter counts
enum GemvKind { kRow1, kFive, kMade };
struct GemvLds {  // byte offsets of a block's LDS
    int p8, sc, red, bytes;
    __host__ __device__ GemvLds(int M, int tiles, bool made) {
        if (made) {
            p8 = kTerm8;
            sc = kTermScale;
            red = tiles * kTermBytes;
            bytes = red + kGemvWaves * 1024;
            return;
        }
        const int slots = tiles * 4 * kMxTerms * M;
        p8 = slots * 16;
        sc = p8 + slots * 8;
        red = sc + tiles * 4 * M * 8;
        bytes = red + kGemvWaves * 1024;
    }
};
// 16 bytes past the caches of an XCD (agent scope).
__device__ __forceinline__ void store_far(__amdgpu_buffer_rsrc_t rs, int at, floatx4 v) {
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), rs, at, 0, 16);
}
template <GemvKind KIND, int WK, int U>
__global__ __launch_bounds__(64 * kGemvWaves, 2) void k_mx_gemv(MxLinearArgs a) {
    constexpr int WN = kGemvWaves / WK, T = WK * U;
    constexpr bool ROW1 = KIND == kRow1, MADE = KIND == kMade;
    extern __shared__ __align__(16) char lds[];
    __shared__ int last;
    // blocks of the same row tiles run on one XCD (every eighth block)
    const int eight = blockIdx.x >> 3, slice = eight % a.slices, nb = eight / a.slices * 8 + (blockIdx.x & 7);
    if (nb >= a.blocks) return;
    const GemvLds at(a.M, min(T, a.nk), MADE);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, c = lane & 15;
    const int M = a.M, R = kMxTerms * M, wk = wave % WK, wn = wave / WK;
    const int t0 = nb * a.per, t1 = min(t0 + a.per, a.nt);
    uint64_t was = 0;
    if (a.slices > 1 && threadIdx.x == 0) was = __hip_atomic_load(a.done + nb, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    float* red = reinterpret_cast<float*>(lds + at.red);
    struct Step {
        u32x4 codes[U];
        uint32_t scale[(U + 3) / 4];
    };
    // U column tiles from j on of row tile t (what lies past the last is not looked at)
    const auto load = [&](Step& s, int t, int j) {
        const size_t tt = min(t, a.nt - 1);
#pragma unroll
        for (int u = 0; u < U; u += 4) s.scale[u / 4] = a.wsc[(tt * a.nq + (min(j + u, a.nk - 1) >> 2)) * 64 + lane];
#pragma unroll
        for (int u = 0; u < U; u++) s.codes[u] = __builtin_nontemporal_load(a.wp + (tt * a.nk + min(j + u, a.nk - 1)) * 64 + lane);
    };
    floatx4 acc = {0.f, 0.f, 0.f, 0.f};
    const auto multiply = [&](const Step& s, int j, int jl) {
        const auto one = [&](auto uc) {
            constexpr int u = decltype(uc)::value, B = u & 3;
            if constexpr (u < U) {
                if (j + u >= a.nk) return;
                const uint32_t sw = s.scale[u / 4] >> (U < 4 ? 8 * (j & 3) : 0);
                const i32x8 w = mx_op4(s.codes[u]);
                if constexpr (ROW1) {
                    const int slot = ((jl + u) * 4 + g) * R + min(c, R - 1);
                    const i32x8 six = mx_op6(*reinterpret_cast<const u32x4*>(lds + slot * 16),
                                             *reinterpret_cast<const u32x2*>(lds + at.p8 + slot * 8));
                    const uint32_t sx = *reinterpret_cast<const uint8_t*>(lds + at.sc + slot);
                    acc = mx_mfma<0, B>(six, sx, w, sw, acc);
                } else {
                    const int m = min(c, M - 1);
                    const char* made = lds + (jl + u) * kTermBytes;
                    const u32x2 sx = *reinterpret_cast<const u32x2*>(
                        MADE ? made + kTermScale + lane * 8 : lds + at.sc + (((jl + u) * 4 + g) * M + m) * 8);
                    const auto six = [&](int q) {
                        if constexpr (MADE)
                            return mx_op6(*reinterpret_cast<const u32x4*>(made + q * 1024 + lane * 16),
                                          *reinterpret_cast<const u32x2*>(made + kTerm8 + q * 512 + lane * 8));
                        const int slot = (((jl + u) * kMxTerms + q) * 4 + g) * M + m;
                        return mx_op6(*reinterpret_cast<const u32x4*>(lds + slot * 16),
                                      *reinterpret_cast<const u32x2*>(lds + at.p8 + slot * 8));
                    };
                    const i32x8 x4 = six(4), x3 = six(3), x2 = six(2), x1 = six(1), x0 = six(0);
                    acc = mx_mfma<0, B>(x4, sx[1], w, sw, acc);
                    acc = mx_mfma<3, B>(x3, sx[0], w, sw, acc);
                    acc = mx_mfma<2, B>(x2, sx[0], w, sw, acc);
                    acc = mx_mfma<1, B>(x1, sx[0], w, sw, acc);
                    acc = mx_mfma<0, B>(x0, sx[0], w, sw, acc);
                }
            }
        };
        one(std::integral_constant<int, 0>{});
        one(std::integral_constant<int, 1>{});
        one(std::integral_constant<int, 2>{});
        one(std::integral_constant<int, 3>{});
        one(std::integral_constant<int, 4>{});
        one(std::integral_constant<int, 5>{});
        one(std::integral_constant<int, 6>{});
        one(std::integral_constant<int, 7>{});
    };
    // x's columns of chunk ch as terms
    const auto split = [&](int j0) {
        const int groups = min(T, a.nk - j0) * 4, tasks = groups * M;
        const auto slot_of = [&](int m, int kb, int q) {
            const int j = kb >> 2, gg = kb & 3;
            return ROW1 ? (j * 4 + gg) * R + m * kMxTerms + q : ((j * kMxTerms + q) * 4 + gg) * M + m;
        };
        const auto put = [&](int slot, const u32x6& t) {
            *reinterpret_cast<u32x4*>(lds + slot * 16) = u32x4{t[0], t[1], t[2], t[3]};
            *reinterpret_cast<u32x2*>(lds + at.p8 + slot * 8) = u32x2{t[4], t[5]};
        };
        // (One row's first terms may add up to 2^128 where its other rows take some
        // off again: terms that are rows of an operand are held at half their size.)
        const auto byte_of = [](uint32_t s) { return (uint8_t)(ROW1 && s != kMxNaN ? s - 1 : s); };
        const auto scales_of = [&](int m, int kb) {  // bytes of the terms' scales
            return reinterpret_cast<uint8_t*>(lds + at.sc) + (ROW1 ? kb * R + m * kMxTerms : (kb * M + m) * 8);
        };
        if (tasks * kMxTerms <= 64 * kGemvWaves) {
            // few groups: a thread a term
            const int i = threadIdx.x / kMxTerms, q = threadIdx.x - i * kMxTerms;
            const int m = i / groups, kb = i - m * groups;
            const floatx32 x = load_group(a.x, i < tasks ? m : M, M, 128 * j0 + 32 * kb, a.K);
            uint32_t s;
            const u32x6 t = mx_term(x, q, s);
            if (i < tasks) {
                put(slot_of(m, kb, q), t);
                scales_of(m, kb)[q] = byte_of(s);
            }
        } else {
            for (int i = threadIdx.x; i < tasks; i += 64 * kGemvWaves) {
                const int m = i / groups, kb = i - m * groups;
                MxTerms r;
                mx_split(load_group(a.x, m, M, 128 * j0 + 32 * kb, a.K), r);
#pragma unroll
                for (int q = 0; q < kMxTerms; q++) put(slot_of(m, kb, q), r.t[q]);
                uint8_t* sc = scales_of(m, kb);
                if constexpr (ROW1) {
#pragma unroll
                    for (int q = 0; q < 4; q++) sc[q] = byte_of(r.scale >> (8 * q) & 0xff);
                    sc[4] = byte_of(r.last);
                } else {
                    *reinterpret_cast<u32x2*>(sc) = u32x2{r.scale, r.last};
                }
            }
        }
    };
    // a wave's sums of row tile t (lane: rows 4 g .. 4 g + 3 of x or of terms, column c) to y
    const auto finish = [&](int t, floatx4 d) {
        const int n = 16 * t + c;
        if constexpr (ROW1) {
            float* mine = red + wave * 256;
#pragma unroll
            for (int i = 0; i < 4; i++) mine[i * 64 + lane] = d[i];
            // (a wave reads back what it wrote)
            float v = 0.f;
#pragma unroll
            for (int q = kMxTerms - 1; q >= 0; q--) {
                const int row = min(g, M - 1) * kMxTerms + q;
                v += mine[(row & 3) * 64 + (row >> 2) * 16 + c];
            }
            if (g < M && n < a.N) mx_store(a, g, n, 2 * v);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (4 * g + i < M && n < a.N) mx_store(a, 4 * g + i, n, d[i]);
        }
    };
    // (partial sums of a block's row tiles: up to 2^31 bytes)
    const __amdgpu_buffer_rsrc_t part =
        make_rsrc(a.part + (size_t)t0 * a.slices * 256, (long long)(t1 - t0) * a.slices * 1024);
    // What the counter held before the call does not matter: the first block
    // that finds another call's mark, or anything else, puts this call's there
    // (one such exchange succeeds, since all start from what was there before),
    // and no block counts before it has seen the mark or tried that.
    const auto set_mark = [&] {
        if (a.slices > 1 && threadIdx.x == 0 && (was ^ a.mark) >= kMarkStep)
            __hip_atomic_compare_exchange_strong(a.done + nb, &was, a.mark, __ATOMIC_RELAXED, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    };
    // one column range and one round of row tiles after another
    const int j00 = slice * a.chunks * T, rounds = (t1 - t0 + WN - 1) / WN;
    Step s;
    load(s, t0 + wn, j00 + wk * U);
    for (int r = 0, ch = 0; r < rounds;) {
        const int j0 = j00 + ch * T, t = t0 + r * WN + wn;
        const bool more = ch + 1 < a.chunks && j0 + T < a.nk;
        if (ch > 0 || r == 0 || a.chunks > 1) {
            if (ch > 0 || r > 0) lds_sync();
            if (MADE && r == 0 && ch == 0) set_mark();
            if constexpr (MADE) {
                typedef __attribute__((address_space(1))) const uint32_t* global_ptr;
                typedef __attribute__((address_space(3))) uint32_t* lds_ptr;
                const int kb = min(T, a.nk - j0) * (kTermBytes / 1024);
                for (int k = wave; k < kb; k += kGemvWaves)
                    __builtin_amdgcn_global_load_lds((global_ptr)(a.terms + (size_t)j0 * kTermBytes + k * 1024 + lane * 16),
                                                     (lds_ptr)(lds + k * 1024), 16, 0, 0);
                block_sync_dma();
            } else {
                split(j0);
                if (r == 0 && ch == 0) set_mark();
                lds_sync();
            }
        }
        const int nr = more ? r : r + 1, nch = more ? ch + 1 : 0;
        const Step now = s;
        load(s, t0 + nr * WN + wn, j00 + nch * T + wk * U);
        multiply(now, j0 + wk * U, wk * U);
        r = nr;
        ch = nch;
        if (more) continue;
        floatx4 d = acc;
        acc = floatx4{0.f, 0.f, 0.f, 0.f};
        // the waves' sums along the columns, in wave order
        if constexpr (WK > 1) {
            if (r > 1) lds_sync();
            if (wk > 0) *reinterpret_cast<floatx4*>(red + (wave * 64 + lane) * 4) = d;
            lds_sync();
            if (wk > 0) continue;
#pragma unroll
            for (int k = 1; k < WK; k++) d += *reinterpret_cast<const floatx4*>(red + ((wave + k) * 64 + lane) * 4);
        }
        if (t >= t1) continue;
        if (a.slices == 1) finish(t, d);
        else store_far(part, ((t - t0) * a.slices + slice) * 1024 + lane * 16, d);
    }
    if (a.slices == 1) return;
    // Partial sums were stored, and are loaded, past the XCD's caches, so that
    // they are there once their stores are waited for; a fence that writes the
    // L2 back costs 38 us here (16 x 1600 x 6400: 48.6 us with it).
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0), lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (threadIdx.x == 0) last = __hip_atomic_fetch_add(a.done + nb, 1ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1 == a.mark + a.slices;
    __syncthreads();
    if (!last) return;
    if (threadIdx.x == 0) __hip_atomic_store(a.done + nb, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    for (int t = t0 + wave; t < t1; t += kGemvWaves) {
        floatx4 p[kGemvSlices];
#pragma unroll
        for (int k = 0; k < kGemvSlices; k++)  // (slices that there are not lie past the resource: zeros)
            p[k] = __builtin_bit_cast(floatx4, __builtin_amdgcn_raw_buffer_load_b128(
                part, k < a.slices ? ((t - t0) * a.slices + k) * 1024 + lane * 16 : kOutOfRange, 0, 16));
#pragma unroll
        for (int k = 1; k < kGemvSlices; k++) p[0] += p[k];
        finish(t, p[0]);
    }
}

// More rows: eight waves, WM along the rows of x (16 each) and WK along the
// columns, over NT row tiles of W. A wave's operands of x go from memory to its
// registers (no two waves need the same), W's codes and scale words to LDS,
// where the WM waves share them: rows two column tiles ahead, codes three, and
// the next tile's first codes from LDS before the block meets. A row tile's five
// products follow each other, which leaves two of three operands where they are
// (on all CUs the matrix cores run at what power allows, 6.2 PFLOP/s with the
// terms outermost, 6.9 so). 2,000 x 4,096 x 4,096 82 to 89 us (174 with x split by
// every block and one buffer): five products of 67 GFLOP, 49 us at 6.9 PFLOP/s;
// the rest is waits for x's terms, 64 KB a step and CU, each used 16 times. A
// larger tile would use them more often, but sums and three sets of operands
// take 320 of a lane's 512 registers already.
template <int MT, int NT, int WM>
struct GemmLds {
    static constexpr int WK = 8 / MT / WM, STAGE = NT * 1024, WORDS = (NT + 3) / 4 * 1024;
    static constexpr int RING = WK * (4 * STAGE + 2 * WORDS), JOIN = (WK - 1) * WM * MT * NT * 1024;
    static constexpr int BYTES = RING > JOIN ? RING : JOIN;
};
template <int MT, int NT, int WM>
__global__ __launch_bounds__(512 / MT, 2 / MT) void k_mx_gemm(MxLinearArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)  // (the host's pass cannot instantiate the loads in its lambdas)
    using L = GemmLds<MT, NT, WM>;
    constexpr int WK = L::WK, NB = NT < 2 ? NT : 2, DMA = (NT + WM - 1) / WM, ROWS = 2 * kMxTerms + 1;
    constexpr int KB = L::WORDS / 1024, LOADS = DMA + MT * ROWS + (KB + WM - 1) / WM;
    extern __shared__ __align__(16) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, c = lane & 15;
    const int wm = wave % WM, wk = wave / WM;
    // blocks that share x's rows run on one XCD (every eighth block)
    const int cols = (a.nt + NT - 1) / NT, each = (gridDim.x + 7) / 8, at = (blockIdx.x & 7) * each + (blockIdx.x >> 3);
    const int mt = (a.M + 15) / 16, by = at / cols, i0 = (by * WM + wm) * MT, t0 = (at - by * cols) * NT;
    if (by * WM * MT >= mt) return;
    // this wave's columns: whole words of four tiles
    const int per = (a.nq + WK - 1) / WK, q0 = wk * per, j1 = min(4 * (q0 + per), a.nk);
    // Resources in place of pointers, whose 64-bit sums per lane the compiler
    // would keep and spill: a wave's rows of x, and the row tiles of W that it
    // loads, which end with its columns (past them are zeros, whose products
    // change nothing: no branch stands around a step).
    __amdgpu_buffer_rsrc_t from[MT], wrs[DMA];
#pragma unroll
    for (int m = 0; m < MT; m++) from[m] = make_rsrc(a.terms + (size_t)min(i0 + m, mt - 1) * a.nk * kTermBytes, (long long)a.nk * kTermBytes);
#pragma unroll
    for (int i = 0; i < DMA; i++)
        wrs[i] = make_rsrc(a.wp + (size_t)min(t0 + min(i * WM + wm, NT - 1), a.nt - 1) * a.nk * 64, (long long)j1 * 1024);
    char* ring = lds + wk * 4 * L::STAGE;
    char* words = lds + WK * 4 * L::STAGE + wk * 2 * L::WORDS;
    struct Six {
        u32x4 lo[kMxTerms];
        u32x2 hi[kMxTerms], s;
    };
    typedef __attribute__((address_space(1))) const uint32_t* global_ptr;
    typedef __attribute__((address_space(3))) uint32_t* lds_ptr;
    typedef __attribute__((address_space(3))) void* lds_void;
    // Load i of column tile j's rows (to x), codes (to stage b) and scale words
    // (`word`, where it `has` one; a KB holds four row tiles', some waves load the same).
    const auto load = [&](auto ic, Six (&x)[MT], int j, int jc, int b, auto has, int word) {
        constexpr int i = decltype(ic)::value;
        if constexpr (i < DMA) {
            __builtin_amdgcn_raw_ptr_buffer_load_lds(wrs[i], (lds_void)(ring + b * L::STAGE + min(i * WM + wm, NT - 1) * 1024), 16,
                                                     lane * 16, min(jc, a.nk) * 1024, 0, 0);
        } else if constexpr (i < DMA + MT * ROWS) {
            constexpr int m = (i - DMA) / ROWS, k = (i - DMA) % ROWS, q = k / 2;
            const int at = min(j, a.nk - 1) * kTermBytes;
            if constexpr (k == 2 * kMxTerms) x[m].s = __builtin_amdgcn_raw_buffer_load_b64(from[m], lane * 8, at + kTermScale, 0);
            else if constexpr (k % 2 == 0) x[m].lo[q] = __builtin_amdgcn_raw_buffer_load_b128(from[m], lane * 16, at + q * 1024, 0);
            else x[m].hi[q] = __builtin_amdgcn_raw_buffer_load_b64(from[m], lane * 8, at + kTerm8 + q * 512, 0);
        } else if constexpr (decltype(has)::value) {
            const int k = ((i - DMA - MT * ROWS) * WM + wm) % KB, n = 4 * k + (lane >> 4);
            const uint32_t* p = a.wsc + ((size_t)min(t0 + n, a.nt - 1) * a.nq + min(word, a.nq - 1)) * 64 + (lane & 15) * 4;
            __builtin_amdgcn_global_load_lds((global_ptr)p, (lds_ptr)(words + (word & 1) * L::WORDS + k * 1024), 16, 0, 0);
        }
    };
    const auto loads = [&](auto lo, auto n, Six (&x)[MT], int j, int jc, int b, auto has, int word) {
        [&]<int... I>(std::integer_sequence<int, I...>) {
            (load(std::integral_constant<int, decltype(lo)::value + I>{}, x, j, jc, b, has, word), ...);
        }(std::make_integer_sequence<int, decltype(n)::value>{});
    };
    floatx4 acc[MT][NT];
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int n = 0; n < NT; n++) acc[m][n] = floatx4{0.f, 0.f, 0.f, 0.f};
    Six x[3][MT];
    uint32_t ws[NT];
    u32x4 w[2 * NB];
    constexpr bool EARLY = NT >= 2 * NB;  // the next words' registers are free before this step's last row tiles
    const auto word_of = [&](int n, int word) {
        ws[n] = *reinterpret_cast<const uint32_t*>(words + (word & 1) * L::WORDS + n * 256 + lane * 4);
    };
    // row tile n's codes of stage b (and where it `has` a word their scale words)
    const auto fetch = [&](u32x4& to, int n, int b, auto has, int word) {
        to = *reinterpret_cast<const u32x4*>(ring + b * L::STAGE + n * 1024 + lane * 16);
        if constexpr (decltype(has)::value) word_of(n, word);
    };
    {
        using Zero = std::integral_constant<int, 0>;
        loads(Zero{}, std::integral_constant<int, LOADS>{}, x[0], 4 * q0, 4 * q0, 0, std::true_type{}, q0);
        loads(Zero{}, std::integral_constant<int, LOADS>{}, x[1], 4 * q0 + 1, 4 * q0 + 1, 1, std::false_type{}, 0);
        loads(Zero{}, std::integral_constant<int, DMA>{}, x[0], 0, 4 * q0 + 2, 2, std::false_type{}, 0);
        block_sync_dma();
#pragma unroll
        for (int n = 0; n < NB; n++) fetch(w[n], n, 0, std::true_type{}, q0);
    }
    // A wave issues in order, and eight at once take 1,300 cycles to hand over a
    // column tile's loads: they go out between the products.
    const auto step = [&](auto uc, auto rc, int j) {
        constexpr int u = decltype(uc)::value, r = decltype(rc)::value % 3;
        // all loads have landed but those of the last step (and of its words)
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(wait_vm(DMA + MT * ROWS, true));
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        const auto& now = x[r];
        [&]<int... N>(std::integer_sequence<int, N...>) {
            const auto one = [&](auto nc) {
                constexpr int n = decltype(nc)::value, from = n * LOADS / NT, to = (n + 1) * LOADS / NT;
                // (slots of w turn over NT row tiles a step)
                constexpr int slot = (NT % (2 * NB) ? n + u * NT : n) % (2 * NB), ahead = (slot + NB) % (2 * NB);
                loads(std::integral_constant<int, from>{}, std::integral_constant<int, to - from>{}, x[(r + 2) % 3], j + 2, j + 3, (u + 3) & 3,
                      std::bool_constant<u == 0>{}, j / 4 + 1);
                if constexpr (n + NB < NT) fetch(w[ahead], n + NB, u, std::bool_constant<u == 0>{}, j / 4);
                else fetch(w[ahead], n + NB - NT, (u + 1) & 3, std::bool_constant<u == 3 && EARLY>{}, j / 4 + 1);
                if constexpr (u == 0 && !EARLY) word_of(n, j / 4);
                __builtin_amdgcn_sched_barrier(0);
                const i32x8 v = mx_op4(w[slot]);
                const auto product = [&](auto qc) {
                    constexpr int q = decltype(qc)::value;
#pragma unroll
                    for (int m = 0; m < MT; m++)
                        acc[m][n] = mx_mfma<q & 3, u>(mx_op6(now[m].lo[q], now[m].hi[q]), now[m].s[q / 4], v, ws[n], acc[m][n]);
                };
                product(std::integral_constant<int, 4>{});
                product(std::integral_constant<int, 3>{});
                product(std::integral_constant<int, 2>{});
                product(std::integral_constant<int, 1>{});
                product(std::integral_constant<int, 0>{});
                __builtin_amdgcn_sched_barrier(0);
            };
            (one(std::integral_constant<int, N>{}), ...);
        }(std::make_integer_sequence<int, NT>{});
    };
    const auto quad = [&](auto rc, int q) {
        constexpr int r = decltype(rc)::value;
        [&]<int... U>(std::integer_sequence<int, U...>) {
            (step(std::integral_constant<int, U>{}, std::integral_constant<int, r + U>{}, 4 * (q0 + q) + U), ...);
        }(std::make_integer_sequence<int, 4>{});
    };
    for (int q = 0;; q++) {
        quad(std::integral_constant<int, 0>{}, q);
        if (++q >= per) break;
        quad(std::integral_constant<int, 1>{}, q);
        if (++q >= per) break;
        quad(std::integral_constant<int, 2>{}, q);
        if (q + 1 >= per) break;
    }
    block_sync_dma();
    if constexpr (WK > 1) {
        block_sync_dma();
        floatx4* join = reinterpret_cast<floatx4*>(lds);
        if (wk > 0)
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int n = 0; n < NT; n++) join[((((wk - 1) * WM + wm) * MT + m) * NT + n) * 64 + lane] = acc[m][n];
        __syncthreads();
        if (wk > 0) return;
#pragma unroll
        for (int k = 0; k < WK - 1; k++)
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int n = 0; n < NT; n++) acc[m][n] += join[(((k * WM + wm) * MT + m) * NT + n) * 64 + lane];
    }
    // (what is added is asked for by up to four row tiles at a time)
    constexpr int EB = NT < 4 ? NT : 4;
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int n0 = 0; n0 < NT; n0 += EB) {
            float bias[EB], r[EB][4];
#pragma unroll
            for (int n = 0; n < EB; n++) {
                const int col = min(16 * (t0 + n0 + n) + c, a.N - 1);
                bias[n] = a.bias ? a.bias[col] : 0.f;
#pragma unroll
                for (int i = 0; i < 4; i++)
                    r[n][i] = a.residual ? a.residual[(size_t)min(16 * (i0 + m) + 4 * g + i, a.M - 1) * a.N + col] : 0.f;
            }
#pragma unroll
            for (int n = 0; n < EB; n++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int row = 16 * (i0 + m) + 4 * g + i, col = 16 * (t0 + n0 + n) + c;
                    float v = acc[m][n0 + n][i] + bias[n];
                    if (a.epi == GORCH_HIP_EPI_GELU) v = gelu_gemm(v);
                    if (row < a.M && col < a.N) a.y[(size_t)row * a.N + col] = v + r[n][i];
                }
        }
#endif
}

// A workspace begins with the counters of every shape's blocks (at most 128 of
// several slices), so that one may serve calls of all sizes in turn; a call finds
// in them what it will.
constexpr size_t kCounterBytes = 1024;
// A counter's value that no workspace holds by chance (2^-58): the bits of a
// count mixed with the process's start, never 0, which a call leaves behind. A
// captured call keeps its own; its replays follow each other.
static uint64_t next_mark() {
    static std::atomic<uint64_t> calls{0};
    static const uint64_t seed = (uint64_t)std::chrono::system_clock::now().time_since_epoch().count() ^ ((uint64_t)(uintptr_t)&calls << 20);
    uint64_t z = seed + 0x9e3779b97f4a7c15ull * (calls.fetch_add(1, std::memory_order_relaxed) + 1);
    z = (z ^ (z >> 30)) * 0xbf58476d1ce4e5b9ull;
    z = (z ^ (z >> 27)) * 0x94d049bb133111ebull;
    return ((z ^ (z >> 31)) | 1ull << 63) / kMarkStep * kMarkStep;
}
static size_t terms_bytes(int M, int K) { return kCounterBytes + (size_t)((M + 15) / 16) * ((K + 127) / 128) * kTermBytes; }

// How the rows of a decode step are cut into blocks: slices of K (at most 16),
// row tiles per block, waves along the columns.
struct GemvPlan {
    GemvKind kind;
    int tiles, slices, chunks, per, blocks, wk;
    size_t terms, part, bytes;
};
static GemvPlan gemv_plan(int M, int N, int K) {
    GemvPlan p{};
    const int nt = (N + 15) / 16, nk = (K + 127) / 128;
    // (a block splits 512 groups, M * nk = 128, in 1.7 us; another kernel takes
    // 3 us for all of them)
    p.kind = M <= 3 ? kRow1 : ((long long)M * nk >= (M > 8 ? 128 : 257) ? kMade : kFive);
    // Column tiles whose terms a block holds: up to 64 KB of them, a round of
    // splitting; made ones 128 KB.
    const int most = p.kind == kMade ? 16 : (M <= 4 ? 32 : (M <= 8 ? 16 : 8));
    p.tiles = 8;
    while (p.tiles < nk && p.tiles < most) p.tiles *= 2;
    const int ranges = (nk + p.tiles - 1) / p.tiles;
    p.slices = std::min(ranges, kGemvSlices);
    // (joining slices takes 2.3 us, as much as loading the terms of 48 tiles)
    if (p.kind == kMade) p.slices = nk <= 48 ? 1 : std::min((nk + 31) / 32, kGemvSlices);
    p.chunks = (ranges + p.slices - 1) / p.slices;
    p.slices = (ranges + p.chunks - 1) / p.chunks;
    // 256 blocks, one a CU, of which each has a row tile at least
    const int blocks = std::max(1, 256 / p.slices);
    p.per = (nt + blocks - 1) / blocks;
    p.blocks = (nt + p.per - 1) / p.per;
    p.wk = 8;
    while (p.wk > p.tiles / 8 && kGemvWaves / p.wk < p.per) p.wk /= 2;
    p.terms = p.kind == kMade ? (size_t)nk * kTermBytes : 0;
    p.part = p.slices == 1 ? 0 : (size_t)p.slices * nt * 1024;
    p.bytes = p.terms + p.part;
    if (p.bytes) p.bytes += kCounterBytes;
    return p;
}

template <GemvKind KIND, int WK, int U>
static int launch_mx_gemv_t(hipStream_t s, const MxLinearArgs& a) {
    static_assert(KIND != kMade || WK * U * kTermBytes + kGemvWaves * 1024 <= 160 << 10);
    const int bytes = GemvLds(a.M, std::min(WK * U, a.nk), KIND == kMade).bytes;
    if (bytes > 64 << 10)
        GH_TRY(check(hipFuncSetAttribute(reinterpret_cast<const void*>(&k_mx_gemv<KIND, WK, U>),
                                         hipFuncAttributeMaxDynamicSharedMemorySize, bytes), "mx_gemv attribute"));
    hipLaunchKernelGGL((k_mx_gemv<KIND, WK, U>), dim3((a.blocks + 7) / 8 * 8 * a.slices), dim3(64 * kGemvWaves), bytes, s, a);
    return GORCH_HIP_OK;
}
template <int WK, int U>
static int launch_mx_gemv_f(hipStream_t s, const MxLinearArgs& a, const GemvPlan& p) {
    if (p.kind == kRow1) return launch_mx_gemv_t<kRow1, WK, U>(s, a);
    if constexpr (WK * U <= 16)
        if (p.kind == kMade) return launch_mx_gemv_t<kMade, WK, U>(s, a);
    return launch_mx_gemv_t<kFive, WK, U>(s, a);
}
static int launch_mx_gemv(hipStream_t s, MxLinearArgs a, char* ws) {
    const GemvPlan p = gemv_plan(a.M, a.N, a.K);
    static_assert(kCounterBytes >= 256 / 2 * sizeof(uint64_t) && kMarkStep > kGemvSlices);
    a.slices = p.slices;
    a.chunks = p.chunks;
    a.per = p.per;
    a.blocks = p.blocks;
    a.done = reinterpret_cast<uint64_t*>(ws);
    a.mark = p.slices > 1 ? next_mark() : 0;
    a.terms = ws + kCounterBytes;
    a.part = reinterpret_cast<float*>(ws + kCounterBytes + p.terms);
    if (p.kind == kMade) hipLaunchKernelGGL(k_mx_terms16, dim3(a.nk), dim3(64 * kMxTerms), 0, s, a);
    if (p.tiles == 8) {
        if (p.wk == 8) return launch_mx_gemv_f<8, 1>(s, a, p);
        if (p.wk == 4) return launch_mx_gemv_f<4, 2>(s, a, p);
        if (p.wk == 2) return launch_mx_gemv_f<2, 4>(s, a, p);
        return launch_mx_gemv_f<1, 8>(s, a, p);
    }
    if (p.tiles == 16) {
        if (p.wk == 8) return launch_mx_gemv_f<8, 2>(s, a, p);
        if (p.wk == 4) return launch_mx_gemv_f<4, 4>(s, a, p);
        return launch_mx_gemv_f<2, 8>(s, a, p);
    }
    return p.wk == 8 ? launch_mx_gemv_f<8, 4>(s, a, p) : launch_mx_gemv_f<4, 8>(s, a, p);
}

// The block (MT x WM row tiles of x, NT of W) of the least estimated time:
// rounds of 256 blocks, times a wave's steps (a column tile each), times what a
// step takes: measured with N = K = 4096 where few blocks ran (other N and K rest
// on that); loading x's terms bounds it, 64 KB a step, which the wider blocks use
// more often. (us, wide
// first: 2000 x 4096 x 4096 91 101 113 143 178 286; 512 x 4096 x 4096 66 43 32
// 41 51 77; 64 x 4096 x 4096 60 37 24 20 15 14.)
struct GemmShape {
    int mt, nt, wm;
    double step;
    const char* name;
};
static constexpr GemmShape kGemmShapes[] = {{2, 16, 4, 1.70, "gemm128x256"}, {2, 8, 4, 0.97, "gemm128x128"},
                                            {1, 8, 4, 1.10, "gemm64x128"},   {1, 4, 4, 0.89, "gemm64x64"},
                                            {1, 4, 2, 1.18, "gemm32x64"},    {1, 2, 2, 1.00, "gemm32x32"}};
static int gemm_shape(int M, int N, int K) {
    const long long mt = (M + 15) / 16, nt = (N + 15) / 16, nq = (K + 511) / 512;
    int best = 0;
    double least = 0;
    for (int i = 0; i < (int)std::size(kGemmShapes); i++) {
        const GemmShape& g = kGemmShapes[i];
        const long long wk = 8 / g.mt / g.wm, blocks = ((mt + g.mt * g.wm - 1) / (g.mt * g.wm)) * ((nt + g.nt - 1) / g.nt);
        const double t = (double)((blocks + 255) / 256) * ((nq + wk - 1) / wk) * g.step;
        if (i == 0 || t < least) best = i, least = t;
    }
    return best;
}
template <int MT, int NT, int WM>
static int launch_mx_gemm_t(hipStream_t s, const MxLinearArgs& a) {
    constexpr int bytes = GemmLds<MT, NT, WM>::BYTES;
    if constexpr (bytes > 64 << 10)
        GH_TRY(check(hipFuncSetAttribute(reinterpret_cast<const void*>(&k_mx_gemm<MT, NT, WM>),
                                         hipFuncAttributeMaxDynamicSharedMemorySize, bytes), "mx_gemm attribute"));
    const long long blocks = (long long)((a.nt + NT - 1) / NT) * (((a.M + 15) / 16 + WM * MT - 1) / (WM * MT));
    hipLaunchKernelGGL((k_mx_gemm<MT, NT, WM>), dim3((unsigned)((blocks + 7) / 8 * 8)), dim3(512 / MT), bytes, s, a);
    return GORCH_HIP_OK;
}
static int launch_mx_gemm(hipStream_t s, MxLinearArgs a, char* ws) {
    a.terms = ws + kCounterBytes;
    hipLaunchKernelGGL(k_mx_terms, dim3((a.nk + 3) / 4, (a.M + 15) / 16), dim3(256), 0, s, a);
    switch (gemm_shape(a.M, a.N, a.K)) {
        case 0: return launch_mx_gemm_t<2, 16, 4>(s, a);
        case 1: return launch_mx_gemm_t<2, 8, 4>(s, a);
        case 2: return launch_mx_gemm_t<1, 8, 4>(s, a);
        case 3: return launch_mx_gemm_t<1, 4, 4>(s, a);
        case 4: return launch_mx_gemm_t<1, 4, 2>(s, a);
        default: return launch_mx_gemm_t<1, 2, 2>(s, a);
    }
}

const char* mx_linear_choice_name(int M, int N, int K) {
    if (M > 16) return kGemmShapes[gemm_shape(M, N, K)].name;
    const GemvPlan p = gemv_plan(M, N, K);
    static const char* const names[3][2] = {{"gemv", "gemv split"}, {"gemv5", "gemv5 split"}, {"gemv5 made", "gemv5 made split"}};
    return names[p.kind == kRow1 ? 0 : (p.kind == kFive ? 1 : 2)][p.slices > 1];
}

}  // namespace gh

using namespace gh;

extern "C" size_t gorch_hip_linear_mxfp4_workspace_size(int M, int N, int K) {
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    return M <= 16 ? gemv_plan(M, N, K).bytes : terms_bytes(M, K);
}

extern "C" int gorch_hip_linear_mxfp4(void* stream, const float* x, const void* Wp, const float* bias, const float* residual,
                                      float* y, int M, int N, int K, int epilogue, void* workspace, size_t workspace_bytes) {
    GH_REQUIRE(M >= 0 && N >= 0 && K >= 0, "gorch_hip_linear_mxfp4: negative size");
    GH_REQUIRE(epilogue == GORCH_HIP_EPI_NONE || epilogue == GORCH_HIP_EPI_GELU, "gorch_hip_linear_mxfp4: unknown epilogue");
    if (M == 0 || N == 0) return GORCH_HIP_OK;
    GH_REQUIRE(K > 0, "gorch_hip_linear_mxfp4: K must be positive");
    GH_REQUIRE(x && Wp && y, "gorch_hip_linear_mxfp4: null pointer");
    GH_REQUIRE(x != y, "gorch_hip_linear_mxfp4: y must not be x");
    GH_SUPPORTED(K % 8 == 0, "gorch_hip_linear_mxfp4: K must be a multiple of 8");
    GH_SUPPORTED((uintptr_t)x % 16 == 0 && (uintptr_t)Wp % 16 == 0 && (uintptr_t)workspace % 16 == 0,
                 "gorch_hip_linear_mxfp4: x, Wp and the workspace must be 16-byte aligned");
    GH_SUPPORTED(M <= 16 * 65535 && N <= 16 * 65535 && K <= 1 << 24, "gorch_hip_linear_mxfp4: M, N or K out of range");
    const size_t need = M <= 16 ? gemv_plan(M, N, K).bytes : terms_bytes(M, K);
    GH_REQUIRE(workspace_bytes >= need && (workspace || need == 0), "gorch_hip_linear_mxfp4: workspace too small");
    hipStream_t s = stream_of(stream);
    GH_TRY(bf16_gate(s));
    MxLinearArgs a{};
    a.x = x;
    a.bias = bias;
    a.residual = residual;
    a.y = y;
    a.M = M;
    a.N = N;
    a.K = K;
    a.epi = epilogue;
    a.nt = (N + 15) / 16;
    a.nk = (K + 127) / 128;
    a.nq = (a.nk + 3) / 4;
    a.wp = static_cast<const u32x4*>(Wp);
    a.wsc = reinterpret_cast<const uint32_t*>(static_cast<const char*>(Wp) + (size_t)a.nt * a.nk * 1024);
    if (M <= 16) GH_TRY(launch_mx_gemv(s, a, static_cast<char*>(workspace)));
    else GH_TRY(launch_mx_gemm(s, a, static_cast<char*>(workspace)));
    count(M <= 16 ? CNT_GEMV : CNT_GEMM);
    return finish(stream, check_launch("linear_mxfp4"));
}
