// mxlinear.hip — Linear over MXFP4 weights (nn/module.go:61-88 with the
// weight's values rounded to four bits): y = residual + epi(x W^T + bias). The
// codes go to the matrix cores as they are; x goes there as the five 6-bit
// terms of mx.h, which keep f32's accuracy.
#include <algorithm>

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
    int chunk;       // column tiles whose terms a block holds at once
    char* terms;     // of more than 16 rows: x's operands (k_mx_terms)
};

// Barrier for LDS alone: loads into registers stay in flight.
__device__ __forceinline__ void lds_sync() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(kWaitLgkm0);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// The 32 values of row m, columns k .. k + 31 (zeros past K or without a row).
__device__ __forceinline__ floatx32 load_group(const float* x, int m, int M, int k, int K) {
    floatx32 v;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        floatx4 f = {0.f, 0.f, 0.f, 0.f};
        if (m < M && k + 4 * i < K) f = *reinterpret_cast<const floatx4*>(x + (size_t)m * K + k + 4 * i);
#pragma unroll
        for (int e = 0; e < 4; e++) v[4 * i + e] = f[e];
    }
    return v;
}

__device__ __forceinline__ void mx_store(const MxLinearArgs& a, int m, int n, float v) {
    if (a.bias) v += a.bias[n];
    if (a.epi == GORCH_HIP_EPI_GELU) v = gelu_gemm(v);
    const size_t at = (size_t)m * a.N + n;
    if (a.residual) v += a.residual[at];
    a.y[at] = v;
}

// Up to 16 rows of x. A block splits x (or `chunk` column tiles of it) into its
// terms in LDS once; its 8 waves are WK along the columns, 8 / WK along the row
// tiles of W, and each streams 1 KB of codes a step into one instruction (ROW1:
// up to 3 rows, whose terms are rows of one operand) or five.
constexpr int kGemvWaves = 8;
struct GemvLds {  // byte offsets of a block's LDS
    int p8, sc, red, bytes;
    __host__ __device__ GemvLds(int M, int chunk) {
        const int slots = chunk * 4 * kMxTerms * M;
        p8 = slots * 16;
        sc = p8 + slots * 8;
        red = sc + chunk * 4 * M * 8;
        bytes = red + 2 * kGemvWaves * 1024;
    }
};
template <bool ROW1, int WK>
__global__ __launch_bounds__(64 * kGemvWaves) void k_mx_gemv(MxLinearArgs a) {
    constexpr int WN = kGemvWaves / WK, U = 4;
    extern __shared__ __align__(16) char lds[];
    const GemvLds at(a.M, a.chunk);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, c = lane & 15;
    const int M = a.M, R = kMxTerms * M;
    const int groups = (a.nt + WN - 1) / WN, wk = wave % WK, wn = wave / WK;
    const int chunks = (a.nk + a.chunk - 1) / a.chunk;
    struct Step {
        u32x4 codes[U];
        uint32_t scale[U];
    };
    const auto load = [&](Step& s, int t, int j, int jb) {
        const int tt = min(t, a.nt - 1);
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int jj = min(min(j + u, jb - 1), a.nk - 1);
            s.codes[u] = __builtin_nontemporal_load(a.wp + ((size_t)tt * a.nk + jj) * 64 + lane);
            s.scale[u] = a.wsc[((size_t)tt * a.nq + (jj >> 2)) * 64 + lane] >> (8 * (jj & 3));
        }
    };
    int turn = 0;
    for (int group = blockIdx.x; group < groups; group += gridDim.x) {
        const int t = group * WN + wn;
        floatx4 acc = {0.f, 0.f, 0.f, 0.f};
        for (int ch = 0; ch < chunks; ch++) {
            const int c0 = ch * a.chunk, c1 = min(c0 + a.chunk, a.nk), per = (c1 - c0 + WK - 1) / WK;
            const int ja = c0 + wk * per, jb = min(ja + per, c1);
            Step s;
            load(s, t, ja, max(jb, 1));
            if (chunks > 1 || group == (int)blockIdx.x) {
                lds_sync();
                for (int i = threadIdx.x; i < (c1 - c0) * 4 * M; i += 64 * kGemvWaves) {
                    const int m = i / ((c1 - c0) * 4), kb = i - m * (c1 - c0) * 4, j = kb >> 2, gg = kb & 3;
                    MxTerms r;
                    mx_split(load_group(a.x, m, M, 128 * c0 + 32 * kb, a.K), r);
#pragma unroll
                    for (int q = 0; q < kMxTerms; q++) {
                        const int slot = ROW1 ? (j * 4 + gg) * R + m * kMxTerms + q : ((j * kMxTerms + q) * 4 + gg) * M + m;
                        *reinterpret_cast<u32x4*>(lds + slot * 16) = u32x4{r.t[q][0], r.t[q][1], r.t[q][2], r.t[q][3]};
                        *reinterpret_cast<u32x2*>(lds + at.p8 + slot * 8) = u32x2{r.t[q][4], r.t[q][5]};
                    }
                    if constexpr (ROW1) {
                        uint8_t* sc = reinterpret_cast<uint8_t*>(lds + at.sc) + (j * 4 + gg) * R + m * kMxTerms;
#pragma unroll
                        for (int q = 0; q < 4; q++) sc[q] = (uint8_t)(r.scale >> (8 * q));
                        sc[4] = (uint8_t)r.last;
                    } else {
                        *reinterpret_cast<u32x2*>(lds + at.sc + ((j * 4 + gg) * M + m) * 8) = u32x2{r.scale, r.last};
                    }
                }
                lds_sync();
            }
            for (int j = ja; j < jb; j += U) {
                const Step now = s;
                load(s, t, j + U, jb);
#pragma unroll
                for (int u = 0; u < U; u++) {
                    if (j + u >= jb) break;
                    const int jl = j + u - c0;
                    const i32x8 w = mx_op4(now.codes[u]);
                    if constexpr (ROW1) {
                        const int slot = (jl * 4 + g) * R + min(c, R - 1);
                        const i32x8 six = mx_op6(*reinterpret_cast<const u32x4*>(lds + slot * 16),
                                                 *reinterpret_cast<const u32x2*>(lds + at.p8 + slot * 8));
                        acc = mx_mfma<0, 0>(six, *reinterpret_cast<const uint8_t*>(lds + at.sc + slot), w, now.scale[u], acc);
                    } else {
                        const int m = min(c, M - 1);
                        const u32x2 sx = *reinterpret_cast<const u32x2*>(lds + at.sc + ((jl * 4 + g) * M + m) * 8);
                        const auto six = [&](int q) {
                            const int slot = ((jl * kMxTerms + q) * 4 + g) * M + m;
                            return mx_op6(*reinterpret_cast<const u32x4*>(lds + slot * 16),
                                          *reinterpret_cast<const u32x2*>(lds + at.p8 + slot * 8));
                        };
                        acc = mx_mfma<0, 0>(six(4), sx[1], w, now.scale[u], acc);
                        acc = mx_mfma<3, 0>(six(3), sx[0], w, now.scale[u], acc);
                        acc = mx_mfma<2, 0>(six(2), sx[0], w, now.scale[u], acc);
                        acc = mx_mfma<1, 0>(six(1), sx[0], w, now.scale[u], acc);
                        acc = mx_mfma<0, 0>(six(0), sx[0], w, now.scale[u], acc);
                    }
                }
            }
        }
        // the waves' sums in wave order; row 4 g + i of a result is at i * 64 + lane
        float* red = reinterpret_cast<float*>(lds + at.red) + turn * kGemvWaves * 256;
        turn ^= 1;
#pragma unroll
        for (int i = 0; i < 4; i++) red[wave * 256 + i * 64 + lane] = acc[i];
        lds_sync();
        for (int i = threadIdx.x; i < WN * M * 16; i += 64 * kGemvWaves) {
            const int n16 = i & 15, m = (i >> 4) % M, w = (i >> 4) / M;
            const int n = (group * WN + w) * 16 + n16;
            if (n >= a.N) continue;
            float v = 0.f;
#pragma unroll
            for (int k = 0; k < WK; k++) {
                const float* from = red + (w * WK + k) * 256 + n16;
                if constexpr (ROW1) {
#pragma unroll
                    for (int q = kMxTerms - 1; q >= 0; q--) {
                        const int row = m * kMxTerms + q;
                        v += from[(row & 3) * 64 + (row >> 2) * 16];
                    }
                } else {
                    v += from[(m & 3) * 64 + (m >> 2) * 16];
                }
            }
            mx_store(a, m, n, v);
        }
    }
}

// More rows: x's operands first, 8 KB for each 16 rows and 128 columns (the
// terms' first 16 bytes, then their last 8, then the scale words, each in lane
// order), in row tile, column tile order.
constexpr int kTermBytes = 8192, kTerm8 = kMxTerms * 1024, kTermScale = kTerm8 + kMxTerms * 512;
__global__ __launch_bounds__(256) void k_mx_terms(MxLinearArgs a) {
    const int lane = threadIdx.x & 63, i = blockIdx.y, j = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (j >= a.nk) return;
    MxTerms r;
    mx_split(load_group(a.x, 16 * i + (lane & 15), a.M, 128 * j + 32 * (lane >> 4), a.K), r);
    char* to = a.terms + ((size_t)i * a.nk + j) * kTermBytes;
#pragma unroll
    for (int q = 0; q < kMxTerms; q++) {
        *reinterpret_cast<u32x4*>(to + q * 1024 + lane * 16) = u32x4{r.t[q][0], r.t[q][1], r.t[q][2], r.t[q][3]};
        *reinterpret_cast<u32x2*>(to + kTerm8 + q * 512 + lane * 8) = u32x2{r.t[q][4], r.t[q][5]};
    }
    *reinterpret_cast<u32x2*>(to + kTermScale + lane * 8) = u32x2{r.scale, r.last};
}

// WM x WN waves of MT x NT tiles of 16 x 16: x's operands through a two-stage
// ring in LDS, W's codes straight to the operand registers.
template <int MT, int NT, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void k_mx_gemm(MxLinearArgs a) {
    constexpr int BMT = MT * WM, NW = WM * WN;
    extern __shared__ __align__(16) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, c = lane & 15;
    const int wm = wave % WM, wn = wave / WM;
    const int i0 = blockIdx.y * BMT, t0 = (blockIdx.x * WN + wn) * NT;
    const auto stage = [&](int j, int b) {
        typedef __attribute__((address_space(1))) const uint32_t* global_ptr;
        typedef __attribute__((address_space(3))) uint32_t* lds_ptr;
#pragma unroll
        for (int k = 0; k < BMT * 8 / NW; k++) {
            const int kb = k * NW + wave;  // KB of the stage
            const char* from = a.terms + ((size_t)(i0 + (kb >> 3)) * a.nk + j) * kTermBytes + (kb & 7) * 1024 + lane * 16;
            __builtin_amdgcn_global_load_lds((global_ptr)from, (lds_ptr)(lds + (b * BMT * 8 + kb) * 1024), 16, 0, 0);
        }
    };
    u32x4 wc[NT];
    uint32_t ws[NT];
    const auto codes = [&](int j) {
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const int t = min(t0 + n, a.nt - 1);
            wc[n] = a.wp[((size_t)t * a.nk + j) * 64 + lane];
            ws[n] = a.wsc[((size_t)t * a.nq + (j >> 2)) * 64 + lane] >> (8 * (j & 3));
        }
    };
    floatx4 acc[MT][NT];
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int n = 0; n < NT; n++) acc[m][n] = floatx4{0.f, 0.f, 0.f, 0.f};
    stage(0, 0);
    codes(0);
    for (int j = 0; j < a.nk; j++) {
        block_sync_dma();
        i32x8 w[NT];
        uint32_t s[NT];
#pragma unroll
        for (int n = 0; n < NT; n++) {
            w[n] = mx_op4(wc[n]);
            s[n] = ws[n];
        }
        if (j + 1 < a.nk) {
            stage(j + 1, (j + 1) & 1);
            codes(j + 1);
        }
        const char* base = lds + ((j & 1) * BMT + wm * MT) * kTermBytes;
#pragma unroll
        for (int m = 0; m < MT; m++) {
            const char* from = base + m * kTermBytes;
            const u32x2 sx = *reinterpret_cast<const u32x2*>(from + kTermScale + lane * 8);
            const auto six = [&](int q) {
                return mx_op6(*reinterpret_cast<const u32x4*>(from + q * 1024 + lane * 16),
                              *reinterpret_cast<const u32x2*>(from + kTerm8 + q * 512 + lane * 8));
            };
            const i32x8 x4 = six(4), x3 = six(3), x2 = six(2), x1 = six(1), x0 = six(0);
#pragma unroll
            for (int n = 0; n < NT; n++) acc[m][n] = mx_mfma<0, 0>(x4, sx[1], w[n], s[n], acc[m][n]);
#pragma unroll
            for (int n = 0; n < NT; n++) acc[m][n] = mx_mfma<3, 0>(x3, sx[0], w[n], s[n], acc[m][n]);
#pragma unroll
            for (int n = 0; n < NT; n++) acc[m][n] = mx_mfma<2, 0>(x2, sx[0], w[n], s[n], acc[m][n]);
#pragma unroll
            for (int n = 0; n < NT; n++) acc[m][n] = mx_mfma<1, 0>(x1, sx[0], w[n], s[n], acc[m][n]);
#pragma unroll
            for (int n = 0; n < NT; n++) acc[m][n] = mx_mfma<0, 0>(x0, sx[0], w[n], s[n], acc[m][n]);
        }
    }
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int row = 16 * (i0 + wm * MT + m) + 4 * g + i, col = 16 * (t0 + n) + c;
                if (row < a.M && col < a.N) mx_store(a, row, col, acc[m][n][i]);
            }
}

constexpr int kGemmRowTiles = 4;  // of the GEMM's blocks
static size_t terms_bytes(int M, int K) {
    const size_t tiles = ((size_t)M + 15) / 16, padded = (tiles + kGemmRowTiles - 1) / kGemmRowTiles * kGemmRowTiles;
    return M <= 16 ? 0 : padded * ((K + 127) / 128) * kTermBytes;
}

static void launch_mx_gemv(hipStream_t s, MxLinearArgs a) {
    // columns whose terms fit 48 KB (with the waves' sums 64: two blocks a CU)
    const int per = 4 * a.M * (kMxTerms * 24 + 8);
    a.chunk = std::min(a.nk, std::max(1, (48 << 10) / per));
    const int bytes = GemvLds(a.M, a.chunk).bytes;
    int wk = 8;
    while (wk > 1 && (a.nk < wk || (long long)a.nt * wk / 8 >= 512)) wk /= 2;
    const int wn = kGemvWaves / wk, groups = (a.nt + wn - 1) / wn;
    const auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(std::min(groups, 512)), dim3(64 * kGemvWaves), bytes, s, a); };
    const auto form = [&](auto k) {
        constexpr int WK = decltype(k)::value;
        a.M <= 3 ? go(k_mx_gemv<true, WK>) : go(k_mx_gemv<false, WK>);
    };
    if (wk == 8) form(std::integral_constant<int, 8>{});
    else if (wk == 4) form(std::integral_constant<int, 4>{});
    else if (wk == 2) form(std::integral_constant<int, 2>{});
    else form(std::integral_constant<int, 1>{});
}

static void launch_mx_gemm(hipStream_t s, const MxLinearArgs& a) {
    const int row_tiles = (a.M + 15) / 16, blocks = (row_tiles + kGemmRowTiles - 1) / kGemmRowTiles;
    hipLaunchKernelGGL(k_mx_terms, dim3((a.nk + 3) / 4, blocks * kGemmRowTiles), dim3(256), 0, s, a);
    constexpr int MT = 2, NT = 4, WM = 2, WN = 2;
    static_assert(MT * WM == kGemmRowTiles);
    hipLaunchKernelGGL((k_mx_gemm<MT, NT, WM, WN>), dim3((a.nt + NT * WN - 1) / (NT * WN), blocks), dim3(64 * WM * WN),
                       2 * kGemmRowTiles * kTermBytes, s, a);
}

}  // namespace gh

using namespace gh;

extern "C" size_t gorch_hip_linear_mxfp4_workspace_size(int M, int N, int K) {
    return M <= 0 || N <= 0 || K <= 0 ? 0 : terms_bytes(M, K);
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
    GH_SUPPORTED(M <= 1 << 20 && N <= 16 * 65535 && K <= 1 << 24, "gorch_hip_linear_mxfp4: M, N or K out of range");
    const size_t need = terms_bytes(M, K);
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
    a.terms = static_cast<char*>(workspace);
    if (M <= 16) launch_mx_gemv(s, a);
    else launch_mx_gemm(s, a);
    count(M <= 16 ? CNT_GEMV : CNT_GEMM);
    return finish(stream, check_launch("linear_mxfp4"));
}
