// mxfp4.hip — weights in MXFP4: the codec between rows of f32 or bf16 and
// codes with a scale byte per group of 32, and the layout that the Linear over
// such weights reads.
#include "mx.h"

namespace gh {

struct MxRows {
    long long rows, stride;  // of the values, in elements
    int cols, groups;        // groups of 32 in a row, the last perhaps shorter
};

// Piece i of 8 values (four to a group, the last group's missing ones too) to
// its row, group and place there. FLAT: rows of whole groups that lie close.
template <bool FLAT>
struct Piece {
    long long row, group, at;  // at: index of its first value
    int col;
    bool live;
    __device__ __forceinline__ Piece(const MxRows& a, long long i, long long n) {
        group = i >> 2;
        live = i < n;
        if constexpr (FLAT) {
            row = 0;
            col = 0;
            at = 8 * i;
        } else {
            row = (unsigned long long)group >> 32 ? group / a.groups : (long long)((uint32_t)group / (uint32_t)a.groups);
            col = 32 * (int)(group - row * a.groups) + 8 * (int)(i & 3);
            live &= col < a.cols;
            at = row * a.stride + col;
        }
    }
    // index of its codes' word
    __device__ __forceinline__ long long word(const MxRows& a, long long i) const {
        return FLAT ? i : row * (a.cols / 8) + col / 8;
    }
};

template <bool BF16>
struct Raw8 {
    u32x4 w[BF16 ? 1 : 2];
    __device__ __forceinline__ void load(const void* in, long long at) {
        const u32x4* p = reinterpret_cast<const u32x4*>(static_cast<const char*>(in) + at * (BF16 ? 2 : 4));
#pragma unroll
        for (int k = 0; k < (BF16 ? 1 : 2); k++) w[k] = __builtin_nontemporal_load(p + k);
    }
    __device__ __forceinline__ void get(float (&x)[8]) const {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            if constexpr (BF16) x[e] = e & 1 ? bf16_hi(w[0][e / 2]) : bf16_lo(w[0][e / 2]);
            else x[e] = __uint_as_float(w[e / 4][e % 4]);
        }
    }
};

// Four lanes a group, eight values each: 16 or 32 bytes in, a word of codes out,
// the group's largest magnitude by two lane exchanges. Bound by memory:
// 151,936 x 1,024 in bf16 67.5 us (5.9 TB/s of 394 MB; a copy of 1 GiB runs at
// 5.2), 33 x 1,000 in f32 2.6 us, a launch's latency. Rows of whole groups that
// lie close are one long row (FLAT), which saves the divisions.
template <bool BF16, bool FLAT>
__global__ __launch_bounds__(256) void k_mxfp4_encode(MxRows a, const void* in, uint32_t* codes, uint8_t* scales) {
    const long long n = a.rows * a.groups * 4, step = (long long)gridDim.x * 256;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < (n + 63) / 64 * 64; i += step) {
        const Piece<FLAT> p(a, i, n);
        Raw8<BF16> raw{};
        if (p.live) raw.load(in, p.at);
        float x[8];
        raw.get(x);
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
        top = max(top, __float_as_uint(dpp_f<kDppQuadSwap1>(__uint_as_float(top))));
        top = max(top, __float_as_uint(dpp_f<kDppQuadSwap2>(__uint_as_float(top))));
        const uint32_t s = mx_scale(top);
        if (p.live) {
            codes[p.word(a, i)] = mx_encode8(x, s);
            if ((i & 3) == 0) scales[p.group] = (uint8_t)s;
        }
    }
}

// The same back: 60 us for 151,936 x 1,024 in bf16 (6.6 TB/s), 2.7 for 33 x 1,000.
template <bool BF16, bool FLAT>
__global__ __launch_bounds__(256) void k_mxfp4_decode(MxRows a, const uint32_t* codes, const uint8_t* scales, void* out) {
    const long long n = a.rows * a.groups * 4, step = (long long)gridDim.x * 256;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += step) {
        const Piece<FLAT> p(a, i, n);
        if (!p.live) continue;
        const u32x4 w = mx_widen8(codes[p.word(a, i)], 1.0f);
        const float s = mx_power(scales[p.group]);
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = (e & 1 ? bf16_hi(w[e / 2]) : bf16_lo(w[e / 2])) * s;
        u32x4* o = reinterpret_cast<u32x4*>(static_cast<char*>(out) + p.at * (BF16 ? 2 : 4));
        if constexpr (BF16) {
            u32x4 y;
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] = f32_to_bf16_bits(x[2 * e]) | ((uint32_t)f32_to_bf16_bits(x[2 * e + 1]) << 16);
            __builtin_nontemporal_store(y, o);
        } else {
#pragma unroll
            for (int k = 0; k < 2; k++) {
                u32x4 y;
#pragma unroll
                for (int e = 0; e < 4; e++) y[e] = __float_as_uint(x[4 * k + e]);
                __builtin_nontemporal_store(y, o + k);
            }
        }
    }
}

// The Linear's layout: for 16 rows t and 128 columns j of the weight, lane l's
// 16 bytes of codes (row 16 t + l % 16, columns 128 j + 32 (l / 16) .. + 31) at
// ((t nk + j) 64 + l) 16, the operand of a matrix instruction as one contiguous
// KB; then the scale bytes, those of four j in a word, at ((t nq + j / 4) 64 +
// l) 4 + j % 4. Rows and columns past the weight's are zeros. Once a weight: 49 us
// for 151,936 x 1,024.
__global__ __launch_bounds__(256) void k_pack_mxfp4(const uint32_t* codes, const uint8_t* scales, u32x4* wp, uint32_t* ws,
                                                    int N, int K, int nk, int nq) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int t = blockIdx.y, q = blockIdx.x, j = 4 * q + wave;  // a block: four j
    __shared__ uint8_t sc[64][4];
    const int n = 16 * t + (lane & 15), k = 128 * j + 32 * (lane >> 4);
    u32x4 c = {0, 0, 0, 0};
    uint32_t s = 0;
    if (n < N && k < K) {
        const uint32_t* src = codes + (size_t)n * (K / 8) + k / 8;
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (k + 8 * e < K) c[e] = src[e];
        s = scales[(size_t)n * ((K + 31) / 32) + k / 32];
    }
    if (j < nk) wp[((size_t)t * nk + j) * 64 + lane] = c;
    sc[lane][wave] = (uint8_t)s;
    __syncthreads();
    if (wave == 0) ws[((size_t)t * nq + q) * 64 + lane] = *reinterpret_cast<const uint32_t*>(sc[lane]);
}

static int codec_args(const char* who, const void* a, const void* b, const void* c, int64_t rows, int64_t cols,
                      int64_t stride, MxRows& r) {
    const auto fail = [&](int rc, const char* what) {
        set_error(std::string(who) + ": " + what);
        return rc;
    };
    if (rows < 0 || cols < 0 || cols > 0x7fffffff) return fail(GORCH_HIP_EINVAL, "negative size, or cols past 2^31 - 1");
    if (cols % 8 != 0) return fail(GORCH_HIP_EUNSUPPORTED, "cols must be a multiple of 8");
    r = MxRows{rows, stride, (int)cols, (int)((cols + kMxGroup - 1) / kMxGroup)};
    if (rows == 0 || cols == 0) return GORCH_HIP_OK;
    if (!a || !b || !c) return fail(GORCH_HIP_EINVAL, "null pointer");
    if (stride < cols && rows > 1) return fail(GORCH_HIP_EINVAL, "the row stride is shorter than a row");
    if (rows > (1ll << 40) / cols) return fail(GORCH_HIP_EUNSUPPORTED, "rows * cols must be at most 2^40");
    return GORCH_HIP_OK;
}

// One piece a thread up to 2^16 blocks, then several.
static dim3 codec_grid(const MxRows& r) {
    const long long blocks = (r.rows * r.groups * 4 + 255) / 256;
    return dim3((unsigned)(blocks < 65536 ? blocks : 65536));
}
static bool flat(const MxRows& r) { return r.cols % kMxGroup == 0 && (r.stride == r.cols || r.rows == 1); }

}  // namespace gh

using namespace gh;

extern "C" int gorch_hip_mxfp4_encode(void* stream, const void* in, int in_bf16, int64_t in_stride, uint8_t* codes,
                                      uint8_t* scales, int64_t rows, int64_t cols) {
    MxRows r;
    GH_TRY(codec_args("gorch_hip_mxfp4_encode", in, codes, scales, rows, cols, in_stride, r));
    if (rows == 0 || cols == 0) return GORCH_HIP_OK;
    GH_SUPPORTED((uintptr_t)in % 16 == 0 && (rows == 1 || in_stride % (in_bf16 ? 8 : 4) == 0) && (uintptr_t)codes % 4 == 0,
                 "gorch_hip_mxfp4_encode: rows must be 16-byte aligned, codes 4-byte aligned");
    const auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, codec_grid(r), dim3(256), 0, stream_of(stream), r, in, reinterpret_cast<uint32_t*>(codes), scales);
    };
    if (flat(r)) in_bf16 ? go(k_mxfp4_encode<true, true>) : go(k_mxfp4_encode<false, true>);
    else in_bf16 ? go(k_mxfp4_encode<true, false>) : go(k_mxfp4_encode<false, false>);
    count(CNT_CODEC);
    return finish(stream, check_launch("mxfp4_encode"));
}

extern "C" int gorch_hip_mxfp4_decode(void* stream, const uint8_t* codes, const uint8_t* scales, void* out, int out_bf16,
                                      int64_t out_stride, int64_t rows, int64_t cols) {
    MxRows r;
    GH_TRY(codec_args("gorch_hip_mxfp4_decode", codes, scales, out, rows, cols, out_stride, r));
    if (rows == 0 || cols == 0) return GORCH_HIP_OK;
    GH_SUPPORTED((uintptr_t)out % 16 == 0 && (rows == 1 || out_stride % (out_bf16 ? 8 : 4) == 0) && (uintptr_t)codes % 4 == 0,
                 "gorch_hip_mxfp4_decode: rows must be 16-byte aligned, codes 4-byte aligned");
    const auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, codec_grid(r), dim3(256), 0, stream_of(stream), r, reinterpret_cast<const uint32_t*>(codes), scales, out);
    };
    if (flat(r)) out_bf16 ? go(k_mxfp4_decode<true, true>) : go(k_mxfp4_decode<false, true>);
    else out_bf16 ? go(k_mxfp4_decode<true, false>) : go(k_mxfp4_decode<false, false>);
    count(CNT_CODEC);
    return finish(stream, check_launch("mxfp4_decode"));
}

extern "C" size_t gorch_hip_packed_mxfp4_bytes(int N, int K) {
    if (N <= 0 || K <= 0) return 0;
    const size_t nt = ((size_t)N + 15) / 16, nk = ((size_t)K + 127) / 128;
    return nt * nk * 1024 + nt * ((nk + 3) / 4) * 256;
}

extern "C" int gorch_hip_pack_mxfp4(void* stream, const uint8_t* codes, const uint8_t* scales, void* Wp, int N, int K) {
    GH_REQUIRE(N >= 0 && K >= 0, "gorch_hip_pack_mxfp4: negative size");
    if (N == 0 || K == 0) return GORCH_HIP_OK;
    GH_REQUIRE(codes && scales && Wp, "gorch_hip_pack_mxfp4: null pointer");
    GH_SUPPORTED(K % 8 == 0, "gorch_hip_pack_mxfp4: K must be a multiple of 8");
    GH_SUPPORTED(N <= 16 * 65535, "gorch_hip_pack_mxfp4: N must be at most 1048560");
    GH_SUPPORTED((uintptr_t)codes % 4 == 0 && (uintptr_t)Wp % 16 == 0,
                 "gorch_hip_pack_mxfp4: codes must be 4-byte aligned, Wp 16-byte aligned");
    const int nt = (N + 15) / 16, nk = (K + 127) / 128, nq = (nk + 3) / 4;
    char* p = static_cast<char*>(Wp);
    hipLaunchKernelGGL(k_pack_mxfp4, dim3(nq, nt), dim3(256), 0, stream_of(stream), reinterpret_cast<const uint32_t*>(codes),
                       scales, reinterpret_cast<u32x4*>(p), reinterpret_cast<uint32_t*>(p + (size_t)nt * nk * 1024), N, K, nk, nq);
    count(CNT_CODEC);
    return finish(stream, check_launch("pack_mxfp4"));
}
