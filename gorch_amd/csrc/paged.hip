// paged.hip — a KV cache in pages: new tokens' q and k finished (per-head
// RMSNorm, RoPE; GQA.ForwardCached's order, nn/gqa.go:300-330) and K and V
// written in bf16 or quantised to e4m3 (gorch_hip_paged_append), and rows
// read back as f32 (gorch_hip_paged_read).
#include "paged.h"

namespace gh {

static bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

int paged_args(const char* who, const gorch_hip_paged_kv* kv, const gorch_hip_paged_batch* b, PagedArgs& a) {
    const auto fail = [&](int rc, const char* what) {
        set_error(std::string(who) + ": " + what);
        return rc;
    };
    if (!kv || !b) return fail(GORCH_HIP_EINVAL, "null cache or batch");
    if (kv->dtype != GORCH_HIP_KV_BF16 && kv->dtype != GORCH_HIP_KV_E4M3) return fail(GORCH_HIP_EINVAL, "unknown cache dtype");
    if (kv->num_pages <= 0 || kv->page_size <= 0 || kv->num_kv <= 0 || kv->head_dim <= 0)
        return fail(GORCH_HIP_EINVAL, "cache sizes must be positive");
    if (b->tokens < 0 || b->seqs < 0 || b->max_pages < 0 || b->max_new < 0 || b->max_kv < 0)
        return fail(GORCH_HIP_EINVAL, "batch sizes must not be negative");
    if (kv->head_dim % 16 != 0 || kv->head_dim > 256)
        return fail(GORCH_HIP_EUNSUPPORTED, "head_dim must be a multiple of 16 up to 256");
    if (kv->num_kv > 0xffff) return fail(GORCH_HIP_EUNSUPPORTED, "num_kv must be below 2^16");
    const long long room = (long long)b->max_pages * kv->page_size;
    // (2^16 below 2^31: the kernels look a few tiles past the last position)
    if (room > 0x7fff0000ll) return fail(GORCH_HIP_EINVAL, "max_pages * page_size must be below 2^31 - 2^16");
    if (b->tokens >= 1 << 24) return fail(GORCH_HIP_EUNSUPPORTED, "tokens must be below 2^24");
    if (b->tokens > 0 && b->seqs > 0) {
        if (!kv->k || !kv->v || !b->cu_seqlens || !b->kv_lens || (b->max_pages > 0 && !b->page_table))
            return fail(GORCH_HIP_EINVAL, "null pool or batch array");
        if (kv->dtype == GORCH_HIP_KV_E4M3 && (!kv->k_scale || !kv->v_scale))
            return fail(GORCH_HIP_EINVAL, "e4m3 pools need k_scale and v_scale");
        if (!aligned(kv->k, 16) || !aligned(kv->v, 16)) return fail(GORCH_HIP_EUNSUPPORTED, "pools must be 16-byte aligned");
    }
    a.k = kv->k;
    a.v = kv->v;
    a.ks = kv->k_scale;
    a.vs = kv->v_scale;
    a.cu = b->cu_seqlens;
    a.lens = b->kv_lens;
    a.table = b->page_table;
    a.tokens = b->tokens;
    a.seqs = b->seqs;
    a.max_pages = b->max_pages;
    a.num_pages = kv->num_pages;
    a.num_kv = kv->num_kv;
    a.hd = kv->head_dim;
    a.limit = b->max_kv > 0 && b->max_kv < room ? b->max_kv : (int)room;
    a.page.set((uint32_t)kv->page_size);
    return GORCH_HIP_OK;
}

// v of the lane M lanes away within a row's lanes (lane ^ M; M = 8, 16, 32),
// on the vector unit's lane network.
template <int M>
__device__ __forceinline__ float across(float v) {
    if constexpr (M == 8) {
        return dpp_f<0x128>(v);  // 16 lanes rotated by 8
    } else {
        const uint32_t u = __float_as_uint(v);
        const bool odd = (threadIdx.x & M) != 0;
        if constexpr (M == 16) {
            const auto w = __builtin_amdgcn_permlane16_swap(u, u, false, false);
            return __uint_as_float(odd ? w[0] : w[1]);
        } else {
            const auto w = __builtin_amdgcn_permlane32_swap(u, u, false, false);
            return __uint_as_float(odd ? w[0] : w[1]);
        }
    }
}
template <int M>
__device__ __forceinline__ double across_d(double v) {
    const unsigned long long b = (unsigned long long)__double_as_longlong(v);
    const uint32_t lo = __float_as_uint(across<M>(__uint_as_float((uint32_t)b))),
                   hi = __float_as_uint(across<M>(__uint_as_float((uint32_t)(b >> 32))));
    return __longlong_as_double((long long)(((unsigned long long)hi << 32) | lo));
}
// Sums and maxima over the NL lanes of a row (NL = 16, 32 or 64).
template <int NL>
__device__ __forceinline__ double row_sum_d(double v) {
    v += dpp_d<kDppQuadSwap1>(v);
    v += dpp_d<kDppQuadSwap2>(v);
    v += dpp_d<kDppRowHalfMirror>(v);
    v += dpp_d<kDppRowMirror>(v);
    if constexpr (NL >= 32) v += across_d<16>(v);
    if constexpr (NL >= 64) v += across_d<32>(v);
    return v;
}
template <int NL>
__device__ __forceinline__ float row_max_f(float v) {
    v = fmaxf(v, dpp_f<kDppQuadSwap1>(v));
    v = fmaxf(v, dpp_f<kDppQuadSwap2>(v));
    v = fmaxf(v, dpp_f<kDppRowHalfMirror>(v));
    v = fmaxf(v, dpp_f<kDppRowMirror>(v));
    if constexpr (NL >= 32) v = fmaxf(v, across<16>(v));
    if constexpr (NL >= 64) v = fmaxf(v, across<32>(v));
    return v;
}

// Rows smaller than this throughout are stored as zeros (their scale's
// reciprocal would leave f32).
constexpr float kTinyRow = 0x1p-100f;

// Four values of a row to its pool row: bf16, or codes of x / scale, scale =
// amax / 448 the row's (NL lanes; every lane of the wave calls it).
template <bool F8, int NL>
__device__ __forceinline__ void store_kv(void* pool, float* scales, long long row, int hd, int c, bool mine, float4 x) {
    if constexpr (F8) {
        const float m = row_max_f<NL>(fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))));
        const float inv = m >= kTinyRow ? 448.0f / m : 0.0f;
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(x.x * inv, x.y * inv, 0, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(x.z * inv, x.w * inv, w, true);
        if (mine && row >= 0) {
            reinterpret_cast<int*>(pool)[(row * hd) / 4 + c] = w;
            if (c == 0) scales[row] = m >= kTinyRow ? m / 448.0f : 0.0f;
        }
    } else if (mine && row >= 0) {
        uint2 w;
        w.x = f32_to_bf16_bits(x.x) | ((uint32_t)f32_to_bf16_bits(x.y) << 16);
        w.y = f32_to_bf16_bits(x.z) | ((uint32_t)f32_to_bf16_bits(x.w) << 16);
        reinterpret_cast<uint2*>(pool)[(row * hd) / 4 + c] = w;
    }
}

struct AppendArgs {
    PagedArgs p;
    const float* q;
    const float* k;
    const float* v;
    long long qs, ks, vs;  // row strides in floats
    float* q_out;
    int hq;  // query heads here: 0 without q
    const float* gq;
    const float* gk;
    float eps;
    const float* cosT;
    const float* sinT;
    int rope_rows, neox;
};

// One token's rows: q heads, then k heads, then v heads, NL lanes a row of hd
// floats (lane c < hd / 4 holds elements 4c .. 4c + 3; FULL: hd = 4 NL), P
// rows per group of lanes. Same operations per row, in the same order, as
// k_norm_rope_rows: x * inv * gain with inv from the f64 sum of squares, then
// the pair rotated with every product and sum rounded on its own.
// Bound by memory: the rows go out before anything else, and the chain
// sequence -> page -> store runs beside them. Large calls (P > 1) read them
// past the caches: 15,518 tokens of 14 + 2 + 2 heads of 64 into e4m3 38.7 ->
// 35.5 us (3.8 TB/s; two or four tokens a block: 39.4, 46). One token 3.6 us
// on the GPU.
template <bool F8, int NL, bool FULL, int P>
__global__ __launch_bounds__(256) void k_paged_append(AppendArgs a) {
#pragma clang fp contract(off)
    constexpr int RPB = 256 / NL;
    const int t = blockIdx.x, hd = FULL ? 4 * NL : a.p.hd, half = hd / 2, nl = hd / 4;
    const int c = threadIdx.x % NL, r0 = blockIdx.y * RPB * P + threadIdx.x / NL;
    const int nkv = a.p.num_kv, rows = a.hq + 2 * nkv;
    const bool lane_in = FULL || c < nl;
    float4 x[P], g[P];
#pragma unroll
    for (int i = 0; i < P; i++) {
        const int r = min(r0 + i * RPB, rows - 1);
        const bool isq = r < a.hq, isk = !isq && r < a.hq + nkv;
        const int h = isq ? r : (isk ? r - a.hq : r - a.hq - nkv);
        const float* src = isq ? a.q + t * a.qs : (isk ? a.k + t * a.ks : a.v + t * a.vs);
        floatx4 v = {0.f, 0.f, 0.f, 0.f};
        if (lane_in) {
            const floatx4* p = reinterpret_cast<const floatx4*>(src + (size_t)h * hd + 4 * c);
            v = P > 1 ? __builtin_nontemporal_load(p) : *p;
        }
        x[i] = make_float4(v[0], v[1], v[2], v[3]);
    }
    SeqAt sq;
    if (!token_seq(a.p, t, sq)) return;
    const int s = sq.s, pos = sq.len - sq.end + t;
    if (pos < 0 || (a.cosT && pos >= a.rope_rows)) return;
    const long long row0 = pool_row(a.p, s, pos, 0);
    if (row0 < 0) return;
    float co[4], sn[4];
    const bool lo = c < nl / 2;
    if (a.cosT) {
        // elements 4c .. 4c + 3 turn by angles 4c mod half .. (neox: 2c, 2c, 2c + 1, 2c + 1)
        const size_t at = (size_t)pos * half + (a.neox ? 2 * c : (lo ? 4 * c : 4 * c - half));
        if (!lane_in) {
            for (int i = 0; i < 4; i++) co[i] = sn[i] = 0.f;
        } else if (a.neox) {
            const float2 cc = *reinterpret_cast<const float2*>(a.cosT + at), ss = *reinterpret_cast<const float2*>(a.sinT + at);
            co[0] = co[1] = cc.x;
            co[2] = co[3] = cc.y;
            sn[0] = sn[1] = ss.x;
            sn[2] = sn[3] = ss.y;
        } else {
            const float4 cc = *reinterpret_cast<const float4*>(a.cosT + at), ss = *reinterpret_cast<const float4*>(a.sinT + at);
            co[0] = cc.x, co[1] = cc.y, co[2] = cc.z, co[3] = cc.w;
            sn[0] = ss.x, sn[1] = ss.y, sn[2] = ss.z, sn[3] = ss.w;
        }
    }
    if (a.gq || a.gk) {
#pragma unroll
        for (int i = 0; i < P; i++) {
            const int r = r0 + i * RPB;
            const float* gain = r < a.hq ? a.gq : (r < a.hq + nkv ? a.gk : nullptr);
            if (gain && lane_in) g[i] = make_float4(gain[4 * c], gain[4 * c + 1], gain[4 * c + 2], gain[4 * c + 3]);
        }
    }
#pragma unroll
    for (int i = 0; i < P; i++) {
        const int r = r0 + i * RPB;
        const bool mine = r < rows && lane_in, isq = r < a.hq, isk = !isq && r < a.hq + nkv;
        const int h = isq ? r : (isk ? r - a.hq : r - a.hq - nkv);
        float4 y = x[i];
        if (a.gq || a.gk) {
            const double ss = row_sum_d<NL>(((double)y.x * (double)y.x + (double)y.y * (double)y.y) +
                                            ((double)y.z * (double)y.z + (double)y.w * (double)y.w));
            if (isq ? a.gq != nullptr : (isk && a.gk != nullptr)) {
                const float inv = (float)rsqrt_f64(div_rcp(ss, (double)hd, 1.0 / hd) + (double)a.eps);
                y = make_float4(y.x * inv * g[i].x, y.y * inv * g[i].y, y.z * inv * g[i].z, y.w * inv * g[i].w);
            }
        }
        if (a.cosT) {
            const float e[4] = {y.x, y.y, y.z, y.w};
            float o[4];
            if (a.neox) {
#pragma unroll
                for (int q = 0; q < 4; q += 2) {
                    o[q] = e[q] * co[q] - e[q + 1] * sn[q];
                    o[q + 1] = e[q] * sn[q] + e[q + 1] * co[q];
                }
            } else {
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    float p;
                    if constexpr (FULL) p = across<NL / 2>(e[q]);
                    else p = __shfl(e[q], (int)(threadIdx.x & 63) + (lo ? nl / 2 : -(nl / 2)));
                    o[q] = lo ? e[q] * co[q] - p * sn[q] : p * sn[q] + e[q] * co[q];
                }
            }
            if (isq || isk) y = make_float4(o[0], o[1], o[2], o[3]);
        }
        if (isq && mine) *reinterpret_cast<float4*>(a.q_out + ((size_t)t * a.hq + h) * hd + 4 * c) = y;
        // the pool rows of a position's heads lie a page's slots apart
        const long long row = mine && !isq ? row0 + (long long)h * a.p.page.d : -1;
        store_kv<F8, NL>(isk ? a.p.k : a.p.v, isk ? a.p.ks : a.p.vs, row, hd, c, mine, y);
    }
}

// TOK tokens a block: their places first, then every load of K and V (a thread
// keeps its four columns), then the stores. Bound by memory: 57,512 tokens of
// 8 x 128 in e4m3 116 us with four tokens a block (5.1 TB/s), 172 with one;
// few tokens have one a block (1,000 in bf16 4.3 us against 5.0).
template <bool F8, int TOK>
__global__ __launch_bounds__(256) void k_paged_read(PagedArgs p, float* ko, float* vo) {
    const int t0 = blockIdx.x * TOK, hd4 = p.hd / 4, n4 = p.num_kv * hd4;
    const int i0 = blockIdx.y * 256 + threadIdx.x, i = min(i0, n4 - 1), h = i / hd4, c = i - h * hd4;
    long long row[TOK];
#pragma unroll
    for (int j = 0; j < TOK; j++) {
        SeqAt sq;
        row[j] = -1;
        if (t0 + j < p.tokens && token_seq(p, t0 + j, sq)) row[j] = pool_row(p, sq.s, sq.len - sq.end + t0 + j, h);
    }
    if (i0 >= n4) return;
    using Raw = typename std::conditional<F8, uint32_t, uint2>::type;
    Raw u[2][TOK];
    float sc[2][TOK];
#pragma unroll
    for (int w = 0; w < 2; w++)
#pragma unroll
        for (int j = 0; j < TOK; j++) {
            if (row[j] < 0 || !(w ? vo : ko)) continue;
            u[w][j] = reinterpret_cast<const Raw*>(w ? p.v : p.k)[row[j] * hd4 + c];
            if constexpr (F8) sc[w][j] = (w ? p.vs : p.ks)[row[j]];
        }
#pragma unroll
    for (int w = 0; w < 2; w++)
#pragma unroll
        for (int j = 0; j < TOK; j++) {
            float* o = w ? vo : ko;
            if (row[j] < 0 || !o) continue;
            float4 x;
            if constexpr (F8) {
                const uint32_t v = u[w][j];
                const float f = sc[w][j];
                x = make_float4(e4m3_f32<0>(v) * f, e4m3_f32<1>(v) * f, e4m3_f32<2>(v) * f, e4m3_f32<3>(v) * f);
            } else {
                x = make_float4(bf16_lo(u[w][j].x), bf16_hi(u[w][j].x), bf16_lo(u[w][j].y), bf16_hi(u[w][j].y));
            }
            *reinterpret_cast<float4*>(o + ((size_t)(t0 + j) * n4 + i) * 4) = x;
        }
}

// Rows per lane group: one while the call's blocks leave CUs idle (a step's
// latency), else as many as spare a token a second block, up to 4.
template <bool F8, int NL, bool FULL>
static void launch_append_nl(hipStream_t s, const AppendArgs& a) {
    constexpr int RPB = 256 / NL;
    const int rows = a.hq + 2 * a.p.num_kv, groups = (rows + RPB - 1) / RPB;
    const auto go = [&](auto kernel, int per) {
        hipLaunchKernelGGL(kernel, dim3(a.p.tokens, (groups + per - 1) / per), dim3(256), 0, s, a);
    };
    if (groups == 1 || (long long)a.p.tokens * groups <= 1024) go(k_paged_append<F8, NL, FULL, 1>, 1);
    else if (groups == 2) go(k_paged_append<F8, NL, FULL, 2>, 2);
    else go(k_paged_append<F8, NL, FULL, 4>, 4);
}
template <bool F8>
static void launch_append(hipStream_t s, const AppendArgs& a) {
    const int hd = a.p.hd;
    if (hd == 64) launch_append_nl<F8, 16, true>(s, a);
    else if (hd < 64) launch_append_nl<F8, 16, false>(s, a);
    else if (hd == 128) launch_append_nl<F8, 32, true>(s, a);
    else if (hd < 128) launch_append_nl<F8, 32, false>(s, a);
    else if (hd == 256) launch_append_nl<F8, 64, true>(s, a);
    else launch_append_nl<F8, 64, false>(s, a);
}

}  // namespace gh

using namespace gh;

extern "C" int gorch_hip_paged_append(void* stream, const gorch_hip_paged_kv* kv, const gorch_hip_paged_batch* b,
                                      const gorch_hip_gqa_weights* w, const float* q, int64_t q_stride, const float* k,
                                      int64_t k_stride, const float* v, int64_t v_stride, float* q_out) {
    AppendArgs a{};
    GH_TRY(paged_args("gorch_hip_paged_append", kv, b, a.p));
    GH_REQUIRE(w, "gorch_hip_paged_append: null heads");
    GH_REQUIRE(w->num_kv == kv->num_kv && w->head_dim == kv->head_dim,
               "gorch_hip_paged_append: the heads and the cache differ in num_kv or head_dim");
    GH_REQUIRE(!q == !q_out, "gorch_hip_paged_append: need both q and q_out or neither");
    GH_REQUIRE(!q || (w->num_q > 0 && w->num_q % w->num_kv == 0), "gorch/nn: GQA NumQ must be divisible by NumKV");
    GH_SUPPORTED(!q || w->num_q <= 0xffff, "gorch_hip_paged_append: num_q must be below 2^16");
    GH_REQUIRE(!w->rope_cos == !w->rope_sin, "gorch_hip_paged_append: need both RoPE tables");
    if (b->tokens == 0 || b->seqs == 0) return GORCH_HIP_OK;
    GH_REQUIRE(k && v, "gorch_hip_paged_append: null k or v");
    const long long kvd = (long long)kv->num_kv * kv->head_dim, qd = (long long)(q ? w->num_q : 0) * kv->head_dim;
    GH_REQUIRE(k_stride >= kvd && v_stride >= kvd && (!q || q_stride >= qd),
               "gorch_hip_paged_append: a row stride is shorter than its row");
    GH_REQUIRE(q_out != q || !q || q_stride == qd || b->tokens == 1,
               "gorch_hip_paged_append: q_out may only be q where q's rows are contiguous");
    GH_SUPPORTED(aligned(q, 16) && aligned(k, 16) && aligned(v, 16) && aligned(q_out, 16) && (!q || q_stride % 4 == 0) &&
                     k_stride % 4 == 0 && v_stride % 4 == 0 && aligned(w->rope_cos, 16) && aligned(w->rope_sin, 16),
                 "gorch_hip_paged_append: rows and RoPE tables must be 16-byte aligned");
    a.q = q;
    a.k = k;
    a.v = v;
    a.qs = q_stride;
    a.ks = k_stride;
    a.vs = v_stride;
    a.q_out = q_out;
    a.hq = q ? w->num_q : 0;
    a.gq = w->q_norm;
    a.gk = w->k_norm;
    a.eps = w->norm_eps;
    a.cosT = w->rope_cos;
    a.sinT = w->rope_sin;
    a.rope_rows = w->rope_max_seq;
    a.neox = w->rope_neox;
    if (kv->dtype == GORCH_HIP_KV_E4M3) launch_append<true>(stream_of(stream), a);
    else launch_append<false>(stream_of(stream), a);
    count(CNT_ELEMENTWISE);
    return finish(stream, check_launch("paged_append"));
}

extern "C" int gorch_hip_paged_read(void* stream, const gorch_hip_paged_kv* kv, const gorch_hip_paged_batch* b,
                                    float* k_out, float* v_out) {
    PagedArgs p{};
    GH_TRY(paged_args("gorch_hip_paged_read", kv, b, p));
    GH_SUPPORTED(aligned(k_out, 16) && aligned(v_out, 16), "gorch_hip_paged_read: outputs must be 16-byte aligned");
    if (b->tokens == 0 || b->seqs == 0 || (!k_out && !v_out)) return GORCH_HIP_OK;
    const auto go = [&](auto kernel, int tok) {
        hipLaunchKernelGGL(kernel, dim3((p.tokens + tok - 1) / tok, (p.num_kv * p.hd / 4 + 255) / 256), dim3(256), 0,
                           stream_of(stream), p, k_out, v_out);
    };
    const bool f8 = kv->dtype == GORCH_HIP_KV_E4M3;
    if (p.tokens < 4096) f8 ? go(k_paged_read<true, 1>, 1) : go(k_paged_read<false, 1>, 1);
    else f8 ? go(k_paged_read<true, 4>, 4) : go(k_paged_read<false, 4>, 4);
    count(CNT_CODEC);
    return finish(stream, check_launch("paged_read"));
}
