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
    const long long room = (long long)b->max_pages * kv->page_size;
    if (room > 0x7fffffffll) return fail(GORCH_HIP_EINVAL, "max_pages * page_size must be below 2^31");
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

// Sums and maxima over the NL lanes of a row (NL a power of two).
template <int NL>
__device__ __forceinline__ double row_sum_d(double v) {
#pragma unroll
    for (int m = 1; m < NL; m *= 2) v += __shfl_xor(v, m);
    return v;
}
template <int NL>
__device__ __forceinline__ float row_max_f(float v) {
#pragma unroll
    for (int m = 1; m < NL; m *= 2) v = fmaxf(v, __shfl_xor(v, m));
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
// floats (lane c < hd / 4 holds elements 4c .. 4c + 3), a wave one row of
// lanes at a time. Same operations per row, in the same order, as
// k_norm_rope_rows: x * inv * gain with inv from the f64 sum of squares, then
// the pair rotated with every product and sum rounded on its own.
template <bool F8, int NL>
__global__ __launch_bounds__(256) void k_paged_append(AppendArgs a) {
#pragma clang fp contract(off)
    constexpr int RPB = 256 / NL;
    const int t = blockIdx.x, hd = a.p.hd, half = hd / 2, nl = hd / 4;
    const int c = threadIdx.x % NL, r = blockIdx.y * RPB + threadIdx.x / NL;
    SeqAt sq;
    if (!token_seq(a.p, t, sq)) return;
    const int s = sq.s, pos = sq.len - sq.end + t;
    if (pos < 0 || (a.cosT && pos >= a.rope_rows) || pool_row(a.p, s, pos, 0) < 0) return;
    const int nkv = a.p.num_kv, rows = a.hq + 2 * nkv;
    const bool live = r < rows, mine = live && c < nl;
    const bool isq = r < a.hq, isk = !isq && r < a.hq + nkv;
    const int h = isq ? r : (isk ? r - a.hq : r - a.hq - nkv);
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f), g = make_float4(1.f, 1.f, 1.f, 1.f);
    const float* src = isq ? a.q + t * a.qs : (isk ? a.k + t * a.ks : a.v + t * a.vs);
    if (mine) x = *reinterpret_cast<const float4*>(src + (size_t)h * hd + 4 * c);
    const float* gain = isq ? a.gq : (isk ? a.gk : nullptr);
    const double ss = row_sum_d<NL>(((double)x.x * (double)x.x + (double)x.y * (double)x.y) +
                                    ((double)x.z * (double)x.z + (double)x.w * (double)x.w));
    if (gain && mine) {
        g = make_float4(gain[4 * c], gain[4 * c + 1], gain[4 * c + 2], gain[4 * c + 3]);
        const float inv = (float)rsqrt_f64(div_rcp(ss, (double)hd, 1.0 / hd) + (double)a.eps);
        x = make_float4(x.x * inv * g.x, x.y * inv * g.y, x.z * inv * g.z, x.w * inv * g.w);
    }
    if (a.cosT) {
        const bool lo = c < nl / 2;
        const int lane = threadIdx.x & 63, other = lo ? lane + nl / 2 : lane - nl / 2;
        const float e[4] = {x.x, x.y, x.z, x.w};
        float o[4];
        for (int i = 0; i < 4; i++) {
            const float p = __shfl(e[a.neox ? i ^ 1 : i], a.neox ? lane : other);
            const int at = a.neox ? 2 * c + i / 2 : (lo ? 4 * c + i : 4 * c + i - half);
            const bool first = a.neox ? (i & 1) == 0 : lo;
            float co = 1.f, si = 0.f;
            if (mine) {
                co = a.cosT[(size_t)pos * half + at];
                si = a.sinT[(size_t)pos * half + at];
            }
            o[i] = first ? e[i] * co - p * si : p * si + e[i] * co;
        }
        if (isq || isk) x = make_float4(o[0], o[1], o[2], o[3]);
    }
    if (isq && mine) *reinterpret_cast<float4*>(a.q_out + ((size_t)t * a.hq + h) * hd + 4 * c) = x;
    const long long row = live && !isq ? pool_row(a.p, s, pos, h) : -1;
    store_kv<F8, NL>(isk ? a.p.k : a.p.v, isk ? a.p.ks : a.p.vs, row, hd, c, mine, x);
}

template <bool F8>
__global__ __launch_bounds__(256) void k_paged_read(PagedArgs p, float* ko, float* vo) {
    const int t = blockIdx.x;
    SeqAt sq;
    if (!token_seq(p, t, sq)) return;
    const int s = sq.s, pos = sq.len - sq.end + t;
    if (pos < 0) return;
    const int n4 = p.num_kv * p.hd / 4, hd4 = p.hd / 4;
    for (int i = threadIdx.x; i < n4; i += 256) {
        const int h = i / hd4, c = i - h * hd4;
        const long long row = pool_row(p, s, pos, h);
        if (row < 0) return;
        for (int w = 0; w < 2; w++) {
            float* o = w ? vo : ko;
            if (!o) continue;
            const void* pool = w ? p.v : p.k;
            float4 x;
            if constexpr (F8) {
                const uint32_t u = reinterpret_cast<const uint32_t*>(pool)[row * hd4 + c];
                const float sc = (w ? p.vs : p.ks)[row];
                x = make_float4(e4m3_f32<0>(u) * sc, e4m3_f32<1>(u) * sc, e4m3_f32<2>(u) * sc, e4m3_f32<3>(u) * sc);
            } else {
                const uint2 u = reinterpret_cast<const uint2*>(pool)[row * hd4 + c];
                x = make_float4(bf16_lo(u.x), bf16_hi(u.x), bf16_lo(u.y), bf16_hi(u.y));
            }
            *reinterpret_cast<float4*>(o + (size_t)t * p.num_kv * p.hd + 4 * i) = x;
        }
    }
}

template <bool F8>
static void launch_append(hipStream_t s, const AppendArgs& a) {
    const int rows = a.hq + 2 * a.p.num_kv, nl = a.p.hd / 4;
    const auto go = [&](auto kernel, int lanes) {
        const int rpb = 256 / lanes;
        hipLaunchKernelGGL(kernel, dim3(a.p.tokens, (rows + rpb - 1) / rpb), dim3(256), 0, s, a);
    };
    if (nl <= 16) go(k_paged_append<F8, 16>, 16);
    else if (nl <= 32) go(k_paged_append<F8, 32>, 32);
    else go(k_paged_append<F8, 64>, 64);
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
    GH_REQUIRE(!w->rope_cos == !w->rope_sin, "gorch_hip_paged_append: need both RoPE tables");
    if (b->tokens == 0 || b->seqs == 0) return GORCH_HIP_OK;
    GH_REQUIRE(k && v, "gorch_hip_paged_append: null k or v");
    const long long kvd = (long long)kv->num_kv * kv->head_dim, qd = (long long)(q ? w->num_q : 0) * kv->head_dim;
    GH_REQUIRE(k_stride >= kvd && v_stride >= kvd && (!q || q_stride >= qd),
               "gorch_hip_paged_append: a row stride is shorter than its row");
    GH_REQUIRE(q_out != q || !q || q_stride == qd || b->tokens == 1,
               "gorch_hip_paged_append: q_out may only be q where q's rows are contiguous");
    GH_SUPPORTED(aligned(q, 16) && aligned(k, 16) && aligned(v, 16) && aligned(q_out, 16) && (!q || q_stride % 4 == 0) &&
                     k_stride % 4 == 0 && v_stride % 4 == 0,
                 "gorch_hip_paged_append: rows must be 16-byte aligned");
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
    if (kv->dtype == GORCH_HIP_KV_E4M3)
        hipLaunchKernelGGL(k_paged_read<true>, dim3(p.tokens), dim3(256), 0, stream_of(stream), p, k_out, v_out);
    else
        hipLaunchKernelGGL(k_paged_read<false>, dim3(p.tokens), dim3(256), 0, stream_of(stream), p, k_out, v_out);
    count(CNT_CODEC);
    return finish(stream, check_launch("paged_read"));
}
