// paged_attention.hip — attention of ragged new tokens over a KV cache in
// pages (gorch_hip_gqa_attention_cached's mathematics, GQA.forwardCached
// nn/gqa.go:308-352):
//   o = sum_j p_j v_j / sum_j p_j, p_j = exp(q . k_j / sqrt(hd) - max_j ...)
// over the positions j that the token sees.
#include "paged.h"

namespace gh {

struct PagedAttnArgs {
    PagedArgs p;
    const float* q;
    float* out;
    int hq, causal;
    float scale;
};

template <bool F8>
__device__ __forceinline__ float pool_value(const void* pool, long long i) {
    if constexpr (F8) return e4m3_f32<0>(reinterpret_cast<const uint8_t*>(pool)[i]);
    return bf16_lo(reinterpret_cast<const uint16_t*>(pool)[i]);
}

// One wave per (query head, token): 64 keys at a time, a lane each for the
// scores, then a lane per column (up to four) for the weighted values.
template <bool F8>
__global__ __launch_bounds__(64) void k_paged_attn_rows(PagedAttnArgs a) {
    __shared__ float qs[256], ps[64];
    __shared__ long long rows[64];
    const int lane = threadIdx.x, h = blockIdx.x, t = blockIdx.y, hd = a.p.hd;
    const int s = wave_find(a.p.seqs, t, [&](int i) { return seq_begin(a.p, i); });
    if (s < 0) return;
    const int end = seq_begin(a.p, s + 1);
    if (t >= end) return;
    const int len = a.p.lens[s], pos = len - end + t;
    const int T = min(a.causal ? pos + 1 : len, a.p.limit);
    const int kvh = h / (a.hq / a.p.num_kv);
    for (int d = lane; d < hd; d += 64) qs[d] = a.q[((size_t)t * a.hq + h) * hd + d] * a.scale;
    float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int j0 = 0; j0 < T; j0 += 64) {
        const long long row = j0 + lane < T ? pool_row(a.p, s, j0 + lane, kvh) : -1;
        __syncthreads();
        float sc = -INFINITY;
        if (row >= 0) {
            float d = 0.f;
            for (int e = 0; e < hd; e++) d += qs[e] * pool_value<F8>(a.p.k, row * hd + e);
            sc = F8 ? d * a.p.ks[row] : d;
        }
        const float mn = fmaxf(m, wave_max(sc)), use = mn == -INFINITY ? 0.f : mn;
        const float p = row >= 0 ? expf(sc - use) : 0.f, al = expf(m - use);
        l = l * al + wave_sum(p);
        ps[lane] = F8 && row >= 0 ? p * a.p.vs[row] : p;
        rows[lane] = row;
        m = mn;
        __syncthreads();
        for (int i = 0; i < 4; i++) o[i] *= al;
        for (int j = 0; j < 64; j++) {
            if (rows[j] < 0) continue;
            for (int i = 0; i < 4; i++)
                if (lane + 64 * i < hd) o[i] += ps[j] * pool_value<F8>(a.p.v, rows[j] * hd + lane + 64 * i);
        }
    }
    for (int i = 0; i < 4; i++)
        if (lane + 64 * i < hd) a.out[((size_t)t * a.hq + h) * hd + lane + 64 * i] = l == 0.f ? 0.f : o[i] / l;
}

static int attn_args(const gorch_hip_paged_kv* kv, const gorch_hip_paged_batch* b, int num_q, PagedAttnArgs& a) {
    GH_TRY(paged_args("gorch_hip_paged_attention", kv, b, a.p));
    GH_REQUIRE(num_q > 0 && num_q % kv->num_kv == 0, "gorch/nn: GQA NumQ must be divisible by NumKV");
    a.hq = num_q;
    a.scale = (float)(1.0 / sqrt((double)kv->head_dim));
    return GORCH_HIP_OK;
}

}  // namespace gh

using namespace gh;

extern "C" size_t gorch_hip_paged_attention_workspace_size(const gorch_hip_paged_kv* kv, const gorch_hip_paged_batch* b,
                                                           int num_q) {
    return 0;
}

extern "C" int gorch_hip_paged_attention(void* stream, const gorch_hip_paged_kv* kv, const gorch_hip_paged_batch* b,
                                         const float* q, int num_q, float* out, int causal, void* workspace,
                                         size_t workspace_bytes) {
    PagedAttnArgs a{};
    GH_TRY(attn_args(kv, b, num_q, a));
    if (b->tokens == 0 || b->seqs == 0) return GORCH_HIP_OK;
    GH_REQUIRE(q && out, "gorch_hip_paged_attention: null q or out");
    GH_SUPPORTED(reinterpret_cast<uintptr_t>(q) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0,
                 "gorch_hip_paged_attention: q and out must be 16-byte aligned");
    GH_TRY(bf16_gate(stream_of(stream)));
    a.q = q;
    a.out = out;
    a.causal = causal != 0;
    GH_SUPPORTED(a.p.tokens <= 65535, "gorch_hip_paged_attention: too many tokens");
    if (kv->dtype == GORCH_HIP_KV_E4M3)
        hipLaunchKernelGGL(k_paged_attn_rows<true>, dim3(num_q, a.p.tokens), dim3(64), 0, stream_of(stream), a);
    else
        hipLaunchKernelGGL(k_paged_attn_rows<false>, dim3(num_q, a.p.tokens), dim3(64), 0, stream_of(stream), a);
    count(CNT_ATTENTION);
    return finish(stream, check_launch("paged_attention"));
}
