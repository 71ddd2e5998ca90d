// logits.hip — a request's rules on its logits before a token is chosen
// (gorch_hip_process_logits; no counterpart in the reference, whose
// GenerateConfig has temperature, top-k and top-p only,
// model/generate.go:13-42).
//
// A block takes a slice of one row's vocabulary: it counts the row's history
// tokens of that slice in LDS (integers, so any order gives the same counts),
// notes the last bias entry of each, and streams the slice's logits through
// the rules. Every block of a row reads the whole history (from L2).
#include "common.h"

namespace gh {

struct LogitsArgs {
    gorch_hip_logits_rules r;
    const float* x;
    float* out;
    int n, slice;
};

constexpr uint32_t kInPrompt = 0x80000000u;  // beside the count of tokens after the prompt

// note: per token of the slice, kInPrompt | count after the prompt; last: the
// last bias entry + 1
__global__ __launch_bounds__(256) void k_process_logits(LogitsArgs a) {
    extern __shared__ uint32_t note[];
    const int row = blockIdx.y, lo = blockIdx.x * a.slice, n = min(a.slice, a.n - lo);
    const gorch_hip_logits_rules& r = a.r;
    uint32_t* last = note + (r.history ? a.slice : 0);
    if (r.history)
        for (int i = threadIdx.x; i < n; i += 256) note[i] = 0;
    if (r.bias)
        for (int i = threadIdx.x; i < n; i += 256) last[i] = 0;
    __syncthreads();
    if (r.history) {
        const int len = r.history_lens ? min(max(r.history_lens[row], 0), r.history_stride) : r.history_stride;
        const int prompt = r.prompt_lens ? r.prompt_lens[row] : 0;
        const int* h = r.history + (size_t)row * r.history_stride;
        for (int i = threadIdx.x; i < len; i += 256) {
            const int id = h[i] - lo;
            if ((unsigned)id >= (unsigned)n) continue;
            if (i < prompt) atomicOr(&note[id], kInPrompt);
            else atomicAdd(&note[id], 1u);
        }
    }
    if (r.bias) {
        const int b0 = min(max(r.bias_rows[row], 0), r.biases), b1 = min(max(r.bias_rows[row + 1], b0), r.biases);
        for (int i = b0 + threadIdx.x; i < b1; i += 256) {
            const int id = r.bias_ids[i] - lo;
            if ((unsigned)id < (unsigned)n) atomicMax(&last[id], (uint32_t)i + 1);
        }
    }
    __syncthreads();
    const float rep = r.repetition ? r.repetition[row] : 1.f, fr = r.frequency ? r.frequency[row] : 0.f,
                pr = r.presence ? r.presence[row] : 0.f;
    for (int i = threadIdx.x; i < n; i += 256) {
        float x = a.x[(size_t)row * a.n + lo + i];
        if (r.history && note[i]) {
            const uint32_t c = note[i] & ~kInPrompt;
            if (r.repetition) x = x > 0.f ? x / rep : x * rep;
            if (c) x = x - fr * (float)c - pr;
        }
        if (r.bias && last[i]) x += r.bias[last[i] - 1];
        if (r.allowed && !(r.allowed[(size_t)row * r.allowed_stride + (lo + i) / 32] >> ((lo + i) % 32) & 1u)) x = -INFINITY;
        a.out[(size_t)row * a.n + lo + i] = x;
    }
}

}  // namespace gh

using namespace gh;

extern "C" int gorch_hip_process_logits(void* stream, const gorch_hip_logits_rules* r, const float* logits, float* out,
                                        int rows, int n) {
    GH_REQUIRE(r && rows >= 0 && n >= 0, "gorch_hip_process_logits: bad arguments");
    GH_REQUIRE(!r->history || r->history_stride >= 0, "gorch_hip_process_logits: negative history_stride");
    GH_REQUIRE(r->biases >= 0 && (r->biases == 0 || (r->bias && r->bias_rows && r->bias_ids)),
               "gorch_hip_process_logits: biases need bias_rows, bias_ids and bias");
    GH_REQUIRE(!r->allowed || (long long)r->allowed_stride * 32 >= n,
               "gorch_hip_process_logits: allowed_stride is shorter than n bits");
    GH_SUPPORTED(rows <= 65535, "gorch_hip_process_logits: more than 65535 rows");
    if (rows == 0 || n == 0) return GORCH_HIP_OK;
    GH_REQUIRE(logits && out, "gorch_hip_process_logits: null logits or out");
    LogitsArgs a{*r, logits, out, n, 4096};
    if (r->biases == 0) a.r.bias = nullptr;
    const size_t lds = (size_t)((a.r.history ? 1 : 0) + (a.r.bias ? 1 : 0)) * a.slice * 4;
    hipLaunchKernelGGL(k_process_logits, dim3((n + a.slice - 1) / a.slice, rows), dim3(256), lds, stream_of(stream), a);
    count(CNT_ELEMENTWISE);
    return finish(stream, check_launch("process_logits"));
}
