// logits.hip — a request's rules on its logits before a token is chosen
// (gorch_hip_process_logits; no counterpart in the reference, whose
// GenerateConfig has temperature, top-k and top-p only,
// model/generate.go:13-42).
//
// A block takes a slice of one row's vocabulary: it counts the row's history
// tokens of that slice in LDS (integers, so any order gives the same counts),
// notes the last bias entry of each, and takes the slice's logits through the
// rules. Every block of a row reads the whole history (from L2). Bound by
// memory: the logits and the mask go out first and arrive while the notes are
// taken.
#include "common.h"

namespace gh {

struct LogitsArgs {
    gorch_hip_logits_rules r;
    const float* x;
    float* out;
    int n, wide_history;
};

constexpr uint32_t kInPrompt = 0x80000000u;  // beside the count of tokens after the prompt

// Blocks of NT threads, U groups of four tokens each. Slices start where x is
// 16-byte aligned, up to three tokens before a multiple of their size, so rows
// of any length move in 16-byte pieces; SAME: out is aligned as x is (else it
// is stored token by token). Large calls (U > 1) pass the caches by, in and
// out: 256 x 151,936 logits with histories of up to 4,000 and 300 biases each
// 69.4 -> 62.6 us (5.1 TB/s; a large copy reaches 4.9), against 81 for blocks of
// 256 threads with four groups, whose history is scanned by half as many.
template <int NT, int U, bool SAME>
__global__ __launch_bounds__(NT) void k_process_logits(LogitsArgs a) {
    constexpr int SLICE = 4 * NT * U, HISTORY = 1024 / NT;
    extern __shared__ __align__(16) uint32_t note[];  // per token: kInPrompt | count after the prompt
    const gorch_hip_logits_rules& r = a.r;
    uint32_t* last = note + (r.history ? SLICE : 0);  // per token: last bias entry + 1
    const int row = blockIdx.y, tid = threadIdx.x;
    const float* x = a.x + (size_t)row * a.n;
    float* out = a.out + (size_t)row * a.n;
    const int lo = (int)blockIdx.x * SLICE - (int)(reinterpret_cast<uintptr_t>(x) / 4 % 4);
    // everything that the block is sure to read goes out at once
    int len = 0, prompt = 0, b0 = 0, b1 = 0;
    const int* h = r.history + (size_t)row * r.history_stride;
    int4 id[HISTORY];
    if (r.history) {
        len = r.history_lens ? min(max(r.history_lens[row], 0), r.history_stride) : r.history_stride;
        prompt = r.prompt_lens ? r.prompt_lens[row] : 0;
        if (a.wide_history)
#pragma unroll
            for (int u = 0; u < HISTORY; u++) {
                const int i = 4 * (u * NT + tid);
                if (i < r.history_stride) id[u] = *reinterpret_cast<const int4*>(h + i);
            }
    }
    if (r.bias) {
        b0 = min(max(r.bias_rows[row], 0), r.biases);
        b1 = min(max(r.bias_rows[row + 1], b0), r.biases);
    }
    floatx4 v[U];
    uint32_t w0[U], w1[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int t = lo + 4 * (u * NT + tid);
        if (t >= 0 && t + 4 <= a.n) {
            const floatx4* p = reinterpret_cast<const floatx4*>(x + t);
            v[u] = U > 1 ? __builtin_nontemporal_load(p) : *p;
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) v[u][i] = t + i >= 0 && t + i < a.n ? x[t + i] : 0.f;
        }
        w0[u] = w1[u] = ~0u;
        if (r.allowed) {
            const uint32_t* m = r.allowed + (size_t)row * r.allowed_stride;
            w0[u] = m[min(max(t, 0), a.n - 1) / 32];
            w1[u] = m[min(max(t + 3, 0), a.n - 1) / 32];
        }
    }
    if (r.history || r.bias) {
        const uint4 none = make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (r.history) reinterpret_cast<uint4*>(note)[u * NT + tid] = none;
            if (r.bias) reinterpret_cast<uint4*>(last)[u * NT + tid] = none;
        }
        __syncthreads();
        if (r.history) {
            auto take = [&](int i, int token) {
                const unsigned at = (unsigned)(token - lo);
                if (i >= len || at >= (unsigned)SLICE || (unsigned)token >= (unsigned)a.n) return;
                if (i < prompt) atomicOr(&note[at], kInPrompt);
                else atomicAdd(&note[at], 1u);
            };
            auto take4 = [&](int i, const int4& t) {
                take(i, t.x);
                take(i + 1, t.y);
                take(i + 2, t.z);
                take(i + 3, t.w);
            };
            if (a.wide_history) {
#pragma unroll
                for (int u = 0; u < HISTORY; u++)
                    if (4 * (u * NT + tid) < len) take4(4 * (u * NT + tid), id[u]);
                for (int i = 4 * (HISTORY * NT + tid); i < len; i += 4 * NT) take4(i, *reinterpret_cast<const int4*>(h + i));
            } else {
                for (int i = tid; i < len; i += NT) take(i, h[i]);
            }
        }
        if (r.bias)
            for (int i = b0 + tid; i < b1; i += NT) {
                const int token = r.bias_ids[i];
                const unsigned at = (unsigned)(token - lo);
                if (at < (unsigned)SLICE && (unsigned)token < (unsigned)a.n) atomicMax(&last[at], (uint32_t)i + 1);
            }
        __syncthreads();
    }
    const float rep = r.repetition ? r.repetition[row] : 1.f, fr = r.frequency ? r.frequency[row] : 0.f,
                pr = r.presence ? r.presence[row] : 0.f;
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int t = lo + 4 * (u * NT + tid);
        floatx4 e = v[u];
        // bits of tokens t .. t + 3 (those before the row or past it are never stored)
        const uint64_t bits = w0[u] | ((uint64_t)w1[u] << 32);
        const uint32_t ok = t >= 0 ? (uint32_t)(bits >> (t % 32)) : (uint32_t)(bits << -t);
        if (r.history) {
            const uint4 w = reinterpret_cast<const uint4*>(note)[u * NT + tid];
            const uint32_t c[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (c[i] == 0) continue;
                const uint32_t k = c[i] & ~kInPrompt;
                if (r.repetition) e[i] = e[i] > 0.f ? e[i] / rep : e[i] * rep;
                if (k) e[i] = e[i] - fr * (float)k - pr;
            }
        }
        if (r.bias) {
            const uint4 w = reinterpret_cast<const uint4*>(last)[u * NT + tid];
            const uint32_t c[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (c[i]) e[i] += r.bias[c[i] - 1];
        }
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (!(ok >> i & 1u)) e[i] = -INFINITY;
        if (SAME && t >= 0 && t + 4 <= a.n) {
            floatx4* p = reinterpret_cast<floatx4*>(out + t);
            if constexpr (U > 1) __builtin_nontemporal_store(e, p);
            else *p = e;
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (t + i >= 0 && t + i < a.n) out[t + i] = e[i];
        }
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
    GH_SUPPORTED(reinterpret_cast<uintptr_t>(logits) % 4 == 0 && n < 0x7fff0000,
                 "gorch_hip_process_logits: logits must be 4-byte aligned, n below 2^31 - 2^16");
    LogitsArgs a{*r, logits, out, n, 0};
    if (r->biases == 0) a.r.bias = nullptr;
    a.wide_history = reinterpret_cast<uintptr_t>(r->history) % 16 == 0 && r->history_stride % 4 == 0;
    const bool same = (reinterpret_cast<uintptr_t>(logits) - reinterpret_cast<uintptr_t>(out)) % 16 == 0;
    const int words = (a.r.history ? 1 : 0) + (a.r.bias ? 1 : 0);
    const auto go = [&](auto kernel, int threads, int slice) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)(((long long)n + 3 + slice - 1) / slice), rows), dim3(threads),
                           (size_t)words * slice * 4, stream_of(stream), a);
    };
    // few rows: slices of 1024 tokens, so that more CUs share the latency;
    // many: of 4096, so that fewer blocks read a row's history
    if ((long long)rows * n < 512 * 4096ll) {
        if (same) go(k_process_logits<256, 1, true>, 256, 1024);
        else go(k_process_logits<256, 1, false>, 256, 1024);
    } else {
        if (same) go(k_process_logits<512, 2, true>, 512, 4096);
        else go(k_process_logits<512, 2, false>, 512, 4096);
    }
    count(CNT_ELEMENTWISE);
    return finish(stream, check_launch("process_logits"));
}
