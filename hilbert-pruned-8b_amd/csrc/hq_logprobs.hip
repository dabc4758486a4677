// hq_logprobs.hip - log probabilities of given tokens, entropy and likeliest tokens of rows of logits (hq_logprobs,
// include/hq_serve.h).
#include <hip/hip_runtime.h>

#include <math.h>

#include "hq_batch.h"
#include "hq_device.h"

namespace {

struct LpArgs {
    const void *x;
    const uint32_t *ids;
    float *logp, *entropy, *top_logp;
    uint32_t *top_ids;
    int64_t stride;
    uint32_t V;
    int n_ids, k;
};

template <bool F32>
DEV float logit(const void *x, size_t at) {
    return F32 ? ((const float *)x)[at] : (float)((const _Float16 *)x)[at];
}

// Logits as unsigned integers in their order: every NaN above +inf, -0 as +0; with the token below them, lower tokens
// first, one 64-bit key orders candidates.
DEV uint32_t order_of(float x) {
    if (x != x) return 0xffffffffu;
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
DEV float from_order(uint32_t o) {
    if (o == 0xffffffffu) return NAN;
    return __builtin_bit_cast(float, o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
DEV uint64_t key_of(float x, uint32_t at) { return (uint64_t)order_of(x) << 32 | (uint32_t)~at; }

// log p of a logit x in a row of maximum m and sum of e^(x - m) = s
DEV float log_p(float x, float m, float logs) {
    if (m == -INFINITY) return -INFINITY;
    return (x - m) - logs;
}

template <class T, class F>
DEV T block_reduce(T v, T *red, F f) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = f(v, (T)__shfl_xor(v, o, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return f(f(red[0], red[1]), f(red[2], red[3]));
}

// One workgroup per row: the maximum, the sums, then each of the top tokens by a pass over the row.
template <bool F32>
__global__ void __launch_bounds__(256) k_logprobs(LpArgs g) {
    __shared__ float red[4];
    __shared__ unsigned long long rk[4];
    const size_t row = blockIdx.x, at = row * (size_t)g.stride;
    const auto add = [](float a, float b) { return a + b; };
    float m = -INFINITY, nan = 0.f;
    for (uint32_t i = threadIdx.x; i < g.V; i += 256) {
        const float x = logit<F32>(g.x, at + i);
        m = fmaxf(m, x);
        if (x != x) nan = x;
    }
    m = block_reduce(m, red, [](float a, float b) { return fmaxf(a, b); });
    nan = block_reduce(nan, red, add);
    float s = 0.f, t = 0.f;
    if (m != -INFINITY)
        for (uint32_t i = threadIdx.x; i < g.V; i += 256) {
            const float d = logit<F32>(g.x, at + i) - m, e = expf(d);
            s += e;
            if (d != -INFINITY) t += d * e;
        }
    s = block_reduce(s, red, add);
    t = block_reduce(t, red, add);
    const float bad = nan + (m == INFINITY ? NAN : 0.f), logs = logf(s);
    if (g.entropy && threadIdx.x == 0) g.entropy[row] = bad + (m == -INFINITY ? 0.f : logs - t / s);
    if (g.logp)
        for (int j = threadIdx.x; j < g.n_ids; j += 256) {
            const uint32_t id = g.ids[row * g.n_ids + j];
            g.logp[row * g.n_ids + j] = id < g.V ? bad + log_p(logit<F32>(g.x, at + id), m, logs) : NAN;
        }
    if (!g.top_ids && !g.top_logp) return;
    unsigned long long below = ~0ull;
    for (int j = 0; j < g.k; j++) {
        unsigned long long best = 0;
        for (uint32_t i = threadIdx.x; i < g.V; i += 256) {
            const unsigned long long key = key_of(logit<F32>(g.x, at + i), i);
            if (key < below && key > best) best = key;
        }
        best = block_reduce(best, rk, [](unsigned long long a, unsigned long long b) { return a > b ? a : b; });
        below = best;
        if (threadIdx.x == 0) {
            if (g.top_ids) g.top_ids[row * g.k + j] = ~(uint32_t)best;
            if (g.top_logp) g.top_logp[row * g.k + j] = bad + log_p(from_order((uint32_t)(best >> 32)), m, logs);
        }
    }
}

}  // namespace

extern "C" int hq_logprobs(const void *logits, int f32, int M, uint32_t V, int64_t stride, const uint32_t *ids, int n_ids, int top_k,
                           float *logp, float *entropy, uint32_t *top_ids, float *top_logp, void *stream) {
    const char *const who = "hq_logprobs";
    if (M < 0 || M > (1 << 24) || V < 1 || V > (1u << 30)) return hq_internal_fail("%s: %d rows of %u (at most 2^24 of 2^30)", who, M, V);
    if (stride < (int64_t)V || stride > ((int64_t)1 << 40)) return hq_internal_fail("%s: stride %lld (at least %u)", who, (long long)stride, V);
    if (n_ids < 0 || n_ids > (1 << 20)) return hq_internal_fail("%s: %d tokens per row", who, n_ids);
    if (top_k < 0 || top_k > HQ_LOGPROBS_MAX_TOP || (uint32_t)top_k > V) return hq_internal_fail("%s: top_k %d (at most %d and V)", who, top_k, HQ_LOGPROBS_MAX_TOP);
    if (M == 0) return 0;
    if (!logits || (n_ids && logp && !ids)) return hq_internal_fail("%s: null argument", who);
    if ((uintptr_t)logits % (f32 ? 4 : 2)) return hq_internal_fail("%s: the logits are misaligned", who);
    if (n_ids == 0) logp = nullptr;
    if (top_k == 0) top_ids = nullptr, top_logp = nullptr;
    if (!logp && !entropy && !top_ids && !top_logp) return 0;
    const LpArgs g = {logits, ids, logp, entropy, top_logp, top_ids, stride, V, n_ids, top_k};
    if (f32) k_logprobs<true><<<(unsigned)M, 256, 0, (hipStream_t)stream>>>(g);
    else k_logprobs<false><<<(unsigned)M, 256, 0, (hipStream_t)stream>>>(g);
    SCK(hipGetLastError());
    return 0;
}
