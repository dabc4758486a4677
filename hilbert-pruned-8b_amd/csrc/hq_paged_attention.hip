// hq_paged_attention.hip - attention of a step's new tokens over the paged cache (hq_attention, include/hq_serve.h).
#include <hip/hip_runtime.h>

#include <math.h>

#include "hq_batch.h"
#include "hq_device.h"

namespace {

struct Args {
    hq_kv_t kv;
    hq_attn_t a;
    const int *tok_pos, *tok_seq;
    const HqSeq *seqs;
    const uint32_t *pages;
    int nh, rep;
};

template <bool Q8>
DEV float kv_at(const void *p, size_t at) {
    return Q8 ? (float)((const int8_t *)p)[at] : (float)((const _Float16 *)p)[at];
}

DEV float wave_max(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}
DEV float wave_sum(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// One wave per token and head: 64 positions at a time, a lane a score, then a lane every 64th dim of the output, with a
// running maximum and sum.
template <bool Q8>
__global__ void __launch_bounds__(64) k_attn_paged(Args g) {
    __shared__ float q[256], ps[64];
    __shared__ uint32_t row[64];
    const int t = blockIdx.x, h = blockIdx.y, lane = threadIdx.x, hd = g.kv.head_dim, kvh = h / g.rep;
    const HqSeq s = g.seqs[g.tok_seq[t]];
    const int n = g.tok_pos[t] + 1, ps_ = g.kv.page_size;
    for (int d = lane; d < hd; d += 64) q[d] = (float)((const _Float16 *)g.a.q)[(size_t)t * g.a.q_stride + (size_t)h * hd + d] * g.a.scale;
    float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int p0 = 0; p0 < n; p0 += 64) {
        __syncthreads();
        const int p = p0 + lane;
        float x = -INFINITY;
        if (p < n) {
            const uint32_t page = g.pages[s.page0 + p / ps_], in = (uint32_t)p % (uint32_t)ps_;
            row[lane] = page * (uint32_t)ps_ + in;
            const size_t at = (size_t)page * g.kv.page_stride + (size_t)in * g.kv.pos_stride + (size_t)kvh * g.kv.head_stride;
            x = 0.f;
            for (int d = 0; d < hd; d++) x += q[d] * kv_at<Q8>(g.kv.k, at + d);
            if (Q8) x *= h2f(g.kv.k_scale[((size_t)page * g.kv.n_kv_heads + kvh) * ps_ + in]);
        }
        const float mn = fmaxf(m, wave_max(x)), m0 = mn == -INFINITY ? 0.f : mn;
        const float e = p < n ? expf(x - m0) : 0.f, f = expf(m - m0);
        ps[lane] = e;
        l = l * f + wave_sum(e);
        m = mn;
        __syncthreads();
        for (int i = 0; i < 4; i++) o[i] *= f;
        for (int j = 0; j < 64 && p0 + j < n; j++) {
            const uint32_t page = row[j] / (uint32_t)ps_, in = row[j] % (uint32_t)ps_;
            const size_t at = (size_t)page * g.kv.page_stride + (size_t)in * g.kv.pos_stride + (size_t)kvh * g.kv.head_stride;
            const float w = Q8 ? ps[j] * h2f(g.kv.v_scale[((size_t)page * g.kv.n_kv_heads + kvh) * ps_ + in]) : ps[j];
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (lane + 64 * i < hd) o[i] += w * kv_at<Q8>(g.kv.v, at + lane + 64 * i);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int d = lane + 64 * i;
        if (d >= hd) continue;
        float y = n > 0 ? o[i] / l : 0.f;
        if (g.a.gate) {
            const size_t at = (size_t)t * g.a.gate_stride + (size_t)h * g.a.gate_head_stride + d;
            y *= 1.0f / (1.0f + expf(-(g.a.gate_f32 ? ((const float *)g.a.gate)[at] : (float)((const _Float16 *)g.a.gate)[at])));
        }
        ((_Float16 *)g.a.out)[(size_t)t * g.a.out_stride + (size_t)h * hd + d] = (_Float16)y;
    }
}

}  // namespace

extern "C" int hq_attention(const hq_batch *b, const hq_kv_t *kv, const hq_attn_t *a, void *stream) {
    const char *const who = "hq_attention";
    if (!b || !kv || !a) return hq_internal_fail("%s: null argument", who);
    if (!b->set) return hq_internal_fail("%s: the batch describes no step (hq_batch_set)", who);
    if (hq_kv_check(who, kv, b)) return -1;
    if (b->n_tokens == 0) return 0;
    if (!a->q || !a->out) return hq_internal_fail("%s: null argument", who);
    if ((uintptr_t)a->q % 16 || (uintptr_t)a->out % 16) return hq_internal_fail("%s: q and out must be 16-byte aligned", who);
    const int64_t most = (int64_t)1 << 40, row = (int64_t)b->n_heads * kv->head_dim;
    if (a->q_stride < 0 || a->q_stride > most || a->q_stride % 8 || a->out_stride < row || a->out_stride > most || a->out_stride % 8)
        return hq_internal_fail("%s: strides %lld and %lld (multiples of 8; out's at least a row's %lld)", who, (long long)a->q_stride,
                                (long long)a->out_stride, (long long)row);
    if (!isfinite(a->scale)) return hq_internal_fail("%s: scale %g", who, (double)a->scale);
    if (a->gate) {
        if ((uintptr_t)a->gate % (a->gate_f32 ? 16 : 8)) return hq_internal_fail("%s: the gate must be aligned to 4 elements", who);
        if (a->gate_stride < 0 || a->gate_stride > most || a->gate_stride % 4 || a->gate_head_stride < 0 || a->gate_head_stride > most || a->gate_head_stride % 4)
            return hq_internal_fail("%s: gate strides %lld and %lld (multiples of 4)", who, (long long)a->gate_stride, (long long)a->gate_head_stride);
    }
    int cur = -1;
    SCK(hipGetDevice(&cur));
    if (cur != b->device) SCK(hipSetDevice(b->device));
    const Args g = {*kv, *a, b->tok_pos, b->tok_seq, b->seqs, b->pages, b->n_heads, b->n_heads / kv->n_kv_heads};
    const dim3 grid((unsigned)b->n_tokens, (unsigned)b->n_heads);
    if (kv->type == HQ_KV_Q8) k_attn_paged<true><<<grid, 64, 0, (hipStream_t)stream>>>(g);
    else k_attn_paged<false><<<grid, 64, 0, (hipStream_t)stream>>>(g);
    SCK(hipGetLastError());
    return 0;
}
