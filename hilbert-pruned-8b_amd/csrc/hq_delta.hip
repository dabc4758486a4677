// hq_delta.hip - the gated delta recurrence of a step's sequences (hq_delta, include/hq_serve.h).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <math.h>

#include "hq_device.h"
#include "hq_scan.h"

namespace {

bool aligned(const void *p, size_t a) { return ((uintptr_t)p % a) == 0; }

struct DeltaArgs {
    hq_state_t st;
    hq_delta_t d;
    const HqSeq *seqs;
    const int *steps;
};

DEV f4 sum_over(f4 x, int lanes) {
    return f4{x[0] + __shfl_xor(x[0], lanes, 64), x[1] + __shfl_xor(x[1], lanes, 64), x[2] + __shfl_xor(x[2], lanes, 64), x[3] + __shfl_xor(x[3], lanes, 64)};
}

// Token by token. A workgroup holds one head's S in registers, 16 rows x 4 columns a lane: column group tid % CG, row group tid / CG.
// With p = S^T k and r = S^T q of the state before the token, formed together, a token costs one meeting of the waves:
//   u = beta (v - e^g p),  o = scale (e^g r + (k q) u),  S' = e^g S + k u.
template <int CG>
__global__ void __launch_bounds__(16 * CG) k_delta_step(DeltaArgs g) {
    constexpr int TB = 8, WAVES = 16 * CG / 64, RED = 8 * CG + 4;
    __shared__ alignas(16) float in[TB][2 * 256 + 4 * CG];  // k, q, v of tokens
    __shared__ alignas(16) float red[2][WAVES][RED];
    const int nv = g.st.n_v_heads, dk = g.st.k_dim, dv = g.st.v_dim;
    const HqSeq seq = g.seqs[g.steps[blockIdx.x / nv]];
    const int h = blockIdx.x % nv, hk = h / (nv / g.st.n_k_heads);
    const int tid = threadIdx.x, nt = blockDim.x, w = tid >> 6, lane = tid & 63, waves = nt >> 6;
    const int cg = tid % CG, rg = tid / CG;
    const bool col = 4 * cg < dv, on = col && 16 * rg < dk;
    f4 S[16];
    const size_t size = (size_t)dk * dv;
#pragma unroll
    for (int i = 0; i < 16; i++) S[i] = f4{0.f, 0.f, 0.f, 0.f};
    if (seq.from >= 0 && on) {
        const float *s = g.st.s + ((size_t)seq.from * nv + h) * size + (size_t)(16 * rg) * dv + 4 * cg;
#pragma unroll
        for (int i = 0; i < 16; i++) S[i] = *(const f4 *)(s + (size_t)i * dv);
    }
    int buf = 0;
    for (int t0 = 0; t0 < seq.n; t0 += TB) {
        const int m = min(TB, seq.n - t0), pieces = (2 * dk + dv) / 8;
        __syncthreads();
        for (int i = tid; i < m * pieces; i += nt) {
            const int t = i / pieces, e = 8 * (i - t * pieces);
            const size_t tok = (size_t)(seq.tok0 + t0 + t);
            const uint16_t *src = e < dk ? g.d.k + tok * g.d.qk_stride + hk * dk + e
                                  : e < 2 * dk ? g.d.q + tok * g.d.qk_stride + hk * dk + (e - dk)
                                               : g.d.v + tok * g.d.v_stride + h * dv + (e - 2 * dk);
            float *to = in[t] + (e < dk ? e : e < 2 * dk ? 256 + e - dk : 512 + e - 2 * dk);
            const h8 x = *(const h8 *)src;
#pragma unroll
            for (int j = 0; j < 8; j++) to[j] = (float)x[j];
        }
        __syncthreads();
        for (int t = 0; t < m; t++) {
            const size_t tok = (size_t)(seq.tok0 + t0 + t);
            const float keep = expf(g.d.decay[tok * nv + h]), beta = g.d.beta[tok * nv + h];
            f4 k[4], p = {0.f, 0.f, 0.f, 0.f}, r = p;
            float kq = 0.f;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                k[i] = f4{0.f, 0.f, 0.f, 0.f};
                f4 q = k[i];
                if (16 * rg < dk) k[i] = *(const f4 *)(in[t] + 16 * rg + 4 * i), q = *(const f4 *)(in[t] + 256 + 16 * rg + 4 * i);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const f4 s = S[4 * i + j];
#pragma unroll
                    for (int e = 0; e < 4; e++) p[e] = fmaf(s[e], k[i][j], p[e]), r[e] = fmaf(s[e], q[j], r[e]);
                    kq = fmaf(k[i][j], q[j], kq);
                }
            }
#pragma unroll
            for (int o = CG; o < 64; o *= 2) p = sum_over(p, o), r = sum_over(r, o), kq += __shfl_xor(kq, o, 64);
            if (lane < CG) {
                *(f4 *)(red[buf][w] + 4 * cg) = p;
                *(f4 *)(red[buf][w] + 4 * CG + 4 * cg) = r;
                if (cg == 0) red[buf][w][8 * CG] = kq;
            }
            __syncthreads();
            p = r = f4{0.f, 0.f, 0.f, 0.f}, kq = 0.f;
            for (int i = 0; i < waves; i++) {
                p += *(const f4 *)(red[buf][i] + 4 * cg);
                r += *(const f4 *)(red[buf][i] + 4 * CG + 4 * cg);
                kq += red[buf][i][8 * CG];
            }
            buf ^= 1;
            f4 u = {0.f, 0.f, 0.f, 0.f}, o = u;
            if (col) {
                const f4 v = *(const f4 *)(in[t] + 512 + 4 * cg);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    u[e] = beta * (v[e] - keep * p[e]);
                    o[e] = g.d.scale * (keep * r[e] + kq * u[e]);
                }
            }
            if (on) {
#pragma unroll
                for (int i = 0; i < 16; i++)
#pragma unroll
                    for (int e = 0; e < 4; e++) S[i][e] = fmaf(k[i / 4][i % 4], u[e], keep * S[i][e]);
            }
            if (rg == 0) {
                if (g.d.norm) {
                    float ss = col ? o[0] * o[0] + o[1] * o[1] + o[2] * o[2] + o[3] * o[3] : 0.f;
#pragma unroll
                    for (int i = CG / 2; i > 0; i >>= 1) ss += __shfl_xor(ss, i, 64);
                    const float inv = 1.0f / sqrtf(ss / (float)dv + g.d.eps);
                    if (col) {
                        const size_t at = tok * g.d.gate_stride + (size_t)h * dv + 4 * cg;
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const float z = g.d.gate_f32 ? ((const float *)g.d.gate)[at + e] : (float)((const _Float16 *)g.d.gate)[at + e];
                            o[e] = o[e] * inv * g.d.norm[4 * cg + e] * (z / (1.0f + expf(-z)));
                        }
                    }
                }
                if (col) *(h4 *)((_Float16 *)g.d.out + tok * g.d.out_stride + (size_t)h * dv + 4 * cg) = h4{(_Float16)o[0], (_Float16)o[1], (_Float16)o[2], (_Float16)o[3]};
            }
        }
    }
    if (seq.to >= 0 && on) {
        float *s = g.st.s + ((size_t)seq.to * nv + h) * size + (size_t)(16 * rg) * dv + 4 * cg;
#pragma unroll
        for (int i = 0; i < 16; i++) *(f4 *)(s + (size_t)i * dv) = S[i];
    }
}

}  // namespace

extern "C" int hq_delta(const hq_scan *c, const hq_state_t *st, const hq_delta_t *d, void *stream) {
    const char *const who = "hq_delta";
    if (!c || !st || !d) return hq_internal_fail("%s: null argument", who);
    if (!c->set) return hq_internal_fail("%s: no step is described (hq_scan_set)", who);
    if (hq_state_check(who, st, c)) return -1;
    if (c->n_steps == 0) return 0;
    if (!st->s || !aligned(st->s, 16)) return hq_internal_fail("%s: 16-byte aligned memory of the states is needed", who);
    if (c->n_tokens) {
        if (!d->q || !d->k || !d->v || !d->decay || !d->beta || !d->out) return hq_internal_fail("%s: null argument", who);
        if (!aligned(d->q, 16) || !aligned(d->k, 16) || !aligned(d->v, 16) || !aligned(d->out, 16)) return hq_internal_fail("%s: q, k, v and out must be 16-byte aligned", who);
        if (!aligned(d->decay, 4) || !aligned(d->beta, 4)) return hq_internal_fail("%s: decay and beta are misaligned", who);
        if (!d->norm != !d->gate) return hq_internal_fail("%s: norm without gate, or the other way round", who);
        if (d->norm && (!aligned(d->norm, 16) || !aligned(d->gate, 16))) return hq_internal_fail("%s: norm and gate must be 16-byte aligned", who);
        if (d->norm && !(d->eps >= 0.f)) return hq_internal_fail("%s: eps %g", who, (double)d->eps);
        const int64_t most = (int64_t)1 << 40;
        for (int64_t s : {d->qk_stride, d->v_stride, d->out_stride, d->norm ? d->gate_stride : 0})
            if (s < 0 || s > most || s % 8) return hq_internal_fail("%s: stride %lld (a multiple of 8)", who, (long long)s);
        if (!(fabsf(d->scale) <= 1e20f)) return hq_internal_fail("%s: scale %g", who, (double)d->scale);
    }
    int cur = -1;
    SCK(hipGetDevice(&cur));
    if (cur != c->device) SCK(hipSetDevice(c->device));
    const DeltaArgs g = {*st, *d, c->seqs, c->steps};
    const int rows = st->k_dim / 16;
    const unsigned grid = (unsigned)c->n_steps * (unsigned)st->n_v_heads;
    hipStream_t s = (hipStream_t)stream;
    const auto threads = [&](int cg) { return (unsigned)std::max(64, (cg * rows + 63) / 64 * 64); };
    if (st->v_dim <= 64) k_delta_step<16><<<grid, threads(16), 0, s>>>(g);
    else if (st->v_dim <= 128) k_delta_step<32><<<grid, threads(32), 0, s>>>(g);
    else k_delta_step<64><<<grid, threads(64), 0, s>>>(g);
    SCK(hipGetLastError());
    return 0;
}
