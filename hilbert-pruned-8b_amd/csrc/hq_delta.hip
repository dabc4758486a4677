// hq_delta.hip - the gated delta recurrence of a step's sequences (hq_delta, include/hq_serve.h).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <math.h>

#include "hq_device.h"
#include "hq_scan.h"

namespace {

bool aligned(const void *p, size_t a) { return ((uintptr_t)p % a) == 0; }

constexpr int64_t MOST_CHUNK_STRIDE = 1 << 22;  // 64 rows of it stay below 2^29 bytes

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

// ------------------------------------------------------------------------------------ by chunks
// Within a chunk of 64 tokens, with G the sums of the log decays, the recurrence is a triangular system:
//   (I + A) U = beta (V - e^G K S),  A_ij = beta_i e^(G_i - G_j) k_i k_j below the diagonal,
//   O = scale (e^G Q S + M U),  M_ij = e^(G_i - G_j) q_i k_j on and below it,
//   S' = e^G_64 S + (e^(G_64 - G) K)^T U,
// so that all that depends on the state is products of matrices, and T = (I + A)^-1 beta and M can be formed for all chunks at once.
// Differences of G are formed in 64 bits (a decay of 0 is a logarithm of -1e4, next to which small ones would drown); none of the
// exponentials exceeds 1. T's entries are at most 1 in magnitude where |k| <= 1 and 0 <= beta <= 1.
//
// Tokens and k_dim are numbered so that what one product leaves in the accumulators is the next one's operand as it stands. Rows 4 q +
// r of the accumulators of block b (b = 0 .. 3 of 16 tokens, lane group q) are token 32 (b / 2) + 8 q + r + 4 (b % 2): blocks 2 s
// and 2 s + 1 together hold, lane group by lane group, the 8 consecutive contraction indices that an operand takes. Tiles of S
// likewise.
//
// Precision: K, Q and V are exact. S, U and T enter products as two fp16 terms each, scaled by a power of two of their column's largest
// (T: of the matrix), good to 2^-22 of it; only for the outputs, which end in fp16, one term of S, M and U does.
constexpr int FRAG_T = 0, FRAG_T_LO = 6, FRAG_M = 12, FRAG_VEC = 18;  // of a chunk's workspace, in KB; fragments (block, half) in the order below
constexpr float T_SCALE = 4096.f;
DEV int frag_of(int b, int s) { return b < 2 ? b : 2 * b - 2 + s; }
DEV int token_of(int b, int row) { return 32 * (b >> 1) + 8 * (row >> 2) + (row & 3) + 4 * (b & 1); }
// A row's 16-byte pieces lie in LDS in an order of the row's own, so that 16 rows' pieces of one column fall into different banks.
template <int CPR>
DEV int piece_at(int row, int c) {
    const int key = CPR >= 16 ? (row & 3) | ((row >> 1) & 12) : ((row >> 1) & 1) | ((row >> 2) & 6);
    return row * CPR + (c ^ key);
}

DEV float pow2(uint32_t e) { return __builtin_bit_cast(float, e << 23); }
// The exponent that takes a largest magnitude to 2^14 .. 2^15 by pow2(268 - e), and back by pow2(e - 14)
DEV uint32_t exponent(float largest) {
    const uint32_t e = __builtin_bit_cast(uint32_t, largest) >> 23;
    return e < 15u ? 15u : e > 253u ? 253u : e;
}

struct ChunkArgs {
    hq_state_t st;
    hq_delta_t d;
    const HqChunk *chunks;
    const HqRun *runs;
    int n_runs;
    char *work;
    float *carry;
};

// T and M of a chunk's value heads; a workgroup takes those of one key head. Wave w forms rows 16 w .. of K K^T and Q K^T, then inverts
// the 16 x 16 block (w, w) of I + A by substitution, a column a lane, and last computes block column w of the inverse from the top
// down, T_ij = -T_ii sum_l A_il T_lj, on the fp32 matrix cores: each block of the column is the next one's operand.
template <int KS>
__global__ void __launch_bounds__(256) k_delta_prep(ChunkArgs g) {
    constexpr int CPR = 4 * KS < 8 ? 8 : 4 * KS, LD = 72, LA = 68, LT = 20;
    __shared__ union {
        u4v kq[2][64 * CPR];
        _Float16 f[3][64 * LD];  // T, its second term, M
    } sh;
    __shared__ alignas(16) float At[64 * LA];  // A transposed
    __shared__ alignas(16) float Td[4][16 * LT];
    __shared__ double gam[4][64];
    __shared__ float bet[4][64], ms[64];
    const int nk = g.st.n_k_heads, nv = g.st.n_v_heads, dk = g.st.k_dim;
    const int at = blockIdx.x / nk, hk = blockIdx.x % nk, rep = nv / nk;
    const HqChunk ch = g.chunks[at];
    const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63, n = lane & 15, q = lane >> 4;
    for (int i = tid; i < 2 * 64 * CPR; i += 256) {
        const int which = i / (64 * CPR), row = (i / CPR) % 64, c = i % CPR;
        u4v x = {0, 0, 0, 0};
        if (row < ch.n && 8 * c < dk) x = *(const u4v *)((which ? g.d.q : g.d.k) + (size_t)(ch.tok0 + row) * g.d.qk_stride + hk * dk + 8 * c);
        sh.kq[which][piece_at<CPR>(row, c)] = x;
    }
    __syncthreads();
    f4 G[4], H[4];
#pragma unroll
    for (int b = 0; b < 4; b++) {
        G[b] = H[b] = f4{0.f, 0.f, 0.f, 0.f};
        if (b > w) continue;
#pragma unroll
        for (int s = 0; s < KS; s++) {
            const h8 x = __builtin_bit_cast(h8, sh.kq[0][piece_at<CPR>(16 * b + n, 4 * s + q)]);
            G[b] = mfma(__builtin_bit_cast(h8, sh.kq[0][piece_at<CPR>(16 * w + n, 4 * s + q)]), x, G[b]);
            H[b] = mfma(__builtin_bit_cast(h8, sh.kq[1][piece_at<CPR>(16 * w + n, 4 * s + q)]), x, H[b]);
        }
    }
    for (int e = 0; e < rep; e++) {
        const int h = hk * rep + e;
        const float gl = lane < ch.n ? g.d.decay[(size_t)(ch.tok0 + lane) * nv + h] : 0.f;
        double sum = (double)(gl < -1e4f ? -1e4f : gl);
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const double y = __shfl_up(sum, o, 64);
            if (lane >= o) sum += y;
        }
        gam[w][lane] = sum;
        bet[w][lane] = lane < ch.n ? g.d.beta[(size_t)(ch.tok0 + lane) * nv + h] : 0.f;
        __syncthreads();  // (the last head's reads of At are done as well)
        f4 M[4];
        float mx[4] = {0.f, 0.f, 0.f, 0.f};
        const int i0 = 16 * w + 4 * q;
#pragma unroll
        for (int b = 0; b < 4; b++) {
            M[b] = f4{0.f, 0.f, 0.f, 0.f};
            if (b > w) continue;
            const int j = 16 * b + n;
            f4 a;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const float x = j <= i0 + r ? expf((float)(gam[w][i0 + r] - gam[w][j])) : 0.f;
                a[r] = j < i0 + r ? bet[w][i0 + r] * x * G[b][r] : 0.f;
                M[b][r] = j <= i0 + r ? x * H[b][r] : 0.f;
                mx[r] = fmaxf(mx[r], fabsf(M[b][r]));
            }
            *(f4 *)(At + j * LA + i0) = a;
        }
#pragma unroll
        for (int r = 0; r < 4; r++) {
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) mx[r] = fmaxf(mx[r], __shfl_xor(mx[r], o, 64));
            const uint32_t ex = exponent(mx[r]);
            if (n == 0) ms[i0 + r] = pow2(ex - 14u);
#pragma unroll
            for (int b = 0; b < 4; b++) M[b][r] *= pow2(268u - ex);
        }
        __syncthreads();
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; i++) x[i] = i == n ? 1.f : 0.f;
#pragma unroll
        for (int j = 0; j < 15; j++)
#pragma unroll
            for (int i4 = (j + 1) / 4; i4 < 4; i4++) {
                const f4 a = *(const f4 *)(At + (16 * w + j) * LA + 16 * w + 4 * i4);
#pragma unroll
                for (int r = 0; r < 4; r++)
                    if (4 * i4 + r > j) x[4 * i4 + r] = fmaf(-a[r], x[j], x[4 * i4 + r]);
            }
#pragma unroll
        for (int i = 0; i < 16; i++)
            if (i / 4 == q) Td[w][i * LT + n] = x[i];
        __syncthreads();
        f4 T[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            T[i] = f4{0.f, 0.f, 0.f, 0.f};
            if (i < w) continue;
            if (i == w) {
#pragma unroll
                for (int r = 0; r < 4; r++) T[i][r] = Td[w][(4 * q + r) * LT + n];
                continue;
            }
            f4 y = {0.f, 0.f, 0.f, 0.f}, z = y;
#pragma unroll
            for (int l = 0; l < i; l++)
                if (l >= w) {
#pragma unroll
                    for (int r = 0; r < 4; r++) y = __builtin_amdgcn_mfma_f32_16x16x4f32(At[(16 * l + 4 * q + r) * LA + 16 * i + n], T[l][r], y, 0, 0, 0);
                }
            const f4 t = *(const f4 *)(Td[i] + n * LT + 4 * q);
#pragma unroll
            for (int r = 0; r < 4; r++) z = __builtin_amdgcn_mfma_f32_16x16x4f32(t[r], y[r], z, 0, 0, 0);
            T[i] = -z;
        }
        const float scale = T_SCALE * bet[w][16 * w + n];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (i < (w & ~1)) continue;  // (above the diagonal: the half of a fragment that is zero)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const float v = T[i][r] * scale;
                const _Float16 hi = (_Float16)v;
                const int o = (16 * i + 4 * q + r) * LD + 16 * w + n;
                sh.f[0][o] = hi;
                sh.f[1][o] = (_Float16)(v - (float)hi);
            }
        }
#pragma unroll
        for (int b = 0; b < 4; b++) {
            if (b > (w | 1)) continue;
#pragma unroll
            for (int r = 0; r < 4; r++) sh.f[2][(i0 + r) * LD + 16 * b + n] = (_Float16)M[b][r];
        }
        __syncthreads();
        char *const to = g.work + ((size_t)at * nv + h) * HQ_CHUNK_BYTES;
        for (int p = w; p < 18; p += 4) {
            const int k = p % 6, b = k < 2 ? k : k / 2 + 1, s = k < 2 ? 0 : k & 1;
            *(u4v *)(to + p * 1024 + lane * 16) = *(const u4v *)(sh.f[p / 6] + token_of(b, n) * LD + 32 * s + 8 * q);
        }
        if (w == 3) {
            float *const v = (float *)(to + FRAG_VEC * 1024);
            v[lane] = expf((float)gam[3][lane]);
            v[64 + lane] = expf((float)(gam[3][63] - gam[3][lane]));
            v[128 + lane] = ms[lane];
            v[192 + lane] = expf((float)gam[3][63]);
        }
    }
}

typedef short s4v __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4v lds_s4v;

// Two fp16 terms of 8 values scaled by sc: accumulator blocks a and b as an operand
DEV void two_terms(const f4 &a, const f4 &b, float sc, h8 &hi, h8 &lo) {
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const float x = (j < 4 ? a[j & 3] : b[j & 3]) * sc;
        hi[j] = (_Float16)x;
        lo[j] = (_Float16)(x - (float)hi[j]);
    }
}
template <int N>
DEV float column_max(const f4 (&x)[N]) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < N; i++) m = fmaxf(fmaxf(fmaxf(fabsf(x[i][0]), fabsf(x[i][1])), fmaxf(fabsf(x[i][2]), fabsf(x[i][3]))), m);
    m = fmaxf(m, __shfl_xor(m, 16, 64));
    return fmaxf(m, __shfl_xor(m, 32, 64));
}

// The chunks of a run in order; a wave holds S for 16 of a head's value columns and needs no other wave's results. All waves of a
// workgroup (W of them with columns, four at least) bring the next chunk's keys, queries, T and M to LDS by DMA meanwhile.
template <int KS, int W>
__global__ void __launch_bounds__(64 * (W < 4 ? 4 : W)) k_delta_scan(ChunkArgs g) {
    constexpr int CPR = 4 * KS < 8 ? 8 : 4 * KS, NW = W < 4 ? 4 : W;
    constexpr int KB = CPR;  // of a chunk's keys: 64 rows of CPR pieces of 16 bytes
    constexpr int BUFS = KS <= 6 ? 2 : 1;  // (two chunks of wider keys do not fit: the next one's wait until this one is done)
    __shared__ alignas(1024) char buf[BUFS][(2 * KB + 19) * 1024];
    const int nk = g.st.n_k_heads, nv = g.st.n_v_heads, dk = g.st.k_dim, dv = g.st.v_dim;
    const int groups = (dv + 16 * W - 1) / (16 * W);
    // workgroup i runs on XCD i % 8: the groups of one head on one, where they share its keys
    const int head = blockIdx.x / (8 * groups) * 8 + blockIdx.x % 8, group = blockIdx.x / 8 % groups;
    if (head >= g.n_runs * nv) return;
    const HqRun run = g.runs[head / nv];
    const int h = head % nv, hk = h / (nv / nk);
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, n = lane & 15, q = lane >> 4;
    const int col = 16 * (group * W + w) + n;
    const bool on = w < W && 16 * (group * W + w) < dv;  // (of a wave as a whole)
    const uint32_t NOWHERE = 0x80000000u;  // past every range: loads give zeros, stores nothing
    const size_t size = (size_t)dk * dv;
    f4 S[2 * KS];
#pragma unroll
    for (int t = 0; t < 2 * KS; t++) S[t] = f4{0.f, 0.f, 0.f, 0.f};
    if (on && run.from != -1) {
        const float *s = (run.from >= 0 ? g.st.s + ((size_t)run.from * nv + h) * size : g.carry + ((size_t)(-2 - run.from) * nv + h) * size) + col;
#pragma unroll
        for (int t = 0; t < 2 * KS; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int d = 32 * (t >> 1) + 8 * q + r + 4 * (t & 1);
                if (d < dk) S[t][r] = s[(size_t)d * dv];
            }
    }
    const int chunks = (run.n + HQ_CHUNK - 1) / HQ_CHUNK;
    const uint32_t row_bytes = (uint32_t)g.d.qk_stride * 2u;
    const auto load = [&](int c) {
        const int rows = min(HQ_CHUNK, run.n - c * HQ_CHUNK);
        const size_t tok = (size_t)(run.tok0 + c * HQ_CHUNK);
        const uint32_t range = (uint32_t)(rows - 1) * row_bytes + (uint32_t)dk * 2u;
        const rsrc_t rk = make_rsrc(g.d.k + tok * g.d.qk_stride + hk * dk, range), rq = make_rsrc(g.d.q + tok * g.d.qk_stride + hk * dk, range);
        const rsrc_t rw = make_rsrc(g.work + ((size_t)(run.chunk0 + c) * nv + h) * HQ_CHUNK_BYTES, (uint32_t)HQ_CHUNK_BYTES);
        const uint32_t to = (uint32_t)(uintptr_t)buf[c % BUFS];
#pragma unroll
        for (int i0 = 0; i0 < KB; i0 += NW) {
            const int i = i0 + w, slot = 64 * i + lane, row = slot / CPR, x = piece_at<CPR>(row, slot % CPR) - row * CPR;  // (its own inverse)
            if (KB % NW && i >= KB) break;
            const uint32_t off = row < rows && 8 * x < dk ? (uint32_t)row * row_bytes + 16u * (uint32_t)x : NOWHERE;
            dma16_untracked(rk, to + 1024u * (uint32_t)i, off);
            dma16_untracked(rq, to + 1024u * (uint32_t)(KB + i), off);
        }
        for (int i = w; i < 19; i += NW) dma16_untracked(rw, to + 1024u * (uint32_t)(2 * KB + i), 1024u * (uint32_t)i + 16u * (uint32_t)lane);
    };
    const uint32_t v_bytes = (uint32_t)g.d.v_stride * 2u, o_bytes = (uint32_t)g.d.out_stride * 2u;
    _Float16 V[16];
    const auto load_v = [&](int c) {
        const int rows = min(HQ_CHUNK, run.n - c * HQ_CHUNK);
        const rsrc_t rv = make_rsrc(g.d.v + (size_t)(run.tok0 + c * HQ_CHUNK) * g.d.v_stride + (size_t)h * dv, (uint32_t)(rows - 1) * v_bytes + (uint32_t)dv * 2u);
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const int row = token_of(i >> 2, 4 * q + (i & 3));
            V[i] = __builtin_bit_cast(_Float16, __builtin_amdgcn_raw_buffer_load_b16(rv, row < rows ? (uint32_t)row * v_bytes + 2u * (uint32_t)col : NOWHERE, 0u, 0));
        }
    };
    if (BUFS == 2) load(0);
    if (on) load_v(0);
    for (int c = 0; c < chunks; c++) {
        if (BUFS == 1) {
            __syncthreads();
            load(c);
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (BUFS == 2 && c + 1 < chunks) load(c + 1);
        if (!on) continue;
        const char *const b0 = buf[c % BUFS];
        const u4v *const K = (const u4v *)b0, *const Q = K + 64 * KB, *const F = K + 128 * KB;
        const float *const vec = (const float *)(F + 64 * FRAG_VEC);
        const auto frag = [&](int i) { return __builtin_bit_cast(h8, F[64 * i + lane]); };
        const int rows = min(HQ_CHUNK, run.n - c * HQ_CHUNK);
        const uint32_t es = exponent(column_max(S));
        h8 Sh[KS], Sl[KS];
#pragma unroll
        for (int s = 0; s < KS; s++) two_terms(S[2 * s], S[2 * s + 1], pow2(268u - es), Sh[s], Sl[s]);
        const float back = pow2(es - 14u);
        f4 X[4], O[4];
#pragma unroll
        for (int b = 0; b < 4; b++) {
            const int row = token_of(b, n);
            f4 p = {0.f, 0.f, 0.f, 0.f}, o = p;
#pragma unroll
            for (int s = 0; s < KS; s++) {
                const h8 k = __builtin_bit_cast(h8, K[piece_at<CPR>(row, 4 * s + q)]);
                p = mfma(k, Sh[s], p);
                p = mfma(k, Sl[s], p);
                o = mfma(__builtin_bit_cast(h8, Q[piece_at<CPR>(row, 4 * s + q)]), Sh[s], o);
            }
            const f4 eg = *(const f4 *)(vec + token_of(b, 4 * q)) * back;
#pragma unroll
            for (int r = 0; r < 4; r++) X[b][r] = (float)V[4 * b + r] - eg[r] * p[r];
            O[b] = eg * o;
        }
        if (c + 1 < chunks) load_v(c + 1);
        const uint32_t ex = exponent(column_max(X));
        h8 Xh[2], Xl[2];
        two_terms(X[0], X[1], pow2(268u - ex), Xh[0], Xl[0]);
        two_terms(X[2], X[3], pow2(268u - ex), Xh[1], Xl[1]);
        f4 U[4];
#pragma unroll
        for (int b = 0; b < 4; b++) {
            f4 u = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s <= b / 2; s++) {
                const h8 t = frag(FRAG_T + frag_of(b, s)), tl = frag(FRAG_T_LO + frag_of(b, s));
                u = mfma(tl, Xh[s], u);
                u = mfma(t, Xl[s], u);
                u = mfma(t, Xh[s], u);
            }
            U[b] = u * (pow2(ex - 14u) / T_SCALE);
        }
        const uint32_t eu = exponent(column_max(U));
        const float su = pow2(268u - eu), bu = pow2(eu - 14u);
        h8 Uh[2], Dh[2], Dl[2];
#pragma unroll
        for (int s = 0; s < 2; s++) {
            h8 unused;
            two_terms(U[2 * s], U[2 * s + 1], su, Uh[s], unused);
            two_terms(U[2 * s] * *(const f4 *)(vec + 64 + token_of(2 * s, 4 * q)), U[2 * s + 1] * *(const f4 *)(vec + 64 + token_of(2 * s + 1, 4 * q)), su, Dh[s], Dl[s]);
        }
        const rsrc_t ro = make_rsrc(g.d.out + (size_t)(run.tok0 + c * HQ_CHUNK) * g.d.out_stride + (size_t)h * dv, (uint32_t)(rows - 1) * o_bytes + (uint32_t)dv * 2u);
#pragma unroll
        for (int b = 0; b < 4; b++) {
            f4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s <= b / 2; s++) o = mfma(frag(FRAG_M + frag_of(b, s)), Uh[s], o);
            const f4 m = *(const f4 *)(vec + 128 + token_of(b, 4 * q)) * bu;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int row = token_of(b, 4 * q + r);
                const _Float16 y = (_Float16)(g.d.scale * fmaf(m[r], o[r], O[b][r]));
                __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(short, y), ro, row < rows ? (uint32_t)row * o_bytes + 2u * (uint32_t)col : NOWHERE, 0u, 0);
            }
        }
        const float keep = vec[192];
        const uint32_t k0 = (uint32_t)(uintptr_t)b0;
#pragma unroll
        for (int t = 0; t < 2 * KS; t++) {
            f4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < 2; s++) {
                // lane i of a group of 16 hands over 4 values of k_dim of row i / 4, and gets one of k_dim of 4 rows
                s4v x[2];
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int row = 32 * s + 8 * q + (n >> 2) + 4 * e;
                    x[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4v *)(uintptr_t)(k0 + 16u * (uint32_t)piece_at<CPR>(row, 4 * (t >> 1) + (n & 3)) + 8u * (uint32_t)(t & 1)));
                }
                const h8 k = __builtin_bit_cast(h8, __builtin_shufflevector(x[0], x[1], 0, 1, 2, 3, 4, 5, 6, 7));
                a = mfma(k, Dl[s], a);
                a = mfma(k, Dh[s], a);
            }
#pragma unroll
            for (int r = 0; r < 4; r++) S[t][r] = fmaf(bu, a[r], keep * S[t][r]);
        }
    }
    if (on && run.to != -1) {
        float *s = (run.to >= 0 ? g.st.s + ((size_t)run.to * nv + h) * size : g.carry + ((size_t)(-2 - run.to) * nv + h) * size) + col;
#pragma unroll
        for (int t = 0; t < 2 * KS; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int d = 32 * (t >> 1) + 8 * q + r + 4 * (t & 1);
                if (d < dk) s[(size_t)d * dv] = S[t][r];
            }
    }
}

// The outputs' norm and gate of chunks, in place: G lanes a head, eight columns a lane. (The outputs have been rounded to fp16 by
// then, 2^-11 of each beside the rounding of the result.)
template <int G>
__global__ void __launch_bounds__(256) k_delta_norm(ChunkArgs g) {
    const int nv = g.st.n_v_heads, dv = g.st.v_dim, u = threadIdx.x % G;
    const HqChunk ch = g.chunks[blockIdx.x];
    for (int i = blockIdx.y * (256 / G) + threadIdx.x / G; i < ch.n * nv; i += gridDim.y * (256 / G)) {
        const int t = i / nv, h = i - t * nv;
        const bool on = 8 * u < dv;
        const size_t tok = (size_t)(ch.tok0 + t), in = (size_t)h * dv + (on ? 8 * u : 0);
        _Float16 *const at = (_Float16 *)g.d.out + tok * g.d.out_stride + in;
        const h8 x = *(const h8 *)at;
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; e++) ss = fmaf((float)x[e], (float)x[e], ss);
        if (!on) ss = 0.f;
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1) ss += __shfl_xor(ss, o, 64);
        const float inv = 1.0f / sqrtf(ss / (float)dv + g.d.eps);
        const size_t zat = tok * g.d.gate_stride + in;
        h8 y;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float z = g.d.gate_f32 ? ((const float *)g.d.gate)[zat + e] : (float)((const _Float16 *)g.d.gate)[zat + e];
            y[e] = (_Float16)((float)x[e] * inv * g.d.norm[(on ? 8 * u : 0) + e] * (z / (1.0f + expf(-z))));
        }
        if (on) *(h8 *)at = y;
    }
}

template <int KS>
void launch_chunks(const ChunkArgs &g, int n_chunks, hipStream_t s) {
    k_delta_prep<KS><<<(unsigned)n_chunks * (unsigned)g.st.n_k_heads, 256, 0, s>>>(g);
    const unsigned heads = ((unsigned)g.n_runs * (unsigned)g.st.n_v_heads + 7) / 8 * 8;
    const auto grid = [&](int W) { return heads * (unsigned)((g.st.v_dim + 16 * W - 1) / (16 * W)); };
    k_delta_scan<KS, 4><<<grid(4), 256, 0, s>>>(g);
}

}  // namespace

extern "C" int hq_delta(const hq_scan *c, const hq_state_t *st, const hq_delta_t *d, void *stream) {
    const char *const who = "hq_delta";
    if (!c || !st || !d) return hq_internal_fail("%s: null argument", who);
    if (!c->set) return hq_internal_fail("%s: no step is described (hq_scan_set)", who);
    if (hq_state_check(who, st, c)) return -1;
    if (c->n_steps == 0 && c->passes.empty()) return 0;
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
        // a chunk's rows are addressed by 32 bits
        if (!c->passes.empty())
            for (int64_t s : {d->qk_stride, d->v_stride, d->out_stride})
                if (s > MOST_CHUNK_STRIDE) return hq_internal_fail("%s: stride %lld (with more than %d new tokens of a sequence at most %lld)", who, (long long)s, HQ_STEP_TOKENS, (long long)MOST_CHUNK_STRIDE);
        if (!(fabsf(d->scale) <= 1e20f)) return hq_internal_fail("%s: scale %g", who, (double)d->scale);
    }
    int cur = -1;
    SCK(hipGetDevice(&cur));
    if (cur != c->device) SCK(hipSetDevice(c->device));
    hipStream_t s = (hipStream_t)stream;
    for (const HqPass &p : c->passes) {
        const ChunkArgs g = {*st, *d, c->chunks + p.chunk0, c->runs + p.run0, p.n_runs, c->work, (float *)(c->work + c->carry_at)};
        if (st->k_dim <= 64) launch_chunks<2>(g, p.n_chunks, s);
        else if (st->k_dim <= 128) launch_chunks<4>(g, p.n_chunks, s);
        else launch_chunks<8>(g, p.n_chunks, s);
        if (d->norm) {
            const int lanes = st->v_dim <= 64 ? 8 : st->v_dim <= 128 ? 16 : 32;
            const dim3 grid((unsigned)p.n_chunks, (unsigned)std::max(1, std::min(32, HQ_CHUNK * st->n_v_heads * lanes / 1024)));
            if (lanes == 8) k_delta_norm<8><<<grid, 256, 0, s>>>(g);
            else if (lanes == 16) k_delta_norm<16><<<grid, 256, 0, s>>>(g);
            else k_delta_norm<32><<<grid, 256, 0, s>>>(g);
        }
        SCK(hipGetLastError());
    }
    if (c->n_steps == 0) return 0;
    const DeltaArgs g = {*st, *d, c->seqs, c->steps};
    const int rows = st->k_dim / 16;
    const unsigned grid = (unsigned)c->n_steps * (unsigned)st->n_v_heads;
    const auto threads = [&](int cg) { return (unsigned)std::max(64, (cg * rows + 63) / 64 * 64); };
    if (st->v_dim <= 64) k_delta_step<16><<<grid, threads(16), 0, s>>>(g);
    else if (st->v_dim <= 128) k_delta_step<32><<<grid, threads(32), 0, s>>>(g);
    else k_delta_step<64><<<grid, threads(64), 0, s>>>(g);
    SCK(hipGetLastError());
    return 0;
}
