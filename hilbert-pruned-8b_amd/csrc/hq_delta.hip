// hq_delta.hip - the gated delta recurrence of a step's sequences (hq_delta, include/hq_serve.h).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <math.h>

#include "hq_device.h"
#include "hq_scan.h"

namespace {

bool aligned(const void *p, size_t a) { return ((uintptr_t)p % a) == 0; }

constexpr int64_t MOST_CHUNK_STRIDE = 1 << 22;  // 64 rows of it stay below 2^29 bytes

// z / (1 + e^-z) with the hardware's exponential and reciprocal (2^-22 of the result together; -inf gives NaN, as the formula)
DEV float silu(float z) { return z * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.4426950408889634f)); }

// x 2^e / sqrt(mean (x 2^e)^2 + eps) of a head's dv values, N of them in each of G neighbouring lanes (zeros behind dv). e is that of the
// scale, which outputs ahead of their norm are formed without, as it goes up to 1e20 and the norm takes it out again. The squares of values that
// are far from 1 leave fp32's range all the same: where their mean is not well inside it, of values over a power of two of the largest.
// (eps 2^-2e comes from the host: formed here it cost k_delta_step registers, 64 single tokens 56.4 us in place of 54.8)
struct Eps {
    float eps, unit;  // unit: eps 2^-2e
    int e;
};
template <int N, int G>
DEV void normalise(float (&x)[N], int dv, const Eps &at) {
    const auto mean = [&](float eps) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < N; i++) ss = fmaf(x[i], x[i], ss);
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1) ss += __shfl_xor(ss, o, 64);
        return ss / (float)dv + eps;
    };
    float ms = mean(at.unit);
    if (!(ms > 1e-30f && ms < INFINITY)) {  // (all of a head's lanes, or none)
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < N; i++) m = max(m, __builtin_bit_cast(uint32_t, fabsf(x[i])));  // (magnitudes: their order as integers)
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o, 64));
        const int to_1 = min(max(127 - (int)(m >> 23), -126), 126);
#pragma unroll
        for (int i = 0; i < N; i++) x[i] = ldexpf(x[i], to_1);
        ms = mean(ldexpf(at.eps, 2 * (to_1 - at.e)));
    }
    const float inv = 1.0f / sqrtf(ms);
#pragma unroll
    for (int i = 0; i < N; i++) x[i] *= inv;
}

struct DeltaArgs {
    hq_state_t st;
    hq_delta_t d;
    const HqSeq *seqs;
    const int *steps;
    Eps eps;  // with a norm: e is the scale's exponent, whose rest d.scale is
};

// The sum of x over the lane groups of eight: all lanes have it. (Elements are bit-cast from plain scalars.)
DEV float sum_groups(float x) {
    const uint32_t v = __builtin_bit_cast(uint32_t, x);
    const auto a = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    const uint32_t a0 = a[0], a1 = a[1];
    const float y = __builtin_bit_cast(float, a0) + __builtin_bit_cast(float, a1);
    const uint32_t w = __builtin_bit_cast(uint32_t, y);
    const auto b = __builtin_amdgcn_permlane16_swap(w, w, false, false);
    const uint32_t b0 = b[0], b1 = b[1];
    const float z = __builtin_bit_cast(float, b0) + __builtin_bit_cast(float, b1);
    return z + __shfl_xor(z, 8, 64);
}

// Token by token. A wave holds 32 columns of a head's S in registers, a lane four of them and an eighth of the rows: no wave waits for
// another within a token. With p = S^T k and r = S^T q of the state before the token, formed together:
//   u = beta (v - e^g p),  o = scale (e^g r + (k q) u),  S' = e^g S + k u.
// What tokens bring besides lies in LDS for eight of them; the outputs' norm, for which a head's waves meet, follows for eight together.
// Bound: the bytes of the states. 64 sequences of one token, 32 heads of 128: 268 MB in 53 us; more tokens: some 330 instructions each.
// FULL: dk = 8 ROWS (less otherwise).
template <int ROWS, bool FULL>
__global__ void __launch_bounds__(512, ROWS <= 16 ? 4 : 2) k_delta_step(DeltaArgs g) {
    constexpr int TB = 8;
    __shared__ alignas(16) _Float16 in[TB][2][8 * ROWS];  // k and q, each lane group's rows in ROWS places
    __shared__ alignas(16) _Float16 in_v[TB][256];
    __shared__ alignas(16) float z[TB][256], o[TB][256];  // gates and outputs
    __shared__ float keep[TB], beta[TB];
    const int nv = g.st.n_v_heads, dk = g.st.k_dim, dv = g.st.v_dim, rows = FULL ? ROWS : dk / 8;
    const HqSeq seq = g.seqs[g.steps[blockIdx.x / nv]];
    const int h = blockIdx.x % nv, hk = h / (nv / g.st.n_k_heads);
    const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 63, cl = lane & 7, rg = lane >> 3;
    const int col = 32 * (int)(blockIdx.y * (nt >> 6) + (tid >> 6)) + 4 * cl;
    const bool on = col < dv;
    const size_t size = (size_t)dk * dv, at = (size_t)(rg * rows) * dv + col;
    f4 S[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; i++) S[i] = f4{0.f, 0.f, 0.f, 0.f};
    if (seq.from >= 0 && on) {
        const float *s = g.st.s + ((size_t)seq.from * nv + h) * size + at;
#pragma unroll
        for (int i = 0; i < ROWS; i++)
            if (i < rows) S[i] = *(const f4 *)(s + (size_t)i * dv);
    }
    for (int t0 = 0; t0 < seq.n; t0 += TB) {
        const int m = min(TB, seq.n - t0), pk = dk / 8, pv = dv / 8;
        const size_t tok0 = (size_t)(seq.tok0 + t0);
        __syncthreads();
        // pieces of eight values: k and q, v, gates
        for (int i = tid; i < m * (2 * pk + 2 * pv); i += nt) {
            const int t = i / (2 * pk + 2 * pv), e = i - t * (2 * pk + 2 * pv);
            const size_t tok = tok0 + t;
            if (e < 2 * pk) {
                const int which = e >= pk, d = 8 * (e - which * pk);
                const h8 x = *(const h8 *)((which ? g.d.q : g.d.k) + tok * g.d.qk_stride + hk * dk + d);
                if (FULL) *(h8 *)(in[t][which] + d) = x;
                else
#pragma unroll
                    for (int j = 0; j < 8; j++) in[t][which][(d + j) / rows * ROWS + (d + j) % rows] = x[j];
            } else if (e < 2 * pk + pv) {
                const int d = 8 * (e - 2 * pk);
                *(h8 *)(in_v[t] + d) = *(const h8 *)(g.d.v + tok * g.d.v_stride + h * dv + d);
            } else if (g.d.norm) {
                const int d = 8 * (e - 2 * pk - pv);
                const size_t from = tok * g.d.gate_stride + (size_t)h * dv + d;
                if (g.d.gate_f32) *(f4 *)(z[t] + d) = *(const f4 *)((const float *)g.d.gate + from), *(f4 *)(z[t] + d + 4) = *(const f4 *)((const float *)g.d.gate + from + 4);
                else {
                    const h8 x = *(const h8 *)((const _Float16 *)g.d.gate + from);
#pragma unroll
                    for (int j = 0; j < 8; j++) z[t][d + j] = (float)x[j];
                }
            }
        }
        if (tid < m) keep[tid] = expf(g.d.decay[(tok0 + tid) * nv + h]), beta[tid] = g.d.beta[(tok0 + tid) * nv + h];
        __syncthreads();
        for (int t = 0; t < m; t++) {
            const float kp = keep[t], bt = beta[t];
            h8 k[ROWS / 8];
            f4 p = {0.f, 0.f, 0.f, 0.f}, r = p;
            float kq = 0.f;
#pragma unroll
            for (int i = 0; i < ROWS / 8; i++) {
                k[i] = *(const h8 *)(in[t][0] + rg * ROWS + 8 * i);
                const h8 q = *(const h8 *)(in[t][1] + rg * ROWS + 8 * i);
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int row = 8 * i + j;
                    if (row >= rows) continue;  // (places behind the rows hold anything)
                    const float a = (float)k[i][j], b = (float)q[j];
#pragma unroll
                    for (int e = 0; e < 4; e++) p[e] = fmaf(S[row][e], a, p[e]), r[e] = fmaf(S[row][e], b, r[e]);
                    kq = fmaf(a, b, kq);
                }
            }
#pragma unroll
            for (int e = 0; e < 4; e++) p[e] = sum_groups(p[e]), r[e] = sum_groups(r[e]);
            kq = sum_groups(kq);
            f4 u = {0.f, 0.f, 0.f, 0.f}, y = u;
            if (on) {
                const h4 v = *(const h4 *)(in_v[t] + col);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    u[e] = bt * ((float)v[e] - kp * p[e]);
                    y[e] = g.d.scale * (kp * r[e] + kq * u[e]);
                }
            }
#pragma unroll
            for (int i = 0; i < ROWS; i++)
                if (i < rows) {
                    const float a = (float)k[i / 8][i % 8];
#pragma unroll
                    for (int e = 0; e < 4; e++) S[i][e] = fmaf(a, u[e], kp * S[i][e]);
                }
            if (rg == 0 && on) {
                if (g.d.norm) *(f4 *)(o[t] + col) = y;
                else *(h4 *)((_Float16 *)g.d.out + (tok0 + t) * g.d.out_stride + (size_t)h * dv + col) = h4{(_Float16)y[0], (_Float16)y[1], (_Float16)y[2], (_Float16)y[3]};
            }
        }
        if (!g.d.norm) continue;
        // a wave a token
        __syncthreads();
        for (int t = tid >> 6; t < m; t += nt >> 6) {
            const int d = 4 * lane;
            f4 at = {0.f, 0.f, 0.f, 0.f};
            if (d < dv) at = *(const f4 *)(o[t] + d);
            float y[4] = {at[0], at[1], at[2], at[3]};
            normalise<4, 64>(y, dv, g.eps);
            if (d >= dv) continue;
            const f4 zz = *(const f4 *)(z[t] + d), nw = *(const f4 *)(g.d.norm + d);
            h4 w;
#pragma unroll
            for (int e = 0; e < 4; e++) w[e] = (_Float16)(y[e] * nw[e] * silu(zz[e]));
            *(h4 *)((_Float16 *)g.d.out + (tok0 + t) * g.d.out_stride + (size_t)h * dv + d) = w;
        }
    }
    if (seq.to >= 0 && on) {
        float *s = g.st.s + ((size_t)seq.to * nv + h) * size + at;
#pragma unroll
        for (int i = 0; i < ROWS; i++)
            if (i < rows) *(f4 *)(s + (size_t)i * dv) = S[i];
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
// Precision: K, Q and V are exact. S, U, T and M enter products as two fp16 terms each, scaled by a power of two of their column's largest
// (T and M: of the matrix; T's is the largest beta, which stands on its diagonal), good to 2^-22 of it. (One term of S, M and U for the outputs, which end in fp16, made them 1.6 to 1.8 times
// as inexact as their own rounding does.)
constexpr int FRAG_T = 0, FRAG_T_LO = 6, FRAG_M = 12, FRAG_M_LO = 18, FRAG_VEC = 24;  // of a chunk's workspace, in KB; fragments (block, half) in the order below
constexpr int T_EXP = 265;  // T's largest entry has an exponent e, and is held as pow2(T_EXP - e) times it, 2^11 .. 2^12
DEV int frag_of(int b, int s) { return b < 2 ? b : 2 * b - 2 + s; }
DEV int token_of(int b, int row) { return 32 * (b >> 1) + 8 * (row >> 2) + (row & 3) + 4 * (b & 1); }
// A row's 16-byte pieces lie in LDS in an order of the row's own, so that what is read together falls into different banks: a piece of
// each of a block's 16 rows (by lanes 0 - 3, 12 - 15 of one lane group with 4 - 11 of the next), or, transposed, four pieces in a row of
// each of four rows. (With the row's number alone as the key, the transposed reads go at half the rate: 94 against 81 us.)
template <int CPR>
DEV int piece_at(int row, int c) {
    const int mid = (row >> 3 & 1 ? 2 : 0) ^ (row >> 4 & 1 ? 3 : 0);
    return row * CPR + (c ^ ((CPR >= 16 ? (row & 3) << 2 : (row & 2) << 1) | mid));
}

typedef float f2 __attribute__((ext_vector_type(2)));
DEV float pow2(int e) { return __builtin_bit_cast(float, (uint32_t)e << 23); }
// A largest magnitude's exponent: its 2^14 .. 2^15 is reached by pow2(268 - e), and left by pow2(e - 14).
DEV int exponent(float largest) {
    const int e = (int)(__builtin_bit_cast(uint32_t, largest) >> 23);
    return min(max(e, 15), 253);
}
DEV int in_range(int e) { return min(max(e, 1), 253); }

struct ChunkArgs {
    hq_state_t st;
    hq_delta_t d;
    const HqChunk *chunks;
    const HqRun *runs;
    int n_runs, n_chunks;
    char *work;
    float *places;  // states of the workspace
    float *outs;    // outputs ahead of their norm, 64 rows of v_dim for each chunk of the pass and value head
    Eps eps;        // as in DeltaArgs
    float one;  // 1: a factor that the compiler does not know, so that a difference is one fused instruction
};

// The largest of a wave's magnitudes, in rows of 16 lanes and across them
DEV float largest(float x) {
    uint32_t v = __builtin_bit_cast(uint32_t, x);
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, false));  // (rows turned by 8, 4, 2, 1 lanes)
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xf, 0xf, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x122, 0xf, 0xf, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x121, 0xf, 0xf, false));
    const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max(a[0], a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return __builtin_bit_cast(float, max(b[0], b[1]));
}

// T and M of a chunk and value head. Wave w forms rows 16 w .. of K K^T and Q K^T, one inverts the 16 x 16 blocks of I + A on the diagonal by
// substitution, a column a lane, and last each computes block column w of the inverse from the top down, T_ij = -T_ii sum_l A_il T_lj, on
// the fp32 matrix cores: each block of the column is the next one's operand.
// e^(G_i - G_j) of a block left of the diagonal is a factor of the row, from the block's first row, times one of the column, to it:
// neither exceeds 1. Sums of logarithms are formed in 64 bits and held as a multiple of 2^-9 and a rest, so that their differences
// lose nothing; below -150 a decay is 0 in 32 bits.
// Bound: a chain of some 9 us (loads, products, substitution, blocks, stores), hidden by four workgroups a CU: 1024 of them (32 chunks of
// 32 heads of 128) 14 us; 8352 of 16384 tokens 86, 56 of which would be their bytes'. (With every wave substituting in a block of its own, a
// fourth of the lanes' work new, and rows of 72 words, three fit a CU: 18 and 109. The wave with the sums of logarithms loads nothing by
// DMA: it would wait for that too.)
template <int KS>
__global__ void __launch_bounds__(256, KS <= 4 ? 4 : 2) k_delta_prep(ChunkArgs g) {
    constexpr int CPR = 4 * KS < 8 ? 8 : 4 * KS, LD = 68, LA = 68, LT = 20;
    __shared__ union {
        u4v kq[2][64 * CPR];
        struct {
            uint32_t t[64 * LD];  // T: its two terms
            union {
                uint32_t m[64 * LD];  // M likewise
                float At[64 * LA];    // A transposed
            };
        };
    } sh;
    __shared__ alignas(16) float Td[4][16 * LT];
    __shared__ alignas(16) f2 gam[64];
    __shared__ alignas(16) float bet[64], ms[4];
    __shared__ int t_exp;
    // workgroup i runs on XCD i % 8: the value heads of a key head on one
    const int nk = g.st.n_k_heads, nv = g.st.n_v_heads, dk = g.st.k_dim, rep = nv / nk;
    const int unit = blockIdx.x / (8 * rep) * 8 + blockIdx.x % 8;
    if (unit >= g.n_chunks * nk) return;
    const int at = unit / nk, hk = unit % nk, h = hk * rep + blockIdx.x / 8 % rep;
    const HqChunk ch = g.chunks[at];
    // (the waves' shares are unlike: turned from workgroup to workgroup, so that no SIMD has all the long ones)
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), w = (wave + (int)(blockIdx.x / 8)) & 3;
    const int lane = tid & 63, n = lane & 15, q = lane >> 4;
    if (w == 0) {
        const float gl = lane < ch.n ? g.d.decay[(size_t)(ch.tok0 + lane) * nv + h] : 0.f;
        const float bl = lane < ch.n ? g.d.beta[(size_t)(ch.tok0 + lane) * nv + h] : 0.f;
        bet[lane] = bl;
        const float most = largest(fabsf(bl));
        if (lane == 0) t_exp = exponent(most);
        double sum = (double)(gl < -150.f ? -150.f : gl) * 1.4426950408889634074;  // to base 2
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const double y = __shfl_up(sum, o, 64);
            if (lane >= o) sum += y;
        }
        const double top = rint(sum * 512.0) * (1.0 / 512.0);
        gam[lane] = f2{(float)top, (float)(sum - top)};
    } else {
        // (a wave that loads by DMA and waits for a register's load waits for both)
        const uint32_t row_bytes = (uint32_t)g.d.qk_stride * 2u, range = (uint32_t)(ch.n - 1) * row_bytes + (uint32_t)dk * 2u;
        const rsrc_t rk = make_rsrc(g.d.k + (size_t)ch.tok0 * g.d.qk_stride + hk * dk, range), rq = make_rsrc(g.d.q + (size_t)ch.tok0 * g.d.qk_stride + hk * dk, range);
#pragma unroll
        for (int c = 0; c < CPR; c += 3) {
            const int i = c + w - 1;
            if (i >= CPR) break;
            const int slot = 64 * i + lane, row = slot / CPR, x = piece_at<CPR>(row, slot % CPR) - row * CPR;  // (its own inverse)
            const uint32_t off = 8 * x < dk ? (uint32_t)row * row_bytes + 16u * (uint32_t)x : 0x80000000u, to = (uint32_t)(uintptr_t)sh.kq + 1024u * (uint32_t)i;
            dma16_untracked(rk, to, off);
            dma16_untracked(rq, to + 1024u * CPR, off);
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    f4 A[4], M[4];
#pragma unroll
    for (int b = 0; b < 4; b++) {
        A[b] = M[b] = f4{0.f, 0.f, 0.f, 0.f};
        if (b > w) continue;
#pragma unroll
        for (int s = 0; s < KS; s++) {
            const h8 x = __builtin_bit_cast(h8, sh.kq[0][piece_at<CPR>(16 * b + n, 4 * s + q)]);
            A[b] = mfma(__builtin_bit_cast(h8, sh.kq[0][piece_at<CPR>(16 * w + n, 4 * s + q)]), x, A[b]);
            M[b] = mfma(__builtin_bit_cast(h8, sh.kq[1][piece_at<CPR>(16 * w + n, 4 * s + q)]), x, M[b]);
        }
    }
    const int i0 = 16 * w + 4 * q;
    const auto decay = [](f2 i, f2 j) { return __builtin_amdgcn_exp2f((i[0] - j[0]) + (i[1] - j[1])); };
    f2 gi[4];
#pragma unroll
    for (int r = 0; r < 4; r++) gi[r] = gam[i0 + r];
    const f2 first = gam[16 * w];
    const f4 beta = *(const f4 *)(bet + i0);
    float mx = 0.f, row[4];
#pragma unroll
    for (int r = 0; r < 4; r++) row[r] = decay(gi[r], first);
    __syncthreads();
#pragma unroll
    for (int b = 0; b < 4; b++) {
        if (b > w) continue;
        const f2 gj = gam[16 * b + n];
        if (b < w) {
            const float col = decay(first, gj);
#pragma unroll
            for (int r = 0; r < 4; r++) A[b][r] = beta[r] * row[r] * (col * A[b][r]), M[b][r] = row[r] * (col * M[b][r]);
        } else {
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const float x = decay(gi[r], gj);  // (above the diagonal anything)
                A[b][r] = n < 4 * q + r ? beta[r] * x * A[b][r] : 0.f;
                M[b][r] = n <= 4 * q + r ? x * M[b][r] : 0.f;
            }
        }
        mx = fmaxf(fmaxf(mx, fabsf(M[b][0])), fabsf(M[b][1]));
        mx = fmaxf(fmaxf(mx, fabsf(M[b][2])), fabsf(M[b][3]));
        *(f4 *)(sh.At + (16 * b + n) * LA + i0) = A[b];
    }
    mx = largest(mx);
    if (lane == 0) ms[w] = mx;
    __syncthreads();
    if (w == 0) {  // (it had the least to do before)
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; i++) x[i] = i == n ? 1.f : 0.f;
#pragma unroll
        for (int j = 0; j < 15; j++)
#pragma unroll
            for (int i4 = (j + 1) / 4; i4 < 4; i4++) {
                const f4 a = *(const f4 *)(sh.At + (16 * q + j) * LA + 16 * q + 4 * i4);
#pragma unroll
                for (int r = 0; r < 4; r++)
                    if (4 * i4 + r > j) x[4 * i4 + r] = fmaf(-a[r], x[j], x[4 * i4 + r]);
            }
#pragma unroll
        for (int i = 0; i < 16; i++) Td[q][i * LT + n] = x[i];
    }
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
                for (int r = 0; r < 4; r++) y = __builtin_amdgcn_mfma_f32_16x16x4f32(sh.At[(16 * l + 4 * q + r) * LA + 16 * i + n], T[l][r], y, 0, 0, 0);
            }
        const f4 t = *(const f4 *)(Td[i] + n * LT + 4 * q);
#pragma unroll
        for (int r = 0; r < 4; r++) z = __builtin_amdgcn_mfma_f32_16x16x4f32(t[r], y[r], z, 0, 0, 0);
        T[i] = -z;
    }
    const float scale = pow2(T_EXP - t_exp) * bet[16 * w + n];
    const int em = exponent(fmaxf(fmaxf(ms[0], ms[1]), fmaxf(ms[2], ms[3])));
    const float to_m = pow2(268 - em);
    const auto terms = [](float v) { return __builtin_bit_cast(uint32_t, h2{(_Float16)v, (_Float16)(v - (float)(_Float16)v)}); };
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (i >= (w & ~1)) {  // (above the diagonal: the half of a fragment that is zero)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                sh.t[(16 * i + 4 * q + r) * LD + 16 * w + n] = terms(T[i][r] * scale);
            }
        }
        if (i <= (w | 1)) {
#pragma unroll
            for (int r = 0; r < 4; r++) sh.m[(i0 + r) * LD + 16 * i + n] = terms(M[i][r] * to_m);
        }
    }
    __syncthreads();
    char *const to = g.work + ((size_t)at * nv + h) * HQ_CHUNK_BYTES + lane * 16;
#pragma unroll
    for (int p0 = 0; p0 < 12; p0 += 4) {
        const int p = p0 + wave, k = p % 6, b = k < 2 ? k : k / 2 + 1, s = k < 2 ? 0 : k & 1;
        const u4v *const x = (const u4v *)((p < 6 ? sh.t : sh.m) + token_of(b, n) * LD + 32 * s + 8 * q);
        const u4v u = x[0], v = x[1];
        // (the terms of neighbouring values lie side by side)
        char *const o = to + ((p < 6 ? FRAG_T : FRAG_M) + k) * 1024;
        *(u4v *)o = u4v{__builtin_amdgcn_perm(u.y, u.x, 0x05040100u), __builtin_amdgcn_perm(u.w, u.z, 0x05040100u),
                        __builtin_amdgcn_perm(v.y, v.x, 0x05040100u), __builtin_amdgcn_perm(v.w, v.z, 0x05040100u)};
        *(u4v *)(o + 6 * 1024) = u4v{__builtin_amdgcn_perm(u.y, u.x, 0x07060302u), __builtin_amdgcn_perm(u.w, u.z, 0x07060302u),
                                     __builtin_amdgcn_perm(v.y, v.x, 0x07060302u), __builtin_amdgcn_perm(v.w, v.z, 0x07060302u)};
    }
    if (wave == 3) {
        float *const v = (float *)(g.work + ((size_t)at * nv + h) * HQ_CHUNK_BYTES + FRAG_VEC * 1024);
        v[lane] = decay(gam[lane], f2{0.f, 0.f});
        v[64 + lane] = decay(gam[63], gam[lane]);
        if (lane == 0) v[128] = g.d.scale * pow2(em - 14), ((int *)v)[129] = t_exp;
    }
}

typedef short s4v __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4v lds_s4v;
typedef const __attribute__((address_space(3))) u4v lds_u4;
typedef const __attribute__((address_space(3))) float lds_f;
typedef const __attribute__((address_space(3))) int lds_i;
typedef const __attribute__((address_space(3))) _Float16 lds_h;

// Two fp16 terms of 8 values scaled by sc: accumulator blocks a and b as an operand. Scaling and conversion stay two instructions:
// fused into one that writes half a register they go at half the rate (9.4 clocks an instruction against 5.4).
DEV h8 halves(const f4 &a, const f4 &b) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const f4 &x = j < 2 ? a : b;
        w[j] = __builtin_bit_cast(uint32_t, h2{(_Float16)x[2 * j & 3], (_Float16)x[(2 * j & 3) + 1]});
        asm("" : "+v"(w[j]));  // (a pair from one conversion is not to be converted again, value by value, where it is subtracted)
    }
    return __builtin_bit_cast(h8, u4v{w[0], w[1], w[2], w[3]});
}
DEV h8 first_term(const f4 &a, const f4 &b, float sc) { return halves(a * sc, b * sc); }
DEV h8 second_term(const f4 &a, const f4 &b, float sc, h8 hi) {
    f4 x, y;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        x[j] = fmaf(a[j], sc, -(float)hi[j]), y[j] = fmaf(b[j], sc, -(float)hi[4 + j]);
        float u = x[j], v = y[j];
        asm("" : "+v"(u), "+v"(v));
        x[j] = u, y[j] = v;
    }
    return halves(x, y);
}
// The largest magnitude of a column: 4 N values of each of the four lanes that have it
template <int N>
DEV float column_max(const f4 (&x)[N]) {
    float m[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < N; i++) {
        m[0] = fmaxf(fmaxf(m[0], fabsf(x[i][0])), fabsf(x[i][1]));
        m[1] = fmaxf(fmaxf(m[1], fabsf(x[i][2])), fabsf(x[i][3]));
    }
    uint32_t v = __builtin_bit_cast(uint32_t, fmaxf(m[0], m[1]));
    const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max(a[0], a[1]);  // (magnitudes: their order as integers)
    const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return __builtin_bit_cast(float, max(b[0], b[1]));
}

// The chunks of a run in order. A workgroup has 16 W value columns of a head; wave w < W holds S for 16 of them, takes it from chunk to
// chunk and needs no other wave's results. The four waves behind them bring the next chunk's operands to LDS by DMA: an instruction of
// it holds its wave for some 70 clocks, which the way from one state to the next, what bounds a long run, has no room for.
//
// A column of S is held in units of a power of two, taken from a bound of its magnitudes (the bound before, decayed, and what a chunk can
// add, 64 times its largest U as no key's element exceeds 1; every 16 chunks the largest itself): so S can enter products without a
// look over it, and fp16's range leaves what the bound is too large by.
//
// Bound: the way from one state to the next, some 750 instructions of one wave in order, which its SIMD has for itself: 4400 clocks a chunk
// (32 heads of 128), the products in them 2100; the outputs' work fills what the state's leaves. Products are started as soon as half of
// their operands are there (both halves first: 3.5 % more). W columns' waves read the same operands from LDS: 4 waves; with 2 (1), one
// sequence of 2048 tokens takes 76 (75) us in place of 80 (in parts 71, for which narrower groups leave no CUs), ten prompts of 16384 354
// (585) in place of 290; with 8 a chunk takes twice as long.
// (wider keys' operands do not all fit the registers: they are read where they are used)
#define STAGE if (KS <= 4) __builtin_amdgcn_sched_barrier(0)
// N times a product and M other instructions (what: 2 arithmetic, 0x100 reads of LDS), in the order of issue
#define MIX(N, what, M)                                          \
    if (KS <= 4) {                                               \
        _Pragma("unroll") for (int i_ = 0; i_ < (N); i_++) {     \
            __builtin_amdgcn_sched_group_barrier(8, 1, 0);       \
            __builtin_amdgcn_sched_group_barrier(what, M, 0);    \
        }                                                        \
    }
// OUT: outputs are formed, in fp16 where they belong or, ahead of their norm, in fp32 (in fp16 they would be rounded twice, and the norm
// takes sizes that fp16 has not). Without: a part's effect on states, Q from zeros or, from I and without values, P (a chunk takes some
// 1.8 us either way: it is the way from state to state that bounds both).
enum { STATES_ONLY, TO_OUT, TO_NORM };
// N times a product, D reads of LDS and V arithmetic instructions
#define MIX2(N, D, V)                                            \
    if (KS <= 4) {                                               \
        _Pragma("unroll") for (int i_ = 0; i_ < (N); i_++) {     \
            __builtin_amdgcn_sched_group_barrier(8, 1, 0);       \
            __builtin_amdgcn_sched_group_barrier(0x100, D, 0);   \
            __builtin_amdgcn_sched_group_barrier(2, V, 0);       \
        }                                                        \
    }
template <int KS, int W, int OUT>
__global__ void __launch_bounds__(64 * (W + 4), 1) k_delta_scan(ChunkArgs g) {
    constexpr int LW = 4;  // waves that load
    constexpr int CPR = 4 * KS < 8 ? 8 : 4 * KS;
    constexpr int KB = CPR, VB = 2 * W;    // KB of a chunk's keys or queries (64 rows of CPR pieces of 16 bytes) and of its values
    constexpr int BUFS = KS <= 4 ? 2 : 1;  // (two chunks of wider keys do not fit: the next one's wait until this one is done)
    constexpr int AHEAD = 2;               // steps of K or Q that are read before their use
    constexpr int FRAGS = OUT ? FRAG_VEC : FRAG_M;
    constexpr int AT_F = OUT ? 2 * KB : KB, AT_VEC = AT_F + FRAGS, AT_V = AT_VEC + 1, SIZE = AT_V + VB;
    static_assert(KB % LW == 0, "whole rounds of loads");
    __shared__ alignas(1024) char lds[BUFS * SIZE * 1024];
    const int nk = g.st.n_k_heads, nv = g.st.n_v_heads, dk = g.st.k_dim, dv = g.st.v_dim;
    const int groups = ((OUT ? dv : max(dk, dv)) + 16 * W - 1) / (16 * W);
    // workgroup i runs on XCD i % 8: the groups of one head on one, where they share its keys
    const int head = blockIdx.x / (8 * groups) * 8 + blockIdx.x % 8, group = blockIdx.x / 8 % groups;
    if (head >= g.n_runs * nv) return;
    const HqRun run = g.runs[head / nv];
    const bool eye = !OUT && run.from == HQ_IDENTITY;
    const int cols = eye ? dk : dv;
    if (!OUT && group * 16 * W >= cols) return;
    const int h = head % nv, hk = h / (nv / nk);
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 15, q = lane >> 4;
    const int chunks = (run.n + HQ_CHUNK - 1) / HQ_CHUNK;
    const auto buffer = [&](int c) { return (uint32_t)(uintptr_t)lds + 1024u * (uint32_t)(SIZE * (c % BUFS)); };
    const auto rows_of = [&](int c) { return (uint32_t)min(HQ_CHUNK, run.n - c * HQ_CHUNK); };
    // Rows behind the run's last lie past the buffers' ranges, as a row of heads is no longer than the stride: loads give zeros, stores
    // nothing. A row's values lie in LDS so that the four rows which a wave reads together fall into different banks.
    const auto v_piece = [](int row, int x) { return VB >= 8 ? x ^ (2 * (row >> 3 & 3)) : x; };
    if (w >= W) {
        const int lw = w - W;
        const uint32_t row_bytes = (uint32_t)g.d.qk_stride * 2u, v_bytes = (uint32_t)g.d.v_stride * 2u;
        uint32_t k_off[KB / LW], v_off[(VB + LW - 1) / LW];
#pragma unroll
        for (int i = 0; i < KB / LW; i++) {
            const int slot = 64 * (LW * i + lw) + lane, row = slot / CPR, x = piece_at<CPR>(row, slot % CPR) - row * CPR;  // (its own inverse)
            k_off[i] = 8 * x < dk ? (uint32_t)row * row_bytes + 16u * (uint32_t)x : 0x80000000u;
        }
#pragma unroll
        for (int i = 0; i < (VB + LW - 1) / LW; i++) {
            const int slot = 64 * (LW * i + lw) + lane, row = slot / VB, x = 8 * (2 * W * group + v_piece(row, slot % VB));
            v_off[i] = x < dv ? (uint32_t)row * v_bytes + 2u * (uint32_t)x : 0x80000000u;
        }
        const auto load = [&](int c) {
            const size_t tok = (size_t)(run.tok0 + c * HQ_CHUNK);
            const uint32_t range = (rows_of(c) - 1u) * row_bytes + (uint32_t)dk * 2u, to = buffer(c) + 1024u * (uint32_t)lw;
            const rsrc_t rk = make_rsrc(g.d.k + tok * g.d.qk_stride + hk * dk, range), rq = make_rsrc(g.d.q + tok * g.d.qk_stride + hk * dk, range);
            const rsrc_t rv = make_rsrc(g.d.v + tok * g.d.v_stride + (size_t)h * dv, eye ? 0u : (rows_of(c) - 1u) * v_bytes + (uint32_t)dv * 2u);
            const rsrc_t rw = make_rsrc(g.work + ((size_t)(run.chunk0 + c) * nv + h) * HQ_CHUNK_BYTES, (uint32_t)HQ_CHUNK_BYTES);
#pragma unroll
            for (int i = 0; i < KB; i += LW) dma16_untracked(rk, to + 1024u * (uint32_t)i, k_off[i / LW]);
#pragma unroll
            for (int i = 0; i < VB; i += LW)
                if (VB % LW == 0 || i + lw < VB) dma16_untracked(rv, to + 1024u * (uint32_t)(AT_V + i), v_off[i / LW]);
#pragma unroll
            for (int i = 0; i <= FRAGS; i += LW)
                if (i + LW <= FRAGS + 1 || i + lw <= FRAGS)
                    dma16_untracked(rw, to + 1024u * (uint32_t)(AT_F + i), 1024u * (uint32_t)(i + lw == FRAGS ? FRAG_VEC : i + lw) + 16u * (uint32_t)lane);
            if (OUT)
#pragma unroll
                for (int i = 0; i < KB; i += LW) dma16_untracked(rq, to + 1024u * (uint32_t)(KB + i), k_off[i / LW]);
        };
        if (BUFS == 2) load(0);
        for (int c = 0; c < chunks; c++) {
            if (BUFS == 1) {
                __syncthreads();
                load(c);
            }
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            if (BUFS == 2 && c + 1 < chunks) load(c + 1);
        }
        return;
    }
    const int col = 16 * (group * W + w) + n;
    const bool on = 16 * (group * W + w) < cols;  // (of a wave as a whole)
    const size_t size = (size_t)dk * dv, place = (size_t)dk * max(dk, dv);
    f4 S[2 * KS];
#pragma unroll
    for (int t = 0; t < 2 * KS; t++) S[t] = f4{0.f, 0.f, 0.f, 0.f};
    if (eye) {
#pragma unroll
        for (int t = 0; t < 2 * KS; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) S[t][r] = 32 * (t >> 1) + 8 * q + r + 4 * (t & 1) == col ? 1.f : 0.f;
    } else if (on && run.from != -1) {
        const float *s = (run.from >= 0 ? g.st.s + ((size_t)run.from * nv + h) * size : g.places + ((size_t)(-2 - run.from) * nv + h) * place) + col;
#pragma unroll
        for (int t = 0; t < 2 * KS; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int d = 32 * (t >> 1) + 8 * q + r + 4 * (t & 1);
                if (d < dk) S[t][r] = s[(size_t)d * dv];
            }
    }
    float bound = column_max(S);
    int unit = exponent(bound) - 14;
    {
        const float to_unit = pow2(in_range(254 - unit));
#pragma unroll
        for (int t = 0; t < 2 * KS; t++) S[t] = S[t] * to_unit;
    }
    constexpr uint32_t O_SIZE = OUT == TO_NORM ? 4 : 2;
    const uint32_t o_bytes = OUT == TO_NORM ? (uint32_t)dv * 4u : (uint32_t)g.d.out_stride * 2u;
    // where a lane's outputs go (wider keys: but the first is formed anew for each chunk, since the kernel spills; 2048 tokens of 16 heads of 256
    // 161 us in place of 165)
    constexpr int PLACES = KS <= 4 ? 16 : 1;
    uint32_t o_off[PLACES], k_in[KS], t_in[KS];
#pragma unroll
    for (int i = 0; i < PLACES; i++) o_off[i] = (uint32_t)token_of(i >> 2, 4 * q + (i & 3)) * o_bytes + O_SIZE * (uint32_t)col;
    // what a lane reads of K and Q, of K transposed and of V, as offsets into a chunk's buffer
#pragma unroll
    for (int s = 0; s < KS; s++) k_in[s] = 16u * (uint32_t)piece_at<CPR>(token_of(0, n), 4 * s + q), t_in[s] = 16u * (uint32_t)piece_at<CPR>(8 * q + (n >> 2), 4 * s + (n & 3));
    // (wider keys: values one by one, since by columns, 12 instructions less, the kernel spills and takes 10 % longer)
    constexpr bool BY_COLUMN = KS <= 4;
    const uint32_t v_in = 1024u * AT_V + (BY_COLUMN ? 16u * (uint32_t)((8 * q + (n >> 2)) * VB + v_piece(8 * q, 2 * w + (n >> 1 & 1))) + 8u * (uint32_t)(n & 1)
                                                    : 16u * (uint32_t)(8 * q * VB + v_piece(8 * q, 2 * w + (n >> 3))) + 2u * (uint32_t)(n & 7));
    // lane i of a group of 16 hands over 4 values of row i / 4, and gets one column's of 4 rows
    const auto read_tr = [](uint32_t at) { return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4v *)(uintptr_t)at); };
    const auto read16 = [](uint32_t at) { return __builtin_bit_cast(h8, *(lds_u4 *)(uintptr_t)at); };
    for (int c = 0; c < chunks; c++) {
        if (BUFS == 1) __syncthreads();
        __syncthreads();
        if (!on) continue;
        const uint32_t base = buffer(c), f_at = base + 1024u * AT_F + 16u * (uint32_t)lane, vec_at = base + 1024u * AT_VEC + 32u * (uint32_t)q;
        uint32_t k_at[KS], t_at[KS];
#pragma unroll
        for (int s = 0; s < KS; s++) k_at[s] = base + k_in[s], t_at[s] = base + t_in[s];
        const auto rows4 = [&](int which, int b) { return __builtin_bit_cast(f4, read16(vec_at + 256u * (uint32_t)which + 4u * (uint32_t)token_of(b, 0))); };
        const float keep = *(lds_f *)(uintptr_t)(base + 1024u * AT_VEC + 4u * 63u), m_unit = OUT ? *(lds_f *)(uintptr_t)(base + 1024u * AT_VEC + 4u * 128u) : 0.f;
        const int t_exp = *(lds_i *)(uintptr_t)(base + 1024u * AT_VEC + 4u * 129u);
        // Reads of LDS are issued a stage ahead of their use (STAGE: nothing moves past it), and what the outputs need is put between the
        // steps of the state.
        const auto read_rows = [&](int what, int s, h8(&x)[4]) {
#pragma unroll
            for (int b = 0; b < 4; b++) x[b] = read16(k_at[s] + 1024u * KB * (uint32_t)what + 16u * CPR * (uint32_t)token_of(b, 0));
        };
        h8 K[KS][4], Q[KS][4];
#pragma unroll
        for (int s = 0; s < AHEAD; s++) read_rows(0, s, K[s]);
        h8 Sh[KS], Sl[KS];
#pragma unroll
        for (int s = 0; s < KS; s++) Sh[s] = halves(S[2 * s], S[2 * s + 1]), Sl[s] = second_term(S[2 * s], S[2 * s + 1], g.one, Sh[s]);
        const float back = pow2(unit);
        f4 X[4], O[4], eg[4];
        h4 V[4];
#pragma unroll
        for (int b = 0; b < 4; b++) X[b] = O[b] = f4{0.f, 0.f, 0.f, 0.f};
        STAGE;
#pragma unroll
        for (int s = 0; s < KS; s++) {
            if (s + AHEAD < KS) read_rows(0, s + AHEAD, K[s + AHEAD]);
            else if (OUT) read_rows(1, s + AHEAD - KS, Q[s + AHEAD - KS]);
            if (s == KS - 1) {
#pragma unroll
                for (int b = 0; b < 4; b++) {
                    eg[b] = rows4(0, b);
                    if (BY_COLUMN) V[b] = __builtin_bit_cast(h4, read_tr(base + v_in + 16u * VB * (uint32_t)token_of(b, 0)));
                    else
#pragma unroll
                        for (int r = 0; r < 4; r++) V[b][r] = *(lds_h *)(uintptr_t)(base + v_in + 16u * VB * (uint32_t)token_of(b, r));
                }
            }
#pragma unroll
            for (int b = 0; b < 4; b++) X[b] = mfma(K[s][b], Sl[s], X[b]);
#pragma unroll
            for (int b = 0; b < 4; b++) X[b] = mfma(K[s][b], Sh[s], X[b]);
            MIX(8, 0x100, 3);
            STAGE;
        }
        const auto old = [&](int s) {
#pragma unroll
            for (int b = 0; b < 4; b++) O[b] = mfma(Q[s][b], Sl[s], O[b]);
#pragma unroll
            for (int b = 0; b < 4; b++) O[b] = mfma(Q[s][b], Sh[s], O[b]);
        };
        if (OUT) {
#pragma unroll
            for (int s = AHEAD; s < KS; s++) read_rows(1, s, Q[s]);
#pragma unroll
            for (int s = 0; s < AHEAD; s++) old(s);
        }
#pragma unroll
        for (int b = 0; b < 4; b++) {
            eg[b] = eg[b] * back;
#pragma unroll
            for (int r = 0; r < 4; r++) X[b][r] = fmaf(-eg[b][r], X[b][r], (float)V[b][r]);
        }
        if (OUT) MIX(8 * AHEAD, 2, 2);
        STAGE;
        h8 T[6], Tl[6];
#pragma unroll
        for (int i = 0; i < 6; i++) T[i] = read16(f_at + 1024u * (uint32_t)(FRAG_T + i)), Tl[i] = read16(f_at + 1024u * (uint32_t)(FRAG_T_LO + i));
        if (OUT)
#pragma unroll
            for (int s = AHEAD; s < KS; s++) old(s);
        const int ex = exponent(column_max(X));
        h8 Xh[2], Xl[2];
#pragma unroll
        for (int s = 0; s < 2; s++) Xh[s] = first_term(X[2 * s], X[2 * s + 1], pow2(268 - ex)), Xl[s] = second_term(X[2 * s], X[2 * s + 1], pow2(268 - ex), Xh[s]);
        f4 U[4];  // in units of 2^(uu - 127)
        const int uu = ex - 14 - (T_EXP - 127 - t_exp);
#pragma unroll
        for (int b = 0; b < 4; b++) U[b] = f4{0.f, 0.f, 0.f, 0.f};
        if (OUT) MIX(8 * (KS - AHEAD), 2, 3);
        STAGE;
        s4v Kt[2][2 * KS][2];
        const auto read_columns = [&](int s) {
#pragma unroll
            for (int t = 0; t < 2 * KS; t++)
#pragma unroll
                for (int e = 0; e < 2; e++)
                    Kt[s][t][e] = read_tr(t_at[t >> 1] + 8u * (uint32_t)(t & 1) + 16u * CPR * (uint32_t)(32 * s + 4 * e));
        };
        const auto column = [&](int s, int t) { return __builtin_bit_cast(h8, __builtin_shufflevector(Kt[s][t][0], Kt[s][t][1], 0, 1, 2, 3, 4, 5, 6, 7)); };
        f4 dec[4];
#pragma unroll
        for (int b = 0; b < 4; b++) dec[b] = rows4(1, b);
        read_columns(0);
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int i = 0; i < 3; i++)
#pragma unroll
                for (int b = 2 * s; b < 4; b++) U[b] = mfma(i == 0 ? Tl[frag_of(b, s)] : T[frag_of(b, s)], i == 1 ? Xl[s] : Xh[s], U[b]);
        MIX(18, 0x100, 1);
        STAGE;
        // the state's products of the chunk's first half start while the second's operands and the outputs' are formed
        const float mu = column_max(U);
        bound = fmaf(bound, keep, 64.f * mu * pow2(in_range(uu)));
        const int next = exponent(bound) - 14;
        const float sd = pow2(in_range(uu - next + 127)), ratio = keep * pow2(in_range(unit - next + 127));
        unit = next;
        h8 Uh[2], Ul[2], Dh[2], Dl[2];
        const auto written = [&](int s) {
            const f4 xd = U[2 * s] * dec[2 * s], yd = U[2 * s + 1] * dec[2 * s + 1];
            Dh[s] = halves(xd, yd), Dl[s] = second_term(xd, yd, g.one, Dh[s]);
        };
        U[0] = U[0] * sd, U[1] = U[1] * sd;
        written(0);
#pragma unroll
        for (int t = 0; t < 2 * KS; t++) S[t] = S[t] * ratio;
        STAGE;
        h8 M[6], Ml[6];
        if (OUT)
#pragma unroll
            for (int i = 0; i < 6; i++) M[i] = read16(f_at + 1024u * (uint32_t)(FRAG_M + i)), Ml[i] = read16(f_at + 1024u * (uint32_t)(FRAG_M_LO + i));
        read_columns(1);
        U[2] = U[2] * sd, U[3] = U[3] * sd;
        written(1);
        if (OUT)
#pragma unroll
            for (int s = 0; s < 2; s++) Uh[s] = halves(U[2 * s], U[2 * s + 1]), Ul[s] = second_term(U[2 * s], U[2 * s + 1], g.one, Uh[s]);
        f4 y[4];
#pragma unroll
        for (int b = 0; b < 4; b++) y[b] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < 2 * KS; t++) S[t] = mfma(column(0, t), Dl[0], S[t]);
#pragma unroll
        for (int t = 0; t < 2 * KS; t++) S[t] = mfma(column(0, t), Dh[0], S[t]);
        MIX2(4 * KS, 2, 5);
        STAGE;
        if (OUT)
#pragma unroll
            for (int s = 0; s < 2; s++)
#pragma unroll
                for (int i = 0; i < 3; i++)
#pragma unroll
                    for (int b = 2 * s; b < 4; b++) y[b] = mfma(i == 0 ? Ml[frag_of(b, s)] : M[frag_of(b, s)], i == 1 ? Ul[s] : Uh[s], y[b]);
        if (OUT)
#pragma unroll
            for (int b = 0; b < 4; b++) O[b] = eg[b] * g.d.scale * O[b];
        if (OUT) MIX(18, 2, 2);
        STAGE;
        const float bu = pow2(next) * m_unit;
        const rsrc_t ro = OUT == TO_NORM ? make_rsrc(g.outs + ((size_t)(run.chunk0 + c) * nv + h) * HQ_CHUNK * dv, rows_of(c) * o_bytes)
                                         : make_rsrc(g.d.out + (size_t)(run.tok0 + c * HQ_CHUNK) * g.d.out_stride + (size_t)h * dv, (rows_of(c) - 1u) * o_bytes + (uint32_t)dv * 2u);
#pragma unroll
        for (int t = 0; t < 2 * KS; t++) S[t] = mfma(column(1, t), Dl[1], S[t]);
#pragma unroll
        for (int t = 0; t < 2 * KS; t++) S[t] = mfma(column(1, t), Dh[1], S[t]);
        uint32_t o_at = o_off[0];
        asm("" : "+v"(o_at));  // (not held from chunk to chunk)
        if (OUT)
#pragma unroll
            for (int b = 0; b < 4; b++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float o = fmaf(bu, y[b][r], O[b][r]);
                    const uint32_t to = PLACES == 16 ? o_off[(4 * b + r) % PLACES] : o_at + (uint32_t)token_of(b, r) * o_bytes;
                    if (OUT == TO_NORM) __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, o), ro, to, 0u, 0);
                    else __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(short, (_Float16)o), ro, to, 0u, 0);
                }
        if (OUT) MIX(4 * KS, 2, 3);
        if ((c & 15) == 15) bound = column_max(S) * pow2(unit);
    }
    if (on && run.to != -1) {
        float *s = (run.to >= 0 ? g.st.s + ((size_t)run.to * nv + h) * size : g.places + ((size_t)(-2 - run.to) * nv + h) * place) + col;
#pragma unroll
        for (int t = 0; t < 2 * KS; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int d = 32 * (t >> 1) + 8 * q + r + 4 * (t & 1);
                if (d < dk) s[(size_t)d * cols] = S[t][r] * pow2(unit);
            }
    }
}

// The states between the parts of a sequence: S of the first part's end, then P S + Q of one after another, in place of Q. A workgroup has
// 16 columns of a head, wave w the rows 16 w .. (and 128 on). The products are of 32 bits: an accumulator's four rows of block m are what
// lane group q has of the contraction's steps 4 m .. 4 m + 3, so that a state's blocks lie in LDS as they come.
// Bound: one way through memory and a chain of products: 32 heads of 128, three parts: 5.9 us (8.8 with a head's columns on eight XCDs).
template <int KS>
__global__ void __launch_bounds__(512) k_delta_join(ChunkArgs g, const HqJoin *joins, int n_joins) {
    constexpr int RT = KS > 4 ? 2 : 1, KT = 8 * RT;
    __shared__ alignas(16) f4 at[2][KT][64];
    const int nv = g.st.n_v_heads, dk = g.st.k_dim, dv = g.st.v_dim, tiles = dv / 16, kt = dk / 16;
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, n = lane & 15, q = lane >> 4;
    // workgroup i runs on XCD i % 8: a head's on one, where they share its P
    const int head = blockIdx.x / (8 * tiles) * 8 + blockIdx.x % 8, h = head % nv, col = 16 * (int)(blockIdx.x / 8 % tiles) + n;
    if (head >= n_joins * nv) return;
    const HqJoin jn = joins[head / nv];
    const size_t size = (size_t)dk * dv, place = (size_t)dk * max(dk, dv);
    const auto state = [&](int i) { return g.places + ((size_t)i * nv + h) * place; };
    f4 x[RT], y[RT], first[RT], P[RT][KT];
    const auto load = [&](const float *s, int t) {
        const float *const p = s + (size_t)(16 * (w + 8 * t) + 4 * q) * dv + col;
        return f4{p[0], p[dv], p[2 * dv], p[3 * dv]};
    };
    const auto store = [&](float *s, int t, f4 v) {
        float *const p = s + (size_t)(16 * (w + 8 * t) + 4 * q) * dv + col;
        p[0] = v[0], p[dv] = v[1], p[2 * dv] = v[2], p[3 * dv] = v[3];
    };
    const auto part = [&](int j) {  // its P and Q
#pragma unroll
        for (int t = 0; t < RT; t++) {
            if (w + 8 * t >= kt) continue;
            y[t] = load(state(jn.place + 1 + j), t);
#pragma unroll
            for (int m = 0; m < KT; m++)
                if (m < kt) P[t][m] = *(const f4 *)(state(jn.place + jn.n + j - 1) + (size_t)(16 * (w + 8 * t) + n) * dk + 16 * m + 4 * q);
        }
    };
#pragma unroll
    for (int t = 0; t < RT; t++)
        if (w + 8 * t < kt) x[t] = load(state(jn.place + 1), t);
    if (jn.n > 2) part(1);
    if (jn.from != -1) {
#pragma unroll
        for (int t = 0; t < RT; t++)
            if (w + 8 * t < kt) first[t] = load(jn.from >= 0 ? g.st.s + ((size_t)jn.from * nv + h) * size : state(-2 - jn.from), t);
    }
    for (int j = 1; j < jn.n - 1; j++) {
#pragma unroll
        for (int t = 0; t < RT; t++)
            if (w + 8 * t < kt) at[j & 1][w + 8 * t][lane] = x[t];
        __syncthreads();  // (and the other half is free again: its readers have all come here)
#pragma unroll
        for (int m = 0; m < KT; m++) {
            if (m >= kt) continue;
            const f4 s = at[j & 1][m][lane];
#pragma unroll
            for (int t = 0; t < RT; t++)
                if (w + 8 * t < kt)
#pragma unroll
                    for (int r = 0; r < 4; r++) y[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(P[t][m][r], s[r], y[t], 0, 0, 0);
        }
#pragma unroll
        for (int t = 0; t < RT; t++)
            if (w + 8 * t < kt) store(state(jn.place + 1 + j), t, x[t] = y[t]);
        if (j + 2 < jn.n) part(j + 1);
    }
    if (jn.from != -1) {
#pragma unroll
        for (int t = 0; t < RT; t++)
            if (w + 8 * t < kt) store(state(jn.place), t, first[t]);
    }
}

// The norm and gate of chunks' outputs, from the workspace to where they belong: G lanes a head, eight columns a lane.
// Bound: bytes. 16384 tokens of 32 heads of 128, gates in fp32: 671 MB in 127 us, 5.3 TB/s (from fp16 outputs 537 MB in 101), a
// workgroup a token of a chunk, gates past the caches that hold the outputs (four tokens and without that: 134; 1100 tokens of 16 heads of 256 72 us in
// all in place of 79).
template <int G, bool F32>
__global__ void __launch_bounds__(256) k_delta_norm(ChunkArgs g) {
    const int nv = g.st.n_v_heads, dv = g.st.v_dim, u = threadIdx.x % G;
    const bool on = 8 * u < dv;
    const HqChunk ch = g.chunks[blockIdx.x];
    const int t = blockIdx.y;
    if (t >= ch.n) return;
    f4 wa = {0.f, 0.f, 0.f, 0.f}, wb = wa;
    if (on) wa = *(const f4 *)(g.d.norm + 8 * u), wb = *(const f4 *)(g.d.norm + 8 * u + 4);
    for (int h = threadIdx.x / G; h < nv; h += 256 / G) {
        const size_t in = (size_t)h * dv + (on ? 8 * u : 0);
        const size_t tok = (size_t)(ch.tok0 + t), zat = tok * g.d.gate_stride + in;
        const float *const from = g.outs + (((size_t)blockIdx.x * nv + h) * HQ_CHUNK + t) * dv + (on ? 8 * u : 0);
        float x[8];
        const f4 xa = *(const f4 *)from, xb = *(const f4 *)(from + 4);
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = on ? xa[e] : 0.f, x[4 + e] = on ? xb[e] : 0.f;
        float z[8];
        if (F32) {
            const f4 a = __builtin_nontemporal_load((const f4 *)((const float *)g.d.gate + zat)), b = __builtin_nontemporal_load((const f4 *)((const float *)g.d.gate + zat + 4));
#pragma unroll
            for (int e = 0; e < 4; e++) z[e] = a[e], z[4 + e] = b[e];
        } else {
            const h8 a = *(const h8 *)((const _Float16 *)g.d.gate + zat);
#pragma unroll
            for (int e = 0; e < 8; e++) z[e] = (float)a[e];
        }
        normalise<8, G>(x, dv, g.eps);
        h8 y;
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = (_Float16)(x[e] * (e < 4 ? wa[e & 3] : wb[e & 3]) * silu(z[e]));
        if (on) *(h8 *)((_Float16 *)g.d.out + tok * g.d.out_stride + in) = y;
    }
}

template <int KS>
void launch_chunks(ChunkArgs g, const HqPass &p, const HqRun *runs, const HqJoin *joins, hipStream_t s) {
    constexpr int W = hq_scan_columns(32 * KS) / 16;
    const int nv = g.st.n_v_heads, dk = g.st.k_dim, dv = g.st.v_dim;
    k_delta_prep<KS><<<((unsigned)g.n_chunks * (unsigned)g.st.n_k_heads + 7) / 8 * 8 * (unsigned)(nv / g.st.n_k_heads), 256, 0, s>>>(g);
    const auto grid = [&](int n, int cols) { return ((unsigned)n * (unsigned)nv + 7) / 8 * 8 * (unsigned)((cols + 16 * W - 1) / (16 * W)); };
    if (p.n_parts) {
        g.runs = runs + p.part0, g.n_runs = p.n_parts;
        k_delta_scan<KS, W, STATES_ONLY><<<grid(p.n_parts, std::max(dk, dv)), 64 * (W + 4), 0, s>>>(g);
        k_delta_join<KS><<<((unsigned)p.n_joins * (unsigned)nv + 7) / 8 * 8 * (unsigned)(dv / 16), 512, 0, s>>>(g, joins + p.join0, p.n_joins);
    }
    g.runs = runs + p.run0, g.n_runs = p.n_runs;
    if (g.d.norm) k_delta_scan<KS, W, TO_NORM><<<grid(p.n_runs, dv), 64 * (W + 4), 0, s>>>(g);
    else k_delta_scan<KS, W, TO_OUT><<<grid(p.n_runs, dv), 64 * (W + 4), 0, s>>>(g);
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
        const int64_t k_row = (int64_t)st->n_k_heads * st->k_dim, v_row = (int64_t)st->n_v_heads * st->v_dim;
        if (d->qk_stride < k_row || d->v_stride < v_row || d->out_stride < v_row)
            return hq_internal_fail("%s: strides %lld, %lld and %lld of tokens whose heads take %lld, %lld and %lld", who, (long long)d->qk_stride, (long long)d->v_stride,
                                    (long long)d->out_stride, (long long)k_row, (long long)v_row, (long long)v_row);
        // a chunk's rows are addressed by 32 bits
        if (!c->passes.empty())
            for (int64_t s : {d->qk_stride, d->v_stride, d->out_stride})
                if (s > MOST_CHUNK_STRIDE) return hq_internal_fail("%s: stride %lld (with more than %d new tokens of a sequence at most %lld)", who, (long long)s, HQ_STEP_ALONE, (long long)MOST_CHUNK_STRIDE);
        if (!(fabsf(d->scale) <= 1e20f)) return hq_internal_fail("%s: scale %g", who, (double)d->scale);
    }
    int cur = -1;
    SCK(hipGetDevice(&cur));
    if (cur != c->device) SCK(hipSetDevice(c->device));
    hipStream_t s = (hipStream_t)stream;
    hq_delta_t in = *d;
    Eps eps = {in.eps, in.eps, 0};
    if (in.norm) in.scale = frexpf(in.scale, &eps.e), eps.unit = ldexpf(eps.eps, -2 * eps.e);
    for (const HqPass &p : c->passes) {
        const ChunkArgs g = {*st, in, c->chunks + p.chunk0, nullptr, 0, p.n_chunks, c->work, (float *)(c->work + c->places_at), (float *)(c->work + c->outs_at), eps, 1.0f};
        if (st->k_dim <= 64) launch_chunks<2>(g, p, c->runs, c->joins, s);
        else if (st->k_dim <= 128) launch_chunks<4>(g, p, c->runs, c->joins, s);
        else launch_chunks<8>(g, p, c->runs, c->joins, s);
        if (d->norm) {
            const int lanes = st->v_dim <= 64 ? 8 : st->v_dim <= 128 ? 16 : 32;
            const dim3 grid((unsigned)p.n_chunks, HQ_CHUNK);
#define HQ_NORM(G)                                                          \
    do {                                                                    \
        if (d->gate_f32) k_delta_norm<G, true><<<grid, 256, 0, s>>>(g);     \
        else k_delta_norm<G, false><<<grid, 256, 0, s>>>(g);                \
    } while (0)
            if (lanes == 8) HQ_NORM(8);
            else if (lanes == 16) HQ_NORM(16);
            else HQ_NORM(32);
#undef HQ_NORM
        }
        SCK(hipGetLastError());
    }
    // A head's waves in one workgroup; few heads with one token and no norm, for which they would have to meet, a wave each: 32 heads 5.0
    // us (in one workgroup 5.2), 128 6.5 (7.0), but of five tokens, whose keys each wave then fetches itself, 9.7 (9.4) and 13.1 (11.8).
    const int waves = (st->v_dim + 31) / 32;
    const bool apart = !d->norm && c->longest_step <= 1 && (int64_t)c->n_steps * st->n_v_heads * waves <= 2 * c->n_cu;
    const unsigned threads = apart ? 64u : 64u * (unsigned)waves;
    // (a launch has fewer than 2^32 threads)
    const int most = std::max(1, (int)((((int64_t)1 << 32) - 1) / ((int64_t)st->n_v_heads * threads)));
    for (int i = 0; i < c->n_steps; i += most) {
        const DeltaArgs g = {*st, in, c->seqs, c->steps + i, eps};
        const dim3 grid((unsigned)std::min(most, c->n_steps - i) * (unsigned)st->n_v_heads, apart ? (unsigned)waves : 1u);
        if (st->k_dim == 64) k_delta_step<8, true><<<grid, threads, 0, s>>>(g);
        else if (st->k_dim < 64) k_delta_step<8, false><<<grid, threads, 0, s>>>(g);
        else if (st->k_dim == 128) k_delta_step<16, true><<<grid, threads, 0, s>>>(g);
        else if (st->k_dim < 128) k_delta_step<16, false><<<grid, threads, 0, s>>>(g);
        else if (st->k_dim == 256) k_delta_step<32, true><<<grid, threads, 0, s>>>(g);
        else k_delta_step<32, false><<<grid, threads, 0, s>>>(g);
        SCK(hipGetLastError());
    }
    return 0;
}
