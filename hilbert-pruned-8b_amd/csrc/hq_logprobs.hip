// hq_logprobs.hip - log probabilities of given tokens, entropy and likeliest tokens of rows of logits (hq_logprobs,
// include/hq_serve.h), and the best continuations of groups of beams (hq_beam).
//
// One pass over the logits: each thread keeps m = max x, s = sum e^(x - m) and t = sum (x - m) e^(x - m) of what it reads,
// rescaled when m grows, so that log p = x - m - log s and the entropy is log s - t / s; both sums have one sign, nothing
// cancels. Few rows are split over workgroups; the last of a row's to arrive joins their sums in part order.
//
// The top k come from the same pass: the k-th largest of the threads' maxima, B, is no larger than the k-th largest logit, so
// only the threads' shares whose maximum reaches B are read again (k of 256 or more, from cache), and the few logits found
// there are ranked by counting. No share is sorted and nothing is inserted anywhere in the stream.
//
// Bound: the bytes of the logits. 512 rows of 151936, fp32: 311 MB in 55 us, 5.6 TB/s (59 where none of them is in cache); fp16: 156 MB in 40.
// Few rows: the chain of launch, loads, the row's last workgroup (5.5 us for one row of 32000, 8 for 16 of 151936, fp16) and the
// second look (3 us more with the top 5 of the one, 7 with the top 20 of the other).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <math.h>

#include "hq_batch.h"
#include "hq_device.h"

namespace {

constexpr int NT = 512, WAVES = NT / 64;
constexpr int MAX_PARTS = 32;      // of a row
constexpr int MAX_BUCKETS = 512;   // shares of a row that the second look chooses from
constexpr int FOUND = 1024, TIES = 256;

struct LpArgs {
    const void *x;
    const uint32_t *ids;
    float *logp, *entropy, *top_logp;
    uint32_t *top_ids;
    int64_t stride;
    uint32_t V;
    int n_ids, k;
    int parts, group;  // workgroups per row; neighbouring threads whose maxima make one bucket
    uint32_t per;      // 16-byte pieces per part
    float *work;       // [rows][parts][4 + NT / group]: m, s, t, -, then the buckets
    int *counters;     // [rows], zero when idle
};

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

// log p of a logit x in a row of maximum m and sum of e^(x - m) = e^logs
DEV float log_p(float x, float m, float logs) {
    if (m == -INFINITY && logs == -INFINITY) return -INFINITY;
    return (x - m) - logs;
}

constexpr float LOG2E = 1.4426950408889634f;
DEV float ex(float d) { return __builtin_amdgcn_exp2f(d * LOG2E); }  // e^d

struct Sums {
    float m, s, t;
    // to a maximum of mn >= m (differences past 1e30 weigh 0 and must not make NaN of t)
    __device__ __forceinline__ void raise(float mn) {
        const float f = m == -INFINITY ? 0.f : ex(m - mn);
        t = m == -INFINITY ? 0.f : (t + fmaxf(m - mn, -1e30f) * s) * f;
        s = m == -INFINITY ? s : s * f;
        m = mn;
    }
    __device__ __forceinline__ void add(Sums o) {
        const float mn = fmaxf(m, o.m);
        raise(mn), o.raise(mn);
        s += o.s, t += o.t;
    }
};

template <bool F32>
constexpr int VEC = F32 ? 4 : 8;  // logits of a 16-byte piece

// Piece v of a row whose first logit is `mis` logits into piece 0: its values, -inf outside the row.
template <bool F32>
DEV void piece(const char *base, uint32_t v, uint32_t n_pieces, uint32_t mis, uint32_t V, float (&x)[VEC<F32>]) {
    const u4v w = *(const u4v *)(base + (size_t)v * 16);
#pragma unroll
    for (int e = 0; e < VEC<F32>; e++) x[e] = F32 ? __builtin_bit_cast(float, (uint32_t)w[e % 4]) : h2f((uint16_t)(w[e / 2 % 4] >> (16 * (e % 2))));
    if (v == 0 || v + 1 == n_pieces) {
#pragma unroll
        for (int e = 0; e < VEC<F32>; e++)
            if (v * VEC<F32> + e - mis >= V) x[e] = -INFINITY;  // (unsigned: before the row too)
    }
}

struct Shared {
    Sums sums[WAVES];
    uint32_t bucket[MAX_BUCKETS];
    int hit[MAX_BUCKETS];
    alignas(16) unsigned long long found[FOUND + TIES], out[64];
    int n_found, n_ties, n_hit, last, count[WAVES];
};

template <bool F32>
struct Row {
    const LpArgs &g;
    const char *base;
    uint32_t mis, n_pieces;
    __device__ __forceinline__ float at(uint32_t i) const {
        const size_t a = (size_t)mis + i;
        return F32 ? ((const float *)base)[a] : (float)((const _Float16 *)base)[a];
    }
    // f(order, token) of the logits that the threads of the `n` buckets sh.hit[] read, but for pieces in which none reaches
    // `least` (a logit; NaN: all pieces are wanted) (whole workgroup)
    template <class F>
    __device__ __forceinline__ void buckets(const Shared &sh, int n, float least, F f) const {
        constexpr int U = 4;  // pieces in flight per thread
        const uint32_t rounds = (g.per + NT - 1) / NT, shift = __builtin_ctz(g.group), total = (uint32_t)n * rounds << shift;
        for (uint32_t j0 = threadIdx.x; j0 < total; j0 += U * NT) {
            float x[U][VEC<F32>];
            uint32_t v[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const uint32_t j = j0 + u * NT, y = j >> shift, h = y / rounds;
                v[u] = n_pieces;
                if (j >= total) continue;
                const uint32_t t = (uint32_t)sh.hit[h] << shift, at = (y - h * rounds) * NT + t % NT + (j & (g.group - 1));  // t: the bucket's first thread
                const uint32_t i = t / NT * g.per + at;
                if (at < g.per && i < n_pieces) {
                    v[u] = i;
                    piece<F32>(base, i, n_pieces, mis, g.V, x[u]);
                }
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                if (v[u] >= n_pieces) continue;
                float mx = x[u][0];
#pragma unroll
                for (int e = 1; e < VEC<F32>; e++) mx = fmaxf(mx, x[u][e]);
                if (mx < least) continue;
#pragma unroll
                for (int e = 0; e < VEC<F32>; e++) {
                    const uint32_t i = v[u] * VEC<F32> + e - mis;
                    if (i < g.V) f(order_of(x[u][e]), i);
                }
            }
        }
    }
    // how many logits of the row are at least `o` in order (whole workgroup)
    __device__ __forceinline__ int count_from(uint32_t o, Shared &sh) const {
        int c = 0;
        for (uint32_t i = threadIdx.x; i < g.V; i += NT) c += order_of(at(i)) >= o;
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) c += __shfl_xor(c, d, 64);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) sh.count[threadIdx.x >> 6] = c;
        __syncthreads();
        c = 0;
        for (int w = 0; w < WAVES; w++) c += sh.count[w];
        return c;
    }
};

// A bound that at least k of the n words of sh.bucket reach (0 where there are fewer), every wave for itself: the k-th largest
// of them, or for small k of the 64 maxima of words a lane, which is little less and takes one count per bit, not four. The
// words that reach it to sh.hit (sh.n_hit, 0 before; any order).
DEV uint32_t choose(Shared &sh, int n, int k) {
    constexpr int W = MAX_BUCKETS / 64;
    const int tid = threadIdx.x, lane = tid & 63;
    uint32_t x[W], top = 0, b = 0;
#pragma unroll
    for (int i = 0; i < W; i++) x[i] = 64 * i + lane < n ? sh.bucket[64 * i + lane] : 0u, top = std::max(top, x[i]);
    if (k <= 32) {
        for (int bit = 31; bit >= 0; bit--)
            if (__popcll(__ballot(top >= (b | 1u << bit))) >= k) b |= 1u << bit;
    } else {
        for (int bit = 31; bit >= 0; bit--) {
            int c = 0;
#pragma unroll
            for (int i = 0; i < W; i++) c += __popcll(__ballot(x[i] >= (b | 1u << bit)));
            if (c >= k) b |= 1u << bit;
        }
    }
    if (tid < n && sh.bucket[tid] >= b) sh.hit[atomicAdd(&sh.n_hit, 1)] = tid;
    return b;
}

// how many of the first n keys of v (there is room for a multiple of eight) are larger
DEV int larger_of(const unsigned long long *v, int n, unsigned long long key) {
    int c = 0;
    for (int i = 0; i < n; i += 8) {
        unsigned long long y[8];
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = v[i + e];
#pragma unroll
        for (int e = 0; e < 8; e++) c += i + e < n && y[e] > key;
    }
    return c;
}

// The row's top k to sh.out as keys, likeliest first: buckets (n of them) hold the orders of their maxima; odd: the row has
// a NaN or +inf, whose buckets say nothing.
template <bool F32>
DEV void top_k(const Row<F32> &row, int n, bool odd, Shared &sh) {
    const int k = row.g.k, tid = threadIdx.x;
    uint32_t B = 0;
    bool exact = odd;
    if (tid == 0) sh.n_hit = odd ? n : 0;
    if (odd) {
        if (tid < n) sh.hit[tid] = tid;
    } else {
        __syncthreads();
        B = choose(sh, n, k);
    }
    for (;;) {
        if (exact) {  // B: the k-th largest logit itself
            B = 0;
            for (int bit = 31; bit >= 0; bit--)
                if (row.count_from(B | 1u << bit, sh) >= k) B |= 1u << bit;
        }
        __syncthreads();
        if (tid == 0) sh.n_found = sh.n_ties = 0;
        __syncthreads();
        const auto take = [&](uint32_t o, uint32_t i) {
            if (o < B) return;
            const unsigned long long key = (unsigned long long)o << 32 | (uint32_t)~i;
            if (o > B) {
                const int at = atomicAdd(&sh.n_found, 1);
                if (at < FOUND) sh.found[at] = key;
            } else {
                const int at = atomicAdd(&sh.n_ties, 1);
                if (at < TIES) sh.found[FOUND + at] = key;
            }
        };
        row.buckets(sh, sh.n_hit, odd ? NAN : from_order(B), take);  // (no bound, B = 0: NaN too)
        __syncthreads();
        if (sh.n_found <= FOUND) break;
        exact = true;  // more than FOUND logits pass the buckets' bound (a sorted row): fewer than k pass the exact one
    }
    int nf = sh.n_found;
    if (nf < k && sh.n_ties > TIES) {
        // the first k - nf logits that equal B, in the order of tokens
        const int need = k - nf;
        int have = 0;
        for (uint32_t i0 = 0; i0 < row.g.V && have < need; i0 += NT) {
            const uint32_t i = i0 + tid;
            const bool tie = i < row.g.V && order_of(row.at(i)) == B;
            const uint64_t mask = __ballot(tie);
            __syncthreads();
            if ((tid & 63) == 0) sh.count[tid >> 6] = __popcll(mask);
            __syncthreads();
            int at = have + __popcll(mask & ((1ull << (tid & 63)) - 1));
            for (int w = 0; w < WAVES; w++) {
                if (w < tid >> 6) at += sh.count[w];
                have += sh.count[w];
            }
            if (tie && at < need) sh.found[FOUND + at] = (unsigned long long)B << 32 | (uint32_t)~i;
        }
        __syncthreads();
        if (tid == 0) sh.n_ties = std::min(have, need);
        __syncthreads();
    }
    const int nt = nf < k ? std::min(sh.n_ties, TIES) : 0, all = nf + nt;
    for (int x = tid; x < all; x += NT) {
        const unsigned long long key = sh.found[x < nf ? x : FOUND + x - nf];
        const int rank = larger_of(sh.found, nf, key) + larger_of(sh.found + FOUND, nt, key);
        if (rank < k) sh.out[rank] = key;
    }
    __syncthreads();
}

template <bool F32>
__global__ void __launch_bounds__(NT) k_logprobs(LpArgs g) {
    __shared__ Shared sh;
    constexpr int U = 2;  // pieces in flight per thread
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const size_t r = blockIdx.x / g.parts;
    const int part = blockIdx.x % g.parts;
    const char *const start = (const char *)g.x + r * (size_t)g.stride * (F32 ? 4 : 2);
    const uint32_t mis = (uint32_t)((uintptr_t)start & 15u) / (F32 ? 4 : 2);
    const Row<F32> row = {g, start - ((uintptr_t)start & 15u), mis, (mis + g.V + VEC<F32> - 1) / VEC<F32>};
    const uint32_t v0 = (uint32_t)part * g.per, v1 = std::min(v0 + g.per, row.n_pieces);
    // the first tokens asked for, before the pass: theirs is a chain of two loads
    const uint32_t asked = g.logp && tid < g.n_ids ? g.ids[r * g.n_ids + tid] : 0u;
    const float x_asked = g.logp && tid < g.n_ids && asked < g.V ? row.at(asked) : 0.f;
    Sums a = {-INFINITY, 0.f, 0.f};
    for (uint32_t v = v0 + tid; v < v1; v += U * NT) {
        float x[U][VEC<F32>];
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (v + u * NT < v1) piece<F32>(row.base, v + u * NT, row.n_pieces, mis, g.V, x[u]);
            else
#pragma unroll
                for (int e = 0; e < VEC<F32>; e++) x[u][e] = -INFINITY;
        }
        float mn = a.m;
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int e = 0; e < VEC<F32>; e++) mn = fmaxf(mn, x[u][e]);
        a.raise(mn);
        const float m0 = mn == -INFINITY ? 0.f : mn;
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int e = 0; e < VEC<F32>; e++) {
                const float d = x[u][e] - m0, p = ex(d);
                a.s += p;
                a.t = fmaf(fmaxf(d, -1e30f), p, a.t);
            }
    }
    const bool want_top = g.top_ids || g.top_logp;
    const int per = NT / g.group;
    uint32_t big = 0;
    if (want_top) {
        float mx = a.m;
        for (int o = 1; o < g.group; o <<= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
        big = order_of(mx);
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) a.add({__shfl_xor(a.m, o, 64), __shfl_xor(a.s, o, 64), __shfl_xor(a.t, o, 64)});
    if (lane == 0) sh.sums[w] = a;
    __syncthreads();
    a = sh.sums[0];
#pragma unroll
    for (int i = 1; i < WAVES; i++) a.add(sh.sums[i]);
    if (g.parts > 1) {
        const uint32_t each = 4 + per;
        const rsrc_t rp = make_rsrc(g.work + r * (size_t)g.parts * each, (uint32_t)g.parts * each * 4u);
        if (tid == 0) buf_store16(rp, f4{a.m, a.s, a.t, 0.f}, (uint32_t)part * each * 4u);
        if (want_top && tid % g.group == 0)
            __builtin_amdgcn_raw_buffer_store_b32(big, rp, ((uint32_t)part * each + 4 + tid / g.group) * 4u, 0u, CPOL_SC1);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (tid == 0) {
            sh.last = atomicAdd(&g.counters[r], 1) == g.parts - 1;
            if (sh.last) atomicExch(&g.counters[r], 0);
        }
        __syncthreads();
        if (!sh.last) return;
        // a part a lane, in either half of every wave and in one order
        const int mine = lane % MAX_PARTS;
        const f4 o = buf_load16_sc1(rp, (uint32_t)std::min(mine, g.parts - 1) * each * 4u, 0);
        if (want_top && tid < g.parts * per)
            sh.bucket[tid] = __builtin_amdgcn_raw_buffer_load_b32(rp, ((uint32_t)(tid / per) * each + 4 + tid % per) * 4u, 0u, CPOL_SC1);
        a = {-INFINITY, 0.f, 0.f};
        if (mine < g.parts) a = {o.x, o.y, o.z};
#pragma unroll
        for (int o = 1; o < MAX_PARTS; o <<= 1) a.add({__shfl_xor(a.m, o, 64), __shfl_xor(a.s, o, 64), __shfl_xor(a.t, o, 64)});
    } else if (want_top && tid % g.group == 0) {
        sh.bucket[tid / g.group] = big;
    }
    // m = +inf: e^(inf - inf) made s NaN; a NaN did too. Nothing but -inf: s = 0, its log -inf.
    const float logs = logf(a.s);
    const bool nothing = a.m == -INFINITY && a.s == 0.f;
    if (g.entropy && tid == 0) g.entropy[r] = nothing ? 0.f : logs - a.t / a.s;
    if (g.logp) {
        if (tid < g.n_ids) g.logp[r * g.n_ids + tid] = asked < g.V ? log_p(x_asked, a.m, logs) : NAN;
        for (int j = tid + NT; j < g.n_ids; j += NT) {
            const uint32_t id = g.ids[r * g.n_ids + j];
            g.logp[r * g.n_ids + j] = id < g.V ? log_p(row.at(id), a.m, logs) : NAN;
        }
    }
    if (!want_top) return;
    __syncthreads();
    top_k<F32>(row, g.parts * per, !(a.s >= 0.f), sh);
    for (int j = tid; j < g.k; j += NT) {
        const unsigned long long key = sh.out[j];
        if (g.top_ids) g.top_ids[r * g.k + j] = ~(uint32_t)key;
        if (g.top_logp) g.top_logp[r * g.k + j] = log_p(from_order((uint32_t)(key >> 32)), a.m, logs);
    }
}

// ------------------------------------------------------------------------------------ beams
// The k best of a group's candidates are among the k likeliest tokens of each of its rows, so each row is read once as above, its
// top k and the logarithm of its sum go to the workspace, and the last workgroup of the group merges the rows: a candidate's place
// is the number of candidates before it, found in every other row by bisection (a row's values fall along its list).
//
// Values of unlike rows are compared, and a beam's tokens are a choice that cannot be taken back, so the sum of a row is kept to
// about 2^-22 of itself: eight exponentials to a 32-bit sum, those to a 64-bit one, an exponent within 2^-22; a value is formed in
// 64 bits. Equal logits of one row compare equal whatever the sum. Threads, waves and parts join by their common maximum first, one
// exponential each, then by sums of what is left: pair by pair, with two exponentials a step, it was 2.5 us more of a chain of 19 steps.
//
// Bound: the bytes of the logits where rows are many: 64 groups of 8 of 151936, fp32 (311 MB), k 16: 69 us, of which the pass over
// them is 55. 16 groups of 8, fp16 (39 MB): 21.6 us; the pass 14 with its launch, the second look 6, the merge 1.4 (as 64-bit values
// in lists; as keys whose values are formed at each comparison 2.4, and with k 64 20 more). One group of 4 of 32000: 12.8 us, a chain of
// launch, loads, two meetings of workgroups and the second look.
struct BeamArgs {
    LpArgs lp;  // its k: places of a row, k or V
    int k;
    const float *score;
    const uint8_t *done;
    uint32_t done_token;
    int n_beams;
    char *rows;        // [rows][row_bytes]: m and the sum (as 64 bits), what the row is; then its k keys
    uint32_t row_bytes;
    int *group_counters;
    float *out_score;
    uint32_t *out_token;
    int32_t *out_beam;
};
enum { BEAM_ROW, BEAM_NONE, BEAM_DONE, BEAM_ODD };  // a row with candidates; none; the one of a done beam; NaN or +inf somewhere

// e^d for d <= 0 to about 2^-23 of itself, NaN for NaN: the exponent as a product and its remainder
DEV float ex_sharp(float d) {
    constexpr float LOG2E_LO = 1.925963033500e-8f, LN2 = 0.69314718055994531f;  // log2 e = LOG2E + LOG2E_LO
    const float c = fmaxf(d, -1e4f), t = c * LOG2E, lo = fmaf(c, LOG2E_LO, fmaf(c, LOG2E, -t));
    const float e = __builtin_amdgcn_exp2f(d * LOG2E);
    return fmaf(e, lo * LN2, e);
}

// s e^m: the sum of the exponentials of some logits, m the largest
struct BeamSum {
    float m;
    double s;
    // of N neighbouring lanes, in an order of its own that is the same in each
    template <int N>
    __device__ __forceinline__ void join() {
        float n = m;
#pragma unroll
        for (int o = 1; o < N; o <<= 1) n = fmaxf(n, __shfl_xor(n, o, 64));
        s = m == -INFINITY ? s : s * (double)ex_sharp(m - n);
#pragma unroll
        for (int o = 1; o < N; o <<= 1) s += __shfl_xor(s, o, 64);
        m = n;
    }
};

// A thread's sum in the pass over a row: 2^(x log2 e - M) with one fused operation an exponent, M = m log2 e - 8 rounded (the same M in
// every exponent, so that its rounding costs nothing; 8 less than the largest exponent, which puts the terms that count on both
// sides of 0, where a rounding of the exponent is 2^-22 at most): with e^(x - m) itself, seven operations, 128 rows of 151936, fp16,
// take 4 us more. Where M's rounding is no longer small or leaves fp32's range
// (|m| of 2^17 or more: no finite fp16 logit, fp32 ones barred with the type's lowest value), e^(x - m).
template <bool F32>
struct BeamPass {
    float m = -INFINITY, M = 0.f;
    double s = 0.0;
    static __device__ __forceinline__ bool far(float m) { return !(fabsf(m) < 0x1p17f); }
    template <int U>
    __device__ __forceinline__ void add(const float (&x)[U][VEC<F32>]) {
        float n = m;
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int e = 0; e < VEC<F32>; e++) n = fmaxf(n, x[u][e]);
        const bool wide = far(n);
        if (n > m) {
            const float N = fmaf(n, LOG2E, -8.f);
            if (!wide && !far(m)) {
                s *= (double)__builtin_amdgcn_exp2f(M - N);
            } else if (m != -INFINITY) {
                s = sum().s * (double)ex_sharp(m - n);
                if (!wide) s *= (double)__builtin_amdgcn_exp2f(fmaf(n, LOG2E, -N));
            }
            m = n, M = N;
        }
        const float n0 = n == -INFINITY ? 0.f : n;
#pragma unroll
        for (int u = 0; u < U; u++) {
            float p = 0.f;
            if (!wide) {
#pragma unroll
                for (int e = 0; e < VEC<F32>; e++) p += __builtin_amdgcn_exp2f(fmaf(x[u][e], LOG2E, -M));
            } else {
#pragma unroll
                for (int e = 0; e < VEC<F32>; e++) p += ex_sharp(x[u][e] - n0);
            }
            s += (double)p;
        }
    }
    __device__ __forceinline__ BeamSum sum() const { return {m, far(m) ? s : s * (double)__builtin_amdgcn_exp2f(fmaf(-m, LOG2E, M))}; }
};

// Lists of a group's k best candidates, best first: values as integers in their order (0: no candidate) and which of the group's
// n_beams * k they are. Two at a time become one, whose places are found by bisection, half the lists from buffer to buffer.
constexpr size_t beam_lists(int n_beams, int k) { return (size_t)(n_beams + (n_beams + 1) / 2) * k * 10; }
DEV unsigned long long order_of(double v) {
    const unsigned long long b = __builtin_bit_cast(unsigned long long, v + 0.0);
    return v == -INFINITY ? 0ull : b >> 63 ? ~b : b | 1ull << 63;
}
DEV float value_of(unsigned long long o) {
    const unsigned long long b = o >> 63 ? o & ~(1ull << 63) : ~o;
    return (float)__builtin_bit_cast(double, b);
}

template <bool F32>
__global__ void __launch_bounds__(NT) k_beam(BeamArgs a) {
    alignas(16) extern __shared__ unsigned long long lds[];  // the row's Shared, then the group's lists
    __shared__ struct {
        float m[WAVES];
        double s[WAVES];
        double logs[HQ_BEAM_MAX];  // of each row of the group: the logarithm of its sum
        float big[HQ_BEAM_MAX], score[HQ_BEAM_MAX];
        int what[HQ_BEAM_MAX], last, odd;
    } top;
    constexpr int U = 2;  // pieces in flight per thread
    const LpArgs &g = a.lp;
    Shared &sh = *(Shared *)lds;
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, k = g.k;
    const size_t r = blockIdx.x / g.parts;
    const int part = blockIdx.x % g.parts;
    const float score = a.score[r];
    int what = a.done && a.done[r] ? BEAM_DONE : BEAM_ROW;
    if (!(score < INFINITY)) what = BEAM_ODD;
    else if (score == -INFINITY) what = BEAM_NONE;
    BeamSum z = {-INFINITY, 0.0};
    if (what != BEAM_ROW) {
        if (part) return;
    } else {
        const char *const start = (const char *)g.x + r * (size_t)g.stride * (F32 ? 4 : 2);
        const uint32_t mis = (uint32_t)((uintptr_t)start & 15u) / (F32 ? 4 : 2);
        const Row<F32> row = {g, start - ((uintptr_t)start & 15u), mis, (mis + g.V + VEC<F32> - 1) / VEC<F32>};
        const uint32_t v0 = (uint32_t)part * g.per, v1 = std::min(v0 + g.per, row.n_pieces);
        BeamPass<F32> pass;
        for (uint32_t v = v0 + tid; v < v1; v += U * NT) {
            float x[U][VEC<F32>];
#pragma unroll
            for (int u = 0; u < U; u++) {
                if (v + u * NT < v1) piece<F32>(row.base, v + u * NT, row.n_pieces, mis, g.V, x[u]);
                else
#pragma unroll
                    for (int e = 0; e < VEC<F32>; e++) x[u][e] = -INFINITY;
            }
            pass.add(x);
        }
        z = pass.sum();
        const int per = NT / g.group;
        float mx = z.m;
        for (int o = 1; o < g.group; o <<= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
        const uint32_t big = order_of(mx);
        z.join<64>();
        if (lane == 0) top.m[w] = z.m, top.s[w] = z.s;
        __syncthreads();
        z = {top.m[lane % WAVES], top.s[lane % WAVES]};
        z.join<WAVES>();
        if (g.parts > 1) {
            const uint32_t each = 4 + per;
            const rsrc_t rp = make_rsrc(g.work + r * (size_t)g.parts * each, (uint32_t)g.parts * each * 4u);
            const unsigned long long bits = __builtin_bit_cast(unsigned long long, z.s);
            if (tid == 0) buf_store16(rp, f4{z.m, __builtin_bit_cast(float, (uint32_t)bits), __builtin_bit_cast(float, (uint32_t)(bits >> 32)), 0.f}, (uint32_t)part * each * 4u);
            if (tid % g.group == 0) __builtin_amdgcn_raw_buffer_store_b32(big, rp, ((uint32_t)part * each + 4 + tid / g.group) * 4u, 0u, CPOL_SC1);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            if (tid == 0) {
                top.last = atomicAdd(&g.counters[r], 1) == g.parts - 1;
                if (top.last) atomicExch(&g.counters[r], 0);
            }
            __syncthreads();
            if (!top.last) return;
            const int mine = lane % MAX_PARTS;  // a part a lane, in one order
            const u4v o = __builtin_bit_cast(u4v, buf_load16_sc1(rp, (uint32_t)std::min(mine, g.parts - 1) * each * 4u, 0));
            if (tid < g.parts * per) sh.bucket[tid] = __builtin_amdgcn_raw_buffer_load_b32(rp, ((uint32_t)(tid / per) * each + 4 + tid % per) * 4u, 0u, CPOL_SC1);
            z = {-INFINITY, 0.0};
            const uint32_t om = o.x;
            if (mine < g.parts) z = {__builtin_bit_cast(float, om), __builtin_bit_cast(double, (unsigned long long)o.z << 32 | o.y)};
            z.join<MAX_PARTS>();
        } else if (tid % g.group == 0) {
            sh.bucket[tid / g.group] = big;
        }
        __syncthreads();
        if (!(z.s >= 0.0)) what = BEAM_ODD;
        else if (z.s == 0.0) what = BEAM_NONE;
        else top_k<F32>(row, g.parts * per, false, sh);
    }
    // the row to the workspace; the last one of the group goes on
    const size_t group = r / a.n_beams;
    const rsrc_t rr = make_rsrc(a.rows + group * (size_t)a.n_beams * a.row_bytes, (uint32_t)a.n_beams * a.row_bytes);
    const uint32_t mine = (uint32_t)(r - group * a.n_beams) * a.row_bytes;
    if (tid == 0) {
        const unsigned long long bits = __builtin_bit_cast(unsigned long long, z.s);
        buf_store16(rr, f4{z.m, __builtin_bit_cast(float, (uint32_t)bits), __builtin_bit_cast(float, (uint32_t)(bits >> 32)), __builtin_bit_cast(float, what)}, mine);
    }
    if (what == BEAM_ROW)
        for (int j = tid; j < 2 * k; j += NT) {
            const unsigned long long key = sh.out[j / 2];
            __builtin_amdgcn_raw_buffer_store_b32((uint32_t)(j & 1 ? key >> 32 : key), rr, mine + 16u + 4u * (uint32_t)j, 0u, CPOL_SC1);
        }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tid == 0) {
        top.last = atomicAdd(&a.group_counters[group], 1) == a.n_beams - 1;
        if (top.last) atomicExch(&a.group_counters[group], 0);
    }
    __syncthreads();
    if (!top.last) return;
    const int B = a.n_beams, L = a.k;
    unsigned long long *val = lds, *val2 = lds + B * L;
    uint16_t *which = (uint16_t *)(val2 + (B + 1) / 2 * L), *which2 = which + B * L;
    if (tid == 0) top.odd = 0;
    __syncthreads();
    if (tid < B) {
        const u4v o = __builtin_bit_cast(u4v, buf_load16_sc1(rr, (uint32_t)tid * a.row_bytes, 0));
        const uint32_t om = o.x, kind = o.w;
        top.big[tid] = __builtin_bit_cast(float, om);
        top.logs[tid] = log(__builtin_bit_cast(double, (unsigned long long)o.z << 32 | o.y));
        top.score[tid] = a.score[group * B + tid];
        top.what[tid] = (int)kind;
        if ((int)kind == BEAM_ODD) top.odd = 1;
    }
    __syncthreads();
    const size_t to = group * (size_t)L;
    if (top.odd) {
        for (int j = tid; j < L; j += NT) a.out_score[to + j] = NAN, a.out_token[to + j] = 0xffffffffu, a.out_beam[to + j] = -1;
        return;
    }
    for (int i = tid; i < B * L; i += NT) {
        const int b = i / L, j = i - b * L, kind = top.what[b];
        double v = -INFINITY;
        if (kind == BEAM_DONE) {
            if (j == 0) v = (double)top.score[b];
        } else if (kind == BEAM_ROW && j < k) {
            const float x = from_order(__builtin_amdgcn_raw_buffer_load_b32(rr, (uint32_t)b * a.row_bytes + 20u + 8u * (uint32_t)j, 0u, CPOL_SC1));
            if (x != -INFINITY) v = (double)top.score[b] + (((double)x - (double)top.big[b]) - top.logs[b]);
        }
        val[i] = order_of(v), which[i] = (uint16_t)i;
    }
    __syncthreads();
    for (int n = B; n > 1; n = (n + 1) / 2) {
        for (int i = tid; i < n * L; i += NT) {
            const int l = i / L, j = i - l * L, other = l ^ 1;
            const unsigned long long v = val[i];
            int at = j;
            if (other < n) {
                const unsigned long long *const y = val + other * L, least = v + (l & 1 ? 0 : 1);  // those that come before: of a lower beam equal ones too
                int lo = 0, hi = L;
                while (lo < hi) {
                    const int mid = (lo + hi) / 2;
                    if (y[mid] >= least) lo = mid + 1;
                    else hi = mid;
                }
                at += lo;
            }
            if (at < L) val2[l / 2 * L + at] = v, which2[l / 2 * L + at] = which[i];
        }
        __syncthreads();
        unsigned long long *const v = val;
        uint16_t *const w = which;
        val = val2, val2 = v, which = which2, which2 = w;
    }
    for (int j = tid; j < L; j += NT) {
        const unsigned long long v = val[j];
        const int b = v ? which[j] / L : -1;
        uint32_t token = 0xffffffffu;
        if (v) token = top.what[b] == BEAM_DONE ? a.done_token : ~__builtin_amdgcn_raw_buffer_load_b32(rr, (uint32_t)b * a.row_bytes + 16u + 8u * (uint32_t)(which[j] - b * L), 0u, CPOL_SC1);
        a.out_score[to + j] = v ? value_of(v) : -INFINITY, a.out_token[to + j] = token, a.out_beam[to + j] = b;
    }
}

__global__ void k_zero(int *p, int n) {
    for (int i = blockIdx.x * 256 + threadIdx.x; i < n; i += gridDim.x * 256) p[i] = 0;
}

// Few rows: parts of three pieces a thread, while the chip has workgroups to spare (two per CU); 16 rows of 151936 with two: 1.9
// us more, with four 0.3 more. Buckets stay within MAX_BUCKETS: more parts, more threads to a bucket.
void split_rows(LpArgs *g, int M, bool f32, int n_cu) {
    const uint32_t pieces = (g->V + (f32 ? 3u : 7u)) / (f32 ? 4u : 8u) + 1;
    g->parts = (int)std::max(1u, std::min({2u * (uint32_t)n_cu / (uint32_t)M, (pieces + 3 * NT - 1) / (3 * NT), (uint32_t)MAX_PARTS}));
    while (g->parts * (NT / g->group) > MAX_BUCKETS) g->group *= 2;
    g->per = (pieces + (uint32_t)g->parts - 1) / (uint32_t)g->parts;
}

// Rows of a launch, which has fewer than 2^32 threads: half of what 512 a row leave. (Rows that are split are far fewer.)
constexpr int LAUNCH_ROWS = 1 << 22;

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
    LpArgs g = {logits, ids, logp, entropy, top_logp, top_ids, stride, V, n_ids, top_k, 1, 1, 0, nullptr, nullptr};
    int device, n_cu;
    if (hq_internal_device(&device, &n_cu)) return -1;
    split_rows(&g, M, f32, n_cu);
    if (g.parts > 1) {
        const size_t each = 4 + NT / (size_t)g.group, sums = (size_t)M * g.parts * each * 4;
        void *work, *cnt;
        size_t grew;
        if (hq_internal_staging(device, stream, HQ_STAGE_LOGPROBS, sums, &work, &grew) ||
            hq_internal_staging(device, stream, HQ_STAGE_LOGPROBS_COUNT, (size_t)M * 4, &cnt, &grew))
            return -1;
        if (grew) {
            k_zero<<<(unsigned)std::min<size_t>(grew / 1024, 1024), 256, 0, (hipStream_t)stream>>>((int *)cnt, (int)(grew / 4));
            SCK(hipGetLastError());
        }
        g.work = (float *)work, g.counters = (int *)cnt;
    }
    for (int r = 0; r < M; r += LAUNCH_ROWS) {
        const size_t at = (size_t)r;
        LpArgs l = g;
        l.x = (const char *)logits + at * (size_t)stride * (f32 ? 4 : 2);
        if (logp) l.ids = ids + at * n_ids, l.logp = logp + at * n_ids;
        if (entropy) l.entropy = entropy + at;
        if (top_ids) l.top_ids = top_ids + at * top_k;
        if (top_logp) l.top_logp = top_logp + at * top_k;
        const unsigned grid = (unsigned)std::min(LAUNCH_ROWS, M - r) * (unsigned)g.parts;
        if (f32) k_logprobs<true><<<grid, NT, 0, (hipStream_t)stream>>>(l);
        else k_logprobs<false><<<grid, NT, 0, (hipStream_t)stream>>>(l);
        SCK(hipGetLastError());
    }
    return 0;
}

extern "C" int hq_beam(const void *logits, int f32, int n_groups, int n_beams, uint32_t V, int64_t stride, const float *score, const uint8_t *done,
                       uint32_t done_token, int k, float *out_score, uint32_t *out_token, int32_t *out_beam, void *stream) {
    const char *const who = "hq_beam";
    if (n_beams < 1 || n_beams > HQ_BEAM_MAX || n_groups < 0 || n_groups > (1 << 24) / n_beams)
        return hq_internal_fail("%s: %d groups of %d beams (1 .. %d beams, at most 2^24 rows)", who, n_groups, n_beams, HQ_BEAM_MAX);
    if (V < 1 || V > (1u << 30) || stride < (int64_t)V || stride > ((int64_t)1 << 40)) return hq_internal_fail("%s: rows of %u (at most 2^30), stride %lld", who, V, (long long)stride);
    if (k < 1 || k > HQ_BEAM_MAX) return hq_internal_fail("%s: k %d (1 .. %d)", who, k, HQ_BEAM_MAX);
    if (n_groups == 0) return 0;
    if (!logits || !score || !out_score || !out_token || !out_beam) return hq_internal_fail("%s: null argument", who);
    if ((uintptr_t)logits % (f32 ? 4 : 2)) return hq_internal_fail("%s: the logits are misaligned", who);
    for (const void *p : {(const void *)score, (const void *)out_score, (const void *)out_token, (const void *)out_beam})
        if ((uintptr_t)p % 4) return hq_internal_fail("%s: scores and outputs must be 4-byte aligned", who);
    const int M = n_groups * n_beams;
    BeamArgs a = {};
    LpArgs &g = a.lp;
    g.stride = stride, g.V = V, g.k = (int)std::min((uint32_t)k, V), g.parts = g.group = 1;
    int device, n_cu;
    if (hq_internal_device(&device, &n_cu)) return -1;
    split_rows(&g, M, f32, n_cu);
    a.done_token = done_token, a.n_beams = n_beams, a.k = k;
    // the rows' results, and behind them the sums of split rows; counters of rows and groups (of a launch: they follow one another)
    a.row_bytes = 16u + 8u * (uint32_t)((g.k + 1) & ~1);
    const int groups = std::min(n_groups, LAUNCH_ROWS / n_beams), most = groups * n_beams;
    const size_t each = 4 + NT / (size_t)g.group, rows = (size_t)most * a.row_bytes, sums = g.parts > 1 ? (size_t)most * g.parts * each * 4 : 0;
    const int n_count = most + groups;
    void *work, *cnt;
    size_t grew;
    if (hq_internal_staging(device, stream, HQ_STAGE_BEAM, rows + sums, &work, &grew) ||
        hq_internal_staging(device, stream, HQ_STAGE_BEAM_COUNT, (size_t)n_count * 4, &cnt, &grew))
        return -1;
    if (grew) {
        k_zero<<<(unsigned)std::min<size_t>(grew / 1024, 1024), 256, 0, (hipStream_t)stream>>>((int *)cnt, (int)(grew / 4));
        SCK(hipGetLastError());
    }
    a.rows = (char *)work, g.work = (float *)((char *)work + rows);
    a.group_counters = (int *)cnt, g.counters = (int *)cnt + groups;
    const size_t lds = std::max(sizeof(Shared), beam_lists(n_beams, k));
    for (int i = 0; i < n_groups; i += groups) {
        const size_t r = (size_t)i * n_beams, o = (size_t)i * k;
        g.x = (const char *)logits + r * (size_t)stride * (f32 ? 4 : 2);
        a.score = score + r, a.done = done ? done + r : nullptr;
        a.out_score = out_score + o, a.out_token = out_token + o, a.out_beam = out_beam + o;
        const unsigned grid = (unsigned)(std::min(groups, n_groups - i) * n_beams) * (unsigned)g.parts;
        if (f32) k_beam<true><<<grid, NT, lds, (hipStream_t)stream>>>(a);
        else k_beam<false><<<grid, NT, lds, (hipStream_t)stream>>>(a);
        SCK(hipGetLastError());
    }
    return 0;
}
