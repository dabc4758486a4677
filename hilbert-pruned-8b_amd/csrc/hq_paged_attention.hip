// hq_paged_attention.hip - attention of a step's new tokens over the paged cache (hq_attention, include/hq_serve.h).
//
// The queries that share a kv head are one matrix: row r = t rep + e of a sequence is its new token t in query head g rep +
// e of kv head g (rep = heads / kv heads), so grouped heads and neighbouring tokens read each key and value once. hq_batch.hip
// cuts a step into items: a block of rows of one kv head over a range of positions. Two bodies do them:
//   k_rows    blocks of 32 rows per wave: a workgroup's waves share tiles of positions in LDS (prompts, chunks)
//   k_stream  16 or 32 rows: each wave streams tiles of its own straight into operand registers (single tokens)
// Both form everything transposed, so that nothing moves between lanes from scores to outputs: S^T = K Q^T leaves row li in
// every lane and positions in its registers, which is the B operand of O^T = V^T P^T. Both run the online softmax: a running
// maximum and sum per row, outputs scaled when the maximum grows.
//
// Precision: fp16 operands, fp32 products, sums, maxima and outputs. Rounded to 16 bits are the weights p alone: off by 2^-11 of
// each or 2^-31 of the row's largest, whichever is more (LIFT below). Their sum takes them as they are multiplied in k_rows over
// an fp16 cache, before the rounding elsewhere. Of a Q8 cache the operands are exact: keys enter as their codes and the scores take the
// scale in fp32; values enter as code * 2^(e-7), e the exponent of their scale: a normal or subnormal fp16 number, finite and
// exact for every finite scale (2^e itself made infinities of codes from 64 on under scales from 1024 on). The scale's mantissa
// joins the weight before that is rounded, the 2^7 the weights' sum. Decoding to fp16 instead doubled the error of the outputs
// (2.1e-4 -> 4.8e-4).
//
// Places that a row does not see weigh 0, and 0 times an infinity or NaN would be NaN: in a tile that some row sees only part
// of, values that are not finite (`odd` below) enter the product as 0, and are added to the outputs of the rows that do see
// them afterwards.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <math.h>
#include <type_traits>

#include "hq_batch.h"
#include "hq_device.h"

namespace {

typedef float f16v __attribute__((ext_vector_type(16)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef short s4 __attribute__((ext_vector_type(4)));

struct Args {
    hq_kv_t kv;
    hq_attn_t a;
    const HqItem *items;
    const uint32_t *pages;
    float *parts;
    int *counters;
    int nh, rep, shift;  // shift: log2 of the page size
    uint32_t inverse;    // 2^32 / rep, rounded up; 0 for rep = 1
    float sc, slack;     // |scale| log2(e); how far a maximum may grow before the outputs are rescaled (raw scores; Q8: in log2 units)
};

// The new token that row `row0 + local` of an item's block is of (local and the remainder e0 together below 2^16 + 256, rep at
// most 2^15: the product is exact).
DEV int token_of(const Args &g, const HqItem &it, int local) {
    const uint32_t x = (uint32_t)(it.e0 + local);
    return it.t0 + (int)(g.inverse ? __umulhi(x, g.inverse) : x);
}

DEV f16v mfma32(h8 a, h8 b, f16v c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

// the maximum / sum of a lane's value and that of the lane 32 away
DEV float max_halves(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    return fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}
DEV float sum_halves(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    return __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
}
DEV float max_lg(float v) { return max_halves(fmaxf(v, __shfl_xor(v, 16, 64))); }
DEV float sum_lg(float v) { return sum_halves(v + __shfl_xor(v, 16, 64)); }

DEV float ex2(float x) { return __builtin_amdgcn_exp2f(x); }
// Weights are 2^(score - m + LIFT), m a row's maximum when its outputs were last rescaled, at most SLACK below the present one
// (log2 units): up to 2^14, 2^15 with a value scale's mantissa, in fp16. LIFT keeps light weights out of fp16's subnormal range:
// without it those below 2^-25 of the largest are 0, and with many of them so is a part of the answer. A smaller SLACK leaves
// more room for LIFT and rescales more often: packed prompts 626 us with 8 and 6, 634 with 6 and 8, 647 with 4 and 10 (624 with 8
// and 0).
constexpr float SLACK = 8.0f, LIFT = 6.0f;
// m of a row (raw scores; Q8: in log2 units) and what its exponents are taken against. Against a reference past FAR, whose rounding is no small part of a weight's exponent, weights would be infinite or all 0: such
// rows take their scores against m first, and are rescaled at every tile, so that the common case has no test of it.
constexpr float FAR = 4194304.0f;
template <bool Q8>
struct Top {
    float m = -INFINITY, ref = 0.f;
    // the score from which on the row is rescaled
    __device__ __forceinline__ float limit(const Args &g) const { return ref == -LIFT ? -INFINITY : m + g.slack; }
    __device__ __forceinline__ float log2_of(const Args &g, float x) const { return fmaf(x, Q8 ? 1.f : g.sc, -LIFT); }
    // m rises to mn: what the outputs are scaled with; far: scores lose m
    __device__ __forceinline__ float raise(const Args &g, float mn, bool &far) {
        const float from = log2_of(g, m), to = log2_of(g, mn);
        far = fabsf(to) > FAR && mn != -INFINITY;
        const float a = m == -INFINITY ? 0.f : ex2(far ? (m - mn) * (Q8 ? 1.f : g.sc) : from - to);
        m = mn, ref = far ? -LIFT : mn == -INFINITY ? 0.f : to;
        return a;
    }
    // of a part, for part_scale
    __device__ __forceinline__ float part(const Args &g) const { return m == -INFINITY ? -INFINITY : log2_of(g, m); }
};
// 2^(x - m) of a part's maximum x (log2 units) against the row's m; a part that saw nothing has x = -inf
DEV float part_scale(float x, float m) { return x == -INFINITY ? 0.f : ex2(x - m); }

// fp16 pairs of the 16-bit words of x that are infinities or NaN
DEV bool odd2(uint32_t x) { return (x & 0x7c00u) == 0x7c00u || (x & 0x7c000000u) == 0x7c000000u; }
DEV bool odd16(u4v x) { return odd2(x.x) || odd2(x.y) || odd2(x.z) || odd2(x.w); }
DEV bool odd(_Float16 x) { return odd2(__builtin_bit_cast(uint16_t, x)); }
// v with 0 for infinities and NaN; the 0/1 pattern of +inf and NaN (up), of -inf and NaN (down)
DEV h8 finite8(h8 v) {
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = odd(v[e]) ? (_Float16)0.f : v[e];
    return v;
}
DEV u4v finite16(u4v v) { return __builtin_bit_cast(u4v, finite8(__builtin_bit_cast(h8, v))); }
DEV h8 pattern8(h8 v, bool up) {
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = odd(v[e]) && !(up ? v[e] < (_Float16)0.f : v[e] > (_Float16)0.f) ? (_Float16)1.f : (_Float16)0.f;
    return v;
}
// an output that saw `up` and `down` such values (counts)
DEV float add_odd(float o, float up, float down) {
    if (up > 0.f) o += INFINITY;
    if (down > 0.f) o -= INFINITY;
    return o;
}

// Q8 codes as fp16: bytes q ^ 0x80 under 0x64 are 1024 + q + 128
DEV h2 codes2(uint32_t w) {
    const h2 bias = {(_Float16)1152.0f, (_Float16)1152.0f};
    return as_h2(w) - bias;
}
// A value scale as the power of two of its exponent (of fp16's lowest normal one below that) and what remains, fp32 in [1, 2),
// below 1 for subnormal scales; the scale itself and 1 where it is not finite. The power comes 2^-7 smaller: 127 2^8 is the
// largest product with a code, 2^-21 the smallest. Q8_SUM makes up for it in the weights' sum.
constexpr float Q8_SUM = 1.0f / 128.0f;
DEV uint16_t exponent_of(uint32_t d) { return (uint16_t)std::max(d & 0x7c00u, 0x400u); }
DEV uint32_t pow2_of(uint32_t d) {
    const uint16_t small = __builtin_bit_cast(uint16_t, (_Float16)(__builtin_bit_cast(_Float16, exponent_of(d)) * (_Float16)Q8_SUM));
    return (d & 0x7c00u) == 0x7c00u ? d : small;
}
DEV float rest_of(uint32_t d) {
    const uint32_t inverse = 0x7f000000u - __builtin_bit_cast(uint32_t, h2f(exponent_of(d)));  // of 2^k: 2^-k
    return (d & 0x7c00u) == 0x7c00u ? 1.f : h2f((uint16_t)d) * __builtin_bit_cast(float, inverse);
}
// 16 codes times d: a power of two, or 1
DEV void decode16(u4v c, _Float16 d, h8 &lo, h8 &hi) {
    const h2 dd = {d, d};
    h2 o[8];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t w = c[i] ^ 0x80808080u;
        o[2 * i] = codes2(perm_lo(w)) * dd;
        o[2 * i + 1] = codes2(perm_hi(w)) * dd;
    }
    lo = h8{o[0].x, o[0].y, o[1].x, o[1].y, o[2].x, o[2].y, o[3].x, o[3].y};
    hi = h8{o[4].x, o[4].y, o[5].x, o[5].y, o[6].x, o[6].y, o[7].x, o[7].y};
}

// Where row `row0 + local` of an item goes (`is`: there is such a row; else the last one's place, for reading), and its gate.
struct OutRow {
    _Float16 *out;
    const char *gate;
    int hd, gate_f32;
    bool is, padding;
    __device__ __forceinline__ OutRow(const Args &g, const HqItem &it, int local) : hd(g.kv.head_dim), gate_f32(g.a.gate_f32), is(it.row0 + local < it.R) {
        local = std::min(local, it.R - 1 - it.row0);
        const int t = token_of(g, it, local), h = it.kvh * g.rep + it.row0 + local - t * g.rep;
        const size_t tok = (size_t)(it.tok0 + t);
        out = (_Float16 *)g.a.out + tok * g.a.out_stride + (size_t)h * hd;
        gate = (const char *)g.a.gate + (tok * g.a.gate_stride + (size_t)h * g.a.gate_head_stride) * (gate_f32 ? 4 : 2);
        padding = it.base + t < 0;  // before position 0: sees nothing, its sums are 0
    }
    // what the sums are multiplied with, l their weights' sum
    __device__ __forceinline__ float scale(float l) const { return padding ? 0.f : 1.0f / l; }
    // gates of dims d .. d + 3 (past head_dim: others; of padding, whose row may hold anything: 0)
    __device__ __forceinline__ f4 gates(int d) const {
        d = std::min(d, hd - 4);
        f4 x;
        if (gate_f32) {
            x = *(const f4 *)(gate + 4 * d);
        } else {
            const h4 y = *(const h4 *)(gate + 2 * d);
            x = f4{(float)y[0], (float)y[1], (float)y[2], (float)y[3]};
        }
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = padding ? 0.f : x[e];
        return x;
    }
    __device__ __forceinline__ void put(int d, f4 v) const {
        if (is && d < hd) *(h4 *)(out + d) = h4{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
    }
};
DEV f4 gated(f4 v, f4 x) {
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] *= 1.0f / (1.0f + expf(-x[e]));
    return v;
}

// A part's row: its sums [HDP], then (maximum in log2 units, sum). Parts are added in their order, so the result does not
// depend on which came first.
template <int HDP>
constexpr int PARTF = HDP + HQ_PART_EXTRA;

constexpr int JOIN_AT_ONCE = 4;  // parts on their way at a time
// Row `local` of an item from its parts, dims d .. d + 3 of it; load(p, at): 16 bytes at float `at` of part p's row.
template <int HDP, class F>
DEV void join_row(const Args &g, const HqItem &it, int local, int d, F load) {
    constexpr int U = JOIN_AT_ONCE;
    const OutRow out(g, it, local);
    const f4 x = g.a.gate ? out.gates(d) : f4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    f4 v = {0.f, 0.f, 0.f, 0.f};
    for (int p0 = 0; p0 < it.n_parts; p0 += U) {
        f4 y[U], z[U];
#pragma unroll
        for (int e = 0; e < U; e++)
            if (p0 + e < it.n_parts) y[e] = load(p0 + e, d), z[e] = load(p0 + e, HDP);
#pragma unroll
        for (int e = 0; e < U; e++) {
            if (p0 + e >= it.n_parts) continue;
            const float mn = fmaxf(m, z[e].x), a = part_scale(m, mn), b = part_scale(z[e].x, mn);
            v = v * a + y[e] * b;
            l = l * a + z[e].y * b;
            m = mn;
        }
    }
    v *= out.scale(l);
    out.put(d, g.a.gate ? gated(v, x) : v);
}

// Few rows: parts are written and read at device scope, and the last of a block's items to arrive joins them, which is
// quicker than another kernel. The parts' weights first, a part a lane; then the sums, the parts of a row over as many groups
// of threads as there are, so that the chain of reads is short. One token of 2 heads behind 10485 positions, 41 parts a head:
// 28 us reading four parts at a time, 10 us so; of 8 heads behind 1000, 4 parts a head: 6.8 and 7.9 us, so few parts go the
// first way. arena: LDS that the workgroup is done with.
template <int HDP, int ROWS, int NT>
constexpr int JOIN_ARENA = (HQ_STREAM_PARTS + 1) * ROWS + 4 * NT;  // floats
template <int HDP, int ROWS, int NT>
DEV void join_parts(const Args &g, const HqItem &it, rsrc_t rp, int *flag, float *arena) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) {
        const bool last = atomicAdd(&g.counters[it.block], 1) == it.n_parts - 1;
        if (last) atomicExch(&g.counters[it.block], 0);
        *flag = last;
    }
    __syncthreads();
    if (!*flag) return;
    constexpr int C = HDP / 4;
    const int rows = std::min(ROWS, it.R - it.row0);
    if (it.n_parts <= JOIN_AT_ONCE) {  // one round trip, and nothing to share
        for (int x = threadIdx.x; x < rows * C; x += NT) {
            const int row = x / C;
            join_row<HDP>(g, it, row, 4 * (x % C), [&](int p, int f) { return buf_load16_sc1(rp, (uint32_t)((p * ROWS + row) * PARTF<HDP> + f) * 4u, 0); });
        }
        return;
    }
    constexpr int NW = NT / 64, RW = ROWS / NW, PL = HQ_STREAM_PARTS / 64, U = 8;
    float *const weight = arena, *const sum = arena + HQ_STREAM_PARTS * ROWS, *const share = sum + ROWS;  // [part][row], [row], [thread][4]
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    auto at = [&](int part, int row, int f) { return (uint32_t)((part * ROWS + row) * PARTF<HDP> + f) * 4u; };
    f4 z[RW][PL];
#pragma unroll
    for (int u = 0; u < RW; u++)
#pragma unroll
        for (int e = 0; e < PL; e++) {
            const int row = w + NW * u, part = lane + 64 * e;
            z[u][e] = f4{-INFINITY, 0.f, 0.f, 0.f};
            if (row < rows && part < it.n_parts) z[u][e] = buf_load16_sc1(rp, at(part, row, HDP), 0);
        }
#pragma unroll
    for (int u = 0; u < RW; u++) {
        const int row = w + NW * u;
        if (row >= rows) continue;
        float m = -INFINITY, l = 0.f;
#pragma unroll
        for (int e = 0; e < PL; e++) m = fmaxf(m, z[u][e].x);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
#pragma unroll
        for (int e = 0; e < PL; e++) {
            const float x = part_scale(z[u][e].x, m);
            weight[(lane + 64 * e) * ROWS + row] = x;
            l += z[u][e].y * x;
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o, 64);
        if (lane == 0) sum[row] = l;
    }
    __syncthreads();
    int groups = 1;
    while (2 * groups * rows * C <= NT) groups *= 2;
    const int width = NT / groups, group = tid / width;
    for (int s0 = 0; s0 < rows * C; s0 += width) {
        const int slot = s0 + tid % width, row = slot / C, d = 4 * (slot % C);
        const bool on = slot < rows * C;
        const OutRow out(g, it, row);
        const f4 x = g.a.gate ? out.gates(d) : f4{0.f, 0.f, 0.f, 0.f};
        f4 v = {0.f, 0.f, 0.f, 0.f};
        if (on)
            for (int p0 = group; p0 < it.n_parts; p0 += groups * U) {
                f4 y[U];
#pragma unroll
                for (int e = 0; e < U; e++) y[e] = p0 + e * groups < it.n_parts ? buf_load16_sc1(rp, at(p0 + e * groups, row, d), 0) : f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int e = 0; e < U; e++)
                    if (p0 + e * groups < it.n_parts) v += y[e] * weight[(p0 + e * groups) * ROWS + row];
            }
        if (groups > 1) {
            *(f4 *)(share + 4 * tid) = v;
            __syncthreads();
            if (group) return;  // (one pass: the rows' threads fit)
            for (int k = 1; k < groups; k++) v += *(const f4 *)(share + 4 * (tid + k * width));
        }
        if (!on) continue;
        v *= out.scale(sum[row]);
        out.put(d, g.a.gate ? gated(v, x) : v);
    }
}

// Many rows: a kernel behind k_rows, so that the whole chip reads the parts; one workgroup per block did it at a tenth of its
// rate (heads of 256, 2 parts of 128 rows a block: 35 us behind the loop, now 11; 64 blocks of 4 parts of 256 rows, 35 MB: 8 us).
// items: the first part of each block; a workgroup takes JOIN_ROWS rows. Bound: the parts' bytes.
constexpr int JOIN_ROWS = 8;
template <int HDP, int ROWS>
__global__ void __launch_bounds__(256) k_join(Args g) {
    constexpr int C = HDP / 4;
    const HqItem it = g.items[blockIdx.x / (ROWS / JOIN_ROWS)];
    const int first = blockIdx.x % (ROWS / JOIN_ROWS) * JOIN_ROWS;
    const float *const parts = g.parts + (size_t)it.part_at * 4;
    for (int x = threadIdx.x; x < JOIN_ROWS * C; x += 256) {
        const int local = first + x / C, d = 4 * (x % C);
        if (it.row0 + local < it.R) join_row<HDP>(g, it, local, d, [&](int p, int at) { return *(const f4 *)(parts + ((size_t)p * ROWS + local) * PARTF<HDP> + at); });
    }
}

// (through the scalar cache: p is the same in every lane; the table does not change while a kernel runs)
typedef const __attribute__((address_space(4))) uint32_t const_u32;
DEV uint32_t page_of(const Args &g, const HqItem &it, int p) { return ((const_u32 *)(uintptr_t)g.pages)[it.page0 + (p >> g.shift)]; }

// f(0) .. f(N - 1), each index a constant
template <int N, class F>
DEV void unrolled(F f) {
    if constexpr (N > 0) {
        unrolled<N - 1>(f);
        f(std::integral_constant<int, N - 1>());
    }
}

// ------------------------------------------------------------------------------------ rows
// Row pitch of an LDS tile and the XOR of its 16-byte pieces: 16 rows that follow each other put a piece on 16 different
// places of the 256 bytes the LDS reads in a clock (operand K), and four rows put 64 bytes on its four quarters (operand V).
template <int HDP>
constexpr int PITCH = HDP <= 64 ? 128 : HDP <= 128 ? 256 : 512;
template <int HDP>
DEV int swizzle(int row) {
    return HDP <= 64 ? ((row & 2) << 1) | ((row >> 2) & 3) : ((row & 3) << 2) | ((row >> 2) & 3);
}

constexpr int KT = 32;  // positions per tile

DEV const void *uniform(const void *p) {
    const uint64_t x = (uint64_t)p;
    return (const void *)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(x >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)x));
}
// LDS DMA: lane i's 16 (4) bytes at base + off land at lds + 16 i (4 i). Untracked by the compiler, which would otherwise wait
// for all of them before every LDS read: callers wait with wait_dma.
// `lanes`: which take part; as data, so that a conditional load is no branch. Called with all lanes on; m0 is restored.
DEV void dma16_global(const void *base, uint32_t off, uint32_t lds, uint64_t lanes) {
    uint32_t save;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_mov_b64 exec, %4\n\ts_nop 1\n\t"
                 "global_load_lds_dwordx4 %2, %3\n\ts_mov_b64 exec, -1\n\ts_mov_b32 m0, %0"
                 : "=&s"(save)
                 : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(off), "s"(uniform(base)), "s"(lanes)
                 : "memory");
}
DEV void dma4_global(const void *at, uint32_t lds, uint64_t lanes) {
    uint32_t save;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_mov_b64 exec, %3\n\ts_nop 1\n\t"
                 "global_load_lds_dword %2, off\n\ts_mov_b64 exec, -1\n\ts_mov_b32 m0, %0"
                 : "=&s"(save)
                 : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(at), "s"(lanes)
                 : "memory");
}
template <int N>
DEV void wait_dma() { asm volatile("s_waitcnt vmcnt(%0)" ::"i"(N) : "memory"); }
// a workgroup barrier that leaves loads and LDS DMA in flight
DEV void barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Tiles that k_rows keeps in LDS, the ones on their way from memory among them: what fits 160 KB (two workgroups of 4 waves
// per CU for head_dim <= 128, else one).
template <int HDP, bool Q8, int NW>
constexpr int DEPTH = HDP <= 128 && NW == 8 ? 6 : Q8 ? 5 : 4;

// A workgroup of NW waves takes 32 NW rows. Tiles of KT positions come into a ring in LDS by DMA, DEPTH - 2 tiles ahead: the
// time of a tile is shorter than the way from HBM. Every wave multiplies every tile: while it turns the scores of a tile into
// weights (vector instructions), the matrix cores form the scores of the next one. It holds its queries, two S^T [KT x 32] and
// O^T [HDP x 32] in registers; V's operand is read transposed from LDS, its key order that of S^T's registers. Q8 tiles are
// decoded a tile ahead from the ring into two more buffers of each matrix, once for all waves.
// Eight waves of 32 rows, two per SIMD, for heads up to 128: a key is read from LDS once per 32 rows and from the cache once
// per 256. 64 rows per wave spill, and four waves in each of two workgroups read every tile twice (10 % slower). Heads above
// 128 leave room for one wave per SIMD.
// Bound: the matrix products, 4 head_dim per row and position (2 % more for the masked ones), and the power they take. Heads of
// 128: 1800 cycles a tile and SIMD, 1024 of them the matrix cores' (54 % busy with what is around the loop), at 1.7 GHz; without
// the loop's DMA 1730 cycles at 1.6 GHz. What made it 1800 from 2300 is fewer scalar instructions and branches: a SIMD has two
// waves to hide them. Two groups of waves half a tile apart (products of values beside exponentials) or priorities changed
// nothing. 16384 tokens of ten prompts, 32 / 8 heads: 615 us, 850 TFLOP/s; 512 tokens behind 32256: 280 us, 970 TFLOP/s. Heads of
// 256: 2150 cycles, 470 of them the DMA's issue, which no second wave hides; 1000 tokens behind 2001, 16 / 4 heads: 64 us, 640
// TFLOP/s. Over a Q8 cache, which is decoded between barriers and has no loop without tests, the prompts take 764 us, the 512
// tokens 345.
template <int HDP, bool Q8, int NW>
__global__ void __launch_bounds__(64 * NW, HDP > 128 ? 1 : 2) k_rows(Args g) {
    constexpr int P = PITCH<HDP>, T = KT, NJ = HDP / 16, ND = HDP / 32, TILE = T * P, D = DEPTH<HDP, Q8, NW>;
    constexpr int RAWP = Q8 ? P / 2 : P, RAW = T * RAWP;  // a ring tile's pitch and bytes
    constexpr int LPR = RAWP / 16, RPI = 64 / LPR, UNITS = T / RPI, NI = 2 * UNITS > NW ? 2 * UNITS / NW : 1;
    constexpr int LEAD = Q8 ? 2 : 1;  // tile i + LEAD is in LDS when tile i's turn comes
    constexpr int RING = Q8 ? 4 * TILE : 0, SCALES = RING + D * 2 * RAW;  // Q8: K, K, V, V decoded; the ring; its scales
    __shared__ __align__(1024) char lds[SCALES + (Q8 ? D * 128 : 0)];
    __shared__ int found_odd;
    __shared__ __align__(16) float fac[Q8 ? 4 * T : 4];  // Q8, two tiles: what a position's scores take (key scale, score scale); its weight
    const HqItem it = g.items[blockIdx.x];
    if (it.kvh < 0) return;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 31, hf = lane >> 5;
    const int hd = g.kv.head_dim, n = it.n;
    const int r0 = it.row0 + 32 * w, mine = std::min(32 * w + li, it.R - 1 - it.row0);  // (rows past the last: that one again)
    const int n_blk = it.base + it.t0 + 1;  // positions every row of the block sees
    const int end = std::min(it.k1, n), tiles = end > it.k0 ? (end - it.k0 + T - 1) / T : 0;
    const int wn = std::min(end, r0 < it.R ? it.base + token_of(g, it, std::min(32 * w + 31, it.R - 1 - it.row0)) + 1 : 0);
    const int wn_all = it.base + token_of(g, it, 32 * w) + 1, lim = it.base + token_of(g, it, mine) + 1;
    if (threadIdx.x == 0) found_odd = 0;

    // The ring: wave w takes rows RPI NI (w % WM) .. of one matrix, a run within 16 rows and so within a page, 16-byte pieces in
    // NI loads. A piece's place in LDS is the lane's, so the lane takes the piece that belongs there. Pieces past head_dim stay 0.
    constexpr int WM = UNITS / NI;  // waves per matrix
    static_assert(RPI * NI <= 16, "a wave's rows stay in a page");
    const uint32_t at0 = (uint32_t)(uintptr_t)lds;
    const size_t es = Q8 ? 1 : 2;
    const bool loads = w < 2 * WM, values = w >= WM;
    const int row_w = RPI * NI * (w % WM);
    const char *const kv0 = (const char *)(values ? g.kv.v : g.kv.k) + (size_t)it.kvh * g.kv.head_stride * es;
    const size_t page_b = (size_t)g.kv.page_stride * es;
    const uint32_t pos_b = (uint32_t)(g.kv.pos_stride * es), pmask = (uint32_t)g.kv.page_size - 1;
    const uint32_t to_w = at0 + RING + (values ? RAW : 0) + row_w * RAWP;
    uint32_t piece_at[NI];  // byte of the lane's piece in its row
    uint32_t row_at[NI];    // byte of that row in the run
    uint64_t on[NI];        // lanes whose piece is one
#pragma unroll
    for (int x = 0; x < NI; x++) {
        const int row = row_w + RPI * x + lane / LPR, place = lane % LPR, piece = Q8 ? place : place ^ swizzle<HDP>(row);
        on[x] = loads ? __ballot(piece * (Q8 ? 16 : 8) < hd) : 0;
        piece_at[x] = (uint32_t)piece * 16u, row_at[x] = (uint32_t)(row & 15) * pos_b;
    }
    // The wave's rows of a tile in memory: their run of 16, the first byte of its last row that is to be read (behind the last
    // position: that one again, its weight is 0). Lane t holds those of tile 64 c + t (Q8: and the pages of the tile's scales),
    // formed again every 64 tiles. (A scalar load of a page per tile would be waited for at every barrier.)
    uint32_t run_lo = 0, run_hi = 0, run_last = 0, pages[2];
    auto fetch_pages = [&](int i) {
        const int p = it.k0 + (i + lane) * T;
        const int first = std::min(p + (row_w & ~15), (n - 1) & ~15);
        const uint32_t page = g.pages[it.page0 + (first >> g.shift)];
        const uint64_t at = (uint64_t)kv0 + (uint64_t)page * page_b + (uint64_t)((uint32_t)first & pmask) * pos_b;
        run_lo = (uint32_t)at, run_hi = (uint32_t)(at >> 32), run_last = (uint32_t)std::min(n - 1 - first, 15) * pos_b;
        if (Q8)
#pragma unroll
            for (int x = 0; x < 2; x++) pages[x] = g.pages[it.page0 + (std::min(p + 16 * x, n - 1) >> g.shift)];
        asm volatile("" : "+v"(run_lo), "+v"(run_hi), "+v"(run_last));  // here, not where they are used
        if (Q8) asm volatile("" : "+v"(pages[0]), "+v"(pages[1]));
    };
    // (with all lanes on: under a mask the register may be a copy made for the lanes that are on, and lane i's of it anything)
    auto of_tile = [&](uint32_t v, int i) { return (uint32_t)__builtin_amdgcn_readlane((int)v, i & 63); };
    struct Run {
        const char *at;
        uint32_t last;
        bool is;  // there is such a tile
    };
    auto run_of = [&](int i) {
        return Run{(const char *)((uint64_t)of_tile(run_hi, i) << 32 | of_tile(run_lo, i)), of_tile(run_last, i), i < tiles};
    };
    // a tile within `inside` (below): all of its rows are there
    const uint32_t all_rows = 15 * pos_b;
    auto run_inside = [&](int i) { return Run{(const char *)((uint64_t)of_tile(run_hi, i) << 32 | of_tile(run_lo, i)), all_rows, true}; };
    // the load of piece x to `slot`
    auto load_piece = [&](const Run &run, int slot, int x) {
        const uint32_t at = std::min(row_at[x], run.last) + piece_at[x];
        dma16_global(run.at, at, to_w + slot * 2 * RAW + RPI * x * RAWP, run.is ? on[x] : 0);
    };
    auto load_scales = [&](int i, int slot) {
        if (!Q8) return;
        // two positions a lane: lanes 0 .. 15 keys', 16 .. 31 values'; whole runs of 16 (what lies behind the last position is
        // not used)
        const uint32_t p = (uint32_t)(it.k0 + i * T + 2 * (lane & 15));
        const uint32_t low = of_tile(pages[0], i), high = of_tile(pages[1], i), page = lane & 8 ? high : low;
        const uint16_t *const sc = lane & 16 ? g.kv.v_scale : g.kv.k_scale;
        dma4_global(sc + ((size_t)page * g.kv.n_kv_heads + it.kvh) * g.kv.page_size + (p & pmask), at0 + SCALES + slot * 128, w == 0 && i < tiles ? 0xffffffffull : 0);
    };
    // until tile i of the `issued` that are on their way or here is here, at most AFTER tiles behind it
    auto wait_tile = [&](int i, int issued, auto after) {
        constexpr int AFTER = decltype(after)::value;
        if (issued - 1 - i < AFTER) wait_dma<0>();
        else if (Q8 && w == 0) wait_dma<AFTER * (NI + 1)>();
        else wait_dma<AFTER * NI>();
    };
    // Q8: tile i's keys (values) out of the ring, decoded, by the whole workgroup: a piece of 16 codes a thread
    auto decode = [&](int i, bool val) {
        if (i >= tiles) return;
        constexpr int PIECES = T * P / 32;
        const int s0 = it.k0 + i * T, slot = i % D, buf = i & 1;
        const uint16_t *const sc = (const uint16_t *)(lds + SCALES + slot * 128) + (val ? 32 : 0);
        for (int x = threadIdx.x; x < PIECES; x += 64 * NW) {
            const int row = x / LPR, piece = x % LPR;
            const u4v c = *(const u4v *)(lds + RING + slot * 2 * RAW + (val ? RAW : 0) + row * RAWP + piece * 16);
            const uint32_t d = s0 + row < n ? sc[row] : 0u;
            h8 lo, hi;
            decode16(c, val ? __builtin_bit_cast(_Float16, (uint16_t)pow2_of(d)) : (_Float16)1.f, lo, hi);
            if (piece * 16 >= hd) lo = hi = h8{};
            if (piece == 0) fac[(2 * val + buf) * T + row] = val ? rest_of(d) : h2f((uint16_t)d) * g.sc;
            if (val && s0 + T > n_blk && (odd16(__builtin_bit_cast(u4v, lo)) || odd16(__builtin_bit_cast(u4v, hi))))
                lo = finite8(lo), hi = finite8(hi), found_odd = 1;
            char *const to = lds + (2 * val + buf) * TILE + row * P;
            const int at = (2 * piece) ^ swizzle<HDP>(row);
            *(h8 *)(to + at * 16) = lo;
            *(h8 *)(to + (at ^ 1) * 16) = hi;
        }
    };
    // fp16: the odd values of tile i, which some row sees only part of, become 0
    auto look = [&](int i) {
        if (i >= tiles || it.k0 + i * T + T <= n_blk) return;
        for (int x = threadIdx.x; x < TILE / 16; x += 64 * NW) {
            u4v *const at = (u4v *)(lds + (i % D) * 2 * RAW + RAW + x * 16);
            const u4v v = *at;
            if (odd16(v)) *at = finite16(v), found_odd = 1;
        }
    };

    float mx = -INFINITY;                      // of the lane's scores of the tile whose turn it is
    h8 q[NJ];
    Top<Q8> top;
    float limit = -INFINITY, l = 0.f;  // top's limit; the weights' sum
    f16v o[ND], sa, sb;  // outputs; scores of a tile and of the next
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
        for (int e = 0; e < 16; e++) o[d][e] = 0.f;

    const uint32_t kx = at0 + (uint32_t)(li * P + ((hf ^ swizzle<HDP>(li)) << 4));
    const int i16 = lane & 15, vrow = 4 * hf + (i16 >> 2), vc = 2 * ((lane >> 4) & 1) + ((i16 & 3) >> 1);
    const uint32_t vx = at0 + (uint32_t)((Q8 ? 2 * TILE : RAW) + vrow * P + ((vc ^ swizzle<HDP>(vrow)) << 4) + 8 * (i16 & 1));
    typedef __attribute__((address_space(3))) s4 lds_s4;
    typedef const __attribute__((address_space(3))) h8 lds_h8;
    // operands of the tile at `buf` (bytes): its keys by dims 16 j ..; dims 32 d .. by positions 16 k ..
    auto key_operand = [&](uint32_t buf, int j) { return *(lds_h8 *)(uintptr_t)((kx + buf) ^ (32u * j)); };
    auto value_operand = [&](uint32_t buf, int d, int k) {
        const uint32_t x = (vx + buf) ^ (64u * d);
        const h4 a = __builtin_bit_cast(h4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(uintptr_t)(x + 16 * P * k)));
        const h4 c = __builtin_bit_cast(h4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(uintptr_t)((x ^ 32u) + 16 * P * k + 8 * P)));
        return h8{a[0], a[1], a[2], a[3], c[0], c[1], c[2], c[3]};
    };
    // y times the key scales of tile i
    auto scale_scores = [&](f16v &y, int i) {
        if (!Q8) return;
#pragma unroll
        for (int c = 0; c < 4; c++) {
            const f4 f = *(const f4 *)&fac[(i & 1) * T + 8 * c + 4 * hf];
#pragma unroll
            for (int e = 0; e < 4; e++) y[4 * c + e] *= f[e];
        }
    };
    auto zero_scores = [&](f16v &y) {
#pragma unroll
        for (int e = 0; e < 16; e++) y[e] = 0.f;
    };
    static_assert(T == 32, "one block of scores a tile");
    // Scores s of tile i to weights, and its values' product; y: the scores of the tile after it (of whatever the buffer holds,
    // behind the last). k_at, v_at: the next tile's keys and this one's values in LDS. Written out in the
    // order of issue: a score product, its share of the exponentials and a load; then a product of values beside the maxima of
    // the new scores; operands are read AHEAD products before theirs.
    auto step = [&](int i, uint32_t k_at, uint32_t v_at, int to, f16v &s, f16v &y, auto within) {
        constexpr bool INSIDE = decltype(within)::value;
        const int s0 = it.k0 + i * T;
        constexpr int AHEAD = 4;
        h8 kr[AHEAD], vr[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; j++) kr[j] = key_operand(k_at, j);
        if (!INSIDE && s0 + T > wn_all) {
#pragma unroll
            for (int e = 0; e < 16; e++) s[e] = s0 + 8 * (e >> 2) + 4 * hf + (e & 3) < lim ? s[e] : -INFINITY;
            mx = s[0];
#pragma unroll
            for (int e = 1; e < 16; e++) mx = fmaxf(mx, s[e]);
        }
        if (__any(mx > limit)) {
            bool far;
            const float a = top.raise(g, fmaxf(top.m, max_halves(mx)), far);
            limit = top.limit(g);
            if (__any(far))
#pragma unroll
                for (int e = 0; e < 16; e++) s[e] -= far ? top.m : 0.f;
            l *= a;
#pragma unroll
            for (int d = 0; d < ND; d++)
#pragma unroll
                for (int e = 0; e < 16; e++) o[d][e] *= a;
        }
        const Run run = INSIDE ? run_inside(i + D - 1) : run_of(i + D - 1);
        zero_scores(y);
        float x[16];
        h8 p[2];
        f4 f[Q8 ? 4 : 1];
        if (Q8)
#pragma unroll
            for (int c = 0; c < 4; c++) f[c] = *(const f4 *)&fac[(2 + (i & 1)) * T + 8 * c + 4 * hf];
        // weights 2 c and 2 c + 1: their exponentials; later, as fp16 (and summed)
        auto weigh = [&](int c) {
#pragma unroll
            for (int e = 2 * c; e < 2 * c + 2; e++) x[e] = ex2(Q8 ? s[e] - top.ref : fmaf(s[e], g.sc, -top.ref));
        };
        auto round = [&](int c) {
            const int e = 2 * c;
            if (Q8) {
                l += x[e] + x[e + 1];
                x[e] *= f[e / 4][e % 4], x[e + 1] *= f[e / 4][e % 4 + 1];
            }
            const h2 y2 = {(_Float16)x[e], (_Float16)x[e + 1]};
            p[e / 8][e % 8] = y2.x, p[e / 8][e % 8 + 1] = y2.y;
            if (!Q8) l = __builtin_amdgcn_fdot2(y2, h2{(_Float16)1.f, (_Float16)1.f}, l, false);  // (the weights as they are multiplied)
        };
        __builtin_amdgcn_sched_barrier(0);
        unrolled<NJ>([&](auto index) {
            constexpr int j = decltype(index)::value;
            y = mfma32(kr[j % AHEAD], q[j], y);
            if constexpr (j + AHEAD < NJ) kr[j % AHEAD] = key_operand(k_at, j + AHEAD);
            else vr[j + AHEAD - NJ] = value_operand(v_at, (j + AHEAD - NJ) % ND, (j + AHEAD - NJ) / ND);
#pragma unroll
            for (int c = 8 * j / NJ; c < 8 * (j + 1) / NJ; c++) {
                weigh(c);
                if (c) round(c - 1);
            }
#pragma unroll
            for (int x = NI * j / NJ; x < NI * (j + 1) / NJ; x++) load_piece(run, to, x);
            if constexpr (j == NJ - 1) load_scales(i + D - 1, to);
            __builtin_amdgcn_sched_barrier(0);
        });
        round(7);
        float my = -INFINITY;
        unrolled<2 * ND>([&](auto index) {
            constexpr int t = decltype(index)::value, d = t % ND;
            o[d] = mfma32(vr[t % AHEAD], p[t / ND], o[d]);
            if constexpr (t + AHEAD < 2 * ND) vr[t % AHEAD] = value_operand(v_at, (t + AHEAD) % ND, (t + AHEAD) / ND);
            if constexpr (t + 1 == ND) scale_scores(y, i + 1);
            if constexpr (t >= ND)
#pragma unroll
                for (int e = 16 * d / ND; e < 16 * (d + 1) / ND; e++) my = fmaxf(my, y[e]);
            __builtin_amdgcn_sched_barrier(0);
        });
        mx = my;
    };
    if (tiles) {
        if (!Q8 && 2 * hd < P)  // what no load writes: 0, for the products and for look() (decode() writes zeros itself)
            for (int x = threadIdx.x; x < D * 2 * RAW / 16; x += 64 * NW) *(u4v *)(lds + x * 16) = u4v{0, 0, 0, 0};
        fetch_pages(0);
        barrier();
        // the first tiles, then the queries (what waits for the pages must not wait for them), then the rest of the ring
        auto load_tile = [&](int i) {
            const Run run = run_of(i);
#pragma unroll
            for (int x = 0; x < NI; x++) load_piece(run, i, x);
            load_scales(i, i);
        };
#pragma unroll
        for (int i = 0; i < LEAD; i++) load_tile(i);
        {
            const int t = lim - 1 - it.base, h = it.kvh * g.rep + it.row0 + mine - t * g.rep;
            const _Float16 *p = (const _Float16 *)g.a.q + (size_t)(it.tok0 + t) * g.a.q_stride + (size_t)h * hd;
#pragma unroll
            for (int j = 0; j < NJ; j++) {
                const int d = 16 * j + 8 * hf;
                q[j] = d < hd ? *(const h8 *)(p + d) : h8{};
            }
        }
        wait_dma<0>();
#pragma unroll
        for (int i = LEAD; i < D - 1; i++) load_tile(i);
        barrier();
        if constexpr (Q8) {
            decode(0, false), decode(1, false), decode(0, true);
        } else {
            look(0);
        }
        barrier();
        if (g.a.scale < 0.f)
#pragma unroll
            for (int j = 0; j < NJ; j++) q[j] = -q[j];
        zero_scores(sa);
#pragma unroll
        for (int j = 0; j < NJ; j++) sa = mfma32(key_operand(0, j), q[j], sa);
        scale_scores(sa, 0);
#pragma unroll
        for (int e = 0; e < 16; e++) mx = fmaxf(mx, sa[e]);
    }
    int before = D - 1, slot = 0, after = 1;  // of tiles i - 1, i and i + 1
    auto tile = [&](int i, f16v &s, f16v &y, auto within) {
        constexpr bool INSIDE = decltype(within)::value;
        // tile i + LEAD is there, the tiles behind it may still be on their way
        if (INSIDE) wait_dma<(D - 2 - LEAD) * NI>();
        else wait_tile(i + LEAD, std::min(i + D - 1, tiles), std::integral_constant<int, D - 2 - LEAD>());
        barrier();
        if (INSIDE || it.k0 + i * T < wn) {
            if (Q8) step(i, (~i & 1) * TILE, (i & 1) * TILE, before, s, y, within);
            else step(i, after * 2 * RAW, slot * 2 * RAW, before, s, y, within);
        } else {
            const Run run = run_of(i + D - 1);
#pragma unroll
            for (int x = 0; x < NI; x++) load_piece(run, before, x);
            load_scales(i + D - 1, before);
        }
        if (!INSIDE && ((i + D) & 63) == 0) fetch_pages(i + D);
        if constexpr (Q8) decode(i + LEAD, false), decode(i + 1, true);
        else if (!INSIDE) look(i + LEAD);
        before = slot, slot = after, after = __builtin_amdgcn_readfirstlane(after == D - 1 ? 0 : after + 1);
    };
    // Two tiles at a time (their score registers change places). Below `inside` every row sees all of both tiles and of the one
    // that is looked at next, and all that is loaded is there: no test but the maximum's is left. (A wave without rows stays out.
    // Q8: a second copy of its longer loop spills, and waits that count loads would wait for the scratch accesses behind them too.)
    // (Tile i + D, which the second of them loads, is a whole one: behind the last position may stand infinities or NaN, which
    // would send the block through the loop over odd values for nothing.)
    const int inside = !Q8 && r0 < it.R ? std::min((end - it.k0) / T - D, (n_blk - it.k0) / T - 1 - LEAD) : 0;
    for (int i = 0; i < tiles; i += 2) {
        if constexpr (!Q8)
            for (; i < inside && ((i + D) & 63) && ((i + 1 + D) & 63); i += 2) {
                tile(i, sa, sb, std::true_type());
                tile(i + 1, sb, sa, std::true_type());
            }
        tile(i, sa, sb, std::false_type());
        if (i + 1 < tiles) tile(i + 1, sb, sa, std::false_type());
    }
    wait_dma<0>();
    __syncthreads();
    if (found_odd) {
        // the odd values of the tiles that some row sees only part of, position by position
#pragma clang loop unroll(disable)
        for (int at = it.k0 + (std::max(n_blk, it.k0) - it.k0) / T * T; at < wn; at++) {
            const uint32_t page = page_of(g, it, at), in = (uint32_t)at & (uint32_t)(g.kv.page_size - 1);
            const char *const v = (const char *)g.kv.v + ((size_t)it.kvh * (size_t)g.kv.head_stride + (size_t)page * (size_t)g.kv.page_stride + (size_t)in * (size_t)g.kv.pos_stride) * es;
            const _Float16 d8 = Q8 ? __builtin_bit_cast(_Float16, (uint16_t)pow2_of(g.kv.v_scale[((size_t)page * g.kv.n_kv_heads + it.kvh) * g.kv.page_size + in])) : (_Float16)0.f;
#pragma unroll
            for (int d = 0; d < ND; d++)
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const int dim = 32 * d + 8 * c + 4 * hf;
                    h4 x = {};
                    if (dim < hd) {
                        if (Q8) {
                            const uint32_t q4 = *(const uint32_t *)(v + dim);
#pragma unroll
                            for (int e = 0; e < 4; e++) x[e] = (_Float16)(float)(int8_t)byte_of(q4, e) * d8;
                        } else {
                            x = *(const h4 *)(v + 2 * dim);
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float y = (float)x[e], rest = y - fminf(fmaxf(y, -65504.f), 65504.f);  // 0, or what is odd of it
                        o[d][4 * c + e] += at < lim ? rest : 0.f;
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
        }
    }
    const float lt = sum_halves(l) * (Q8 ? Q8_SUM : 1.f);
    if (it.n_parts > 1) {
        float *const to = g.parts + (size_t)it.part_at * 4 + (size_t)(it.part * 32 * NW + 32 * w + li) * PARTF<HDP>;
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int c = 0; c < 4; c++) *(f4 *)(to + 32 * d + 8 * c + 4 * hf) = f4{o[d][4 * c], o[d][4 * c + 1], o[d][4 * c + 2], o[d][4 * c + 3]};
        if (hf == 0) *(f4 *)(to + HDP) = f4{top.part(g), lt, 0.f, 0.f};
        return;
    }
    // outputs through LDS (the ring is done with): 16 bytes a lane, whole rows an instruction
    constexpr int PITCH_O = 2 * HDP + 16, LPO = HDP / 8;
    static_assert(NW * 32 * PITCH_O <= sizeof lds, "the waves' outputs in the ring");
    char *const mem = lds + w * 32 * PITCH_O;
    const OutRow out(g, it, 32 * w + li);
    const float inv = out.scale(lt);
    auto to_lds = [&](auto with) {
        constexpr bool GATED = decltype(with)::value;
#pragma unroll
        for (int d = 0; d < ND; d++) {
            f4 x[4];
            if (GATED)
#pragma unroll
                for (int c = 0; c < 4; c++) x[c] = out.gates(32 * d + 8 * c + 4 * hf);
#pragma unroll
            for (int c = 0; c < 4; c++) {
                f4 v = f4{o[d][4 * c], o[d][4 * c + 1], o[d][4 * c + 2], o[d][4 * c + 3]} * inv;
                if (GATED) v = gated(v, x[c]);
                *(h4 *)(mem + li * PITCH_O + 2 * (32 * d + 8 * c + 4 * hf)) = h4{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
            }
        }
    };
    if (g.a.gate) to_lds(std::true_type());
    else to_lds(std::false_type());
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int i = 0; i < LPO / 2; i++) {
        const int x = lane + 64 * i, row = x / LPO, d = 8 * (x % LPO);
        if (r0 + row >= it.R || d >= hd) continue;
        const int t = token_of(g, it, 32 * w + row), h = it.kvh * g.rep + r0 + row - t * g.rep;
        *(u4v *)((_Float16 *)g.a.out + (size_t)(it.tok0 + t) * g.a.out_stride + (size_t)h * hd + d) = *(const u4v *)(mem + row * PITCH_O + 2 * d);
    }
}

// ------------------------------------------------------------------------------------ stream
// A workgroup of NW waves takes 16 QB rows; the waves take tiles of 32 positions in turn, each with a softmax of its own, and
// the waves' (maximum, sum, output) are added in wave order at the end. A lane (li = lane % 16, lg = lane / 16) loads keys
// straight into the operand (key li, 16 bytes of dims), and of V the DPL dims DPL li .. of the eight positions 4 lg + r and
// 16 + 4 lg + r, which are the positions of its score registers; pairs of positions are put together by v_perm into the
// operand of block b, whose row li is dim DPL li + b. Nothing goes through LDS before the end: few rows use an operand once.
// Bound: the cache's bytes. 64 tokens behind 200 .. 8192 positions, 32 / 8 heads of 128: 113 us, 5.1 TB/s; 8 behind 20000 ..
// 40000 of a Q8 cache: 97 us, 5.0 TB/s. 32 rows of heads of 128 do not fit the registers of two workgroups per CU and spill (412
// bytes a lane, Q8 324): 16 sequences with 5 new tokens each behind 500 .. 8000, 32 / 8 heads: 54 us, Q8 46. A single sequence: the chain of page, keys, softmax and join, 6.8 us behind 1000
// positions (8 heads of 64).
template <int HDP, int QB, int NW>
struct StreamLds {
    float os[NW][16 * QB][HDP + 4], ms[NW][16 * QB], ls[NW][16 * QB];
    int last;
};
template <int HDP, bool Q8, int QB, int NW>
DEV void stream_item(const Args &g, const HqItem &it, StreamLds<HDP, QB, NW> &lds) {
    constexpr int DPL = HDP / 16, NJ = HDP / 32, ROWS = 16 * QB, VW = Q8 ? DPL / 4 : DPL / 2;
    constexpr int KL = Q8 ? HDP / 64 : HDP / 32;  // 16-byte loads of a key
    auto &os = lds.os;
    auto &ms = lds.ms, &ls = lds.ls;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 15, lg = lane >> 4;
    const int hd = g.kv.head_dim;
    const int n = it.n, n_all = it.base + it.t0 + 1;  // positions that some row, that every row sees
    const int end = std::min(it.k1, n);

    h8 q[QB][NJ];
    int lim[QB];
#pragma unroll
    for (int b = 0; b < QB; b++) {
        const int local = std::min(16 * b + li, it.R - 1 - it.row0), t = token_of(g, it, local), h = it.kvh * g.rep + it.row0 + local - t * g.rep;
        lim[b] = it.base + t + 1;
        const _Float16 *p = (const _Float16 *)g.a.q + (size_t)(it.tok0 + t) * g.a.q_stride + (size_t)h * hd;
#pragma unroll
        for (int j = 0; j < NJ; j++) {
            const int d = Q8 ? 64 * (j / 2) + 16 * lg + 8 * (j % 2) : 32 * j + 8 * lg;
            q[b][j] = d < hd ? *(const h8 *)(p + d) : h8{};
            if (g.a.scale < 0.f) q[b][j] = -q[b][j];
        }
    }
    const size_t es = Q8 ? 1 : 2;
    const char *const kb0 = (const char *)g.kv.k + (size_t)it.kvh * g.kv.head_stride * es, *const vb0 = (const char *)g.kv.v + (size_t)it.kvh * g.kv.head_stride * es;
    const uint32_t pos_b = (uint32_t)(g.kv.pos_stride * es), pmask = (uint32_t)g.kv.page_size - 1;
    const size_t page_b = (size_t)g.kv.page_stride * es;

    u4v kf[2][KL];
    uint32_t vf[2][4][VW];
    u2v ksc[2], vsc[2], pow2[2];
    uint32_t pgk[2], pgn[2];  // pages of the tile whose keys are loaded next, of the one whose values are
    auto fetch = [&](int s0, uint32_t (&pg)[2]) {
#pragma unroll
        for (int b = 0; b < 2; b++) pg[b] = page_of(g, it, std::min(s0 + 16 * b, n - 1));
    };
    auto load_k = [&](int s0, const uint32_t (&pg)[2]) {
#pragma unroll
        for (int b = 0; b < 2; b++) {
            const uint32_t in = (uint32_t)std::min(s0 + 16 * b + li, n - 1) & pmask;
            const char *p = kb0 + (size_t)pg[b] * page_b;
#pragma unroll
            for (int j = 0; j < KL; j++) {
                const int d = (Q8 ? 64 * j + 16 * lg : 32 * j + 8 * lg);
                kf[b][j] = d < hd ? *(const u4v *)(p + (in * pos_b + (uint32_t)d * (uint32_t)es)) : u4v{0, 0, 0, 0};
            }
            if (Q8) ksc[b] = *(const u2v *)(g.kv.k_scale + ((size_t)pg[b] * g.kv.n_kv_heads + it.kvh) * g.kv.page_size + ((uint32_t)(s0 + 16 * b + 4 * lg) & pmask));
        }
    };
    auto load_v = [&](int s0, const uint32_t (&pg)[2]) {
#pragma unroll
        for (int b = 0; b < 2; b++) {
            const char *p = vb0 + (size_t)pg[b] * page_b;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const uint32_t in = (uint32_t)std::min(s0 + 16 * b + 4 * lg + r, n - 1) & pmask;
                // dims past head_dim: the last ones again (dropped)
                const int d = std::min(DPL * li, hd - DPL);
                const char *at = p + (in * pos_b + (uint32_t)d * (uint32_t)es);
                if constexpr (VW == 1) vf[b][r][0] = *(const uint32_t *)at;
                else if constexpr (VW == 2) {
                    const u2v x = *(const u2v *)at;
                    vf[b][r][0] = x.x, vf[b][r][1] = x.y;
                } else {
#pragma unroll
                    for (int c = 0; c < VW / 4; c++) {
                        const u4v x = *(const u4v *)(at + 16 * c);
#pragma unroll
                        for (int e = 0; e < 4; e++) vf[b][r][4 * c + e] = x[e];
                    }
                }
            }
            if (Q8) vsc[b] = *(const u2v *)(g.kv.v_scale + ((size_t)pg[b] * g.kv.n_kv_heads + it.kvh) * g.kv.page_size + ((uint32_t)(s0 + 16 * b + 4 * lg) & pmask));
        }
    };

    Top<Q8> top[QB];
    float l[QB];
    f4 o[QB][DPL];
#pragma unroll
    for (int b = 0; b < QB; b++) {
        l[b] = 0.f;
#pragma unroll
        for (int c = 0; c < DPL; c++) o[b][c] = f4{0.f, 0.f, 0.f, 0.f};
    }
    constexpr int STEP = 32 * NW;
    int s0 = it.k0 + 32 * w;
    if (s0 < end) {
        fetch(s0, pgk);
        load_k(s0, pgk);
    }
    for (; s0 < end; s0 += STEP) {
        load_v(s0, pgk);
        if (s0 + STEP < end) fetch(s0 + STEP, pgn);
        f4 s[QB][2];
#pragma unroll
        for (int b = 0; b < QB; b++) s[b][0] = s[b][1] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < NJ; j++)
#pragma unroll
            for (int p = 0; p < 2; p++) {
                h8 kk;
                if (Q8) {
                    const uint32_t w0 = kf[p][j / 2][2 * (j % 2)] ^ 0x80808080u, w1 = kf[p][j / 2][2 * (j % 2) + 1] ^ 0x80808080u;
                    const h2 a0 = codes2(perm_lo(w0)), a1 = codes2(perm_hi(w0)), a2 = codes2(perm_lo(w1)), a3 = codes2(perm_hi(w1));
                    kk = h8{a0.x, a0.y, a1.x, a1.y, a2.x, a2.y, a3.x, a3.y};
                } else {
                    kk = __builtin_bit_cast(h8, kf[p][Q8 ? 0 : j]);
                }
#pragma unroll
                for (int b = 0; b < QB; b++) s[b][p] = mfma(kk, q[b][j], s[b][p]);
            }
        if (Q8) {
#pragma unroll
            for (int p = 0; p < 2; p++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float d = h2f((uint16_t)(ksc[p][r / 2] >> (16 * (r % 2)))) * g.sc;
#pragma unroll
                    for (int b = 0; b < QB; b++) s[b][p][r] *= d;
                }
        }
        if (s0 + STEP < end) load_k(s0 + STEP, pgn);
        const bool cut = s0 + 32 > n_all;  // some row does not see all of the tile
        if (Q8 && s0 + 32 > n) {  // nothing is known of scales behind the last position
#pragma unroll
            for (int p = 0; p < 2; p++)
#pragma unroll
                for (int r = 0; r < 4; r++)
                    if (s0 + 16 * p + 4 * lg + r >= n) vsc[p][r / 2] &= r % 2 ? 0x0000ffffu : 0xffff0000u;
        }
        float rest[2][4];
        if (Q8) {
#pragma unroll
            for (int p = 0; p < 2; p++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const uint32_t d = vsc[p][r / 2] >> (16 * (r % 2)) & 0xffffu;
                    rest[p][r] = rest_of(d);
                    pow2[p][r / 2] = r % 2 ? pow2[p][r / 2] | pow2_of(d) << 16 : pow2_of(d);
                }
        }
        h8 pr[QB];
#pragma unroll
        for (int b = 0; b < QB; b++) {
            if (cut)
#pragma unroll
                for (int p = 0; p < 2; p++)
#pragma unroll
                    for (int r = 0; r < 4; r++) s[b][p][r] = s0 + 16 * p + 4 * lg + r < lim[b] ? s[b][p][r] : -INFINITY;
            float mx = s[b][0][0];
#pragma unroll
            for (int p = 0; p < 2; p++)
#pragma unroll
                for (int r = 0; r < 4; r++) mx = fmaxf(mx, s[b][p][r]);
            if (__any(mx > top[b].limit(g))) {
                bool far;
                const float a = top[b].raise(g, fmaxf(top[b].m, max_lg(mx)), far);
                if (__any(far))
#pragma unroll
                    for (int p = 0; p < 2; p++)
#pragma unroll
                        for (int r = 0; r < 4; r++) s[b][p][r] -= far ? top[b].m : 0.f;
                l[b] *= a;
#pragma unroll
                for (int c = 0; c < DPL; c++) o[b][c] *= a;
            }
#pragma unroll
            for (int p = 0; p < 2; p++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float x = ex2(Q8 ? s[b][p][r] - top[b].ref : fmaf(s[b][p][r], g.sc, -top[b].ref));
                    l[b] += x;
                    pr[b][4 * p + r] = (_Float16)(Q8 ? x * rest[p][r] : x);
                }
        }
        // operand of block c: dim DPL li + c of the eight positions
        auto operand = [&](int c) {
            uint32_t x[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int p = k / 2, r = 2 * (k % 2);
                if (Q8) {
                    // byte c of two positions' words
                    const uint32_t sel = 0x0c000c00u | (uint32_t)((c & 3) + 4) << 16 | (uint32_t)(c & 3);
                    const uint32_t y = __builtin_amdgcn_perm(vf[p][r + 1][c / 4] ^ 0x80808080u, vf[p][r][c / 4] ^ 0x80808080u, sel) | 0x64006400u;
                    x[k] = __builtin_bit_cast(uint32_t, codes2(y) * as_h2(pow2[p][r / 2]));
                } else {
                    x[k] = __builtin_amdgcn_perm(vf[p][r + 1][c / 2], vf[p][r][c / 2], c & 1 ? 0x07060302u : 0x05040100u);
                }
            }
            return __builtin_bit_cast(h8, u4v{x[0], x[1], x[2], x[3]});
        };
        bool bad = false;
        if (cut) {
#pragma unroll
            for (int p = 0; p < 2; p++) {
                // (Q8: values are not finite where their scale is not)
                if (Q8) bad |= odd2(vsc[p].x) || odd2(vsc[p].y);
                else
#pragma unroll
                    for (int r = 0; r < 4; r++)
#pragma unroll
                        for (int c = 0; c < VW; c++) bad |= odd2(vf[p][r][c]);
            }
        }
        if (cut && __any(bad)) {
#pragma unroll
            for (int b = 0; b < QB; b++) {
                h8 seen;
#pragma unroll
                for (int p = 0; p < 2; p++)
#pragma unroll
                    for (int r = 0; r < 4; r++) seen[4 * p + r] = (_Float16)(s0 + 16 * p + 4 * lg + r < lim[b] ? 1.f : 0.f);
#pragma unroll
                for (int c = 0; c < DPL; c++) {
                    const h8 v = operand(c);
                    const f4 zero = {0.f, 0.f, 0.f, 0.f};
                    o[b][c] = mfma(finite8(v), pr[b], o[b][c]);
                    const f4 up = mfma(pattern8(v, true), seen, zero), down = mfma(pattern8(v, false), seen, zero);
#pragma unroll
                    for (int e = 0; e < 4; e++) o[b][c][e] = add_odd(o[b][c][e], up[e], down[e]);
                }
            }
        } else {
#pragma unroll
            for (int c = 0; c < DPL; c++) {
                const h8 v = operand(c);
#pragma unroll
                for (int b = 0; b < QB; b++) o[b][c] = mfma(v, pr[b], o[b][c]);
            }
        }
#pragma unroll
        for (int b = 0; b < 2; b++) pgk[b] = pgn[b];
    }

    // the waves' parts, in wave order
#pragma unroll
    for (int b = 0; b < QB; b++) {
        const float lt = sum_lg(l[b]) * (Q8 ? Q8_SUM : 1.f);
        if (lg == 0) ms[w][16 * b + li] = top[b].part(g), ls[w][16 * b + li] = lt;
    }
    __syncthreads();
#pragma unroll
    for (int b = 0; b < QB; b++) {
        float mm = ms[0][16 * b + li];
#pragma unroll
        for (int v = 1; v < NW; v++) mm = fmaxf(mm, ms[v][16 * b + li]);
        const float f = part_scale(ms[w][16 * b + li], mm);
#pragma unroll
        for (int c = 0; c < DPL; c++) o[b][c] *= f;
    }
    static_assert(NW == 4, "one round of the waves' outputs through LDS");
#pragma unroll
    for (int b = 0; b < QB; b++)
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int c = 0; c < DPL; c += 4)
                *(f4 *)&os[w][16 * b + li][DPL * (4 * lg + r) + c] = f4{o[b][c][r], o[b][c + 1][r], o[b][c + 2][r], o[b][c + 3][r]};
    __syncthreads();
    const rsrc_t rp = make_rsrc(g.parts + (size_t)it.part_at * 4, it.n_parts > 1 ? (uint32_t)it.n_parts * ROWS * PARTF<HDP> * 4u : 0u);
    for (int x = threadIdx.x; x < ROWS * (HDP / 4); x += 64 * NW) {
        const int row = x / (HDP / 4), d = 4 * (x % (HDP / 4));
        f4 v = *(const f4 *)&os[0][row][d];
        float mm = ms[0][row];
#pragma unroll
        for (int u = 1; u < NW; u++) {
            v += *(const f4 *)&os[u][row][d];
            mm = fmaxf(mm, ms[u][row]);
        }
        float lt = 0.f;
#pragma unroll
        for (int u = 0; u < NW; u++) lt += ls[u][row] * part_scale(ms[u][row], mm);
        if (it.n_parts == 1) {
            const OutRow out(g, it, row);
            v *= out.scale(lt);
            out.put(d, g.a.gate ? gated(v, out.gates(d)) : v);
        } else {
            const uint32_t at = (uint32_t)((it.part * ROWS + row) * PARTF<HDP>) * 4u;
            buf_store16(rp, v, at + (uint32_t)d * 4u);
            if (d == 0) buf_store16(rp, f4{mm, lt, 0.f, 0.f}, at + HDP * 4u);
        }
    }
    static_assert(JOIN_ARENA<HDP, ROWS, 64 * NW> * 4 <= sizeof os, "the parts' weights in the waves' arena");
    if (it.n_parts > 1) join_parts<HDP, ROWS, 64 * NW>(g, it, rp, &lds.last, &os[0][0][0]);
}

// QB: the most rows of an item, by 16. Steps that have items of 32 rows do those of 16 in the same kernel: they need no more
// of it, and one behind the other they would each wait for their longest item.
template <int HDP, bool Q8, int QB, int NW>
__global__ void __launch_bounds__(64 * NW, HDP > 128 ? 1 : 2) k_stream(Args g) {
    __shared__ __align__(16) char lds[sizeof(StreamLds<HDP, QB, NW>)];
    const HqItem it = g.items[blockIdx.x];
    if (QB == 1 || it.R <= 16) stream_item<HDP, Q8, 1, NW>(g, it, *(StreamLds<HDP, 1, NW> *)lds);
    else stream_item<HDP, Q8, QB, NW>(g, it, *(StreamLds<HDP, QB, NW> *)lds);
}

template <bool Q8>
hipError_t launch(int body, int width, int stream_rows, Args g, unsigned grid, const HqItem *joins, unsigned n_joins, hipStream_t st) {
#define HQ_STREAMS(H, QB) k_stream<H, Q8, QB, 4><<<grid, 256, 0, st>>>(g)
#define HQ_ROWS(H, NW)                                                                                    \
    do {                                                                                                  \
        k_rows<H, Q8, NW><<<grid, 64 * NW, 0, st>>>(g);                                                   \
        g.items = joins;                                                                                  \
        if (n_joins) k_join<H, 32 * NW><<<n_joins * (32 * NW / JOIN_ROWS), 256, 0, st>>>(g);              \
    } while (0)
    const bool two = stream_rows > 16;
    if (body == HQ_STREAM) {
        if (width == 256) HQ_STREAMS(256, 1);
        else if (width == 128) two ? HQ_STREAMS(128, 2) : HQ_STREAMS(128, 1);
        else two ? HQ_STREAMS(64, 2) : HQ_STREAMS(64, 1);
    } else if (body == HQ_ROWS256) {
        if (width == 128) HQ_ROWS(128, 8);
        else if (width == 96) HQ_ROWS(96, 8);
        else HQ_ROWS(64, 8);
    } else {
        if (width == 256) HQ_ROWS(256, 4);
        else if (width == 192) HQ_ROWS(192, 4);
        else if (width == 128) HQ_ROWS(128, 4);
        else if (width == 96) HQ_ROWS(96, 4);
        else HQ_ROWS(64, 4);
    }
#undef HQ_ROWS
#undef HQ_STREAMS
    return hipGetLastError();
}

}  // namespace

// (a part's row is PARTF<width> floats: its size in the plan and in the kernels comes from this one rule)
int hq_attn_width(int body, int hd) {
    if (body == HQ_STREAM) return hd <= 64 ? 64 : hd <= 128 ? 128 : 256;
    return hd <= 64 ? 64 : hd <= 96 ? 96 : hd <= 128 ? 128 : hd <= 192 ? 192 : 256;
}

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
    if (!(fabsf(a->scale) <= 1e20f)) return hq_internal_fail("%s: scale %g", who, (double)a->scale);
    if (a->gate) {
        if ((uintptr_t)a->gate % (a->gate_f32 ? 16 : 8)) return hq_internal_fail("%s: the gate must be aligned to 4 elements", who);
        if (a->gate_stride < 0 || a->gate_stride > most || a->gate_stride % 4 || a->gate_head_stride < 0 || a->gate_head_stride > most || a->gate_head_stride % 4)
            return hq_internal_fail("%s: gate strides %lld and %lld (multiples of 4)", who, (long long)a->gate_stride, (long long)a->gate_head_stride);
    }
    int cur = -1;
    SCK(hipGetDevice(&cur));
    if (cur != b->device) SCK(hipSetDevice(b->device));
    Args g = {*kv, *a, nullptr, b->pages, b->parts, b->counters, b->n_heads, b->n_heads / kv->n_kv_heads, __builtin_ctz((unsigned)kv->page_size), 0, 0.f, 0.f};
    if (g.rep > 1) g.inverse = (uint32_t)((((uint64_t)1 << 32) + (uint64_t)g.rep - 1) / (uint64_t)g.rep);
    // (a smaller scale leaves every weight alike in fp32; 0 would make NaN of masked scores)
    g.sc = std::max(fabsf(a->scale) * 1.4426950408889634f, 1e-30f);
    g.slack = kv->type == HQ_KV_Q8 ? SLACK : SLACK / g.sc;
    for (int body = 0; body < HQ_BODIES; body++) {
        if (!b->n_items[body]) continue;
        g.items = b->items[body];
        const int width = hq_attn_width(body, kv->head_dim);
        SCK((kv->type == HQ_KV_Q8 ? launch<true> : launch<false>)(body, width, b->stream_rows, g, (unsigned)b->n_items[body], b->joins[body], (unsigned)b->n_joins[body], (hipStream_t)stream));
    }
    return 0;
}
