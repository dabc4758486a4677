// hq_scan.hip - the sequences and states of a step through recurrent layers (hq_scan_*, include/hq_serve.h), and what stands in
// front of their recurrence: causal convolution, norms and gates (hq_delta_append).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <math.h>
#include <new>
#include <string.h>
#include <vector>

#include "hq_device.h"
#include "hq_scan.h"

namespace {

constexpr size_t MOST_WORK = (size_t)640 << 20;  // of the chunks of a pass (their outputs ahead of a norm are beside it, 2.6 times as much at most)

bool aligned(const void *p, size_t a) { return ((uintptr_t)p % a) == 0; }

int use_device(int device) {
    int cur = -1;
    SCK(hipGetDevice(&cur));
    if (cur != device) SCK(hipSetDevice(device));
    return 0;
}

int check_geometry(const char *who, const hq_state_t *st) {
    if (st->n_k_heads < 1 || st->n_k_heads > 1024 || st->n_v_heads < 1 || st->n_v_heads > 1024 || st->n_v_heads % st->n_k_heads)
        return hq_internal_fail("%s: %d value heads over %d key heads (1 .. 1024, a multiple)", who, st->n_v_heads, st->n_k_heads);
    for (int d : {st->k_dim, st->v_dim})
        if (d < 16 || d > 256 || d % 16) return hq_internal_fail("%s: heads of %d and %d (multiples of 16, 16 .. 256)", who, st->k_dim, st->v_dim);
    if (st->conv_taps < 1 || st->conv_taps > 8) return hq_internal_fail("%s: a convolution of %d taps (1 .. 8)", who, st->conv_taps);
    if (st->n_slots < 1 || st->n_slots > 0x7fffffffu) return hq_internal_fail("%s: %u slots", who, st->n_slots);
    return 0;
}

// Few long runs leave most of the chip idle, each a chain of chunks. Cut into parts that fill it, a workgroup a CU, first every part's
// effect on a state is formed (P and Q, all parts side by side, without outputs), then the states between them, then the outputs of all
// parts side by side: two chains of a part's length and a product a part instead of one. It costs two launches, the states' way through
// memory and the products. One sequence, 32 heads of 128, us, in one chain / in parts: 1000 tokens 46.5 / 48.5, 1300 57.5 / 54, 2048 80 / 71, 4096
// 153 / 118, 6001 219 / 161, 16000 562 / 395; 2048 of 8 heads of 128 74 / 54, of 32 heads of 64 67 / 46. JOIN_CHUNKS chunks are more than it
// costs here (some 6), on the side of the one chain.
constexpr int JOIN_CHUNKS = 9, LEAST_PART = 4;
void split_runs(const hq_state_t *st, int n_cu, std::vector<HqPass> *passes, std::vector<HqRun> *runs, std::vector<HqJoin> *joins, int *places) {
    const int cols = hq_scan_columns(st->k_dim);
    const int64_t units = (int64_t)st->n_v_heads * ((st->v_dim + cols - 1) / cols), p_units = (int64_t)st->n_v_heads * ((st->k_dim + cols - 1) / cols);
    std::vector<HqRun> all, parts;
    const auto chunks_of = [](int n) { return (n + HQ_CHUNK - 1) / HQ_CHUNK; };
    for (HqPass &p : *passes) {
        int longest = 0, used = 2;  // (passes follow one another: their parts' places are the same, behind the 2 between passes)
        for (int i = 0; i < p.n_runs; i++) longest = std::max(longest, chunks_of((*runs)[p.run0 + i].n));
        const auto fits = [&](int part) {  // a workgroup a CU
            int64_t outputs = 0, effects = 0, rest = 0;  // (runs shorter than a part: one after another in its time)
            for (int i = 0; i < p.n_runs; i++) {
                const int64_t chunks = chunks_of((*runs)[p.run0 + i].n), n = (chunks + part - 1) / part;
                if (n == 1) rest += chunks;
                else outputs += n * units, effects += (n - 1) * units + (n - 2) * p_units;
            }
            return outputs + (rest + part - 1) / part * units <= n_cu && effects <= n_cu;
        };
        int part = LEAST_PART, above = longest;  // the shortest that fits: `above` does, or is the whole
        while (part < above) {
            const int mid = (part + above) / 2;
            if (fits(mid)) above = mid;
            else part = mid + 1;
        }
        const bool split = longest > 2 * part + JOIN_CHUNKS;
        const int run0 = (int)all.size();
        parts.clear();
        p.join0 = (int)joins->size();
        for (int i = 0; i < p.n_runs; i++) {
            const HqRun r = (*runs)[p.run0 + i];
            const int chunks = chunks_of(r.n), n = split ? (chunks + part - 1) / part : 1;
            if (n == 1) {
                all.push_back(r);
                continue;
            }
            const int each = (chunks + n - 1) / n, m = (chunks + each - 1) / each;  // (m: with parts of one length, as many as there are)
            const int first = used, place = -2 - first;
            used += 2 * m - 2, *places = std::max(*places, used);
            joins->push_back({r.from, first, m});
            for (int j = 0; j < m; j++) {
                HqRun q = {r.tok0 + j * each * HQ_CHUNK, std::min(each * HQ_CHUNK, r.n - j * each * HQ_CHUNK), r.chunk0 + j * each, j ? place - j : r.from == -1 ? -1 : place,
                           j == m - 1 ? r.to : -1};
                all.push_back(q);
                if (j == m - 1) break;
                q.from = j ? -1 : r.from, q.to = place - 1 - j;
                parts.push_back(q);
                if (!j) continue;
                q.from = HQ_IDENTITY, q.to = place - m - j + 1;
                parts.push_back(q);
            }
        }
        p.run0 = run0, p.n_runs = (int)all.size() - run0;
        p.part0 = (int)all.size(), p.n_parts = (int)parts.size();
        all.insert(all.end(), parts.begin(), parts.end());
        p.n_joins = (int)joins->size() - p.join0;
    }
    runs->swap(all);
}

}  // namespace

int hq_state_check(const char *who, const hq_state_t *st, const hq_scan *c) {
    if (check_geometry(who, st)) return -1;
    const hq_state_t &g = c->geom;
    if (st->n_k_heads != g.n_k_heads || st->n_v_heads != g.n_v_heads || st->k_dim != g.k_dim || st->v_dim != g.v_dim ||
        st->conv_taps != g.conv_taps || st->n_slots != g.n_slots)
        return hq_internal_fail("%s: the states (%u slots, %d / %d heads of %d and %d, %d taps) are not those hq_scan_set was given (%u "
                                "slots, %d / %d heads of %d and %d, %d taps)", who, st->n_slots, st->n_k_heads, st->n_v_heads, st->k_dim, st->v_dim,
                                st->conv_taps, g.n_slots, g.n_k_heads, g.n_v_heads, g.k_dim, g.v_dim, g.conv_taps);
    return 0;
}

extern "C" int hq_scan_create(int device, int max_seqs, int max_tokens, hq_scan **out) {
    if (!out) return hq_internal_fail("hq_scan_create: null argument");
    *out = nullptr;
    if (max_seqs < 1 || max_seqs > (1 << 20) || max_tokens < 0 || max_tokens > (1 << 24))
        return hq_internal_fail("hq_scan_create: %d sequences, %d tokens (at least 1, 0; at most 2^20, 2^24)", max_seqs, max_tokens);
    if (use_device(device)) return -1;
    hq_scan *c = new (std::nothrow) hq_scan();
    if (!c) return hq_internal_fail("hq_scan_create: out of memory");
    c->device = device;
    c->max_seqs = max_seqs, c->max_tokens = max_tokens;
    hipError_t e = hipDeviceGetAttribute(&c->n_cu, hipDeviceAttributeMultiprocessorCount, device);
    if (e == hipSuccess) e = hipEventCreateWithFlags(&c->sent, hipEventDisableTiming);
    if (e != hipSuccess) {
        hq_scan_free(c);
        return hq_internal_fail("hq_scan_create: %s", hipGetErrorString(e));
    }
    *out = c;
    return 0;
}

extern "C" void hq_scan_free(hq_scan *c) {
    if (!c) return;
    (void)use_device(c->device);
    (void)hipDeviceSynchronize();
    if (c->dev) (void)hipFree(c->dev);
    if (c->work) (void)hipFree(c->work);
    if (c->host) (void)hipHostFree(c->host);
    if (c->sent) (void)hipEventDestroy(c->sent);
    delete c;
}

extern "C" int hq_scan_set(hq_scan *c, const hq_state_t *st, int n_seqs, const int32_t *n_new, const int32_t *from, const int32_t *to, void *stream) {
    const char *const who = "hq_scan_set";
    if (!c || !st) return hq_internal_fail("%s: null argument", who);
    if (check_geometry(who, st)) return -1;
    if (n_seqs < 0 || n_seqs > c->max_seqs) return hq_internal_fail("%s: %d sequences (the step takes %d)", who, n_seqs, c->max_seqs);
    if (n_seqs && (!n_new || !from || !to)) return hq_internal_fail("%s: null argument", who);
    int64_t T = 0;
    const auto slot = [&](int s) { return s >= -1 && (s < 0 || (uint32_t)s < st->n_slots); };
    for (int i = 0; i < n_seqs; i++) {
        if (n_new[i] < 0) return hq_internal_fail("%s: sequence %d has %d new tokens", who, i, n_new[i]);
        if (!slot(from[i]) || !slot(to[i])) return hq_internal_fail("%s: sequence %d goes from slot %d to slot %d (there are %u)", who, i, from[i], to[i], st->n_slots);
        T += n_new[i];
    }
    if (T > c->max_tokens) return hq_internal_fail("%s: %lld new tokens (the step takes %d)", who, (long long)T, c->max_tokens);
    std::vector<HqTile> tiles;
    std::vector<int> steps;
    std::vector<HqChunk> chunks;
    std::vector<HqRun> runs;
    std::vector<HqPass> passes;
    std::vector<HqJoin> joins;
    // chunks of a pass: what fits MOST_WORK, and 64 at least
    const size_t per_chunk = (size_t)st->n_v_heads * HQ_CHUNK_BYTES;
    const int most_chunks = (int)std::max<size_t>(64, MOST_WORK / per_chunk);
    int places = 0;  // for states
    try {
        // slots that are written: each by one sequence, and read by no other
        std::vector<std::pair<int, int>> w, r;
        for (int i = 0; i < n_seqs; i++) {
            if (to[i] >= 0) w.push_back({to[i], i});
            if (from[i] >= 0) r.push_back({from[i], i});
        }
        std::sort(w.begin(), w.end());
        std::sort(r.begin(), r.end());
        size_t j = 0;
        for (size_t i = 0; i < w.size(); i++) {
            if (i && w[i].first == w[i - 1].first) return hq_internal_fail("%s: sequences %d and %d leave their states in slot %d", who, w[i - 1].second, w[i].second, w[i].first);
            while (j < r.size() && r[j].first < w[i].first) j++;
            for (size_t k = j; k < r.size() && r[k].first == w[i].first; k++)
                if (r[k].second != w[i].second) return hq_internal_fail("%s: sequence %d goes on from slot %d, where sequence %d leaves its state", who, r[k].second, w[i].first, w[i].second);
        }
        std::vector<std::pair<int, int>> long_seqs;
        int64_t all = 0, few = 0;
        int longest = 0;
        for (int i = 0; i < n_seqs; i++) all += n_new[i] > 0, few += n_new[i] > HQ_STEP_BESIDE && n_new[i] <= HQ_STEP_TOKENS, longest = std::max(longest, n_new[i]);
        const int cols = hq_scan_columns(st->k_dim);
        int by_steps = HQ_STEP_TOKENS;
        if (longest > HQ_STEP_ALONE && all * st->n_v_heads * ((st->v_dim + cols - 1) / cols) <= c->n_cu) by_steps = 0;
        else if (longest > HQ_STEP_TOKENS && few * st->n_v_heads <= 4 * c->n_cu) by_steps = HQ_STEP_BESIDE;
        for (int i = 0, tok = 0; i < n_seqs; tok += n_new[i], i++) {
            if (n_new[i] == 0 && (to[i] < 0 || to[i] == from[i])) continue;
            for (int t = 0; t == 0 || t < n_new[i]; t += HQ_CONV_TILE) tiles.push_back({i, t, std::min(HQ_CONV_TILE, n_new[i] - t)});
            if (n_new[i] <= by_steps) {
                steps.push_back(i);
                continue;
            }
            long_seqs.push_back({i, tok});
        }
        for (const auto &l : long_seqs) {
            int from_now = from[l.first];
            for (int t = 0; t < n_new[l.first];) {
                if (passes.empty() || passes.back().n_chunks == most_chunks) passes.push_back({(int)chunks.size(), 0, (int)runs.size(), 0, 0, 0, 0, 0});
                HqPass &p = passes.back();
                const int n = std::min<int64_t>((int64_t)n_new[l.first] - t, (int64_t)(most_chunks - p.n_chunks) * HQ_CHUNK);
                const bool cut = t + n < n_new[l.first];
                const int carry = -2 - (int)(passes.size() & 1);
                runs.push_back({l.second + t, n, p.n_chunks, from_now, cut ? carry : to[l.first]});
                for (int j = 0; j < n; j += HQ_CHUNK) chunks.push_back({l.second + t + j, std::min(HQ_CHUNK, n - j)}), p.n_chunks++;
                p.n_runs++;
                from_now = carry;
                if (cut) places = 2;
                t += n;
            }
        }
        split_runs(st, c->n_cu, &passes, &runs, &joins, &places);
        for (const HqPass &p : passes)
            std::stable_sort(runs.begin() + p.run0, runs.begin() + p.run0 + p.n_runs, [](const HqRun &a, const HqRun &b) { return a.n > b.n; });
        std::stable_sort(steps.begin(), steps.end(), [&](int a, int b) { return n_new[a] > n_new[b]; });
    } catch (const std::exception &) {
        return hq_internal_fail("%s: out of memory", who);
    }
    if (use_device(c->device)) return -1;
    c->set = false;
    if (c->sending) {  // the pinned copy is free again when the last transfer has read it
        SCK(hipEventSynchronize(c->sent));
        c->sending = false;
    }
    const size_t words = (size_t)n_seqs * (sizeof(HqSeq) / 4) + tiles.size() * (sizeof(HqTile) / 4) + steps.size() + chunks.size() * (sizeof(HqChunk) / 4) +
                         runs.size() * (sizeof(HqRun) / 4) + joins.size() * (sizeof(HqJoin) / 4) + 16;
    if (words > c->words) {
        const size_t want = words + words / 2;
        SCK(hipDeviceSynchronize());
        if (c->dev) SCK(hipFree(c->dev));
        c->dev = nullptr;
        if (c->host) SCK(hipHostFree(c->host));
        c->host = nullptr;
        c->words = 0;
        SCK(hipMalloc((void **)&c->dev, want * 4));
        SCK(hipHostMalloc((void **)&c->host, want * 4, hipHostMallocDefault));
        c->words = want;
    }
    size_t most = 0;  // chunks of a pass
    for (const HqPass &p : passes) most = std::max(most, (size_t)p.n_chunks);
    const size_t outs_at = most * per_chunk, places_at = outs_at + most * HQ_CHUNK * (size_t)st->n_v_heads * (size_t)st->v_dim * 4;
    size_t work = places_at;
    work += (size_t)places * st->n_v_heads * st->k_dim * std::max(st->k_dim, st->v_dim) * 4;
    if (work > c->work_bytes) {
        SCK(hipDeviceSynchronize());
        if (c->work) SCK(hipFree(c->work));
        c->work = nullptr;
        c->work_bytes = 0;
        SCK(hipMalloc((void **)&c->work, work));
        c->work_bytes = work;
    }
    int *w = c->host;
    const auto dev = [&]() { return c->dev + (w - c->host); };
    c->seqs = (const HqSeq *)dev();
    for (int i = 0, t = 0; i < n_seqs; t += n_new[i], i++, w += sizeof(HqSeq) / 4) {
        const HqSeq s = {t, n_new[i], from[i], to[i]};
        memcpy(w, &s, sizeof s);
    }
    c->tiles = (const HqTile *)dev(), c->n_tiles = (int)tiles.size();
    if (!tiles.empty()) memcpy(w, tiles.data(), tiles.size() * sizeof(HqTile));
    w += tiles.size() * (sizeof(HqTile) / 4);
    c->steps = dev(), c->n_steps = (int)steps.size(), c->longest_step = steps.empty() ? 0 : n_new[steps[0]];
    if (!steps.empty()) memcpy(w, steps.data(), steps.size() * 4);
    w += steps.size();
    c->chunks = (const HqChunk *)dev();
    if (!chunks.empty()) memcpy(w, chunks.data(), chunks.size() * sizeof(HqChunk));
    w += chunks.size() * (sizeof(HqChunk) / 4);
    c->runs = (const HqRun *)dev();
    if (!runs.empty()) memcpy(w, runs.data(), runs.size() * sizeof(HqRun));
    w += runs.size() * (sizeof(HqRun) / 4);
    c->joins = (const HqJoin *)dev();
    if (!joins.empty()) memcpy(w, joins.data(), joins.size() * sizeof(HqJoin));
    w += joins.size() * (sizeof(HqJoin) / 4);
    c->passes.swap(passes);
    c->outs_at = outs_at, c->places_at = places_at;
    const size_t used = (size_t)(w - c->host);
    if (used) {
        SCK(hipMemcpyAsync(c->dev, c->host, used * 4, hipMemcpyHostToDevice, (hipStream_t)stream));
        SCK(hipEventRecord(c->sent, (hipStream_t)stream));
        c->sending = true;
    }
    c->n_seqs = n_seqs, c->n_tokens = (int)T;
    c->geom = *st;
    c->set = true;
    return 0;
}

// ------------------------------------------------------------------------------------ convolution, norms and gates
namespace {

struct AppendArgs {
    hq_state_t st;
    hq_delta_in_t r;
    const HqSeq *seqs;
    const HqTile *tiles;
};

typedef float f8 __attribute__((ext_vector_type(8)));

template <bool F32>
DEV f8 load8(const void *p, size_t at) {
    if (F32) {
        const f4 a = *(const f4 *)((const float *)p + at), b = *(const f4 *)((const float *)p + at + 4);
        return f8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    }
    const h8 x = *(const h8 *)((const _Float16 *)p + at);
    return f8{(float)x[0], (float)x[1], (float)x[2], (float)x[3], (float)x[4], (float)x[5], (float)x[6], (float)x[7]};
}

template <bool F32>
DEV float load1(const void *p, size_t at) { return F32 ? ((const float *)p)[at] : (float)((const _Float16 *)p)[at]; }

DEV float silu(float z) { return z * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.4426950408889634f)); }  // 2^-22 of itself

// A workgroup takes the heads (of queries, keys, values: one sequence of them) 256 / G blockIdx.y .. of a tile's tokens, G lanes a
// head, eight channels a lane; the last blockIdx.y the tile's gates. A lane holds a window of its channels' last inputs, so that each
// input is read once for a tile and taps - 1 times more at its border, four tokens ahead of its use. The tile with a sequence's first
// token reads the slot's inputs and writes those that the sequence leaves: the same lane the same channels, so one slot may be both.
// TAPS: conv_taps, or with EXACT false more: taps beyond it have no input and no weight.
// Bound: bytes. 2048 tokens of 8192 channels, fp32: 100 MB in 26.5 us, 3.8 TB/s, a few us of them the launch and its ends (57 with a load
// a token waited for, and weights one by one); 16 single tokens 5.1 us, launch and two loads that wait for each other.
template <bool F32, int G, int TAPS, bool EXACT>
__global__ void __launch_bounds__(256) k_delta_append(AppendArgs g) {
    const HqTile tile = g.tiles[blockIdx.x];
    const HqSeq seq = g.seqs[tile.seq];
    const int nk = g.st.n_k_heads, nv = g.st.n_v_heads, dk = g.st.k_dim, dv = g.st.v_dim, taps = EXACT ? TAPS : g.st.conv_taps;
    const size_t channels = 2 * (size_t)nk * dk + (size_t)nv * dv;
    const int tok0 = seq.tok0 + tile.t0;
    if (blockIdx.y == gridDim.y - 1) {
        for (int i = threadIdx.x; i < tile.n * nv; i += 256) {
            const int t = i / nv, h = i - t * nv;
            const size_t at = (size_t)(tok0 + t) * g.r.ab_stride + h, o = (size_t)(tok0 + t) * nv + h;
            const float y = load1<F32>(g.r.a, at) + g.r.dt_bias[h];
            g.r.decay[o] = -expf(g.r.a_log[h]) * (fmaxf(y, 0.f) + log1pf(expf(-fabsf(y))));
            g.r.beta[o] = 1.0f / (1.0f + expf(-load1<F32>(g.r.b, at)));
        }
        return;
    }
    const int u = threadIdx.x % G, j = blockIdx.y * (256 / G) + threadIdx.x / G;
    if (j >= 2 * nk + nv) return;  // (of whole lane groups)
    const bool is_v = j >= 2 * nk;
    const bool on = 8 * u < (is_v ? dv : dk);
    const size_t ch = (is_v ? 2 * (size_t)nk * dk + (size_t)(j - 2 * nk) * dv : (size_t)j * dk) + (on ? 8 * u : 0);
    // the input of token t of the sequence
    const auto input = [&](int t) {
        if (t >= 0) return load8<F32>(g.r.x, (size_t)(seq.tok0 + t) * g.r.x_stride + ch);
        if (seq.from >= 0) return load8<true>(g.st.conv, ((size_t)seq.from * (taps - 1) + (taps - 1 + t)) * channels + ch);
        return f8{};
    };
    f8 x[TAPS - 1 + HQ_CONV_TILE];  // from TAPS - 1 tokens before the tile on
    f8 w[TAPS];                     // of the inputs TAPS - 1 .. 0 tokens back
#pragma unroll
    for (int i = 0; i < TAPS - 1; i++) {
        x[i] = f8{};
        if (i >= TAPS - taps) x[i] = input(tile.t0 - (TAPS - 1) + i);
    }
    constexpr int AHEAD = 4;
    const auto fetch = [&](int t) {
        if (t < tile.n) x[TAPS - 1 + t] = load8<F32>(g.r.x, (size_t)(tok0 + t) * g.r.x_stride + ch);
    };
#pragma unroll
    for (int t = 0; t < AHEAD; t++) fetch(t);
    if (EXACT && TAPS % 4 == 0) {
#pragma unroll
        for (int e = 0; e < 8; e++)
#pragma unroll
            for (int i = 0; i < TAPS; i += 4) {
                const f4 v = *(const f4 *)(g.r.conv_w + (ch + e) * TAPS + i);
#pragma unroll
                for (int r = 0; r < 4; r++)
                    if (i + r < TAPS) w[i + r][e] = v[r];
            }
    } else {
#pragma unroll
        for (int i = 0; i < TAPS; i++)
#pragma unroll
            for (int e = 0; e < 8; e++) w[i][e] = i >= TAPS - taps ? g.r.conv_w[(ch + e) * taps + i - (TAPS - taps)] : 0.f;
    }
    const auto keep = [&](int r, f8 v) {
        f4 *o = (f4 *)(g.st.conv + ((size_t)seq.to * (taps - 1) + r) * channels + ch);
        o[0] = f4{v[0], v[1], v[2], v[3]};
        o[1] = f4{v[4], v[5], v[6], v[7]};
    };
    const bool leaves = tile.t0 == 0 && seq.to >= 0 && on;
    if (leaves && tile.n < seq.n) {
        // the sequence goes on behind the tile: its last taps - 1 inputs are its last tokens' (a tile holds as many)
#pragma unroll
        for (int r = 0; r < TAPS - 1; r++)
            if (r < taps - 1) keep(r, input(seq.n - (taps - 1) + r));
    }
#pragma unroll
    for (int t = 0; t < HQ_CONV_TILE; t++) {
        if (t >= tile.n) break;
        fetch(t + AHEAD < HQ_CONV_TILE ? t + AHEAD : HQ_CONV_TILE);
        f8 y;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < TAPS; i++) s = fmaf(w[i][e], x[t + i][e], s);
            y[e] = silu(s);
        }
        float inv = 1.0f;
        if (!is_v) {  // (not the same for all lanes of a wave, but for those that exchange)
            const auto sum = [&]() {
                float ss = 0.f;
#pragma unroll
                for (int e = 0; e < 8; e++) ss = fmaf(y[e], y[e], ss);
                if (!on) ss = 0.f;
#pragma unroll
                for (int o = G / 2; o > 0; o >>= 1) ss += __shfl_xor(ss, o, 64);
                return ss;
            };
            float ss = sum() + g.r.eps;
            if (!(ss > 1e-30f && ss < INFINITY)) {  // squares beyond fp32's range: of values over a power of two of the largest
                uint32_t m = 0;
#pragma unroll
                for (int e = 0; e < 8; e++) m = max(m, __builtin_bit_cast(uint32_t, fabsf(y[e])));  // (magnitudes: their order as integers)
                if (!on) m = 0;
#pragma unroll
                for (int o = G / 2; o > 0; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o, 64));
                const int to_1 = min(max(127 - (int)(m >> 23), -126), 126);
#pragma unroll
                for (int e = 0; e < 8; e++) y[e] = ldexpf(y[e], to_1);
                ss = sum() + ldexpf(g.r.eps, 2 * to_1);
            }
            inv = 1.0f / sqrtf(ss);
        }
        h8 o;
#pragma unroll
        for (int e = 0; e < 8; e++) o[e] = (_Float16)(y[e] * inv);
        if (on) *(h8 *)((_Float16 *)g.r.qkv + (size_t)(tok0 + t) * channels + ch) = o;
    }
    if (leaves && tile.n == seq.n) {
        // the last taps - 1 of the old inputs and the new ones
#pragma unroll
        for (int n = 0; n <= HQ_CONV_TILE; n++) {
            if (n != tile.n) continue;
#pragma unroll
            for (int r = 0; r < TAPS - 1; r++)
                if (r >= TAPS - taps) keep(r - (TAPS - taps), x[n + r]);
        }
    }
}

}  // namespace

extern "C" int hq_delta_append(const hq_scan *c, const hq_state_t *st, const hq_delta_in_t *r, void *stream) {
    const char *const who = "hq_delta_append";
    if (!c || !st || !r) return hq_internal_fail("%s: null argument", who);
    if (!c->set) return hq_internal_fail("%s: no step is described (hq_scan_set)", who);
    if (hq_state_check(who, st, c)) return -1;
    if (c->n_tiles == 0) return 0;
    if (st->conv_taps > 1 && (!st->conv || !aligned(st->conv, 16))) return hq_internal_fail("%s: 16-byte aligned memory of the convolution's inputs is needed", who);
    if (!r->conv_w || !aligned(r->conv_w, 16)) return hq_internal_fail("%s: 16-byte aligned weights are needed", who);
    if (c->n_tokens) {
        if (!r->x || !r->a || !r->b || !r->a_log || !r->dt_bias || !r->qkv || !r->decay || !r->beta) return hq_internal_fail("%s: null argument", who);
        if (!aligned(r->x, 16) || !aligned(r->qkv, 16)) return hq_internal_fail("%s: x and qkv must be 16-byte aligned", who);
        const size_t size = r->f32 ? 4 : 2;
        if (!aligned(r->a, size) || !aligned(r->b, size) || !aligned(r->a_log, 4) || !aligned(r->dt_bias, 4) || !aligned(r->decay, 4) || !aligned(r->beta, 4))
            return hq_internal_fail("%s: a, b, their parameters or outputs are misaligned", who);
        const int64_t most = (int64_t)1 << 40;
        if (r->x_stride < 0 || r->x_stride > most || r->x_stride % 8 || r->ab_stride < 0 || r->ab_stride > most)
            return hq_internal_fail("%s: strides %lld (a multiple of 8), %lld", who, (long long)r->x_stride, (long long)r->ab_stride);
    }
    if (!(r->eps >= 0.f)) return hq_internal_fail("%s: eps %g", who, (double)r->eps);
    if (use_device(c->device)) return -1;
    const AppendArgs g = {*st, *r, c->seqs, c->tiles};
    const int widest = std::max(st->k_dim, st->v_dim), lanes = widest <= 64 ? 8 : widest <= 128 ? 16 : 32, per = 256 / lanes;
    const int heads = 2 * st->n_k_heads + st->n_v_heads;
    const dim3 grid((unsigned)c->n_tiles, (unsigned)((heads + per - 1) / per) + 1u);
    hipStream_t s = (hipStream_t)stream;
#define HQ_APPEND_G(F, G)                                                            \
    do {                                                                             \
        if (st->conv_taps == 4) k_delta_append<F, G, 4, true><<<grid, 256, 0, s>>>(g); \
        else if (st->conv_taps < 4) k_delta_append<F, G, 4, false><<<grid, 256, 0, s>>>(g); \
        else k_delta_append<F, G, 8, false><<<grid, 256, 0, s>>>(g);                 \
    } while (0)
#define HQ_APPEND(F)                       \
    do {                                   \
        if (lanes == 8) HQ_APPEND_G(F, 8); \
        else if (lanes == 16) HQ_APPEND_G(F, 16); \
        else HQ_APPEND_G(F, 32);           \
    } while (0)
    if (r->f32) HQ_APPEND(true);
    else HQ_APPEND(false);
#undef HQ_APPEND
#undef HQ_APPEND_G
    SCK(hipGetLastError());
    return 0;
}
