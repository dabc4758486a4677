// hq_batch.hip - a serving step's sequences (hq_batch_*, include/hq_serve.h), and the rotary positions and cache append of
// its new tokens.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <math.h>
#include <new>
#include <queue>
#include <string.h>
#include <vector>

#include "hq_batch.h"
#include "hq_device.h"

namespace {

bool aligned(const void *p, size_t a) { return ((uintptr_t)p % a) == 0; }

int use_device(int device) {
    int cur = -1;
    SCK(hipGetDevice(&cur));
    if (cur != device) SCK(hipSetDevice(device));
    return 0;
}

// the geometry alone (hq_batch_set needs no pointers)
int check_geometry(const char *who, const hq_kv_t *kv) {
    if (kv->type != HQ_KV_F16 && kv->type != HQ_KV_Q8) return hq_internal_fail("%s: cache type %d (HQ_KV_F16 = 0, HQ_KV_Q8 = 1)", who, kv->type);
    if (kv->page_size < 16 || kv->page_size > 4096 || (kv->page_size & (kv->page_size - 1)))
        return hq_internal_fail("%s: page_size %d (a power of two, 16 .. 4096)", who, kv->page_size);
    if (kv->head_dim < 16 || kv->head_dim > 256 || kv->head_dim % 16)
        return hq_internal_fail("%s: head_dim %d (a multiple of 16, at most 256)", who, kv->head_dim);
    if (kv->n_kv_heads < 1 || kv->n_kv_heads > 1024) return hq_internal_fail("%s: %d kv heads (1 .. 1024)", who, kv->n_kv_heads);
    if (kv->n_pages < 1 || (uint64_t)kv->n_pages * (uint64_t)kv->page_size >= (1ull << 31))
        return hq_internal_fail("%s: %u pages of %d positions (1 page or more, below 2^31 positions)", who, kv->n_pages, kv->page_size);
    return 0;
}

// ------------------------------------------------------------------------------------ hq_attention's work
struct Block {
    HqItem it;
    int len;   // positions, of its last row
    int rows;  // of its body
};

// Blocks of rows become items (see HqItem). Cutting a long block's positions fills the chip where blocks are few or uneven,
// at the price of a part's way through memory, about `over` positions' time for each item. The length of a piece is the one
// of a few whose items, dealt longest first to `slots` workgroups at a time, end first; none is shorter than `least`.
int piece_length(const std::vector<Block> &bl, int unit, int slots, int over, int least) {
    int64_t total = 0;
    int longest = 0;
    for (const Block &b : bl) total += b.len, longest = std::max(longest, b.len);
    int best = longest;
    double best_end = 1e300;
    std::vector<int> cost;
    for (int f = 0; f <= 4; f++) {
        const int L = f ? (int)std::max<int64_t>((total / (slots * f) + unit - 1) / unit * unit, least) : std::max(longest, unit);
        if (f && L >= longest) continue;
        cost.clear();
        for (const Block &b : bl) {
            const int n = std::max(1, (b.len + L / 2) / L), each = (b.len + n - 1) / n;
            for (int i = 0; i < n; i++) cost.push_back(each + (n > 1 ? 2 * over : over));
        }
        std::sort(cost.begin(), cost.end(), [](int a, int b) { return a > b; });
        std::priority_queue<double, std::vector<double>, std::greater<double>> q;
        for (int i = 0; i < slots; i++) q.push(0);
        double end = 0;
        for (int c : cost) {
            const double e = q.top() + c;
            q.pop(), q.push(e);
            end = std::max(end, e);
        }
        if (end < best_end) best_end = end, best = L;
    }
    return best;
}

struct Plan {
    std::vector<HqItem> items[HQ_BODIES], joins[HQ_BODIES];
    int stream_rows = 16;
    int blocks = 0;          // counters
    uint64_t part_units = 0; // of 16 bytes
};

constexpr int XCDS = 8;

void plan_attention(const hq_kv_t &kv, int n_heads, int n_cu, int n_seqs, const int32_t *n_new, const int32_t *n_pos, Plan *out) {
    const int rep = n_heads / kv.n_kv_heads;
    const auto body_of = [&](int R) { return R <= 16 || (R <= 32 && kv.head_dim <= 128) ? HQ_STREAM : R <= 128 || kv.head_dim > 128 ? HQ_ROWS128 : HQ_ROWS256; };
    // A step with blocks of 256 rows does those of 128 in the same kernel, half its waves idle, while their positions are fewer
    // than the time of a kernel of their own: about 256 positions on every workgroup that would run it.
    int64_t small = 0;
    bool large = false;
    for (int i = 0; i < n_seqs; i++) {
        const int body = body_of(n_new[i] * rep);
        if (body == HQ_ROWS128 && n_new[i]) small += (int64_t)n_pos[i] * kv.n_kv_heads;
        large |= body == HQ_ROWS256;
    }
    const bool together = large && small < 256 * 2 * n_cu;
    std::vector<Block> bl[HQ_BODIES];
    int tok0 = 0, page0 = 0;
    for (int i = 0; i < n_seqs; i++) {
        const int R = n_new[i] * rep, base = n_pos[i] - n_new[i];
        int body = body_of(R);
        if (body == HQ_ROWS128 && together) body = HQ_ROWS256;
        const int rows = body == HQ_ROWS256 ? 256 : body == HQ_ROWS128 ? 128 : R <= 16 ? 16 : 32;
        if (body == HQ_STREAM) out->stream_rows = std::max(out->stream_rows, rows);
        for (int h = 0; h < kv.n_kv_heads && R; h++)
            for (int row0 = (R - 1) / rows * rows; row0 >= 0; row0 -= rows) {
                const int see = base + (std::min(R, row0 + rows) - 1) / rep + 1, n = std::max(0, see);
                bl[body].push_back({{h, tok0, base, R, row0, row0 / rep, row0 % rep, see, 0, n, page0, 0, 1, 0, 0}, n, rows});
            }
        tok0 += n_new[i];
        page0 += (n_pos[i] + kv.page_size - 1) / kv.page_size;
    }
    for (int body = 0; body < HQ_BODIES; body++) {
        if (bl[body].empty()) continue;
        const bool stream = body == HQ_STREAM;
        const int unit = stream ? 128 : 64;
        const int slots = n_cu * (stream || (body == HQ_ROWS128 && kv.head_dim <= 128) ? 2 : 1);  // workgroups at a time
        const int L = piece_length(bl[body], unit, slots, stream ? 128 : 192, 256);
        std::vector<HqItem> all;
        for (const Block &b : bl[body]) {
            const int units = (b.len + unit - 1) / unit, n = std::max(1, std::min({(b.len + L / 2) / L, units, stream ? HQ_STREAM_PARTS : units}));
            HqItem it = b.it;
            it.n_parts = n;
            if (n > 1) {
                if (stream) it.block = out->blocks++;
                it.part_at = (uint32_t)out->part_units;
                out->part_units += (uint64_t)n * b.rows * (hq_attn_width(body, kv.head_dim) + HQ_PART_EXTRA) / 4;
            }
            for (int p = 0; p < n; p++) {
                it.part = p;
                it.k0 = (int)((int64_t)units * p / n) * unit;
                it.k1 = p == n - 1 ? b.len : (int)((int64_t)units * (p + 1) / n) * unit;
                all.push_back(it);
                if (p == 0 && n > 1 && !stream) out->joins[body].push_back(it);
            }
        }
        const auto longer = [](const HqItem &a, const HqItem &b) { return a.k1 - a.k0 > b.k1 - b.k0; };
        std::vector<HqItem> &to = out->items[body];
        if (stream) {
            std::stable_sort(all.begin(), all.end(), longer);
            to = all;
            continue;
        }
        // blocks of one sequence and kv head read the same keys and values: items go to the XCDs (workgroup i runs on XCD
        // i % 8) in eight runs, each longest first: of equal work, or, where every item has a workgroup's place of its own, of
        // equal numbers (30 decoded sequences and a chunk of 1000, 256 items of unlike lengths: 103 -> 77 us then)
        int64_t total = 0, run = 0;
        for (const HqItem &it : all) total += it.k1 - it.k0 + unit;
        std::vector<HqItem> q[XCDS];
        for (size_t i = 0; i < all.size(); i++) {
            const HqItem &it = all[i];
            const int64_t mid = run + (it.k1 - it.k0 + unit) / 2;
            const int64_t to_xcd = (int)all.size() <= slots ? (int64_t)(i * XCDS / all.size()) : mid * XCDS / total;
            q[std::min<int64_t>(to_xcd, XCDS - 1)].push_back(it);
            run += it.k1 - it.k0 + unit;
        }
        size_t most = 0;
        for (auto &v : q) std::stable_sort(v.begin(), v.end(), longer), most = std::max(most, v.size());
        for (size_t j = 0; j < most; j++)
            for (auto &v : q) {
                HqItem none = {};
                none.kvh = -1;
                to.push_back(j < v.size() ? v[j] : none);
            }
    }
}

}  // namespace

int hq_kv_check(const char *who, const hq_kv_t *kv, const hq_batch *b) {
    if (check_geometry(who, kv)) return -1;
    const hq_kv_t &g = b->geom;
    if (kv->type != g.type || kv->page_size != g.page_size || kv->n_kv_heads != g.n_kv_heads || kv->head_dim != g.head_dim || kv->n_pages != g.n_pages)
        return hq_internal_fail("%s: the cache (type %d, %u pages of %d, %d heads of %d) is not the one hq_batch_set was given (type %d, %u "
                                "pages of %d, %d heads of %d)", who, kv->type, kv->n_pages, kv->page_size, kv->n_kv_heads, kv->head_dim, g.type,
                                g.n_pages, g.page_size, g.n_kv_heads, g.head_dim);
    if (!kv->k || !kv->v) return hq_internal_fail("%s: the cache has no memory", who);
    if (!aligned(kv->k, 16) || !aligned(kv->v, 16)) return hq_internal_fail("%s: k and v must be 16-byte aligned", who);
    if (kv->type == HQ_KV_Q8 && (!kv->k_scale || !kv->v_scale || !aligned(kv->k_scale, 16) || !aligned(kv->v_scale, 16)))
        return hq_internal_fail("%s: a Q8 cache needs 16-byte aligned scales", who);
    if (kv->pos_stride >= ((int64_t)1 << 30) / kv->page_size) return hq_internal_fail("%s: a page's positions span 2^30 elements or more", who);
    for (int64_t s : {kv->page_stride, kv->pos_stride, kv->head_stride})
        if (s < 0 || s % 16 || s > ((int64_t)1 << 40)) return hq_internal_fail("%s: cache stride %lld (a multiple of 16)", who, (long long)s);
    return 0;
}

extern "C" int hq_batch_create(int device, int max_seqs, int max_tokens, int max_pages, hq_batch **out) {
    if (!out) return hq_internal_fail("hq_batch_create: null argument");
    *out = nullptr;
    if (max_seqs < 1 || max_seqs > (1 << 20) || max_tokens < 0 || max_tokens > (1 << 24) || max_pages < 0 || max_pages > (1 << 24))
        return hq_internal_fail("hq_batch_create: %d sequences, %d tokens, %d pages per sequence (at least 1, 0, 0; at most 2^20, 2^24, 2^24)",
                                max_seqs, max_tokens, max_pages);
    if (use_device(device)) return -1;
    hq_batch *b = new (std::nothrow) hq_batch();
    if (!b) return hq_internal_fail("hq_batch_create: out of memory");
    b->device = device;
    b->max_seqs = max_seqs, b->max_tokens = max_tokens, b->max_pages = max_pages;
    hipError_t e = hipDeviceGetAttribute(&b->n_cu, hipDeviceAttributeMultiprocessorCount, device);
    if (e == hipSuccess) e = hipEventCreateWithFlags(&b->sent, hipEventDisableTiming);
    if (e != hipSuccess) {
        hq_batch_free(b);
        return hq_internal_fail("hq_batch_create: %s", hipGetErrorString(e));
    }
    *out = b;
    return 0;
}

extern "C" void hq_batch_free(hq_batch *b) {
    if (!b) return;
    (void)use_device(b->device);
    (void)hipDeviceSynchronize();
    if (b->dev) (void)hipFree(b->dev);
    if (b->parts) (void)hipFree(b->parts);
    if (b->host) (void)hipHostFree(b->host);
    if (b->sent) (void)hipEventDestroy(b->sent);
    delete b;
}

extern "C" int hq_batch_set(hq_batch *b, const hq_kv_t *kv, int n_heads, int n_seqs, const int32_t *n_new, const int32_t *n_pos,
                            const uint32_t *pages, int pages_ld, void *stream) {
    const char *const who = "hq_batch_set";
    if (!b || !kv) return hq_internal_fail("%s: null argument", who);
    if (check_geometry(who, kv)) return -1;
    if (n_heads < 1 || n_heads % kv->n_kv_heads || n_heads > 32768)
        return hq_internal_fail("%s: %d heads over %d kv heads", who, n_heads, kv->n_kv_heads);
    if (n_seqs < 0 || n_seqs > b->max_seqs) return hq_internal_fail("%s: %d sequences (the batch takes %d)", who, n_seqs, b->max_seqs);
    if (n_seqs && (!n_new || !n_pos)) return hq_internal_fail("%s: null argument", who);
    const int ps = kv->page_size;
    int64_t T = 0, P = 0;
    for (int i = 0; i < n_seqs; i++) {
        if (n_new[i] < 0 || n_pos[i] < 0 || n_pos[i] > (1 << 28)) return hq_internal_fail("%s: sequence %d has %d new tokens of %d", who, i, n_new[i], n_pos[i]);
        T += n_new[i];
        const int64_t need = ((int64_t)n_pos[i] + ps - 1) / ps;
        if (need > b->max_pages) return hq_internal_fail("%s: sequence %d needs %lld pages (the batch takes %d)", who, i, (long long)need, b->max_pages);
        if (need > pages_ld || (need && !pages)) return hq_internal_fail("%s: sequence %d needs %lld pages, its row of the table has %d", who, i, (long long)need, pages ? pages_ld : 0);
        for (int64_t p = 0; p < need; p++)
            if (pages[(size_t)i * (size_t)pages_ld + (size_t)p] >= kv->n_pages)
                return hq_internal_fail("%s: page %lld of sequence %d is %u (the cache has %u)", who, (long long)p, i, pages[(size_t)i * (size_t)pages_ld + (size_t)p], kv->n_pages);
        P += need;
    }
    if (T > b->max_tokens) return hq_internal_fail("%s: %lld new tokens (the batch takes %d)", who, (long long)T, b->max_tokens);
    if (T * n_heads >= (1ll << 31)) return hq_internal_fail("%s: %lld tokens of %d heads", who, (long long)T, n_heads);
    if (P >= (1ll << 30)) return hq_internal_fail("%s: %lld pages in all", who, (long long)P);
    if (use_device(b->device)) return -1;
    b->set = false;
    if (b->sending) {  // the pinned copy is free again when the last transfer has read it
        SCK(hipEventSynchronize(b->sent));
        b->sending = false;
    }
    Plan plan;
    try {
        plan_attention(*kv, n_heads, b->n_cu, n_seqs, n_new, n_pos, &plan);
    } catch (const std::exception &) {
        return hq_internal_fail("%s: out of memory", who);
    }
    if (plan.part_units >> 32) return hq_internal_fail("%s: %llu MiB of workspace", who, (unsigned long long)(plan.part_units >> 16));
    size_t n_items = 0;
    for (int i = 0; i < HQ_BODIES; i++) n_items += plan.items[i].size() + plan.joins[i].size();
    const size_t words = n_items * (sizeof(HqItem) / 4) + 2 * (size_t)T + (size_t)plan.blocks + (size_t)P + 16;
    if (words > b->words) {
        const size_t want = std::max(words, words + words / 2);
        SCK(hipDeviceSynchronize());
        if (b->dev) SCK(hipFree(b->dev));
        b->dev = nullptr;
        if (b->host) SCK(hipHostFree(b->host));
        b->host = nullptr;
        b->words = 0;
        SCK(hipMalloc((void **)&b->dev, want * 4));
        SCK(hipHostMalloc((void **)&b->host, want * 4, hipHostMallocDefault));
        b->words = want;
    }
    if (plan.part_units * 16 > b->part_bytes) {
        SCK(hipDeviceSynchronize());
        if (b->parts) SCK(hipFree(b->parts));
        b->parts = nullptr;
        b->part_bytes = 0;
        SCK(hipMalloc((void **)&b->parts, plan.part_units * 16));
        b->part_bytes = plan.part_units * 16;
    }
    int *w = b->host;
    const auto dev = [&]() { return b->dev + (w - b->host); };
    for (int i = 0; i < HQ_BODIES; i++) {
        const auto send = [&](const std::vector<HqItem> &v, const HqItem **at, int *n) {
            *at = (const HqItem *)dev();
            *n = (int)v.size();
            if (!v.empty()) memcpy(w, v.data(), v.size() * sizeof(HqItem));
            w += v.size() * (sizeof(HqItem) / 4);
        };
        send(plan.items[i], &b->items[i], &b->n_items[i]);
        send(plan.joins[i], &b->joins[i], &b->n_joins[i]);
    }
    b->stream_rows = plan.stream_rows;
    b->counters = dev();
    if (plan.blocks) memset(w, 0, (size_t)plan.blocks * 4);
    w += plan.blocks;
    b->pages = (const uint32_t *)dev();
    for (int i = 0; i < n_seqs; i++) {
        const int need = (n_pos[i] + ps - 1) / ps;
        if (need) memcpy(w, pages + (size_t)i * (size_t)pages_ld, (size_t)need * 4);
        w += need;
    }
    b->tok_pos = dev(), b->tok_slot = b->tok_pos + T;
    int *const slot = w + T;
    for (int i = 0, t = 0; i < n_seqs; i++)
        for (int j = 0; j < n_new[i]; j++, t++) {
            const int p = n_pos[i] - n_new[i] + j;
            w[t] = p;
            slot[t] = p < 0 ? -1 : (int)(pages[(size_t)i * (size_t)pages_ld + (size_t)(p / ps)] * (uint32_t)ps + (uint32_t)(p % ps));
        }
    w = slot + T;
    const size_t used = (size_t)(w - b->host);
    if (used) {
        SCK(hipMemcpyAsync(b->dev, b->host, used * 4, hipMemcpyHostToDevice, (hipStream_t)stream));
        SCK(hipEventRecord(b->sent, (hipStream_t)stream));
        b->sending = true;
    }
    b->n_seqs = n_seqs, b->n_tokens = (int)T, b->n_heads = n_heads;
    b->geom = *kv;
    b->set = true;
    return 0;
}

// ------------------------------------------------------------------------------------ rotary positions
namespace {

__global__ void __launch_bounds__(256) k_rope_table(const float *__restrict__ inv_freq, int half, int n, float *__restrict__ out) {
    for (size_t i = blockIdx.x * (size_t)256 + threadIdx.x; i < (size_t)n * half; i += (size_t)gridDim.x * 256) {
        const double a = (double)(i / half) * (double)inv_freq[i % half];
        out[2 * i] = (float)cos(a);
        out[2 * i + 1] = (float)sin(a);
    }
}

struct RopeArgs {
    hq_kv_t kv;
    hq_rope_t r;
    const int *tok_pos, *tok_slot;
    int nh, n_tokens, first;  // first: of the launch's tokens
    uint8_t axis[128];  // of each frequency
};

typedef float f2 __attribute__((ext_vector_type(2)));

template <bool F32>
DEV f4 load4(const void *p, size_t at) {
    if (F32) return *(const f4 *)((const float *)p + at);
    const h4 x = *(const h4 *)((const _Float16 *)p + at);
    return f4{(float)x[0], (float)x[1], (float)x[2], (float)x[3]};
}

DEV void store4(_Float16 *p, f4 x) { *(h4 *)p = h4{(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3]}; }

// x' = x c - y s, y' = y c + x s for the pairs (x, y) = (i, i + rot_dim / 2), c and s of the token's position.
// G lanes take a head of a token (G: head_dim / 8 rounded up to a power of two), each two pieces of four dims: below
// rot_dim the dims 4u .. 4u + 3 and their partners rot_dim / 2 further, so that a pair never leaves a lane, then eight dims in a
// row. Heads j < nh are queries, the next n_kv_heads keys, the last n_kv_heads values. A workgroup takes heads of token
// blockIdx.x: its cosines and sines are read once.
// Bound: bytes. 2048 tokens of 32 + 8 + 8 heads of 128, fp32 in: 75 MB in 15.7 us, 4.8 TB/s; 8191 of 16 + 4 + 4 of 256, fp16: 201
// MB in 46 us, 62 where the inputs come from HBM; 16 tokens: 3.7 us, a launch. To a Q8 cache: 2048 tokens 18 us, 8191 51. Slower
// at 8191, with the inputs in cache (not compared from HBM): a workgroup per 8 heads (67 us), workgroups over several tokens (52
// .. 58), the next head's values read ahead (50).
template <bool F32, int G>
__global__ void __launch_bounds__(256, 8) k_rope_append(RopeArgs g) {
    const int t = g.first + (int)blockIdx.x, hd = g.kv.head_dim, nkv = g.kv.n_kv_heads, half = g.r.rot_dim / 2;
    const int u = threadIdx.x % G, first = threadIdx.x / G;
    const int d0 = 4 * u < half ? 4 * u : 2 * half + 8 * (u - half / 4), d1 = 4 * u < half ? half + 4 * u : d0 + 4;
    const bool on = 8 * u < hd, turn = 4 * u < half;
    const int where = g.tok_pos[t], slot = g.tok_slot[t];
    f4 c = {1.f, 1.f, 1.f, 1.f}, s = {0.f, 0.f, 0.f, 0.f};
    if (turn) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int p = g.r.positions ? g.r.positions[(size_t)g.axis[4 * u + e] * g.n_tokens + t] : where;
            const bool ok = (unsigned)p < (unsigned)g.r.n_table;
            const f2 cs = ok ? *(const f2 *)(g.r.table + ((size_t)p * half + 4 * u + e) * 2) : f2{NAN, NAN};
            c[e] = cs.x, s[e] = cs.y;
        }
    }
    for (int j = blockIdx.y * (256 / G) + first; j < g.nh + 2 * nkv; j += gridDim.y * (256 / G)) {
        const bool is_q = j < g.nh, is_v = j >= g.nh + nkv;
        const int h = is_q ? j : (j - g.nh) % nkv;
        const void *src = is_q ? g.r.q : is_v ? g.r.v : g.r.k;
        const size_t at = is_q ? (size_t)t * g.r.q_stride + (size_t)h * g.r.q_head_stride : (size_t)t * g.r.kv_stride + (size_t)h * hd;
        f4 a = {0.f, 0.f, 0.f, 0.f}, b = a;
        if (on) a = load4<F32>(src, at + d0), b = load4<F32>(src, at + d1);
        if (g.r.q_norm && !is_v) {
            float ss = 0.f;
#pragma unroll
            for (int e = 0; e < 4; e++) ss += a[e] * a[e] + b[e] * b[e];
#pragma unroll
            for (int o = G / 2; o > 0; o >>= 1) ss += __shfl_xor(ss, o, 64);
            const float inv = 1.0f / sqrtf(ss / (float)hd + g.r.eps);
            const float *w = is_q ? g.r.q_norm : g.r.k_norm;
            if (on) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    a[e] = a[e] * inv * (g.r.norm_offset + w[d0 + e]);
                    b[e] = b[e] * inv * (g.r.norm_offset + w[d1 + e]);
                }
            }
        }
        if (turn && !is_v) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float x = a[e], y = b[e];
                a[e] = x * c[e] - y * s[e];
                b[e] = y * c[e] + x * s[e];
            }
        }
        if (is_q) {
            if (where < 0) a = b = f4{0.f, 0.f, 0.f, 0.f};  // padding
            if (on) {
                _Float16 *o = (_Float16 *)g.r.q_out + ((size_t)t * g.nh + h) * hd;
                store4(o + d0, a), store4(o + d1, b);
            }
            continue;
        }
        if (slot < 0) continue;
        const int page = slot / g.kv.page_size, in = slot % g.kv.page_size;
        const size_t to = (size_t)page * g.kv.page_stride + (size_t)in * g.kv.pos_stride + (size_t)h * g.kv.head_stride;
        if (g.kv.type == HQ_KV_F16) {
            _Float16 *o = (_Float16 *)(is_v ? g.kv.v : g.kv.k) + to;
            if (on) store4(o + d0, a), store4(o + d1, b);
            continue;
        }
        // Q8: the largest magnitude of the head (a NaN among them makes the scale NaN), codes to nearest
        float mx = 0.f, bad = 0.f;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            mx = fmaxf(mx, fmaxf(fabsf(a[e]), fabsf(b[e])));
            bad += 0.f * a[e] + 0.f * b[e];  // NaN where a value is not finite
        }
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1) {
            mx = fmaxf(mx, __shfl_xor(mx, o, 64));
            bad += __shfl_xor(bad, o, 64);
        }
        const _Float16 d = (_Float16)(mx / 127.0f + bad);
        const float df = (float)d;
        uint32_t w0 = 0, w1 = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float x = df > 0.f ? rintf(a[e] / df) : 0.f, y = df > 0.f ? rintf(b[e] / df) : 0.f;
            w0 |= ((uint32_t)(int)fminf(fmaxf(x, -127.f), 127.f) & 0xffu) << (8 * e);
            w1 |= ((uint32_t)(int)fminf(fmaxf(y, -127.f), 127.f) & 0xffu) << (8 * e);
        }
        int8_t *o = (int8_t *)(is_v ? g.kv.v : g.kv.k) + to;
        if (on) *(uint32_t *)(o + d0) = w0, *(uint32_t *)(o + d1) = w1;
        if (u == 0) ((_Float16 *)(is_v ? g.kv.v_scale : g.kv.k_scale))[((size_t)page * nkv + h) * g.kv.page_size + in] = d;
    }
}

}  // namespace

extern "C" int hq_rope_table(const float *inv_freq, int rot_dim, int n, float *table, void *stream) {
    if (!inv_freq || !table) return hq_internal_fail("hq_rope_table: null argument");
    if (rot_dim < 2 || rot_dim > 256 || rot_dim % 2 || n < 1) return hq_internal_fail("hq_rope_table: rot_dim %d, %d positions", rot_dim, n);
    if (!aligned(table, 8)) return hq_internal_fail("hq_rope_table: the table must be 8-byte aligned");
    float *d = nullptr;
    SCK(hipMalloc((void **)&d, (size_t)rot_dim / 2 * 4));
    hipError_t e = hipMemcpy(d, inv_freq, (size_t)rot_dim / 2 * 4, hipMemcpyHostToDevice);
    if (e == hipSuccess) {
        const size_t blocks = std::min<size_t>(((size_t)n * (rot_dim / 2) + 255) / 256, 65536);
        k_rope_table<<<(unsigned)blocks, 256, 0, (hipStream_t)stream>>>(d, rot_dim / 2, n, table);
        e = hipGetLastError();
        if (e == hipSuccess) e = hipStreamSynchronize((hipStream_t)stream);
    }
    (void)hipFree(d);
    if (e != hipSuccess) return hq_internal_fail("hq_rope_table: %s", hipGetErrorString(e));
    return 0;
}

extern "C" int hq_rope_append(const hq_batch *b, const hq_kv_t *kv, const hq_rope_t *r, void *stream) {
    const char *const who = "hq_rope_append";
    if (!b || !kv || !r) return hq_internal_fail("%s: null argument", who);
    if (!b->set) return hq_internal_fail("%s: the batch describes no step (hq_batch_set)", who);
    if (hq_kv_check(who, kv, b)) return -1;
    if (b->n_tokens == 0) return 0;
    if (!r->q || !r->k || !r->v || !r->q_out) return hq_internal_fail("%s: null argument", who);
    if (!aligned(r->q, 16) || !aligned(r->k, 16) || !aligned(r->v, 16) || !aligned(r->q_out, 16))
        return hq_internal_fail("%s: q, k, v and q_out must be 16-byte aligned", who);
    const int64_t most = (int64_t)1 << 40;
    if (r->q_stride < 0 || r->q_stride > most || r->q_stride % 8 || r->kv_stride < 0 || r->kv_stride > most || r->kv_stride % 8 ||
        r->q_head_stride < kv->head_dim || r->q_head_stride > most || r->q_head_stride % 8)
        return hq_internal_fail("%s: strides %lld, %lld, %lld (multiples of 8; a head's at least head_dim)", who, (long long)r->q_stride,
                                (long long)r->q_head_stride, (long long)r->kv_stride);
    if (r->rot_dim < 0 || r->rot_dim % 8 || r->rot_dim > kv->head_dim)
        return hq_internal_fail("%s: rot_dim %d (a multiple of 8, at most head_dim = %d)", who, r->rot_dim, kv->head_dim);
    if (r->rot_dim && (!r->table || r->n_table < 1 || !aligned(r->table, 8))) return hq_internal_fail("%s: an 8-byte aligned table of positions is needed", who);
    if (!r->q_norm != !r->k_norm) return hq_internal_fail("%s: q_norm without k_norm, or the other way round", who);
    if (r->q_norm && !(r->eps >= 0.f)) return hq_internal_fail("%s: eps %g", who, (double)r->eps);
    RopeArgs g;
    memset(g.axis, 0, sizeof g.axis);
    if (r->positions) {
        if (!r->axis || r->n_axes < 1 || r->n_axes > 8) return hq_internal_fail("%s: positions on %d axes (1 .. 8, with the axis of each frequency)", who, r->n_axes);
        for (int i = 0; i < r->rot_dim / 2; i++) {
            if (r->axis[i] >= r->n_axes) return hq_internal_fail("%s: frequency %d turns by axis %d of %d", who, i, r->axis[i], r->n_axes);
            g.axis[i] = r->axis[i];
        }
    }
    if (use_device(b->device)) return -1;
    g.kv = *kv, g.r = *r;
    g.tok_pos = b->tok_pos, g.tok_slot = b->tok_slot, g.nh = b->n_heads, g.n_tokens = b->n_tokens;
    const int lanes = kv->head_dim <= 64 ? 8 : kv->head_dim <= 128 ? 16 : 32, heads = b->n_heads + 2 * kv->n_kv_heads, per = 256 / lanes;
    // few tokens: their heads over several workgroups, while there are fewer than 8 per CU
    const int y = std::min((heads + per - 1) / per, std::max(8 * b->n_cu / b->n_tokens, 1));
    hipStream_t st = (hipStream_t)stream;
    for (g.first = 0; g.first < b->n_tokens; g.first += 1 << 23) {  // (a launch has fewer than 2^32 threads)
        const dim3 grid((unsigned)std::min(1 << 23, b->n_tokens - g.first), (unsigned)y);
#define HQ_ROPE(F, G) k_rope_append<F, G><<<grid, 256, 0, st>>>(g)
        if (r->f32) {
            if (lanes == 8) HQ_ROPE(true, 8);
            else if (lanes == 16) HQ_ROPE(true, 16);
            else HQ_ROPE(true, 32);
        } else {
            if (lanes == 8) HQ_ROPE(false, 8);
            else if (lanes == 16) HQ_ROPE(false, 16);
            else HQ_ROPE(false, 32);
        }
        SCK(hipGetLastError());
    }
#undef HQ_ROPE
    return 0;
}
