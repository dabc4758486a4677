// hq_pages.hip - pages of a cache that sequences share, branch from and leave (hq_pages_*), and their copies (hq_kv_copy,
// include/hq_serve.h).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <new>
#include <string.h>
#include <vector>

#include "hq_batch.h"
#include "hq_device.h"

// ------------------------------------------------------------------------------------ who holds which page
struct hq_pages {
    uint32_t n_pages;
    int page_size;
    struct Seq {
        int n_pos = 0;
        std::vector<uint32_t> pages;
    };
    std::vector<Seq> seqs;
    std::vector<int> holders;    // of each page
    std::vector<int> readers;    // waiting copies that read it: it is not handed out while there are any
    std::vector<uint32_t> free;  // a heap, the lowest page first
    std::vector<uint32_t> src, dst;  // waiting copies
    std::vector<int32_t> n;
    std::vector<int> waits;      // the one into each page, or -1
    std::vector<uint32_t> out_src, out_dst;  // those handed to the caller
    std::vector<int32_t> out_n;

    void put(uint32_t p) {  // (free has room for every page)
        free.push_back(p);
        std::push_heap(free.begin(), free.end(), std::greater<uint32_t>());
    }
    uint32_t take() {
        std::pop_heap(free.begin(), free.end(), std::greater<uint32_t>());
        const uint32_t p = free.back();
        free.pop_back();
        holders[p] = 1;
        return p;
    }
    void push(uint32_t from, uint32_t to, int32_t m) {  // (there is room)
        waits[to] = (int)dst.size();
        src.push_back(from), dst.push_back(to), n.push_back(m);
        readers[from]++;
    }
    // The pages that go back to the pool with one of p's holders: itself, and one that only a copy into it still reads. (Of the pages of
    // one sequence no two wait for one page's copy: each is another part of what they are copied from.)
    size_t returns(uint32_t p) const {
        if (holders[p] > 1) return 0;
        const int i = waits[p];
        return (readers[p] == 0) + (i >= 0 && readers[src[(size_t)i]] == 1 && holders[src[(size_t)i]] == 0);
    }
    void drop(uint32_t p) {
        if (--holders[p]) return;
        if (const int i = waits[p]; i >= 0) {  // a copy into a page that nobody holds any more is not wanted
            const uint32_t s = src[(size_t)i];
            src[(size_t)i] = src.back(), dst[(size_t)i] = dst.back(), n[(size_t)i] = n.back();
            waits[dst[(size_t)i]] = i, waits[p] = -1;
            src.pop_back(), dst.pop_back(), n.pop_back();
            if (--readers[s] == 0 && holders[s] == 0) put(s);
        }
        if (readers[p] == 0) put(p);
    }
};

namespace {

int seq_check(const char *who, const hq_pages *p, int seq) {
    if (!p) return hq_internal_fail("%s: null argument", who);
    if (seq < 0 || (size_t)seq >= p->seqs.size()) return hq_internal_fail("%s: sequence %d (there are %zu)", who, seq, p->seqs.size());
    return 0;
}

}  // namespace

extern "C" int hq_pages_create(uint32_t n_pages, int page_size, int max_seqs, hq_pages **out) {
    const char *const who = "hq_pages_create";
    if (!out) return hq_internal_fail("%s: null argument", who);
    *out = nullptr;
    if (page_size < 16 || page_size > 4096 || (page_size & (page_size - 1))) return hq_internal_fail("%s: page_size %d (a power of two, 16 .. 4096)", who, page_size);
    if (n_pages < 1 || (uint64_t)n_pages * (uint64_t)page_size >= (1ull << 31))
        return hq_internal_fail("%s: %u pages of %d positions (1 page or more, below 2^31 positions)", who, n_pages, page_size);
    if (max_seqs < 1 || max_seqs > (1 << 20)) return hq_internal_fail("%s: %d sequences (1 .. 2^20)", who, max_seqs);
    hq_pages *p = nullptr;
    try {
        p = new hq_pages();
        p->n_pages = n_pages, p->page_size = page_size;
        p->seqs.resize((size_t)max_seqs);
        p->holders.assign(n_pages, 0);
        p->readers.assign(n_pages, 0);
        p->waits.assign(n_pages, -1);
        p->free.resize(n_pages);
        for (uint32_t i = 0; i < n_pages; i++) p->free[i] = i;  // in order: a heap
    } catch (const std::exception &) {
        delete p;
        return hq_internal_fail("%s: out of memory", who);
    }
    *out = p;
    return 0;
}

extern "C" void hq_pages_free(hq_pages *p) { delete p; }

extern "C" int hq_pages_resize(hq_pages *p, int seq, int n_keep, int n_pos) {
    const char *const who = "hq_pages_resize";
    if (seq_check(who, p, seq)) return -1;
    hq_pages::Seq &s = p->seqs[(size_t)seq];
    if (n_keep < 0 || n_keep > s.n_pos || n_pos < n_keep || (uint64_t)n_pos > (uint64_t)p->n_pages * (uint64_t)p->page_size)
        return hq_internal_fail("%s: sequence %d of %d positions is to keep %d and have %d (of a cache of %u pages of %d)", who, seq, s.n_pos, n_keep, n_pos,
                                p->n_pages, p->page_size);
    const size_t ps = (size_t)p->page_size, have = s.pages.size(), need = ((size_t)n_pos + ps - 1) / ps;
    // pages from `first` on take new positions: those that others hold are replaced
    const size_t first = n_pos > n_keep ? (size_t)n_keep / ps : need, stay = std::min(have, need);
    size_t want = need > have ? need - have : 0;
    for (size_t i = first; i < stay; i++) want += p->holders[s.pages[i]] > 1;
    // too few in the pool: those that the sequence itself gives back come first
    const bool give_first = want > p->free.size();
    if (give_first) {
        size_t given = 0;
        for (size_t i = need; i < have; i++) given += p->returns(s.pages[i]);
        if (want > p->free.size() + given) return hq_internal_fail("%s: sequence %d needs %zu pages more (%zu are free)", who, seq, want, p->free.size() + given);
    }
    try {
        s.pages.reserve(need);
        if (p->src.size() == std::min({p->src.capacity(), p->dst.capacity(), p->n.capacity()})) {  // (twice the room: not a new place for all of them at each call)
            const size_t room = std::max<size_t>(16, 2 * p->src.size());
            p->src.reserve(room), p->dst.reserve(room), p->n.reserve(room);
        }
    } catch (const std::exception &) {
        return hq_internal_fail("%s: out of memory", who);
    }
    const auto give = [&]() {
        for (; s.pages.size() > need; s.pages.pop_back()) p->drop(s.pages.back());
    };
    if (give_first) give();
    for (size_t i = first; i < stay; i++) {
        const uint32_t old = s.pages[i];
        if (p->holders[old] == 1) continue;
        const int kept = (int)std::min<size_t>((size_t)n_keep > i * ps ? (size_t)n_keep - i * ps : 0, ps);
        const uint32_t page = s.pages[i] = p->take();
        if (kept) {
            // what the old page is itself still waiting for comes from there
            uint32_t from = old;
            int n = kept;
            if (const int j = p->waits[old]; j >= 0) from = p->src[(size_t)j], n = std::min(n, (int)p->n[(size_t)j]);
            p->push(from, page, n);
        }
        p->drop(old);
    }
    give();
    while (s.pages.size() < need) s.pages.push_back(p->take());
    s.n_pos = n_pos;
    return 0;
}

extern "C" int hq_pages_fork(hq_pages *p, int parent, int child, int n_pos) {
    const char *const who = "hq_pages_fork";
    if (seq_check(who, p, parent) || seq_check(who, p, child)) return -1;
    const hq_pages::Seq &a = p->seqs[(size_t)parent];
    hq_pages::Seq &b = p->seqs[(size_t)child];
    if (b.n_pos || parent == child) return hq_internal_fail("%s: sequence %d has %d positions (a child must have none)", who, child, b.n_pos);
    if (n_pos < 0 || n_pos > a.n_pos) return hq_internal_fail("%s: %d positions of sequence %d, which has %d", who, n_pos, parent, a.n_pos);
    const size_t need = ((size_t)n_pos + (size_t)p->page_size - 1) / (size_t)p->page_size;
    try {
        b.pages.assign(a.pages.begin(), a.pages.begin() + (ptrdiff_t)need);
    } catch (const std::exception &) {
        return hq_internal_fail("%s: out of memory", who);
    }
    for (uint32_t page : b.pages) p->holders[page]++;
    b.n_pos = n_pos;
    return 0;
}

extern "C" int hq_pages_compact(hq_pages *p) {
    const char *const who = "hq_pages_compact";
    if (!p) return hq_internal_fail("%s: null argument", who);
    if (!p->dst.empty()) return hq_internal_fail("%s: %zu copies wait (hq_pages_copies)", who, p->dst.size());
    const uint32_t used = p->n_pages - (uint32_t)p->free.size();
    std::vector<uint32_t> to;
    try {
        to.resize(p->n_pages);
        size_t moves = 0;
        for (uint32_t i = used; i < p->n_pages; i++) moves += p->holders[i] > 0;
        p->src.reserve(moves), p->dst.reserve(moves), p->n.reserve(moves);
    } catch (const std::exception &) {
        return hq_internal_fail("%s: out of memory", who);
    }
    uint32_t hole = 0;
    for (uint32_t i = 0; i < p->n_pages; i++) {
        to[i] = i;
        if (i < used || !p->holders[i]) continue;
        while (p->holders[hole]) hole++;  // (as many free pages lie below `used` as held ones above)
        to[i] = hole;
        p->holders[hole] = p->holders[i];
        p->push(i, hole, p->page_size);
    }
    for (uint32_t i : p->src) p->holders[i] = 0;
    for (hq_pages::Seq &s : p->seqs)
        for (uint32_t &page : s.pages) page = to[page];
    p->free.clear();
    for (uint32_t i = 0; i < p->n_pages; i++)
        if (!p->holders[i] && !p->readers[i]) p->free.push_back(i);  // in order: a heap
    return 0;
}

extern "C" int hq_pages_copies(hq_pages *p, const uint32_t **src, const uint32_t **dst, const int32_t **n_pos, int *n) {
    const char *const who = "hq_pages_copies";
    if (!p || !src || !dst || !n_pos || !n) return hq_internal_fail("%s: null argument", who);
    p->out_src.swap(p->src), p->out_dst.swap(p->dst), p->out_n.swap(p->n);
    p->src.clear(), p->dst.clear(), p->n.clear();
    for (uint32_t d : p->out_dst) p->waits[d] = -1;
    for (uint32_t s : p->out_src)
        if (--p->readers[s] == 0 && p->holders[s] == 0) p->put(s);
    *src = p->out_src.data(), *dst = p->out_dst.data(), *n_pos = p->out_n.data(), *n = (int)p->out_src.size();
    return 0;
}

extern "C" int hq_pages_table(const hq_pages *p, const int32_t *seqs, int n, uint32_t *pages, int pages_ld) {
    const char *const who = "hq_pages_table";
    if (!p || n < 0 || pages_ld < 0 || (n && (!seqs || (pages_ld && !pages)))) return hq_internal_fail("%s: null argument", who);
    for (int i = 0; i < n; i++) {
        if (seq_check(who, p, seqs[i])) return -1;
        const size_t have = p->seqs[(size_t)seqs[i]].pages.size();
        if (have > (size_t)pages_ld) return hq_internal_fail("%s: sequence %d has %zu pages, a row %d", who, seqs[i], have, pages_ld);
    }
    for (int i = 0; i < n; i++) {
        const std::vector<uint32_t> &s = p->seqs[(size_t)seqs[i]].pages;
        uint32_t *row = pages + (size_t)i * (size_t)pages_ld;
        std::copy(s.begin(), s.end(), row);
        std::fill(row + s.size(), row + pages_ld, 0u);
    }
    return 0;
}

extern "C" int hq_pages_count(const hq_pages *p, int seq, int *n_pos, uint32_t *n_free) {
    if (seq_check("hq_pages_count", p, seq)) return -1;
    if (n_pos) *n_pos = p->seqs[(size_t)seq].n_pos;
    if (n_free) *n_free = (uint32_t)p->free.size();
    return 0;
}

// ------------------------------------------------------------------------------------ copies
namespace {

constexpr int CACHES = 40, PAIRS = 256;  // of a launch: they lie in its arguments (4 KB at most), so that nothing is
                                         // allocated or sent before it; 36 layers in launches of 8 caches 29 us, in one 16
constexpr int NT = 256, VEC = 4;        // pieces of 16 bytes in flight per thread

struct CopyArgs {
    void *at[CACHES][2];
    uint16_t *scale[CACHES][2];
    uint32_t src[PAIRS], dst[PAIRS];
    uint16_t n[PAIRS];
    int64_t page_bytes, outer_bytes, inner_bytes;
    // the first n positions of a page are runs of memory: `inner` of each of n (or 1) outer ones, each `run` pieces, n times that
    // where a run holds all positions
    int inner, run;
    bool per_pos;  // outer: the positions
    int heads, page_size, caches;
};

// Bound: bytes, read and written once. 192 whole pages of 128 KB, keys and values of 8 layers (806 MB moved): 157 us, 5.1 TB/s, as a
// large copy. 32 pages of which about half is used (67 MB): 16.9 us, 13 of them the bytes, the rest the launch and its ends;
// without the divisions, or with eight pieces in flight, no less.
__global__ void __launch_bounds__(NT) k_kv_copy(CopyArgs g) {
    const int pair = blockIdx.y, c = blockIdx.z % g.caches, kind = blockIdx.z / g.caches;
    const size_t src = g.src[pair], dst = g.dst[pair];
    const uint32_t n = g.n[pair];
    if (kind >= 2) {  // scales
        uint16_t *const s = g.scale[c][kind - 2];
        const uint32_t all = (uint32_t)g.heads * n;
        for (uint32_t i = blockIdx.x * NT + threadIdx.x; i < all; i += gridDim.x * NT) {
            const uint32_t h = i / n, p = i - h * n;
            s[(dst * g.heads + h) * g.page_size + p] = s[(src * g.heads + h) * g.page_size + p];
        }
        return;
    }
    char *const at = (char *)g.at[c][kind];
    const uint32_t run = (uint32_t)g.run * (g.per_pos ? 1u : n), all = run * (uint32_t)g.inner * (g.per_pos ? n : 1u);
    for (uint32_t i0 = blockIdx.x * (NT * VEC) + threadIdx.x; i0 < all; i0 += gridDim.x * (NT * VEC)) {
        u4v x[VEC];
        size_t o[VEC];
#pragma unroll
        for (int v = 0; v < VEC; v++) {
            const uint32_t i = i0 + v * NT, r = i / run, e = i - r * run, a = r / (uint32_t)g.inner, b = r - a * (uint32_t)g.inner;
            o[v] = (size_t)a * g.outer_bytes + (size_t)b * g.inner_bytes + (size_t)e * 16;
            if (i < all) x[v] = *(const u4v *)(at + src * g.page_bytes + o[v]);
        }
#pragma unroll
        for (int v = 0; v < VEC; v++)
            if (i0 + v * NT < all) *(u4v *)(at + dst * g.page_bytes + o[v]) = x[v];
    }
}

}  // namespace

extern "C" int hq_kv_copy(const hq_kv_t *kv, int n_kv, const uint32_t *src, const uint32_t *dst, const int32_t *n_pos, int n, void *stream) {
    const char *const who = "hq_kv_copy";
    if (n_kv < 0 || n < 0 || (n_kv && !kv) || (n && (!src || !dst))) return hq_internal_fail("%s: null argument, or %d caches and %d copies", who, n_kv, n);
    for (int i = 0; i < n_kv; i++) {
        hq_batch b = {};
        b.geom = kv[0];
        if (hq_kv_check(who, &kv[i], &b)) return -1;
        if (kv[i].page_stride != kv[0].page_stride || kv[i].pos_stride != kv[0].pos_stride || kv[i].head_stride != kv[0].head_stride)
            return hq_internal_fail("%s: caches 0 and %d differ in their strides", who, i);
    }
    if (!n_kv || !n) return 0;
    const hq_kv_t &k = kv[0];
    for (int i = 0; i < n; i++) {
        if (src[i] >= k.n_pages || dst[i] >= k.n_pages) return hq_internal_fail("%s: copy %d is of page %u to page %u (the cache has %u)", who, i, src[i], dst[i], k.n_pages);
        if (n_pos && (n_pos[i] < 0 || n_pos[i] > k.page_size)) return hq_internal_fail("%s: copy %d is of %d positions (a page has %d)", who, i, n_pos[i], k.page_size);
    }
    try {
        std::vector<uint32_t> w(dst, dst + n), r(src, src + n);
        std::sort(w.begin(), w.end());
        std::sort(r.begin(), r.end());
        for (size_t i = 1; i < w.size(); i++)
            if (w[i] == w[i - 1]) return hq_internal_fail("%s: two copies to page %u", who, w[i]);
        for (size_t i = 0, j = 0; i < w.size(); i++) {
            while (j < r.size() && r[j] < w[i]) j++;
            if (j < r.size() && r[j] == w[i]) return hq_internal_fail("%s: page %u is read by one copy and written by another", who, w[i]);
        }
    } catch (const std::exception &) {
        return hq_internal_fail("%s: out of memory", who);
    }
    const int bytes = k.type == HQ_KV_Q8 ? 1 : 2, row = k.head_dim * bytes / 16;
    CopyArgs g;
    g.page_bytes = k.page_stride * bytes, g.heads = k.n_kv_heads, g.page_size = k.page_size;
    if (k.pos_stride == (int64_t)k.n_kv_heads * k.head_dim && k.head_stride == k.head_dim) {  // all positions in one run
        g.inner = 1, g.run = k.n_kv_heads * row, g.per_pos = false, g.outer_bytes = g.inner_bytes = 0;
    } else if (k.pos_stride == k.head_dim) {  // a head's positions in one run
        g.inner = k.n_kv_heads, g.run = row, g.per_pos = false, g.outer_bytes = 0, g.inner_bytes = k.head_stride * bytes;
    } else {
        g.inner = k.n_kv_heads, g.run = row, g.per_pos = true, g.outer_bytes = k.pos_stride * bytes, g.inner_bytes = k.head_stride * bytes;
    }
    const unsigned pieces = (unsigned)k.page_size * (unsigned)(k.n_kv_heads * row);
    const unsigned blocks = std::min((pieces + NT * VEC - 1) / (NT * VEC), 4096u);
    for (int c0 = 0; c0 < n_kv; c0 += CACHES)
        for (int p0 = 0; p0 < n; p0 += PAIRS) {
            const int pairs = std::min(PAIRS, n - p0);
            g.caches = std::min(CACHES, n_kv - c0);
            for (int c = 0; c < g.caches; c++) {
                g.at[c][0] = kv[c0 + c].k, g.at[c][1] = kv[c0 + c].v;
                g.scale[c][0] = kv[c0 + c].k_scale, g.scale[c][1] = kv[c0 + c].v_scale;
            }
            for (int i = 0; i < pairs; i++) g.src[i] = src[p0 + i], g.dst[i] = dst[p0 + i], g.n[i] = (uint16_t)(n_pos ? n_pos[p0 + i] : k.page_size);
            const dim3 grid(blocks, (unsigned)pairs, (unsigned)(g.caches * (k.type == HQ_KV_Q8 ? 4 : 2)));
            k_kv_copy<<<grid, NT, 0, (hipStream_t)stream>>>(g);
            SCK(hipGetLastError());
        }
    return 0;
}
