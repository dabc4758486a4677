// hq_batch.h - a serving step's description on the device (hq_batch.hip), as the paged kernels read it.
#ifndef HQ_BATCH_H
#define HQ_BATCH_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "hq_internal.h"
#include "hq_serve.h"

// One workgroup's work in hq_attention: rows row0 .. of kv head kvh of a sequence (row t rep + e: its new token t, query head
// kvh rep + e; R rows in all) over positions k0 .. k1 - 1; part `part` of the n_parts that its block of rows is cut into.
struct HqItem {
    int kvh;        // -1: nothing
    int tok0;       // the sequence's first new token
    int base;       // the position of it
    int R, row0;
    int t0, e0;     // row0 / rep and row0 % rep
    int n;          // positions that the block's last row sees
    int k0, k1;
    int page0;      // its pages
    int part, n_parts;
    int block;        // HQ_STREAM: the block's counter, where n_parts > 1
    uint32_t part_at; // its parts, in units of 16 bytes of hq_batch::parts
};
// Kernel bodies of hq_attention by the rows a workgroup takes.
enum { HQ_STREAM, HQ_ROWS128, HQ_ROWS256, HQ_BODIES };  // HQ_STREAM: 16, or 32 where the item has more rows
constexpr int HQ_STREAM_PARTS = 128;  // most parts of a block of HQ_STREAM
// The dims that a body's kernel for a head_dim holds; a part's row has HQ_PART_EXTRA floats more.
int hq_attn_width(int body, int head_dim);
constexpr int HQ_PART_EXTRA = 4;

struct hq_batch {
    int device, n_cu;
    int max_seqs, max_tokens, max_pages;  // capacities; pages per sequence
    // the step
    int n_seqs, n_tokens, n_heads;
    hq_kv_t geom;  // the cache's type, page size, heads, head_dim and pages
    bool set;
    // device arrays, parts of `dev`
    const int *tok_pos;   // position of token t in its sequence
    const int *tok_slot;  // page * page_size + slot, or -1: not stored
    const uint32_t *pages;
    const HqItem *items[HQ_BODIES];
    int n_items[HQ_BODIES];
    int stream_rows;  // the most rows of an item of HQ_STREAM: 16 or 32
    const HqItem *joins[HQ_BODIES];  // HQ_ROWS*: the first part of each block that is cut into several
    int n_joins[HQ_BODIES];
    int *counters;      // one per block of HQ_STREAM cut into parts; zero between calls
    float *parts;       // rows of such blocks
    size_t part_bytes;  // allocated
    // storage: one pinned copy of `dev`, which the next set waits for
    int *host, *dev;
    size_t words;  // of each
    hipEvent_t sent;
    bool sending;
};

// A kv argument against the batch's geometry and the alignment rules: 0, or -1 with a message naming `who`.
int hq_kv_check(const char *who, const hq_kv_t *kv, const hq_batch *b);

#define SCK(call)                                                                                         \
    do {                                                                                                  \
        hipError_t e_ = (call);                                                                           \
        if (e_ != hipSuccess)                                                                             \
            return hq_internal_fail("HIP %s failed: %s (%s:%d)", #call, hipGetErrorString(e_), __FILE__, __LINE__); \
    } while (0)

#endif
