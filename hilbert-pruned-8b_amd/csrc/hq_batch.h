// hq_batch.h - a serving step's description on the device (hq_batch.hip), as the paged kernels read it.
#ifndef HQ_BATCH_H
#define HQ_BATCH_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "hq_internal.h"
#include "hq_serve.h"

// One sequence: its new tokens tok0 .. tok0 + n_new - 1, of which the last n_new stand at positions n_pos - n_new ..
// n_pos - 1 (negative: padding), and its pages, pages[page0 ..].
struct HqSeq {
    int tok0, n_new, n_pos, page0;
};

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
    const int *tok_seq;
    const HqSeq *seqs;
    const uint32_t *pages;
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
