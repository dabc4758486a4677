// hq_scan.h - a step's sequences and states on the device (hq_scan.hip), as the kernels of recurrent layers read them.
#ifndef HQ_SCAN_H
#define HQ_SCAN_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <vector>

#include "hq_internal.h"
#include "hq_serve.h"

struct HqSeq {
    int tok0, n;   // its first new token and how many there are
    int from, to;  // slots, or -1
};
// Tokens t0 .. t0 + n - 1 of sequence seq, for one workgroup.
struct HqTile {
    int seq, t0, n;
};
constexpr int HQ_CONV_TILE = 8;  // most tokens of a tile of hq_delta_append

// hq_delta by chunks of 64 tokens. A chunk's operands that depend on its value head but not on the state are formed first, for many
// chunks at a time (a pass), into HQ_CHUNK_BYTES of workspace each: 24 fragments and a vector of 1 KB (hq_delta.hip).
// Most new tokens of a sequence that it takes token by token. Alone (32 heads of 128, us, by chunks behind the stroke): 16 sequences of 5
// tokens, 21 / 39, of 12, 34 / 39, of 16, 39 / 39; 64 of 16, 117 / 139. Where all sequences' workgroups by chunks find a CU each, a
// chain of tokens is the longer one sooner: one sequence of 8, 12.4 / 13.8, of 12, 17.2 / 14.0; 4 of 8, 15.1 / 16.5, of 12, 20.2 / 16.5; so there
// all go by chunks as soon as one has more than 8. Beside sequences of more than 16 it is a launch more: a chunk of 2048 and 8 of 5 tokens, 87 / 85,
// and 32 of 5, 107 / 100, and 32 of 16, 141 / 102; but 64 of 5, 138 / 162, and 64 of one, 128 / 160; so there those of more than 4 tokens go by
// chunks where they have four heads a CU at most.
constexpr int HQ_STEP_TOKENS = 16, HQ_STEP_ALONE = 8, HQ_STEP_BESIDE = 4;
constexpr int HQ_CHUNK = 64;
constexpr size_t HQ_CHUNK_BYTES = 25 * 1024;
struct HqChunk {
    int tok0, n;
};
// A sequence, or a part of one: its tokens, its first chunk in the pass, slots as in HqSeq, or places of the workspace for states: -2 - i
// is place i. Places 0 and 1 have states on their way from one pass to the next.
constexpr int HQ_IDENTITY = -0x7fffffff;  // from: S = I, and the values are zeros
struct HqRun {
    int tok0, n, chunk0;
    int from, to;
};
// A sequence that a pass takes in `n` parts at a time. What a part does to a state is S' = P S + Q. Places of the workspace: `place` a copy
// of the sequence's state, from there on the states behind parts 0 .. n - 2 (at first Q), then P of parts 1 .. n - 2.
struct HqJoin {
    int from, place, n;
};
struct HqPass {
    int chunk0, n_chunks;  // of hq_scan::chunks
    int run0, n_runs;      // of hq_scan::runs
    int part0, n_parts;    // of hq_scan::runs: those that only lead to states, before
    int join0, n_joins;    // of hq_scan::joins: and what makes the parts' first states of them
};
// columns of a head's state that one workgroup takes through a run
constexpr int hq_scan_columns(int k_dim) { return k_dim > 128 ? 32 : 64; }

struct hq_scan {
    int device, n_cu;
    int max_seqs, max_tokens;
    // the step
    int n_seqs, n_tokens;
    hq_state_t geom;
    bool set;
    // device arrays, parts of `dev`
    const HqSeq *seqs;
    const HqTile *tiles;  // of hq_delta_append: every sequence's first tile, which has its convolution's state, is there
    int n_tiles;
    const int *steps;  // the sequences that hq_delta takes token by token, longest first
    int n_steps, longest_step;  // (its tokens)
    const HqChunk *chunks;  // and those that it takes by chunks
    const HqRun *runs;      // (a pass's longest first)
    const HqJoin *joins;
    std::vector<HqPass> passes;
    char *work;             // chunks of a pass, then their outputs ahead of a norm (fp32: 64 rows of n_v_heads * v_dim a chunk), then places for
                            // states, each n_v_heads * k_dim * max(k_dim, v_dim) long
    size_t work_bytes, outs_at, places_at;
    // storage: one pinned copy of `dev`, which the next set waits for
    int *host, *dev;
    size_t words;
    hipEvent_t sent;
    bool sending;
};

// A state argument against the step's geometry: 0, or -1 with a message naming `who`.
int hq_state_check(const char *who, const hq_state_t *st, const hq_scan *c);

#define SCK(call)                                                                                         \
    do {                                                                                                  \
        hipError_t e_ = (call);                                                                           \
        if (e_ != hipSuccess)                                                                             \
            return hq_internal_fail("HIP %s failed: %s (%s:%d)", #call, hipGetErrorString(e_), __FILE__, __LINE__); \
    } while (0)

#endif
