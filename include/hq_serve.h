/* hq_serve.h - operators of a serving loop: many sequences whose keys and values live in one paged cache.
 *
 * A step of such a loop takes each sequence's new tokens (a whole prompt, a chunk of one, a single decoded token) through
 * the layers together. hq_batch_set describes the step once; every layer then calls hq_rope_append (rotary positions of
 * the new queries and keys, keys and values into the pages) and hq_attention (the new queries over their sequences), and
 * after the last layer hq_logprobs turns rows of logits into log probabilities. include/hq_backend.h's hip_batch_*
 * functions run a whole model this way.
 *
 * Conventions as in hq.h: 0, or -1 with a message in hq_last_error(); arguments are checked on the host before anything
 * is queued; calls are asynchronous on `stream` and allocate nothing, except where stated. Matrices are row-major, strides
 * count elements. fp16 is held as uint16_t.
 */
#ifndef HQ_SERVE_H
#define HQ_SERVE_H

#include "hq.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- the paged cache (memory of the caller) */
enum {
    HQ_KV_F16 = 0, /* fp16 */
    HQ_KV_Q8 = 1   /* 8-bit codes (int8, -127 .. 127) and one fp16 scale for each position and kv head: value = code * scale */
};

/* Keys and values of one layer: element d of position slot s of page p of kv head h stands at
 * k[p * page_stride + s * pos_stride + h * head_stride + d] (and the same in v), so both usual orders of a page, positions
 * or heads outermost, are strides. Q8 scales stand at k_scale[(p * n_kv_heads + h) * page_size + s].
 * page_size: a power of two, 16 .. 4096; head_dim: a multiple of 16, at most 256; the strides: multiples of 16; k and v
 * 16-byte aligned. There is no limit on the cache's bytes; pages * page_size is below 2^31, page_size * pos_stride below
 * 2^30. */
typedef struct {
    int type, page_size, n_kv_heads, head_dim;
    uint32_t n_pages;
    void *k, *v;
    uint16_t *k_scale, *v_scale;
    int64_t page_stride, pos_stride, head_stride;
} hq_kv_t;

/* ---- one step's sequences */
typedef struct hq_batch hq_batch;

/* A batch description for up to max_seqs sequences, max_tokens new tokens in all and max_pages pages per sequence.
 * hq_batch_free waits for the device. */
int hq_batch_create(int device, int max_seqs, int max_tokens, int max_pages, hq_batch **out);
void hq_batch_free(hq_batch *b);

/* Describes a step (host arrays; copied before the call returns, sent to the device on `stream`): sequence i has n_pos[i]
 * positions, its new tokens among them, the last n_new[i] of which are the step's tokens; position p of it lies in slot
 * p % page_size of page pages[i * pages_ld + p / page_size]. The step's tokens are numbered sequence after sequence. Both
 * counts may be 0. With n_new > n_pos the first n_new - n_pos tokens are padding before position 0: they see nothing, are
 * not stored, and give zeros. kv: the cache's geometry (its pointers may differ in each call that follows); n_heads: query
 * heads, a multiple of the kv heads (head h reads kv head h / (n_heads / n_kv_heads)). Page numbers are checked here.
 * Also plans hq_attention's work and grows its workspace: the only call on device memory of this header, with hq_batch_create,
 * hq_scan_create and hq_scan_set, and the growing of hq_logprobs' and hq_beam's workspaces, that allocates. It waits until the last set's transfer is done, and with growing for
 * the device. Calls that use the batch must be ordered after it on the device, and the next set after them; calls that
 * overlap in time need batches of their own. */
int hq_batch_set(hq_batch *b, const hq_kv_t *kv, int n_heads, int n_seqs, const int32_t *n_new, const int32_t *n_pos,
                 const uint32_t *pages, int pages_ld, void *stream);

/* ---- rotary positions, and the append to the cache */
/* Cosines and sines of n positions, [n, rot_dim / 2] pairs (cos, sin) in fp32: of p * inv_freq[i] (host array), formed in
 * 64 bits. Waits for the stream. */
int hq_rope_table(const float *inv_freq, int rot_dim, int n, float *table, void *stream);

typedef struct {
    /* the new tokens' projections, fp16 (f32 = 0) or fp32: head h of token t at q + t * q_stride + h * q_head_stride
     * (head_dim, or more where other values stand between the heads, as an output gate does), k and v + t * kv_stride +
     * h * head_dim. 16-byte aligned, strides multiples of 8. */
    const void *q, *k, *v;
    int f32;
    int64_t q_stride, q_head_stride, kv_stride;
    /* optional RMSNorm of each head's query and key before the rotation (both or neither): x / sqrt(mean(x^2) + eps) *
     * (norm_offset + w), fp32 [head_dim] on the device */
    const float *q_norm, *k_norm;
    float norm_offset, eps;
    /* the rotation of the first rot_dim dims (a multiple of 8, 0 .. head_dim; pairs i and i + rot_dim / 2) by the table's
     * row of the token's position; n_table rows */
    const float *table;
    int n_table, rot_dim;
    /* positions on the device, [axes, tokens]; frequency i turns by axis[i] (host array of rot_dim / 2, each below n_axes,
     * at most 8 axes; copied): time, height and width of image and video tokens. NULL: one axis, the token's position in
     * its sequence. A position outside the table makes that token's rotated values NaN. */
    const int32_t *positions;
    const uint8_t *axis;
    int n_axes;
    uint16_t *q_out; /* [tokens, n_heads, head_dim] fp16, 16-byte aligned: the queries hq_attention takes */
} hq_rope_t;

/* For every new token: the queries, normalised and rotated, to q_out; the keys likewise, and the values, to the token's
 * slot of the cache. fp32 arithmetic, each result rounded once (Q8: to code * fp16(max |x| / 127); a head with an infinity
 * or NaN becomes all NaN). One kernel. */
int hq_rope_append(const hq_batch *b, const hq_kv_t *kv, const hq_rope_t *r, void *stream);

/* ---- attention */
typedef struct {
    const uint16_t *q; /* fp16: head h of token t at q + t * q_stride + h * head_dim; 16-byte aligned, stride a multiple of 8 */
    int64_t q_stride;
    float scale;       /* of the scores, 1 / sqrt(head_dim) as a rule; at most 1e20 in magnitude */
    /* optional output gate, fp16 or fp32 (gate_f32): out = o * 1 / (1 + exp(-gate)); head h of token t at gate +
     * t * gate_stride + h * gate_head_stride, aligned to 4 elements, strides multiples of 4 */
    const void *gate;
    int gate_f32;
    int64_t gate_stride, gate_head_stride;
    uint16_t *out;     /* fp16, head h of token t at out + t * out_stride + h * head_dim; alignment as q's */
    int64_t out_stride;
} hq_attn_t;

/* out = softmax(scale * q . K) V for every new token and head over positions 0 .. the token's own of its sequence, which
 * the cache holds (the step's own among them: hq_rope_append first). fp16 products (a weight is off by 2^-11 of itself or
 * 2^-31 of its row's largest, whichever is more), everything else fp32. Positions after a token, and what else a page holds,
 * do not affect it whatever their bits. The result does not depend on how the work was split over time: the same batch gives
 * the same bits. */
int hq_attention(const hq_batch *b, const hq_kv_t *kv, const hq_attn_t *a, void *stream);

/* ---- log probabilities */
#define HQ_LOGPROBS_MAX_TOP 64
/* Of M rows of V logits (fp16, or fp32 with f32; row m at logits + m * stride): logp[m, j] = log softmax(row)[ids[m, j]]
 * for n_ids tokens per row (ids on the device; an id >= V gives NaN), entropy[m] in nats, and the top_k
 * (<= HQ_LOGPROBS_MAX_TOP, <= V) likeliest tokens with their log probabilities, likeliest first, equal logits by the lower
 * token. logp, entropy, top_ids and top_logp may each be NULL (top_ids and top_logp as they are wanted). fp32 throughout.
 * A barred token has the logit -inf: log probability -inf, no part in the entropy. A row of nothing but -inf gives -inf
 * everywhere and entropy 0; a row with a NaN or +inf gives NaN everywhere (its top_ids put NaN first, then +inf).
 * Its workspace belongs to (device, stream), grows on first use of a larger shape, and goes with hq_stream_destroy; a captured call keeps the
 * one that it was captured with until then (capture after an eager call of the shape on the stream; graphs captured on one stream run one at
 * a time). */
int hq_logprobs(const void *logits, int f32, int M, uint32_t V, int64_t stride, const uint32_t *ids, int n_ids, int top_k,
                float *logp, float *entropy, uint32_t *top_ids, float *top_logp, void *stream);

/* ---- layers with a recurrent state: gated delta attention
 *
 * Such a layer keeps, in place of keys and values, one matrix S (k_dim x v_dim) for each value head and sequence, and the last
 * inputs of a causal convolution. Both lie in slots of the caller's memory; a step reads each sequence's slot and writes the same
 * or another one, so that a sequence that branches (a beam, a second sample) costs no copy. hq_scan_set describes a step once;
 * every such layer then calls hq_delta_append (convolution, norms and gates of the projections) and hq_delta (the recurrence). */
typedef struct {
    int n_k_heads, n_v_heads; /* queries and keys; values: a multiple, value head h takes key head h / (n_v_heads / n_k_heads) */
    int k_dim, v_dim;         /* multiples of 16, 16 .. 256 */
    int conv_taps;            /* 1 .. 8 */
    uint32_t n_slots;         /* below 2^31 */
    /* fp32, 16-byte aligned: S of slot i and head h at s + (i * n_v_heads + h) * k_dim * v_dim, v_dim contiguous; the inputs of
     * slot i at conv + i * (conv_taps - 1) * channels, rows of channels = 2 n_k_heads k_dim + n_v_heads v_dim, the oldest first */
    float *s, *conv;
} hq_state_t;

/* A step's sequences, for up to max_seqs of them and max_tokens new tokens in all. hq_scan_free waits for the device. */
typedef struct hq_scan hq_scan;
int hq_scan_create(int device, int max_seqs, int max_tokens, hq_scan **out);
void hq_scan_free(hq_scan *c);
/* Describes a step (host arrays, copied): sequence i has n_new[i] new tokens (0 or more; the step's tokens are numbered sequence
 * after sequence), goes on from the state in slot from[i] (-1: begins, all zeros) and leaves the state behind them in slot to[i]
 * (-1: nowhere). Without new tokens the state is copied. Several sequences may go on from one slot. No two leave theirs in one
 * slot, nor in a slot that another goes on from. st: the geometry (its pointers may differ in each call that follows). Plans the
 * work and grows the workspace: allocation, waiting and order as with hq_batch_set (steps that overlap in time need descriptions of
 * their own; a captured graph of a step's calls is good until the next hq_scan_set). */
int hq_scan_set(hq_scan *c, const hq_state_t *st, int n_seqs, const int32_t *n_new, const int32_t *from, const int32_t *to, void *stream);

typedef struct {
    /* the new tokens' projections, fp16 (f32 = 0) or fp32: channels of token t at x + t * x_stride in the order query heads, key
     * heads, value heads; n_v_heads values each at a and b + t * ab_stride. x 16-byte aligned, x_stride a multiple of 8. */
    const void *x, *a, *b;
    int f32;
    int64_t x_stride, ab_stride;
    const float *conv_w;         /* [channels, conv_taps] on the device, the newest input's tap last; 16-byte aligned */
    const float *a_log, *dt_bias; /* [n_v_heads] on the device */
    float eps;
    uint16_t *qkv;               /* [tokens, channels] fp16, 16-byte aligned */
    float *decay, *beta;         /* [tokens, n_v_heads] */
} hq_delta_in_t;

/* For every new token: y = silu(sum_j conv_w[j] x[t - (conv_taps - 1) + j]) over the sequence's inputs (the slot's before its
 * first new one), heads of queries and keys divided by sqrt(sum y^2 + eps), to qkv; decay = -e^a_log softplus(a + dt_bias), the
 * logarithm of the state's decay; beta = 1 / (1 + e^-b). Each sequence's last conv_taps - 1 inputs to its slot. fp32 arithmetic,
 * results rounded once. Outputs must not overlap inputs. One kernel. */
int hq_delta_append(const hq_scan *c, const hq_state_t *st, const hq_delta_in_t *r, void *stream);

typedef struct {
    /* fp16: head h of token t at q and k + t * qk_stride + h * k_dim, v + t * v_stride + h * v_dim; 16-byte aligned, strides
     * multiples of 8, those and out_stride no less than the heads of a token (and at most 2^22 where a sequence has more than 8
     * new tokens) */
    const uint16_t *q, *k, *v;
    int64_t qk_stride, v_stride;
    const float *decay, *beta; /* [tokens, n_v_heads]; decay: a logarithm, 0 or less, -inf allowed */
    float scale;               /* of the outputs, 1 / sqrt(k_dim) as a rule */
    /* optional norm and output gate: out = o / sqrt(mean(o^2) + eps) * norm * gate / (1 + e^-gate), over each head's v_dim; norm
     * fp32 [v_dim] on the device, gate fp16 or fp32 (gate_f32), head h of token t at gate + t * gate_stride + h * v_dim; both or
     * neither, 16-byte aligned, gate_stride a multiple of 8 */
    const float *norm;
    const void *gate;
    int gate_f32;
    int64_t gate_stride;
    float eps;
    uint16_t *out; /* fp16, head h of token t at out + t * out_stride + h * v_dim; 16-byte aligned, out_stride a multiple of 8 */
    int64_t out_stride;
} hq_delta_t;

/* For every new token, value head and its key head, from the sequence's state: S' = e^decay S; S = S' + k (beta (v - S'^T k))^T;
 * o = scale S^T q. States to their slots. Keys are to have a norm of at most 1 and beta to lie in 0 .. 1 (as hq_delta_append gives
 * them): the recurrence itself grows without bound otherwise. States and sums are fp32; sequences of more than 16 new tokens (fewer,
 * where it is the faster way) are taken in chunks of 64 tokens from their first, as products on the matrix cores whose operands are two
 * fp16 terms each (2^-22 of a column's largest, of a chunk's strengths of the chunk's largest). Outputs are rounded once, behind the norm. A value that is
 * not a number stays in its value column (and head, with the norm), but there it may reach outputs of its chunk's earlier tokens. The
 * same step gives the same bits. out must not overlap what is read. Kernels in a row, no allocation. */
int hq_delta(const hq_scan *c, const hq_state_t *st, const hq_delta_t *d, void *stream);

/* ---- pages of sequences that branch and end */
/* Which pages of a cache each of max_seqs sequences holds (host memory only; one thread at a time). Pages that several sequences
 * share are counted; a page goes back to the pool with its last holder. */
typedef struct hq_pages hq_pages;
int hq_pages_create(uint32_t n_pages, int page_size, int max_seqs, hq_pages **out);
void hq_pages_free(hq_pages *p);
/* Sequence seq has n_pos positions from now on, of which it keeps the first n_keep (at most n_pos and those it has): pages are
 * taken from the pool, the lowest first, or go back to it (0, 0: all of them). Where positions behind n_keep lie in a page that
 * others hold too, the sequence gets one of its own in its place, with a copy of what it keeps there (hq_pages_copies). Too few
 * pages in the pool, with those that it gives back itself: -1, and nothing is changed. */
int hq_pages_resize(hq_pages *p, int seq, int n_keep, int n_pos);
/* child, which must have no positions, gets the first n_pos of parent's and shares their pages. */
int hq_pages_fork(hq_pages *p, int parent, int child, int n_pos);
/* Pages are moved so that those held are the lowest ones. No copies may wait (hq_pages_copies). */
int hq_pages_compact(hq_pages *p);
/* The copies that resize and compact have asked for since the last call of this function, as hq_kv_copy takes them; they must run
 * before a step reads or writes the pages. The arrays belong to p, until its next call. A page that a waiting copy reads is in
 * nobody's hands again only after this call. */
int hq_pages_copies(hq_pages *p, const uint32_t **src, const uint32_t **dst, const int32_t **n_pos, int *n);
/* The pages of n sequences as rows of hq_batch_set's table: row i, pages_ld wide, those of seqs[i] (places behind them: 0). */
int hq_pages_table(const hq_pages *p, const int32_t *seqs, int n, uint32_t *pages, int pages_ld);
/* A sequence's positions, and the pages that resize could take now. Either may be NULL. */
int hq_pages_count(const hq_pages *p, int seq, int *n_pos, uint32_t *n_free);

/* Positions 0 .. n_pos[i] - 1 (n_pos NULL: all) of page src[i] to page dst[i], i < n, in the n_kv caches of kv (layers of one
 * geometry): keys, values and scales. src, dst, n_pos are the host's; all n copies are as if at once: no dst may be another's dst
 * or any src. Asynchronous; the arrays may change when the call returns. */
int hq_kv_copy(const hq_kv_t *kv, int n_kv, const uint32_t *src, const uint32_t *dst, const int32_t *n_pos, int n, void *stream);

/* ---- beam search */
#define HQ_BEAM_MAX 64 /* beams of a group, and candidates chosen */
/* The k best continuations of each of n_groups groups of n_beams beams. Row i * n_beams + j of the logits (fp16, or fp32 with f32;
 * V each, row m at logits + m * stride) and score[i * n_beams + j] belong to beam j of group i; its candidates are the tokens v
 * with the value score + log softmax(row)[v]. A beam with done != 0 (done may be NULL) has the one candidate done_token, with its
 * score as the value. To out_score, out_token and out_beam [n_groups, k], best first, equal values by the lower beam; of one
 * beam's, whose values may be equal where its logits are not (next to a score of -1e30, say), the larger logit, then the lower token; candidates of -inf (barred tokens, beams with a score of -inf) are none, and places beyond the last candidate get
 * -inf, UINT32_MAX and -1. Rows of done beams and of those with a score of -inf are not read. A NaN or +inf in a group's scores or
 * in a row that is read: NaN, UINT32_MAX and -1 in all of the group's places. Values are formed and compared in 64 bits from 32-bit
 * exponentials. Its workspace belongs to (device, stream) as hq_logprobs' does. score and
 * the outputs must not overlap. */
int hq_beam(const void *logits, int f32, int n_groups, int n_beams, uint32_t V, int64_t stride, const float *score, const uint8_t *done,
            uint32_t done_token, int k, float *out_score, uint32_t *out_token, int32_t *out_beam, void *stream);

#ifdef __cplusplus
}
#endif
#endif
