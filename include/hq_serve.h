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
 * Also plans hq_attention's work and grows its workspace: the only call of this header, with hq_batch_create and the
 * growing of hq_logprobs' workspace, that allocates. It waits until the last set's transfer is done, and with growing for
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
 * Its workspace belongs to (device, stream), grows on first use of a larger shape, and goes with hq_stream_destroy. */
int hq_logprobs(const void *logits, int f32, int M, uint32_t V, int64_t stride, const uint32_t *ids, int n_ids, int top_k,
                float *logp, float *entropy, uint32_t *top_ids, float *top_logp, void *stream);

#ifdef __cplusplus
}
#endif
#endif
