/*
 * sera_attn.h - C ABI of the paged key/value cache and its attention on
 * MI355X (gfx950): what a decoder layer runs between the q/k/v products and
 * the o product of sera_q4k.h.
 *
 * The conventions are those of sera_q4k.h: plain C types, device pointers,
 * a stream is a hipStream_t passed as void* (NULL = the null stream). Every
 * function enqueues on the given stream and returns without synchronizing;
 * none allocates device memory, so all of them can be captured into a graph.
 * Return codes: 0 success, -1 invalid arguments, -3 launch failed;
 * sera_q4k_last_error() gives the message. No other set-up call is needed.
 *
 * The cache: `pages` pages of page_tokens tokens in one allocation. A page
 * is one run of sera_kv_page_bytes() bytes (page p starts at data + p * that,
 * so a page is copied as bytes); inside it each kv head has one run
 *
 *   K        [page_tokens][head_dim]            elements
 *   V        [page_tokens / 16][head_dim][16]   elements
 *   K scale  [page_tokens] float                SERA_KV_Q8 only
 *   V scale  [page_tokens] float                SERA_KV_Q8 only
 *
 * (16 tokens of one V channel lie side by side, the order in which the
 * products take them). Elements:
 *
 *   SERA_KV_F16  fp16, rounded to nearest even
 *   SERA_KV_Q8   int8 codes and one float scale for each token and kv head,
 *                separately for K and V: scale = max|x| / 127, code =
 *                x / scale rounded to nearest even (the quotient exact), a
 *                value stands for code * scale. A zero vector has scale 0; a
 *                vector with an infinity or NaN reads back as NaN.
 *
 * A page may be in the tables of several sequences (a shared prefix): the
 * calls read it for each of them. Two sequences of one write must not have
 * new rows in the same page slot.
 */
#ifndef SERA_ATTN_H
#define SERA_ATTN_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of rows (q, k, v, out), by their GGUF type ids. */
#define SERA_TYPE_F32 0u
#define SERA_TYPE_F16 1u
#define SERA_TYPE_BF16 30u

/* Cache types: GGUF's id for fp16, and 256 + GGUF's Q8_0 for this library's
 * 8-bit layout. */
#define SERA_KV_F16 1u
#define SERA_KV_Q8 264u

typedef struct {
    uint32_t type;         /* SERA_KV_F16 or SERA_KV_Q8 */
    int32_t page_tokens;   /* a power of two, 16..1024 */
    int32_t kv_heads;      /* 1..1024 */
    int32_t head_dim;      /* 64 or 128 */
    int64_t pages;
    void *data;            /* device, 16-byte aligned, pages * page bytes */
} sera_kv_cache;

/* Sequences of one call. Their new rows are packed one after the other in
 * the row operands: sequence b has rows row_start[b] .. row_start[b+1]-1,
 * which are the last positions of its kv_len[b] positions. Position j of
 * sequence b lies in page page_table[b * table_stride + j / page_tokens].
 * The three arrays are device memory and are read when the work runs, so a
 * replayed graph takes the lengths that are there then; the bounds max_new
 * and max_kv are the host's, and hold for every such run. The host cannot
 * check the arrays, the kernels do: a sequence whose rows or length are
 * outside the bounds writes nothing and its rows (those inside [0, rows)) come
 * out as NaN; where row_start decreases, sequences overlap and what the batch's
 * rows come out as is not defined (some may be left as they are); a page id outside [0, pages) is never followed: its tokens are
 * not written, and read as NaN. Positions below zero (a sequence with more
 * rows than length) are not written, and read as zeros. */
typedef struct {
    int32_t sequences;
    int32_t rows;          /* packed rows in the operands */
    int32_t max_new;       /* most new rows of one sequence */
    int32_t max_kv;        /* longest kv_len, <= table_stride * page_tokens */
    int64_t table_stride;  /* page_table entries from one sequence to the next */
    const int32_t *row_start;   /* [sequences + 1] */
    const int32_t *kv_len;      /* [sequences], new rows included */
    const int32_t *page_table;
} sera_kv_batch;

/* Bytes of one page; 0 for a type, page size, head count or head size that
 * the library does not have. */
size_t sera_kv_page_bytes(uint32_t type, int page_tokens, int kv_heads, int head_dim);

/* Writes the new rows' keys and values into the cache. k and v are [rows]
 * [kv_heads * head_dim] of `type`, with k_stride and v_stride elements from
 * one row to the next (views into a fused q/k/v buffer pass its width); rows
 * and strides are 16-byte aligned. */
int sera_kv_write(const sera_kv_cache *cache, const sera_kv_batch *batch, uint32_t type, const void *k,
                  int64_t k_stride, const void *v, int64_t v_stride, void *stream);

/* Reads the same positions back: the values that the cache stands for
 * (code * scale in fp32), rounded to `type`. A batch whose rows cover whole contexts
 * (row_start[b+1] - row_start[b] = kv_len[b]) reads those. */
int sera_kv_read(const sera_kv_cache *cache, const sera_kv_batch *batch, uint32_t type, void *k, int64_t k_stride,
                 void *v, int64_t v_stride, void *stream);

/* Scratch for sera_attention with these bounds and `heads` query heads on
 * the current device (0: none is needed, or the arguments are refused by the
 * call as well): partial sums of contexts that are split over workgroups, which
 * is done only as far as compute units would be idle. So it is bounded, by 39
 * MB on 256 compute units, and not monotone in the batch: one that fills the device
 * needs none, a smaller one may need more. */
size_t sera_attention_workspace_bytes(const sera_kv_cache *cache, const sera_kv_batch *batch, int heads);

/* out[row][head] = softmax(scale * q . K^T) V of each new row over its
 * sequence's cache, one token or a long chunk. q and out are [rows]
 * [heads * head_dim] of `type` with their own strides; query head h reads
 * kv head h / (heads / kv_heads). The row at position p sees the positions
 * j <= p; with window > 0 only j > p - window, and the first `sinks`
 * positions, which stay visible (a window of max_kv or more hides none). (The
 * new rows' keys and values are written before, by sera_kv_write.) A position
 * that a row does not see has no effect on it, whatever it holds. A row that
 * sees nothing comes out as zeros.
 *
 * Products run on fp16 matrix instructions with fp32 sums: for fp16 and bf16
 * rows with q and the softmax weights rounded once to fp16, for fp32 rows
 * with both split into two fp16 terms (22 bits), so the result keeps fp32's
 * accuracy against the cached values. A value that is not finite makes the rows
 * that see it not finite in its channel (an infinity may come out as NaN).
 *
 * Sequences may differ in rows: where most have a token or so and some have
 * long chunks, both kinds run in the kernel that suits them. A call makes one
 * to three launches.
 *
 * workspace: 16-byte aligned device scratch of at least
 * sera_attention_workspace_bytes(), used by one call at a time; its content
 * between calls does not matter. Results repeat bit for bit. */
int sera_attention(const sera_kv_cache *cache, const sera_kv_batch *batch, uint32_t type, const void *q,
                   int64_t q_stride, void *out, int64_t out_stride, int heads, float scale, int window, int sinks,
                   void *workspace, size_t workspace_bytes, void *stream);

/* ---- norm and rotation on the way into the cache ------------------------ */

/* Which channels of a head turn together: i and i + rotated/2, or 2i and
 * 2i + 1 (i < rotated/2). */
#define SERA_ROPE_HALVES 0
#define SERA_ROPE_NEIGHBOURS 1

/* What a layer's q and k heads go through: with a gamma, RMSNorm over the
 * head's channels,
 *   x' = (x * (1 / sqrt(mean(x^2) + eps))) * gamma,
 * then the first `rotated` channels are turned pair by pair:
 *   (a, b) -> (a cos t - b sin t, a sin t + b cos t),  t = position * inv_freq[i].
 * The angle is taken in 64 bits and reduced before it is rounded, so far
 * positions lose nothing; the rest is in fp32, rounded once to the rows' or the
 * cache's type. */
typedef struct {
    const float *inv_freq;  /* device, [rotated / 2]; may be NULL when nothing rotates */
    const float *q_gamma;   /* device, [head_dim], 16-byte aligned; NULL: q is not normed */
    const float *k_gamma;   /* the same for k */
    float eps;              /* 0 or more */
    int32_t rotated;        /* channels: 0, head_dim / 4, head_dim / 2 or head_dim */
    int32_t pairing;        /* SERA_ROPE_HALVES or SERA_ROPE_NEIGHBOURS */
} sera_qk_rope;

/* sera_kv_write of rows whose k heads are normed and rotated on the way, and
 * the same for q's heads, from q to q_out (rows of `type` with strides of their
 * own; q_out may be q with the same stride, and must not overlap it otherwise).
 * k and v are left as they are. `heads` (a multiple of kv_heads) is q's.
 * positions: device, [rows], the position that each row is rotated by, or NULL
 * for its place in the sequence. They differ where a cache was thinned
 * (sera_kv_evict) and its tokens have other places than they had in the text.
 * Rows of a sequence outside the bounds come out of q as NaN, those in front of
 * a sequence's start as zeros; rows of no sequence are left as they are. One
 * launch. */
int sera_kv_write_rope(const sera_kv_cache *cache, const sera_kv_batch *batch, const sera_qk_rope *rope, uint32_t type,
                       const void *q, int64_t q_stride, void *q_out, int64_t q_out_stride, int heads, const void *k,
                       int64_t k_stride, const void *v, int64_t v_stride, const int32_t *positions, void *stream);

/* ---- a cache of bounded length ------------------------------------------ */

/* sera_attention, which also adds up the weight that every position gets: for
 * sequence b, kv head h and position j < kv_len[b]
 *   weights[b][h][j] = before[b][h][j] + sum of the softmax weights of j over
 *                      the sequence's new rows and h's query heads,
 * where `before` counts for positions in front of the new rows only: the new
 * ones start at zero, whatever their places held. Both are device float arrays
 * [sequences][kv_heads][weights_stride] (weights_stride >= max_kv); `before`
 * may be `weights` (the sums go on in place) or NULL (they start with this
 * call), and must not overlap it otherwise. Places from kv_len on are left as
 * they are, and so is all of a sequence outside the bounds. Rows whose scores
 * have no softmax (one that is NaN or +inf, or all of them -inf: a lost page,
 * keys that are not finite) give NaN to the positions that they see. A batch
 * without rows does nothing. kv_heads * max_kv is to stay below 2^34 (one
 * launch makes the sums). Results repeat bit for bit. The
 * workspace is its own size, which grows with rows * heads * max_kv where few
 * rows go to long contexts (their scores are kept for the sums, 4 bytes each).
 */
size_t sera_attention_weights_workspace_bytes(const sera_kv_cache *cache, const sera_kv_batch *batch, int heads);
int sera_attention_weights(const sera_kv_cache *cache, const sera_kv_batch *batch, uint32_t type, const void *q,
                           int64_t q_stride, void *out, int64_t out_stride, int heads, float scale, int window,
                           int sinks, const float *before, float *weights, int64_t weights_stride, void *workspace,
                           size_t workspace_bytes, void *stream);

/* Shortens every sequence of more than `keep` positions to `keep`: of each kv
 * head the first `sinks` positions stay, the last `recent` ones, and of those
 * between the ones with the largest weights (of equal ones the first; NaN
 * counts as less than anything), keep - sinks - recent of them. What stays
 * keeps its order and moves, with its bytes, to the places 0, 1, .. of the
 * pages in new_table [sequences][new_stride] (new_stride * page_tokens >=
 * min(keep, max_kv)); its weights move to the same places of new_weights (both
 * [sequences][kv_heads][weights_stride], not overlapping; places behind are
 * left as they are). A sequence of up to `keep` positions moves as it is.
 * new_len[b] is the new length, kept [sequences][kv_heads][keep] the old
 * positions in order, -1 behind the last. Of the batch only sequences, max_kv,
 * table_stride, kv_len and page_table are used.
 *
 * The new pages belong to one sequence each and are not among the old ones of
 * any (they take the bytes while others still read theirs), so old pages may go
 * on being shared; but a sequence of up to `keep` positions may name its own
 * old pages again, in the same order. new_len must not overlap kv_len. A
 * sequence whose length is outside 0..max_kv moves nothing, has new_len -1 and
 * only -1 in kept; tokens of a page that is not in the pool arrive as NaN, and
 * to a new page that is not none are written. kv_heads * min(keep, max_kv) is
 * to stay below 2^29 (one launch moves it). Two launches. */
int sera_kv_evict(const sera_kv_cache *cache, const sera_kv_batch *batch, int keep, int recent, int sinks,
                  const float *weights, float *new_weights, int64_t weights_stride, const int32_t *new_table,
                  int64_t new_stride, int32_t *new_len, int32_t *kept, void *stream);

#ifdef __cplusplus
}
#endif

#endif
