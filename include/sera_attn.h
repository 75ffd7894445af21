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

#ifdef __cplusplus
}
#endif

#endif
