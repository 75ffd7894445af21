/*
 * sera_attn_runtime.hip - host side of include/sera_attn.h and
 * include/sera_logprobs.h: argument checks and launches. Nothing here allocates device memory or synchronizes.
 */
#include "attn_common.h"
#include "logprobs.h"
#include "sera_launch.h"

#include "../../include/sera_logprobs.h"

#include <math.h>
#include <stdarg.h>
#include <stdio.h>

namespace {

int fail(int code, const char *fmt, ...) {
    char msg[240];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(msg, sizeof(msg), fmt, ap);
    va_end(ap);
    return sera_report_error(code, msg);
}

bool type_ok(uint32_t type) { return type == SERA_TYPE_F32 || type == SERA_TYPE_F16 || type == SERA_TYPE_BF16; }
int type_bytes(uint32_t type) { return type == SERA_TYPE_F32 ? 4 : 2; }

constexpr int kMaxPageTokens = 1024, kMaxKvHeads = 1024, kMaxHeads = 16384;
constexpr int64_t kMaxPages = 0x7fffffff;
/* Positions, rows and grid units are 32-bit in the kernels, with tile ends
 * and rows * group past them: both stay far below 2^31. */
constexpr int kMaxPositions = 1 << 28, kMaxRows = 1 << 22, kMaxSequences = 1 << 20;

bool geometry_ok(uint32_t type, int page_tokens, int kv_heads, int head_dim) {
    return (type == SERA_KV_F16 || type == SERA_KV_Q8) && page_tokens >= 16 && page_tokens <= kMaxPageTokens &&
           (page_tokens & (page_tokens - 1)) == 0 && kv_heads >= 1 && kv_heads <= kMaxKvHeads &&
           (head_dim == 64 || head_dim == 128);
}

/* The kernels' view of cache and batch. */
kv_args args_of(const sera_kv_cache *c, const sera_kv_batch *b) {
    kv_args a;
    a.data = (uint8_t *)c->data;
    a.head_bytes = kv_head_bytes(c->type, c->page_tokens, c->head_dim);
    a.page_bytes = (size_t)a.head_bytes * (size_t)c->kv_heads;
    a.page_shift = __builtin_ctz((unsigned)c->page_tokens);
    a.pages = (int)c->pages;
    a.kv_heads = c->kv_heads;
    a.sequences = b->sequences;
    a.rows = b->rows;
    a.max_new = b->max_new;
    a.max_kv = b->max_kv;
    a.table_stride = b->table_stride;
    a.row_start = b->row_start;
    a.kv_len = b->kv_len;
    a.table = b->page_table;
    return a;
}

/* 0, or a failure: of the cache's form... */
int check_cache(const char *tag, const sera_kv_cache *c, const sera_kv_batch *b) {
    if (!c || !b) return fail(-1, "%s: null cache or batch", tag);
    if (!geometry_ok(c->type, c->page_tokens, c->kv_heads, c->head_dim))
        return fail(-1, "%s: cache type %u, %d tokens a page, %d kv heads of %d: want type %u or %u, a power of two "
                    "16..%d, 1..%d heads of 64 or 128", tag, c->type, c->page_tokens, c->kv_heads, c->head_dim,
                    SERA_KV_F16, SERA_KV_Q8, kMaxPageTokens, kMaxKvHeads);
    return 0;
}

/* ... of its memory... */
int check_pool(const char *tag, const sera_kv_cache *c) {
    if (c->pages < 1 || c->pages > kMaxPages) return fail(-1, "%s: %lld pages", tag, (long long)c->pages);
    if (!c->data || ((uintptr_t)c->data & 15u))
        return fail(-1, "%s: the cache's data must be a 16-byte aligned device pointer", tag);
    return 0;
}

/* ... and of the sequences' lengths and pages. */
int check_lengths(const char *tag, const sera_kv_cache *c, const sera_kv_batch *b) {
    if (b->max_kv < 1 || b->max_kv > kMaxPositions || b->table_stride < 1 ||
        b->table_stride < ((int64_t)b->max_kv + c->page_tokens - 1) / c->page_tokens)
        return fail(-1, "%s: max_kv=%d outside 1..%d, or over %lld table entries of %d tokens", tag, b->max_kv,
                    kMaxPositions, (long long)b->table_stride, c->page_tokens);
    if (!b->kv_len || !b->page_table) return fail(-1, "%s: null kv_len or page_table", tag);
    if (((uintptr_t)b->kv_len & 3u) || ((uintptr_t)b->page_table & 3u))
        return fail(-1, "%s: kv_len and page_table must be 4-byte aligned", tag);
    return 0;
}

/* 0, or a failure. *empty: there are no rows, nothing is to be launched. */
int check(const char *tag, const sera_kv_cache *c, const sera_kv_batch *b, bool *empty) {
    if (check_cache(tag, c, b)) return -1;
    if (b->sequences < 0 || b->sequences > kMaxSequences || b->rows < 0 || b->rows > kMaxRows)
        return fail(-1, "%s: %d rows of %d sequences outside 0..%d and 0..%d", tag, b->rows, b->sequences, kMaxRows,
                    kMaxSequences);
    *empty = b->rows == 0;
    if (*empty) return 0;
    if (b->sequences == 0) return fail(-1, "%s: %d rows of no sequence", tag, b->rows);
    if (check_pool(tag, c)) return -1;
    if (b->max_new < 1 || b->max_new > b->rows)
        return fail(-1, "%s: max_new=%d outside 1..%d rows", tag, b->max_new, b->rows);
    if (!b->row_start || ((uintptr_t)b->row_start & 3u))
        return fail(-1, "%s: row_start is null or not 4-byte aligned", tag);
    return check_lengths(tag, c, b);
}

int check_rows(const char *tag, const char *name, uint32_t type, const void *p, int64_t stride, int64_t width) {
    if (!p) return fail(-1, "%s: null %s", tag, name);
    if (stride < width || stride > ((int64_t)1 << 40)) return fail(-1, "%s: %s rows of %lld elements %lld apart", tag,
                                                                   name, (long long)width, (long long)stride);
    if (((uintptr_t)p & 15u) || (stride * type_bytes(type)) % 16)
        return fail(-1, "%s: %s and its row stride must be 16-byte aligned", tag, name);
    return 0;
}

int move(bool write, const sera_kv_cache *c, const sera_kv_batch *b, uint32_t type, void *k, int64_t ks, void *v,
         int64_t vs, void *stream) {
    const char *tag = write ? "sera_kv_write" : "sera_kv_read";
    bool empty;
    if (check(tag, c, b, &empty)) return -1;
    if (!type_ok(type)) return fail(-1, "%s: row type %u is not F32, F16 or BF16", tag, type);
    if (empty) return 0;
    const int64_t width = (int64_t)c->kv_heads * c->head_dim;
    if (check_rows(tag, "k", type, k, ks, width) || check_rows(tag, "v", type, v, vs, width)) return -1;
    return sera_launch_kv_move(write, c->type, type, c->head_dim, args_of(c, b), k, ks, v, vs,
                               (hipStream_t)stream) == hipSuccess ? 0 : fail(-3, "%s: launch failed", tag);
}

/* Compute units of the current device, kept per device. */
int device_cus() {
    static int known[64];
    int d = 0, n = 0;
    if (hipGetDevice(&d) != hipSuccess || d < 0 || d >= 64) return 256;
    if (known[d]) return known[d];
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, d) != hipSuccess || n < 1) return 256;
    known[d] = n;
    return n;
}

bool overlap(const void *a, const void *b, int64_t bytes) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return (x < y ? y - x : x - y) < (uintptr_t)bytes;
}

/* Two arrays of sums, one for each of `arrays` (sequence, kv head). */
int check_weights(const char *tag, const float *a, const float *b, int64_t arrays, int64_t stride, int max_kv) {
    if (!a || !b || ((uintptr_t)a & 3u) || ((uintptr_t)b & 3u))
        return fail(-1, "%s: weights must be 4-byte aligned device pointers", tag);
    if (stride < max_kv || stride > ((int64_t)1 << 40) / arrays)
        return fail(-1, "%s: weights of %d positions %lld apart", tag, max_kv, (long long)stride);
    return 0;
}

size_t workspace_of(const sera_kv_cache *cache, const sera_kv_batch *batch, int heads, bool weigh) {
    if (!cache || !batch || !geometry_ok(cache->type, cache->page_tokens, cache->kv_heads, cache->head_dim)) return 0;
    if (heads < 1 || heads > kMaxHeads || heads % cache->kv_heads) return 0;
    if (batch->rows < 1 || batch->rows > kMaxRows || batch->sequences < 1 || batch->sequences > kMaxSequences ||
        batch->max_new < 1 || batch->max_new > batch->rows || batch->max_kv < 1 || batch->max_kv > kMaxPositions)
        return 0;
    return sera_attn_workspace(args_of(cache, batch), cache->head_dim, heads, device_cus(), weigh);
}

/* Attention; with `weigh`, the sums of its weights. */
int attend(const char *tag, const sera_kv_cache *cache, const sera_kv_batch *batch, uint32_t type, const void *q,
           int64_t q_stride, void *out, int64_t out_stride, int heads, float scale, int window, int sinks, bool weigh,
           const float *before, float *weights, int64_t weights_stride, void *workspace, size_t workspace_bytes,
           void *stream) {
    bool empty;
    if (check(tag, cache, batch, &empty)) return -1;
    if (!type_ok(type)) return fail(-1, "%s: row type %u is not F32, F16 or BF16", tag, type);
    if (heads < 1 || heads > kMaxHeads || heads % cache->kv_heads)
        return fail(-1, "%s: %d query heads over %d kv heads", tag, heads, cache->kv_heads);
    if (window < 0 || sinks < 0) return fail(-1, "%s: window=%d, sinks=%d below zero", tag, window, sinks);
    if (!isfinite(scale)) return fail(-1, "%s: the scale is not finite", tag);
    if (empty) return 0;
    if ((int64_t)batch->rows * heads > 0x7fffffff - (weigh ? 63 : 0))      /* the sums go by blocks of 32 columns */
        return fail(-1, "%s: %d rows of %d heads reach 2^31", tag, batch->rows, heads);
    const int64_t width = (int64_t)heads * cache->head_dim;
    if (check_rows(tag, "q", type, q, q_stride, width) || check_rows(tag, "out", type, out, out_stride, width))
        return -1;
    if (weigh) {
        const int64_t sums = (int64_t)batch->sequences * cache->kv_heads;
        if (cache->kv_heads * (((int64_t)batch->max_kv + 1023) / 1024) > kAttnMaxGrid)
            return fail(-1, "%s: %d positions of %d kv heads are more than one launch sums", tag, batch->max_kv,
                        cache->kv_heads);
        if (check_weights(tag, before ? before : weights, weights, sums, weights_stride, batch->max_kv)) return -1;
        if (before && before != weights && overlap(before, weights, sums * weights_stride * 4))
            return fail(-1, "%s: before and weights overlap and are not the same", tag);
    }
    const kv_args a = args_of(cache, batch);
    attn_args t = {};
    t.q = q;
    t.out = out;
    t.q_stride = q_stride;
    t.out_stride = out_stride;
    t.heads = heads;
    t.group = heads / cache->kv_heads;
    t.scale_log2 = (float)((double)scale * 1.4426950408889634);
    /* A window of all positions is none. Below that it is under kMaxPositions, so p - window stays inside an int for
     * every position p of a row, those in front of a sequence's start (p >= -kMaxRows) among them. */
    t.window = window < batch->max_kv ? window : 0;
    t.sinks = sinks;
    t.workspace = (float *)workspace;
    t.cus = device_cus();
    const size_t need = workspace_of(cache, batch, heads, weigh);
    if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15u)))
        return fail(-1, "%s: the workspace must be 16-byte aligned and hold %zu bytes (%zu given)", tag, need,
                    workspace ? workspace_bytes : (size_t)0);
    if (weigh) {
        t.before = before;
        t.weights = weights;
        t.weights_stride = weights_stride;
    }
    return sera_launch_attn(cache->type, type, cache->head_dim, a, t, (hipStream_t)stream) == hipSuccess
               ? 0 : fail(-3, "%s: launch failed", tag);
}

}  // namespace

extern "C" {

size_t sera_kv_page_bytes(uint32_t type, int page_tokens, int kv_heads, int head_dim) {
    if (!geometry_ok(type, page_tokens, kv_heads, head_dim)) return 0;
    return (size_t)kv_head_bytes(type, page_tokens, head_dim) * (size_t)kv_heads;
}

int sera_kv_write(const sera_kv_cache *cache, const sera_kv_batch *batch, uint32_t type, const void *k,
                  int64_t k_stride, const void *v, int64_t v_stride, void *stream) {
    return move(true, cache, batch, type, (void *)k, k_stride, (void *)v, v_stride, stream);
}

int sera_kv_read(const sera_kv_cache *cache, const sera_kv_batch *batch, uint32_t type, void *k, int64_t k_stride,
                 void *v, int64_t v_stride, void *stream) {
    return move(false, cache, batch, type, k, k_stride, v, v_stride, stream);
}

size_t sera_attention_workspace_bytes(const sera_kv_cache *cache, const sera_kv_batch *batch, int heads) {
    return workspace_of(cache, batch, heads, false);
}

size_t sera_attention_weights_workspace_bytes(const sera_kv_cache *cache, const sera_kv_batch *batch, int heads) {
    return workspace_of(cache, batch, heads, true);
}

int sera_attention(const sera_kv_cache *cache, const sera_kv_batch *batch, uint32_t type, const void *q,
                   int64_t q_stride, void *out, int64_t out_stride, int heads, float scale, int window, int sinks,
                   void *workspace, size_t workspace_bytes, void *stream) {
    return attend("sera_attention", cache, batch, type, q, q_stride, out, out_stride, heads, scale, window, sinks,
                  false, nullptr, nullptr, 0, workspace, workspace_bytes, stream);
}

int sera_attention_weights(const sera_kv_cache *cache, const sera_kv_batch *batch, uint32_t type, const void *q,
                           int64_t q_stride, void *out, int64_t out_stride, int heads, float scale, int window,
                           int sinks, const float *before, float *weights, int64_t weights_stride, void *workspace,
                           size_t workspace_bytes, void *stream) {
    return attend("sera_attention_weights", cache, batch, type, q, q_stride, out, out_stride, heads, scale, window,
                  sinks, true, before, weights, weights_stride, workspace, workspace_bytes, stream);
}

int sera_kv_write_rope(const sera_kv_cache *cache, const sera_kv_batch *batch, const sera_qk_rope *rope, uint32_t type,
                       const void *q, int64_t q_stride, void *q_out, int64_t q_out_stride, int heads, const void *k,
                       int64_t k_stride, const void *v, int64_t v_stride, const int32_t *positions, void *stream) {
    const char *tag = "sera_kv_write_rope";
    bool empty;
    if (check(tag, cache, batch, &empty)) return -1;
    if (!rope) return fail(-1, "%s: null rope", tag);
    if (!type_ok(type)) return fail(-1, "%s: row type %u is not F32, F16 or BF16", tag, type);
    if (heads < 1 || heads > kMaxHeads || heads % cache->kv_heads)
        return fail(-1, "%s: %d query heads over %d kv heads", tag, heads, cache->kv_heads);
    const int dim = cache->head_dim;
    if (rope->rotated != 0 && rope->rotated != dim && rope->rotated != dim / 2 && rope->rotated != dim / 4)
        return fail(-1, "%s: %d of %d channels rotate: want 0, a quarter, a half or all", tag, rope->rotated, dim);
    if (rope->pairing != SERA_ROPE_HALVES && rope->pairing != SERA_ROPE_NEIGHBOURS)
        return fail(-1, "%s: pairing %d is not HALVES or NEIGHBOURS", tag, rope->pairing);
    if (!(rope->eps >= 0.0f) || !isfinite(rope->eps)) return fail(-1, "%s: eps must be finite and 0 or more", tag);
    if (empty) return 0;
    if (rope->rotated && (!rope->inv_freq || ((uintptr_t)rope->inv_freq & 3u)))
        return fail(-1, "%s: inv_freq must be a 4-byte aligned device pointer", tag);
    if (((uintptr_t)rope->q_gamma & 15u) || ((uintptr_t)rope->k_gamma & 15u))
        return fail(-1, "%s: q_gamma and k_gamma must be 16-byte aligned", tag);
    if ((uintptr_t)positions & 3u) return fail(-1, "%s: positions must be 4-byte aligned", tag);
    const int64_t width = (int64_t)heads * dim, kv_width = (int64_t)cache->kv_heads * dim;
    if (check_rows(tag, "q", type, q, q_stride, width) || check_rows(tag, "q_out", type, q_out, q_out_stride, width) ||
        check_rows(tag, "k", type, k, k_stride, kv_width) || check_rows(tag, "v", type, v, v_stride, kv_width))
        return -1;
    if (q == q_out && q_stride != q_out_stride)
        return fail(-1, "%s: q_out is q with another stride (%lld and %lld)", tag, (long long)q_out_stride,
                    (long long)q_stride);
    rope_args r = {};
    r.inv_freq = rope->inv_freq;
    r.q_gamma = rope->q_gamma;
    r.k_gamma = rope->k_gamma;
    r.positions = positions;
    r.eps = rope->eps;
    r.half = rope->rotated / 2;
    r.neighbours = rope->pairing == SERA_ROPE_NEIGHBOURS;
    r.heads = heads;
    r.cus = device_cus();
    return sera_launch_kv_rope(cache->type, type, dim, args_of(cache, batch), r, q, q_stride, q_out, q_out_stride, k,
                               k_stride, v, v_stride, (hipStream_t)stream) == hipSuccess
               ? 0 : fail(-3, "%s: launch failed", tag);
}

int sera_kv_evict(const sera_kv_cache *cache, const sera_kv_batch *batch, int keep, int recent, int sinks,
                  const float *weights, float *new_weights, int64_t weights_stride, const int32_t *new_table,
                  int64_t new_stride, int32_t *new_len, int32_t *kept, void *stream) {
    const char *tag = "sera_kv_evict";
    if (check_cache(tag, cache, batch)) return -1;
    if (batch->sequences < 0 || batch->sequences > kMaxSequences)
        return fail(-1, "%s: %d sequences outside 0..%d", tag, batch->sequences, kMaxSequences);
    if (keep < 1 || keep > kMaxPositions || recent < 0 || sinks < 0 || (int64_t)recent + sinks > keep)
        return fail(-1, "%s: keep=%d of which recent=%d and sinks=%d: want 1..%d, and no more than that", tag, keep,
                    recent, sinks, kMaxPositions);
    if (batch->sequences == 0) return 0;
    if (check_pool(tag, cache) || check_lengths(tag, cache, batch)) return -1;
    const int64_t most = keep < batch->max_kv ? keep : batch->max_kv;
    if (new_stride < (most + cache->page_tokens - 1) / cache->page_tokens)
        return fail(-1, "%s: %lld new positions in %lld pages of %d tokens", tag, (long long)most,
                    (long long)new_stride, cache->page_tokens);
    if (cache->kv_heads * ((most + 31) / 32) > kAttnMaxGrid)
        return fail(-1, "%s: %lld positions that stay, of %d kv heads, are more than one launch moves", tag,
                    (long long)most, cache->kv_heads);
    if (!new_table || !new_len || !kept || ((uintptr_t)new_table & 3u) || ((uintptr_t)new_len & 3u) ||
        ((uintptr_t)kept & 3u))
        return fail(-1, "%s: new_table, new_len and kept must be 4-byte aligned device pointers", tag);
    if (overlap(new_len, batch->kv_len, (int64_t)batch->sequences * 4))
        return fail(-1, "%s: new_len must not overlap kv_len", tag);
    const int64_t sums = (int64_t)batch->sequences * cache->kv_heads;
    if (check_weights(tag, weights, new_weights, sums, weights_stride, batch->max_kv)) return -1;
    if (overlap(weights, new_weights, sums * weights_stride * 4))
        return fail(-1, "%s: weights and new_weights overlap", tag);
    evict_args t = {};
    t.keep = keep;
    t.recent = recent;
    t.sinks = sinks;
    t.weights = weights;
    t.new_weights = new_weights;
    t.weights_stride = weights_stride;
    t.new_table = new_table;
    t.new_stride = new_stride;
    t.new_len = new_len;
    t.kept = kept;
    return sera_launch_kv_evict(cache->type, cache->head_dim, args_of(cache, batch), t, (hipStream_t)stream) ==
                   hipSuccess ? 0 : fail(-3, "%s: launch failed", tag);
}

int sera_logprobs(uint32_t type, const void *logits, int64_t stride, int rows, int vocab, const int32_t *tokens,
                  int per_row, float *token_logprobs, float *entropy, int top, int32_t *top_ids, float *top_logprobs,
                  void *workspace, size_t workspace_bytes, void *stream) {
    const char *tag = "sera_logprobs";
    if (!type_ok(type)) return fail(-1, "%s: row type %u is not F32, F16 or BF16", tag, type);
    if (rows < 0 || rows > kMaxRows || vocab < 1 || vocab > kMaxPositions)
        return fail(-1, "%s: %d rows of %d outside 0..%d and 1..%d", tag, rows, vocab, kMaxRows, kMaxPositions);
    if (top < 0 || top > SERA_LOGPROBS_MAX_TOP || top > vocab)
        return fail(-1, "%s: top=%d outside 0..%d, or over the %d tokens", tag, top, SERA_LOGPROBS_MAX_TOP, vocab);
    if (per_row < 0 || (int64_t)per_row * rows > 0x7fffffff)
        return fail(-1, "%s: per_row=%d below zero, or over 2^31 tokens of %d rows", tag, per_row, rows);
    if (rows == 0 || (per_row == 0 && top == 0 && !entropy)) return 0;
    if (stride < vocab || stride > ((int64_t)1 << 40))
        return fail(-1, "%s: rows of %d elements %lld apart", tag, vocab, (long long)stride);
    if (!logits || ((uintptr_t)logits & (uintptr_t)(type_bytes(type) - 1)))
        return fail(-1, "%s: logits must be a device pointer aligned to its elements", tag);
    if (per_row && (!tokens || !token_logprobs || ((uintptr_t)tokens & 3u) || ((uintptr_t)token_logprobs & 3u)))
        return fail(-1, "%s: tokens and token_logprobs must be 4-byte aligned device pointers", tag);
    if (top && (!top_ids || !top_logprobs || ((uintptr_t)top_ids & 3u) || ((uintptr_t)top_logprobs & 3u)))
        return fail(-1, "%s: top_ids and top_logprobs must be 4-byte aligned device pointers", tag);
    if ((uintptr_t)entropy & 3u) return fail(-1, "%s: entropy must be 4-byte aligned", tag);
    const size_t need = sera_logprobs_workspace_bytes(rows, vocab, top);
    if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15u)))
        return fail(-1, "%s: the workspace must be 16-byte aligned and hold %zu bytes (%zu given)", tag, need,
                    workspace ? workspace_bytes : (size_t)0);
    logprobs_args p = {};
    p.logits = logits;
    p.stride = stride;
    p.rows = rows;
    p.vocab = vocab;
    p.tokens = tokens;
    p.per_row = per_row;
    p.token_logprobs = token_logprobs;
    p.entropy = entropy;
    p.top = top;
    p.top_ids = top_ids;
    p.top_logprobs = top_logprobs;
    p.splits = sera_logprobs_splits(rows, vocab, device_cus());
    p.sums = sera_logprobs_sums(rows, p.splits);
    p.workspace = (float *)workspace;
    return sera_launch_logprobs(type, p, (hipStream_t)stream) == hipSuccess ? 0 : fail(-3, "%s: launch failed", tag);
}

size_t sera_logprobs_workspace_bytes(int rows, int vocab, int top) {
    if (rows < 1 || rows > kMaxRows || vocab < 1 || vocab > kMaxPositions || top < 0 || top > SERA_LOGPROBS_MAX_TOP ||
        top > vocab)
        return 0;
    const int splits = sera_logprobs_splits(rows, vocab, device_cus());
    return splits < 2 ? 0 : sera_logprobs_sums(rows, splits) * 4 + (size_t)rows * splits * top * 8;
}

}  // extern "C"
