/*
 * sera_attn_runtime.hip - host side of include/sera_attn.h: argument checks
 * and launches. Nothing here allocates device memory or synchronizes.
 */
#include "attn_common.h"
#include "sera_launch.h"

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

/* 0, or a failure. *empty: there are no rows, nothing is to be launched. */
int check(const char *tag, const sera_kv_cache *c, const sera_kv_batch *b, bool *empty) {
    if (!c || !b) return fail(-1, "%s: null cache or batch", tag);
    if (!geometry_ok(c->type, c->page_tokens, c->kv_heads, c->head_dim))
        return fail(-1, "%s: cache type %u, %d tokens a page, %d kv heads of %d: want type %u or %u, a power of two "
                    "16..%d, 1..%d heads of 64 or 128", tag, c->type, c->page_tokens, c->kv_heads, c->head_dim,
                    SERA_KV_F16, SERA_KV_Q8, kMaxPageTokens, kMaxKvHeads);
    if (b->sequences < 0 || b->sequences > kMaxSequences || b->rows < 0 || b->rows > kMaxRows)
        return fail(-1, "%s: %d rows of %d sequences outside 0..%d and 0..%d", tag, b->rows, b->sequences, kMaxRows,
                    kMaxSequences);
    *empty = b->rows == 0;
    if (*empty) return 0;
    if (b->sequences == 0) return fail(-1, "%s: %d rows of no sequence", tag, b->rows);
    if (c->pages < 1 || c->pages > kMaxPages) return fail(-1, "%s: %lld pages", tag, (long long)c->pages);
    if (!c->data || ((uintptr_t)c->data & 15u))
        return fail(-1, "%s: the cache's data must be a 16-byte aligned device pointer", tag);
    if (b->max_new < 1 || b->max_new > b->rows)
        return fail(-1, "%s: max_new=%d outside 1..%d rows", tag, b->max_new, b->rows);
    if (b->max_kv < 1 || b->max_kv > kMaxPositions || b->table_stride < 1 ||
        b->table_stride < ((int64_t)b->max_kv + c->page_tokens - 1) / c->page_tokens)
        return fail(-1, "%s: max_kv=%d outside 1..%d, or over %lld table entries of %d tokens", tag, b->max_kv,
                    kMaxPositions, (long long)b->table_stride, c->page_tokens);
    if (!b->row_start || !b->kv_len || !b->page_table) return fail(-1, "%s: null row_start, kv_len or page_table", tag);
    if (((uintptr_t)b->row_start & 3u) || ((uintptr_t)b->kv_len & 3u) || ((uintptr_t)b->page_table & 3u))
        return fail(-1, "%s: row_start, kv_len and page_table must be 4-byte aligned", tag);
    return 0;
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
    if (!cache || !batch || !geometry_ok(cache->type, cache->page_tokens, cache->kv_heads, cache->head_dim)) return 0;
    if (heads < 1 || heads > kMaxHeads || heads % cache->kv_heads) return 0;
    if (batch->rows < 1 || batch->rows > kMaxRows || batch->sequences < 1 || batch->sequences > kMaxSequences ||
        batch->max_new < 1 || batch->max_new > batch->rows || batch->max_kv < 1 || batch->max_kv > kMaxPositions)
        return 0;
    return sera_attn_workspace(args_of(cache, batch), cache->head_dim, heads, device_cus());
}

int sera_attention(const sera_kv_cache *cache, const sera_kv_batch *batch, uint32_t type, const void *q,
                   int64_t q_stride, void *out, int64_t out_stride, int heads, float scale, int window, int sinks,
                   void *workspace, size_t workspace_bytes, void *stream) {
    const char *tag = "sera_attention";
    bool empty;
    if (check(tag, cache, batch, &empty)) return -1;
    if (!type_ok(type)) return fail(-1, "%s: row type %u is not F32, F16 or BF16", tag, type);
    if (heads < 1 || heads > kMaxHeads || heads % cache->kv_heads)
        return fail(-1, "%s: %d query heads over %d kv heads", tag, heads, cache->kv_heads);
    if (window < 0 || sinks < 0) return fail(-1, "%s: window=%d, sinks=%d below zero", tag, window, sinks);
    if (!isfinite(scale)) return fail(-1, "%s: the scale is not finite", tag);
    if (empty) return 0;
    if ((int64_t)batch->rows * heads > 0x7fffffff)
        return fail(-1, "%s: %d rows of %d heads reach 2^31", tag, batch->rows, heads);
    const int64_t width = (int64_t)heads * cache->head_dim;
    if (check_rows(tag, "q", type, q, q_stride, width) || check_rows(tag, "out", type, out, out_stride, width))
        return -1;
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
    const size_t need = sera_attn_workspace(a, cache->head_dim, heads, t.cus);
    if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15u)))
        return fail(-1, "%s: the workspace must be 16-byte aligned and hold %zu bytes (%zu given)", tag, need,
                    workspace ? workspace_bytes : (size_t)0);
    return sera_launch_attn(cache->type, type, cache->head_dim, a, t, (hipStream_t)stream) == hipSuccess
               ? 0 : fail(-3, "%s: launch failed", tag);
}

}  // extern "C"
