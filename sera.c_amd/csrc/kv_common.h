/*
 * kv_common.h - the paged cache on the device: layout, batch lookup and
 * element conversions shared by the cache and the attention kernels
 * (internal; the layout itself is stated in include/sera_attn.h).
 */
#ifndef SERA_KV_COMMON_H
#define SERA_KV_COMMON_H

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/sera_attn.h"

/* What the kernels take of a sera_kv_cache and a sera_kv_batch. */
struct kv_args {
    uint8_t *data;
    size_t page_bytes;       /* one page, all kv heads */
    uint32_t head_bytes;     /* one kv head's run of a page */
    int page_shift;          /* log2(page_tokens) */
    int pages;
    int kv_heads;
    int sequences, rows, max_new, max_kv;
    int64_t table_stride;
    const int32_t *row_start, *kv_len, *table;
};

/* Bytes of one element; the head's run of a page. */
static inline uint32_t kv_head_bytes(uint32_t type, int page_tokens, int head_dim) {
    const uint32_t n = (uint32_t)page_tokens * (uint32_t)head_dim;
    return type == SERA_KV_F16 ? 4u * n : 2u * n + 8u * (uint32_t)page_tokens;
}

/* One sequence of a batch, checked against the host's bounds. */
struct kv_seq {
    int b;          /* sequence, or -1: none */
    int row0, n;    /* its packed rows */
    int len;        /* its positions */
    bool bad;       /* rows or length outside the bounds */
};

__device__ __forceinline__ kv_seq kv_sequence_of(const kv_args &a, int b, int r0, int r1, int len) {
    kv_seq s;
    s.b = b;
    s.bad = r0 < 0 || r1 < r0 || r1 > a.rows || r1 - r0 > a.max_new || len < 0 || len > a.max_kv;
    const int lo = min(max(r0, 0), a.rows), hi = min(max(r1, lo), a.rows);
    s.row0 = lo;
    s.n = hi - lo;
    s.len = len;
    return s;
}

__device__ __forceinline__ kv_seq kv_sequence(const kv_args &a, int b) {
    return kv_sequence_of(a, b, a.row_start[b], a.row_start[b + 1], a.kv_len[b]);
}

/* Grids over (sequence, unit of `per` rows) when only the packed rows' count
 * is known on the host: sequence b has the slots from row_start[b] / per +
 * extra * b on. That leaves it floor(n / per) + extra slots or more, in
 * floor(rows / per) + extra * sequences in all. Returns the sequence and the
 * unit in it of slot `slot` (wave-uniform): a 64-way search, one load of
 * row_start per level, a single one up to 64 sequences. With a scale, a unit
 * is `per` of rows * scale (which stays below 2^31). */
__device__ __forceinline__ int kv_find(const kv_args &a, int slot, int per, int extra, int *unit,
                                       int scale = 1) {
    const int lane = (int)(threadIdx.x & 63);
    int lo = 0, span = a.sequences;          /* the answer is in [lo, lo + span) */
    int base = 0;
    while (span > 0) {
        const int step = (span + 63) / 64;
        const int b = lo + lane * step;
        int key = 0x7fffffff;
        if (lane * step < span) {
            const int r = min(max(a.row_start[b], 0), a.rows);
            key = r * scale / per + extra * b;
        }
        const int hits = __popcll(__ballot(key <= slot));
        if (!hits) return -1;                /* unordered row_start */
        base = __shfl(key, hits - 1, 64);
        lo += (hits - 1) * step;
        if (step == 1) break;
        span = min(step, a.sequences - lo);
    }
    *unit = __builtin_amdgcn_readfirstlane(slot - base);
    if (*unit < 0) return -1;
    return __builtin_amdgcn_readfirstlane(lo);
}

/* kv_find and the sequence found (b -1: none). Up to 63 sequences the lanes hold all of row_start and kv_len after
 * one round of loads; otherwise the sequence is read after the search. */
__device__ __forceinline__ kv_seq kv_find_sequence(const kv_args &a, int slot, int per, int extra, int *unit) {
    kv_seq s;
    s.b = -1;
    if (a.sequences > 63) {
        const int b = kv_find(a, slot, per, extra, unit);
        return b < 0 ? s : kv_sequence(a, b);
    }
    const int lane = (int)(threadIdx.x & 63);
    const int r = lane <= a.sequences ? a.row_start[lane] : 0, len = lane < a.sequences ? a.kv_len[lane] : 0;
    const int key = lane < a.sequences ? min(max(r, 0), a.rows) / per + extra * lane : 0x7fffffff;
    const int b = __popcll(__ballot(key <= slot)) - 1;
    if (b < 0) return s;
    *unit = slot - __builtin_amdgcn_readlane(key, b);
    if (*unit < 0) return s;
    return kv_sequence_of(a, b, __builtin_amdgcn_readlane(r, b), __builtin_amdgcn_readlane(r, b + 1),
                          __builtin_amdgcn_readlane(len, b));
}

static inline int64_t kv_slots(int rows, int sequences, int per, int extra) {
    return (int64_t)rows / per + (int64_t)extra * sequences;
}

/* Row elements. */
__device__ __forceinline__ float kv_to_f32(float x) { return x; }
__device__ __forceinline__ float kv_to_f32(_Float16 x) { return (float)x; }
__device__ __forceinline__ float kv_to_f32(__bf16 x) { return (float)x; }
template <typename T>
__device__ __forceinline__ T kv_from_f32(float x) { return (T)x; }

#endif
