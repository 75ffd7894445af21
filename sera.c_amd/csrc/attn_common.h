/*
 * attn_common.h - what the attention kernels take beside the cache and the
 * batch, and their launchers (internal).
 */
#ifndef SERA_ATTN_COMMON_H
#define SERA_ATTN_COMMON_H

#include "kv_common.h"

struct attn_args {
    const void *q;
    void *out;
    int64_t q_stride, out_stride;   /* elements */
    int heads, group;               /* query heads, query heads per kv head */
    float scale_log2;               /* scale * log2(e) */
    int window, sinks;              /* window 0: none */
    int few_columns;                /* sequences of up to this many rows x group go to the few-row kernel, others to
                                     * the tile kernel */
    int few_rows;                   /* rows of one of its partial results */
    float *workspace;
    int cus;                        /* compute units of the device */
};

/* How a kernel's part of a call is cut up, in 32-token tiles. */
struct attn_plan {
    int columns;         /* rows of q (tokens x heads of a group) that a workgroup has; 0: the kernel has no part */
    int waves;           /* few-row kernel: of a workgroup */
    int slots;           /* tile kernel: row tiles, of `columns` rows each, at most */
    int splits, chunk;   /* workgroups over a context, tiles of each */
};
constexpr int kAttnShift = 5;       /* log2 of a tile's tokens */

hipError_t sera_launch_kv_move(bool write, uint32_t cache_type, uint32_t type, int dim, const kv_args &a, void *k,
                               int64_t k_stride, void *v, int64_t v_stride, hipStream_t s);
size_t sera_attn_workspace(const kv_args &a, int dim, int heads, int cus);
hipError_t sera_launch_attn_few(uint32_t cache_type, uint32_t type, int dim, const kv_args &a, const attn_args &t,
                                const attn_plan &p, hipStream_t s);
hipError_t sera_launch_attn(uint32_t cache_type, uint32_t type, int dim, const kv_args &a, const attn_args &t,
                            hipStream_t s);
hipError_t sera_launch_attn_tile(uint32_t cache_type, uint32_t type, int dim, const kv_args &a, const attn_args &t,
                                 const attn_plan &p, hipStream_t s);

#endif
