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
    float2 *norms;                  /* attn_norm of each row, [rows][heads], for the weights, or NULL */
    float *scores;                  /* s' of the few-row kernel, [sequences][kv_heads][pitch / 32][few_rows][32], or
                                     * NULL */
    size_t pitch;
    const float *before;            /* sums so far, or NULL */
    float *weights;                 /* [sequences][kv_heads][weights_stride] */
    int64_t weights_stride;
};

/* How the weights' sums are made. */
struct attn_sums {
    int few_rows;                   /* columns of a sequence in the few-row kernel, at most; 0: it has no part */
    int splits, chunk, dim;         /* of its partial results */
    size_t pitch;                   /* positions that scores have a place for, of each sequence */
    int groups, share;              /* of all other sequences: workgroups of a sequence and head at most, units
                                     * (blocks of 32 columns over 512 positions) of one */
    int64_t units;                  /* of a sequence and head, at most */
    size_t slots;                   /* places of 512 sums for a sequence and head */
    size_t scores_bytes;            /* of the workspace; the ranges' sums lie behind */
    float *scores, *partial;
};

/* Norm and rotation of q's and k's heads. */
struct rope_args {
    const float *inv_freq, *q_gamma, *k_gamma;
    const int32_t *positions;
    float eps;
    int half;                       /* pairs of channels that turn */
    bool neighbours;
    int heads;                      /* q's */
    int cus;                        /* compute units of the device */
};

/* What shortening a cache takes beside it and the batch. */
struct evict_args {
    int keep, recent, sinks;
    const float *weights;
    float *new_weights;
    int64_t weights_stride;
    const int32_t *new_table;
    int64_t new_stride;
    int32_t *new_len, *kept;
};

/* How a kernel's part of a call is cut up, in 32-token tiles. */
struct attn_plan {
    int columns;         /* rows of q (tokens x heads of a group) that a workgroup has; 0: the kernel has no part */
    int waves;           /* few-row kernel: of a workgroup */
    int slots;           /* tile kernel: row tiles, of `columns` rows each, at most */
    int splits, chunk;   /* workgroups over a context, tiles of each */
};
/* Workgroups of 256 threads in x: a launch has less than 2^32 threads there. */
constexpr int64_t kAttnMaxGrid = ((int64_t)1 << 24) - 1;
constexpr int kAttnShift = 5;       /* log2 of a tile's tokens */

hipError_t sera_launch_kv_move(bool write, uint32_t cache_type, uint32_t type, int dim, const kv_args &a, void *k,
                               int64_t k_stride, void *v, int64_t v_stride, hipStream_t s);
size_t sera_attn_workspace(const kv_args &a, int dim, int heads, int cus, bool weigh);
hipError_t sera_launch_attn_few(uint32_t cache_type, uint32_t type, int dim, const kv_args &a, const attn_args &t,
                                const attn_plan &p, hipStream_t s);
hipError_t sera_launch_attn(uint32_t cache_type, uint32_t type, int dim, const kv_args &a, const attn_args &t,
                            hipStream_t s);
hipError_t sera_launch_attn_tile(uint32_t cache_type, uint32_t type, int dim, const kv_args &a, const attn_args &t,
                                 const attn_plan &p, hipStream_t s);
attn_sums sera_attn_sums_plan(const kv_args &a, int few_rows, int group, int cus, size_t *bytes);
void sera_attn_sums_shorten(attn_sums &p, const kv_args &a, const attn_args &t, int group);
hipError_t sera_launch_attn_sums(uint32_t cache_type, uint32_t type, int dim, const kv_args &a, const attn_args &t,
                                 const attn_sums &p, bool many, hipStream_t s);
hipError_t sera_launch_kv_rope(uint32_t cache_type, uint32_t type, int dim, const kv_args &a, const rope_args &r,
                               const void *q, int64_t q_stride, void *q_out, int64_t q_out_stride, const void *k,
                               int64_t k_stride, const void *v, int64_t v_stride, hipStream_t s);
hipError_t sera_launch_kv_evict(uint32_t cache_type, int dim, const kv_args &a, const evict_args &t, hipStream_t s);

#endif
