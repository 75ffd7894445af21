/*
 * attn_sums.h - the weights' sums of few rows from their scores: device code of the kernel that makes all sums
 * (attn_weights.hip) and of the one that joins split contexts beside it (attn.hip).
 */
#ifndef ATTN_SUMS_H
#define ATTN_SUMS_H

#include "attn_device.h"

constexpr int kFewNorms = 32;       /* columns of the few-row kernel */

/* The norms of a sequence's and kv head's columns, by four waves: as the few-row kernel left them, or of a context
 * split over workgroups from what each of those left (as the join has them, which may run at the same time). */
__device__ __forceinline__ void attn_few_norms(const kv_args &a, const attn_args &t, const attn_sums &p,
                                               const kv_seq &s, int head, float2 *norms) {
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), rows = s.n * t.group;
    if (p.splits < 2) {
        if (tid < rows) {
            const int i = tid / t.group;
            norms[tid] = t.norms[(size_t)(s.row0 + i) * t.heads + head * t.group + tid - i * t.group];
        }
        return;
    }
    const attn_range range = attn_range_of(t, max(s.len - s.n, 0), s.len, kAttnShift);
    const int used = max((range.count + p.chunk - 1) / p.chunk, 1);
    const size_t step = attn_partial_floats(p.few_rows, p.dim);
    const float *const at = t.workspace + ((size_t)s.b * a.kv_heads + head) * p.splits * step +
                            (size_t)p.few_rows * p.dim + lane * step;
    attn_f2 ml[kFewNorms / 4];
#pragma unroll
    for (int k = 0; k < kFewNorms / 4; k++) {
        const int r = wave + 4 * k;
        ml[k] = attn_f2{kAttnLowest, 0.0f};
        if (lane < used && r < rows) ml[k] = *(const attn_f2 *)(at + 2 * r);
    }
#pragma unroll
    for (int k = 0; k < kFewNorms / 4; k++) {
        const int r = wave + 4 * k;
        if (r >= rows) break;
        float top = ml[k][0];
        top = fmaxf(top, xor_partner<1>(top));
        top = fmaxf(top, xor_partner<2>(top));
        top = fmaxf(top, xor_partner<4>(top));
        top = fmaxf(top, xor_partner<8>(top));
        top = fmaxf(top, xor_partner<16>(top));
        top = fmaxf(top, xor_partner<32>(top));
        float l = lane < used ? ml[k][1] * attn_exp2(ml[k][0] - top) : 0.0f;
        l += xor_partner<1>(l);
        l += xor_partner<2>(l);
        l += xor_partner<4>(l);
        l += xor_partner<8>(l);
        l += xor_partner<16>(l);
        l += xor_partner<32>(l);
        if (lane == 0) norms[r] = attn_norm(top, l);
    }
}

/* Whether a row of the sequence may see any of positions j .. j+n-1. What none sees, in front of the first row's window and
 * behind the sinks, has no scores: the attention kernel goes by the same range, and leaves their places as they are. */
__device__ __forceinline__ bool attn_few_seen(const attn_args &t, const kv_seq &s, int j, int n) {
    return t.window == 0 || j < t.sinks || j + n - 1 > max(s.len - s.n, 0) - t.window;
}

/* The sums of positions j .. j+3. */
__device__ __forceinline__ attn_f4 attn_few_sums(const attn_args &t, const attn_sums &p, const kv_seq &s, size_t place,
                                                 int j, const float2 *norms) {
    constexpr int BATCH = 8;        /* loads on their way */
    const int first = s.len - s.n, rows = s.n * t.group;
    constexpr int TILE = 1 << kAttnShift;
    const float *const x = p.scores + (place * p.pitch + (j & -TILE)) * p.few_rows + j % TILE;
    attn_f4 w = {0.0f, 0.0f, 0.0f, 0.0f};
    if (!attn_few_seen(t, s, j, 4)) return w;
    for (int r = 0, i = 0, g = 0; r < rows; r += BATCH) {
        attn_f4 y[BATCH];
        float2 l[BATCH];
        int pos[BATCH];
#pragma unroll
        for (int k = 0; k < BATCH; k++) {
            y[k] = *(const attn_f4 *)(x + min(r + k, rows - 1) * TILE);
            l[k] = norms[min(r + k, rows - 1)];
            pos[k] = r + k < rows ? first + i : -1;
            if (++g == t.group) {
                g = 0;
                i++;
            }
        }
#pragma unroll
        for (int k = 0; k < BATCH; k++)
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (pos[k] >= 0 && attn_sees(t, pos[k], j + e))
                    w[e] = fmaf(attn_exp2(y[k][e] - l[k].x), l[k].y, w[e]);
    }
    return w;
}

/* They go behind what was there before, but for the new rows' positions. */
__device__ __forceinline__ void attn_put_sums(const attn_args &t, const kv_seq &s, size_t place, int j, attn_f4 w) {
    const int first = s.len - s.n;
    const size_t at = place * (size_t)t.weights_stride + j;
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (j + e < s.len) t.weights[at + e] = (t.before && j + e < first ? t.before[at + e] : 0.0f) + w[e];
}

#endif
