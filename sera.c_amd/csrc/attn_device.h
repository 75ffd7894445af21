/*
 * attn_device.h - what the attention kernels share on the device: the
 * visible range of a sequence's rows, query fragments, the mask, and the
 * treatment of what the cache holds in places that a row does not see.
 */
#ifndef SERA_ATTN_DEVICE_H
#define SERA_ATTN_DEVICE_H

#include "attn_common.h"
#include "sera_dpp.h"

typedef _Float16 attn_h2 __attribute__((ext_vector_type(2)));
typedef _Float16 attn_h8 __attribute__((ext_vector_type(8)));
typedef float attn_f2 __attribute__((ext_vector_type(2)));
typedef float attn_f4 __attribute__((ext_vector_type(4)));
typedef float attn_f16 __attribute__((ext_vector_type(16)));
typedef uint32_t attn_u2 __attribute__((ext_vector_type(2)));
typedef uint32_t attn_u4 __attribute__((ext_vector_type(4)));

constexpr float kAttnLowest = -3.402823466e38f;
/* Weights are held as 2^(s - m + kAttnBias), m the running maximum. m may lag
 * behind the true maximum by kAttnLag, so they reach 2^15, inside fp16, and a
 * weight keeps its 11 (two terms: 22) bits down to 2^-21 (2^-10) of the
 * largest; below that its error is 2^-31 of the largest. The factor 2^kAttnBias
 * is in the sum of the weights as well and leaves with the division. */
constexpr float kAttnBias = 7.0f, kAttnLag = 8.0f;

/* Tiles of 2^shift positions that the rows from position p0 (>= 0) to len-1 see:
 * the sinks' tiles, then those from the first row's window to the end. */
struct attn_range {
    int sink_tiles, low, count;
    __device__ __forceinline__ int tile(int v) const { return v < sink_tiles ? v : low + v - sink_tiles; }
};

__device__ __forceinline__ attn_range attn_range_of(const attn_args &t, int p0, int end, int shift) {
    attn_range r;
    const int first = t.window > 0 ? max(p0 - t.window + 1, 0) : 0;
    r.low = first >> shift;
    /* sinks can be as large as an int: no sum before the minimum */
    r.sink_tiles = t.window > 0 ? min((min(t.sinks, first) + (1 << shift) - 1) >> shift, r.low) : 0;
    r.count = end > 0 ? r.sink_tiles + ((end + (1 << shift) - 1) >> shift) - r.low : 0;
    return r;
}

/* The tiles v0 <= v < v1 of a range that rows with positions p0 .. p1 (those with p0 < 0 see no tile whole) all see
 * whole, but for tiles of sinks. */
struct attn_whole {
    int v0, v1;
};

__device__ __forceinline__ attn_whole attn_whole_of(const attn_args &t, const attn_range &r, int p0, int p1,
                                                    int shift) {
    attn_whole w;
    const int past = r.sink_tiles - r.low;       /* v - tile */
    const int from = t.window > 0 ? max(p1 - t.window + 1, 0) : 0;
    w.v0 = max(((from + (1 << shift) - 1) >> shift) + past, r.sink_tiles);
    w.v1 = p0 < 0 ? 0 : ((p0 + 1) >> shift) + past;
    return w;
}

/* Whether every row with positions p0 .. p1 sees all positions j .. j+n-1. */
__device__ __forceinline__ bool attn_all_seen(const attn_args &t, int j, int n, int p0, int p1) {
    return j + n - 1 <= p0 && (t.window == 0 || j > p1 - t.window || j + n <= t.sinks);
}

__device__ __forceinline__ bool attn_sees(const attn_args &t, int p, int j) {
    return j <= p && (t.window == 0 || j > p - t.window || j < t.sinks);
}

/* The page of positions pos .. pos+15 of sequence b, or -1 if its id is
 * outside the pool. Past the end: page 0, which is in the pool (its content
 * is masked). */
__device__ __forceinline__ int attn_page(const kv_args &a, int b, int pos, int len) {
    if (pos >= len) return 0;
    const int page = a.table[(size_t)b * a.table_stride + (pos >> a.page_shift)];
    return page < 0 || page >= a.pages ? -1 : page;
}

__device__ __forceinline__ float attn_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

/* What a score becomes a weight by, 2^(s' - z) * r, from a row's maximum and its sum of weights. z is log2 of the sum but
 * for a factor of 2; what that addition rounds off goes into r with the rest, so that scores keep all of their bits. A
 * row without weights has an r of 0. */
__device__ __forceinline__ float2 attn_norm(float m, float l) {
    const float shift = m - kAttnBias, e = (float)__builtin_amdgcn_frexp_expf(l), z = shift + e, y = z - shift;
    const float off = (shift - (z - y)) + (e - y);
    return make_float2(z, l == 0.0f ? __builtin_nanf("") : attn_exp2(-off) / __builtin_amdgcn_frexp_mantf(l));
}

/* The power of two that brings the largest |q| of a row near 2^10 (products
 * and sums then stay clear of fp16's and fp32's borders whatever the rows' size),
 * as its exponent. */
__device__ __forceinline__ int attn_q_exponent(float amax) {
    const int e = (int)((__float_as_uint(amax) >> 23) & 255u);
    return e == 0 || e == 255 ? (amax > 0.0f && e == 0 ? 126 : 0) : min(max(137 - e, -126), 126);
}

__device__ __forceinline__ attn_h2 attn_pack(float a, float b) {
    const attn_f2 f = {a, b};
    return __builtin_convertvector(f, attn_h2);
}

/* x as one fp16 or the sum of two: hi = x rounded, lo = the rest (exact in fp32) rounded. The rest is
 * written as an FMA with a -1 that the compiler does not see through, so it and its rounding become one mixed
 * instruction (v_fma_mixlo/hi_f16). */
template <bool TWO>
__device__ __forceinline__ void attn_split(const float *x, attn_h8 &hi, attn_h8 &lo) {
    float minus = -1.0f;
    asm("" : "+s"(minus));
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const attn_h2 h = attn_pack(x[i], x[i + 1]);
        hi[i] = h[0];
        hi[i + 1] = h[1];
        if (TWO) {
            lo[i] = (_Float16)fmaf((float)h[0], minus, x[i]);
            lo[i + 1] = (_Float16)fmaf((float)h[1], minus, x[i + 1]);
        }
    }
}

/* Eight int8 codes as fp16, exact: 1024 + (code + 128) is the fp16 number
 * with the byte in its low bits. */
__device__ __forceinline__ attn_h8 attn_codes(uint32_t a, uint32_t b) {
    const uint32_t x = a ^ 0x80808080u, y = b ^ 0x80808080u, c = 0x64646464u;
    attn_u4 w;
    w[0] = __builtin_amdgcn_perm(c, x, 0x04010400u);
    w[1] = __builtin_amdgcn_perm(c, x, 0x04030402u);
    w[2] = __builtin_amdgcn_perm(c, y, 0x04010400u);
    w[3] = __builtin_amdgcn_perm(c, y, 0x04030402u);
    attn_h8 h = __builtin_bit_cast(attn_h8, w);
    const _Float16 k = (_Float16)1152.0f;
    return h - attn_h8{k, k, k, k, k, k, k, k};
}

/* Non-finite values of v: 1 in `odd` there (0 elsewhere) and 0 in v. Returns
 * whether there is one. */
__device__ __forceinline__ bool attn_take_odd(attn_h8 &v, attn_h8 &odd) {
    attn_u4 w = __builtin_bit_cast(attn_u4, v), f;
    bool any = false;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const bool lo = (w[i] & 0x7c00u) == 0x7c00u, hi = (w[i] & 0x7c000000u) == 0x7c000000u;
        any |= lo | hi;
        f[i] = (lo ? 0x3c00u : 0u) | (hi ? 0x3c000000u : 0u);
        w[i] &= (lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u);
    }
    v = __builtin_bit_cast(attn_h8, w);
    odd = __builtin_bit_cast(attn_h8, f);
    return any;
}

/* log2 of a V scale: 8-bit caches take the running maximum over s +
 * log2(V scale), so that weight * scale fits fp16 however far the scales are
 * apart. It is held inside -84 .. 121, for weights and their sum to stay normal
 * fp32 numbers: a weight is at most 2^(84 + kAttnBias + kAttnLag) = 2^99, the sum of 2^28 of them (all positions that a
 * sequence can have) 2^127; values whose scales are all below 2^-84 lose bits, and
 * vectors of zeros (scale 0) count as such. A NaN stays out of the maximum (fmaxf
 * takes the other). */
__device__ __forceinline__ float attn_log_scale(float vs) {
    const float l = __builtin_amdgcn_logf(fabsf(vs));
    return l < -84.0f ? -84.0f : l > 121.0f ? 121.0f : l;
}

template <typename T>
__device__ __forceinline__ void attn_load8(const T *p, float *x) {
    struct __attribute__((aligned(16))) vec { T v[8]; };
    const vec w = *(const vec *)p;
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = kv_to_f32(w.v[i]);
}

template <typename T, int N>
struct __attribute__((aligned(sizeof(T) * N))) attn_vec {
    T v[N];
};

template <typename T>
__device__ __forceinline__ void attn_store4(T *p, const float *x) {
    attn_vec<T, 4> o;
#pragma unroll
    for (int i = 0; i < 4; i++) o.v[i] = kv_from_f32<T>(x[i]);
    *(attn_vec<T, 4> *)p = o;
}

/* Row tiles of `per` rows (tokens x heads of a group) of the tile kernel's
 * sequences, numbered through the sequences without gaps: a workgroup that finds
 * no rows still takes a turn on a compute unit, and where every second one does
 * (sequences of one tile each, with slots for two), half of the units get
 * nothing but those: 16 sequences of 256 rows took as long as 32. Up to
 * kAttnCounted sequences are counted, one load of a wave for 64 of them;
 * beyond, kv_find's gaps are few against the rest. */
constexpr int kAttnCounted = 256;

__device__ __forceinline__ int attn_tiles_of(const kv_args &a, const attn_args &t, int b, int per) {
    if (b >= a.sequences) return 0;
    const int r0 = min(max(a.row_start[b], 0), a.rows), r1 = min(max(a.row_start[b + 1], r0), a.rows);
    const int rows = (r1 - r0) * t.group;
    return rows <= t.few_columns ? 0 : (rows + per - 1) / per;
}

/* Sequence and tile of it in place `slot`, counted from the last: late rows see most and start first. -1: none.
 * Where row_start decreases, sequences overlap and may have more tiles together than there are slots: the first
 * ones are not run. */
__device__ __forceinline__ int attn_find_tile(const kv_args &a, const attn_args &t, int per, int slots, int slot,
                                              int *tile) {
    const int lane = (int)(threadIdx.x & 63);
    if (a.sequences > kAttnCounted) return kv_find(a, slots - 1 - slot, per, 1, tile, t.group);
    int n[kAttnCounted / 64], upto[kAttnCounted / 64], total = 0;
#pragma unroll
    for (int i = 0; i < kAttnCounted / 64; i++) {
        n[i] = upto[i] = 0;
        if (64 * i >= a.sequences) continue;
        upto[i] = n[i] = attn_tiles_of(a, t, 64 * i + lane, per);
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int x = __shfl_up(upto[i], o, 64);
            upto[i] += lane >= o ? x : 0;
        }
        upto[i] += total;
        total = __builtin_amdgcn_readfirstlane(__shfl(upto[i], 63, 64));
    }
    const int place = total - 1 - slot;
    if (place < 0) return -1;
    for (int i = 0; i < kAttnCounted / 64; i++) {
        const unsigned long long past = __ballot(upto[i] > place);
        if (past) {
            const int l = __builtin_ctzll(past);
            const int own = __shfl(n[i], l, 64);
            *tile = __builtin_amdgcn_readfirstlane(place - (__shfl(upto[i], l, 64) - own));
            /* not one of its tiles: only where overlapping sequences' sum left an int */
            return (unsigned)*tile < (unsigned)__builtin_amdgcn_readfirstlane(own) ? 64 * i + l : -1;
        }
    }
    return -1;
}

/* Partial results of a split context, in the workspace. Few rows: a unit of `rows` rows for each sequence, kv head and
 * split, rows of D sums and then (m, l) of every row. Tiles: by packed row, which stays inside the batch's rows
 * whatever row_start holds: D sums for each (row, query head, split), and behind them all (m, l) in the same order. */
__device__ __forceinline__ size_t attn_partial_floats(int rows, int dim) { return (size_t)rows * (dim + 2); }

#endif
