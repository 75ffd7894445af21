/*
 * kv_device.h - what the kernels that put rows into the paged cache share on
 * the device (internal): 16-token blocks, row accesses, the 8-bit quantizer
 * and the store of half a block.
 *
 * 8-bit quantizer: scale d = max|x| / 127 over the vector (an exact maximum,
 * one IEEE division), code = x / d rounded half to even, as the exact
 * quotient rounds: q0 = rint(x * (1/d)) is off by at most one and only next to a
 * border; x - q0 * d is exact there (one FMA; both terms are multiples of
 * half of d's last place and the difference is below d), so comparing it
 * with d / 2 puts q0 right, without a division per element.
 *
 * No floating-point contraction here: the quantizer's steps are rounded one
 * by one (hipcc fuses a * b + c by default).
 */
#ifndef SERA_KV_DEVICE_H
#define SERA_KV_DEVICE_H

#include "kv_common.h"
#include "sera_dpp.h"

#pragma clang fp contract(off)

namespace {

constexpr int kBlock = 16;   /* tokens of a unit: V's transposed group */

/* The 16-token block `unit` of a sequence's new positions: its first
 * position, and which of its tokens are new. */
struct kv_unit {
    int pos0, t0, t1;   /* tokens t0 .. t1-1 of the block at pos0 */
};

__device__ __forceinline__ kv_unit kv_unit_of(const kv_seq &s, int unit) {
    kv_unit u;
    const int first = s.len - s.n;                 /* may be below zero */
    const int start = max(first, 0);
    u.pos0 = ((start >> 4) + unit) << 4;
    u.t0 = max(start - u.pos0, 0);
    u.t1 = min(s.len - u.pos0, kBlock);
    return u;
}

/* N consecutive elements. */
template <typename T, int N>
struct __attribute__((aligned(sizeof(T) * N))) kv_vec {
    T v[N];
};

/* How a wave accesses 16 rows of D elements, 16 bytes of T at a time. */
template <typename T, int D>
struct kv_rows {
    static constexpr int VEC = 16 / (int)sizeof(T), LANES = D / VEC, ROWS = 64 / LANES, N = kBlock / ROWS;
    /* token and first channel of access i of a lane */
    static __device__ __forceinline__ int token(int i, int lane) { return i * ROWS + lane / LANES; }
    static __device__ __forceinline__ int channel(int lane) { return lane % LANES * VEC; }
};

/* The largest of m over the lanes that share a row. */
template <int LANES>
__device__ __forceinline__ float kv_row_max(float m) {
    m = fmaxf(m, xor_partner<1>(m));
    m = fmaxf(m, xor_partner<2>(m));
    m = fmaxf(m, xor_partner<4>(m));
    if constexpr (LANES >= 16) m = fmaxf(m, xor_partner<8>(m));
    if constexpr (LANES >= 32) m = fmaxf(m, xor_partner<16>(m));
    return m;
}

/* Scale of a row (NaN if an element is not finite), and the factors for its
 * codes: `up` lifts vectors so small that 1 / d would overflow (both factors
 * are powers of two, exact). */
struct kv_scale {
    float d, up, du, inv, half;
};

template <int VEC, int LANES>
__device__ __forceinline__ kv_scale kv_vector_scale(const float *x) {
    float m = 0.0f;
#pragma unroll
    for (int e = 0; e < VEC; e++) m = fmaxf(m, x[e] == x[e] ? fabsf(x[e]) : INFINITY);
    m = kv_row_max<LANES>(m);
    kv_scale s;
    s.d = m <= 3.402823466e38f ? m / 127.0f : __builtin_nanf("");
    s.up = m < 0x1p-60f ? 0x1p64f : 1.0f;
    s.du = s.d * s.up;
    s.inv = 1.0f / s.du;
    s.half = 0.5f * s.du;
    return s;
}

__device__ __forceinline__ int kv_code(float x, const kv_scale &s) {
    if (!(s.d > 0.0f)) return 0;
    const float xu = x * s.up;
    float q = rintf(xu * s.inv);
    const float r = fmaf(-q, s.du, xu);
    const float a = fabsf(r);
    const bool odd = ((int)q & 1) != 0;
    if (a > s.half || (a == s.half && odd)) q += r > 0.0f ? 1.0f : -1.0f;
    return (int)fminf(fmaxf(q, -127.0f), 127.0f);
}

/* Tokens u.t0 .. u.t1-1 of half a block (8 tokens from h0 on) of one head into its run of a page: K as rows, V turned
 * in LDS (`turn`, the wave's own). `from`: the lane's place (its first channel) in the row of the block's token 0.
 * `change`(x, t) is applied to the lane's elements of token t in fp32, for all lanes of a wave at once. */
template <int TYPE, typename T, int D, typename F>
__device__ __forceinline__ void kv_put_half(const kv_args &a, const kv_unit &u, int h0, bool is_v, uint8_t *run,
                                            const T *from, int64_t stride,
                                            uint32_t (*turn)[D * (TYPE == (int)SERA_KV_Q8 ? 1 : 2) / 4], int lane,
                                            const F &change) {
    using R = kv_rows<T, D>;
    constexpr bool Q8 = TYPE == (int)SERA_KV_Q8;
    constexpr int VEC = R::VEC, N = R::N / 2, ES = Q8 ? 1 : 2, TOKENS = kBlock / 2;
    const size_t kv_bytes = ((size_t)D << a.page_shift) * ES;
    const int slot = u.pos0 & ((1 << a.page_shift) - 1);
    const int d0 = R::channel(lane);
    uint8_t *to = run + (is_v ? kv_bytes : 0) + (size_t)slot * (D * ES);

    kv_vec<T, VEC> in[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int t = h0 + R::token(i, lane);
#pragma unroll
        for (int e = 0; e < VEC; e++) in[i].v[e] = (T)0.0f;
        if (t >= u.t0 && t < u.t1) in[i] = *(const kv_vec<T, VEC> *)(from + t * stride);
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int t = h0 + R::token(i, lane);
        const bool new_row = t >= u.t0 && t < u.t1;
        float x[VEC];
#pragma unroll
        for (int e = 0; e < VEC; e++) x[e] = kv_to_f32(in[i].v[e]);
        change(x, t);
        if constexpr (Q8) {
            const kv_scale sc = kv_vector_scale<VEC, R::LANES>(x);
            kv_vec<int8_t, VEC> o;
#pragma unroll
            for (int e = 0; e < VEC; e++) o.v[e] = (int8_t)kv_code(x[e], sc);
            if (new_row && d0 == 0)
                ((float *)(run + 2 * kv_bytes))[((size_t)is_v << a.page_shift) + slot + t] = sc.d;
            if (is_v) *(kv_vec<int8_t, VEC> *)((int8_t *)turn[t - h0] + d0) = o;
            else if (new_row) *(kv_vec<int8_t, VEC> *)(to + t * D + d0) = o;
        } else {
            kv_vec<_Float16, VEC> o;
#pragma unroll
            for (int e = 0; e < VEC; e++) o.v[e] = (_Float16)x[e];
            if (is_v) *(kv_vec<_Float16, VEC> *)((_Float16 *)turn[t - h0] + d0) = o;
            else if (new_row) *(kv_vec<_Float16, VEC> *)(to + (t * D + d0) * 2) = o;
        }
    }
    if (!is_v) return;
    asm volatile("" ::: "memory");          /* the wave's own LDS, which it accesses in order */
    if (u.t1 - u.t0 < TOKENS) {             /* some of the tokens: one element at a time */
        for (int t = u.t0; t < u.t1; t++)
            for (int d = lane; d < D; d += 64) {
                if (Q8) to[16 * d + t] = ((const uint8_t *)turn[t - h0])[d];
                else ((uint16_t *)to)[16 * d + t] = ((const uint16_t *)turn[t - h0])[d];
            }
        return;
    }
    if constexpr (Q8) {                     /* dword column c: channels 4c .. 4c+3; a lane takes D / 64 of them */
        const int c = lane * (D / 64) / 4, j = lane * (D / 64) % 4;
        uint32_t w[TOKENS];
#pragma unroll
        for (int t = 0; t < TOKENS; t++) w[t] = turn[t][c];
#pragma unroll
        for (int e = 0; e < D / 64; e++) {
            kv_vec<uint32_t, 2> o;
            const uint32_t pick = 0x0c0c0400u + (uint32_t)(j + e) * 0x0101u;       /* byte j + e of two dwords */
#pragma unroll
            for (int q = 0; q < 2; q++)
                o.v[q] = __builtin_amdgcn_perm(w[4 * q + 1], w[4 * q], pick) |
                         __builtin_amdgcn_perm(w[4 * q + 3], w[4 * q + 2], pick) << 16;
            *(kv_vec<uint32_t, 2> *)(to + 16 * (lane * (D / 64) + e) + h0) = o;
        }
    } else {                                /* dword column c: channels 2c, 2c+1, of all or half of the tokens */
        constexpr int MINE = D / 16;
        const int c = lane % (D / 2), t0 = lane / (D / 2) * MINE;
        uint32_t w[MINE];
#pragma unroll
        for (int t = 0; t < MINE; t++) w[t] = turn[t0 + t][c];
#pragma unroll
        for (int e = 0; e < 2; e++) {
            kv_vec<uint32_t, MINE / 2> o;
#pragma unroll
            for (int q = 0; q < MINE / 2; q++)
                o.v[q] = __builtin_amdgcn_perm(w[2 * q + 1], w[2 * q], e ? 0x07060302u : 0x05040100u);
            *(kv_vec<uint32_t, MINE / 2> *)(to + 32 * (2 * c + e) + 2 * (h0 + t0)) = o;
        }
    }
}

}  // namespace

#endif
