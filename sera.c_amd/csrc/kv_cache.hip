/*
 * kv_cache.hip - rows into the paged cache and back: the write, which rounds
 * to fp16 or quantizes to 8 bits, and the read of the values that the cache
 * stands for.
 *
 * Both move data once and are bound by memory (or, for a few tokens, by the
 * launch). A wave takes one kv head of one 16-token block of a sequence,
 * lane l the channels E*l .. E*l+E-1 (E = head_dim / 64) of all 16 tokens:
 * row accesses are whole rows across the wave, and a lane ends with 16
 * tokens of its own channels, which is the order V is stored in, so nothing
 * passes through LDS. The block's loads are independent (up to 32 in flight
 * per lane).
 *
 * 8-bit quantizer: scale d = max|x| / 127 over the vector (an exact maximum,
 * one IEEE division), code = x / d rounded half to even, as the exact
 * quotient rounds: q0 = rint(x * (1/d)) is off by at most one and only next to a
 * border; x - q0 * d is exact there (one FMA; both terms are multiples of
 * half of d's last place and the difference is below d), so comparing it
 * with d / 2 puts q0 right, without a division per element.
 */
#include "attn_common.h"
#include "sera_launch.h"

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

__device__ __forceinline__ float kv_wave_max(float v) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}

/* E consecutive elements of a row. */
template <typename T, int E>
struct kv_vec {
    T v[E];
} __attribute__((aligned(sizeof(T) * E)));

/* Scale of a vector spread over the wave (NaN if an element is not finite),
 * and the factors for its codes: `up` lifts vectors so small that 1 / d
 * would overflow (both factors are powers of two, exact). */
struct kv_scale {
    float d, up, du, inv, half;
};

template <int E>
__device__ __forceinline__ kv_scale kv_vector_scale(const float *x) {
    float m = 0.0f;
    bool odd = false;
#pragma unroll
    for (int e = 0; e < E; e++) {
        m = fmaxf(m, fabsf(x[e]));
        odd |= !(fabsf(x[e]) <= 3.402823466e38f);
    }
    m = kv_wave_max(m);
    kv_scale s;
    s.d = __ballot(odd) ? __builtin_nanf("") : m / 127.0f;
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

}  // namespace

template <int TYPE, typename T, int D>
__global__ __launch_bounds__(256) void sera_kv_write_kernel(kv_args a, const T *__restrict__ k, int64_t k_stride,
                                                            const T *__restrict__ v, int64_t v_stride) {
    constexpr int E = D / 64;
    const int lane = threadIdx.x & 63;
    const int head = (int)blockIdx.y * 4 + (int)(threadIdx.x >> 6);
    int unit;
    const int b = kv_find(a, (int)blockIdx.x, kBlock, 2, &unit);
    if (b < 0 || head >= a.kv_heads) return;
    const kv_seq s = kv_sequence(a, b);
    if (s.bad) return;
    const kv_unit u = kv_unit_of(s, unit);
    if (u.t0 >= u.t1) return;
    const int page = a.table[(size_t)b * a.table_stride + (u.pos0 >> a.page_shift)];
    if (page < 0 || page >= a.pages) return;
    uint8_t *run = a.data + (size_t)page * a.page_bytes + (size_t)head * a.head_bytes;
    const int slot = u.pos0 & ((1 << a.page_shift) - 1);
    const size_t kv_elems = (size_t)D << a.page_shift;
    /* row of the block's token 0; only tokens t0 .. t1-1 have one */
    const int64_t row = (int64_t)s.row0 + u.pos0 - (s.len - s.n);
    const int d0 = E * lane;
    const T *kp = k + row * k_stride + (int64_t)head * D + d0, *vp = v + row * v_stride + (int64_t)head * D + d0;
    const bool full = u.t0 == 0 && u.t1 == kBlock;

    kv_vec<T, E> kx[kBlock], vx[kBlock];
#pragma unroll
    for (int t = 0; t < kBlock; t++)
        if (t >= u.t0 && t < u.t1) {
            kx[t] = *(const kv_vec<T, E> *)(kp + t * k_stride);
            vx[t] = *(const kv_vec<T, E> *)(vp + t * v_stride);
        } else {
#pragma unroll
            for (int e = 0; e < E; e++) kx[t].v[e] = vx[t].v[e] = (T)0.0f;
        }

    if (TYPE == (int)SERA_KV_F16) {
        _Float16 *ko = (_Float16 *)run + (size_t)slot * D + d0;
        _Float16 *vo = (_Float16 *)run + kv_elems + (size_t)slot * D + (size_t)d0 * 16;
#pragma unroll
        for (int t = 0; t < kBlock; t++)
            if (t >= u.t0 && t < u.t1) {
                kv_vec<_Float16, E> o;
#pragma unroll
                for (int e = 0; e < E; e++) o.v[e] = (_Float16)kv_to_f32(kx[t].v[e]);
                *(kv_vec<_Float16, E> *)(ko + t * D) = o;
            }
#pragma unroll
        for (int e = 0; e < E; e++) {
            if (full) {
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    kv_vec<_Float16, 8> o;
#pragma unroll
                    for (int t = 0; t < 8; t++) o.v[t] = (_Float16)kv_to_f32(vx[8 * h + t].v[e]);
                    *(kv_vec<_Float16, 8> *)(vo + 16 * e + 8 * h) = o;
                }
            } else {
#pragma unroll
                for (int t = 0; t < kBlock; t++)
                    if (t >= u.t0 && t < u.t1) vo[16 * e + t] = (_Float16)kv_to_f32(vx[t].v[e]);
            }
        }
    } else {
        int8_t *ko = (int8_t *)run + (size_t)slot * D + d0;
        int8_t *vo = (int8_t *)run + kv_elems + (size_t)slot * D + (size_t)d0 * 16;
        float *ks = (float *)(run + 2 * kv_elems) + slot, *vs = ks + ((size_t)1 << a.page_shift);
        kv_vec<int8_t, 16> vq[E];
#pragma unroll
        for (int t = 0; t < kBlock; t++) {
            const bool in = t >= u.t0 && t < u.t1;
            float x[E], y[E];
#pragma unroll
            for (int e = 0; e < E; e++) {
                x[e] = kv_to_f32(kx[t].v[e]);
                y[e] = kv_to_f32(vx[t].v[e]);
            }
            const kv_scale sx = kv_vector_scale<E>(x), sy = kv_vector_scale<E>(y);
            kv_vec<int8_t, E> o;
#pragma unroll
            for (int e = 0; e < E; e++) {
                o.v[e] = (int8_t)kv_code(x[e], sx);
                vq[e].v[t] = (int8_t)kv_code(y[e], sy);
            }
            if (in) {
                *(kv_vec<int8_t, E> *)(ko + t * D) = o;
                if (lane == 0) {
                    ks[t] = sx.d;
                    vs[t] = sy.d;
                }
            }
        }
#pragma unroll
        for (int e = 0; e < E; e++) {
            if (full) {
                *(kv_vec<int8_t, 16> *)(vo + 16 * e) = vq[e];
            } else {
#pragma unroll
                for (int t = 0; t < kBlock; t++)
                    if (t >= u.t0 && t < u.t1) vo[16 * e + t] = vq[e].v[t];
            }
        }
    }
}

/* Rows of bad sequences and pages come out as NaN, positions below zero as
 * zeros: unit 0 also fills the rows in front of the sequence's start. */
template <int TYPE, typename T, int D>
__global__ __launch_bounds__(256) void sera_kv_read_kernel(kv_args a, T *__restrict__ k, int64_t k_stride,
                                                           T *__restrict__ v, int64_t v_stride) {
    constexpr int E = D / 64;
    const int lane = threadIdx.x & 63;
    const int head = (int)blockIdx.y * 4 + (int)(threadIdx.x >> 6);
    int unit;
    const int b = kv_find(a, (int)blockIdx.x, kBlock, 2, &unit);
    if (b < 0 || head >= a.kv_heads) return;
    const kv_seq s = kv_sequence(a, b);
    const int d0 = E * lane;
    const int64_t col = (int64_t)head * D + d0;
    const int before = s.bad ? s.n : min(max(s.n - s.len, 0), s.n);
    if (unit == 0 && before > 0) {
        kv_vec<T, E> o;
#pragma unroll
        for (int e = 0; e < E; e++) o.v[e] = kv_from_f32<T>(s.bad ? __builtin_nanf("") : 0.0f);
        for (int64_t r = s.row0; r < s.row0 + before; r++) {
            *(kv_vec<T, E> *)(k + r * k_stride + col) = o;
            *(kv_vec<T, E> *)(v + r * v_stride + col) = o;
        }
    }
    if (s.bad) return;
    const kv_unit u = kv_unit_of(s, unit);
    if (u.t0 >= u.t1) return;
    const int page = a.table[(size_t)b * a.table_stride + (u.pos0 >> a.page_shift)];
    const bool lost = page < 0 || page >= a.pages;
    const uint8_t *run = a.data + (lost ? 0 : (size_t)page * a.page_bytes) + (size_t)head * a.head_bytes;
    const int slot = u.pos0 & ((1 << a.page_shift) - 1);
    const size_t kv_elems = (size_t)D << a.page_shift;
    const int64_t row = (int64_t)s.row0 + u.pos0 - (s.len - s.n);
    T *kp = k + row * k_stride + col, *vp = v + row * v_stride + col;

    float kx[kBlock][E], vx[kBlock][E];
    if (TYPE == (int)SERA_KV_F16) {
        const _Float16 *ki = (const _Float16 *)run + (size_t)slot * D + d0;
        const _Float16 *vi = (const _Float16 *)run + kv_elems + (size_t)slot * D + (size_t)d0 * 16;
        kv_vec<_Float16, E> kr[kBlock];
        kv_vec<_Float16, 8> vr[E][2];
#pragma unroll
        for (int t = 0; t < kBlock; t++) kr[t] = *(const kv_vec<_Float16, E> *)(ki + t * D);
#pragma unroll
        for (int e = 0; e < E; e++)
#pragma unroll
            for (int h = 0; h < 2; h++) vr[e][h] = *(const kv_vec<_Float16, 8> *)(vi + 16 * e + 8 * h);
#pragma unroll
        for (int t = 0; t < kBlock; t++)
#pragma unroll
            for (int e = 0; e < E; e++) {
                kx[t][e] = (float)kr[t].v[e];
                vx[t][e] = (float)vr[e][t >> 3].v[t & 7];
            }
    } else {
        const int8_t *ki = (const int8_t *)run + (size_t)slot * D + d0;
        const int8_t *vi = (const int8_t *)run + kv_elems + (size_t)slot * D + (size_t)d0 * 16;
        const float *ks = (const float *)(run + 2 * kv_elems) + slot, *vs = ks + ((size_t)1 << a.page_shift);
        kv_vec<int8_t, E> kr[kBlock];
        kv_vec<int8_t, 16> vr[E];
#pragma unroll
        for (int t = 0; t < kBlock; t++) kr[t] = *(const kv_vec<int8_t, E> *)(ki + t * D);
#pragma unroll
        for (int e = 0; e < E; e++) vr[e] = *(const kv_vec<int8_t, 16> *)(vi + 16 * e);
#pragma unroll
        for (int t = 0; t < kBlock; t++)
#pragma unroll
            for (int e = 0; e < E; e++) {
                kx[t][e] = (float)kr[t].v[e] * ks[t];
                vx[t][e] = (float)vr[e].v[t] * vs[t];
            }
    }
#pragma unroll
    for (int t = 0; t < kBlock; t++)
        if (t >= u.t0 && t < u.t1) {
            kv_vec<T, E> ko, vo;
#pragma unroll
            for (int e = 0; e < E; e++) {
                ko.v[e] = kv_from_f32<T>(lost ? __builtin_nanf("") : kx[t][e]);
                vo.v[e] = kv_from_f32<T>(lost ? __builtin_nanf("") : vx[t][e]);
            }
            *(kv_vec<T, E> *)(kp + t * k_stride) = ko;
            *(kv_vec<T, E> *)(vp + t * v_stride) = vo;
        }
}

namespace {

template <int TYPE, typename T, int D>
hipError_t kv_move(bool write, const kv_args &a, void *k, int64_t ks, void *v, int64_t vs, hipStream_t s) {
    const dim3 grid((unsigned)kv_slots(a.rows, a.sequences, kBlock, 2), (unsigned)((a.kv_heads + 3) / 4));
    if (write)
        hipLaunchKernelGGL((sera_kv_write_kernel<TYPE, T, D>), grid, dim3(256), 0, s, a, (const T *)k, ks,
                           (const T *)v, vs);
    else
        hipLaunchKernelGGL((sera_kv_read_kernel<TYPE, T, D>), grid, dim3(256), 0, s, a, (T *)k, ks, (T *)v, vs);
    return hipGetLastError();
}

template <int TYPE, typename T>
hipError_t kv_move_d(bool write, int dim, const kv_args &a, void *k, int64_t ks, void *v, int64_t vs, hipStream_t s) {
    return dim == 64 ? kv_move<TYPE, T, 64>(write, a, k, ks, v, vs, s)
                     : kv_move<TYPE, T, 128>(write, a, k, ks, v, vs, s);
}

template <int TYPE>
hipError_t kv_move_t(bool write, uint32_t type, int dim, const kv_args &a, void *k, int64_t ks, void *v, int64_t vs,
                     hipStream_t s) {
    if (type == SERA_TYPE_F32) return kv_move_d<TYPE, float>(write, dim, a, k, ks, v, vs, s);
    if (type == SERA_TYPE_F16) return kv_move_d<TYPE, _Float16>(write, dim, a, k, ks, v, vs, s);
    return kv_move_d<TYPE, __bf16>(write, dim, a, k, ks, v, vs, s);
}

}  // namespace

/* Arguments are checked by the caller (sera_attn_runtime.hip). */
hipError_t sera_launch_kv_move(bool write, uint32_t cache_type, uint32_t type, int dim, const kv_args &a, void *k,
                               int64_t k_stride, void *v, int64_t v_stride, hipStream_t s) {
    return cache_type == SERA_KV_F16
               ? kv_move_t<(int)SERA_KV_F16>(write, type, dim, a, k, k_stride, v, v_stride, s)
               : kv_move_t<(int)SERA_KV_Q8>(write, type, dim, a, k, k_stride, v, v_stride, s);
}
