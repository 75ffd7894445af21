/*
 * kv_cache.hip - rows into the paged cache and back: the write, which rounds
 * to fp16 or quantizes to 8 bits, and the read of the values that the cache
 * stands for.
 *
 * Both move data once and are bound by memory (or, for a few tokens, by the
 * launch and three dependent loads: sequence, page, data). A wave takes K or V
 * of one kv head of one 16-token block of a sequence, a half of it to write (more
 * waves for the quantizer: 2048 tokens into an 8-bit cache and back 17.6 us, 19.9
 * with whole blocks). Rows are accessed in 16-byte
 * pieces (D / VEC lanes to a row, several rows to an access); K's place in the cache is
 * the same order. V's is not: 16 tokens of a channel lie side by side, so a wave
 * turns its block in LDS of its own, in dwords that are unpacked by byte
 * permutes. 37922 tokens out of an 8-bit cache as fp32 rows: 79-88 us, 4.4-5.0
 * TB/s (a large copy: 5.2); ragged bf16 chunks into an fp16 cache 6 us for 15 MB.
 *
 * 8-bit quantizer: scale d = max|x| / 127 over the vector (an exact maximum,
 * one IEEE division), code = x / d rounded half to even, as the exact
 * quotient rounds: q0 = rint(x * (1/d)) is off by at most one and only next to a
 * border; x - q0 * d is exact there (one FMA; both terms are multiples of
 * half of d's last place and the difference is below d), so comparing it
 * with d / 2 puts q0 right, without a division per element.
 */
#include "attn_common.h"
#include "sera_dpp.h"
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

/* N consecutive elements. */
template <typename T, int N>
struct __attribute__((aligned(sizeof(T) * N))) kv_vec {
    T v[N];
};

typedef uint32_t kv_u4 __attribute__((ext_vector_type(4)));
typedef uint32_t kv_u2 __attribute__((ext_vector_type(2)));

/* Stores past the caches: rows read back are larger than what they come from and only stream through (37922 tokens
 * out of an 8-bit cache take 80 us so, 94 us with ordinary stores; out of an fp16 cache 118 and 116). */
template <typename T, int N>
__device__ __forceinline__ void kv_store_past(T *p, const kv_vec<T, N> &v) {
    if constexpr (sizeof(v) == 16) __builtin_nontemporal_store(__builtin_bit_cast(kv_u4, v), (kv_u4 *)p);
    else __builtin_nontemporal_store(__builtin_bit_cast(kv_u2, v), (kv_u2 *)p);
}

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

}  // namespace

template <int TYPE, typename T, int D>
__global__ __launch_bounds__(256) void sera_kv_write_kernel(kv_args a, const T *__restrict__ k, int64_t k_stride,
                                                            const T *__restrict__ v, int64_t v_stride) {
    using R = kv_rows<T, D>;
    constexpr bool Q8 = TYPE == (int)SERA_KV_Q8;
    constexpr int VEC = R::VEC, N = R::N / 2, ES = Q8 ? 1 : 2, ROW = D * ES / 4;  /* dwords of a row in LDS */
    constexpr int TOKENS = kBlock / 2;
    __shared__ uint32_t turn[4][TOKENS][ROW];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int item = (int)blockIdx.y * 4 + wave, head = item >> 2, h0 = (item & 1) * TOKENS;
    const bool is_v = item & 2;
    int unit;
    const kv_seq s = kv_find_sequence(a, (int)blockIdx.x, kBlock, 2, &unit);
    if (s.b < 0 || head >= a.kv_heads || s.bad) return;
    kv_unit u = kv_unit_of(s, unit);
    u.t0 = max(u.t0, h0);
    u.t1 = min(u.t1, h0 + TOKENS);
    if (u.t0 >= u.t1) return;
    const int page = a.table[(size_t)s.b * a.table_stride + (u.pos0 >> a.page_shift)];
    if (page < 0 || page >= a.pages) return;
    const size_t kv_bytes = ((size_t)D << a.page_shift) * ES;
    uint8_t *run = a.data + (size_t)page * a.page_bytes + (size_t)head * a.head_bytes;
    const int slot = u.pos0 & ((1 << a.page_shift) - 1);
    const int64_t stride = is_v ? v_stride : k_stride;
    /* row of the block's token 0; only tokens t0 .. t1-1 have one */
    const int64_t row = (int64_t)s.row0 + u.pos0 - (s.len - s.n);
    const int d0 = R::channel(lane);
    const T *from = (is_v ? v : k) + row * stride + (int64_t)head * D + d0;
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
        if constexpr (Q8) {
            const kv_scale sc = kv_vector_scale<VEC, R::LANES>(x);
            kv_vec<int8_t, VEC> o;
#pragma unroll
            for (int e = 0; e < VEC; e++) o.v[e] = (int8_t)kv_code(x[e], sc);
            if (new_row && d0 == 0)
                ((float *)(run + 2 * kv_bytes))[((size_t)is_v << a.page_shift) + slot + t] = sc.d;
            if (is_v) *(kv_vec<int8_t, VEC> *)((int8_t *)turn[wave][t - h0] + d0) = o;
            else if (new_row) *(kv_vec<int8_t, VEC> *)(to + t * D + d0) = o;
        } else {
            kv_vec<_Float16, VEC> o;
#pragma unroll
            for (int e = 0; e < VEC; e++) o.v[e] = (_Float16)x[e];
            if (is_v) *(kv_vec<_Float16, VEC> *)((_Float16 *)turn[wave][t - h0] + d0) = o;
            else if (new_row) *(kv_vec<_Float16, VEC> *)(to + (t * D + d0) * 2) = o;
        }
    }
    if (!is_v) return;
    asm volatile("" ::: "memory");          /* the wave's own LDS, which it accesses in order */
    if (u.t1 - u.t0 < TOKENS) {             /* some of the tokens: one element at a time */
        for (int t = u.t0; t < u.t1; t++)
            for (int d = lane; d < D; d += 64) {
                if (Q8) to[16 * d + t] = ((const uint8_t *)turn[wave][t - h0])[d];
                else ((uint16_t *)to)[16 * d + t] = ((const uint16_t *)turn[wave][t - h0])[d];
            }
        return;
    }
    if constexpr (Q8) {                     /* dword column c: channels 4c .. 4c+3; a lane takes D / 64 of them */
        const int c = lane * (D / 64) / 4, j = lane * (D / 64) % 4;
        uint32_t w[TOKENS];
#pragma unroll
        for (int t = 0; t < TOKENS; t++) w[t] = turn[wave][t][c];
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
        for (int t = 0; t < MINE; t++) w[t] = turn[wave][t0 + t][c];
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

/* Rows of bad sequences and pages come out as NaN, positions below zero as
 * zeros: unit 0 also fills the rows in front of the sequence's start. */
template <int TYPE, typename T, int D>
__global__ __launch_bounds__(256) void sera_kv_read_kernel(kv_args a, T *__restrict__ k, int64_t k_stride,
                                                           T *__restrict__ v, int64_t v_stride) {
    using R = kv_rows<T, D>;
    constexpr bool Q8 = TYPE == (int)SERA_KV_Q8;
    constexpr int VEC = R::VEC, N = R::N, ES = Q8 ? 1 : 2;
    __shared__ kv_vec<uint32_t, 4> turn[4][D * ES];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int item = (int)blockIdx.y * 4 + wave, head = item >> 1;
    const bool is_v = item & 1;
    int unit;
    const kv_seq s = kv_find_sequence(a, (int)blockIdx.x, kBlock, 2, &unit);
    if (s.b < 0 || head >= a.kv_heads) return;
    const int64_t stride = is_v ? v_stride : k_stride;
    T *out = (is_v ? v : k) + (int64_t)head * D;
    const int before = s.bad ? s.n : min(max(s.n - s.len, 0), s.n);
    if (unit == 0 && before > 0) {
        kv_vec<T, VEC> o;
#pragma unroll
        for (int e = 0; e < VEC; e++) o.v[e] = kv_from_f32<T>(s.bad ? __builtin_nanf("") : 0.0f);
        for (int64_t r = s.row0 + lane / R::LANES; r < s.row0 + before; r += R::ROWS)
            *(kv_vec<T, VEC> *)(out + r * stride + R::channel(lane)) = o;
    }
    if (s.bad) return;
    const kv_unit u = kv_unit_of(s, unit);
    if (u.t0 >= u.t1) return;
    const int page = a.table[(size_t)s.b * a.table_stride + (u.pos0 >> a.page_shift)];
    const bool lost = page < 0 || page >= a.pages;
    const size_t kv_bytes = ((size_t)D << a.page_shift) * ES;
    const uint8_t *run = a.data + (lost ? 0 : (size_t)page * a.page_bytes) + (size_t)head * a.head_bytes;
    const int slot = u.pos0 & ((1 << a.page_shift) - 1);
    const uint8_t *from = run + (is_v ? kv_bytes : 0) + (size_t)slot * (D * ES);
    out += ((int64_t)s.row0 + u.pos0 - (s.len - s.n)) * stride;      /* of the block's token 0 */
    float scale = lost ? __builtin_nanf("") : 1.0f;                  /* of token `lane` */
    if (Q8 && lane < kBlock && !lost)
        scale = ((const float *)(run + 2 * kv_bytes))[((size_t)is_v << a.page_shift) + slot + lane];

    if (!is_v) {
        kv_vec<uint8_t, VEC * ES> in[N];
#pragma unroll
        for (int i = 0; i < N; i++)
            in[i] = *(const kv_vec<uint8_t, VEC * ES> *)(from + (R::token(i, lane) * D + R::channel(lane)) * ES);
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int t = R::token(i, lane);
            const float f = __shfl(scale, t, 64);
            kv_vec<T, VEC> o;
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                const uint16_t bits = (uint16_t)(in[i].v[e * ES] | in[i].v[e * ES + ES - 1] << 8);
                const float x = Q8 ? (float)(int8_t)in[i].v[e] : (float)__builtin_bit_cast(_Float16, bits);
                o.v[e] = kv_from_f32<T>(x * f);
            }
            if (t >= u.t0 && t < u.t1) kv_store_past(out + t * stride + R::channel(lane), o);
        }
        return;
    }
    /* V: channels 4c .. 4c+3 lie D / 4 places apart in LDS, so that lanes of consecutive c read side by side. */
    kv_vec<uint32_t, 4> in[D * ES / 64];
#pragma unroll
    for (int i = 0; i < D * ES / 64; i++) in[i] = ((const kv_vec<uint32_t, 4> *)from)[64 * i + lane];
#pragma unroll
    for (int i = 0; i < D * ES / 64; i++) {
        const int at = 64 * i + lane, ch = at / ES;
        turn[wave][(ch % 4 * (D / 4) + ch / 4) * ES + at % ES] = in[i];
    }
    asm volatile("" ::: "memory");
    constexpr int PER = 4 / ES;             /* tokens of a dword */
#pragma unroll
    for (int i = 0; i < D * kBlock / (4 * PER * 64); i++) {
        const int x = 64 * i + lane, c = x % (D / 4), q = x / (D / 4);    /* tokens PER * q .. of channels 4c .. */
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; j++) w[j] = turn[wave][(j * (D / 4) + c) * ES + q / 4].v[q % 4];
#pragma unroll
        for (int z = 0; z < PER; z++) {
            const int t = PER * q + z;
            const float f = __shfl(scale, t, 64);
            kv_vec<T, 4> o;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint16_t bits = (uint16_t)(w[j] >> (32 / PER * z));
                const float y = Q8 ? (float)(int8_t)bits : (float)__builtin_bit_cast(_Float16, bits);
                o.v[j] = kv_from_f32<T>(y * f);
            }
            if (t >= u.t0 && t < u.t1) kv_store_past(out + t * stride + 4 * c, o);
        }
    }
}

namespace {

template <int TYPE, typename T, int D>
hipError_t kv_move(bool write, const kv_args &a, void *k, int64_t ks, void *v, int64_t vs, hipStream_t s) {
    /* K and V of a head; written in halves of a block */
    const dim3 grid((unsigned)kv_slots(a.rows, a.sequences, kBlock, 2),
                    (unsigned)(write ? a.kv_heads : (2 * a.kv_heads + 3) / 4));
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
