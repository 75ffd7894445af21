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
 */
#include "attn_common.h"
#include "kv_device.h"
#include "sera_launch.h"

#pragma clang fp contract(off)

namespace {

typedef uint32_t kv_u4 __attribute__((ext_vector_type(4)));
typedef uint32_t kv_u2 __attribute__((ext_vector_type(2)));

/* Stores past the caches: rows read back are larger than what they come from and only stream through (37922 tokens
 * out of an 8-bit cache take 80 us so, 94 us with ordinary stores; out of an fp16 cache 118 and 116). */
template <typename T, int N>
__device__ __forceinline__ void kv_store_past(T *p, const kv_vec<T, N> &v) {
    if constexpr (sizeof(v) == 16) __builtin_nontemporal_store(__builtin_bit_cast(kv_u4, v), (kv_u4 *)p);
    else __builtin_nontemporal_store(__builtin_bit_cast(kv_u2, v), (kv_u2 *)p);
}

struct kv_same {
    template <typename X>
    __device__ __forceinline__ void operator()(X *, int) const {}
};

}  // namespace

template <int TYPE, typename T, int D>
__global__ __launch_bounds__(256) void sera_kv_write_kernel(kv_args a, const T *__restrict__ k, int64_t k_stride,
                                                            const T *__restrict__ v, int64_t v_stride) {
    constexpr int TOKENS = kBlock / 2, ROW = D * (TYPE == (int)SERA_KV_Q8 ? 1 : 2) / 4;   /* dwords of a row in LDS */
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
    uint8_t *run = a.data + (size_t)page * a.page_bytes + (size_t)head * a.head_bytes;
    const int64_t stride = is_v ? v_stride : k_stride;
    /* row of the block's token 0; only tokens t0 .. t1-1 have one */
    const int64_t row = (int64_t)s.row0 + u.pos0 - (s.len - s.n);
    const T *from = (is_v ? v : k) + row * stride + (int64_t)head * D + kv_rows<T, D>::channel(lane);
    kv_put_half<TYPE, T, D>(a, u, h0, is_v, run, from, stride, turn[wave], lane, kv_same());
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
