/*
 * kv_rope.hip - rows into the paged cache with q's and k's heads normed and rotated on the way.
 *
 *   x' = (x * (1 / sqrt(mean(x^2) + eps))) * gamma          over a head's channels
 *   (a, b) -> (a cos t - b sin t, a sin t + b cos t)        t = position * inv_freq[i]
 *
 * A workgroup has a 16-token block of a sequence and some of its heads. The block's sines and cosines are made once,
 * in LDS, for all of them: position * inv_freq / 2 pi in 64 bits, less the whole turns, then fp32. A head's channels
 * lie in the 16-byte accesses of one row's lanes, so the mean and the partner of a channel come from other lanes of
 * the row. q goes back to rows, k and v to the cache as kv_write puts them there. The workgroups of a block lie
 * beside each other, as its rows do in memory.
 *
 * Bound by memory: each row is read and written once. A prompt of 2048 fp32 rows (64 heads of q, 8 of k and v, 128
 * channels, fp16 cache): 39 us for 160 MB, 4.1 TB/s of the 5.2 that a copy reaches, 42 us (37 at the least) into an 8-bit
 * cache; of bf16 rows into an 8-bit cache 26 us for 80 MB. 16 single tokens: 6.4 us, which is latency.
 */
#include "attn_common.h"
#include "kv_device.h"
#include "sera_launch.h"

#include <type_traits>

#pragma clang fp contract(off)

namespace {

/* x of the lane `apart` (1, 2, 4, 8 or 16) away. */
template <int VEC>
__device__ __forceinline__ void rope_partner(const float *x, float *y, int apart) {
    switch (apart) {
#define SERA_CASE(N)                                                      \
    case N:                                                               \
        _Pragma("unroll") for (int e = 0; e < VEC; e++) y[e] = xor_partner<N>(x[e]); \
        break;
        SERA_CASE(1)
        SERA_CASE(2)
        SERA_CASE(4)
        SERA_CASE(8)
        SERA_CASE(16)
#undef SERA_CASE
    default:
#pragma unroll
        for (int e = 0; e < VEC; e++) y[e] = x[e];
    }
}

template <int LANES>
__device__ __forceinline__ float rope_row_sum(float s) {
    s += xor_partner<1>(s);
    s += xor_partner<2>(s);
    s += xor_partner<4>(s);
    if constexpr (LANES >= 16) s += xor_partner<8>(s);
    if constexpr (LANES >= 32) s += xor_partner<16>(s);
    return s;
}

/* The norm and the turn of a lane's channels of one head of a token. */
template <typename T, int D>
struct rope_turn {
    using R = kv_rows<T, D>;
    float gamma[R::VEC], eps;
    const float (*cosine)[64], (*sine)[64];   /* by token of the block and pair */
    int half, d0;                             /* pairs; the lane's first channel */
    bool norm, neighbours;

    __device__ __forceinline__ void operator()(float *x, int t) const {
        constexpr int VEC = R::VEC;
        if (norm) {
            float s = 0.0f;
#pragma unroll
            for (int e = 0; e < VEC; e++) s = fmaf(x[e], x[e], s);
            const float r = 1.0f / sqrtf(rope_row_sum<R::LANES>(s) * (1.0f / D) + eps);
#pragma unroll
            for (int e = 0; e < VEC; e++) x[e] = x[e] * r * gamma[e];
        }
        if (half == 0) return;
        const bool turns = d0 < 2 * half;
        if (neighbours) {
            const int i = turns ? d0 / 2 : 0;
#pragma unroll
            for (int e = 0; e < VEC; e += 2) {
                const float c = cosine[t][i + e / 2], s = sine[t][i + e / 2];
                const float a = x[e], b = x[e + 1];
                x[e] = turns ? fmaf(a, c, -(b * s)) : a;
                x[e + 1] = turns ? fmaf(a, s, b * c) : b;
            }
        } else {
            const int i = d0 & (half - 1);
            const float sign = d0 < half ? -1.0f : 1.0f;
            float y[VEC];
            rope_partner<VEC>(x, y, half / VEC);
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                const float c = cosine[t][i + e], s = sine[t][i + e] * sign;
                x[e] = turns ? fmaf(x[e], c, y[e] * s) : x[e];
            }
        }
    }
};

struct kv_same {
    template <typename X>
    __device__ __forceinline__ void operator()(X *, int) const {}
};

}  // namespace

/* Item i of a block: q's head i, or behind those of a kv head the halves of its K and of its V. A workgroup has `per`
 * of them. */
template <int TYPE, typename T, int D>
__global__ __launch_bounds__(256) void sera_kv_rope_kernel(kv_args a, rope_args r, const T *q, int64_t q_stride,
                                                           T *q_out, int64_t q_out_stride, const T *__restrict__ k,
                                                           int64_t k_stride, const T *__restrict__ v,
                                                           int64_t v_stride, int per) {
    using R = kv_rows<T, D>;
    constexpr int VEC = R::VEC, N = R::N, TOKENS = kBlock / 2, ROW = D * (TYPE == (int)SERA_KV_Q8 ? 1 : 2) / 4;
    __shared__ uint32_t turn[4][TOKENS][ROW];
    __shared__ __attribute__((aligned(16))) float cosine[kBlock][64], sine[kBlock][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int items = r.heads + 4 * a.kv_heads, groups = (items + per - 1) / per;
    const int first_item = (int)(blockIdx.x % groups) * per;
    int unit;
    const kv_seq s = kv_find_sequence(a, (int)(blockIdx.x / groups), kBlock, 2, &unit);
    if (s.b < 0) return;
    const int last_item = min(first_item + per, items), d0 = R::channel(lane);
    /* rows without a place in the cache */
    const int before = s.bad ? s.n : min(max(s.n - s.len, 0), s.n);
    if (unit == 0 && before > 0) {
        kv_vec<T, VEC> o;
#pragma unroll
        for (int e = 0; e < VEC; e++) o.v[e] = kv_from_f32<T>(s.bad ? __builtin_nanf("") : 0.0f);
        for (int it = first_item + wave; it < min(last_item, r.heads); it += 4)
            for (int64_t row = s.row0 + lane / R::LANES; row < s.row0 + before; row += R::ROWS)
                *(kv_vec<T, VEC> *)(q_out + row * q_out_stride + (int64_t)it * D + d0) = o;
    }
    if (s.bad) return;
    const kv_unit u = kv_unit_of(s, unit);
    if (u.t0 >= u.t1) return;
    const int page = a.table[(size_t)s.b * a.table_stride + (u.pos0 >> a.page_shift)];
    const int64_t row = (int64_t)s.row0 + u.pos0 - (s.len - s.n);     /* of the block's token 0 */

    /* The next of q's heads, on its way while the angles are made and while the one before it is turned. */
    kv_vec<T, VEC> in[N];
    const auto load = [&](int it, int i) {
        const int t = min(max(R::token(i, lane), u.t0), u.t1 - 1);
        in[i] = *(const kv_vec<T, VEC> *)(q + (row + t) * q_stride + (int64_t)it * D + d0);
    };
    const auto some = [&](int i) { return (i + 1) * R::ROWS > u.t0 && i * R::ROWS < u.t1; };
    int it = first_item + wave;
    const int last_q = min(last_item, r.heads);
    if (it < last_q)
#pragma unroll
        for (int i = 0; i < N; i++)
            if (some(i)) load(it, i);
    if (r.half) {
        const int shift = __builtin_ctz(r.half);
        for (int x = tid; x < (u.t1 - u.t0) << shift; x += 256) {
            const int t = u.t0 + (x >> shift), i = x & (r.half - 1);
            const int at = r.positions ? r.positions[row + t] : u.pos0 + t;
            double turns = (double)at * (double)r.inv_freq[i] * 0.15915494309189535;   /* 1 / (2 pi) */
            turns -= rint(turns);
            const float h = (float)(2.0 * turns), rest = (float)((2.0 * turns - h) * M_PI);   /* what h rounds off */
            float s, c;
            sincospif(h, &s, &c);
            sine[t][i] = fmaf(rest, c, s);
            cosine[t][i] = fmaf(-rest, s, c);
        }
    }
    __syncthreads();

    rope_turn<T, D> change;
    change.eps = r.eps;
    change.cosine = cosine;
    change.sine = sine;
    change.half = r.half;
    change.d0 = d0;
    change.neighbours = r.neighbours;
    const auto gamma_of = [&](const float *g) {
        change.norm = g != nullptr;
        if (g)
#pragma unroll
            for (int e = 0; e < VEC; e++) change.gamma[e] = g[d0 + e];
    };
    const auto heads = [&](auto whole) {        /* whole: all 16 tokens, so that what is on its way can be counted */
        for (; it < last_q; it += 4) {
            const int next = min(it + 4, last_q - 1);
#pragma unroll
            for (int i = 0; i < N; i++) {
                if (!whole.value && !some(i)) continue;
                const int t = R::token(i, lane);
                float x[VEC];
#pragma unroll
                for (int e = 0; e < VEC; e++) x[e] = kv_to_f32(in[i].v[e]);
                load(next, i);
                change(x, t);
                kv_vec<T, VEC> o;
#pragma unroll
                for (int e = 0; e < VEC; e++) o.v[e] = kv_from_f32<T>(x[e]);
                if (whole.value || (t >= u.t0 && t < u.t1))
                    *(kv_vec<T, VEC> *)(q_out + (row + t) * q_out_stride + (int64_t)it * D + d0) = o;
            }
        }
    };
    gamma_of(r.q_gamma);
    if (u.t0 == 0 && u.t1 == kBlock) heads(std::true_type());
    else heads(std::false_type());
    gamma_of(r.k_gamma);
    for (; it < last_item; it += 4) {
        const int x = it - r.heads, head = x >> 2, h0 = (x & 1) * TOKENS;
        kv_unit part = u;
        part.t0 = max(u.t0, h0);
        part.t1 = min(u.t1, h0 + TOKENS);
        if (part.t0 >= part.t1 || page < 0 || page >= a.pages) continue;
        uint8_t *run = a.data + (size_t)page * a.page_bytes + (size_t)head * a.head_bytes;
        if (x & 2)
            kv_put_half<TYPE, T, D>(a, part, h0, true, run, v + row * v_stride + (int64_t)head * D + d0, v_stride,
                                    turn[wave], lane, kv_same());
        else
            kv_put_half<TYPE, T, D>(a, part, h0, false, run, k + row * k_stride + (int64_t)head * D + d0, k_stride,
                                    turn[wave], lane, change);
    }
}

namespace {

template <int TYPE, typename T, int D>
void rope_go(const kv_args &a, const rope_args &r, const void *q, int64_t qs, void *q_out, int64_t qos, const void *k,
             int64_t ks, const void *v, int64_t vs, hipStream_t s) {
    /* Items of a workgroup: one for each wave, and more of them only where that leaves 4 workgroups for every compute
     * unit, as each makes its block's angles and finds its sequence anew. A prompt of 2048 rows of 64 heads (fp32): 4
     * items 45 us, 16 39 us; 9 chunks of up to 701 rows of 20 heads of 64 (bf16): 4 items 12.9 us, 12 9.5 us; single
     * tokens of 16: 4 items 6.4 us, 8 7.6 us. */
    const int64_t slots = kv_slots(a.rows, a.sequences, kBlock, 2), blocks = slots < a.rows ? slots : a.rows;
    const int64_t items = r.heads + 4 * a.kv_heads, want = 4 * ((blocks * items + 16 * r.cus - 1) / (16 * r.cus));
    /* and as many as a launch's limit takes, where nearly all slots of very many sequences are empty (2^20 of them have
     * 2^21 slots, for up to 7 workgroups each) */
    const int64_t groups = kAttnMaxGrid / slots, least = (items + groups - 1) / groups;
    const int64_t wanted = want > least ? want : least;
    const int per = (int)(wanted < items ? wanted : items);
    hipLaunchKernelGGL((sera_kv_rope_kernel<TYPE, T, D>), dim3((unsigned)(slots * ((items + per - 1) / per))),
                       dim3(256), 0, s, a, r, (const T *)q, qs, (T *)q_out, qos, (const T *)k, ks, (const T *)v, vs,
                       per);
}

template <int TYPE, typename T>
void rope_d(int dim, const kv_args &a, const rope_args &r, const void *q, int64_t qs, void *q_out, int64_t qos,
            const void *k, int64_t ks, const void *v, int64_t vs, hipStream_t s) {
    if (dim == 64) rope_go<TYPE, T, 64>(a, r, q, qs, q_out, qos, k, ks, v, vs, s);
    else rope_go<TYPE, T, 128>(a, r, q, qs, q_out, qos, k, ks, v, vs, s);
}

template <int TYPE>
void rope_t(uint32_t type, int dim, const kv_args &a, const rope_args &r, const void *q, int64_t qs, void *q_out,
            int64_t qos, const void *k, int64_t ks, const void *v, int64_t vs, hipStream_t s) {
    if (type == SERA_TYPE_F32) rope_d<TYPE, float>(dim, a, r, q, qs, q_out, qos, k, ks, v, vs, s);
    else if (type == SERA_TYPE_F16) rope_d<TYPE, _Float16>(dim, a, r, q, qs, q_out, qos, k, ks, v, vs, s);
    else rope_d<TYPE, __bf16>(dim, a, r, q, qs, q_out, qos, k, ks, v, vs, s);
}

}  // namespace

/* Arguments are checked by the caller (sera_attn_runtime.hip). */
hipError_t sera_launch_kv_rope(uint32_t cache_type, uint32_t type, int dim, const kv_args &a, const rope_args &r,
                               const void *q, int64_t q_stride, void *q_out, int64_t q_out_stride, const void *k,
                               int64_t k_stride, const void *v, int64_t v_stride, hipStream_t s) {
    if (cache_type == SERA_KV_F16)
        rope_t<(int)SERA_KV_F16>(type, dim, a, r, q, q_stride, q_out, q_out_stride, k, k_stride, v, v_stride, s);
    else
        rope_t<(int)SERA_KV_Q8>(type, dim, a, r, q, q_stride, q_out, q_out_stride, k, k_stride, v, v_stride, s);
    return hipGetLastError();
}
