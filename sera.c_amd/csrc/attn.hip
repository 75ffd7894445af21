/*
 * attn.hip - attention of packed rows over the paged cache.
 *
 *   s_j = scale * q . k_j,  o = sum_j 2^(s_j' - m) v_j / sum_j 2^(s_j' - m)
 *
 * with s' = s * log2(e) and m a running maximum, in one pass over the
 * visible positions j.
 */
#include "attn_common.h"
#include "sera_launch.h"

namespace {

/* One wave: the sums of one row over the visible positions in
 * [j0, j1), with plain FMAs. Lane l has the channels E*l .. E*l+E-1. */
template <int TYPE, int D>
struct attn_row {
    static constexpr int E = D / 64;
    float m, l, o[E];

    __device__ void run(const kv_args &a, const kv_seq &s, int head, const float *q, float c, int p, int window,
                        int sinks, int j0, int j1) {
        const int lane = threadIdx.x & 63;
        m = -3.402823466e38f;
        l = 0.0f;
#pragma unroll
        for (int e = 0; e < E; e++) o[e] = 0.0f;
        const int mask = (1 << a.page_shift) - 1;
        const size_t kv_elems = (size_t)D << a.page_shift;
        const int low = window > 0 ? max(p - window + 1, 0) : 0;
        for (int j = j0; j < min(j1, p + 1); j++) {
            if (j < low && j >= sinks) {
                j = min(low, j1) - 1;
                continue;
            }
            const int page = a.table[(size_t)s.b * a.table_stride + (j >> a.page_shift)];
            const bool lost = page < 0 || page >= a.pages;
            const uint8_t *run = a.data + (lost ? 0 : (size_t)page * a.page_bytes) + (size_t)head * a.head_bytes;
            const int slot = j & mask;
            const size_t ke = (size_t)slot * D + E * lane;
            const size_t ve = kv_elems + (size_t)(slot >> 4) * (16 * D) + (size_t)E * lane * 16 + (slot & 15);
            float acc = 0.0f, vx[E], ks = 1.0f, vs = 1.0f;
            if (TYPE == (int)SERA_KV_Q8) {
                const float *sc = (const float *)(run + 2 * kv_elems) + slot;
                ks = sc[0];
                vs = sc[(size_t)1 << a.page_shift];
            }
#pragma unroll
            for (int e = 0; e < E; e++) {
                float kx;
                if (TYPE == (int)SERA_KV_F16) {
                    kx = (float)((const _Float16 *)run)[ke + e];
                    vx[e] = (float)((const _Float16 *)run)[ve + 16 * e];
                } else {
                    kx = (float)((const int8_t *)run)[ke + e];
                    vx[e] = (float)((const int8_t *)run)[ve + 16 * e] * vs;
                }
                acc = fmaf(kx, q[e], acc);
            }
#pragma unroll
            for (int x = 32; x >= 1; x >>= 1) acc += __shfl_xor(acc, x, 64);
            const float t = lost ? __builtin_nanf("") : acc * ks * c;
            const float mn = fmaxf(m, t), f = exp2f(m - mn), w = exp2f(t - mn);
            l = fmaf(l, f, w);
#pragma unroll
            for (int e = 0; e < E; e++) o[e] = fmaf(o[e], f, w * vx[e]);
            m = mn;
        }
    }
};

}  // namespace

template <int TYPE, typename T, int D>
__global__ __launch_bounds__(256) void sera_attn_row_kernel(kv_args a, attn_args t) {
    constexpr int E = D / 64;
    const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (unit >= (int64_t)a.rows * t.heads) return;
    const int row = (int)(unit / t.heads), h = (int)(unit % t.heads), lane = threadIdx.x & 63;
    int i;
    const int b = kv_find(a, row, 1, 0, &i);
    const T *q = (const T *)t.q + row * t.q_stride + (int64_t)h * D + E * lane;
    T *out = (T *)t.out + row * t.out_stride + (int64_t)h * D + E * lane;
    if (b < 0) return;
    const kv_seq s = kv_sequence(a, b);
    if (i >= s.n) return;
    attn_row<TYPE, D> r;
    const int p = s.len - s.n + i;
    float qx[E];
#pragma unroll
    for (int e = 0; e < E; e++) qx[e] = kv_to_f32(q[e]);
    if (!s.bad) r.run(a, s, h / t.group, qx, t.scale_log2, p, t.window, t.sinks, 0, s.len);
#pragma unroll
    for (int e = 0; e < E; e++)
        out[e] = kv_from_f32<T>(s.bad ? __builtin_nanf("") : p < 0 ? 0.0f : r.o[e] / r.l);
}

namespace {

template <int TYPE, typename T, int D>
hipError_t attn_go(const kv_args &a, const attn_args &t, hipStream_t s) {
    hipLaunchKernelGGL((sera_attn_row_kernel<TYPE, T, D>), dim3((unsigned)(((int64_t)a.rows * t.heads + 3) / 4)),
                       dim3(256), 0, s, a, t);
    return hipGetLastError();
}

template <int TYPE, typename T>
hipError_t attn_d(int dim, const kv_args &a, const attn_args &t, hipStream_t s) {
    return dim == 64 ? attn_go<TYPE, T, 64>(a, t, s) : attn_go<TYPE, T, 128>(a, t, s);
}

template <int TYPE>
hipError_t attn_t(uint32_t type, int dim, const kv_args &a, const attn_args &t, hipStream_t s) {
    if (type == SERA_TYPE_F32) return attn_d<TYPE, float>(dim, a, t, s);
    if (type == SERA_TYPE_F16) return attn_d<TYPE, _Float16>(dim, a, t, s);
    return attn_d<TYPE, __bf16>(dim, a, t, s);
}

}  // namespace

size_t sera_attn_workspace(const kv_args &a, int dim, int heads, int cus) { return 0; }

/* Arguments are checked by the caller (sera_attn_runtime.hip). */
hipError_t sera_launch_attn(uint32_t cache_type, uint32_t type, int dim, const kv_args &a, const attn_args &t,
                            hipStream_t s) {
    return cache_type == SERA_KV_F16 ? attn_t<(int)SERA_KV_F16>(type, dim, a, t, s)
                                     : attn_t<(int)SERA_KV_Q8>(type, dim, a, t, s);
}
