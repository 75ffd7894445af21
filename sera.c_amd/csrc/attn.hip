/*
 * attn.hip - attention of packed rows over the paged cache.
 *
 *   s_j = scale * q . k_j,  o = sum_j 2^(s_j' - m) v_j / sum_j 2^(s_j' - m)
 *
 * with s' = s * log2(e) and m a running maximum, in one pass over the
 * visible positions j.
 */
#include "attn_device.h"
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

namespace {

constexpr int kMaxSplits = 64;

/* The workspace has no window in its size (it is asked for before the call
 * that names one), so the split is chosen without it and a window only
 * shortens the chunks. */
attn_plan plan_of(uint32_t cache_type, const kv_args &a, int heads, int cus) {
    attn_plan p = {};
    const int columns = a.max_new * (heads / a.kv_heads);
    if ((int64_t)a.max_new * (heads / a.kv_heads) > 32) return p;
    p.columns = columns <= 16 ? 16 : 32;
    p.waves = 4;
    const int tile = sera_attn_few_tile(cache_type);
    const int tiles = (a.max_kv + tile - 1) / tile;
    const int64_t units = (int64_t)a.sequences * a.kv_heads;
    /* Two workgroups per CU are resident at once: more of them only repeat the start. */
    int64_t want = 2 * (int64_t)cus / units;
    const int most = (tiles + p.waves - 1) / p.waves;       /* a tile for every wave */
    if (want > most) want = most;
    if (want > kMaxSplits) want = kMaxSplits;
    p.splits = want < 1 ? 1 : (int)want;
    p.chunk = (tiles + p.splits - 1) / p.splits;
    return p;
}

}  // namespace

/* Joins the partial sums of a row: a wave for each (row, query head). */
template <typename T, int D>
__global__ __launch_bounds__(256) void sera_attn_join_kernel(kv_args a, attn_args t, int splits, int chunk, int shift) {
    constexpr int E = D / 64;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int i;
    const int b = kv_find(a, (int)blockIdx.x, 1, 0, &i);
    if (b < 0) return;
    const kv_seq s = kv_sequence(a, b);
    if (s.bad || i >= s.n) return;
    const int part_rows = a.max_new * t.group, p = s.len - s.n + i;
    const attn_range range = attn_range_of(t, max(s.len - s.n, 0), s.len, shift);
    const int used = max((range.count + chunk - 1) / chunk, 1);
    for (int h = (int)blockIdx.y * 4 + wave; h < t.heads; h += (int)gridDim.y * 4) {
        const int head = h / t.group, r = i * t.group + h % t.group;
        const size_t step = attn_partial_floats(part_rows, D);
        const float *part = t.workspace + ((size_t)b * a.kv_heads + head) * splits * step;
        float m = kAttnLowest, l = 0.0f;
        if (lane < used) {
            const attn_f2 x = *(const attn_f2 *)(part + lane * step + (size_t)part_rows * D + 2 * r);
            m = x[0];
            l = x[1];
        }
        float top = m;
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
        const float f = lane < used ? attn_exp2(m - top) : 0.0f;
        l *= f;
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) l += __shfl_xor(l, o, 64);
        float y[E] = {};
        for (int k = 0; k < used; k++) {
            const attn_vec<float, E> x = *(const attn_vec<float, E> *)(part + k * step + (size_t)r * D + E * lane);
            const float w = __shfl(f, k, 64);
#pragma unroll
            for (int e = 0; e < E; e++) y[e] = fmaf(x.v[e], w, y[e]);
        }
        attn_vec<T, E> o;
#pragma unroll
        for (int e = 0; e < E; e++) o.v[e] = kv_from_f32<T>(p < 0 ? 0.0f : y[e] / l);
        *(attn_vec<T, E> *)((T *)t.out + (s.row0 + i) * t.out_stride + (int64_t)h * D + E * lane) = o;
    }
}

namespace {

template <typename T>
void join_t(int dim, const kv_args &a, const attn_args &t, const attn_plan &p, int shift, hipStream_t s) {
    const dim3 grid((unsigned)a.rows, (unsigned)((t.heads + 3) / 4));
    if (dim == 64)
        hipLaunchKernelGGL((sera_attn_join_kernel<T, 64>), grid, dim3(256), 0, s, a, t, p.splits, p.chunk, shift);
    else
        hipLaunchKernelGGL((sera_attn_join_kernel<T, 128>), grid, dim3(256), 0, s, a, t, p.splits, p.chunk, shift);
}

}  // namespace

size_t sera_attn_workspace(uint32_t cache_type, const kv_args &a, int dim, int heads, int cus) {
    const attn_plan p = plan_of(cache_type, a, heads, cus);
    if (p.splits < 2) return 0;
    return (size_t)a.sequences * a.kv_heads * p.splits * (size_t)a.max_new * (heads / a.kv_heads) * (dim + 2) *
           sizeof(float);
}

/* Arguments are checked by the caller (sera_attn_runtime.hip). */
hipError_t sera_launch_attn(uint32_t cache_type, uint32_t type, int dim, const kv_args &a, const attn_args &t,
                            hipStream_t s) {
    attn_plan p = plan_of(cache_type, a, t.heads, t.cus);
    if (!p.columns)
        return cache_type == SERA_KV_F16 ? attn_t<(int)SERA_KV_F16>(type, dim, a, t, s)
                                         : attn_t<(int)SERA_KV_Q8>(type, dim, a, t, s);
    const int tile = sera_attn_few_tile(cache_type);
    if (t.window > 0) {
        const int64_t sinks = t.sinks < a.max_kv ? t.sinks : a.max_kv;
        const int64_t tiles = (sinks + tile - 1) / tile + ((int64_t)t.window + a.max_new + tile - 2) / tile + 1;
        const int64_t chunk = (tiles + p.splits - 1) / p.splits;
        if (chunk < p.chunk) p.chunk = (int)chunk;
    }
    hipError_t e = sera_launch_attn_few(cache_type, type, dim, a, t, p, s);
    if (e != hipSuccess || p.splits < 2) return e;
    const int shift = __builtin_ctz((unsigned)tile);
    if (type == SERA_TYPE_F32) join_t<float>(dim, a, t, p, shift, s);
    else if (type == SERA_TYPE_F16) join_t<_Float16>(dim, a, t, p, shift, s);
    else join_t<__bf16>(dim, a, t, p, shift, s);
    return hipGetLastError();
}
