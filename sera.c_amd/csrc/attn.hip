/*
 * attn.hip - attention of packed rows over the paged cache: which kernel takes
 * a call and how it is cut up, and the kernel that joins contexts split over
 * workgroups.
 *
 *   s_j = scale * q . k_j,  o = sum_j 2^(s_j' - m) v_j / sum_j 2^(s_j' - m)
 *
 * with s' = s * log2(e) and m a running maximum, in one pass over the
 * visible positions j.
 */
#include "attn_device.h"
#include "sera_launch.h"

namespace {

constexpr int kMaxSplits = 64;

/* The workspace has no window in its size (it is asked for before the call
 * that names one), so the split is chosen without it and a window only
 * shortens the chunks. */
attn_plan plan_of(uint32_t cache_type, const kv_args &a, int heads, int cus) {
    attn_plan p = {};
    p.shift = 5;
    const int group = heads / a.kv_heads;
    const int64_t columns = (int64_t)a.max_new * group;
    int64_t want;
    int least;           /* tiles of a chunk, at least */
    if (columns <= 32) {
        p.columns = columns <= 8 ? 8 : columns <= 16 ? 16 : 32;
        p.waves = 4;
        p.slots = a.sequences;
        /* Split contexts only as far as there are CUs without a workgroup: joining costs a launch, and more workgroups a
         * CU repeat the start (32 windows of 1024 tokens, 256 workgroups: 34 us whole, 40 in two; 24 contexts of 1050-2100
         * tokens, 192 workgroups: 32 us whole, 33 in two, 31 in four; one context of 8000, 8 workgroups whole: 17 us in 32,
         * 18 in 63). */
        want = (int64_t)cus / ((int64_t)a.sequences * a.kv_heads);
        least = p.waves;                      /* a tile for every wave */
    } else {
        p.waves = 8;
        const int64_t all = (int64_t)a.rows * group;
        /* 256 rows a workgroup load each key and value for the most rows, if that leaves every CU one. If not, 128
         * rows (two groups of waves over the tokens) for contexts up to 8192 tokens, where partial sums cost more
         * than they give: 16 branches of 256 rows over 1568 tokens take 74 us so and 93 us as 256 rows split in two;
         * 512 rows x 8 over 32768 tokens 1175 us so and 1031 us split. */
        p.columns = 256;
        while (p.columns > 64 && columns <= p.columns / 2) p.columns /= 2;
        if (p.columns == 256 && (all + 255) / 256 * a.kv_heads < cus && a.max_kv <= 8192) p.columns = 128;
        p.slots = (int)(all / p.columns + a.sequences);
        const int64_t units = (all + p.columns - 1) / p.columns * a.kv_heads;
        want = cus / units;
        least = 8;
    }
    const int tiles = (a.max_kv + (1 << p.shift) - 1) >> p.shift;
    if (want > (tiles + least - 1) / least) want = (tiles + least - 1) / least;
    if (want > kMaxSplits) want = kMaxSplits;
    p.splits = want < 1 ? 1 : (int)want;
    p.chunk = (tiles + p.splits - 1) / p.splits;
    return p;
}

}  // namespace

/* Joins the partial sums of a row: a wave for each (row, query head).
 * per 0: a unit of partial sums has a sequence's rows (all max_new); otherwise `per` rows of the tile kernel. */
template <typename T, int D>
__global__ __launch_bounds__(256) void sera_attn_join_kernel(kv_args a, attn_args t, int per, int splits, int chunk,
                                                             int shift) {
    constexpr int E = D / 64;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int i;
    const kv_seq s = kv_find_sequence(a, (int)blockIdx.x, 1, 0, &i);
    if (s.b < 0 || s.bad || i >= s.n) return;
    const int first = s.len - s.n, rows = s.n * t.group, unit_rows = per ? per : a.max_new * t.group;
    const int tile0 = per ? attn_first_tile(a, t.group, per, s.b, s.row0) : 0;
    for (int h = (int)blockIdx.y * 4 + wave; h < t.heads; h += (int)gridDim.y * 4) {
        const int head = h / t.group, row = i * t.group + h % t.group, unit = row / unit_rows;
        const int r = row - unit * unit_rows, last = min((unit + 1) * unit_rows, rows) - 1;
        const attn_range range = attn_range_of(t, max(first + unit * unit_rows / t.group, 0),
                                               first + last / t.group + 1, shift);
        const int used = max((range.count + chunk - 1) / chunk, 1);
        const size_t step = attn_partial_floats(unit_rows, D);
        const int slot = per ? tile0 + unit : s.b;
        const float *part = t.workspace + ((size_t)slot * a.kv_heads + head) * splits * step;
        const float *from = part + (size_t)r * D + E * lane;
        /* sums are loaded 16 splits at a time, the first together with the maxima that weigh them */
        constexpr int BATCH = 16;
        attn_vec<float, E> x[BATCH];
#pragma unroll
        for (int k = 0; k < BATCH; k++) x[k] = *(const attn_vec<float, E> *)(from + min(k, used - 1) * step);
        float m = kAttnLowest, l = 0.0f;
        if (lane < used) {
            const attn_f2 ml = *(const attn_f2 *)(part + lane * step + (size_t)unit_rows * D + 2 * r);
            m = ml[0];
            l = ml[1];
        }
        float top = m;
        top = fmaxf(top, xor_partner<1>(top));
        top = fmaxf(top, xor_partner<2>(top));
        top = fmaxf(top, xor_partner<4>(top));
        top = fmaxf(top, xor_partner<8>(top));
        top = fmaxf(top, xor_partner<16>(top));
        top = fmaxf(top, xor_partner<32>(top));
        const float f = lane < used ? attn_exp2(m - top) : 0.0f;
        l *= f;
        l += xor_partner<1>(l);
        l += xor_partner<2>(l);
        l += xor_partner<4>(l);
        l += xor_partner<8>(l);
        l += xor_partner<16>(l);
        l += xor_partner<32>(l);
        float y[E] = {};
        for (int base = 0; base < used; base += BATCH) {
            if (base > 0)
#pragma unroll
                for (int k = 0; k < BATCH; k++)
                    x[k] = *(const attn_vec<float, E> *)(from + min(base + k, used - 1) * step);
#pragma unroll
            for (int k = 0; k < BATCH; k++) {
                const float w = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f), (base + k) & 63));
#pragma unroll
                for (int e = 0; e < E; e++) y[e] = base + k < used ? fmaf(x[k].v[e], w, y[e]) : y[e];
            }
        }
        attn_vec<T, E> o;
#pragma unroll
        for (int e = 0; e < E; e++) o.v[e] = kv_from_f32<T>(first + i < 0 ? 0.0f : y[e] / l);
        *(attn_vec<T, E> *)((T *)t.out + (s.row0 + i) * t.out_stride + (int64_t)h * D + E * lane) = o;
    }
}

namespace {

template <typename T>
void join_t(int dim, const kv_args &a, const attn_args &t, const attn_plan &p, hipStream_t s) {
    const dim3 grid((unsigned)a.rows, (unsigned)((t.heads + 3) / 4));
    const int per = p.columns > 32 ? p.columns : 0;
    if (dim == 64)
        hipLaunchKernelGGL((sera_attn_join_kernel<T, 64>), grid, dim3(256), 0, s, a, t, per, p.splits, p.chunk, p.shift);
    else
        hipLaunchKernelGGL((sera_attn_join_kernel<T, 128>), grid, dim3(256), 0, s, a, t, per, p.splits, p.chunk, p.shift);
}

}  // namespace

size_t sera_attn_workspace(uint32_t cache_type, const kv_args &a, int dim, int heads, int cus) {
    const attn_plan p = plan_of(cache_type, a, heads, cus);
    if (p.splits < 2) return 0;
    const size_t rows = p.columns > 32 ? (size_t)p.columns : (size_t)a.max_new * (heads / a.kv_heads);
    return (size_t)p.slots * a.kv_heads * p.splits * rows * (dim + 2) * sizeof(float);
}

/* Arguments are checked by the caller (sera_attn_runtime.hip). */
hipError_t sera_launch_attn(uint32_t cache_type, uint32_t type, int dim, const kv_args &a, const attn_args &t,
                            hipStream_t s) {
    attn_plan p = plan_of(cache_type, a, t.heads, t.cus);
    if (t.window > 0) {
        const int64_t tile = 1 << p.shift, sinks = t.sinks < a.max_kv ? t.sinks : a.max_kv;
        const int64_t tiles = (sinks + tile - 1) / tile + ((int64_t)t.window + a.max_new + tile - 2) / tile + 1;
        const int64_t chunk = (tiles + p.splits - 1) / p.splits;
        if (chunk < p.chunk) p.chunk = (int)chunk;
    }
    hipError_t e = p.columns > 32 ? sera_launch_attn_tile(cache_type, type, dim, a, t, p, s)
                                  : sera_launch_attn_few(cache_type, type, dim, a, t, p, s);
    if (e != hipSuccess || p.splits < 2) return e;
    if (type == SERA_TYPE_F32) join_t<float>(dim, a, t, p, s);
    else if (type == SERA_TYPE_F16) join_t<_Float16>(dim, a, t, p, s);
    else join_t<__bf16>(dim, a, t, p, s);
    return hipGetLastError();
}
