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

constexpr int kMaxSplits = 64, kFewColumns = 32;

void split_of(attn_plan &p, const kv_args &a, int64_t want, int least) {
    const int tiles = (a.max_kv + (1 << kAttnShift) - 1) >> kAttnShift, most = (tiles + least - 1) / least;
    if (want > most) want = most;
    if (want > kMaxSplits) want = kMaxSplits;
    p.splits = want < 1 ? 1 : (int)want;
    p.chunk = (tiles + p.splits - 1) / p.splits;
}

struct attn_plans {
    attn_plan few, tile;
    int few_columns, few_rows;
    size_t few_bytes, bytes;     /* workspace: partial sums of the few-row kernel, then of the tiles */
};

/* The workspace has no window in its size (it is asked for before the call
 * that names one), so the split is chosen without it and a window only
 * shortens the chunks. */
attn_plans plan_of(const kv_args &a, int dim, int heads, int cus) {
    attn_plans p = {};
    const int group = heads / a.kv_heads;
    const int64_t columns = (int64_t)a.max_new * group;
    /* One kernel takes all sequences, unless they differ much: where they have less than half of the longest one's
     * rows on average, those of a token or so (a group's rows, rounded up to what the few-row kernel holds) go to it
     * and the others to the tiles, in two launches (a chunk of 512 rows over 4096 positions and 31 tokens over 3000
     * each: 235 us, 279 all in tiles; from an 8-bit cache 229 and 305; 64 rows and 63 tokens over 3000: 188 and 333,
     * 132 and 352). */
    if (columns <= kFewColumns) p.few_columns = 0x7fffffff;
    else if (group <= kFewColumns && 2ll * a.rows < (int64_t)a.sequences * a.max_new)
        p.few_columns = group <= 8 ? 8 : group <= 16 ? 16 : 32;
    if (p.few_columns) {
        const int most = columns < p.few_columns ? (int)columns : p.few_columns;
        p.few.columns = most <= 8 ? 8 : most <= 16 ? 16 : 32;
        p.few_rows = columns <= kFewColumns ? (int)columns : p.few_columns / group * group;
        /* Split contexts only as far as there are CUs without a workgroup: joining costs a launch, and more
         * workgroups a CU repeat the start (32 windows of 1024 tokens, 256 workgroups: 33 us whole, 38 in two; 24
         * contexts of 1050-2100 tokens, 192 workgroups: 39 us whole, 44 in two, from an 8-bit cache 25 and 29; one
         * context of 8000, 8 workgroups whole: 15 us in 32, 17 in 63). At least a tile for each of the four waves. */
        split_of(p.few, a, (int64_t)cus / ((int64_t)a.sequences * a.kv_heads), 4);
    }
    if (columns > kFewColumns) {
        const int64_t all = (int64_t)a.rows * group;
        /* 256 rows a workgroup load each key and value for the most rows, if that leaves every CU one. If not, 128
         * rows (two groups of waves over the tokens) for contexts up to 8192 tokens, where partial sums cost more
         * than they give: 16 branches of 256 rows over 1568 tokens take 73 us so and 87 us as 256 rows split in two;
         * 512 rows x 8 over 8192 tokens 276 us and 271 us, over 32768 (8 bits) 1160 us and 1035 us. */
        p.tile.columns = 256;
        while (p.tile.columns > 64 && columns <= p.tile.columns / 2) p.tile.columns /= 2;
        if (p.tile.columns == 256 && (all + 255) / 256 * a.kv_heads < cus && a.max_kv <= 8192) p.tile.columns = 128;
        /* A sequence has a ragged tile at most; of those counted one by one, only sequences of more than few_columns
         * have any. */
        const int64_t ragged = all / (p.few_columns + 1);
        p.tile.slots = (int)(all / p.tile.columns +
                             (a.sequences <= kAttnCounted && ragged < a.sequences ? ragged : a.sequences));
        split_of(p.tile, a, cus / ((all + p.tile.columns - 1) / p.tile.columns * a.kv_heads), 8);
    }
    const size_t row = (size_t)a.kv_heads * (dim + 2) * sizeof(float);
    if (p.few.splits > 1) p.few_bytes = ((size_t)a.sequences * p.few.splits * p.few_rows * row + 15) & ~(size_t)15;
    p.bytes = p.few_bytes;
    if (p.tile.splits > 1) p.bytes += (size_t)a.rows * group * p.tile.splits * row;
    return p;
}

}  // namespace

/* Joins the partial sums of a row: a wave for each (row, query head). How many
 * splits have any goes by unit: a sequence's rows in the few-row kernel, `columns`
 * of them in the tile kernel. Latency, mostly: sequence, then maxima and sums together
 * (one context of 513 tokens in 5 splits: 4 us; 32768 rows in two: 22 us for
 * 50 MB, 28 when the sums of a row tile lay together and not those of a row). */
template <typename T, int D>
__global__ __launch_bounds__(256) void sera_attn_join_kernel(kv_args a, attn_args t, attn_plan few, attn_plan tile,
                                                             size_t tile_sums) {
    constexpr int E = D / 64;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int i;
    const kv_seq s = kv_find_sequence(a, (int)blockIdx.x, 1, 0, &i);
    if (s.b < 0 || s.bad || i >= s.n) return;
    const int first = s.len - s.n, rows = s.n * t.group;
    const bool is_few = rows <= t.few_columns;
    const int splits = is_few ? few.splits : tile.splits, chunk = is_few ? few.chunk : tile.chunk;
    if (splits < 2) return;
    const int unit_rows = is_few ? t.few_rows : tile.columns;
    for (int h = (int)blockIdx.y * 4 + wave; h < t.heads; h += (int)gridDim.y * 4) {
        const int head = h / t.group, row = i * t.group + h % t.group, unit = row / unit_rows;
        const int last = min((unit + 1) * unit_rows, rows) - 1;
        const attn_range range = attn_range_of(t, max(first + unit * unit_rows / t.group, 0),
                                               first + last / t.group + 1, kAttnShift);
        const int used = max((range.count + chunk - 1) / chunk, 1);
        /* sums, and maxima with their weights' sums, of this row's first split, and how far apart those of two splits
         * are: in floats, of which the workspace has some 10^7 */
        const int place = is_few ? s.b * a.kv_heads + head : (s.row0 + i) * t.heads + h;
        const int step = is_few ? (int)attn_partial_floats(unit_rows, D) : D, ml_step = is_few ? step : 2;
        const int sums = place * splits * step + (is_few ? row * D : 0);
        const int ml_at = is_few ? sums - row * D + unit_rows * D + 2 * row
                                 : (a.rows * t.heads * D + 2 * place) * splits;
        const float *const base = t.workspace + (is_few ? 0 : tile_sums);
        const auto sum_of = [&](int split) {
            return *(const attn_vec<float, E> *)(base + (uint32_t)(sums + min(split, used - 1) * step + E * lane));
        };
        /* sums are loaded 16 splits at a time (2, if there are no more), the first together with the maxima that weigh
         * them */
        constexpr int BATCH = 16;
        attn_vec<float, E> x[BATCH];
        x[0] = sum_of(0);
        x[1] = sum_of(1);
        if (used > 2)
#pragma unroll
            for (int k = 2; k < BATCH; k++) x[k] = sum_of(k);
        float m = kAttnLowest, l = 0.0f;
        if (lane < used) {
            const attn_f2 ml = *(const attn_f2 *)(base + (uint32_t)(ml_at + lane * ml_step));
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
        for (int split = 0; split < used; split += BATCH) {
            if (split > 0)
#pragma unroll
                for (int k = 0; k < BATCH; k++) x[k] = sum_of(split + k);
#pragma unroll
            for (int k = 0; k < BATCH; k++) {
                const float w = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f), (split + k) & 63));
#pragma unroll
                for (int e = 0; e < E; e++) y[e] = split + k < used ? fmaf(x[k].v[e], w, y[e]) : y[e];
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
void join_t(int dim, const kv_args &a, const attn_args &t, const attn_plans &p, hipStream_t s) {
    const dim3 grid((unsigned)a.rows, (unsigned)((t.heads + 3) / 4));
    const size_t at = p.few_bytes / sizeof(float);
    if (dim == 64)
        hipLaunchKernelGGL((sera_attn_join_kernel<T, 64>), grid, dim3(256), 0, s, a, t, p.few, p.tile, at);
    else
        hipLaunchKernelGGL((sera_attn_join_kernel<T, 128>), grid, dim3(256), 0, s, a, t, p.few, p.tile, at);
}

/* A window's rows see fewer tiles than a whole context has. */
void shorten(attn_plan &p, const kv_args &a, const attn_args &t) {
    if (!p.columns || t.window == 0) return;
    const int64_t tile = 1 << kAttnShift, sinks = t.sinks < a.max_kv ? t.sinks : a.max_kv;
    const int64_t tiles = (sinks + tile - 1) / tile + ((int64_t)t.window + a.max_new + tile - 2) / tile + 1;
    const int64_t chunk = (tiles + p.splits - 1) / p.splits;
    if (chunk < p.chunk) p.chunk = (int)chunk;
}

}  // namespace

size_t sera_attn_workspace(const kv_args &a, int dim, int heads, int cus) {
    return plan_of(a, dim, heads, cus).bytes;
}

/* Arguments are checked by the caller (sera_attn_runtime.hip). */
hipError_t sera_launch_attn(uint32_t cache_type, uint32_t type, int dim, const kv_args &a, const attn_args &args,
                            hipStream_t s) {
    attn_plans p = plan_of(a, dim, args.heads, args.cus);
    attn_args t = args;
    t.few_columns = p.few_columns;
    t.few_rows = p.few_rows;
    shorten(p.few, a, t);
    shorten(p.tile, a, t);
    /* Whole contexts, a CU to each workgroup: eight waves of an 8-bit cache, whose conversions they share (24 contexts of
     * 1050-2100 tokens: 25.5 us, 28.7 with four). From fp16 the four are as fast (40 and 40), and split contexts
     * have few tiles for more (one of 513 tokens: 11 us with four, 14 with eight). */
    p.few.waves = cache_type == SERA_KV_Q8 && p.few.columns <= 16 && p.few.splits == 1 &&
                  (int64_t)a.sequences * a.kv_heads <= args.cus ? 8 : 4;
    hipError_t e = hipSuccess;
    if (p.tile.columns) {
        attn_args u = t;
        u.workspace += p.few_bytes / sizeof(float);
        e = sera_launch_attn_tile(cache_type, type, dim, a, u, p.tile, s);
    }
    if (e == hipSuccess && p.few.columns) e = sera_launch_attn_few(cache_type, type, dim, a, t, p.few, s);
    if (e != hipSuccess || !p.bytes) return e;
    if (type == SERA_TYPE_F32) join_t<float>(dim, a, t, p, s);
    else if (type == SERA_TYPE_F16) join_t<_Float16>(dim, a, t, p, s);
    else join_t<__bf16>(dim, a, t, p, s);
    return hipGetLastError();
}
