/*
 * attn_few.hip - attention of a few new rows per sequence (decode): the keys
 * and values of a sequence are read once, for the rows of all query heads
 * that share them.
 *
 *   S^T = K Q^T          A = K (tokens), B = Q^T (columns: rows of q)
 *   O^T = V^T P^T        A = V^T (channels), B = P^T (tokens x columns)
 *
 * on 16x16x32 fp16 MFMAs, both products with the cache as A operand, so it goes
 * from memory to the matrix cores in the registers it is loaded into. A
 * lane of quarter t = lane / 16 gets the scores of the tokens 4t..4t+3 of a
 * 16-token A operand in its column; which token each A row is, is free, and
 * chosen so that the scores a lane has are the ones it needs as B operand of the second
 * product: nothing moves between lanes but the maximum (two steps) and, at the end,
 * the sum of the weights.
 *
 * Up to 8 rows of fp32 (PAIR) have both parts of their split in one operand, the high ones in columns 0..7, the low
 * ones in 8..15, whose products are added: half of the MFMAs and of the registers for them.
 *
 * A workgroup has the rows of one sequence and kv head (up to 16 * CT
 * columns) and a range of tiles; its waves take tiles in turn, each with a
 * running maximum of its own, and join through LDS at the end. Long contexts are
 * split over workgroups, joined by sera_attn_join_kernel.
 *
 * Bound by memory once contexts are long: 64 of 8192 tokens (2.15 GB of fp16) in
 * 352 us, 6.1 TB/s (368 us back to back in a graph). A call costs about 9 us (fp16; 10 us 8 bits) beyond the bytes
 * at that rate: launch, two rounds of dependent loads (sequence and pages; data),
 * the last tile's products and the joins. K's and V's registers are loaded again
 * as soon as a tile's products have taken them, 16 KB a wave on the way (8 KB of
 * codes).
 */
#include "attn_device.h"
#include "sera_launch.h"

namespace {

constexpr int kMaxTiles = 512;    /* whose page ids are in LDS at a time */

/* Tile geometry: 32 tokens. A lane loads 16-byte pieces of K rows (8 fp16
 * channels, or 16 codes, which feed two MFMAs), and of V 8 tokens of a
 * channel (16 bytes of fp16, 8 of codes). */
template <int TYPE, int D>
struct few_shape {
    static constexpr bool Q8 = TYPE == (int)SERA_KV_Q8;
    static constexpr int TT = 32, SHIFT = 5;
    static constexpr int QT = TT / 4;             /* tokens of a lane quarter, consecutive */
    static constexpr int NS = TT / 16;            /* 16-token A operands */
    static constexpr int KC = D / 32;             /* MFMA steps over the channels */
    static constexpr int KP = Q8 ? KC / 2 : KC;   /* 16-byte pieces of a K row per lane */
    static constexpr int NC = D / 16;             /* channel blocks */
};

template <int TYPE>
struct few_piece { typedef attn_u4 v; };
template <>
struct few_piece<(int)SERA_KV_Q8> { typedef attn_u2 v; };

}  // namespace

template <int TYPE, typename T, int D, int CT, int NW, int OCC, bool PAIR>
__global__ __launch_bounds__(64 * NW, OCC) void sera_attn_few_kernel(kv_args a, attn_args t, int splits, int chunk) {
    using F = few_shape<TYPE, D>;
    constexpr bool Q8 = F::Q8, TWO = sizeof(T) == 4 && !PAIR;      /* a second fragment for the low parts */
    constexpr int TT = F::TT, QT = F::QT, NS = F::NS, KC = F::KC, KP = F::KP, NC = F::NC;
    constexpr int RS = D + 4;                     /* row stride in LDS: rows start 4 banks apart */
    __shared__ int ids[kMaxTiles * (TT / 16)];
    __shared__ float red[NW][16][RS];
    __shared__ float ml[NW][2][16 * CT];

    const int b = (int)(blockIdx.z * gridDim.y + blockIdx.y);
    if (b >= a.sequences) return;
    const int head = (int)blockIdx.x % a.kv_heads, split = (int)blockIdx.x / a.kv_heads;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, quarter = lane >> 4, v0 = split * chunk;
    /* Without a window a split's first table entries are known before the sequence is: their load goes along with the
     * sequence's (max_kv bounds the table, whatever the length). */
    const int64_t early = (int64_t)v0 * TT + 16 * tid;
    int early_id = 0;
    if (t.window == 0 && early < a.max_kv) early_id = a.table[(size_t)b * a.table_stride + (early >> a.page_shift)];
    const kv_seq s = kv_sequence(a, b);
    if (s.n == 0 || s.n * t.group > t.few_columns) return;
    const int64_t q0 = (int64_t)head * t.group * D;
    if (s.bad) {
        if (split == 0)
            for (int64_t x = tid; x < (int64_t)s.n * t.group * D; x += 64 * NW)
                ((T *)t.out)[(s.row0 + x / (t.group * D)) * t.out_stride + q0 + x % (t.group * D)] =
                    kv_from_f32<T>(__builtin_nanf(""));
        return;
    }
    const int pn = s.len - 1, p0 = max(s.len - s.n, 0), rows = s.n * t.group;
    const attn_range range = attn_range_of(t, p0, s.len, F::SHIFT);
    const int v1 = min(v0 + chunk, range.count);
    if (split > 0 && v0 >= range.count) return;

    /* Page ids of tiles g .. g + kMaxTiles, and from there the wave's tiles. */
    auto list_pages = [&](int g) {
        for (int e = tid; e < min(v1 - g, kMaxTiles) * (TT / 16); e += 64 * NW) {
            const int at = range.tile(g + e / (TT / 16)) * TT + e % (TT / 16) * 16;
            if (t.window == 0 && g == v0 && e == tid)
                ids[e] = at >= s.len ? 0 : early_id < 0 || early_id >= a.pages ? -1 : early_id;
            else
                ids[e] = attn_page(a, b, at, s.len);
        }
    };
    list_pages(v0);

    /* Query fragments: lane (column, quarter) has 8 channels of each MFMA step, in the order of
     * the K pieces. */
    attn_h8 qh[CT][KC], ql[CT][TWO ? KC : 1];
    float c[CT];
    int pos[CT];
    const float sign = t.scale_log2 < 0.0f ? -1.0f : 1.0f;
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
        const int r = min(ct * 16 + (PAIR ? col & 7 : col), rows - 1), i = r / t.group;
        pos[ct] = s.len - s.n + i;
        const T *q = (const T *)t.q + (s.row0 + i) * t.q_stride + q0 + (r - i * t.group) * D;
        float x[KC][8], top = 0.0f;
#pragma unroll
        for (int k = 0; k < KC; k++) {
            attn_load8(q + (Q8 ? 64 * (k >> 1) + 16 * quarter + 8 * (k & 1) : 32 * k + 8 * quarter), x[k]);
#pragma unroll
            for (int j = 0; j < 8; j++) top = fmaxf(top, fabsf(x[k][j]));
        }
        top = fmaxf(top, xor_partner<16>(top));
        top = fmaxf(top, xor_partner<32>(top));
        const int e = attn_q_exponent(top);
        const float up = ldexpf(sign, e);
        c[ct] = ldexpf(fabsf(t.scale_log2), -e);
#pragma unroll
        for (int k = 0; k < KC; k++) {
#pragma unroll
            for (int j = 0; j < 8; j++) x[k][j] *= up;
            attn_h8 lo;
            attn_split<TWO || PAIR>(x[k], qh[ct][k], lo);
            if (TWO) ql[ct][k] = lo;
            if (PAIR) qh[ct][k] = col < 8 ? qh[ct][k] : lo;
        }
    }

    float m[CT], l[CT];
    attn_f4 o[CT][NC];
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
        m[ct] = kAttnLowest;
        l[ct] = 0.0f;
#pragma unroll
        for (int k = 0; k < NC; k++) o[ct][k] = attn_f4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    __syncthreads();

    const int mask = (1 << a.page_shift) - 1;
    const size_t kv_bytes = ((size_t)D << a.page_shift) * (Q8 ? 1 : 2);      /* K's (and V's) part of a head's run */
    const uint8_t *base = a.data + (size_t)head * a.head_bytes;
    /* Tokens of this lane: A row `col` of operand u is token QT * (col / 4) + 4 u + col % 4; its scores are
     * the tokens QT * quarter + 4 u + i. V pieces are those same tokens of one channel. */
    const int k_token = QT * (col >> 2) + (col & 3), v_token = QT * quarter;
    attn_u4 kr[NS][KP];
    typename few_piece<TYPE>::v vr[NC];
    attn_f4 ks[Q8 ? NS : 1], vs[Q8 ? NS : 1];
    int v_id = 0;

    /* The pieces of a tile. A lost page reads page 0 in its place (in the pool; its scores become NaN). */
    int g = v0;
    bool odd = false;       /* this lane took values that are not finite out of a tile */
    auto load_k = [&](int v) {
        const int j = range.tile(v) * TT, *id = ids + (v - g) * (TT / 16);
        const uint8_t *run = base + (size_t)max(id[k_token >> 4], 0) * a.page_bytes;
        const uint8_t *p = run + (size_t)((j + k_token) & mask) * (D * (Q8 ? 1 : 2)) + 16 * quarter;
#pragma unroll
        for (int u = 0; u < NS; u++)
#pragma unroll
            for (int k = 0; k < KP; k++) kr[u][k] = *(const attn_u4 *)(p + 4 * u * D * (Q8 ? 1 : 2) + 64 * k);
        if (Q8) {
            const uint8_t *sr = base + (size_t)max(id[v_token >> 4], 0) * a.page_bytes + 2 * kv_bytes;
            const attn_f4 *sp = (const attn_f4 *)((const float *)sr + ((j + v_token) & mask));
#pragma unroll
            for (int u = 0; u < NS; u++) {
                ks[u] = sp[u];
                vs[u] = *(const attn_f4 *)((const float *)(sp + u) + ((size_t)1 << a.page_shift));
            }
        }
    };
    auto load_v = [&](int v) {
        const int j = range.tile(v) * TT;
        v_id = ids[(v - g) * (TT / 16) + (v_token >> 4)];
        const uint8_t *p = base + (size_t)max(v_id, 0) * a.page_bytes + kv_bytes +
                           (size_t)((j + v_token) & mask & ~15) * (D * (Q8 ? 1 : 2)) +
                           (16 * col + (v_token & 15)) * (Q8 ? 1 : 2);
#pragma unroll
        for (int k = 0; k < NC; k++) vr[k] = *(const typename few_piece<TYPE>::v *)(p + (Q8 ? 256 : 512) * k);
    };

    for (; g < v1; g += kMaxTiles) {
        const int end = min(v1, g + kMaxTiles);
        if (g > v0) {
            __syncthreads();
            list_pages(g);
            __syncthreads();
        }
        int v = g + wave;
        if (v < end) {
            load_k(v);
            load_v(v);
        }
        for (; v < end; v += NW) {
            const int j0 = range.tile(v) * TT + v_token;     /* this lane's first token */
            const bool seen = attn_all_seen(t, range.tile(v) * TT, TT, p0, pn) && s.n <= s.len;
            const bool lost = v_id < 0;
            attn_f4 acc[CT][NS];
    #pragma unroll
            for (int ct = 0; ct < CT; ct++)
    #pragma unroll
                for (int u = 0; u < NS; u++) acc[ct][u] = attn_f4{0.0f, 0.0f, 0.0f, 0.0f};
    #pragma unroll
            for (int u = 0; u < NS; u++)
    #pragma unroll
                for (int k = 0; k < KC; k++) {
                    const attn_h8 kf = Q8 ? attn_codes(kr[u][k / 2][2 * (k & 1)], kr[u][k / 2][2 * (k & 1) + 1])
                                          : __builtin_bit_cast(attn_h8, kr[u][k % KP]);
    #pragma unroll
                    for (int ct = 0; ct < CT; ct++) {
                        acc[ct][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qh[ct][k], acc[ct][u], 0, 0, 0);
                        if (TWO)
                            acc[ct][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, ql[ct][k], acc[ct][u], 0, 0, 0);
                    }
                }
            if (PAIR)
#pragma unroll
                for (int u = 0; u < NS; u++)
#pragma unroll
                    for (int i = 0; i < 4; i++) acc[0][u][i] += xor_partner<8>(acc[0][u][i]);
            attn_f4 vsn[Q8 ? NS : 1];
            float lv[Q8 ? NS : 1][4];
            if (Q8)
    #pragma unroll
                for (int u = 0; u < NS; u++) {
                    vsn[u] = vs[u];
    #pragma unroll
                    for (int i = 0; i < 4; i++) lv[u][i] = attn_log_scale(vs[u][i]);
    #pragma unroll
                    for (int ct = 0; ct < CT; ct++) acc[ct][u] *= ks[u];
                }
            if (v + NW < end) load_k(v + NW);

            attn_h8 ph[CT], pl[CT];
    #pragma unroll
            for (int ct = 0; ct < CT; ct++) {
                float x[4 * NS], top = kAttnLowest;
    #pragma unroll
                for (int u = 0; u < NS; u++)
    #pragma unroll
                    for (int i = 0; i < 4; i++) x[4 * u + i] = acc[ct][u][i] * c[ct];
                if (__ballot(lost))
    #pragma unroll
                    for (int u = 0; u < NS; u++)
    #pragma unroll
                        for (int i = 0; i < 4; i++) x[4 * u + i] = lost ? __builtin_nanf("") : x[4 * u + i];
                if (!seen)
    #pragma unroll
                    for (int u = 0; u < NS; u++)
    #pragma unroll
                        for (int i = 0; i < 4; i++)
                            x[4 * u + i] = attn_sees(t, pos[ct], j0 + 4 * u + i) ? x[4 * u + i] : -INFINITY;
    #pragma unroll
                for (int u = 0; u < NS; u++)
    #pragma unroll
                    for (int i = 0; i < 4; i++)
                        top = fmaxf(top, Q8 ? x[4 * u + i] + lv[u % (Q8 ? NS : 1)][i] : x[4 * u + i]);
                top = fmaxf(top, xor_partner<16>(top));
                top = fmaxf(top, xor_partner<32>(top));
                if (__ballot(top > m[ct] + kAttnLag)) {
                    const float f = attn_exp2(m[ct] - fmaxf(top, m[ct]));
                    m[ct] = fmaxf(top, m[ct]);
                    l[ct] *= f;
    #pragma unroll
                    for (int k = 0; k < NC; k++) o[ct][k] *= f;
                }
                const float shift = m[ct] - kAttnBias;
    #pragma unroll
                for (int u = 0; u < NS; u++)
    #pragma unroll
                    for (int i = 0; i < 4; i++) {
                        float w = attn_exp2(x[4 * u + i] - shift);
                        l[ct] += w;
                        if (Q8) {
                            w *= vsn[u % (Q8 ? NS : 1)][i];
                            if (!seen) w = attn_sees(t, pos[ct], j0 + 4 * u + i) ? w : 0.0f;
                        }
                        x[4 * u + i] = w;
                    }
                    attn_split<TWO || PAIR>(x, ph[ct], pl[ct]);
                if (PAIR) ph[ct] = col < 8 ? ph[ct] : pl[ct];
            }
#pragma unroll
            for (int n = 0; n < NC; n++) {
                attn_h8 vf;
                if constexpr (Q8) vf = attn_codes(vr[n][0], vr[n][1]);
                else vf = __builtin_bit_cast(attn_h8, vr[n]);
                if (!Q8 && !seen) {
                    attn_h8 bad;
                    odd |= attn_take_odd(vf, bad);
                }
#pragma unroll
                for (int ct = 0; ct < CT; ct++) {
                    o[ct][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, ph[ct], o[ct][n], 0, 0, 0);
                    if (TWO) o[ct][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pl[ct], o[ct][n], 0, 0, 0);
                }
            }
            if (v + NW < end) load_v(v + NW);
        }
        /* fp16 values that are not finite, in tiles that a row does not see whole, were taken out: a product would
         * carry them into rows that do not see them (0 * inf). The rows that do get NaN in their channels. */
        if (!Q8 && __ballot(odd)) {
            for (v = g + wave; v < end; v += NW) {
                const int j = range.tile(v) * TT;
                if (attn_all_seen(t, j, TT, p0, pn) && s.n <= s.len) continue;
                load_v(v);
#pragma unroll
                for (int ct = 0; ct < CT; ct++) {
                    attn_h8 sees;
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        sees[i] = attn_sees(t, pos[ct], j + v_token + i) ? (_Float16)1.0f : (_Float16)0.0f;
#pragma unroll
                    for (int n = 0; n < NC; n++) {
                        attn_h8 w, bad;
                        if constexpr (!Q8) w = __builtin_bit_cast(attn_h8, vr[n]);
                        attn_take_odd(w, bad);
                        attn_f4 hit = {0.0f, 0.0f, 0.0f, 0.0f};
                        hit = __builtin_amdgcn_mfma_f32_16x16x32_f16(bad, sees, hit, 0, 0, 0);
#pragma unroll
                        for (int i = 0; i < 4; i++) o[ct][n][i] = hit[i] > 0.0f ? __builtin_nanf("") : o[ct][n][i];
                        __builtin_amdgcn_sched_barrier(0);      /* one at a time: few registers */
                    }
                }
            }
            odd = false;
        }
    }

    if (PAIR)
#pragma unroll
        for (int n = 0; n < NC; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) o[0][n][i] += xor_partner<8>(o[0][n][i]);
    /* Join the waves: columns of 16 rows at a time. */
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
        l[ct] += xor_partner<16>(l[ct]);
        l[ct] += xor_partner<32>(l[ct]);
        if (quarter == 0) {
            ml[wave][0][ct * 16 + col] = m[ct];
            ml[wave][1][ct * 16 + col] = l[ct];
        }
    }
    __syncthreads();
    float *const part = t.workspace +
        (((size_t)b * a.kv_heads + head) * splits + split) * attn_partial_floats(t.few_rows, D);
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
        if (ct * 16 >= rows) break;
        float top = kAttnLowest;
#pragma unroll
        for (int w = 0; w < NW; w++) top = fmaxf(top, ml[w][0][ct * 16 + col]);
        const float f = attn_exp2(m[ct] - top);
        if (ct) __syncthreads();
#pragma unroll
        for (int n = 0; n < NC; n++) *(attn_f4 *)&red[wave][col][16 * n + 4 * quarter] = o[ct][n] * f;
        __syncthreads();
        for (int e = tid; e < 16 * (D / 4); e += 64 * NW) {
            const int r = e / (D / 4), d = 4 * (e % (D / 4)), rr = ct * 16 + r;
            if (rr >= rows) break;
            attn_f4 sum = *(const attn_f4 *)&red[0][r][d];
#pragma unroll
            for (int w = 1; w < NW; w++) sum += *(const attn_f4 *)&red[w][r][d];
            float mt = kAttnLowest, lt = 0.0f;
#pragma unroll
            for (int w = 0; w < NW; w++) mt = fmaxf(mt, ml[w][0][rr]);
#pragma unroll
            for (int w = 0; w < NW; w++) lt += ml[w][1][rr] * attn_exp2(ml[w][0][rr] - mt);
            if (splits > 1) {
                *(attn_f4 *)(part + (size_t)rr * D + d) = sum;
                if (d == 0) {
                    part[(size_t)t.few_rows * D + 2 * rr] = mt;
                    part[(size_t)t.few_rows * D + 2 * rr + 1] = lt;
                }
            } else {
                const int i = rr / t.group;
                float y[4];
#pragma unroll
                for (int x = 0; x < 4; x++) y[x] = s.len - s.n + i < 0 ? 0.0f : sum[x] / lt;
                attn_store4((T *)t.out + (s.row0 + i) * t.out_stride + q0 + (rr - i * t.group) * D + d, y);
            }
        }
    }
}

namespace {

template <int TYPE, typename T, int D, int CT, int NW, int OCC, bool PAIR>
void few_go(const kv_args &a, const attn_args &t, const attn_plan &p, hipStream_t s) {
    const int y = a.sequences < 32768 ? a.sequences : 32768;
    hipLaunchKernelGGL((sera_attn_few_kernel<TYPE, T, D, CT, NW, OCC, PAIR>),
                       dim3((unsigned)(a.kv_heads * p.splits), (unsigned)y, (unsigned)((a.sequences + y - 1) / y)),
                       dim3(64 * NW), 0, s, a, t, p.splits, p.chunk);
}

/* Waves per SIMD: as many as the registers (no spills) leave. */
template <int TYPE, typename T, int D>
void few_ct(const kv_args &a, const attn_args &t, const attn_plan &p, hipStream_t s) {
    constexpr bool Q8 = TYPE == (int)SERA_KV_Q8, F32 = sizeof(T) == 4;
    constexpr int PAIRED = Q8 ? 3 : D == 128 ? 2 : 4;
    constexpr int PLAIN = D == 128 ? Q8 && !F32 ? 3 : 2 : Q8 || F32 ? 3 : 4;
    if (p.columns == 32) return few_go<TYPE, T, D, 2, 4, F32 && D == 128 ? 1 : 2, false>(a, t, p, s);
    if constexpr (Q8) {
        if (p.waves == 8 && F32 && p.columns == 8) return few_go<TYPE, T, D, 1, 8, 2, F32>(a, t, p, s);
        if (p.waves == 8) return few_go<TYPE, T, D, 1, 8, 2, false>(a, t, p, s);
    }
    if (F32 && p.columns == 8) return few_go<TYPE, T, D, 1, 4, PAIRED, F32>(a, t, p, s);
    few_go<TYPE, T, D, 1, 4, PLAIN, false>(a, t, p, s);
}

template <int TYPE, typename T>
void few_d(int dim, const kv_args &a, const attn_args &t, const attn_plan &p, hipStream_t s) {
    dim == 64 ? few_ct<TYPE, T, 64>(a, t, p, s) : few_ct<TYPE, T, 128>(a, t, p, s);
}

template <int TYPE>
void few_t(uint32_t type, int dim, const kv_args &a, const attn_args &t, const attn_plan &p, hipStream_t s) {
    if (type == SERA_TYPE_F32) few_d<TYPE, float>(dim, a, t, p, s);
    else if (type == SERA_TYPE_F16) few_d<TYPE, _Float16>(dim, a, t, p, s);
    else few_d<TYPE, __bf16>(dim, a, t, p, s);
}

}  // namespace


hipError_t sera_launch_attn_few(uint32_t cache_type, uint32_t type, int dim, const kv_args &a, const attn_args &t,
                                const attn_plan &p, hipStream_t s) {
    if (cache_type == SERA_KV_F16) few_t<(int)SERA_KV_F16>(type, dim, a, t, p, s);
    else few_t<(int)SERA_KV_Q8>(type, dim, a, t, p, s);
    return hipGetLastError();
}
