/*
 * attn_tile.hip - attention of many new rows per sequence (prefill, chunks of
 * a prompt, branches of many tokens).
 *
 *   S^T = K Q^T          A = K (tokens), B = Q^T (columns: rows of q)
 *   O^T = V^T P^T        A = V^T (channels), B = P^T (tokens x columns)
 *
 * on 32x32x16 fp16 MFMAs. A workgroup has 32 * RG rows of one sequence and kv
 * head (tokens x heads of the group, so all heads share what is loaded); its
 * waves are RG groups of rows times KG groups of tokens. K and V pass through LDS
 * as fp16 in 32-token tiles, two steps of buffers deep, already in the order that
 * the A operands are read in: K rows with the token bits 2 and 3 exchanged, so
 * that the scores a lane gets are its B operand of the second product, 16-byte
 * units of a row exchanged by the row (xor) against bank conflicts; V in units of
 * (16 tokens, 32 channels), read as one run. A lane's 16 scores belong to one
 * row, so the softmax is in the lane but for one step between the halves of a wave.
 */
#include "attn_device.h"
#include "sera_launch.h"

namespace {

constexpr int kListed = 512;    /* tiles whose page ids are in LDS at a time */

template <int D, int RG, int KG>
struct tile_shape {
    static constexpr int NW = RG * KG, NT = 64 * NW;
    static constexpr int NSUB = KG > 2 ? KG : 2;     /* 32-token tiles of a step */
    static constexpr int UNITS = 32 * D / 8;         /* 16-byte fp16 units of K (and V) in a tile */
    static constexpr int KC = D / 16, NC = D / 32;
    static constexpr int XOR = D / 8 < 16 ? D / 8 - 1 : 15;
};

__device__ __forceinline__ int swap_token(int r) { return (r & ~12) | ((r & 4) << 1) | ((r & 8) >> 1); }

template <int D, int RG, int KG>
struct tile_lds {
    using S = tile_shape<D, RG, KG>;
    attn_u4 k[2][S::NSUB][S::UNITS], v[2][S::NSUB][S::UNITS];
    float scale[2][S::NSUB][3][32];          /* K scale, V scale, log2 of the V scale */
    int ids[2 * kListed];
};

}  // namespace

template <int TYPE, typename T, int D, int RG, int KG>
__global__ __launch_bounds__(64 * RG * KG, 2) void sera_attn_tile_kernel(kv_args a, attn_args t, int slots, int splits,
                                                                         int chunk) {
    using S = tile_shape<D, RG, KG>;
    constexpr bool Q8 = TYPE == (int)SERA_KV_Q8, TWO = sizeof(T) == 4;
    constexpr int NT = S::NT, NSUB = S::NSUB, UNITS = S::UNITS, KC = S::KC, NC = S::NC, BR = 32 * RG;
    constexpr int PIECES = NSUB * UNITS * 2 / (Q8 ? 2 : 1) / NT;     /* 16-byte loads of a thread and step */
    constexpr int ES = Q8 ? 1 : 2;
    __shared__ tile_lds<D, RG, KG> lds;

    int slot = (int)(blockIdx.z * gridDim.y + blockIdx.y);
    if (slot >= slots) return;
    slot = slots - 1 - slot;                          /* the last rows see most: they start first */
    const int head = (int)blockIdx.x % a.kv_heads, split = (int)blockIdx.x / a.kv_heads;
    int unit;
    const int b = kv_find(a, slot, BR, 1, &unit, t.group);
    if (b < 0) return;
    const kv_seq s = kv_sequence(a, b);
    const int rows = s.n * t.group, r0 = unit * BR;
    if (r0 >= rows) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 31, half = lane >> 5;
    const int64_t q0 = (int64_t)head * t.group * D;
    if (s.bad) {
        if (split == 0)
            for (int x = tid; x < min(rows - r0, BR) * D; x += NT) {
                const int r = r0 + x / D, i = r / t.group;
                ((T *)t.out)[(s.row0 + i) * t.out_stride + q0 + (r - i * t.group) * D + x % D] =
                    kv_from_f32<T>(__builtin_nanf(""));
            }
        return;
    }
    const int first = s.len - s.n;                    /* position of row 0 */
    const int end = first + min(r0 + BR - 1, rows - 1) / t.group + 1;
    const attn_range range = attn_range_of(t, max(first + r0 / t.group, 0), end, 5);
    const int v0 = split * chunk, v1 = min(v0 + chunk, range.count);
    if (split > 0 && v0 >= range.count) return;

    /* This wave's rows, and where they end. */
    const int rg = wave % RG, kg = wave / RG;
    const int w0 = r0 + 32 * rg, row = min(w0 + col, rows - 1), at = row / t.group;
    const int pos = first + at;
    const int pw0 = first + min(w0, rows - 1) / t.group, pw1 = first + min(w0 + 31, rows - 1) / t.group;
    const bool idle = w0 >= rows;

    attn_h8 qh[KC], ql[TWO ? KC : 1];
    float c;
    {
        const T *q = (const T *)t.q + (s.row0 + at) * t.q_stride + q0 + (row - at * t.group) * D + 8 * half;
        float top = 0.0f;
        /* twice over the row (the second time from cache): its size first, then the fragments */
#pragma unroll
        for (int k = 0; k < KC; k++) {
            float x[8];
            attn_load8(q + 16 * k, x);
#pragma unroll
            for (int j = 0; j < 8; j++) top = fmaxf(top, fabsf(x[j]));
        }
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const int e = attn_q_exponent(top);
        const float up = ldexpf(t.scale_log2 < 0.0f ? -1.0f : 1.0f, e);
        c = ldexpf(fabsf(t.scale_log2), -e);
#pragma unroll
        for (int k = 0; k < KC; k++) {
            float x[8];
            attn_load8(q + 16 * k, x);
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] *= up;
            attn_h8 lo;
            attn_split<TWO>(x, qh[k], lo);
            if (TWO) ql[k] = lo;
        }
    }

    float m = kAttnLowest, l = 0.0f;
    attn_f16 o[NC];
#pragma unroll
    for (int n = 0; n < NC; n++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[n][i] = 0.0f;

    const int mask = (1 << a.page_shift) - 1;
    const size_t kv_bytes = ((size_t)D << a.page_shift) * ES;
    const uint8_t *base = a.data + (size_t)head * a.head_bytes;
    attn_u4 raw[PIECES];
    float raw_scale = 0.0f;
    int g = v0;

    /* Piece e of this thread of the step at tile v: which tile, K or V, and its place. */
    auto stage_load = [&](int v, int stop) {
        constexpr int PER = UNITS * 2 / (Q8 ? 2 : 1);       /* pieces of a tile, K then V */
#pragma unroll
        for (int e = 0; e < PIECES; e++) {
            const int x = e * NT + tid, sub = x / PER, y = x % PER;
            if (v + sub >= stop) continue;
            const int j = range.tile(v + sub) * 32;
            const bool is_k = y < PER / 2;
            const int z = is_k ? y : y - PER / 2;
            int token, off;
            if (is_k) {
                constexpr int ROW = D * ES / 16;
                const int r = z / ROW;
                token = swap_token(r);
                off = (Q8 ? z % ROW : (z % ROW) ^ (r & S::XOR)) * 16;
            } else if (Q8) {
                token = z / D * 16;
                off = z % D * 16;
            } else {
                token = z / (2 * D) * 16;
                off = (z % (2 * D) / 64 * 32 + z % 32) * 32 + z / 32 % 2 * 16;
            }
            const int id = max(lds.ids[2 * (v - g + sub) + (token >> 4)], 0);
            raw[e] = *(const attn_u4 *)(base + (size_t)id * a.page_bytes + (is_k ? 0 : kv_bytes) +
                                        (size_t)((j + token) & mask) * (D * ES) + off);
        }
        if (Q8 && tid < NSUB * 64 && v + (tid >> 6) < stop) {
            const int j = range.tile(v + (tid >> 6)) * 32, token = tid & 31;
            const int id = max(lds.ids[2 * (v - g + (tid >> 6)) + (token >> 4)], 0);
            raw_scale = ((const float *)(base + (size_t)id * a.page_bytes + 2 * kv_bytes))
                [((size_t)(tid >> 5 & 1) << a.page_shift) + ((j + token) & mask)];
        }
    };
    auto stage_store = [&](int v, int stop, int buf) {
        constexpr int PER = UNITS * 2 / (Q8 ? 2 : 1);
#pragma unroll
        for (int e = 0; e < PIECES; e++) {
            const int x = e * NT + tid, sub = x / PER, y = x % PER;
            if (v + sub >= stop) continue;
            const bool is_k = y < PER / 2;
            const int z = is_k ? y : y - PER / 2;
            attn_u4 *to = is_k ? lds.k[buf][sub] : lds.v[buf][sub];
            if (!Q8) {
                to[z] = raw[e];
            } else {
                const attn_u4 x0 = __builtin_bit_cast(attn_u4, attn_codes(raw[e][0], raw[e][1]));
                const attn_u4 x1 = __builtin_bit_cast(attn_u4, attn_codes(raw[e][2], raw[e][3]));
                int u0, u1;
                if (is_k) {
                    constexpr int ROW = D / 16;
                    const int r = z / ROW, u = 2 * (z % ROW);
                    u0 = r * (D / 8) + (u ^ (r & S::XOR));
                    u1 = r * (D / 8) + ((u + 1) ^ (r & S::XOR));
                } else {
                    u0 = z / D * (2 * D) + z % D / 32 * 64 + z % 32;
                    u1 = u0 + 32;
                }
                to[u0] = x0;
                to[u1] = x1;
            }
        }
        if (Q8 && tid < NSUB * 64 && v + (tid >> 6) < stop) {
            float (*to)[32] = lds.scale[buf][tid >> 6];
            to[tid >> 5 & 1][tid & 31] = raw_scale;
            if (tid & 32) to[2][tid & 31] = attn_log_scale(raw_scale);
        }
    };

    auto compute = [&](int v, int buf, int sub) {
        const int j = range.tile(v) * 32;
        if (idle || j > pw1 || (t.window > 0 && j + 31 <= pw0 - t.window && j >= t.sinks)) return;
        const bool seen = first >= 0 && attn_all_seen(t, j, 32, pw0, pw1);
        const int id0 = lds.ids[2 * (v - g)], id1 = lds.ids[2 * (v - g) + 1];
        attn_f16 x;
#pragma unroll
        for (int i = 0; i < 16; i++) x[i] = 0.0f;
#pragma unroll
        for (int k = 0; k < KC; k++) {
            const attn_h8 kf = __builtin_bit_cast(attn_h8,
                lds.k[buf][sub][col * (D / 8) + ((2 * k + half) ^ (col & S::XOR))]);
            x = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qh[k], x, 0, 0, 0);
            if (TWO) x = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, ql[TWO ? k : 0], x, 0, 0, 0);
        }
        /* Score i belongs to token 16 * (i / 8) + 8 * half + i % 8. */
        attn_f4 vs[Q8 ? 4 : 1];
        float top = kAttnLowest;
        if (Q8) {
            const float (*sc)[32] = lds.scale[buf][sub];
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const attn_f4 ks = *(const attn_f4 *)&sc[0][16 * (i / 8) + 8 * half + i % 8];
                vs[i / 4] = *(const attn_f4 *)&sc[1][16 * (i / 8) + 8 * half + i % 8];
#pragma unroll
                for (int y = 0; y < 4; y++) x[i + y] *= ks[y] * c;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 16; i++) x[i] *= c;
        }
        if ((id0 | id1) < 0)
#pragma unroll
            for (int i = 0; i < 16; i++) x[i] = (i < 8 ? id0 : id1) < 0 ? __builtin_nanf("") : x[i];
        if (!seen)
#pragma unroll
            for (int i = 0; i < 16; i++)
                x[i] = attn_sees(t, pos, j + 16 * (i / 8) + 8 * half + i % 8) ? x[i] : -INFINITY;
        if (Q8) {
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const attn_f4 lv = *(const attn_f4 *)&lds.scale[buf][sub][2][16 * (i / 8) + 8 * half + i % 8];
#pragma unroll
                for (int y = 0; y < 4; y++) top = fmaxf(top, x[i + y] + lv[y]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 16; i++) top = fmaxf(top, x[i]);
        }
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        if (__ballot(top > m + kAttnLag)) {
            const float f = attn_exp2(m - fmaxf(top, m));
            m = fmaxf(top, m);
            l *= f;
#pragma unroll
            for (int n = 0; n < NC; n++) o[n] *= f;
        }
        const float shift = m - kAttnBias;
        attn_h8 ph[2], pl[2];
#pragma unroll
        for (int k = 0; k < 2; k++) {
            float w[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                w[i] = attn_exp2(x[8 * k + i] - shift);
                l += w[i];
                if (Q8) {
                    w[i] *= vs[Q8 ? 2 * k + i / 4 : 0][i % 4];
                    if (!seen) w[i] = attn_sees(t, pos, j + 16 * k + 8 * half + i) ? w[i] : 0.0f;
                }
            }
            attn_split<TWO>(w, ph[k], pl[k]);
        }
#pragma unroll
        for (int n = 0; n < NC; n++)
#pragma unroll
            for (int k = 0; k < 2; k++) {
                attn_h8 vf = __builtin_bit_cast(attn_h8, lds.v[buf][sub][k * 2 * D + n * 64 + lane]);
                if (!Q8 && !seen) {
                    /* fp16 values that are not finite: rows that see them get NaN in their channels, others nothing */
                    attn_h8 odd;
                    if (__ballot(attn_take_odd(vf, odd))) {
                        attn_h8 sees;
#pragma unroll
                        for (int i = 0; i < 8; i++)
                            sees[i] = attn_sees(t, pos, j + 16 * k + 8 * half + i) ? (_Float16)1.0f : (_Float16)0.0f;
                        attn_f16 hit;
#pragma unroll
                        for (int i = 0; i < 16; i++) hit[i] = 0.0f;
                        hit = __builtin_amdgcn_mfma_f32_32x32x16_f16(odd, sees, hit, 0, 0, 0);
#pragma unroll
                        for (int i = 0; i < 16; i++) o[n][i] = hit[i] > 0.0f ? __builtin_nanf("") : o[n][i];
                    }
                }
                o[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, ph[k], o[n], 0, 0, 0);
                if (TWO) o[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, pl[k], o[n], 0, 0, 0);
            }
    };

    for (; g < v1; g += kListed) {
        const int stop = min(v1, g + kListed);
        __syncthreads();
        for (int e = tid; e < 2 * (stop - g); e += NT)
            lds.ids[e] = attn_page(a, b, range.tile(g + (e >> 1)) * 32 + 16 * (e & 1), s.len);
        __syncthreads();
        stage_load(g, stop);
        stage_store(g, stop, 0);
        int buf = 0;
        for (int v = g; v < stop; v += NSUB) {
            __syncthreads();
            if (v + NSUB < stop) stage_load(v + NSUB, stop);
#pragma unroll
            for (int sub = 0; sub < NSUB; sub += KG)
                if (v + sub + kg < stop) compute(v + sub + kg, buf, sub + kg);
            if (v + NSUB < stop) stage_store(v + NSUB, stop, buf ^ 1);
            buf ^= 1;
        }
    }

    l += __shfl_xor(l, 32, 64);
    /* Join the token groups: the upper half of them hands its sums over, lane by lane. */
#pragma unroll
    for (int h = KG / 2; h >= 1; h >>= 1) {
        attn_f4 *box = (attn_f4 *)lds.k + ((size_t)rg + RG * (kg % h)) * (64 * NC * 4);
        float *mlbox = (float *)lds.ids + 128 * (rg + RG * (kg % h));
        static_assert(sizeof(attn_f4) * RG * (KG / 2) * 64 * NC * 4 <= sizeof(lds.k) + sizeof(lds.v), "join space");
        static_assert(sizeof(float) * RG * (KG / 2) * 128 <= sizeof(lds.ids), "join space");
        __syncthreads();
        if (kg >= h && kg < 2 * h) {
#pragma unroll
            for (int n = 0; n < NC; n++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    box[(n * 4 + i) * 64 + lane] = attn_f4{o[n][4 * i], o[n][4 * i + 1], o[n][4 * i + 2], o[n][4 * i + 3]};
            mlbox[lane] = m;
            mlbox[64 + lane] = l;
        }
        __syncthreads();
        if (kg < h) {
            const float m2 = mlbox[lane], top = fmaxf(m, m2), f = attn_exp2(m - top), f2 = attn_exp2(m2 - top);
            l = l * f + mlbox[64 + lane] * f2;
            m = top;
#pragma unroll
            for (int n = 0; n < NC; n++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const attn_f4 y = box[(n * 4 + i) * 64 + lane];
#pragma unroll
                    for (int z = 0; z < 4; z++) o[n][4 * i + z] = o[n][4 * i + z] * f + y[z] * f2;
                }
        }
    }
    if (kg > 0 || w0 + col >= rows) return;
    if (splits > 1) {
        float *part = t.workspace + (((size_t)slot * a.kv_heads + head) * splits + split) * attn_partial_floats(BR, D);
        const int r = 32 * rg + col;
#pragma unroll
        for (int n = 0; n < NC; n++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                *(attn_f4 *)(part + (size_t)r * D + 32 * n + 8 * i + 4 * half) =
                    attn_f4{o[n][4 * i], o[n][4 * i + 1], o[n][4 * i + 2], o[n][4 * i + 3]};
        if (half == 0) {
            part[(size_t)BR * D + 2 * r] = m;
            part[(size_t)BR * D + 2 * r + 1] = l;
        }
        return;
    }
    T *out = (T *)t.out + (s.row0 + at) * t.out_stride + q0 + (row - at * t.group) * D + 4 * half;
#pragma unroll
    for (int n = 0; n < NC; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float y[4];
#pragma unroll
            for (int z = 0; z < 4; z++) y[z] = pos < 0 ? 0.0f : o[n][4 * i + z] / l;
            attn_store4(out + 32 * n + 8 * i, y);
        }
}

namespace {

template <int TYPE, typename T, int D, int RG, int KG>
void tile_go(const kv_args &a, const attn_args &t, const attn_plan &p, hipStream_t s) {
    const int y = p.slots < 32768 ? p.slots : 32768;
    hipLaunchKernelGGL((sera_attn_tile_kernel<TYPE, T, D, RG, KG>),
                       dim3((unsigned)(a.kv_heads * p.splits), (unsigned)y, (unsigned)((p.slots + y - 1) / y)),
                       dim3(64 * RG * KG), 0, s, a, t, p.slots, p.splits, p.chunk);
}

template <int TYPE, typename T, int D>
void tile_rg(const kv_args &a, const attn_args &t, const attn_plan &p, hipStream_t s) {
    if (p.columns == 256) tile_go<TYPE, T, D, 8, 1>(a, t, p, s);
    else if (p.columns == 128) tile_go<TYPE, T, D, 4, 2>(a, t, p, s);
    else tile_go<TYPE, T, D, 2, 4>(a, t, p, s);
}

template <int TYPE, typename T>
void tile_d(int dim, const kv_args &a, const attn_args &t, const attn_plan &p, hipStream_t s) {
    dim == 64 ? tile_rg<TYPE, T, 64>(a, t, p, s) : tile_rg<TYPE, T, 128>(a, t, p, s);
}

template <int TYPE>
void tile_t(uint32_t type, int dim, const kv_args &a, const attn_args &t, const attn_plan &p, hipStream_t s) {
    if (type == SERA_TYPE_F32) tile_d<TYPE, float>(dim, a, t, p, s);
    else if (type == SERA_TYPE_F16) tile_d<TYPE, _Float16>(dim, a, t, p, s);
    else tile_d<TYPE, __bf16>(dim, a, t, p, s);
}

}  // namespace

hipError_t sera_launch_attn_tile(uint32_t cache_type, uint32_t type, int dim, const kv_args &a, const attn_args &t,
                                 const attn_plan &p, hipStream_t s) {
    if (cache_type == SERA_KV_F16) tile_t<(int)SERA_KV_F16>(type, dim, a, t, p, s);
    else tile_t<(int)SERA_KV_Q8>(type, dim, a, t, p, s);
    return hipGetLastError();
}
