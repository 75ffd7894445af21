/*
 * attn_weights.hip - the weight that every cached position gets from the rows of a call, after its attention:
 *
 *   w_j = sum over rows i, query heads of 2^(s'_ij - z_i) r_i,   2^z_i / r_i = sum_j 2^(s'_ij)
 *
 * with s' = scale * q . k * log2(e), as attention has them, and z and r left by its kernels (t.norms).
 *
 * Few rows: the kernel that streams the cache has the scores; it leaves them (4 bytes for each position and column),
 * and what is left to do is one pass over those.
 *
 * Many rows: the products again, S^T = K Q^T on 32x32x16 MFMAs, the keys of 512 positions in a workgroup's registers
 * (64 a wave, A operand) and the columns (rows of q times heads of the group) passing by in blocks of 32: loaded by
 * rows, scaled, split into fp16 terms and laid into LDS in the order of B fragments by all waves, a block ahead of
 * the products. A lane has one column of a block, so z is one number a lane, and its sums stay in the lane until the
 * end. Blocks of columns that see any of 512 positions are the units of work (positions alone are few: 32 workgroups
 * for a prompt of 2048 and 8 kv heads); every workgroup has an equal run of them, of fewer where a window hides
 * most, and the last kernel adds the runs' sums in their order.
 *
 * Many rows are bound by the matrix instructions, and beside them by the exponentials and the columns' way through
 * LDS: the weights of one half of a wave's positions are made under the products of the other, and of the two waves
 * of a SIMD one converts columns while the other multiplies. r goes into z there, rounded to fp32 (2^-24 |z| of a
 * weight, less than its score's own error: z is log2 of the sum of 2^s' but for a factor of 2, whatever the scales of
 * 8-bit values); as a factor of every weight it cost 5%. 1024 rows of 64 heads at the end
 * of 16384 positions (8 kv heads, 128 channels, fp16 cache): 435 us with 16-bit rows, 600 us with fp32 ones, whose
 * products are two (0.8 of the rate of a large library product); a prompt of 2048 fp32 rows: 110 us behind the
 * attention's 160 us. Few rows are bound by memory: 64 sequences of 8192 positions (8 kv heads, groups of 8, bf16
 * rows) leave 134 MB of scores in the 457 us in which the attention streams 2.1 GB of cache, and one pass over them
 * takes 33 us (4.1 TB/s).
 */
#include "attn_sums.h"
#include "sera_launch.h"

namespace {

constexpr int kWaves = 8, kWaveTokens = 64, kTokens = kWaves * kWaveTokens;  /* positions of a wave, a workgroup */

template <typename T, int D>
struct sum_shape {
    static constexpr bool TWO = sizeof(T) == 4;
    static constexpr int KC = D / 16, NB = kWaveTokens / 32;
    static constexpr int VEC = 16 / (int)sizeof(T);            /* elements of a 16-byte load */
    static constexpr int TPC = D / VEC < 16 ? D / VEC : 16;    /* threads to a column */
    static constexpr int LOADS = D / (TPC * VEC);              /* of a thread */
    static constexpr int UNITS = KC * 2 * 32;                  /* 16-byte units of a block's high (or low) terms */
};

typedef __attribute__((address_space(3))) attn_u4 sum_local_u4;
typedef __attribute__((address_space(3))) void sum_local;

/* Place of unit u = 2 kc + half of column `col`: (u, col), columns exchanged so that the units that a row's threads
 * write at once lie in different banks. */
__device__ __forceinline__ int sum_unit(int u, int col) { return u * 32 + (col ^ (((u & 3) << 1) | ((u >> 2) & 1))); }

/* Blocks of 32 columns, c0 .. c1-1, that see any of a tile's positions. */
struct sum_blocks {
    int c0, c1;
};
__device__ __forceinline__ sum_blocks sum_blocks_of(const attn_args &t, const kv_seq &s, int tile) {
    const int first = s.len - s.n, j = tile * kTokens;
    int64_t end = s.n;
    if (t.window > 0 && j >= t.sinks)                   /* rows from here on see nothing of it, nor do those in front */
        end = min(end, max((int64_t)j + kTokens - 1 + t.window - first, (int64_t)0));
    sum_blocks r;
    r.c0 = (int)((int64_t)max(j - first, 0) * t.group / 32);
    r.c1 = (int)((end * t.group + 31) / 32);
    return r;
}

}  // namespace

template <int TYPE, typename T, int D>
__global__ __launch_bounds__(64 * kWaves, 2) void sera_attn_columns_kernel(kv_args a, attn_args t, attn_sums p) {
    using S = sum_shape<T, D>;
    constexpr bool Q8 = TYPE == (int)SERA_KV_Q8, TWO = S::TWO;
    constexpr int ES = Q8 ? 1 : 2, KC = S::KC, NB = S::NB, UNITS = S::UNITS;
    constexpr int LOADS = S::LOADS, VEC = S::VEC, TPC = S::TPC;
    __shared__ attn_u4 box[2][TWO ? 2 : 1][UNITS];
    __shared__ float cz[2][2][32];                        /* each column's factor, and z */
    __shared__ attn_f4 key_scale[Q8 ? kTokens / 4 : 1];

    const int b = (int)(blockIdx.z * gridDim.y + blockIdx.y);
    if (b >= a.sequences) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int head = (int)blockIdx.x % a.kv_heads, group_index = (int)blockIdx.x / a.kv_heads;
    const kv_seq s = kv_sequence(a, b);
    const int rows = s.n * t.group;
    if (s.bad || rows <= t.few_columns) return;
    const int first = s.len - s.n, mask = (1 << a.page_shift) - 1, col = lane & 31, half = lane >> 5;

    /* This workgroup's units: the tile that the first one is in, by counting as many tiles as there are threads at a
     * time. */
    const int tiles = (s.len + kTokens - 1) / kTokens;
    const int64_t u0 = (int64_t)group_index * p.share;
    int tile = -1, c_first = 0;
    {
        __shared__ int64_t ends[kWaves];
        __shared__ int found[2];
        if (tid == 0) found[0] = -1;
        int64_t before = 0;
        for (int x = 0; x < tiles; x += 64 * kWaves) {
            int n = 0;
            sum_blocks r = {0, 0};
            if (x + tid < tiles) {
                r = sum_blocks_of(t, s, x + tid);
                n = max(r.c1 - r.c0, 0);
            }
            int64_t upto = n;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int64_t y = __shfl_up(upto, o, 64);
                upto += lane >= o ? y : 0;
            }
            if (lane == 63) ends[wave] = upto;
            __syncthreads();
            int64_t from = before;
            for (int w = 0; w < kWaves; w++) {
                from += w < wave ? ends[w] : 0;
                before += ends[w];
            }
            from += upto - n;
            if (u0 >= from && u0 < from + n) {
                found[0] = x + tid;
                found[1] = r.c0 + (int)(u0 - from);
            }
            __syncthreads();
            if (found[0] >= 0) break;
        }
        tile = __builtin_amdgcn_readfirstlane(found[0]);
        c_first = __builtin_amdgcn_readfirstlane(found[1]);
    }
    if (tiles == 0 || tile < 0) return;
    int left = p.share;
    const float sign = t.scale_log2 < 0.0f ? -1.0f : 1.0f;
    const int my_col = tid / TPC, sub = tid % TPC, step_i = 32 / t.group, step_g = 32 - step_i * t.group;
    const uint8_t *base = a.data + (size_t)head * a.head_bytes;
    for (; tile < tiles && left > 0; tile++, c_first = -1) {
        const int tile0 = tile * kTokens, j0 = tile0 + wave * kWaveTokens;
        const sum_blocks range = sum_blocks_of(t, s, tile);
        const int c0 = c_first < 0 ? range.c0 : c_first, c1 = min(range.c1, c0 + left);
        if (c0 >= c1) continue;
        left -= c1 - c0;

        /* This thread's column of the block that comes next, and its loads (32 columns may need fewer threads than
         * there are). */
        int at_r = 32 * c0 + my_col, at_i = at_r / t.group, at_g = at_r - at_i * t.group;
        attn_vec<T, VEC> in[2][LOADS];
        float2 z[2];
        bool there[2];                    /* not past the last column, which have no weight */
        const bool loads = 32 * TPC == 64 * kWaves || my_col < 32;
        const auto load = [&](int place) {
            if (!loads) return;
            there[place] = at_r < rows;
            const int i = there[place] ? at_i : s.n - 1, h = head * t.group + (there[place] ? at_g : t.group - 1);
            const T *q = (const T *)t.q + (s.row0 + i) * t.q_stride + (int64_t)h * D + VEC * sub;
#pragma unroll
            for (int k = 0; k < LOADS; k++) in[place][k] = *(const attn_vec<T, VEC> *)(q + TPC * VEC * k);
            z[place] = t.norms[(size_t)(s.row0 + i) * t.heads + h];
            at_r += 32;
            at_i += step_i;
            at_g += step_g;
            if (at_g >= t.group) {
                at_g -= t.group;
                at_i++;
            }
        };
        const auto put = [&](int place, int buf) {
            if (!loads) return;
            float x[LOADS][VEC], top = 0.0f;
#pragma unroll
            for (int k = 0; k < LOADS; k++)
#pragma unroll
                for (int e = 0; e < VEC; e++) {
                    x[k][e] = kv_to_f32(in[place][k].v[e]);
                    top = fmaxf(top, fabsf(x[k][e]));
                }
            top = fmaxf(top, xor_partner<1>(top));
            top = fmaxf(top, xor_partner<2>(top));
            top = fmaxf(top, xor_partner<4>(top));
            if (TPC == 16) top = fmaxf(top, xor_partner<8>(top));
            const int e2 = attn_q_exponent(top);
            const float up = ldexpf(sign, e2);
            if (sub == 0) {
                cz[buf][0][my_col] = ldexpf(fabsf(t.scale_log2), -e2);
                cz[buf][1][my_col] = there[place] ? z[place].x - __builtin_amdgcn_logf(z[place].y) : INFINITY;
            }
#pragma unroll
            for (int k = 0; k < LOADS; k++) {
                attn_vec<_Float16, VEC> hi, lo;
#pragma unroll
                for (int e = 0; e < VEC; e++) {            /* scaled and rounded in one mixed instruction each */
                    hi.v[e] = (_Float16)fmaf(x[k][e], up, 0.0f);
                    if (TWO) lo.v[e] = (_Float16)fmaf(x[k][e], up, -(float)hi.v[e]);
                }
                const int ch = TPC * VEC * k + VEC * sub;
                uint8_t *to = (uint8_t *)&box[buf][0][sum_unit(ch >> 3, my_col)] + (ch & 7) * 2;
                *(attn_vec<_Float16, VEC> *)to = hi;
                if (TWO) *(attn_vec<_Float16, VEC> *)(to + UNITS * 16) = lo;
            }
        };
        load(0);
        if (c0 + 1 < c1) load(1);

        /* Keys: row `col` of A operand n is position j0 + 32 n + col. */
        attn_h8 kf[NB][KC];
        uint32_t lost[NB];
#pragma unroll
        for (int n = 0; n < NB; n++) {
            const int j = j0 + 32 * n + col, id = attn_page(a, b, j & ~15, s.len);
            lost[n] = (uint32_t)__ballot(id < 0);
            const uint8_t *run = base + (size_t)max(id, 0) * a.page_bytes;
            const uint8_t *k = run + (size_t)(j & mask) * (D * ES) + 8 * half * ES;
#pragma unroll
            for (int kc = 0; kc < KC; kc++) {
                if constexpr (Q8) {
                    const attn_u2 w = *(const attn_u2 *)(k + 16 * kc);
                    kf[n][kc] = attn_codes(w[0], w[1]);
                } else {
                    kf[n][kc] = *(const attn_h8 *)(k + 32 * kc);
                }
            }
            if (Q8) {
                const float scale = ((const float *)(run + 2 * ((size_t)D << a.page_shift)))[j & mask];
                if (half == 0) ((float *)key_scale)[wave * kWaveTokens + 32 * n + col] = scale;
            }
        }

        /* They have to have landed here: a wait for them in the loop would be one for the columns on their way. */
#pragma unroll
        for (int n = 0; n < NB; n++)
#pragma unroll
            for (int kc = 0; kc < KC; kc++) asm volatile("" : "+v"(kf[n][kc]));

        uint32_t at[4];                   /* addresses of units 2 kc + half, less 64 kc of them, by kc % 4 */
#pragma unroll
        for (int k = 0; k < 4; k++)
            at[k] = (uint32_t)(uintptr_t)(sum_local *)box + (uint32_t)(sum_unit(2 * k + half, col) - 64 * k) * 16u;

        float sum[NB][16];
#pragma unroll
        for (int n = 0; n < NB; n++)
#pragma unroll
            for (int i = 0; i < 16; i++) sum[n][i] = 0.0f;
        /* Row and head of the block's first and last column, without divisions. */
        int i0 = 32 * c0 / t.group, g0 = 32 * c0 - i0 * t.group;
        int i1 = (32 * c0 + 31) / t.group, g1 = 32 * c0 + 31 - i1 * t.group;
        put(0, 0);
        __syncthreads();
        /* Score i of a lane is of position 8 (i / 4) + 4 half + i % 4 of its 32. The weights of scores i .. i+3,
         * which every row of the block sees, or those of 32 n + .. <= last... */
        const auto key_scales = [&](int n, int i) {
            return key_scale[Q8 ? wave * (kWaveTokens / 4) + 8 * n + 2 * (i / 4) + half : 0];
        };
        constexpr int PARTS = TWO ? 2 : 1, STAGES = KC * PARTS, DEPTH = STAGES < 6 ? STAGES - 1 : 6, PER = 16 / STAGES;
        attn_f16 x[NB];
        attn_f4 scales;
        const auto weigh = [&](int n, int i, float up, float z) {
            if (Q8 && i % 4 == 0) scales = key_scales(n, i);
            sum[n][i] += attn_exp2(fmaf(Q8 ? x[n][i] * scales[i % 4] : x[n][i], up, -z));
        };
        const auto weigh_to = [&](int n, int i, float up, float z, int last) {
            if (Q8 && i % 4 == 0) scales = key_scales(n, i);
            const float w = attn_exp2(fmaf(Q8 ? x[n][i] * scales[i % 4] : x[n][i], up, -z));
            sum[n][i] += 32 * n + 8 * (i / 4) + i % 4 <= last ? w : 0.0f;
        };
        /* ... and all 16 with the mask, of block c. */
        const auto weigh_masked = [&](int n, int c, float up, float z) {
            int side = half;
            asm volatile("" : "+v"(side));       /* nothing of this is kept through the loop */
            const int r = 32 * c + col, pos = first + min(r, rows - 1) / t.group;
#pragma unroll
            for (int i = 0; i < 16; i++) {
                if (Q8 && i % 4 == 0) scales = key_scales(n, i);
                const int tok = 8 * (i / 4) + 4 * side + i % 4;
                float w = attn_exp2(fmaf(Q8 ? x[n][i] * scales[i % 4] : x[n][i], up, -z));
                w = lost[n] >> tok & 1u ? __builtin_nanf("") : w;
                sum[n][i] += r < rows && attn_sees(t, pos, j0 + 32 * n + tok) ? w : 0.0f;
            }
        };
        /* The scores of 32 positions and the block in `buf`, a fragment's MFMA a stage, with the fragments read DEPTH
         * stages ahead and other work under them. */
        const auto products = [&](int n, int buf, auto under) {
            const auto fragment = [&](int st) {
                const int kc = st / PARTS, part = st % PARTS;
                return __builtin_bit_cast(attn_h8, *(const sum_local_u4 *)(uintptr_t)(
                    at[kc & 3] + (uint32_t)(buf * PARTS * UNITS * 16) + (uint32_t)((part * UNITS + 64 * kc) * 16)));
            };
            attn_h8 f[DEPTH + 1];
#pragma unroll
            for (int st = 0; st < DEPTH; st++) f[st] = fragment(st);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int st = 0; st < STAGES; st++) {
                const attn_f16 none = {};
                const attn_h8 w = f[st % (DEPTH + 1)];
                if (st + DEPTH < STAGES) f[(st + DEPTH) % (DEPTH + 1)] = fragment(st + DEPTH);
                x[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[n][st / PARTS], w, st ? x[n] : none, 0, 0, 0);
                under(st);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        /* Block c is in buffer `buf`, block c + 1 in registers `buf ^ 1`, block c + 2 comes into `buf`. The weights
         * of the first 32 positions are made under the products of the others, theirs under those of the next block's
         * first. */
        float up1 = 0.0f, z1 = 0.0f;      /* of the block whose x[1] waits */
        int last1 = 0;
        bool waits = false, plain1 = false, whole1 = false;
        const bool simple = !(lost[0] | lost[1]) && t.window == 0;     /* the mask is the order of positions alone */
        const bool early = wave >= kWaves / 2;
        const auto step = [&](int c, int buf) {
            if (c + 2 < c1) load(buf);
            /* Of the two waves of a SIMD one converts the next block before its products, the other behind them. */
            if (early && c + 1 < c1) put(buf ^ 1, buf ^ 1);
            const int p0 = first + i0, p1 = min(first + i1, s.len - 1);
            /* blocks in front of this wave's positions see none of them */
            if (p1 >= j0) {
                const bool whole = attn_all_seen(t, j0, kWaveTokens, p0, p1) && !(lost[0] | lost[1]);
                const bool plain = whole || simple;
                if (waits && whole1) {
                    products(0, buf, [&](int st) {
#pragma unroll
                        for (int e = 0; e < PER; e++) weigh(1, st * PER + e, up1, z1);
                    });
                } else if (waits && plain1) {
                    products(0, buf, [&](int st) {
#pragma unroll
                        for (int e = 0; e < PER; e++) weigh_to(1, st * PER + e, up1, z1, last1);
                    });
                } else {
                    if (waits) weigh_masked(1, c - 1, up1, z1);
                    products(0, buf, [](int) {});
                }
                up1 = cz[buf][0][col];
                z1 = cz[buf][1][col];
                whole1 = whole;
                if (!whole) {       /* the last of the wave's positions that the lane's column sees, less its first */
                    const int r = 32 * c + col;
                    last1 = r < rows ? first + r / t.group - j0 - 4 * half : -1;
                }
                if (whole) {
                    products(1, buf, [&](int st) {
#pragma unroll
                        for (int e = 0; e < PER; e++) weigh(0, st * PER + e, up1, z1);
                    });
                } else if (plain) {
                    products(1, buf, [&](int st) {
#pragma unroll
                        for (int e = 0; e < PER; e++) weigh_to(0, st * PER + e, up1, z1, last1);
                    });
                } else {
                    products(1, buf, [](int) {});
                    weigh_masked(0, c, up1, z1);
                }
                waits = true;
                plain1 = plain;
            }
            i0 += step_i;
            i1 += step_i;
            g0 += step_g;
            g1 += step_g;
            if (g0 >= t.group) {
                g0 -= t.group;
                i0++;
            }
            if (g1 >= t.group) {
                g1 -= t.group;
                i1++;
            }
            if (!early && c + 1 < c1) put(buf ^ 1, buf ^ 1);
            __syncthreads();
        };
        for (int c = c0; c < c1; c += 2) {
            step(c, 0);
            if (c + 1 < c1) step(c + 1, 1);
        }
        if (waits) weigh_masked(1, c1 - 1, up1, z1);

        /* The tile's sums (or this workgroup's part of them) go to a place of their own, number group_index + tile:
         * each next one of a sequence and head has the next workgroup, the next tile or both. */
        float *const to = p.partial + (((size_t)b * a.kv_heads + head) * p.slots + group_index + tile) * kTokens +
                          wave * kWaveTokens;
#pragma unroll
        for (int n = 0; n < NB; n++)
#pragma unroll
            for (int i = 0; i < 16; i++) {
                float w = sum[n][i];
                w += xor_partner<1>(w);
                w += xor_partner<2>(w);
                w += xor_partner<4>(w);
                w += xor_partner<8>(w);
                w += xor_partner<16>(w);
                if (col == 0) to[32 * n + 8 * (i / 4) + 4 * half + i % 4] = w;
            }
        __syncthreads();        /* the next tile's first block goes where the last one's is read */
    }
}

/* The sums of few rows from their scores, and of many from the workgroups' parts: four positions a thread. */
__global__ __launch_bounds__(256) void sera_attn_sums_kernel(kv_args a, attn_args t, attn_sums p) {
    __shared__ float2 norms[kFewNorms];
    const int b = (int)(blockIdx.z * gridDim.y + blockIdx.y);
    if (b >= a.sequences) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int head = (int)blockIdx.x % a.kv_heads, block0 = (int)blockIdx.x / a.kv_heads * 1024;
    const int w0 = block0 + 256 * wave, j = w0 + 4 * lane, tile = w0 / kTokens;
    const kv_seq s = kv_sequence(a, b);
    if (s.bad || block0 >= s.len) return;
    const bool few = s.n * t.group <= t.few_columns;
    if (few && attn_few_seen(t, s, block0, 1024)) {
        attn_few_norms(a, t, p, s, head, norms);
        __syncthreads();
    }
    if (w0 >= s.len) return;
    const size_t place = (size_t)b * a.kv_heads + head;
    attn_f4 w = {0.0f, 0.0f, 0.0f, 0.0f};
    if (few) {
        if (j < s.len) w = attn_few_sums(t, p, s, place, j, norms);
    } else {
        constexpr int BATCH = 8;        /* loads on their way */
        /* units in front of the tile's */
        int64_t u0 = 0;
        for (int x = lane; x < tile; x += 64) {
            const sum_blocks r = sum_blocks_of(t, s, x);
            u0 += max(r.c1 - r.c0, 0);
        }
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) u0 += __shfl_xor(u0, o, 64);
        const sum_blocks range = sum_blocks_of(t, s, tile);
        const int64_t u1 = u0 + max(range.c1 - range.c0, 0);
        if (u0 < u1) {
            const int g0 = (int)(u0 / p.share), g1 = (int)((u1 - 1) / p.share);
            const float *x = p.partial + (place * p.slots + tile) * kTokens + j % kTokens;
            for (int g = g0; g <= g1; g += BATCH) {
                attn_f4 y[BATCH];
#pragma unroll
                for (int k = 0; k < BATCH; k++) y[k] = *(const attn_f4 *)(x + (size_t)min(g + k, g1) * kTokens);
#pragma unroll
                for (int k = 0; k < BATCH; k++)
                    if (g + k <= g1) w += y[k];
            }
        }
    }
    attn_put_sums(t, s, place, j, w);
}

namespace {

template <int TYPE, typename T, int D>
void columns_go(const kv_args &a, const attn_args &t, const attn_sums &p, hipStream_t s) {
    const int y = a.sequences < 32768 ? a.sequences : 32768;
    hipLaunchKernelGGL((sera_attn_columns_kernel<TYPE, T, D>),
                       dim3((unsigned)(p.groups * a.kv_heads), (unsigned)y, (unsigned)((a.sequences + y - 1) / y)),
                       dim3(64 * kWaves), 0, s, a, t, p);
}

template <int TYPE, typename T>
void columns_d(int dim, const kv_args &a, const attn_args &t, const attn_sums &p, hipStream_t s) {
    dim == 64 ? columns_go<TYPE, T, 64>(a, t, p, s) : columns_go<TYPE, T, 128>(a, t, p, s);
}

template <int TYPE>
void columns_t(uint32_t type, int dim, const kv_args &a, const attn_args &t, const attn_sums &p, hipStream_t s) {
    if (type == SERA_TYPE_F32) columns_d<TYPE, float>(dim, a, t, p, s);
    else if (type == SERA_TYPE_F16) columns_d<TYPE, _Float16>(dim, a, t, p, s);
    else columns_d<TYPE, __bf16>(dim, a, t, p, s);
}

}  // namespace

/* A workgroup runs on a CU; each has an equal share of all units, of 8 at least: the start of one costs some 5. */
static void share_units(attn_sums &p, const kv_args &a, int cus) {
    const int64_t sequences = (a.rows + a.max_new - 1) / a.max_new;
    int64_t share = (p.units * sequences * a.kv_heads + cus - 1) / cus;
    if (share < 8) share = 8;
    if (share > 0x3fffffff) share = 0x3fffffff;
    if (p.groups && share * p.groups < p.units) share = (p.units + p.groups - 1) / p.groups;
    p.share = (int)share;
    p.groups = (int)((p.units + share - 1) / share);
}

/* With a window a sequence has fewer units, and they are shared anew; the workspace, whose size knows no window, has room
 * for as many workgroups as before and no more. A row sees as many tiles as its window touches, and those of sinks; each
 * tile that rows see any of has two blocks begun. 1024 rows of 64 heads at the end of 16384 positions with a window of
 * 512 and 4 sinks (8 kv heads, fp32 rows, fp16 cache): the sums take 110 us, in shares of the whole context 870, as few
 * workgroups had any. */
void sera_attn_sums_shorten(attn_sums &p, const kv_args &a, const attn_args &t, int group) {
    if (!t.window || !p.groups) return;
    const int64_t rows = a.max_new, blocks = (rows * group + 31) / 32;
    const int64_t touched = ((int64_t)t.window + kTokens - 2) / kTokens + 1;
    const int64_t sinks = ((int64_t)(t.sinks < a.max_kv ? t.sinks : a.max_kv) + kTokens - 1) / kTokens;
    const int64_t units = sinks * blocks + (rows * touched * group + 31) / 32 +
                          2 * ((rows + t.window + kTokens - 2) / kTokens + 1);
    if (units >= p.units) return;
    p.units = units;
    share_units(p, a, t.cus);
}

/* How the sums are made, with few_rows columns of each sequence at most in the kernel of few rows (0: none goes
 * there) and groups of `group` columns for each of max_new rows at most elsewhere (0: none). Bytes of workspace in
 * *bytes. */
attn_sums sera_attn_sums_plan(const kv_args &a, int few_rows, int group, int cus, size_t *bytes) {
    attn_sums p = {};
    p.pitch = ((size_t)a.max_kv + 31) & ~(size_t)31;
    p.few_rows = few_rows;
    const size_t arrays = (size_t)a.sequences * a.kv_heads;
    p.scores_bytes = (few_rows * arrays * p.pitch * sizeof(float) + 15) & ~(size_t)15;
    *bytes = p.scores_bytes;
    if (!group) return p;
    /* The units of a sequence of max_new rows over max_kv positions: of tile t those of rows behind it, of all rows
     * at most. A block begun counts, so a shorter sequence has no more. */
    const int64_t tiles = ((int64_t)a.max_kv + kTokens - 1) / kTokens;
    const int64_t blocks = ((int64_t)a.max_new * group + 31) / 32;
    const int64_t part = ((int64_t)a.max_kv - blocks * 32 / group) / kTokens;  /* tiles in front of all rows, about */
    int64_t units = 0;
    const int64_t whole = part < 0 ? 0 : part > tiles ? tiles : part;
    units += whole * blocks;
    for (int64_t x = whole; x < tiles; x++) {
        const int64_t n = ((int64_t)a.max_kv - x * kTokens) * group / 32 + 2;
        units += n < blocks ? n : blocks;
    }
    p.units = units;
    share_units(p, a, cus);
    p.slots = (size_t)(p.groups + tiles);
    *bytes += arrays * p.slots * kTokens * sizeof(float);
    return p;
}

/* After attention (sera_launch_attn). many: some sequences are not the few-row kernel's. */
hipError_t sera_launch_attn_sums(uint32_t cache_type, uint32_t type, int dim, const kv_args &a, const attn_args &args,
                                 const attn_sums &p, bool many, hipStream_t s) {
    attn_args t = args;
    if (!p.few_rows) t.few_columns = -1;            /* sequences without rows are the others' too */
    if (many) {
        if (cache_type == SERA_KV_F16) columns_t<(int)SERA_KV_F16>(type, dim, a, t, p, s);
        else columns_t<(int)SERA_KV_Q8>(type, dim, a, t, p, s);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    const int y = a.sequences < 32768 ? a.sequences : 32768;
    const int64_t four = ((int64_t)a.max_kv + 1023) / 1024;
    hipLaunchKernelGGL(sera_attn_sums_kernel, dim3((unsigned)(four * a.kv_heads), (unsigned)y,
                                                   (unsigned)((a.sequences + y - 1) / y)), dim3(256), 0, s, a, t, p);
    return hipGetLastError();
}
