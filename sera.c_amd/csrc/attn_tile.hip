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
 * as fp16 in steps of two 32-token tiles, which come by direct-to-LDS loads two to three
 * steps ahead (8-bit codes into a ring of their own, from where they are
 * converted once for all waves), already in the order that the A operands are
 * read in: K rows with the token bits 2 and 3 exchanged, so that the scores a
 * lane gets are its B operand of the second product, 16-byte units of a row
 * exchanged by the row (xor) against bank conflicts; V in units of (16 tokens,
 * 32 channels), read as one run. A lane's 16 scores belong to one row, so the
 * softmax is in the lane but for one step between the halves of a wave.
 *
 * fp32 rows hold q and the weights as two fp16 terms each: twice the MFMAs,
 * the same reads of K and V. What bounds it: a tile of a wave is 32 (fp32 rows; 16 otherwise)
 * MFMAs of 32 cycles, about 100 VALU instructions, 16 fragment reads; the two
 * waves of a SIMD overlap part of it, MFMAs are busy 40% of the time
 * (prefill of 2048 tokens). Registers decide the rest: 64 for the sums and 64 for q
 * (fp32 rows, 128 channels) leave room for one tile of scores, not for the
 * next one's beside it, and a value spilled and reloaded in the loop waits for
 * all loads on their way. 64 rows a wave at one wave per SIMD were slower
 * (356 us against 178 for that prefill: nothing hides a wave's own latencies), and so
 * was a strict turn-taking of the two waves by barriers (no gain).
 * 2048 tokens x 64 heads: 150 us, 920 TFLOP/s of fp16 products (fp32 rows),
 * 98 us, 700 (16-bit rows), in calls one after another; 168 and 111 us where a
 * graph leaves no gap between them. A large matrix product reaches 1180 here. 512 rows over
 * 32768 8-bit tokens: 1030 us, 1060 TFLOP/s.
 */
#include "attn_device.h"
#include "sera_launch.h"

namespace {

constexpr int kListed = 512;    /* tiles whose page ids are in LDS at a time */

template <int TYPE, int D, int RG, int KG>
struct tile_shape {
    static constexpr bool Q8 = TYPE == (int)SERA_KV_Q8;
    static constexpr int NW = RG * KG, NT = 64 * NW;
    static constexpr int NSUB = 2;                   /* 32-token tiles of a step */
    static constexpr int UNITS = 32 * D / 8;         /* 16-byte fp16 units of K (and V) in a tile */
    static constexpr int KC = D / 16, NC = D / 32;
    static constexpr int XOR = D / 8 < 16 ? D / 8 - 1 : 15;
    static constexpr int PER = UNITS * 2 / (Q8 ? 2 : 1);    /* 16-byte loads of a tile, K's then V's */
    static constexpr int PIECES = NSUB * PER / NT;          /* of a thread and step */
    /* Buffers of the step whose V is read, of the next one, whose K is read already, and, fp16, of those on
     * their way; 8-bit codes land in a ring of their own and are converted. */
    static constexpr int RING = Q8 ? 2 : NW == 8 ? 4 : 3;
    static constexpr int BUFS = Q8 ? 3 : RING;
    static constexpr int AHEAD = Q8 ? 2 : RING - 1;         /* steps on their way at first */
    static constexpr int LOADS = PIECES + (Q8 ? 1 : 0);     /* of a wave and step */
};

__device__ __forceinline__ int swap_token(int r) { return (r & ~12) | ((r & 4) << 1) | ((r & 8) >> 1); }

template <int TYPE, int D, int RG, int KG>
struct tile_lds {
    using S = tile_shape<TYPE, D, RG, KG>;
    attn_u4 buf[S::BUFS][S::NSUB][2][S::UNITS];                /* K, V */
    attn_u4 raw[S::Q8 ? S::RING : 1][S::Q8 ? S::PIECES * S::NT : 1];
    float raw_scale[S::Q8 ? S::RING : 1][S::Q8 ? S::NT : 1];
    float scale[S::Q8 ? 3 : 1][S::NSUB][3][32];                /* K scale, V scale, log2 of the V scale */
    float row_scale[S::NW][32];                                /* of q's rows, at the start */
    alignas(16) int ids[2 * kListed + 4];
    int lost;                                                  /* a page of those is lost */
    int any;                                                    /* tiles with values taken out, and which */
    uint8_t odd[S::Q8 ? 4 : kListed];
};

/* 32 rows of D elements, 16 bytes of T a lane. */
template <typename T, int D>
struct tile_rows {
    static constexpr int VEC = 16 / (int)sizeof(T), LANES = D / VEC, ROWS = 64 / LANES, N = 32 / ROWS;
};

/* The largest of m over LANES lanes that share a row. */
template <int LANES>
__device__ __forceinline__ float tile_row_max(float m) {
    m = fmaxf(m, xor_partner<1>(m));
    m = fmaxf(m, xor_partner<2>(m));
    m = fmaxf(m, xor_partner<4>(m));
    if constexpr (LANES >= 16) m = fmaxf(m, xor_partner<8>(m));
    if constexpr (LANES >= 32) m = fmaxf(m, xor_partner<16>(m));
    return m;
}

typedef const __attribute__((address_space(1))) void attn_global;
typedef __attribute__((address_space(3))) void attn_local;
typedef __attribute__((address_space(3))) attn_u4 attn_local_u4;

/* All but the last LEFT of this wave's loads have landed. */
template <int LEFT>
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LEFT) : "memory"); }

/* The loads of a step have landed when at most `after` later steps (of LOADS each) are on their way. */
template <int LOADS>
__device__ __forceinline__ void wait_step(int after) {
    if (after >= 2) wait_loads<2 * LOADS>();
    else if (after == 1) wait_loads<LOADS>();
    else wait_loads<0>();
}

__device__ __forceinline__ void barrier_lds() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

}  // namespace

/* Waves per SIMD: 8 waves of 128 channels take a CU's registers and LDS; two
 * workgroups of 64 channels fit where their registers do (a ragged window
 * prefill of fp16 rows: 42 us, 57 us with one). */
template <int TYPE, typename T, int D, int RG, int KG>
constexpr int tile_occupancy() {
    return RG * KG / 4 * (D == 64 && RG * KG == 8 && TYPE == (int)SERA_KV_F16 && sizeof(T) == 2 ? 2 : 1);
}

template <int TYPE, typename T, int D, int RG, int KG>
__global__ __launch_bounds__(64 * RG * KG, (tile_occupancy<TYPE, T, D, RG, KG>()))
void sera_attn_tile_kernel(kv_args a, attn_args t, int slots, int splits, int chunk) {
    using S = tile_shape<TYPE, D, RG, KG>;
    constexpr bool Q8 = S::Q8, TWO = sizeof(T) == 4;
    constexpr int NT = S::NT, NSUB = S::NSUB, UNITS = S::UNITS, KC = S::KC, NC = S::NC, BR = 32 * RG;
    constexpr int PER = S::PER, PIECES = S::PIECES, ES = Q8 ? 1 : 2;
    __shared__ tile_lds<TYPE, D, RG, KG> lds;

    const int slot = (int)(blockIdx.z * gridDim.y + blockIdx.y);
    if (slot >= slots) return;
    const int head = (int)blockIdx.x % a.kv_heads, split = (int)blockIdx.x / a.kv_heads;
    int unit;
    const int b = attn_find_tile(a, t, BR, slots, slot, &unit);
    if (b < 0) return;
    const kv_seq s = kv_sequence(a, b);
    const int rows = s.n * t.group, r0 = unit * BR;
    if (r0 >= rows || rows <= t.few_columns) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 31, half = lane >> 5;
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
    const int w0 = r0 + 32 * rg;
    /* Token and head of the workgroup's row `local`, without a division: (x + 1/2) / group is a 1/(2 group) or more
     * from every whole number, its error in fp32 below (1 + 256 / group) 2^-22. */
    const int at0 = r0 / t.group, rem0 = r0 - at0 * t.group;
    const float inv_group = 1.0f / (float)t.group;
    auto place = [&](int local, int &h) {
        const int x = rem0 + min(local, rows - 1 - r0), q = (int)(((float)x + 0.5f) * inv_group);
        h = x - q * t.group;
        return at0 + q;
    };
    int unused;
    const int pos = first + place(32 * rg + col, unused);
    const int pw0 = first + min(w0, rows - 1) / t.group, pw1 = first + min(w0 + 31, rows - 1) / t.group;
    const attn_whole whole = attn_whole_of(t, range, first < 0 ? -1 : pw0, pw1, 5);                /* of this wave */
    const attn_whole all = attn_whole_of(t, range, max(first + r0 / t.group, 0), end - 1, 5);      /* of all waves */
    /* Tiles that a row of this wave sees: of those before `last`, sinks and those from `from` on. */
    const int last = w0 >= rows ? 0 : (pw1 >= 0 ? pw1 >> 5 : -1) + 1 + range.sink_tiles - range.low;
    const int from = t.window > 0 ? (max(pw0 - t.window + 1, 0) >> 5) + range.sink_tiles - range.low : 0;

    /* This wave's rows of q, on their way while pages are looked up. */
    using R = tile_rows<T, D>;
    const int part = lane % R::LANES * R::VEC, part_row = 32 * rg + lane / R::LANES;
    attn_vec<T, R::VEC> q_in[R::N];
#pragma unroll
    for (int i = 0; i < R::N; i++) {
        int h;
        const int at = place(part_row + i * R::ROWS, h);
        q_in[i] = *(const attn_vec<T, R::VEC> *)((const T *)t.q + (s.row0 + at) * t.q_stride + q0 + h * D + part);
    }

    attn_h8 qh[KC], ql[TWO ? KC : 1];
    float c = 0.0f, m = kAttnLowest, l = 0.0f, l1 = 0.0f;

    const int mask = (1 << a.page_shift) - 1;
    const size_t kv_bytes = ((size_t)D << a.page_shift) * ES;
    const uint8_t *base = a.data + (size_t)head * a.head_bytes;
    int g = v0, stop = v0;
    bool lost = false;

    /* The loads of a step are 16-token blocks of UB pieces, tile by tile: K's two, V's two. A wave's 64 pieces of
     * round e are of block e * (NT / UB) + wave * 64 / UB; a thread has the same place in all its blocks, so one
     * offset for K's and one for V's. */
    constexpr int UB = D * ES, STEP_UNITS = NSUB * PER;
    int off_k, off_v;
    {
        constexpr int ROW = D * ES / 16;
        const int z = tid % UB, row = z / ROW, u = z % ROW;
        off_k = swap_token(row) * (D * ES) + (Q8 ? u : u ^ (row & S::XOR)) * 16;
        off_v = Q8 ? z * 16 : (z / 64 * 32 + z % 32) * 32 + z / 32 % 2 * 16;
    }
    /* Starts the loads of the step at tile v into ring place r. Past the last tile they read page 0. */
    auto stage_load = [&](int v, int r) {
        int id[4];
        const attn_u4 four = *(const attn_u4 *)&lds.ids[2 * (v - g)];
#pragma unroll
        for (int i = 0; i < 4; i++) id[i] = max(__builtin_amdgcn_readfirstlane((int)four[i]), 0);
        const int wb = wave * 64 / UB;
#pragma unroll
        for (int e = 0; e < PIECES; e++) {
            const int block = e * (NT / UB) + wb, sub = block >> 2, odd = block & 1;
            const bool is_v = block & 2;
            const int page = sub ? odd ? id[3] : id[2] : odd ? id[1] : id[0];
            const uint8_t *p = base + (size_t)page * a.page_bytes + (is_v ? kv_bytes : 0) +
                               (size_t)((range.tile(v + sub) * 32 + 16 * odd) & mask) * (D * ES);
            asm("" : "+s"(p));     /* a scalar address and the thread's 32-bit offset, kept apart */
            attn_u4 *to = (Q8 ? lds.raw[0] : lds.buf[0][0][0]) + r * STEP_UNITS + e * NT + wave * 64;
            __builtin_amdgcn_global_load_lds((attn_global *)(p + (uint32_t)(is_v ? off_v : off_k)), (attn_local *)to,
                                             16, 0, 0);
        }
        if (Q8) {      /* both scales of a tile; every wave loads some, those of the first NSUB are used */
            const int token = lane & 31, sub = wave % NSUB;
            const int page = token & 16 ? sub ? id[3] : id[1] : sub ? id[2] : id[0];
            const float *p = (const float *)(base + (size_t)page * a.page_bytes + 2 * kv_bytes) +
                             ((size_t)half << a.page_shift) + ((range.tile(v + sub) * 32 + token) & mask);
            __builtin_amdgcn_global_load_lds((attn_global *)p, (attn_local *)&lds.raw_scale[r][wave * 64], 4, 0, 0);
        }
    };
    /* Converts this thread's codes of ring place r into buffer `to`. */
    auto convert = [&](int r, int to) {
#pragma unroll
        for (int e = 0; e < PIECES; e++) {
            const int x = e * NT + tid, y = x % PER, z = y % (PER / 2);
            const attn_u4 w = lds.raw[r][x];
            const attn_u4 x0 = __builtin_bit_cast(attn_u4, attn_codes(w[0], w[1]));
            const attn_u4 x1 = __builtin_bit_cast(attn_u4, attn_codes(w[2], w[3]));
            attn_u4 *p = lds.buf[to][x / PER][y >= PER / 2];
            if (y < PER / 2) {
                constexpr int ROW = D / 16;
                const int row = z / ROW, u = 2 * (z % ROW);
                p[row * (D / 8) + (u ^ (row & S::XOR))] = x0;
                p[row * (D / 8) + ((u + 1) ^ (row & S::XOR))] = x1;
            } else {
                const int u = z / D * (2 * D) + z % D / 32 * 64 + z % 32;
                p[u] = x0;
                p[u + 32] = x1;
            }
        }
        if (wave < NSUB) {
            const float x = lds.raw_scale[r][tid];
            float (*p)[32] = lds.scale[to][wave];
            p[half][col] = x;
            if (half) p[2][col] = attn_log_scale(x);
        }
    };

    constexpr int AHEAD = S::AHEAD;
    /* The pages of the tiles from g on, and the first loads. */
    auto begin = [&]() {
        stop = min(v1, g + kListed);
        const int steps = (stop - g + NSUB - 1) / NSUB;
        barrier_lds();
        if (tid == 0) lds.lost = 0;
        barrier_lds();
        for (int e = tid; e < 2 * (stop - g) + 4; e += NT) {
            int id = 0;
            if (e < 2 * (stop - g)) id = attn_page(a, b, range.tile(g + (e >> 1)) * 32 + 16 * (e & 1), s.len);
            lds.ids[e] = id;
            if (id < 0) lds.lost = 1;
        }
        if (!Q8) {
            for (int e = tid; e < stop - g; e += NT) lds.odd[e] = 0;
            if (tid == 0) lds.any = 0;
        }
        __syncthreads();
        lost = __builtin_amdgcn_readfirstlane(lds.lost) != 0;
        for (int st = 0; st < min(AHEAD, steps); st++) stage_load(g + st * NSUB, st);
    };

    /* q's rows, scaled, as fragments: through LDS in the buffer that is loaded last, half of the channels of the high
     * and then of the low parts at a time. (Fragments straight from memory would touch 64 places an access.) */
    auto fragments_of_q = [&]() {
        uint8_t *box = (uint8_t *)lds.buf[S::BUFS - 1] + wave * (32 * D);
        static_assert(S::NW * 32 * D <= sizeof(lds.buf[0]), "room for q");
        attn_vec<_Float16, R::VEC> hi[R::N], lo[R::N];
        float minus = -1.0f;
        asm("" : "+s"(minus));
#pragma unroll
        for (int i = 0; i < R::N; i++) {
            float x[R::VEC], most = 0.0f;
#pragma unroll
            for (int z = 0; z < R::VEC; z++) {
                x[z] = kv_to_f32(q_in[i].v[z]);
                most = fmaxf(most, fabsf(x[z]));
            }
            const int e = attn_q_exponent(tile_row_max<R::LANES>(most));
            const float up = ldexpf(t.scale_log2 < 0.0f ? -1.0f : 1.0f, e);
            /* not 0: a masked score is -inf * c */
            if (part == 0)
                lds.row_scale[wave][i * R::ROWS + lane / R::LANES] =
                    fmaxf(ldexpf(fabsf(t.scale_log2), -e), 1.17549435e-38f);
#pragma unroll
            for (int z = 0; z < R::VEC; z += 2) {
                const float a0 = x[z] * up, a1 = x[z + 1] * up;
                const attn_h2 h = attn_pack(a0, a1);
                hi[i].v[z] = h[0];
                hi[i].v[z + 1] = h[1];
                if (TWO) {
                    lo[i].v[z] = (_Float16)fmaf((float)h[0], minus, a0);
                    lo[i].v[z + 1] = (_Float16)fmaf((float)h[1], minus, a1);
                }
            }
        }
        constexpr int HALF_UNITS = D / 16;
#pragma unroll
        for (int turn = 0; turn < (TWO ? 4 : 2); turn++) {
            const int first_channel = turn % 2 * (D / 2);
            asm volatile("" ::: "memory");         /* the wave's own LDS, which it accesses in order */
            if (part >= first_channel && part < first_channel + D / 2)
#pragma unroll
                for (int i = 0; i < R::N; i++) {
                    const int r = i * R::ROWS + lane / R::LANES, byte = 2 * (part - first_channel);
                    const int at = r * D + (((byte >> 4) ^ (r & (HALF_UNITS - 1))) << 4) + (byte & 15);
                    *(attn_vec<_Float16, R::VEC> *)(box + at) = turn < 2 ? hi[i] : lo[i];
                }
            asm volatile("" ::: "memory");
#pragma unroll
            for (int k = 0; k < KC / 2; k++) {
                const int at = col * D + (((2 * k + half) ^ (col & (HALF_UNITS - 1))) << 4);
                const attn_h8 f = *(const attn_h8 *)(box + at);
                if (turn < 2) qh[turn * (KC / 2) + k] = f;
                else if (TWO) ql[TWO ? (turn - 2) * (KC / 2) + k : 0] = f;
            }
        }
        c = lds.row_scale[wave][col];
    };

    if (v0 < v1) {
        begin();
        fragments_of_q();
    }
    attn_f16 o[NC];
#pragma unroll
    for (int n = 0; n < NC; n++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[n][i] = 0.0f;

    attn_f16 x;                        /* scores: score i is of token 16 * (i / 8) + 8 * half + i % 8 */
    attn_f4 vs[Q8 ? 4 : 1];            /* and the scales of those tokens' values */
    float top = kAttnLowest;           /* their largest, as an exponent */
    const int half8 = 8 * half;

    /* Fragment i of the products: V's of this tile (i < 2 NC), then K's of the next one. K's units are xored in
     * address bits that the fragment's number has to itself, so one address serves all. */
    constexpr uint32_t TILE_BYTES = UNITS * 16;
    const uint32_t lds_at = (uint32_t)(uintptr_t)(attn_local *)lds.buf;
    const uint32_t k_at = lds_at + col * (D * 2) + ((half ^ (col & S::XOR)) << 4);
    const uint32_t v_at = lds_at + TILE_BYTES + lane * 16;
    auto fragment = [&](int i, uint32_t k_tile, uint32_t v_tile) {
        const uint32_t at = i < 2 * NC ? v_at + v_tile + (uint32_t)i * 1024u
                                       : (k_at + k_tile) ^ (uint32_t)((i - 2 * NC) << 5);
        return __builtin_bit_cast(attn_h8, *(const attn_local_u4 *)(uintptr_t)at);
    };
    /* The scores x are complete: 8-bit keys' scales, and the largest. */
    auto finish = [&](int buf, int sub) {
        top = kAttnLowest;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int at = 16 * (i / 2) + half8 + 4 * (i % 2);
            attn_f4 ks, lv;
            if (Q8) {
                ks = *(const attn_f4 *)&lds.scale[buf][sub][0][at];
                lv = *(const attn_f4 *)&lds.scale[buf][sub][2][at];
            }
#pragma unroll
            for (int z = 0; z < 4; z++) {
                if (Q8) x[4 * i + z] *= ks[z];
                top = fmaxf(top, Q8 ? fmaf(x[4 * i + z], c, lv[z]) : x[4 * i + z]);
            }
            if (Q8 && i == 1) __builtin_amdgcn_sched_barrier(0);      /* registers: half of the scales at a time */
        }
        if (!Q8) top *= c;
    };
    auto scores = [&](int buf, int sub) {
        uint32_t kt = (buf * NSUB + sub) * 2 * TILE_BYTES;
        asm volatile("" : "+s"(kt));          /* the addresses are made here, not kept */
#pragma unroll
        for (int i = 0; i < 16; i++) x[i] = 0.0f;
#pragma unroll
        for (int k = 0; k < KC; k++) {
            const attn_h8 f = fragment(2 * NC + k, kt, 0);
            x = __builtin_amdgcn_mfma_f32_32x32x16_f16(f, qh[k], x, 0, 0, 0);
            if (TWO) x = __builtin_amdgcn_mfma_f32_32x32x16_f16(f, ql[TWO ? k : 0], x, 0, 0, 0);
        }
        finish(buf, sub);
    };
    /* Mask of tile v, and the running maximum with it. False: no row of this wave sees any of it. */
    auto look = [&](int v, int buf, int sub) {
        if (v >= last || (v < from && range.tile(v) * 32 >= t.sinks)) return false;
        if (Q8)
#pragma unroll
            for (int i = 0; i < 4; i++)
                vs[i] = *(const attn_f4 *)&lds.scale[buf][sub][1][16 * (i / 2) + half8 + 4 * (i % 2)];
        if (lost || v < whole.v0 || v >= whole.v1) {
            const int j = range.tile(v) * 32;
            const int id0 = lds.ids[2 * (v - g)], id1 = lds.ids[2 * (v - g) + 1];
            top = kAttnLowest;
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int at = 16 * (i / 8) + half8 + i % 8;
                const bool sees = attn_sees(t, pos, j + at);
                x[i] = !sees ? -INFINITY : (i < 8 ? id0 : id1) < 0 ? __builtin_nanf("") : x[i];
                top = fmaxf(top, Q8 ? fmaf(x[i], c, lds.scale[Q8 ? buf : 0][sub][2][at]) : x[i] * c);
                if (Q8) vs[i / 4][i % 4] = sees ? vs[i / 4][i % 4] : 0.0f;
                if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);
            }
        }
        top = fmaxf(top, xor_partner<32>(top));
        if (__ballot(top > m + kAttnLag)) {
            const float f = attn_exp2(m - fmaxf(top, m));
            m = fmaxf(top, m);
            l *= f;
            l1 *= f;
#pragma unroll
            for (int n = 0; n < NC; n++) o[n] *= f;
        }
        return true;
    };
    /* The weights of tile (buf, sub) from its scores x, its sums, and the scores of the next tile (nb, ns) into x: in
     * stages of one fragment's MFMAs each, in a fixed order, with the fragments read DEPTH stages ahead. The second
     * half of the weights is made under the MFMAs of the first. */
    auto tile = [&](int buf, int sub, int nb, int ns) {
        constexpr int DEPTH = D == 64 ? 1 : 2, STAGES = KC + 2 * NC;
        __builtin_amdgcn_s_setprio(1);       /* a wave in its products goes before one that is not */
        const float shift = kAttnBias - m;
        float minus = -1.0f;
        asm("" : "+s"(minus));
        const uint32_t kt = (nb * NSUB + ns) * 2 * TILE_BYTES, vt = (buf * NSUB + sub) * 2 * TILE_BYTES;
        attn_h8 f[DEPTH + 1], ph[2], pl[2];
        auto weigh = [&](int e) {
            float a0 = attn_exp2(fmaf(x[e], c, shift)), a1 = attn_exp2(fmaf(x[e + 1], c, shift));
            l += a0;
            l1 += a1;
            if (Q8) {
                a0 *= vs[Q8 ? e / 4 : 0][e % 4];
                a1 *= vs[Q8 ? e / 4 : 0][e % 4 + 1];
            }
            const attn_h2 h = attn_pack(a0, a1);
            ph[e / 8][e % 8] = h[0];
            ph[e / 8][e % 8 + 1] = h[1];
            if (TWO) {
                pl[e / 8][e % 8] = (_Float16)fmaf((float)h[0], minus, a0);
                pl[e / 8][e % 8 + 1] = (_Float16)fmaf((float)h[1], minus, a1);
            }
        };
#pragma unroll
        for (int i = 0; i < DEPTH; i++) f[i] = fragment(i, kt, vt);
#pragma unroll
        for (int e = 0; e < 8; e += 2) weigh(e);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int st = 0; st < STAGES; st++) {
            const attn_h8 w = f[st % (DEPTH + 1)];
            if (st + DEPTH < STAGES) f[(st + DEPTH) % (DEPTH + 1)] = fragment(st + DEPTH, kt, vt);
            const int n = st % NC, k = st < 2 * NC ? st / NC : st - 2 * NC;
            if (st < 2 * NC) {
                o[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(w, ph[k], o[n], 0, 0, 0);
                if (TWO) o[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(w, pl[k], o[n], 0, 0, 0);
            } else {
                if (k == 0)
#pragma unroll
                    for (int i = 0; i < 16; i++) x[i] = 0.0f;
                x = __builtin_amdgcn_mfma_f32_32x32x16_f16(w, qh[k], x, 0, 0, 0);
                if (TWO) x = __builtin_amdgcn_mfma_f32_32x32x16_f16(w, ql[TWO ? k : 0], x, 0, 0, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
            if (st < NC) {
#pragma unroll
                for (int e = 8 + st * (8 / NC); e < 8 + (st + 1) * (8 / NC); e += 2) weigh(e);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        __builtin_amdgcn_s_setprio(0);
        finish(nb, ns);
    };

    /* fp16 values that are not finite, in tiles that some rows of the workgroup see and others do not: a product
     * would carry them into rows that do not see them (0 * inf). They are taken out of the step's buffer, each
     * thread looking at what it loaded, and their tiles marked... */
    auto take_out = [&](int v, int buf) {
        if (Q8 || (v >= all.v0 && v + NSUB <= all.v1)) return;
#pragma unroll
        for (int e = 0; e < PIECES; e++) {
            const int x = e * NT + wave * 64, y = x % PER, tile = v + x / PER;
            if (y < PER / 2 || tile >= stop || (tile >= all.v0 && tile < all.v1)) continue;
            int here = lane;
            asm volatile("" : "+v"(here));
            attn_u4 *p = &lds.buf[buf][x / PER][1][y % (PER / 2) + here];
            attn_h8 w = __builtin_bit_cast(attn_h8, *p), bad;
            if (attn_take_odd(w, bad)) {
                *p = __builtin_bit_cast(attn_u4, w);
                lds.odd[tile - g] = 1;
                lds.any = 1;
            }
        }
    };
    /* ... and in the end the rows that see one get NaN in its channel. */
    auto put_back = [&](int v) {
        int col = lane & 31, half = lane >> 5;
        asm volatile("" : "+v"(col), "+v"(half));       /* nothing of this is kept through the loop */
        const int j = range.tile(v) * 32;
#pragma unroll 1
        for (int k = 0; k < 2; k++) {
            const int id = max(__builtin_amdgcn_readfirstlane(lds.ids[2 * (v - g) + k]), 0);
            const uint8_t *p = base + (size_t)id * a.page_bytes + kv_bytes +
                               (size_t)((j + 16 * k) & mask) * (D * ES) + col * 32 + half * 16;
            attn_h8 sees;
#pragma unroll
            for (int i = 0; i < 8; i++)
                sees[i] = attn_sees(t, pos, j + 16 * k + 8 * half + i) ? (_Float16)1.0f : (_Float16)0.0f;
#pragma unroll
            for (int n = 0; n < NC; n++) {
                attn_h8 w = *(const attn_h8 *)(p + n * 1024), bad;
                attn_take_odd(w, bad);
                attn_f16 hit;
#pragma unroll
                for (int i = 0; i < 16; i++) hit[i] = 0.0f;
                hit = __builtin_amdgcn_mfma_f32_32x32x16_f16(bad, sees, hit, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 16; i++) o[n][i] = hit[i] > 0.0f ? __builtin_nanf("") : o[n][i];
                __builtin_amdgcn_sched_barrier(0);      /* one at a time: this must not spill what the loop holds */
            }
        }
    };

    for (; g < v1; g += kListed) {
        if (g > v0) begin();
        const int steps = (stop - g + NSUB - 1) / NSUB;
        wait_step<S::LOADS>(min(AHEAD, steps) - 1);
        if (Q8) convert(0, 0);
        else take_out(g, 0);
        barrier_lds();
        if (Q8 && AHEAD < steps) stage_load(g + AHEAD * NSUB, 0);
        if (g + kg < stop) scores(0, kg);
        /* The scores of the next tile run beside the weights of this one. */
        int buf = 0, r = 0;           /* this step's buffer; its place in the ring of codes */
        for (int st = 0; st < steps; st++) {
            const int next = buf == S::BUFS - 1 ? 0 : buf + 1;
#pragma unroll
            for (int sub = 0; sub < NSUB; sub += KG) {
                const int v = g + st * NSUB + sub + kg;
                const bool live = v < stop && look(v, buf, sub + kg);
                const bool turn = sub + KG >= NSUB;
                if (turn && st + 1 < steps) {
                    /* This step's scores are all taken: on to the next step's buffer. */
                    if (!Q8) {
                        wait_step<S::LOADS>(min(steps - 2 - st, AHEAD - 2));
                        take_out(g + (st + 1) * NSUB, next);
                    } else {
                        r ^= 1;
                        wait_step<S::LOADS>(min(steps - 2 - st, AHEAD - 1));
                        convert(r, next);
                    }
                    barrier_lds();
                    if (!Q8 && st + AHEAD < steps)
                        stage_load(g + (st + AHEAD) * NSUB, buf == 0 ? S::BUFS - 1 : buf - 1);
                    if (Q8 && st + 1 + AHEAD < steps) stage_load(g + (st + 1 + AHEAD) * NSUB, r);
                }
                /* Past the last tile these are scores of whatever the buffer holds, used by nothing. */
                const int nb = turn ? next : buf, ns = turn ? kg : sub + KG + kg;
                if (live) tile(buf, sub + kg, nb, ns);
                else scores(nb, ns);
            }
            buf = next;
        }
        if (!Q8 && lds.any)
            for (int v = g; v < stop; v++)
                if (lds.odd[v - g]) put_back(v);
    }

    l += l1;
    l += xor_partner<32>(l);
    /* Join the token groups: the upper half of them hands its sums over, lane by lane. */
#pragma unroll
    for (int h = KG / 2; h >= 1; h >>= 1) {
        attn_f4 *box = (attn_f4 *)lds.buf + ((size_t)rg + RG * (kg % h)) * (64 * NC * 4);
        float *mlbox = (float *)lds.ids + 128 * (rg + RG * (kg % h));
        static_assert(sizeof(attn_f4) * RG * (KG / 2) * 64 * NC * 4 <= sizeof(lds.buf), "join space");
        static_assert(sizeof(float) * RG * (KG / 2) * 128 <= sizeof(lds.ids), "join space");
        __syncthreads();
        if (kg >= h && kg < 2 * h) {
#pragma unroll
            for (int n = 0; n < NC; n++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    box[(n * 4 + i) * 64 + lane] =
                        attn_f4{o[n][4 * i], o[n][4 * i + 1], o[n][4 * i + 2], o[n][4 * i + 3]};
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
    /* The result by rows, through LDS: a lane has 16 bytes of two rows' pieces in turn, stores are whole rows. */
    __syncthreads();
    if (kg > 0) return;
    float *box = (float *)lds.buf + rg * (32 * D);
    static_assert(RG * 32 * D * sizeof(float) <= sizeof(lds.buf) + sizeof(lds.raw), "room for the result");
    const float scale = splits > 1 ? 1.0f : 1.0f / l;
#pragma unroll
    for (int n = 0; n < NC; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            attn_f4 y;
#pragma unroll
            for (int z = 0; z < 4; z++) y[z] = splits == 1 && pos < 0 ? 0.0f : o[n][4 * i + z] * scale;
            *(attn_f4 *)(box + col * D + (((8 * n + 2 * i + half) ^ (col & (D / 4 - 1))) << 2)) = y;
        }
    asm volatile("" ::: "memory");
    /* Partial sums by packed row, query head and split; their maxima and sums behind them all. */
    float *const ml = t.workspace + (size_t)a.rows * t.heads * splits * D;
    auto partial = [&](int local) {
        int h;
        const int at = place(local, h);
        return ((size_t)(s.row0 + at) * t.heads + head * t.group + h) * splits + split;
    };
    if (splits > 1 && half == 0 && w0 + col < rows) {
        const size_t k = partial(32 * rg + col);
        ml[2 * k] = m;
        ml[2 * k + 1] = l;
    }
    constexpr int ROWS = 64 / (D / 4);
#pragma unroll 4
    for (int i = 0; i < 32 / ROWS; i++) {
        const int r = i * ROWS + lane / (D / 4), u = lane % (D / 4);
        if (w0 + r >= rows) break;
        const attn_f4 y = *(const attn_f4 *)(box + r * D + ((u ^ (r & (D / 4 - 1))) << 2));
        if (splits > 1) {
            *(attn_f4 *)(t.workspace + partial(32 * rg + r) * D + 4 * u) = y;
        } else {
            int h;
            const int at = place(32 * rg + r, h);
            attn_store4((T *)t.out + (s.row0 + at) * t.out_stride + q0 + h * D + 4 * u, (const float *)&y);
        }
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
    else tile_go<TYPE, T, D, 2, 2>(a, t, p, s);
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
