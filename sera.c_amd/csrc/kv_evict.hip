/*
 * kv_evict.hip - shortening of cached sequences: which positions of a kv head stay, and their move to new pages.
 *
 * Choice: a workgroup for each sequence and kv head. Weights become whole numbers of the same order; the smallest one
 * that stays is built bit by bit, each bit by counting how many are as large. Then each wave walks a run of positions
 * of its own, held in registers up to 16384 positions, and writes what stays behind what the runs before it keep,
 * which a count of each run says.
 *
 * Move: a wave for K or V of 16 new places of a head. A K row is a run of bytes. A V token is an element of each
 * channel's 16, so whole blocks of 16 old tokens come as they lie, go through LDS, and the tokens that stay are
 * picked from there.
 *
 * The move is bound by memory, the choice by the latency of its steps. 64 sequences of 8192 positions to half (8 kv
 * heads, 128 channels, fp16 cache): 32 us and 533 us, for 2.7 GB the rate of a copy; of V's blocks of 16 tokens hardly
 * one is without any that stays, so V is read whole. 24 sequences of up to 3001 (8-bit cache): 16 us and 27 us.
 */
#include "attn_common.h"
#include "sera_dpp.h"
#include "sera_launch.h"

namespace {

constexpr int kKeepWaves = 4;

/* A weight as a whole number of the same order, from 2 on; NaN is 1. */
__device__ __forceinline__ uint32_t keep_key(float w) {
    const uint32_t u = __float_as_uint(w + 0.0f);       /* -0 becomes 0 */
    return w != w ? 1u : (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

/* The sum over a wave, wave-uniform. */
__device__ __forceinline__ int keep_wave_sum(int n) {
    n += xor_partner<1>(n);
    n += xor_partner<2>(n);
    n += xor_partner<4>(n);
    n += xor_partner<8>(n);
    n += xor_partner<16>(n);
    n += xor_partner<32>(n);
    return __builtin_amdgcn_readfirstlane(n);
}

typedef uint32_t move_u4 __attribute__((ext_vector_type(4)));

}  // namespace

/* R: 64-position rows of a wave's run that are held in registers (the run fits); 0: they are read again each time. */
template <int R>
__global__ __launch_bounds__(64 * kKeepWaves) void sera_kv_keep_kernel(kv_args a, evict_args t) {
    __shared__ int part[2][kKeepWaves][4], part_eq[kKeepWaves];
    const int b = (int)(blockIdx.z * gridDim.y + blockIdx.y), head = (int)blockIdx.x;
    if (b >= a.sequences) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int len = a.kv_len[b];
    const bool bad = len < 0 || len > a.max_kv, all = !bad && len <= t.keep;
    const size_t place = (size_t)b * a.kv_heads + head;
    int *__restrict__ kept = t.kept + place * t.keep;
    const float *__restrict__ w = t.weights + place * t.weights_stride;
    float *__restrict__ to = t.new_weights + place * t.weights_stride;
    const int count = bad ? 0 : min(len, t.keep);
    if (head == 0 && tid == 0) t.new_len[b] = bad ? -1 : count;
    for (int x = count + tid; x < t.keep; x += 64 * kKeepWaves) kept[x] = -1;
    if (bad) return;
    if (all) {
        for (int x = tid; x < len; x += 64 * kKeepWaves) {
            kept[x] = x;
            to[x] = w[x];
        }
        return;
    }
    const int lo = t.sinks, hi = len - t.recent;

    /* A wave's run of positions. Those outside the middle count as the largest there are, places behind the run as
     * none. */
    const int run = ((len + kKeepWaves - 1) / kKeepWaves + 63) & ~63;
    const int from = min(wave * run, len), end = min(from + run, len);
    uint32_t key[R ? R : 1];
    const auto key_of = [&](float v, int j) { return j >= end ? 0u : j < lo || j >= hi ? 0xffffffffu : keep_key(v); };
    if (R) {
        float v[R ? R : 1];
#pragma unroll
        for (int r = 0; r < R; r++) v[r] = w[min(from + 64 * r + lane, len - 1)];
#pragma unroll
        for (int r = 0; r < R; r++) key[r] = key_of(v[r], from + 64 * r + lane);
    }
    /* For every row of the run: its first position and its keys. */
    const auto rows = [&](auto each) {
        if constexpr (R > 0) {
#pragma unroll
            for (int r = 0; r < R; r++) each(from + 64 * r, key[r]);
        } else {
            for (int x = from; x < end; x += 64) each(x, key_of(w[min(x + lane, len - 1)], x + lane));
        }
    };

    /* Of all, those outside the middle among them, t.keep stay: those above `cut`, and the first `ties` of those
     * equal to it. The cut is the t.keep-th largest, built bit by bit; as soon as exactly that many reach it, it is
     * the number below. */
    uint32_t cut = 0u;
    int larger = 0, turn = 0;
    bool exact = false;
    for (int bit = 30; bit >= 0 && !exact; bit -= 2) {          /* two bits: three counts */
        int n[3] = {0, 0, 0};
        rows([&](int, uint32_t k) {
#pragma unroll
            for (int i = 0; i < 3; i++) n[i] += k >= (cut | (uint32_t)(i + 1) << bit);
        });
        turn ^= 1;
#pragma unroll
        for (int i = 0; i < 3; i++) {
            n[i] = keep_wave_sum(n[i]);
            if (lane == 0) part[turn][wave][i] = n[i];
        }
        __syncthreads();
        const uint32_t base = cut;
#pragma unroll
        for (int i = 0; i < 3; i++) {
            int all = 0;
#pragma unroll
            for (int x = 0; x < kKeepWaves; x++) all += part[turn][x][i];
            /* the highest that as many reach; the one above it has fewer */
            if (all >= t.keep) cut = base | (uint32_t)(i + 1) << bit;
            else if (cut == (i ? base | (uint32_t)i << bit : base)) larger = all;
            exact |= all == t.keep;
            if (all <= t.keep) break;
        }
    }
    if (exact) {
        cut--;
        larger = t.keep;
    }
    const int ties = t.keep - larger;

    int sure = 0, equal = 0;
    rows([&](int, uint32_t k) {
        sure += k > cut;
        equal += k == cut && k != 0u;
    });
    sure = keep_wave_sum(sure);
    equal = keep_wave_sum(equal);
    __syncthreads();
    if (lane == 0) {
        part[0][wave][0] = sure;
        part_eq[wave] = equal;
    }
    __syncthreads();
    int at = 0, seen = 0;
#pragma unroll
    for (int x = 0; x < kKeepWaves; x++)
        if (x < wave) {
            at += part[0][x][0] + max(min(ties - seen, part_eq[x]), 0);
            seen += part_eq[x];
        }
    const unsigned long long below = (1ull << lane) - 1ull;
    const auto put = [&](int x, uint32_t k, float v) {
        const bool tie = k == cut && k != 0u;
        const unsigned long long tied = __ballot(tie);
        const bool stays = k > cut || (tie && seen + __popcll(tied & below) < ties);
        const unsigned long long staying = __ballot(stays);
        if (stays) {
            const int p = at + __popcll(staying & below);
            kept[p] = x + lane;
            to[p] = v;
        }
        at += __popcll(staying);
        seen += __popcll(tied);
    };
    if constexpr (R > 0) {
        constexpr int BATCH = 8;        /* loads on their way */
#pragma unroll
        for (int r = 0; r < R; r += BATCH) {
            float v[BATCH];
#pragma unroll
            for (int i = 0; i < BATCH; i++) v[i] = w[min(from + 64 * (r + i) + lane, len - 1)];
#pragma unroll
            for (int i = 0; i < BATCH; i++) put(from + 64 * (r + i), key[r + i], v[i]);
        }
    } else {
        for (int x = from; x < end; x += 64) {
            const float v = w[min(x + lane, len - 1)];
            put(x, key_of(v, x + lane), v);
        }
    }
}

/* ES: bytes of an element. */
template <int ES, int D>
__global__ __launch_bounds__(256) void sera_kv_move_kernel(kv_args a, evict_args t, int blocks) {
    constexpr int ROW = D * ES, LANES = ROW / 16, ROWS = 64 / LANES, N = 16 / ROWS;
    constexpr int DW = 4 * ES;                           /* dwords of a channel's 16 tokens */
    __shared__ uint32_t turn[2][DW][D];      /* of the waves that move V: a block, dword by dword of all channels */
    const int b = (int)(blockIdx.z * gridDim.y + blockIdx.y);
    if (b >= a.sequences) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int head = (int)blockIdx.x % a.kv_heads, block = ((int)blockIdx.x / a.kv_heads) * 2 + (wave >> 1);
    const bool is_v = wave & 1;
    if (block >= blocks) return;
    const int len = a.kv_len[b];
    if (len < 0 || len > a.max_kv) return;
    const int t0 = 16 * block, n = min(min(len, t.keep) - t0, 16), mask = (1 << a.page_shift) - 1;
    if (n <= 0) return;
    const int new_page = t.new_table[(size_t)b * t.new_stride + (t0 >> a.page_shift)];
    if (new_page < 0 || new_page >= a.pages) return;

    /* lane x (mod 16): the page and the place of token x */
    const int x = min(lane & 15, n - 1);
    const int pos = t.kept[((size_t)b * a.kv_heads + head) * t.keep + t0 + x];
    int page = a.table[(size_t)b * a.table_stride + (pos >> a.page_shift)];
    if (page < 0 || page >= a.pages) page = -1;
    if (len <= t.keep && __builtin_amdgcn_readfirstlane(page) == new_page) return;      /* in its place already */

    const size_t kv_bytes = (size_t)ROW << a.page_shift;
    const uint8_t *src = a.data + (size_t)head * a.head_bytes;
    uint8_t *dst = a.data + (size_t)new_page * a.page_bytes + (size_t)head * a.head_bytes;
    const int new_slot = t0 & mask;
    if (ES == 1 && lane < n) {
        const size_t off = 2 * kv_bytes + (((size_t)is_v << a.page_shift)) * 4;
        const float scale = page < 0 ? __builtin_nanf("")
                                     : *(const float *)(src + (size_t)page * a.page_bytes + off + 4 * (pos & mask));
        *(float *)(dst + off + 4 * (new_slot + lane)) = scale;
    }
    const uint32_t lost = ES == 2 ? 0x7e007e00u : 0u;        /* fp16 NaN; codes of a lost page have a NaN scale */
    if (!is_v) {
        const int off = lane % LANES * 16;
        move_u4 w[N];
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int y = i * ROWS + lane / LANES;
            const int p = __shfl(page, y, 64), at = __shfl(pos, y, 64) & mask;
            w[i] = move_u4{lost, lost, lost, lost};
            if (p >= 0) w[i] = *(const move_u4 *)(src + (size_t)p * a.page_bytes + (size_t)at * ROW + off);
        }
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int y = i * ROWS + lane / LANES;
            if (y < n) *(move_u4 *)(dst + (size_t)(new_slot + y) * ROW + off) = w[i];
        }
        return;
    }
    uint32_t w[D / 64][DW], (*const box)[D] = turn[wave >> 1];
#pragma unroll
    for (int i = 0; i < D / 64; i++)
#pragma unroll
        for (int k = 0; k < DW; k++) w[i][k] = 0u;
    int there = -1;                                      /* the position of the block in LDS */
#pragma unroll
    for (int y = 0; y < 16; y++) {
        const int p = __builtin_amdgcn_readlane(page, y), from = __builtin_amdgcn_readlane(pos, y), o = from & 15;
        if (y < n && from - o != there) {
            there = from - o;
            const uint8_t *block = src + (size_t)max(p, 0) * a.page_bytes + kv_bytes + (size_t)(there & mask) * ROW;
#pragma unroll
            for (int i = 0; i < D / 64; i++)
#pragma unroll
                for (int k = 0; k < ES; k++) {
                    move_u4 x = ((const move_u4 *)(block + (size_t)(64 * i + lane) * (16 * ES)))[k];
                    if (p < 0) x = move_u4{lost, lost, lost, lost};
#pragma unroll
                    for (int e = 0; e < 4; e++) box[4 * k + e][64 * i + lane] = x[e];
                }
            asm volatile("" ::: "memory");               /* the wave's own LDS, which it accesses in order */
        }
#pragma unroll
        for (int i = 0; i < D / 64; i++) {
            const uint32_t v = box[o * ES / 4][64 * i + lane] >> (o * ES % 4 * 8);
            w[i][y * ES / 4] |= (v & (ES == 2 ? 0xffffu : 0xffu)) << (y * ES % 4 * 8);
        }
        asm volatile("" ::: "memory");
    }
#pragma unroll
    for (int i = 0; i < D / 64; i++) {
        uint8_t *to = dst + kv_bytes + (size_t)new_slot * ROW + 16 * (64 * i + lane) * ES;
        if (n == 16) {
#pragma unroll
            for (int k = 0; k < ES; k++)
                ((move_u4 *)to)[k] = move_u4{w[i][4 * k], w[i][4 * k + 1], w[i][4 * k + 2], w[i][4 * k + 3]};
        } else {
#pragma unroll
            for (int y = 0; y < 16; y++) {
                const uint32_t v = w[i][y * ES / 4] >> (y * ES % 4 * 8);
                if (y < n) {
                    if (ES == 2) ((uint16_t *)to)[y] = (uint16_t)v;
                    else to[y] = (uint8_t)v;
                }
            }
        }
    }
}

/* Arguments are checked by the caller (sera_attn_runtime.hip). */
hipError_t sera_launch_kv_evict(uint32_t cache_type, int dim, const kv_args &a, const evict_args &t, hipStream_t s) {
    const int y = a.sequences < 32768 ? a.sequences : 32768;
    const unsigned z = (unsigned)((a.sequences + y - 1) / y);
    const dim3 heads((unsigned)a.kv_heads, (unsigned)y, z), threads(64 * kKeepWaves);
    if (a.max_kv <= 16 * 64 * kKeepWaves) hipLaunchKernelGGL(sera_kv_keep_kernel<16>, heads, threads, 0, s, a, t);
    else if (a.max_kv <= 32 * 64 * kKeepWaves) hipLaunchKernelGGL(sera_kv_keep_kernel<32>, heads, threads, 0, s, a, t);
    else if (a.max_kv <= 64 * 64 * kKeepWaves) hipLaunchKernelGGL(sera_kv_keep_kernel<64>, heads, threads, 0, s, a, t);
    else hipLaunchKernelGGL(sera_kv_keep_kernel<0>, heads, threads, 0, s, a, t);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const int most = t.keep < a.max_kv ? t.keep : a.max_kv, blocks = (most + 15) / 16;
    const dim3 grid((unsigned)(a.kv_heads * ((blocks + 1) / 2)), (unsigned)y, z);
    if (cache_type == SERA_KV_F16) {
        if (dim == 64) hipLaunchKernelGGL((sera_kv_move_kernel<2, 64>), grid, dim3(256), 0, s, a, t, blocks);
        else hipLaunchKernelGGL((sera_kv_move_kernel<2, 128>), grid, dim3(256), 0, s, a, t, blocks);
    } else {
        if (dim == 64) hipLaunchKernelGGL((sera_kv_move_kernel<1, 64>), grid, dim3(256), 0, s, a, t, blocks);
        else hipLaunchKernelGGL((sera_kv_move_kernel<1, 128>), grid, dim3(256), 0, s, a, t, blocks);
    }
    return hipGetLastError();
}
