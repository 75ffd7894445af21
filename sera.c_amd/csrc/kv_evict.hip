/*
 * kv_evict.hip - shortening of cached sequences: which positions of a kv head stay, and their move to new pages.
 *
 * Choice: a workgroup for each sequence and kv head. Weights become whole numbers of the same order; the smallest one
 * that stays is built of four digits of 8 bits, each from counts in LDS of how many have which. Then each wave walks
 * a run of positions of its own, held in registers up to 24576 positions, and writes what stays behind what the runs
 * before it keep, which a count of each run says.
 *
 * Move: a wave for K or V of 16 new places of a head. A K row is a run of bytes. A V token is an element of each
 * channel's 16, so whole blocks of 16 old tokens come as they lie, go through LDS, and the tokens that stay are
 * picked from there.
 *
 * The move is bound by memory, the choice by the latency of its steps. 64 sequences of 8192 positions to half (8 kv
 * heads, 128 channels, fp16 cache): 21 us and 533 us, for 2.7 GB the rate of a copy; of V's blocks of 16 tokens
 * hardly one is without any that stays, so V is read whole. 24 sequences of up to 3001 (8-bit cache): 8.3 us and 27
 * us. The choice alone, of one sequence: 3001 positions 7.6 us, 16000 19 us, 200000 286 us.
 */
#include "attn_common.h"
#include "sera_dpp.h"
#include "sera_launch.h"

namespace {

constexpr uint32_t kProtected = 0xffffffffu;            /* more than any weight's number */

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

/* W waves. R: 64-position rows of a wave's run that are held in registers (the run fits); 0: they are read again each
 * time. */
template <int W, int R>
__global__ __launch_bounds__(64 * W) void sera_kv_keep_kernel(kv_args a, evict_args t) {
    __shared__ int counts[4][256], part[W], part_eq[W];
    const int b = (int)(blockIdx.z * gridDim.y + blockIdx.y), head = (int)blockIdx.x;
    if (b >= a.sequences) return;
    constexpr int BATCH = R == 0 || R > 8 ? 8 : R;      /* loads on their way */
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int len = a.kv_len[b];
    const bool bad = len < 0 || len > a.max_kv, all = !bad && len <= t.keep;
    const size_t place = (size_t)b * a.kv_heads + head;
    int *__restrict__ kept = t.kept + place * t.keep;
    const float *__restrict__ w = t.weights + place * t.weights_stride;
    float *__restrict__ to = t.new_weights + place * t.weights_stride;
    const int count = bad ? 0 : min(len, t.keep);
    if (head == 0 && tid == 0) t.new_len[b] = bad ? -1 : count;
    for (int x = count + tid; x < t.keep; x += 64 * W) kept[x] = -1;
    if (bad) return;
    if (all) {
        for (int x = tid; x < len; x += 64 * W) {
            kept[x] = x;
            to[x] = w[x];
        }
        return;
    }
    const int lo = t.sinks, hi = len - t.recent;
    for (int x = tid; x < 4 * 256; x += 64 * W) counts[x >> 8][x & 255] = 0;
    __syncthreads();

    /* A wave's run of positions. Those outside the middle count as the largest there are, places behind the run as
     * none. */
    const int run = ((len + W - 1) / W + 63) & ~63;
    const int from = min(wave * run, len), end = min(from + run, len);
    uint32_t key[R ? R : 1];
    const auto key_of = [&](float v, int j) { return j >= end ? 0u : j < lo || j >= hi ? kProtected : keep_key(v); };
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
            for (int x = from; x < end; x += 64 * BATCH) {
                float v[BATCH];
#pragma unroll
                for (int i = 0; i < BATCH; i++) v[i] = w[min(x + 64 * i + lane, len - 1)];
#pragma unroll
                for (int i = 0; i < BATCH; i++) each(x + 64 * i, key_of(v[i], x + 64 * i + lane));
            }
        }
    };

    /* Of the middle `ties` stay: those above `cut`, and the first of those equal to it. The cut is the ties-th
     * largest, built of four digits: how many have each digit behind those found so far, and which one the ties-th
     * has. As soon as all of a digit stay, the cut is the number below. */
    int ties = t.keep - t.sinks - t.recent;
    uint32_t cut = ties ? 0u : kProtected - 1u;
    for (int place = 3; place >= 0 && ties; place--) {
        int *const count = counts[place];
        rows([&](int, uint32_t k) {
            const bool in = k != 0u && k != kProtected && (place == 3 || (k ^ cut) >> (8 * place + 8) == 0u);
            const uint64_t all = __ballot(in);
            if (!all) return;
            const uint32_t digit = k >> (8 * place) & 255u;
            const uint32_t one = __builtin_amdgcn_readlane(digit, __builtin_ctzll(all));
            if (__ballot(in && digit != one) == 0) {            /* equal weights would queue for one counter */
                if (lane == 0) atomicAdd(&count[one], __popcll(all));
            } else if (in) {
                atomicAdd(&count[digit], 1);
            }
        });
        __syncthreads();
        /* A lane has four digits, the highest lane the highest. */
        int n[4], above = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) above += n[i] = count[4 * lane + i];
        int upto = above;                                       /* of this lane and those over it */
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int x = __shfl_down(upto, o, 64);
            upto += lane + o < 64 ? x : 0;
        }
        above = upto - above;
        int digit = -1, over = 0, same = 0;
#pragma unroll
        for (int i = 3; i >= 0; i--) {
            if (above < ties && ties <= above + n[i]) digit = 4 * lane + i, over = above, same = n[i];
            above += n[i];
        }
        const int has = __builtin_ctzll(__ballot(digit >= 0));  /* one lane has: more than `ties` are in the middle */
        cut |= (uint32_t)__builtin_amdgcn_readlane(digit, has) << (8 * place);
        ties -= __builtin_amdgcn_readlane(over, has);
        if (ties == __builtin_amdgcn_readlane(same, has)) {
            cut--;
            ties = 0;
        }
    }

    int sure = 0, equal = 0;
    rows([&](int, uint32_t k) {
        sure += k > cut;
        equal += k == cut && k != 0u;
    });
    sure = keep_wave_sum(sure);
    equal = keep_wave_sum(equal);
    if (lane == 0) {
        part[wave] = sure;
        part_eq[wave] = equal;
    }
    __syncthreads();
    int at = 0, seen = 0;
#pragma unroll
    for (int x = 0; x < W; x++)
        if (x < wave) {
            at += part[x] + max(min(ties - seen, part_eq[x]), 0);
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
#pragma unroll
        for (int r = 0; r < R; r += BATCH) {
            float v[BATCH];
#pragma unroll
            for (int i = 0; i < BATCH; i++) v[i] = w[min(from + 64 * (r + i) + lane, len - 1)];
#pragma unroll
            for (int i = 0; i < BATCH; i++) put(from + 64 * (r + i), key[r + i], v[i]);
        }
    } else {
        for (int x = from; x < end; x += 64 * BATCH) {
            float v[BATCH];
#pragma unroll
            for (int i = 0; i < BATCH; i++) v[i] = w[min(x + 64 * i + lane, len - 1)];
#pragma unroll
            for (int i = 0; i < BATCH; i++) put(x + 64 * i, key_of(v[i], x + 64 * i + lane), v[i]);
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
    const dim3 heads((unsigned)a.kv_heads, (unsigned)y, z);
    /* Eight waves for short sequences, where more of them only wait for each other (24 of 3001 positions 8.3 us, 8.4 with
     * sixteen, 10.6 with four), then sixteen (64 of 8192: 20.9 us, 22.1 with eight; one of 16000: 18.8 and 23.4), and
     * beyond what those hold as well, where the weights are read up to six times, for four digits, the counts and the
     * places (one of 65536: 83 us, 123 with eight; of 200000: 286 and 434). The form goes by the bound, as the lengths
     * are the device's: 24 of 3001 take 13.5 us with a bound of 16000, 13.2 with one of 131072. */
#define SERA_KEEP(W, R) hipLaunchKernelGGL((sera_kv_keep_kernel<W, R>), heads, dim3(64 * W), 0, s, a, t)
    if (a.max_kv <= 8 * 64 * 8) SERA_KEEP(8, 8);
    else if (a.max_kv <= 8 * 64 * 16) SERA_KEEP(16, 8);
    else if (a.max_kv <= 16 * 64 * 16) SERA_KEEP(16, 16);
    else if (a.max_kv <= 24 * 64 * 16) SERA_KEEP(16, 24);
    else SERA_KEEP(16, 0);
#undef SERA_KEEP
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
