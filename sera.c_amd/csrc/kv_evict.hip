/*
 * kv_evict.hip - shortening of cached sequences: which positions of a kv head
 * stay, and their move to new pages.
 *
 * Choice: a workgroup for each sequence and kv head. Weights become whole numbers
 * of the same order; the smallest one that stays (of the middle positions) is built bit by
 * bit, each bit by counting how many are as large. Then each wave walks a run
 * of positions of its own and writes what stays behind what the runs before it
 * keep, which a count of each run says.
 *
 * Move: a wave for K or V of 16 new places of a head. A K row is a run of
 * bytes; a V token is an element of each channel's 16.
 */
#include "attn_common.h"
#include "sera_launch.h"

namespace {

constexpr int kKeepWaves = 16;

/* A weight as a whole number of the same order, at least 1; NaN is 0. */
__device__ __forceinline__ uint32_t keep_key(float w) {
    const uint32_t u = __float_as_uint(w + 0.0f);       /* -0 becomes 0 */
    return w != w ? 0u : (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

typedef uint32_t move_u4 __attribute__((ext_vector_type(4)));

}  // namespace

__global__ __launch_bounds__(64 * kKeepWaves) void sera_kv_keep_kernel(kv_args a, evict_args t) {
    __shared__ int part[2][kKeepWaves], part_eq[kKeepWaves];
    const int b = (int)(blockIdx.z * gridDim.y + blockIdx.y), head = (int)blockIdx.x;
    if (b >= a.sequences) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int len = a.kv_len[b];
    const bool bad = len < 0 || len > a.max_kv, all = !bad && len <= t.keep;
    const size_t place = (size_t)b * a.kv_heads + head;
    int *kept = t.kept + place * t.keep;
    const float *w = t.weights + place * t.weights_stride;
    float *to = t.new_weights + place * t.weights_stride;
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
    const int lo = t.sinks, hi = len - t.recent, want = t.keep - t.sinks - t.recent;     /* hi - lo > want */

    /* The want-th largest key of the middle (all ones if none is wanted), and how many are larger. */
    uint32_t least = want > 0 ? 0u : 0xffffffffu;
    int larger = 0, turn = 0;
    const auto count_from = [&](uint32_t key) {
        int n = 0;
        for (int x = lo + 64 * wave; x < hi; x += 64 * kKeepWaves)
            n += __popcll(__ballot(x + lane < hi && keep_key(w[min(x + lane, hi - 1)]) >= key));
        turn ^= 1;
        if (lane == 0) part[turn][wave] = n;
        __syncthreads();
        n = 0;
#pragma unroll
        for (int x = 0; x < kKeepWaves; x++) n += part[turn][x];
        return n;
    };
    if (want > 0) {
        for (int bit = 31; bit >= 0; bit--) {
            const uint32_t key = least | 1u << bit;
            const int n = count_from(key);
            if (n >= want) least = key;
            else larger = n;
        }
    }
    const int ties = want - larger;      /* of those equal to `least`, the first ones */

    /* Each wave's run of positions: what it keeps for sure, and its ties. */
    const int run = ((len + kKeepWaves - 1) / kKeepWaves + 63) & ~63, from = min(wave * run, len), end = min(from + run, len);
    int sure = 0, equal = 0;
    for (int x = from; x < end; x += 64) {
        const int j = x + lane;
        const bool middle = j >= lo && j < hi;
        const uint32_t key = j < end ? keep_key(w[j]) : 0u;
        sure += __popcll(__ballot(j < end && (!middle || (want > 0 && key > least))));
        equal += __popcll(__ballot(j < end && middle && want > 0 && key == least));
    }
    __syncthreads();
    if (lane == 0) {
        part[0][wave] = sure;
        part_eq[wave] = equal;
    }
    __syncthreads();
    int at = 0, seen = 0;
    for (int x = 0; x < wave; x++) {
        at += part[0][x] + max(min(ties - seen, part_eq[x]), 0);
        seen += part_eq[x];
    }
    for (int x = from; x < end; x += 64) {
        const int j = x + lane;
        const bool middle = j >= lo && j < hi;
        const float value = j < end ? w[j] : 0.0f;
        const uint32_t key = keep_key(value);
        const unsigned long long below = (1ull << lane) - 1ull;
        const bool tie = j < end && middle && want > 0 && key == least;
        const unsigned long long tied = __ballot(tie);
        const bool stays = j < end && (!middle || (want > 0 && key > least) ||
                                       (tie && seen + __popcll(tied & below) < ties));
        const unsigned long long staying = __ballot(stays);
        if (stays) {
            const int p = at + __popcll(staying & below);
            kept[p] = j;
            to[p] = value;
        }
        at += __popcll(staying);
        seen += __popcll(tied);
    }
}

/* ES: bytes of an element. */
template <int ES, int D>
__global__ __launch_bounds__(256) void sera_kv_move_kernel(kv_args a, evict_args t, int blocks) {
    constexpr int ROW = D * ES, LANES = ROW / 16, ROWS = 64 / LANES, N = 16 / ROWS;
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
    for (int d = lane; d < D; d += 64) {
        uint32_t w[4 * ES];
#pragma unroll
        for (int i = 0; i < 4 * ES; i++) w[i] = 0u;
#pragma unroll
        for (int y = 0; y < 16; y++) {
            const int p = __builtin_amdgcn_readlane(page, y), at = __builtin_amdgcn_readlane(pos, y) & mask;
            uint32_t v = lost & (ES == 2 ? 0xffffu : 0xffu);
            if (p >= 0) {
                const uint8_t *from = src + (size_t)p * a.page_bytes + kv_bytes + (size_t)(at & ~15) * ROW +
                                      (16 * d + (at & 15)) * ES;
                v = ES == 2 ? (uint32_t)*(const uint16_t *)from : (uint32_t)*from;
            }
            w[y * ES / 4] |= v << (y * ES % 4 * 8);
        }
        uint8_t *to = dst + kv_bytes + (size_t)new_slot * ROW + 16 * d * ES;
        if (n == 16) {
#pragma unroll
            for (int i = 0; i < ES; i++) ((move_u4 *)to)[i] = move_u4{w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]};
        } else {
#pragma unroll
            for (int y = 0; y < 16; y++) {
                const uint32_t v = w[y * ES / 4] >> (y * ES % 4 * 8);
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
    hipLaunchKernelGGL(sera_kv_keep_kernel, dim3((unsigned)a.kv_heads, (unsigned)y, z), dim3(64 * kKeepWaves), 0, s, a, t);
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
