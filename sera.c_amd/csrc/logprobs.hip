/*
 * logprobs.hip - log probabilities, entropy and the most likely tokens of
 * rows of logits, in one pass over them.
 *
 * With m the running maximum, s = sum e^(x - m) and t = sum e^(x - m) (x - m):
 *
 *   log p(x) = (x - m) - log s       H = log s - t / s
 *
 * A wave takes a piece of a row, 64 lanes x 16 bytes at a time. The top: a
 * wave holds candidates in LDS as 64-bit keys, the logit as a whole number of the same order
 * above the inverted id, so no two are alike and equal logits are in the order of
 * their ids. An element that is below the top-th candidate of the last cut is passed over, which is
 * a comparison of a lane's largest one for almost all; the others are
 * appended, and a full list is cut to the top again. The four lists of a workgroup
 * are cut to one; a row that is split over workgroups leaves (m, s, t) and a
 * list of each, which a second launch joins in the same way.
 */
#include "logprobs.h"
#include "sera_dpp.h"
#include "sera_launch.h"

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

namespace {

constexpr int kWaves = 4, kRoom = 256;             /* candidates of a wave */
constexpr float kLowest = -3.402823466e38f, kLog2E = 1.4426950408889634f;

typedef unsigned long long lp_key;

/* x as a whole number of the same order; at least 1 for all but a NaN. */
__device__ __forceinline__ uint32_t lp_order(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);      /* -0 becomes 0 */
    return x != x ? 0u : (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float lp_value(uint32_t o) {
    return __uint_as_float((o & 0x80000000u) ? o & 0x7fffffffu : ~o);
}

/* The value that a key's element has at least; below that of -inf lie only prefixes of it. */
__device__ __forceinline__ float lp_least_value(lp_key k) {
    const uint32_t o = (uint32_t)(k >> 32);
    return o < 0x00800000u ? -INFINITY : lp_value(o);
}

/* Running sums of a lane. m is not -inf. */
struct lp_sum {
    float m, s, t;
};

__device__ __forceinline__ void lp_join(lp_sum &a, const lp_sum &b) {
    const float m = fmaxf(a.m, b.m);
    /* differences beyond 200 have no weight left; held there, no product with 0 is undefined */
    const float da = fmaxf(a.m - m, -200.0f), db = fmaxf(b.m - m, -200.0f);
    const float fa = __builtin_amdgcn_exp2f(da * kLog2E), fb = __builtin_amdgcn_exp2f(db * kLog2E);
    a.t = fa * (a.t + da * a.s) + fb * (b.t + db * b.s);
    a.s = fa * a.s + fb * b.s;
    a.m = m;
}

template <int OFF>
__device__ __forceinline__ void lp_join_lane(lp_sum &a) {
    lp_sum b;
    b.m = xor_partner<OFF>(a.m);
    b.s = xor_partner<OFF>(a.s);
    b.t = xor_partner<OFF>(a.t);
    lp_join(a, b);
}
__device__ __forceinline__ void lp_join_wave(lp_sum &a) {
    lp_join_lane<1>(a);
    lp_join_lane<2>(a);
    lp_join_lane<4>(a);
    lp_join_lane<8>(a);
    lp_join_lane<16>(a);
    lp_join_lane<32>(a);
}

/* The candidates of a wave: n keys in LDS (wave-uniform), of which those below `least` need not be looked at. */
struct lp_list {
    lp_key *keys;
    int n, top;
    lp_key least;

    /* The `top` largest of the n keys to the front. */
    __device__ __forceinline__ void cut(int lane) {
        if (n <= top) return;
        lp_key k[kRoom / 64];
        asm volatile("" ::: "memory");          /* the wave's own LDS, which it accesses in order */
#pragma unroll
        for (int i = 0; i < kRoom / 64; i++) k[i] = 64 * i + lane < n ? keys[64 * i + lane] : 0;
        /* the top-th largest, bit by bit; all bits of keys that are never alike: as soon as exactly `top` are as large,
         * the rest of the bits do not matter */
        lp_key least_of = 0;
        for (int bit = 63; bit >= 0; bit--) {
            const lp_key at = least_of | 1ull << bit;
            int count = 0;
#pragma unroll
            for (int i = 0; i < kRoom / 64; i++) count += __popcll(__ballot(k[i] >= at));
            if (count >= top) least_of = at;
            if (count == top) break;
        }
        int to = 0;
#pragma unroll
        for (int i = 0; i < kRoom / 64; i++) {
            const bool stays = k[i] >= least_of && k[i] != 0;
            const lp_key all = __ballot(stays);
            if (stays) keys[to + __popcll(all & ((1ull << lane) - 1))] = k[i];
            to += __popcll(all);
        }
        asm volatile("" ::: "memory");
        n = to;
        least = least_of;
    }

    /* Those of the lanes' keys that are not below the cut. 0: none. */
    __device__ __forceinline__ void add(lp_key key, int lane) {
        lp_key all = __ballot(key != 0 && key >= least);
        if (!all) return;
        if (n + __popcll(all) > kRoom) {
            cut(lane);
            all = __ballot(key != 0 && key >= least);
        }
        if (key != 0 && key >= least) keys[n + __popcll(all & ((1ull << lane) - 1))] = key;
        n += __popcll(all);
        asm volatile("" ::: "memory");
    }

    /* In falling order: the place of each (one a lane, n <= 64). */
    __device__ __forceinline__ int place(lp_key mine) const {
        int above = 0;
        for (int i = 0; i < n; i++) above += keys[i] > mine;
        return above;
    }
};

template <typename T>
__device__ __forceinline__ float lp_f32(T x) { return (float)x; }

}  // namespace

/* Joins the waves of a workgroup, and its lists into that of wave 0. */
__device__ __forceinline__ void lp_join_group(lp_sum &a, lp_list &list, lp_key (*keys)[kRoom], float (*sums)[3],
                                              int *counts, int lane, int wave) {
    lp_join_wave(a);
    list.cut(lane);
    if (lane == 0) {
        sums[wave][0] = a.m;
        sums[wave][1] = a.s;
        sums[wave][2] = a.t;
        counts[wave] = list.n;
    }
    __syncthreads();
    if (wave) return;
    for (int w = 1; w < kWaves; w++) {
        const lp_sum b = {sums[w][0], sums[w][1], sums[w][2]};
        lp_join(a, b);
        list.add(lane < counts[w] ? keys[w][lane] : 0, lane);
    }
    list.cut(lane);
}

/* What is asked of a row, from its sums and its list, by wave 0. */
template <typename T>
__device__ __forceinline__ void lp_finish(const logprobs_args &p, int64_t row, const lp_sum &a, const lp_list &list,
                                          int lane) {
    const T *x = (const T *)p.logits + row * p.stride;
    const bool fine = a.s > 0.0f && a.s < INFINITY;
    const float nan = __builtin_nanf(""), log_s = logf(a.s);
    for (int i = lane; i < p.per_row; i += 64) {
        const int token = p.tokens[row * p.per_row + i];
        float y = nan;
        if (fine && token >= 0 && token < p.vocab) y = (lp_f32(x[token]) - a.m) - log_s;
        p.token_logprobs[row * p.per_row + i] = y;
    }
    if (p.entropy && lane == 0) p.entropy[row] = fine ? log_s - a.t / a.s : nan;
    if (lane < p.top) {
        const lp_key mine = lane < list.n ? list.keys[lane] : 0;
        const int at = fine && lane < list.n ? list.place(mine) : lane;
        p.top_ids[row * p.top + at] = fine ? (int)~(uint32_t)mine : -1;
        p.top_logprobs[row * p.top + at] = fine ? (lp_value((uint32_t)(mine >> 32)) - a.m) - log_s : nan;
    }
}

template <typename T>
__global__ __launch_bounds__(64 * kWaves) void sera_logprobs_kernel(logprobs_args p) {
    constexpr int VEC = 16 / (int)sizeof(T), UNROLL = 4;
    struct __attribute__((aligned(16))) vec { T v[VEC]; };
    __shared__ lp_key keys[kWaves][kRoom];
    __shared__ float sums[kWaves][3];
    __shared__ int counts[kWaves];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t row = blockIdx.x;
    const int split = blockIdx.y;
    const T *x = (const T *)p.logits + row * p.stride;
    /* 16-byte units of the row, from the one that holds its first element; the first and the last may be partly its */
    const int skip = (int)((uintptr_t)x & 15u) / (int)sizeof(T);
    const int units = (p.vocab + skip + VEC - 1) / VEC, pieces = p.splits * kWaves;
    const int per = (units + pieces - 1) / pieces, u0 = (split * kWaves + wave) * per, u1 = min(u0 + per, units);

    lp_list list;
    list.keys = keys[wave];
    list.n = 0;
    list.top = p.top;
    list.least = 0;
    float least_value = -INFINITY;
    lp_sum a = {kLowest, 0.0f, 0.0f};
    const auto load = [&](int u, vec *w) {
        if (u * VEC >= skip && u + 64 * UNROLL <= u1 && (u + 64 * UNROLL) * VEC - skip <= p.vocab) {
#pragma unroll
            for (int i = 0; i < UNROLL; i++) w[i] = *(const vec *)(x + ((u + 64 * i + lane) * VEC - skip));
        } else {
#pragma unroll
            for (int i = 0; i < UNROLL; i++)
#pragma unroll
                for (int e = 0; e < VEC; e++) {
                    const int at = u + 64 * i + lane, id = at * VEC - skip + e;
                    w[i].v[e] = at < u1 && id >= 0 && id < p.vocab ? x[id] : (T)-INFINITY;
                }
        }
    };
    for (int u = u0; u < u1; u += 64 * UNROLL) {
        vec in[UNROLL];
        load(u, in);
        float y[UNROLL][VEC], top = -INFINITY;
#pragma unroll
        for (int i = 0; i < UNROLL; i++)
#pragma unroll
            for (int e = 0; e < VEC; e++) y[i][e] = lp_f32(in[i].v[e]);
#pragma unroll
        for (int i = 0; i < UNROLL; i++)
#pragma unroll
            for (int e = 0; e < VEC; e++) top = fmaxf(top, y[i][e]);
        if (__ballot(top > a.m)) {
            const float m = fmaxf(a.m, top), d = fmaxf(a.m - m, -200.0f), f = __builtin_amdgcn_exp2f(d * kLog2E);
            a.t = f * (a.t + d * a.s);
            a.s *= f;
            a.m = m;
        }
#pragma unroll
        for (int i = 0; i < UNROLL; i++)
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                const float d = y[i][e] - a.m, w = __builtin_amdgcn_exp2f(d * kLog2E);
                a.s += w;
                a.t = fmaf(w, fmaxf(d, -200.0f), a.t);
            }
        if (p.top && __ballot(top >= least_value)) {
#pragma unroll
            for (int i = 0; i < UNROLL; i++)
#pragma unroll
                for (int e = 0; e < VEC; e++) {
                    const int at = u + 64 * i + lane, id = at * VEC - skip + e;
                    const bool in = at < u1 && id >= 0 && id < p.vocab;
                    if (__ballot(in && y[i][e] >= least_value)) {
                        list.add(in ? (lp_key)lp_order(y[i][e]) << 32 | (uint32_t)~id : 0, lane);
                        least_value = lp_least_value(list.least);
                    }
                }
        }
    }
    lp_join_group(a, list, keys, sums, counts, lane, wave);
    if (wave) return;
    if (p.splits == 1) return lp_finish<T>(p, row, a, list, lane);
    const size_t part = (size_t)row * p.splits + split;
    float *const ws = p.workspace;
    if (lane == 0) {
        ws[3 * part] = a.m;
        ws[3 * part + 1] = a.s;
        ws[3 * part + 2] = a.t;
    }
    if (lane < p.top)
        ((lp_key *)(ws + p.sums))[part * p.top + lane] = lane < list.n ? list.keys[lane] : 0;
}

template <typename T>
__global__ __launch_bounds__(64 * kWaves) void sera_logprobs_join_kernel(logprobs_args p) {
    __shared__ lp_key keys[kWaves][kRoom];
    __shared__ float sums[kWaves][3];
    __shared__ int counts[kWaves];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t row = blockIdx.x;
    const float *const ws = p.workspace + 3 * (size_t)row * p.splits;
    const lp_key *const parts = (const lp_key *)(p.workspace + p.sums) + (size_t)row * p.splits * p.top;
    lp_list list;
    list.keys = keys[wave];
    list.n = 0;
    list.top = p.top;
    list.least = 0;
    lp_sum a = {kLowest, 0.0f, 0.0f};
    for (int i = 64 * wave + lane; i < p.splits; i += 64 * kWaves) {
        const lp_sum b = {ws[3 * i], ws[3 * i + 1], ws[3 * i + 2]};
        lp_join(a, b);
    }
    for (int i = 64 * wave; i < p.splits * p.top; i += 64 * kWaves)
        list.add(i + lane < p.splits * p.top ? parts[i + lane] : 0, lane);
    lp_join_group(a, list, keys, sums, counts, lane, wave);
    if (wave == 0) lp_finish<T>(p, row, a, list, lane);
}

namespace {

constexpr int kLeastUnits = 256;      /* 16-byte units of a workgroup, at least */

template <typename T>
hipError_t lp_go(const logprobs_args &p, hipStream_t s) {
    hipLaunchKernelGGL(sera_logprobs_kernel<T>, dim3((unsigned)p.rows, (unsigned)p.splits), dim3(64 * kWaves), 0, s, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.splits == 1) return e;
    hipLaunchKernelGGL(sera_logprobs_join_kernel<T>, dim3((unsigned)p.rows), dim3(64 * kWaves), 0, s, p);
    return hipGetLastError();
}

}  // namespace

/* Workgroups of a row. */
int sera_logprobs_splits(int rows, int vocab, int cus) {
    const int64_t most = vocab / 4 / kLeastUnits, want = 2ll * cus / rows;
    const int64_t n = most < want ? most : want;
    return n < 1 ? 1 : n > 128 ? 128 : (int)n;
}

/* Floats of the partial sums (even, the lists lie behind them), and bytes of all. */
size_t sera_logprobs_sums(int rows, int splits) { return ((size_t)rows * splits * 3 + 3) & ~(size_t)3; }

hipError_t sera_launch_logprobs(uint32_t type, const logprobs_args &p, hipStream_t s) {
    if (type == 0u) return lp_go<float>(p, s);
    if (type == 1u) return lp_go<_Float16>(p, s);
    return lp_go<__bf16>(p, s);
}
