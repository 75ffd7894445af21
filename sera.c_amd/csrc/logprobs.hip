/*
 * logprobs.hip - log probabilities, entropy and the most likely tokens of rows of logits, in one pass over them.
 *
 * With m the running maximum, s = sum e^(x - m) and t = sum e^(x - m) (x - m):
 *
 *   log p(x) = (x - m) - log s       H = log s - t / s
 *
 * (x log2(e) - m log2(e) in one instruction instead of a difference and a product would leave an error of m's size:
 * exponents of 2^20 and more come out wrong.)
 *
 * A wave takes a piece of a row, 16 elements of a lane at a time. The top: a wave holds candidates in LDS as 64-bit
 * keys, the logit as a whole number of the same order above the inverted id, so no two are alike and equal logits are
 * in the order of their ids. The workgroup keeps the maximum of each lane number over its waves: the top-th largest
 * of these 64 bounds the top from below, and what is not below it has to be looked at. For almost all elements that
 * is one comparison of the largest of 16. A step that has such elements reads them once more, out of the cache, so
 * that the many others keep no registers for it. A full list is cut to its top, and so are at the end the four lists
 * of a workgroup to one; a row that is split over workgroups leaves (m, s, t) and a list of each, which a second
 * launch joins in the same way.
 *
 * Bound by reading the logits, and of 16-bit ones by the vector instructions (8 an element and an exponential). 2047
 * rows of 151937 bf16 logits: 120 us without a top (5.2 TB/s, what a copy reaches), 130 us with the top 8; 1008 rows
 * of 151936 fp32 logits with the top 8: 115 us (5.3 TB/s). 16 rows: 11 + 4 us, 1 row: 8.5 + 6 us, which is latency. A
 * long top of short rows costs more than the rows, as nearly every step has some of it: the top 64 of 538 rows of
 * 19950 54 us, the top 5 18 us, none 11 us. A threshold of each wave by itself, its list's top-th, made the first 250
 * us: four times as many steps had something to look at.
 */
#include "logprobs.h"
#include "../../include/sera_logprobs.h"
#include "sera_dpp.h"
#include "sera_launch.h"

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

namespace {

constexpr int kWaves = 4, kRoom = 256;             /* candidates of a wave */
constexpr int kMostSplits = 64;                    /* of a row */
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
/* A value that is less than all of this order and more (-0 is no less than 0); -inf below those of numbers. */
__device__ __forceinline__ float lp_below(uint32_t o) {
    return o < 0x00800001u ? -INFINITY : lp_value(o - (o == 0x80000000u ? 2 : 1));
}

/* Running sums of a lane, in 64 bits (which take 16 elements' at a time): a token that stands out has nearly all of
 * s, and the entropy is what the others add to it. m is not -inf. */
struct lp_sum {
    float m;
    double s, t;
};

/* The sums around a maximum m that is as large or larger. */
__device__ __forceinline__ void lp_raise(lp_sum &a, float m) {
    const float d = fmaxf(a.m - m, -200.0f);  /* beyond, no weight is left; held, no product with 0 is undefined */
    const double f = __builtin_amdgcn_exp2f(d * kLog2E);
    a.t = f * fma((double)d, a.s, a.t);
    a.s *= f;
    a.m = m;
}
__device__ __forceinline__ void lp_join(lp_sum &a, lp_sum b) {
    const float m = fmaxf(a.m, b.m);
    lp_raise(a, m);
    lp_raise(b, m);
    a.s += b.s;
    a.t += b.t;
}

template <int OFF>
__device__ __forceinline__ double lp_partner(double x) {
    return __hiloint2double(__float_as_int(xor_partner<OFF>(__int_as_float(__double2hiint(x)))),
                            __float_as_int(xor_partner<OFF>(__int_as_float(__double2loint(x)))));
}
template <int OFF>
__device__ __forceinline__ void lp_join_lane(lp_sum &a) {
    lp_sum b;
    b.m = xor_partner<OFF>(a.m);
    b.s = lp_partner<OFF>(a.s);
    b.t = lp_partner<OFF>(a.t);
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

/* The bits that any lane has, wave-uniform. */
__device__ __forceinline__ uint32_t lp_any(uint32_t x) {
    int y = (int)x;
    y |= xor_partner<1>(y);
    y |= xor_partner<2>(y);
    y |= xor_partner<4>(y);
    y |= xor_partner<8>(y);
    y |= xor_partner<16>(y);
    y |= xor_partner<32>(y);
    return (uint32_t)__builtin_amdgcn_readfirstlane(y);
}

/* The n-th largest of a wave's numbers, or one between it and the next smaller (so as many are as large); if there
 * are fewer than n above 0, one that those are not below. Two bits at a time, as a bit's latency is a comparison, a
 * count and a branch, and only from the first to the last bit in which those above 0 differ (of the logits that may
 * be in a top few do, and the low ones of bf16 never). *larger: how many are over it, if it is the number itself. */
template <int N>
__device__ __forceinline__ uint32_t lp_nth(const uint32_t (&k)[N], int n, bool *exact, int *larger) {
    uint32_t any = 0, lacks = 0;
#pragma unroll
    for (int i = 0; i < N; i++) {
        any |= k[i];
        lacks |= k[i] ? ~k[i] : 0u;
    }
    any = lp_any(any);
    const uint32_t differ = any & lp_any(lacks), common = any & ~differ;
    *larger = 0;
    *exact = false;
    if (!differ) return common;
    int bit = (31 - __builtin_clz(differ)) & ~1;
    uint32_t at = common & ~((4u << bit) - 1u);
    for (;; bit -= 2) {
        int count[3] = {0, 0, 0};
#pragma unroll
        for (int j = 0; j < 3; j++)
#pragma unroll
            for (int i = 0; i < N; i++) count[j] += __popcll(__ballot(k[i] >= (at | (uint32_t)(j + 1) << bit)));
        const int up = (count[0] >= n) + (count[1] >= n) + (count[2] >= n);
        *larger = up == 0 ? count[0] : up == 1 ? count[1] : up == 2 ? count[2] : *larger;
        at |= (uint32_t)up << bit;
        if (count[0] == n || count[1] == n || count[2] == n) {
            *exact = true;
            return at;
        }
        const uint32_t rest = (1u << bit) - 1u;
        if (!(differ & rest)) return at | (common & rest);
    }
}

/* The same of 64-bit numbers. */
template <int N>
__device__ __forceinline__ lp_key lp_nth_key(const lp_key (&k)[N], int n) {
    uint32_t part[N];
    bool exact;
    int larger;
#pragma unroll
    for (int i = 0; i < N; i++) part[i] = (uint32_t)(k[i] >> 32);
    const uint32_t high = lp_nth(part, n, &exact, &larger);
    if (exact || high == 0) return (lp_key)high << 32;
#pragma unroll
    for (int i = 0; i < N; i++) part[i] = (uint32_t)(k[i] >> 32) == high ? (uint32_t)k[i] : 0u;
    return (lp_key)high << 32 | lp_nth(part, n - larger, &exact, &larger);
}

/* The candidates of a wave: n keys in LDS (wave-uniform), of which those below `least` need not be looked at. */
struct lp_list {
    lp_key *keys;
    int n, top;
    lp_key least;

    /* The `top` largest of the n <= 64 N keys to the front. */
    template <int N>
    __device__ __forceinline__ void cut_of(int lane) {
        lp_key k[N];
        asm volatile("" ::: "memory");          /* the wave's own LDS, which it accesses in order */
#pragma unroll
        for (int i = 0; i < N; i++) k[i] = 64 * i + lane < n ? keys[64 * i + lane] : 0;
        least = lp_nth_key(k, top);
        n = 0;
#pragma unroll
        for (int i = 0; i < N; i++) put(k[i], k[i] >= least && k[i] != 0, lane);
    }
    __device__ __forceinline__ void cut(int lane) {
        if (n <= top) return;
        if (n <= 128) cut_of<2>(lane);
        else cut_of<kRoom / 64>(lane);
    }

    /* The keys of some lanes behind the others; there is room. */
    __device__ __forceinline__ void put(lp_key key, bool in, int lane) {
        const lp_key all = __ballot(in);
        if (in) keys[n + __popcll(all & ((1ull << lane) - 1))] = key;
        n += __popcll(all);
        asm volatile("" ::: "memory");
    }

    /* In falling order: the place of each (one a lane, n <= 64). */
    __device__ __forceinline__ int place(lp_key mine) const {
        int above = 0;
#pragma unroll 8
        for (int i = 0; i < n; i++) above += keys[i] > mine;
        return above;
    }
};

template <typename T>
__device__ __forceinline__ float lp_f32(T x) { return (float)x; }

/* 16 bytes of a row, kept as words so that nothing waits for them before their elements are wanted. */
typedef uint32_t lp_words __attribute__((ext_vector_type(4)));
typedef const lp_words __attribute__((address_space(1))) *lp_global;
union lp_unit {
    lp_words words;
    uint32_t word[4];
};
template <typename T>
__device__ __forceinline__ float lp_element(const lp_unit &u, int e) {
    constexpr int PER = 4 / (int)sizeof(T), BITS = 8 * (int)sizeof(T);
    const uint32_t bits = u.word[e / PER] >> BITS * (e % PER);
    T x;
    __builtin_memcpy(&x, &bits, sizeof(T));
    return lp_f32(x);
}
/* What is read of a row that has no whole unit. */
__device__ const lp_words lp_no_unit = {0u, 0u, 0u, 0u};

}  // namespace

/* Joins the waves of a workgroup: the sums for all of them, the lists into that of wave 0. */
__device__ __forceinline__ void lp_join_group(lp_sum &a, lp_list &list, lp_key (*keys)[kRoom], lp_sum *sums,
                                              int *counts, int lane, int wave) {
    lp_join_wave(a);
    if (lane == 0) {
        sums[wave] = a;
        counts[wave] = list.n;
    }
    __syncthreads();
    int all = 0;
    for (int w = 0; w < kWaves; w++) all += counts[w];
    if (all > kRoom) {                  /* else one cut of them together does */
        list.cut(lane);
        __syncthreads();
        if (lane == 0) counts[wave] = list.n;
        __syncthreads();
    }
    a = sums[0];
    for (int w = 1; w < kWaves; w++) lp_join(a, sums[w]);
    if (wave) return;
    for (int w = 1; w < kWaves; w++)
        for (int i = lane, n = counts[w]; i - lane < n; i += 64) list.put(keys[w][min(i, n - 1)], i < n, lane);
    list.cut(lane);
}

/* What is asked of a row, from its sums and its list: the top by wave 0, tokens and entropy by the others. */
template <typename T>
__device__ __forceinline__ void lp_finish(const logprobs_args &p, int64_t row, const lp_sum &a, const lp_list &list,
                                          int lane, int wave) {
    const T *x = (const T *)p.logits + row * p.stride;
    const bool fine = a.s > 0.0 && a.s < INFINITY;
    const float nan = __builtin_nanf("");
    const double log_s = log(a.s);
    if (wave) {
        for (int i = 64 * (wave - 1) + lane; i < p.per_row; i += 64 * (kWaves - 1)) {
            const int token = p.tokens[row * p.per_row + i];
            float y = nan;
            if (fine && token >= 0 && token < p.vocab) y = (float)((double)(lp_f32(x[token]) - a.m) - log_s);
            p.token_logprobs[row * p.per_row + i] = y;
        }
        if (p.entropy && threadIdx.x == 64) p.entropy[row] = fine ? (float)(log_s - a.t / a.s) : nan;
    } else if (lane < p.top) {
        const lp_key mine = lane < list.n ? list.keys[lane] : 0;
        const int at = fine && lane < list.n ? list.place(mine) : lane;
        p.top_ids[row * p.top + at] = fine ? (int)~(uint32_t)mine : -1;
        const float y = lp_value((uint32_t)(mine >> 32));
        p.top_logprobs[row * p.top + at] = fine ? (float)((double)(y - a.m) - log_s) : nan;
    }
}

/* 8 waves of a SIMD hold 2047 rows at once (157 us when it was 164 with 7). fp32 logits need more registers, and
 * memory is the bound there. */
template <typename T>
__global__ __launch_bounds__(64 * kWaves, sizeof(T) == 4 ? 6 : 8) void sera_logprobs_kernel(logprobs_args p) {
    constexpr int VEC = 16 / (int)sizeof(T), UNROLL = 16 / VEC;
    __shared__ lp_key keys[kWaves][kRoom];
    __shared__ lp_sum sums[kWaves];
    __shared__ int counts[kWaves];
    __shared__ uint32_t most[64], bound;            /* of the lanes' largest, and what follows from them */
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t row = blockIdx.x;
    const int split = blockIdx.y, piece = split * kWaves + wave, pieces = p.splits * kWaves;
    const T *x = (const T *)p.logits + row * p.stride;
    /* The row's whole 16-byte units, in equal shares; the elements in front of them are a step of the first wave,
     * those behind them one of the last. */
    const int front = min((int)(-(uintptr_t)x & 15u) / (int)sizeof(T), p.vocab);
    const int units = (p.vocab - front) / VEC, back = p.vocab - front - units * VEC;
    const int per = (units + pieces - 1) / pieces, u0 = min(piece * per, units), u1 = min(u0 + per, units);
    const int steps = (u1 - u0 + 64 * UNROLL - 1) / (64 * UNROLL);
    const int from = piece == 0 && front ? -1 : 0, to = steps + (piece == pieces - 1 && back);

    lp_list list;
    list.keys = keys[wave];
    list.n = 0;
    list.top = p.top;
    list.least = 0;
    lp_sum a = {kLowest, 0.0, 0.0};

    /* Unit i of a step for a lane: the id of its first element, and how many of its elements there are. */
    const auto unit = [&](int step, int i, int lane, int *id) {
        if (step >= 0 && step < steps) {
            const int at = u0 + 64 * (UNROLL * step + i) + lane;
            *id = front + VEC * min(at, u1 - 1);
            return at < u1 ? VEC : 0;
        }
        const int n = step < 0 ? front : back;
        *id = (step < 0 ? 0 : p.vocab - back) + min(lane, n - 1);
        return i == 0 && lane < n ? 1 : 0;
    };
    /* Always and in one way, so that nothing waits for a load before the next step; what a step has not got is taken
     * out of it there. */
    const lp_global first = (lp_global)(units ? (const lp_words *)(x + front) : &lp_no_unit);
    const auto load = [&](int step, lp_unit *w) {
#pragma unroll
        for (int i = 0; i < UNROLL; i++)
            w[i].words = first[max(min(u0 + 64 * (UNROLL * step + i) + lane, u1 - 1), 0)];
    };

    /* What is not over `least` has no place in the top; but -inf has one until the list is as long. */
    float least = p.top ? -INFINITY : INFINITY;
    int known = 0;                                  /* candidates when the bound was found */
    const auto look = [&](int step, float top) {
        const uint32_t now = lp_order(top), had = atomicMax(&most[lane], now), mine[1] = {had > now ? had : now};
        if (list.n - known >= p.top || least == -INFINITY) {       /* else the bound has not gone far */
            bool exact;
            int larger;
            const uint32_t nth = lp_nth(mine, p.top, &exact, &larger);
            if (lane == 0) atomicMax(&bound, nth);
            least = fmaxf(least, lp_below(nth));
            known = list.n;
        }
        const bool all = least == -INFINITY && list.n < p.top;
        uint64_t lanes = __ballot(top > least || all);
        while (lanes) {                             /* 4 lanes' elements at a time */
            int of = 64;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (lane >> 4 == j && lanes) of = __builtin_ctzll(lanes);
                lanes &= lanes - 1;
            }
            int id;
            const int n = unit(step, (lane & 15) / VEC, of, &id), e = (lane & 15) % VEC;
            float y = -INFINITY;
            if (of < 64 && e < n) y = lp_f32(x[id += e]);
            const bool is = of < 64 && e < n && (y > least || all);
            if (list.n > kRoom - 64) {
                list.cut(lane);
                known = -kRoom;
            }
            list.put((lp_key)lp_order(y) << 32 | (uint32_t)~id, is && y == y, lane);
        }
        /* The ids that follow are higher: equal logits come behind the list's. */
        least = fmaxf(least, lp_least_value(list.least));
    };

    if (threadIdx.x < 64) most[lane] = 0;
    if (threadIdx.x == 0) bound = 0;
    lp_unit in[UNROLL];
    load(from, in);
    __syncthreads();
    for (int step = from; step < to; step++) {
        float y[16], top = -INFINITY;
        least = fmaxf(least, lp_below(__hip_atomic_load(&bound, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP)));
#pragma unroll
        for (int k = 0; k < 16; k++) y[k] = lp_element<T>(in[k / VEC], k % VEC);
        load(step + 1, in);
        if (step < 0 || u0 + 64 * UNROLL * (step + 1) > u1) {
#pragma unroll
            for (int k = 0; k < 16; k++) {
                int id;
                const int n = unit(step, k / VEC, lane, &id);
                if (k % VEC >= n) y[k] = -INFINITY;
                else if (k == 0 && n < VEC) y[k] = lp_f32(x[id]);
            }
        }
#pragma unroll
        for (int k = 0; k < 16; k++) top = fmaxf(top, y[k]);
        if (__ballot(top > a.m)) lp_raise(a, fmaxf(a.m, top));
        float s = 0.0f, t = 0.0f;       /* of this step: small weights one by one would be lost beside a large sum */
#pragma unroll
        for (int k = 0; k < 16; k++) {
            const float d = y[k] - a.m, w = __builtin_amdgcn_exp2f(d * kLog2E);
            s += w;
            t = fmaf(w, fmaxf(d, -200.0f), t);
        }
        a.s += s;
        a.t += t;
        if (__ballot(top > least) || (least == -INFINITY && list.n < p.top)) look(step, top);
    }
    lp_join_group(a, list, keys, sums, counts, lane, wave);
    if (p.splits == 1) return lp_finish<T>(p, row, a, list, lane, wave);
    if (wave) return;
    const size_t part = (size_t)row * p.splits + split;
    if (lane == 0) ((lp_sum *)p.workspace)[part] = a;
    if (lane < p.top)
        ((lp_key *)(p.workspace + p.sums))[part * p.top + lane] = lane < list.n ? list.keys[lane] : 0;
}

template <typename T>
__global__ __launch_bounds__(64 * kWaves) void sera_logprobs_join_kernel(logprobs_args p) {
    __shared__ lp_key keys[kWaves][kRoom];
    __shared__ lp_sum sums[kWaves];
    __shared__ int counts[kWaves];
    __shared__ uint32_t most[64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t row = blockIdx.x;
    const lp_sum *const ws = (const lp_sum *)p.workspace + (size_t)row * p.splits;
    const lp_key *const parts = (const lp_key *)(p.workspace + p.sums) + (size_t)row * p.splits * p.top;
    lp_list list;
    list.keys = keys[wave];
    list.n = 0;
    list.top = p.top;
    list.least = 0;
    lp_sum a = {kLowest, 0.0, 0.0};
    lp_key key[kMostSplits * SERA_LOGPROBS_MAX_TOP / (64 * kWaves)];
    const int n = p.splits * p.top;
    uint32_t largest = 0;
#pragma unroll
    for (int i = 0; i < (int)(sizeof(key) / sizeof(key[0])); i++) {
        const int at = 64 * kWaves * i + (int)threadIdx.x;
        key[i] = at < n ? parts[at] : 0;
    }
    if ((int)threadIdx.x < p.splits) a = ws[threadIdx.x];
    if (threadIdx.x < 64) most[lane] = 0;
    __syncthreads();
    if (p.top) {
#pragma unroll
        for (int i = 0; i < (int)(sizeof(key) / sizeof(key[0])); i++) {
            const uint32_t high = (uint32_t)(key[i] >> 32);
            largest = high > largest ? high : largest;
        }
        atomicMax(&most[lane], largest);
        __syncthreads();
        const uint32_t mine[1] = {most[lane]};
        bool exact;
        int larger;
        const lp_key least = (lp_key)lp_nth(mine, p.top, &exact, &larger) << 32;
#pragma unroll 1
        for (int i = 0; i < n; i += 64 * kWaves) {
            if (list.n > kRoom - 64) list.cut(lane);
            list.put(key[0], key[0] != 0 && key[0] >= least, lane);
#pragma unroll
            for (int j = 1; j < (int)(sizeof(key) / sizeof(key[0])); j++) key[j - 1] = key[j];
        }
    }
    lp_join_group(a, list, keys, sums, counts, lane, wave);
    lp_finish<T>(p, row, a, list, lane, wave);
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
    return n < 1 ? 1 : n > kMostSplits ? kMostSplits : (int)n;
}

/* Floats of the partial sums (the lists lie behind them, 16-byte aligned). */
size_t sera_logprobs_sums(int rows, int splits) {
    return ((size_t)rows * splits * sizeof(lp_sum) / sizeof(float) + 3) & ~(size_t)3;
}

hipError_t sera_launch_logprobs(uint32_t type, const logprobs_args &p, hipStream_t s) {
    if (type == 0u) return lp_go<float>(p, s);
    if (type == 1u) return lp_go<_Float16>(p, s);
    return lp_go<__bf16>(p, s);
}
