/*
 * attn_weights.hip - the weight that every cached position gets from the rows
 * of a call, after its attention:
 *
 *   w_j = sum over rows i, query heads of 2^(s'_ij - z_i),   z_i = log2(sum_j 2^(s'_ij))
 *
 * with s' = scale * q . k * log2(e), as attention has them, and z left by its
 * kernels. A wave has 32 positions of a kv head, their keys in registers as
 * A operand, and passes over the columns (rows of q times heads of the group), 16 at a
 * time; a lane sums the columns it sees, lanes are joined at the end.
 */
#include "attn_device.h"
#include "sera_launch.h"

namespace {

constexpr int kWaves = 4, kTokens = 32;

}  // namespace

template <int TYPE, typename T, int D>
__global__ __launch_bounds__(64 * kWaves) void sera_attn_weights_kernel(kv_args a, attn_args t) {
    constexpr bool Q8 = TYPE == (int)SERA_KV_Q8, TWO = sizeof(T) == 4;
    constexpr int ES = Q8 ? 1 : 2, KC = D / 32, KP = Q8 ? KC / 2 : KC, NS = kTokens / 16;
    const int b = (int)(blockIdx.z * gridDim.y + blockIdx.y);
    if (b >= a.sequences) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int head = (int)blockIdx.x % a.kv_heads;
    const int j0 = ((int)blockIdx.x / a.kv_heads * kWaves + wave) * kTokens;
    const int col = lane & 15, quarter = lane >> 4;
    const kv_seq s = kv_sequence(a, b);
    if (s.bad || j0 >= s.len) return;
    const int first = s.len - s.n, rows = s.n * t.group, mask = (1 << a.page_shift) - 1;

    /* Keys: A row `col` of operand u is token 16 u + col. */
    const uint8_t *base = a.data + (size_t)head * a.head_bytes;
    attn_h8 kf[NS][KC];
    attn_f4 ks[NS];
    bool lost[NS];
#pragma unroll
    for (int u = 0; u < NS; u++) {
        const int id = attn_page(a, b, j0 + 16 * u, s.len);
        lost[u] = id < 0;
        const uint8_t *run = base + (size_t)max(id, 0) * a.page_bytes;
        const int slot = (j0 + 16 * u) & mask;
        const uint8_t *p = run + (size_t)(slot + col) * (D * ES) + 16 * quarter;
#pragma unroll
        for (int k = 0; k < KP; k++) {
            const attn_u4 w = *(const attn_u4 *)(p + 64 * k);
            if (Q8) {
                kf[u][2 * k] = attn_codes(w[0], w[1]);
                kf[u][2 * k + 1] = attn_codes(w[2], w[3]);
            } else {
                kf[u][k] = __builtin_bit_cast(attn_h8, w);
            }
        }
        if (Q8)
            ks[u] = *(const attn_f4 *)(run + 2 * ((size_t)D << a.page_shift) + 4 * (size_t)(slot + 4 * quarter));
    }

    float sum[NS][4] = {};
    const float sign = t.scale_log2 < 0.0f ? -1.0f : 1.0f;
    /* rows in front of the first that sees position j0 see none of these, unless they are sinks' positions */
    const int c0 = max(j0 - first, 0) * t.group / 16;
    for (int c = c0; c < (rows + 15) / 16; c++) {
        const int r = min(16 * c + col, rows - 1), i = r / t.group, h = head * t.group + r - i * t.group;
        const T *q = (const T *)t.q + (s.row0 + i) * t.q_stride + (int64_t)h * D;
        float x[KC][8], top = 0.0f;
#pragma unroll
        for (int k = 0; k < KC; k++) {
            attn_load8(q + (Q8 ? 64 * (k >> 1) + 16 * quarter + 8 * (k & 1) : 32 * k + 8 * quarter), x[k]);
#pragma unroll
            for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(x[k][e]));
        }
        const float z = t.lse[(size_t)(s.row0 + i) * t.heads + h];
        top = fmaxf(top, xor_partner<16>(top));
        top = fmaxf(top, xor_partner<32>(top));
        const int e2 = attn_q_exponent(top);
        const float up = ldexpf(sign, e2), down = ldexpf(fabsf(t.scale_log2), -e2);
        attn_f4 acc[NS];
#pragma unroll
        for (int u = 0; u < NS; u++) acc[u] = attn_f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < KC; k++) {
#pragma unroll
            for (int e = 0; e < 8; e++) x[k][e] *= up;
            attn_h8 qh, ql;
            attn_split<TWO>(x[k], qh, ql);
#pragma unroll
            for (int u = 0; u < NS; u++) {
                acc[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[u][k], qh, acc[u], 0, 0, 0);
                if (TWO) acc[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[u][k], ql, acc[u], 0, 0, 0);
            }
        }
#pragma unroll
        for (int u = 0; u < NS; u++) {
            if (Q8) acc[u] *= ks[u];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int j = j0 + 16 * u + 4 * quarter + e;
                const bool sees = 16 * c + col < rows && attn_sees(t, first + i, j);
                const float w = lost[u] ? __builtin_nanf("") : attn_exp2(acc[u][e] * down - z);
                sum[u][e] += sees ? w : 0.0f;
            }
        }
    }
    const size_t place = ((size_t)b * a.kv_heads + head) * (size_t)t.weights_stride;
#pragma unroll
    for (int u = 0; u < NS; u++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            float w = sum[u][e];
            w += xor_partner<1>(w);
            w += xor_partner<2>(w);
            w += xor_partner<4>(w);
            w += xor_partner<8>(w);
            const int j = j0 + 16 * u + 4 * quarter + e;
            if (col == 0 && j < s.len)
                t.weights[place + j] = (t.before && j < first ? t.before[place + j] : 0.0f) + w;
        }
}

namespace {

template <int TYPE, typename T, int D>
void weights_go(const kv_args &a, const attn_args &t, hipStream_t s) {
    const int y = a.sequences < 32768 ? a.sequences : 32768;
    const int64_t tiles = ((int64_t)a.max_kv + kWaves * kTokens - 1) / (kWaves * kTokens);
    hipLaunchKernelGGL((sera_attn_weights_kernel<TYPE, T, D>),
                       dim3((unsigned)(tiles * a.kv_heads), (unsigned)y, (unsigned)((a.sequences + y - 1) / y)),
                       dim3(64 * kWaves), 0, s, a, t);
}

template <int TYPE, typename T>
void weights_d(int dim, const kv_args &a, const attn_args &t, hipStream_t s) {
    dim == 64 ? weights_go<TYPE, T, 64>(a, t, s) : weights_go<TYPE, T, 128>(a, t, s);
}

template <int TYPE>
void weights_t(uint32_t type, int dim, const kv_args &a, const attn_args &t, hipStream_t s) {
    if (type == SERA_TYPE_F32) weights_d<TYPE, float>(dim, a, t, s);
    else if (type == SERA_TYPE_F16) weights_d<TYPE, _Float16>(dim, a, t, s);
    else weights_d<TYPE, __bf16>(dim, a, t, s);
}

}  // namespace

hipError_t sera_launch_attn_weights(uint32_t cache_type, uint32_t type, int dim, const kv_args &a, const attn_args &t,
                                    hipStream_t s) {
    if (cache_type == SERA_KV_F16) weights_t<(int)SERA_KV_F16>(type, dim, a, t, s);
    else weights_t<(int)SERA_KV_Q8>(type, dim, a, t, s);
    return hipGetLastError();
}
