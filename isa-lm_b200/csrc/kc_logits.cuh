/* Logits of a batch of rows before a token is chosen: penalties for tokens of
 * a row's history, biases and a mask of allowed tokens, in one pass.
 *
 * For the token v of a row whose history holds it c times:
 *   c > 0:  z = z > 0 ? z / repeat : z * repeat     (model/sampler.c:30-42)
 *           z = z - frequency * c,  z = z - presence
 *   z = z + bias of v (the last entry of the row's list that names v)
 *   z = -inf where v's bit of the row's mask is 0
 * every operation IEEE round to nearest in 32 bits, in this order.
 *
 * Bound by memory: 8 bytes a logit, an eighth for the mask. A CTA takes 4096
 * logits of one row; it requests them first, then counts the row's history
 * tokens that fall into its stretch in shared memory while they arrive. */
#pragma once
#include <cstdint>

#include "kc_kernels.cuh"

namespace kc {

constexpr int LG_THREADS = 256;
constexpr int LG_VEC = 4;                              /* float4 per thread */
constexpr int LG_CHUNK = LG_THREADS * LG_VEC * 4;      /* logits per CTA */

struct LogitsArgs {
    const float *in;
    float *out;
    long long ld_in, ld_out;
    int vocab;
    const int *hist, *hist_len;
    long long ld_hist;
    int hist_cap;
    const float *repeat, *presence, *frequency;
    float repeat1;                  /* the rows' repeat where `repeat` is NULL */
    const int *bias_off, *bias_ids;
    const float *bias_vals;
    int n_bias;
    const uint32_t *mask;
    long long ld_mask;
    unsigned *err;
};

template <bool HIST, bool BIAS>
__global__ void __launch_bounds__(LG_THREADS) logits_kernel(const LogitsArgs a) {
    __shared__ int s_count[HIST ? LG_CHUNK : 1];
    __shared__ int s_bias[BIAS ? LG_CHUNK : 1];        /* the last list entry of each token, -1 none */
    const int tid = threadIdx.x, V = a.vocab;
    const long long row = blockIdx.x;
    const float *in = a.in + row * a.ld_in;
    float *out = a.out + row * a.ld_out;
    /* vector j of the row covers elements 4 j - sh .. 4 j - sh + 3, 16-byte aligned in `in` */
    const int sh = (int)(((uintptr_t)in >> 2) & 3);
    const bool same = (int)(((uintptr_t)out >> 2) & 3) == sh;
    const int e0 = (int)blockIdx.y * LG_CHUNK - sh;    /* the chunk's first element (below 0: none) */
    float z[LG_VEC][4];
#pragma unroll
    for (int k = 0; k < LG_VEC; k++) {
        const int e = e0 + 4 * (tid + k * LG_THREADS);
        if (e >= 0 && e <= V - 4) {
            const float4 x = __ldcs((const float4 *)(in + e));
            z[k][0] = x.x; z[k][1] = x.y; z[k][2] = x.z; z[k][3] = x.w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) z[k][i] = e + i >= 0 && e + i < V ? in[e + i] : 0.0f;
        }
    }
    float rep = 1.0f, pres = 0.0f, freq = 0.0f;
    if constexpr (HIST || BIAS) {
        for (int i = tid; i < LG_CHUNK; i += LG_THREADS) {
            if constexpr (HIST) s_count[i] = 0;
            if constexpr (BIAS) s_bias[i] = -1;
        }
        __syncthreads();
        if constexpr (HIST) {
            int n = a.hist_len ? a.hist_len[row] : a.hist_cap;
            if (n > a.hist_cap) {
                if (tid == 0 && blockIdx.y == 0) atomicOr(a.err, 1u);
                n = a.hist_cap;
            }
            const int *h = a.hist + row * a.ld_hist;
            for (int i = tid; i < n; i += LG_THREADS) {
                const int t = h[i];
                if (t >= 0 && t < V && t >= e0 && t - e0 < LG_CHUNK) atomicAdd(&s_count[t - e0], 1);
            }
            rep = a.repeat ? a.repeat[row] : a.repeat1;
            if (a.presence) pres = a.presence[row];
            if (a.frequency) freq = a.frequency[row];
        }
        if constexpr (BIAS) {
            int b0 = a.bias_off[row], b1 = a.bias_off[row + 1];
            if (b0 < 0 || b1 < b0 || b1 > a.n_bias) {
                if (tid == 0 && blockIdx.y == 0) atomicOr(a.err, 2u);
                b0 = b1 = 0;
            }
            for (int i = b0 + tid; i < b1; i += LG_THREADS) {
                const int t = a.bias_ids[i];
                if (t >= 0 && t < V && t >= e0 && t - e0 < LG_CHUNK) atomicMax(&s_bias[t - e0], i);
            }
        }
        __syncthreads();
    }
    const uint32_t *mask = a.mask ? a.mask + row * a.ld_mask : nullptr;
#pragma unroll
    for (int k = 0; k < LG_VEC; k++) {
        const int o = 4 * (tid + k * LG_THREADS), e = e0 + o;
        if (e + 3 < 0 || e >= V) continue;
        /* the vector's mask bits: one word or two */
        unsigned bits = 0xfu;
        if (mask) {
            const int ea = max(e, 0), eb = min(e + 3, V - 1);
            const uint32_t wa = __ldg(mask + (ea >> 5));
            const uint32_t wb = (eb >> 5) != (ea >> 5) ? __ldg(mask + (eb >> 5)) : wa;
            bits = 0u;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int v = min(max(e + i, ea), eb);
                const uint32_t w = (v >> 5) == (ea >> 5) ? wa : wb;
                bits |= ((w >> (v & 31)) & 1u) << i;
            }
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float x = z[k][i];
            if constexpr (HIST) {
                const int c = s_count[o + i];
                if (c > 0) {
                    x = x > 0.0f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
                    x = __fsub_rn(x, __fmul_rn(freq, (float)c));
                    x = __fsub_rn(x, pres);
                }
            }
            if constexpr (BIAS) {
                const int b = s_bias[o + i];
                if (b >= 0) x = __fadd_rn(x, a.bias_vals[b]);
            }
            z[k][i] = (bits >> i) & 1u ? x : -INFINITY;
        }
        if (same && e >= 0 && e <= V - 4) {
            __stcs((float4 *)(out + e), make_float4(z[k][0], z[k][1], z[k][2], z[k][3]));
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (e + i >= 0 && e + i < V) out[e + i] = z[k][i];
        }
    }
}

}  // namespace kc
