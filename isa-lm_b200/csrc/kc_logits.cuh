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
constexpr int LG_HIST = 8;                             /* history tokens a thread requests at once */
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
    const int *bias_off, *bias_ids;
    const float *bias_vals;
    int n_bias;
    const uint32_t *mask;
    long long ld_mask;
    unsigned *err;
};

template <bool HIST, bool BIAS>
__global__ void __launch_bounds__(LG_THREADS) logits_kernel(const LogitsArgs a) {
    __shared__ __align__(16) int s_count[HIST ? LG_CHUNK : 1];
    __shared__ __align__(16) int s_bias[BIAS ? LG_CHUNK : 1];        /* the last list entry of each token, -1 none */
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
    /* the words that hold bits e .. e + 3 of each vector */
    uint32_t ma[LG_VEC], mb[LG_VEC];
#pragma unroll
    for (int k = 0; k < LG_VEC; k++) {
        ma[k] = mb[k] = 0xffffffffu;
        const int e = e0 + 4 * (tid + k * LG_THREADS), w = e >> 5;
        if (a.mask && e + 3 >= 0 && e < V) {
            const uint32_t *mask = a.mask + row * a.ld_mask;
            if (w >= 0) ma[k] = mb[k] = __ldg(mask + w);
            if (((e + 3) >> 5) != w && ((e + 3) >> 5) <= (V - 1) >> 5) mb[k] = __ldg(mask + ((e + 3) >> 5));
        }
    }
    float rep = 1.0f, pres = 0.0f, freq = 0.0f;
    if constexpr (HIST || BIAS) {
        const int *h = a.hist + row * a.ld_hist;
        int t0[HIST ? LG_HIST : 1], n = 0;
        if constexpr (HIST) {
#pragma unroll
            for (int k = 0; k < LG_HIST; k++) {
                const int i = tid + k * LG_THREADS;
                t0[k] = i < a.hist_cap ? __ldg(h + i) : -1;
            }
            n = a.hist_len ? a.hist_len[row] : a.hist_cap;
            rep = a.repeat ? a.repeat[row] : 1.0f;
            if (a.presence) pres = a.presence[row];
            if (a.frequency) freq = a.frequency[row];
        }
        for (int i = tid; i < LG_CHUNK / 4; i += LG_THREADS) {
            if constexpr (HIST) ((int4 *)s_count)[i] = make_int4(0, 0, 0, 0);
            if constexpr (BIAS) ((int4 *)s_bias)[i] = make_int4(-1, -1, -1, -1);
        }
        __syncthreads();
        if constexpr (HIST) {
            if (n > a.hist_cap) {
                if (tid == 0 && blockIdx.y == 0) atomicOr(a.err, 1u);
                n = a.hist_cap;
            }
            auto seen = [&](int t) {
                if (t >= 0 && t < V && t >= e0 && t - e0 < LG_CHUNK) atomicAdd(&s_count[t - e0], 1);
            };
#pragma unroll
            for (int k = 0; k < LG_HIST; k++)
                if (tid + k * LG_THREADS < n) seen(t0[k]);
            for (int i = tid + LG_HIST * LG_THREADS; i < n; i += LG_THREADS) seen(__ldg(h + i));
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
#pragma unroll
    for (int k = 0; k < LG_VEC; k++) {
        const int o = 4 * (tid + k * LG_THREADS), e = e0 + o;
        if (e + 3 < 0 || e >= V) continue;
        /* the vector's mask bits, from its two words (elements before the row have e < 0: any bit will do) */
        const unsigned bits = __funnelshift_r(ma[k], mb[k], (unsigned)e & 31u);
        int4 cn = make_int4(0, 0, 0, 0), bn = make_int4(-1, -1, -1, -1);
        if constexpr (HIST) cn = *(const int4 *)(s_count + o);
        if constexpr (BIAS) bn = *(const int4 *)(s_bias + o);
        const int cc[4] = { cn.x, cn.y, cn.z, cn.w }, bb[4] = { bn.x, bn.y, bn.z, bn.w };
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float x = z[k][i];
            if constexpr (HIST) {
                const int c = cc[i];
                if (c > 0) {
                    x = x > 0.0f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
                    x = __fsub_rn(x, __fmul_rn(freq, (float)c));
                    x = __fsub_rn(x, pres);
                }
            }
            if constexpr (BIAS) {
                const int b = bb[i];
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
