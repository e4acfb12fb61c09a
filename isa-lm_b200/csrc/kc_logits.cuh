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
 * Bound by memory: 8 bytes a logit, an eighth for the mask. A CTA takes 8192
 * logits of one row; it requests them first, then counts the row's history
 * tokens that fall into its stretch in shared memory while they arrive. */
#pragma once
#include <cstdint>

#include "kc_kernels.cuh"

namespace kc {

constexpr int LG_THREADS = 512;
constexpr int LG_VEC = 4;                              /* float4 per thread */
constexpr int LG_HIST = 4;                             /* history tokens a thread requests at once */
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

/* Shared memory: for each logit of the chunk the times its token is in the
 * history, and the last list entry that names it (-1: none). */
template <bool HIST, bool BIAS>
constexpr int logits_smem() { return ((HIST ? 4 : 0) + (BIAS ? 4 : 0)) * LG_CHUNK; }

template <bool HIST, bool BIAS>
__global__ void __launch_bounds__(LG_THREADS) logits_kernel(const LogitsArgs a) {
    extern __shared__ __align__(16) int lg_smem[];
    int *s_count = lg_smem, *s_bias = lg_smem + (HIST ? LG_CHUNK : 0);
    const int tid = threadIdx.x, V = a.vocab;
    const long long row = blockIdx.x;
    const float *in = a.in + row * a.ld_in;
    float *out = a.out + row * a.ld_out;
    /* vector j of the row covers elements 4 j - sh .. 4 j - sh + 3, 16-byte aligned in `in` */
    const int sh = (int)(((uintptr_t)in >> 2) & 3);
    const bool same = (int)(((uintptr_t)out >> 2) & 3) == sh;
    const int e0 = (int)blockIdx.y * LG_CHUNK - sh;    /* the chunk's first element (below 0: none) */
    /* everything that comes from memory is requested before anything waits */
    int t0[HIST ? LG_HIST : 1], n = 0, b0 = 0, b1 = 0, i0 = -1;
    const int *h = a.hist + row * a.ld_hist;
    float rep = 1.0f, pres = 0.0f, freq = 0.0f;
    if constexpr (BIAS) {
        b0 = __ldg(a.bias_off + row);
        b1 = __ldg(a.bias_off + row + 1);
    }
    if constexpr (HIST) {
        n = a.hist_len ? __ldg(a.hist_len + row) : a.hist_cap;
#pragma unroll
        for (int k = 0; k < LG_HIST; k++) {
            const int i = tid + k * LG_THREADS;
            t0[k] = i < a.hist_cap ? __ldg(h + i) : -1;
        }
        if (a.repeat) rep = __ldg(a.repeat + row);
        if (a.presence) pres = __ldg(a.presence + row);
        if (a.frequency) freq = __ldg(a.frequency + row);
    }
    float z[LG_VEC][4];
    uint32_t ma[LG_VEC], mb[LG_VEC];                   /* the mask words that hold bits e .. e + 3 of each vector */
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
        ma[k] = mb[k] = 0xffffffffu;
        if (a.mask && e + 3 >= 0 && e < V) {
            const uint32_t *mask = a.mask + row * a.ld_mask;
            const int wa = e >> 5, wb = (e + 3) >> 5;  /* (e below 0: word -1, whose bits no logit has) */
            if (wa >= 0) ma[k] = mb[k] = __ldg(mask + wa);
            if (wb != wa && wb <= (V - 1) >> 5) mb[k] = __ldg(mask + wb);
        }
    }
    if constexpr (HIST || BIAS) {
        if constexpr (BIAS) {
            if (b0 < 0 || b1 < b0 || b1 > a.n_bias) {
                if (tid == 0 && blockIdx.y == 0) atomicOr(a.err, 2u);
                b0 = b1 = 0;
            }
            if (b0 + tid < b1) i0 = __ldg(a.bias_ids + b0 + tid);
        }
        for (int i = tid; i < LG_CHUNK / 4; i += LG_THREADS) {
            if constexpr (HIST) ((int4 *)s_count)[i] = make_int4(0, 0, 0, 0);
            if constexpr (BIAS) ((int4 *)s_bias)[i] = make_int4(-1, -1, -1, -1);
        }
        __syncthreads();
        auto here = [&](int t) { return (unsigned)t < (unsigned)V && (unsigned)(t - e0) < (unsigned)LG_CHUNK; };
        if constexpr (HIST) {
            if (n > a.hist_cap) {
                if (tid == 0 && blockIdx.y == 0) atomicOr(a.err, 1u);
                n = a.hist_cap;
            }
#pragma unroll
            for (int k = 0; k < LG_HIST; k++)
                if (tid + k * LG_THREADS < n && here(t0[k])) atomicAdd(&s_count[t0[k] - e0], 1);
            for (int i = tid + LG_HIST * LG_THREADS; i < n; i += LG_THREADS) {
                const int t = __ldg(h + i);
                if (here(t)) atomicAdd(&s_count[t - e0], 1);
            }
        }
        if constexpr (BIAS) {
            if (i0 >= 0 && here(i0)) atomicMax(&s_bias[i0 - e0], b0 + tid);
            for (int i = b0 + tid + LG_THREADS; i < b1; i += LG_THREADS) {
                const int t = __ldg(a.bias_ids + i);
                if (here(t)) atomicMax(&s_bias[t - e0], i);
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < LG_VEC; k++) {
        const int o = 4 * (tid + k * LG_THREADS), e = e0 + o;
        if (e + 3 < 0 || e >= V) continue;
        /* few logits have a history or a bias: four at a time are looked at */
        if constexpr (HIST) {
            const int4 t = *(const int4 *)(s_count + o);
            if (t.x | t.y | t.z | t.w) {
                const int c[4] = { t.x, t.y, t.z, t.w };
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (c[i] > 0) {
                        float x = z[k][i];
                        x = x > 0.0f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
                        x = __fsub_rn(x, __fmul_rn(freq, (float)c[i]));
                        z[k][i] = __fsub_rn(x, pres);
                    }
            }
        }
        if constexpr (BIAS) {
            const int4 t = *(const int4 *)(s_bias + o);
            if ((t.x & t.y & t.z & t.w) >= 0) {
                const int b[4] = { t.x, t.y, t.z, t.w };
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (b[i] >= 0) z[k][i] = __fadd_rn(z[k][i], a.bias_vals[b[i]]);
            }
        }
        const unsigned bits = __funnelshift_r(ma[k], mb[k], (unsigned)e & 31u);
#pragma unroll
        for (int i = 0; i < 4; i++) z[k][i] = (bits >> i) & 1u ? z[k][i] : -INFINITY;
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
