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
 * logits of one row. It requests them and the row's history first, counts in
 * shared memory which history tokens and biases fall into its stretch while the
 * logits arrive, writes them through the mask, and then goes over the few that
 * are touched, listed once each, whose values it makes meanwhile. 64 rows of
 * 128256: 12.0 us with a mask alone, 17.0 us with 2048 tokens of history and 100
 * biases each, from memory (floor 10.4). Measured beside it and not taken: every logit looking
 * at its own counter, 1.9 times the instructions; stretches of 16384 logits that
 * share one look at the history, the same time, since one wave of CTAs then
 * counts while the memory waits and streams while the counters do. */
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
    const int *bias_off, *bias_ids;
    const float *bias_vals;
    int n_bias;
    const uint32_t *mask;
    long long ld_mask;
    unsigned *err;
};

template <bool HIST, bool BIAS>
__global__ void __launch_bounds__(LG_THREADS, 5) logits_kernel(const LogitsArgs a) {
    /* for each logit of the chunk the times its token is in the history (16 bits; a longer history and biases are
     * two launches), above it one more than the last entry of the row's list that names it, 0: none; and the
     * touched logits, once each */
    constexpr bool ANY = HIST || BIAS;
    constexpr int NH = BIAS ? 4 : 8;                   /* history tokens a thread requests at once */
    __shared__ __align__(16) uint32_t s_word[ANY ? LG_CHUNK : 4];
    __shared__ unsigned short s_list[ANY ? LG_CHUNK : 1];
    __shared__ int s_n;
    launch_next();
    stream_order();
    const int tid = threadIdx.x, V = a.vocab;
    const long long row = blockIdx.x;
    const float *in = a.in + row * a.ld_in;
    float *out = a.out + row * a.ld_out;
    const uint32_t *mask = a.mask ? a.mask + row * a.ld_mask : nullptr;
    /* vector j of the row covers elements 4 j - sh .. 4 j - sh + 3, 16-byte aligned in `in` */
    const int sh = (int)(((uintptr_t)in >> 2) & 3);
    const bool same = (int)(((uintptr_t)out >> 2) & 3) == sh;
    const int e0 = (int)blockIdx.y * LG_CHUNK - sh;    /* the chunk's first element (below 0: none) */
    /* every vector of the chunk is whole, aligned in `out` too, and its mask bits lie in one word */
    const bool whole = sh == 0 && same && e0 + LG_CHUNK <= V;
    /* everything that comes from memory is requested before anything waits */
    int t0[HIST ? NH : 1], n = 0, b0 = 0, b1 = 0, i0 = -1;
    const int *h = a.hist + row * a.ld_hist;
    float rep = 1.0f, pres = 0.0f, freq = 0.0f;
    if constexpr (BIAS) {
        b0 = a.bias_off[row];
        b1 = a.bias_off[row + 1];
    }
    if constexpr (HIST) {
        n = a.hist_len ? a.hist_len[row] : a.hist_cap;
#pragma unroll
        for (int k = 0; k < NH; k++) {
            const int i = tid + k * LG_THREADS;
            t0[k] = i < a.hist_cap ? h[i] : -1;
        }
        if (a.repeat) rep = a.repeat[row];
        if (a.presence) pres = a.presence[row];
        if (a.frequency) freq = a.frequency[row];
    }
    float4 z[LG_VEC];
    uint32_t mw[LG_VEC];                               /* the vectors' mask bits from bit 0 on */
    if (whole) {
#pragma unroll
        for (int k = 0; k < LG_VEC; k++) {
            const int e = e0 + 4 * (tid + k * LG_THREADS);
            z[k] = load_once(in + e);
            mw[k] = mask ? mask[e >> 5] >> (e & 31) : 0xfu;
        }
    } else {
#pragma unroll
        for (int k = 0; k < LG_VEC; k++) {
            const int e = e0 + 4 * (tid + k * LG_THREADS);
            z[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            mw[k] = 0xfu;
            if (e + 3 < 0 || e >= V) continue;
            if (e >= 0 && e <= V - 4) {
                z[k] = load_once(in + e);
            } else {
                if (e >= 0) z[k].x = in[e];
                if (e + 1 >= 0 && e + 1 < V) z[k].y = in[e + 1];
                if (e + 2 >= 0 && e + 2 < V) z[k].z = in[e + 2];
                if (e + 3 < V) z[k].w = in[e + 3];
            }
            if (mask) {
                uint32_t wa = 0xffffffffu, wb;         /* (elements below 0 are no logits: any bit will do) */
                if (e >= 0) wa = mask[e >> 5];
                wb = wa;
                if ((e + 3) >> 5 != e >> 5 && (e + 3) >> 5 <= (V - 1) >> 5) wb = mask[(e + 3) >> 5];
                mw[k] = __funnelshift_r(wa, wb, (unsigned)e & 31u);
            }
        }
    }
    if constexpr (ANY) {
        if constexpr (BIAS) {
            if (b0 < 0 || b1 < b0 || b1 > a.n_bias) {
                if (tid == 0 && blockIdx.y == 0) atomicOr(a.err, 2u);
                b0 = b1 = 0;
            }
            if (b0 + tid < b1) i0 = a.bias_ids[b0 + tid];
        }
        for (int i = tid; i < LG_CHUNK / 4; i += LG_THREADS) ((uint4 *)s_word)[i] = make_uint4(0u, 0u, 0u, 0u);
        if (tid == 0) s_n = 0;
        __syncthreads();
        auto here = [&](int t) { return (unsigned)t < (unsigned)V && (unsigned)(t - e0) < (unsigned)LG_CHUNK; };
        auto touch = [&](int o) { s_list[atomicAdd(&s_n, 1)] = (unsigned short)o; };
        if constexpr (HIST) {
            if ((unsigned)n > (unsigned)a.hist_cap) {
                if (tid == 0 && blockIdx.y == 0) atomicOr(a.err, 1u);
                n = n < 0 ? 0 : a.hist_cap;
            }
            auto seen = [&](int t) {
                if (here(t) && atomicAdd(&s_word[t - e0], 1u) == 0u) touch(t - e0);
            };
#pragma unroll
            for (int k = 0; k < NH; k++)
                if (tid + k * LG_THREADS < n) seen(t0[k]);
            for (int i = tid + NH * LG_THREADS; i < n; i += LG_THREADS) seen(h[i]);
        }
        if constexpr (BIAS) {
            constexpr int SH = HIST ? 16 : 0;
            constexpr uint32_t LOW = HIST ? 0xffffu : 0u;
            auto named = [&](int t, int i) {           /* the largest entry, above the count */
                if (!here(t)) return;
                uint32_t *w = &s_word[t - e0], old = *(volatile uint32_t *)w;
                while ((old >> SH) < (uint32_t)(i + 1)) {
                    const uint32_t was = atomicCAS(w, old, (old & LOW) | ((uint32_t)(i + 1) << SH));
                    if (was == old) {
                        if (old == 0u) touch(t - e0);
                        break;
                    }
                    old = was;
                }
            };
            if (i0 >= 0) named(i0, tid);
            for (int i = tid + LG_THREADS; i < b1 - b0; i += LG_THREADS) named(a.bias_ids[b0 + i], i);
        }
    }
    /* the few that are touched and allowed: their values are made while the others are written. (Where `out` is
     * `in`, what is read here may have been written already: with the same value, since it is allowed.) */
    int to = -1, m = 0;
    float tx = 0.0f;
    auto edit = [&](int i) {
        const int o = s_list[i], t = e0 + o;
        const uint32_t v = s_word[o];
        const int c = HIST && BIAS ? (int)(v & 0xffffu) : (HIST ? (int)v : 0);
        const int b = HIST && BIAS ? (int)(v >> 16) - 1 : (BIAS ? (int)v - 1 : -1);
        const uint32_t w = mask ? mask[t >> 5] : 0xffffffffu;
        const float bv = b >= 0 ? a.bias_vals[b0 + b] : 0.0f;
        tx = ((volatile const float *)in)[t];
        to = (w >> (t & 31)) & 1u ? t : -1;
        if (c > 0) {
            tx = tx > 0.0f ? __fdiv_rn(tx, rep) : __fmul_rn(tx, rep);
            tx = __fsub_rn(tx, __fmul_rn(freq, (float)c));
            tx = __fsub_rn(tx, pres);
        }
        if (b >= 0) tx = __fadd_rn(tx, bv);
    };
    if constexpr (ANY) {
        __syncthreads();
        m = s_n;
        if (tid < m) edit(tid);
    }
    /* the logits through the mask */
#pragma unroll
    for (int k = 0; k < LG_VEC; k++) {
        const int e = e0 + 4 * (tid + k * LG_THREADS);
        z[k].x = mw[k] & 1u ? z[k].x : -INFINITY;
        z[k].y = mw[k] & 2u ? z[k].y : -INFINITY;
        z[k].z = mw[k] & 4u ? z[k].z : -INFINITY;
        z[k].w = mw[k] & 8u ? z[k].w : -INFINITY;
        if (whole || (same && e >= 0 && e <= V - 4)) {
            __stcs((float4 *)(out + e), z[k]);
        } else {
            if (e >= 0 && e < V) out[e] = z[k].x;
            if (e + 1 >= 0 && e + 1 < V) out[e + 1] = z[k].y;
            if (e + 2 >= 0 && e + 2 < V) out[e + 2] = z[k].z;
            if (e + 3 >= 0 && e + 3 < V) out[e + 3] = z[k].w;
        }
    }
    if constexpr (ANY) {
        __syncthreads();
        for (int i = tid; i < m; i += LG_THREADS) {
            if (i != tid) edit(i);
            if (to >= 0) out[to] = tx;
        }
    }
}

}  // namespace kc
