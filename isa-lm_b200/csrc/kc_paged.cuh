/* A paged KV cache for several sequences: the rows of new tokens into it, and
 * the attention of one new token per sequence over it.
 *
 * The pool holds K and V as [page][kv head][slot][head_dim] in the cache's type
 * (f32, f16, or int8 with one float scale for each row of a head, as
 * [page][kv head][slot]), so the rows of a head within a page are contiguous.
 * table[seq][p / page_size] names the page of position p of a sequence.
 * Page numbers, lengths and positions come from device memory: they are checked
 * where they are read, and a bad one is skipped and flagged, never followed. */
#pragma once
#include <cuda_fp16.h>
#include <cstdint>

#include "kc_kernels.cuh"
#include "krafla_cuda.h"

namespace kc {

/* error bits of the serving operators' word */
enum { SE_HIST = 1, SE_BIAS = 2, SE_LEN = 4, SE_PAGE = 8, SE_ROW = 16 };

struct PagedKV {
    uint8_t *k, *v;
    float *kd, *vd;
    const int *table;
    int n_seqs, ld_table, n_pages, page, n_kv, hd;
};

/* ------------------------------------------------------------ append */

struct AppendArgs {
    PagedKV kv;
    const float *q, *k, *v;
    long long ldq, ldk, ldv, ldo;
    float *q_out;
    const float *cos, *sin;      /* [n_pos][hd / 2] */
    const float *q_norm, *k_norm;
    float eps;
    const int *seqs, *pos;
    int rows, n_heads, n_pos;
    unsigned *err;
};

constexpr int AP_THREADS = 256;

/* The sum over the LPH lanes that hold a head's row. */
template <int LPH, class T>
__device__ __forceinline__ T head_sum(T v) {
#pragma unroll
    for (int o = LPH / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

/* Norm (y = x / sqrt(mean(x^2) + eps) * w) and rotation of adjacent pairs of
 * the 4 * NV values that each lane of a head holds, in type T. */
template <class T, int LPH, int NV>
__device__ __forceinline__ void norm_rope(const float (&x)[NV][4], float (&y)[NV][4], const float *w, float eps, int hd,
                                          const float *cs, const float *sn, int lane) {
    T inv = (T)1;
    if (w) {
        T s = (T)0;
#pragma unroll
        for (int j = 0; j < NV; j++)
#pragma unroll
            for (int i = 0; i < 4; i++) s += (T)x[j][i] * (T)x[j][i];
        s = head_sum<LPH>(s);
        if constexpr (sizeof(T) == 8) inv = 1.0 / sqrt(s / (double)hd + (double)eps);
        else inv = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(s, (float)hd), eps)));
    }
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int d = 4 * (lane + j * LPH);
        if (d >= hd) continue;
        const float2 c = __ldg((const float2 *)(cs + d / 2)), s = __ldg((const float2 *)(sn + d / 2));
        float4 g = make_float4(1.0f, 1.0f, 1.0f, 1.0f);
        if (w) g = make_float4(__ldg(w + d), __ldg(w + d + 1), __ldg(w + d + 2), __ldg(w + d + 3));
        const T a = (T)x[j][0] * inv * (T)g.x, b = (T)x[j][1] * inv * (T)g.y;
        const T e = (T)x[j][2] * inv * (T)g.z, f = (T)x[j][3] * inv * (T)g.w;
        y[j][0] = (float)(a * (T)c.x - b * (T)s.x);
        y[j][1] = (float)(a * (T)s.x + b * (T)c.x);
        y[j][2] = (float)(e * (T)c.y - f * (T)s.y);
        y[j][3] = (float)(e * (T)s.y + f * (T)c.y);
    }
}

/* One head of one row per group of LPH lanes, 4 * NV values a lane. Bound by
 * memory: every value is read once and written once.
 *
 * K rows of an 8-bit cache are normed and rotated in 64 bits and rounded once,
 * so that which side of a step's border a value falls on does not depend on
 * the order of the norm's sum; queries and wider caches use 32 bits. */
template <int KV, int LPH, int NV>
__global__ void __launch_bounds__(AP_THREADS) append_kernel(const AppendArgs a) {
    const int lane = threadIdx.x % LPH;
    const int heads = a.n_heads + 2 * a.kv.n_kv, hd = a.kv.hd;
    const long long item = ((long long)blockIdx.x * AP_THREADS + threadIdx.x) / LPH, total = (long long)a.rows * heads;
    const bool live = item < total;
    const int row = live ? (int)(item / heads) : 0, h = live ? (int)(item % heads) : 0;
    const bool isq = h < a.n_heads, isv = h >= a.n_heads + a.kv.n_kv;
    const int hh = isq ? h : (isv ? h - a.n_heads - a.kv.n_kv : h - a.n_heads);
    const float *src = isq ? a.q + row * a.ldq : (isv ? a.v + row * a.ldv : a.k + row * a.ldk);
    src += (size_t)hh * hd;
    float x[NV][4], y[NV][4];
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int d = 4 * (lane + j * LPH);
        float4 t = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (live && d < hd) t = __ldcs((const float4 *)(src + d));
        x[j][0] = t.x; x[j][1] = t.y; x[j][2] = t.z; x[j][3] = t.w;
    }
    /* where the row goes: the same for all lanes of the head */
    const int seq = live ? (a.seqs ? a.seqs[row] : row) : -1, p = live ? a.pos[row] : 0;
    bool ok = seq >= 0;
    int page = 0, slot = 0;
    if (ok) {
        const int pi = p >= 0 ? p / a.kv.page : 0;
        slot = p - pi * a.kv.page;
        if (seq >= a.kv.n_seqs || p < 0 || p >= a.n_pos || pi >= a.kv.ld_table) ok = false;
        else {
            page = a.kv.table[(size_t)seq * a.kv.ld_table + pi];
            ok = page >= 0 && page < a.kv.n_pages;
        }
        if (!ok && lane == 0 && h == 0) atomicOr(a.err, (unsigned)SE_ROW);
    }
    /* no early return: the lanes of a warp meet in the sums */
    const float *cs = a.cos + (size_t)(ok ? p : 0) * (hd / 2), *sn = a.sin + (size_t)(ok ? p : 0) * (hd / 2);
    if (isv) {
#pragma unroll
        for (int j = 0; j < NV; j++)
#pragma unroll
            for (int i = 0; i < 4; i++) y[j][i] = x[j][i];
    }
    /* (the norm's shuffles are taken by all lanes of a warp: heads of different
     * kinds may share it, so each kind's pass runs warp-wide where one needs it) */
    float t[NV][4];
    const bool any_q = __any_sync(0xffffffffu, isq), any_k = __any_sync(0xffffffffu, !isq && !isv);
    if (KV != KC_Q8_0 || any_q) {
        norm_rope<float, LPH, NV>(x, t, a.q_norm ? (isq ? a.q_norm : a.k_norm) : nullptr, a.eps, hd, cs, sn, lane);
        if (isq || (KV != KC_Q8_0 && !isv)) {
#pragma unroll
            for (int j = 0; j < NV; j++)
#pragma unroll
                for (int i = 0; i < 4; i++) y[j][i] = t[j][i];
        }
    }
    if (KV == KC_Q8_0 && any_k) {
        norm_rope<double, LPH, NV>(x, t, a.k_norm, a.eps, hd, cs, sn, lane);
        if (!isq && !isv) {
#pragma unroll
            for (int j = 0; j < NV; j++)
#pragma unroll
                for (int i = 0; i < 4; i++) y[j][i] = t[j][i];
        }
    }
    float amax = 0.0f;
    if constexpr (KV == KC_Q8_0) {
#pragma unroll
        for (int j = 0; j < NV; j++)
            if (4 * (lane + j * LPH) < hd)
                amax = fmaxf(amax, fmaxf(fmaxf(fabsf(y[j][0]), fabsf(y[j][1])), fmaxf(fabsf(y[j][2]), fabsf(y[j][3]))));
#pragma unroll
        for (int o = LPH / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    }
    if (!ok) return;
    if (isq) {
        float *dst = a.q_out + row * a.ldo + (size_t)hh * hd;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int d = 4 * (lane + j * LPH);
            if (d < hd) *(float4 *)(dst + d) = make_float4(y[j][0], y[j][1], y[j][2], y[j][3]);
        }
        return;
    }
    const size_t r = ((size_t)page * a.kv.n_kv + hh) * a.kv.page + slot;
    uint8_t *pool = isv ? a.kv.v : a.kv.k;
    /* the single-scale row rule of the model's 8-bit cache (ops/ops.c:81-96) */
    const bool tiny = amax < 1e-30f;
    const float id = KV == KC_Q8_0 && !tiny ? __fdiv_rn(127.0f, amax) : 0.0f;
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int d = 4 * (lane + j * LPH);
        if (d >= hd) continue;
        if constexpr (KV == KC_F32) {
            ((float4 *)pool)[(r * hd + d) / 4] = make_float4(y[j][0], y[j][1], y[j][2], y[j][3]);
        } else if constexpr (KV == KC_F16) {
            __half2 lo = __floats2half2_rn(y[j][0], y[j][1]), hi = __floats2half2_rn(y[j][2], y[j][3]);
            ((uint2 *)pool)[(r * hd + d) / 4] = make_uint2(*(unsigned *)&lo, *(unsigned *)&hi);
        } else {
            unsigned w = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                int qi = 0;
                if (!tiny) {
                    const float u = truncf(__fadd_rn(__fmul_rn(y[j][i], id), copysignf(0.5f, y[j][i])));
                    qi = (int)fminf(fmaxf(u, -127.0f), 127.0f);
                }
                w |= ((unsigned)qi & 0xffu) << (8 * i);
            }
            ((unsigned *)pool)[(r * hd + d) / 4] = w;
        }
    }
    if (KV == KC_Q8_0 && lane == 0) (isv ? a.kv.vd : a.kv.kd)[r] = tiny ? 0.0f : __fdiv_rn(amax, 127.0f);
}

/* ------------------------------------------------------------ attention */

/* out = sum_t exp(s_t - m) v_t / sum_t exp(s_t - m), s_t = q . k_t * scale (or
 * softcap * tanh of that over softcap) for t in [max(0, len - window), len).
 *
 * Work is cut into quanta of AT_WARPS tiles of TP positions of one unit (a
 * sequence's KV head, or a chunk of 8 * MT of its query heads). The quanta of
 * all units in a row are shared out evenly over the CTAs, so that ragged
 * lengths leave none idle; a CTA's share may begin and end inside a unit, whose
 * pieces paged_join_kernel puts together. Within a quantum each warp has a tile,
 * its own ring of shared-memory slots (cp.async) and its own running softmax;
 * the warps meet once per unit.
 *
 * Both products run on the tensor cores with the query heads as the 16-row
 * side: rows 0-7 hold the high halves of eight heads' values, rows 8-15 what
 * the high halves leave (two f16 of 11 bits each, or two tf32), so a product
 * keeps 22 bits of a 32-bit query or softmax weight, at no more instructions
 * than one f16 row block takes. The sums of a tile leave the tensor core once
 * per tile and are carried in f32. */
constexpr int AT_WARPS = 4;
constexpr int AT_THREADS = AT_WARPS * 32;
constexpr int AT_COMB = 4;                /* heads that the warps of a CTA put together at a time */

template <int KV>
struct AttType;
template <>
struct AttType<KC_F32> { static constexpr int ES = 4, TP = 8; };
template <>
struct AttType<KC_F16> { static constexpr int ES = 2, TP = 16; };
template <>
struct AttType<KC_Q8_0> { static constexpr int ES = 1, TP = 32; };

struct AttendArgs {
    PagedKV kv;
    const float *q;
    float *out;
    long long ldq, ldo;
    const int *lens;
    int n_seqs, n_heads, group, chunks;   /* chunks: head chunks per KV head */
    int window;
    float scale, softcap;
    int min_quanta;                       /* least quanta of a CTA's share */
    float *part;                          /* [2 * CTAs] partial results */
    int4 *desc;                           /* [CTAs] what to join */
    unsigned *err;
};

/* One piece of a unit: 8 * MT heads' sums [HD], then their maxima, then their weights' sums. */
template <int HD, int MT>
constexpr int part_floats() { return 8 * MT * (HD + 2); }

__device__ __forceinline__ void cp_async16z(uint32_t dst, const void *src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0));
}
__device__ __forceinline__ void cp_async4z(uint32_t dst, const void *src, bool live) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(live ? 4 : 0));
}
template <int N>
__device__ __forceinline__ void cp_async_wait_but() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldsm4(unsigned (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm4t(unsigned (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ float4 lds4(uint32_t a) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
/* rows 8-15 of A are zero */
__device__ __forceinline__ void mma_s8(int (&c)[4], unsigned a0, unsigned a2, unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %5}, {%7, %8}, {%0, %1, %2, %3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(0), "r"(a2), "r"(b0), "r"(b1));
}

__device__ __forceinline__ unsigned h2u(__half2 h) { return *(unsigned *)&h; }
/* two floats as f16 pairs: the high parts, and what they leave */
__device__ __forceinline__ void split_f16(float a, float b, unsigned &hi, unsigned &lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    hi = h2u(h);
    lo = h2u(__floats2half2_rn(a - f.x, b - f.y));
}
__device__ __forceinline__ unsigned to_tf32(float a) {
    unsigned r;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(a));
    return r;
}
__device__ __forceinline__ void split_tf32(float a, unsigned &hi, unsigned &lo) {
    hi = to_tf32(a);
    lo = to_tf32(a - __uint_as_float(hi));
}

/* Positions [first, len) of sequence b, quanta of QP positions, clamped to what the table can hold. */
__device__ __forceinline__ int seq_span(const AttendArgs &a, int b, int &first, bool &bad) {
    int n = a.lens[b];
    const long long cap = (long long)a.kv.ld_table * a.kv.page;
    bad = n < 0 || n > cap;
    if (n < 0) n = 0;
    if (n > cap) n = (int)cap;
    first = a.window > 0 && n > a.window ? n - a.window : 0;
    return n;
}

/* Shared memory of a warp's ring slot: K rows, V rows, and (8-bit) their scales. */
template <int KV, int HD>
constexpr int slot_bytes() { return 2 * 32 * HD + (KV == KC_Q8_0 ? 2 * 32 * 4 : 0); }
template <int KV, int HD, int MT, int S>
constexpr int attend_smem() {
    return AT_WARPS * (S * (slot_bytes<KV, HD>() + 16) + AT_COMB * HD * 4 + 2 * 8 * MT * 4);
}

/* sum / weights; nothing attended gives zeros */
__device__ __forceinline__ float4 over(float4 o, float l) {
    const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
    return make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
}

/* The share of CTA i of n of `total` quanta: [i total / n, (i + 1) total / n). */
__device__ __forceinline__ long long share_lo(long long i, long long n, long long total) { return i * total / n; }

template <int KV, int HD, int MT, int S>
__global__ void __launch_bounds__(AT_THREADS, HD <= 128 ? 2 : 1) paged_attend_kernel(const __grid_constant__ AttendArgs a) {
    constexpr int ES = AttType<KV>::ES, TP = AttType<KV>::TP, QP = AT_WARPS * TP;
    constexpr int PITCH = HD * ES, CPR = PITCH / 16;   /* bytes and 16-byte chunks of a row */
    constexpr int NT = TP / 8;                         /* 8-position column blocks of the scores */
    constexpr int SLOT = slot_bytes<KV, HD>();
    constexpr int HC = 8 * MT;
    extern __shared__ __align__(128) unsigned char at_raw[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int r = lane >> 2, c = lane & 3;             /* fragment row (head) and column group */
    unsigned char *ring = at_raw + (size_t)warp * S * SLOT;
    int4 *info = (int4 *)(at_raw + AT_WARPS * S * SLOT) + warp * S;   /* what each slot holds */
    float *comb = (float *)(at_raw + AT_WARPS * S * (SLOT + 16));     /* finish: the warps' sums */
    float *cml = comb + AT_WARPS * AT_COMB * HD;                      /* and their maxima and weights' sums */
    const uint32_t ring_s = smem_u32(ring);
    const int U = a.kv.n_kv * a.chunks;                /* units per sequence */

    cudaTriggerProgrammaticLaunchCompletion();

    /* ---- this CTA's share ---- */
    __shared__ long long s_sum[AT_WARPS];
    __shared__ long long s_lo, s_total;
    __shared__ int s_b, s_cnt, s_ncta;
    __shared__ long long s_base;                       /* quanta of the sequences before s_b */
    {
        const int per = (a.n_seqs + AT_THREADS - 1) / AT_THREADS;
        const int b0 = min(tid * per, a.n_seqs), b1 = min(b0 + per, a.n_seqs);
        long long sum = 0;
        bool any_bad = false;
        for (int b = b0; b < b1; b++) {
            int f;
            bool bad;
            const int n = seq_span(a, b, f, bad);
            any_bad |= bad;
            sum += (n - f + QP - 1) / QP;
        }
        if (any_bad && blockIdx.x == 0) atomicOr(a.err, (unsigned)SE_LEN);
        long long pre = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long t = __shfl_up_sync(0xffffffffu, pre, o);
            if (lane >= o) pre += t;
        }
        if (lane == 31) s_sum[warp] = pre;
        if (tid == 0) s_b = a.n_seqs;
        __syncthreads();
        long long off = 0, all = 0;
#pragma unroll
        for (int w = 0; w < AT_WARPS; w++) {
            if (w < warp) off += s_sum[w];
            all += s_sum[w];
        }
        pre += off - sum;                              /* quanta per unit before b0 */
        const long long total = all * U;
        const long long ncta = max(1ll, min((long long)gridDim.x, (total + a.min_quanta - 1) / a.min_quanta));
        const long long lo = blockIdx.x < ncta ? share_lo(blockIdx.x, ncta, total) : total;
        const long long hi = blockIdx.x < ncta ? share_lo(blockIdx.x + 1, ncta, total) : total;
        if (lo < hi && lo >= pre * U && lo < (pre + sum) * U) {
            long long at = pre;
            int b = b0;
            for (; b < b1; b++) {
                int f;
                bool bad;
                const int n = seq_span(a, b, f, bad), nq = (n - f + QP - 1) / QP;
                if (lo < (at + nq) * U) break;
                at += nq;
            }
            s_b = b;
            s_base = at * U;
            s_lo = lo;
        }
        if (tid == 0) {
            s_cnt = (int)(hi - lo);
            s_ncta = (int)ncta;
            s_total = total;
        }
        __syncthreads();
    }
    const int cnt = s_cnt;
    /* sequences without positions: zeros */
    for (int b = blockIdx.x; b < a.n_seqs; b += gridDim.x) {
        int f;
        bool bad;
        if (seq_span(a, b, f, bad) == 0)
            for (int i = tid; i < a.n_heads * a.kv.hd; i += AT_THREADS) a.out[b * a.ldo + i] = 0.0f;
    }
    if (cnt == 0) {
        if (tid == 0) a.desc[blockIdx.x] = make_int4(-1, 0, 0, 0);
        return;
    }

    /* ---- the loader's place: sequence, unit of it, quantum of that ---- */
    int lb = s_b, first, len, nq, lu, lq;
    bool bad_;
    len = seq_span(a, lb, first, bad_);
    nq = (len - first + QP - 1) / QP;
    {
        const long long rel = s_lo - s_base;
        lu = (int)(rel / nq);
        lq = (int)(rel - (long long)lu * nq);
    }
    const int b0_ = lb, u0_ = lu, lq0 = lq;                                /* the first unit's quanta before this share */
    const long long unit0_at = s_base + (long long)lu * nq;   /* where the first unit begins */
    int left = cnt;
    const int prow = lane & (TP - 1);                  /* the tile row whose page this lane looks up */
    int pg = -1, pslot = 0;
    bool pin = false;
    auto look = [&]() {                                /* page of the lane's row of the loader's tile */
        const int p = first + (lq * AT_WARPS + warp) * TP + prow;
        pin = p < len;
        if (pin) {
            const int pi = p / a.kv.page;
            pslot = p - pi * a.kv.page;
            pg = __ldg(a.kv.table + (size_t)lb * a.kv.ld_table + pi);
        }
    };
    auto issue = [&](int stage) {
        const int g = lu / a.chunks;
        const bool ok = pin && pg >= 0 && pg < a.kv.n_pages;
        if (pin && !ok) atomicOr(a.err, (unsigned)SE_PAGE);
        const unsigned live = __ballot_sync(0xffffffffu, ok) & (unsigned)((1ull << TP) - 1);
        const unsigned row = ok ? (unsigned)(((size_t)pg * a.kv.n_kv + g) * a.kv.page + pslot) : 0u;
        const uint32_t sk = ring_s + stage * SLOT, sv = sk + 32 * HD;
        const size_t rowb = (size_t)a.kv.hd * ES;
#pragma unroll
        for (int e = 0; e < HD / 16; e++) {
            const int idx = lane + 32 * e, t = idx / CPR, ch = idx % CPR;
            const unsigned rr = __shfl_sync(0xffffffffu, row, t);
            const bool lv = ((live >> t) & 1u) && ch * 16 < (int)rowb;
            const size_t off = (size_t)rr * rowb + (lv ? ch * 16 : 0);
            int kx, vx;                                /* swizzles: which of 8 bank groups a row starts at */
            if constexpr (KV == KC_F32) {
                kx = ((t & 1) << 2) | ((t >> 1) & 3);
                vx = t & 7;
            } else {
                kx = vx = CPR >= 8 ? (t & 7) : ((t >> 1) & 3);
            }
            cp_async16z(sk + t * PITCH + ((ch ^ kx) << 4), a.kv.k + off, lv);
            cp_async16z(sv + t * PITCH + ((ch ^ vx) << 4), a.kv.v + off, lv);
        }
        if constexpr (KV == KC_Q8_0) {
            cp_async4z(sk + 64 * HD + lane * 4, a.kv.kd + row, ok);
            cp_async4z(sk + 64 * HD + 128 + lane * 4, a.kv.vd + row, ok);
        }
        if (lane == 0) info[stage] = make_int4(lb, lu, (int)live, (lq == nq - 1 || left == 1) ? (lq == nq - 1 ? 3 : 1) : 0);
    };
    auto advance = [&]() {
        left--;
        if (left == 0) return;
        if (++lq == nq) {
            lq = 0;
            if (++lu == U) {
                lu = 0;
                do {
                    if (++lb >= a.n_seqs) {            /* (lengths changed under the kernel) */
                        left = 0;
                        return;
                    }
                    len = seq_span(a, lb, first, bad_);
                    nq = (len - first + QP - 1) / QP;
                } while (nq == 0);
            }
        }
        look();
    };
    look();
#pragma unroll
    for (int s = 0; s < S - 1; s++) {
        if (left > 0) {
            issue(s);
            advance();
        }
        cp_async_commit();
    }

    /* ---- the compute side ---- */
    constexpr int QR = KV == KC_F32 ? HD / 8 * 4 : (KV == KC_F16 ? HD / 16 * 4 : HD / 32 * 2);
    unsigned qf[MT][QR];                               /* the query fragments */
    float qc[MT];                                      /* score of a raw product, times log2 e without a soft-cap */
    constexpr int NACC = HD / 4;
    float acc[MT][NACC], m[MT], l[MT];
    const float LOG2E = 1.4426950408889634f;
    int cu_b = -1, cu_u = -1;
    bool fresh = true;                                 /* the unit of the next tile begins in this share */

    auto load_q = [&](int b, int u) {
        const int g = u / a.chunks, h0 = (u - g * a.chunks) * HC, nh = min(HC, a.group - h0);
        const float *qb = a.q + b * a.ldq + (size_t)(g * a.group + h0) * a.kv.hd;
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
            const bool on = mt * 8 + r < nh;
            const float *qh = qb + (size_t)(mt * 8 + r) * a.kv.hd;
            const float post = a.softcap > 0.0f ? 1.0f : LOG2E;
            if constexpr (KV == KC_F16) {
                float x[HD / 4];
                float mx = 0.0f;
#pragma unroll
                for (int j = 0; j < HD / 16; j++)
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const int d = 16 * j + 8 * i + 2 * c;
                        float2 t = make_float2(0.0f, 0.0f);
                        if (on && d < a.kv.hd) t = __ldg((const float2 *)(qh + d));
                        x[4 * j + 2 * i] = t.x;
                        x[4 * j + 2 * i + 1] = t.y;
                        mx = fmaxf(mx, fmaxf(fabsf(t.x), fabsf(t.y)));
                    }
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                /* the largest |q| of the head is brought to [2^12, 2^13), a power of two exactly, so
                 * that the low parts of all but vanishing values stay normal f16 */
                int ex = (int)((__float_as_uint(mx) >> 23) & 255) - 127;
                ex = min(max(ex, -100), 100);
                const float up = __uint_as_float((unsigned)(127 + 12 - ex) << 23);
                qc[mt] = a.scale * __uint_as_float((unsigned)(127 - 12 + ex) << 23) * post;
#pragma unroll
                for (int j = 0; j < HD / 16; j++)
#pragma unroll
                    for (int i = 0; i < 2; i++)
                        split_f16(x[4 * j + 2 * i] * up, x[4 * j + 2 * i + 1] * up, qf[mt][4 * j + 2 * i],
                                  qf[mt][4 * j + 2 * i + 1]);
            } else if constexpr (KV == KC_F32) {
#pragma unroll
                for (int j = 0; j < HD / 16; j++) {
                    const int d = 16 * j + 4 * c;
                    float4 t = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    if (on && d < a.kv.hd) t = __ldg((const float4 *)(qh + d));
                    split_tf32(t.x, qf[mt][8 * j], qf[mt][8 * j + 1]);
                    split_tf32(t.y, qf[mt][8 * j + 2], qf[mt][8 * j + 3]);
                    split_tf32(t.z, qf[mt][8 * j + 4], qf[mt][8 * j + 5]);
                    split_tf32(t.w, qf[mt][8 * j + 6], qf[mt][8 * j + 7]);
                }
                qc[mt] = a.scale * post;
            } else {
                /* the query head quantized as a cache row is (ops/ops.c:229-233) */
                float x[HD / 4];
                float mx = 0.0f;
#pragma unroll
                for (int j = 0; j < HD / 16; j++) {
                    const int d = 16 * j + 4 * c;
                    float4 t = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    if (on && d < a.kv.hd) t = __ldg((const float4 *)(qh + d));
                    x[4 * j] = t.x; x[4 * j + 1] = t.y; x[4 * j + 2] = t.z; x[4 * j + 3] = t.w;
                    mx = fmaxf(mx, fmaxf(fmaxf(fabsf(t.x), fabsf(t.y)), fmaxf(fabsf(t.z), fabsf(t.w))));
                }
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                const bool tiny = mx < 1e-30f;
                const float id = tiny ? 0.0f : __fdiv_rn(127.0f, mx), qd = tiny ? 0.0f : __fdiv_rn(mx, 127.0f);
#pragma unroll
                for (int j = 0; j < HD / 16; j++) {
                    unsigned w = 0;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float u = truncf(__fadd_rn(__fmul_rn(x[4 * j + i], id), copysignf(0.5f, x[4 * j + i])));
                        const int qi = tiny ? 0 : (int)fminf(fmaxf(u, -127.0f), 127.0f);
                        w |= ((unsigned)qi & 0xffu) << (8 * i);
                    }
                    qf[mt][j] = w;
                }
                qc[mt] = __fmul_rn(qd, a.scale) * post;
            }
        }
    };

    /* one tile of TP positions in ring slot `stage` */
    auto compute = [&](int stage, unsigned live) {
        const uint32_t sk = ring_s + stage * SLOT, sv = sk + 32 * HD;
        float s[MT][NT][2];
        if constexpr (KV == KC_F16) {
            float d[MT][NT][4];
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int i = 0; i < 4; i++) d[mt][nt][i] = 0.0f;
            const uint32_t kb = sk + (lane & 7) * PITCH;
            const int x = (lane >> 3) ^ (lane & 7);
#pragma unroll
            for (int jj = 0; jj < HD / 32; jj++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    unsigned b[4];
                    ldsm4(b, kb + nt * 8 * PITCH + (((4 * jj) ^ x) << 4));
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) {
                        const unsigned a0[4] = { qf[mt][8 * jj], qf[mt][8 * jj + 1], qf[mt][8 * jj + 2], qf[mt][8 * jj + 3] };
                        const unsigned a1[4] = { qf[mt][8 * jj + 4], qf[mt][8 * jj + 5], qf[mt][8 * jj + 6], qf[mt][8 * jj + 7] };
                        mma_f16(d[mt][nt], a0, b[0], b[1]);
                        mma_f16(d[mt][nt], a1, b[2], b[3]);
                    }
                }
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    s[mt][nt][0] = (d[mt][nt][0] + d[mt][nt][2]) * qc[mt];
                    s[mt][nt][1] = (d[mt][nt][1] + d[mt][nt][3]) * qc[mt];
                }
        } else if constexpr (KV == KC_F32) {
            float dh[MT][4], dl[MT][4];
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int i = 0; i < 4; i++) dh[mt][i] = dl[mt][i] = 0.0f;
            const uint32_t kb = sk + r * PITCH;
            const int x = c ^ (((r & 1) << 2) | (r >> 1));
#pragma unroll
            for (int jj = 0; jj < HD / 16; jj++) {
                const float4 t = lds4(kb + (((4 * jj) ^ x) << 4));
                unsigned h[4], w[4];
                split_tf32(t.x, h[0], w[0]);
                split_tf32(t.y, h[1], w[1]);
                split_tf32(t.z, h[2], w[2]);
                split_tf32(t.w, h[3], w[3]);
#pragma unroll
                for (int mt = 0; mt < MT; mt++) {
                    const unsigned a0[4] = { qf[mt][8 * jj], qf[mt][8 * jj + 1], qf[mt][8 * jj + 2], qf[mt][8 * jj + 3] };
                    const unsigned a1[4] = { qf[mt][8 * jj + 4], qf[mt][8 * jj + 5], qf[mt][8 * jj + 6], qf[mt][8 * jj + 7] };
                    mma_tf32(dh[mt], a0, h[0], h[1]);
                    mma_tf32(dl[mt], a0, w[0], w[1]);
                    mma_tf32(dh[mt], a1, h[2], h[3]);
                    mma_tf32(dl[mt], a1, w[2], w[3]);
                }
            }
#pragma unroll
            for (int mt = 0; mt < MT; mt++) {
                s[mt][0][0] = ((dh[mt][0] + dh[mt][2]) + (dl[mt][0] + dl[mt][2])) * qc[mt];
                s[mt][0][1] = ((dh[mt][1] + dh[mt][3]) + (dl[mt][1] + dl[mt][3])) * qc[mt];
            }
        } else {
            int d[MT][NT][4];
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int i = 0; i < 4; i++) d[mt][nt][i] = 0;
            const uint32_t kb = sk + (lane & 7) * PITCH;
            const int x = (lane >> 3) ^ (CPR >= 8 ? (lane & 7) : ((lane >> 1) & 3));
#pragma unroll
            for (int jj = 0; jj < HD / 64; jj++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    unsigned b[4];
                    ldsm4(b, kb + nt * 8 * PITCH + (((4 * jj) ^ x) << 4));
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) {
                        mma_s8(d[mt][nt], qf[mt][4 * jj], qf[mt][4 * jj + 1], b[0], b[1]);
                        mma_s8(d[mt][nt], qf[mt][4 * jj + 2], qf[mt][4 * jj + 3], b[2], b[3]);
                    }
                }
            const float *kd = (const float *)(ring + stage * SLOT + 64 * HD);
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                const float2 e = *(const float2 *)(kd + nt * 8 + 2 * c);
#pragma unroll
                for (int mt = 0; mt < MT; mt++) {
                    s[mt][nt][0] = (float)d[mt][nt][0] * qc[mt] * e.x;
                    s[mt][nt][1] = (float)d[mt][nt][1] * qc[mt] * e.y;
                }
            }
        }
        /* soft-cap, mask, running softmax in base 2 */
        constexpr float LIFT = KV == KC_F32 ? 0.0f : 15.0f;   /* weights in (0, 2^15]: small ones stay normal f16 */
        float corr[MT];
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
            float mx = -INFINITY;
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    float v = s[mt][nt][i];
                    if (a.softcap > 0.0f) v = a.softcap * tanhf(__fdiv_rn(v, a.softcap)) * LOG2E;
                    v = (live >> (nt * 8 + 2 * c + i)) & 1u ? v : -INFINITY;
                    s[mt][nt][i] = v;
                    mx = fmaxf(mx, v);
                }
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const float mn = fmaxf(m[mt], mx), base = mn == -INFINITY ? 0.0f : mn;
            corr[mt] = exp2f(m[mt] - base);
            m[mt] = mn;
            float sum = 0.0f;
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const float p = exp2f(s[mt][nt][i] - base + LIFT);
                    s[mt][nt][i] = p;
                    sum += p;
                }
            l[mt] = l[mt] * corr[mt] + sum;
        }
        /* the weighted sum of V's rows */
        if constexpr (KV == KC_F16) {
            unsigned w[MT][4];
#pragma unroll
            for (int mt = 0; mt < MT; mt++) {
                split_f16(s[mt][0][0], s[mt][0][1], w[mt][0], w[mt][1]);
                split_f16(s[mt][1][0], s[mt][1][1], w[mt][2], w[mt][3]);
            }
            const uint32_t vb = sv + ((lane & 7) + (lane & 8)) * PITCH;
            const int x = (lane >> 4) ^ (lane & 7);
#pragma unroll
            for (int jj = 0; jj < HD / 16; jj++) {
                unsigned b[4];
                ldsm4t(b, vb + (((2 * jj) ^ x) << 4));
#pragma unroll
                for (int mt = 0; mt < MT; mt++) {
                    float d0[4] = { 0.0f, 0.0f, 0.0f, 0.0f }, d1[4] = { 0.0f, 0.0f, 0.0f, 0.0f };
                    mma_f16(d0, w[mt], b[0], b[1]);
                    mma_f16(d1, w[mt], b[2], b[3]);
                    float *o = &acc[mt][4 * jj];
                    o[0] = o[0] * corr[mt] + (d0[0] + d0[2]);
                    o[1] = o[1] * corr[mt] + (d0[1] + d0[3]);
                    o[2] = o[2] * corr[mt] + (d1[0] + d1[2]);
                    o[3] = o[3] * corr[mt] + (d1[1] + d1[3]);
                }
            }
        } else if constexpr (KV == KC_F32) {
            unsigned w[MT][4];
#pragma unroll
            for (int mt = 0; mt < MT; mt++) {
                split_tf32(s[mt][0][0], w[mt][0], w[mt][1]);
                split_tf32(s[mt][0][1], w[mt][2], w[mt][3]);
            }
            const uint32_t v0 = sv + (2 * c) * PITCH, v1 = v0 + PITCH;
            const int x0 = r ^ (2 * c), x1 = r ^ (2 * c + 1);
#pragma unroll
            for (int j = 0; j < HD / 32; j++) {
                const float4 ya = lds4(v0 + (((8 * j) ^ x0) << 4)), yb = lds4(v1 + (((8 * j) ^ x1) << 4));
                const float y0[4] = { ya.x, ya.y, ya.z, ya.w }, y1[4] = { yb.x, yb.y, yb.z, yb.w };
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    unsigned h0, h1, g0, g1;
                    split_tf32(y0[i], h0, g0);
                    split_tf32(y1[i], h1, g1);
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) {
                        float d0[4] = { 0.0f, 0.0f, 0.0f, 0.0f };
                        mma_tf32(d0, w[mt], g0, g1);
                        mma_tf32(d0, w[mt], h0, h1);
                        float *o = &acc[mt][8 * j + i];
                        o[0] = o[0] * corr[mt] + (d0[0] + d0[2]);
                        o[4] = o[4] * corr[mt] + (d0[1] + d0[3]);
                    }
                }
            }
        } else {
            /* the rows' scales join the weights; a power of two keeps the product in f16's range */
            const float *vd = (const float *)(ring + stage * SLOT + 64 * HD + 128);
            const float top = warp_max(fabsf(vd[lane]));
            int ex = (int)((__float_as_uint(top) >> 23) & 255) - 127;
            ex = min(max(ex, -100), 100);
            const float dn = __uint_as_float((unsigned)(127 - 1 - ex) << 23), upf = __uint_as_float((unsigned)(127 + 1 + ex) << 23);
            unsigned w[MT][2][4];
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                const float2 e = *(const float2 *)(vd + nt * 8 + 2 * c);
#pragma unroll
                for (int mt = 0; mt < MT; mt++)
                    split_f16(s[mt][nt][0] * (e.x * dn), s[mt][nt][1] * (e.y * dn), w[mt][nt >> 1][2 * (nt & 1)],
                              w[mt][nt >> 1][2 * (nt & 1) + 1]);
            }
            const uint32_t vb = sv + ((lane & 7) + (lane & 8)) * PITCH;
            const int x = (lane >> 4) ^ (CPR >= 8 ? (lane & 7) : ((lane >> 1) & 3));
            const __half2 bias = __half2half2(__ushort_as_half(0x6480));   /* 1152 */
            auto bytes = [&](unsigned u, unsigned &even, unsigned &odd) {
                /* signed bytes of two rows -> f16: 0x6400 | (v + 128) is 1024 + 128 + v */
                const unsigned v = u ^ 0x80808080u;
                unsigned e = __byte_perm(v, 0x64646464u, 0x4240), o = __byte_perm(v, 0x64646464u, 0x4341);
                even = h2u(__hsub2(*(__half2 *)&e, bias));
                odd = h2u(__hsub2(*(__half2 *)&o, bias));
            };
#pragma unroll
            for (int jj = 0; jj < HD / 32; jj++) {
                float d[MT][4][4];
#pragma unroll
                for (int mt = 0; mt < MT; mt++)
#pragma unroll
                    for (int k = 0; k < 4; k++)
#pragma unroll
                        for (int i = 0; i < 4; i++) d[mt][k][i] = 0.0f;
#pragma unroll
                for (int ks = 0; ks < 2; ks++) {
                    unsigned b[4];
                    ldsm4t(b, vb + ks * 16 * PITCH + (((2 * jj) ^ x) << 4));
                    unsigned e0, o0, e1, o1;
                    bytes(b[0], e0, o0);
                    bytes(b[1], e1, o1);
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) {
                        mma_f16(d[mt][0], w[mt][ks], e0, e1);
                        mma_f16(d[mt][1], w[mt][ks], o0, o1);
                    }
                    bytes(b[2], e0, o0);
                    bytes(b[3], e1, o1);
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) {
                        mma_f16(d[mt][2], w[mt][ks], e0, e1);
                        mma_f16(d[mt][3], w[mt][ks], o0, o1);
                    }
                }
#pragma unroll
                for (int mt = 0; mt < MT; mt++)
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        float *o = &acc[mt][8 * jj + 4 * k];
                        o[0] = o[0] * corr[mt] + (d[mt][2 * k][0] + d[mt][2 * k][2]) * upf;
                        o[1] = o[1] * corr[mt] + (d[mt][2 * k + 1][0] + d[mt][2 * k + 1][2]) * upf;
                        o[2] = o[2] * corr[mt] + (d[mt][2 * k][1] + d[mt][2 * k][3]) * upf;
                        o[3] = o[3] * corr[mt] + (d[mt][2 * k + 1][1] + d[mt][2 * k + 1][3]) * upf;
                    }
            }
        }
    };

    /* the unit's end in this share: the warps' sums together, into the output or a piece,
     * AT_COMB heads at a time */
    auto finish = [&](int b, int u, bool complete) {
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
            float t = l[mt];
            t += __shfl_xor_sync(0xffffffffu, t, 1);
            t += __shfl_xor_sync(0xffffffffu, t, 2);
            if (c == 0) {
                cml[warp * 2 * HC + mt * 8 + r] = m[mt];
                cml[warp * 2 * HC + HC + mt * 8 + r] = t;
            }
        }
        const int g = u / a.chunks, h0 = (u - g * a.chunks) * HC, nh = min(HC, a.group - h0);
        float *piece = a.part + ((size_t)2 * blockIdx.x + (fresh ? 1 : 0)) * part_floats<HD, MT>();
#pragma unroll
        for (int ps = 0; ps < HC / AT_COMB; ps++) {
            if (ps * AT_COMB >= nh) break;
            const int mt = ps / 2;
            if ((r >> 2) == (ps & 1)) {
                float *row = comb + (warp * AT_COMB + (r & 3)) * HD;
                const int x = (r & 3) * 8;             /* rows start at different banks */
#pragma unroll
                for (int j = 0; j < HD / 32; j++) {
                    if constexpr (KV == KC_F32) {
                        /* acc[8 j + i]: dim 32 j + 8 c + i */
                        float *p = row + ((32 * j + 8 * c) ^ x);
                        *(float4 *)p = make_float4(acc[mt][8 * j], acc[mt][8 * j + 1], acc[mt][8 * j + 2], acc[mt][8 * j + 3]);
                        *(float4 *)(p + 4) =
                            make_float4(acc[mt][8 * j + 4], acc[mt][8 * j + 5], acc[mt][8 * j + 6], acc[mt][8 * j + 7]);
                    } else if constexpr (KV == KC_F16) {
#pragma unroll
                        for (int k = 0; k < 4; k++)    /* acc[2 n + i]: dim 8 n + 2 c + i, n = 4 j + k */
                            *(float2 *)(row + ((32 * j + 8 * k + 2 * c) ^ x)) =
                                make_float2(acc[mt][8 * j + 2 * k], acc[mt][8 * j + 2 * k + 1]);
                    } else {
#pragma unroll
                        for (int k = 0; k < 2; k++)    /* acc[4 n + i]: dim 16 n + 4 c + i, n = 2 j + k */
                            *(float4 *)(row + ((32 * j + 16 * k + 4 * c) ^ x)) =
                                make_float4(acc[mt][8 * j + 4 * k], acc[mt][8 * j + 4 * k + 1],
                                            acc[mt][8 * j + 4 * k + 2], acc[mt][8 * j + 4 * k + 3]);
                    }
                }
            }
            __syncthreads();
            for (int idx = tid; idx < AT_COMB * (HD / 4); idx += AT_THREADS) {
                const int hl = idx / (HD / 4), h = ps * AT_COMB + hl, d = 4 * (idx - hl * (HD / 4));
                if (h >= nh) continue;
                float mw[AT_WARPS], M = -INFINITY, L = 0.0f;
#pragma unroll
                for (int w = 0; w < AT_WARPS; w++) {
                    mw[w] = cml[w * 2 * HC + h];
                    M = fmaxf(M, mw[w]);
                }
                const float base = M == -INFINITY ? 0.0f : M;
                float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int w = 0; w < AT_WARPS; w++) {
                    const float f = exp2f(mw[w] - base);
                    const float4 t = *(const float4 *)(comb + (w * AT_COMB + hl) * HD + (d ^ (hl * 8)));
                    L += f * cml[w * 2 * HC + HC + h];
                    o.x += f * t.x;
                    o.y += f * t.y;
                    o.z += f * t.z;
                    o.w += f * t.w;
                }
                if (complete) {
                    if (d < a.kv.hd)
                        *(float4 *)(a.out + b * a.ldo + (size_t)(g * a.group + h0 + h) * a.kv.hd + d) = over(o, L);
                } else {
                    *(float4 *)(piece + h * HD + d) = o;
                    if (d == 0) {
                        piece[HC * HD + h] = M;
                        piece[HC * HD + HC + h] = L;
                    }
                }
            }
            __syncthreads();
        }
    };

    bool join = false, first_unit = true;
    for (int it = 0; it < cnt; it++) {
        cp_async_wait_but<S - 2>();
        __syncwarp();
        if (left > 0) {
            issue((it + S - 1) % S);
            advance();
        }
        cp_async_commit();
        const int stage = it % S;
        const int4 f = info[stage];
        if (f.x != cu_b || f.y != cu_u) {
            cu_b = f.x;
            cu_u = f.y;
            fresh = it > 0 || lq0 == 0;
            load_q(cu_b, cu_u);
#pragma unroll
            for (int mt = 0; mt < MT; mt++) {
                m[mt] = -INFINITY;
                l[mt] = 0.0f;
#pragma unroll
                for (int i = 0; i < NACC; i++) acc[mt][i] = 0.0f;
            }
        }
        if (f.z) compute(stage, (unsigned)f.z);
        if (f.w & 1) {
            if (first_unit) join = !fresh && (f.w & 2);
            first_unit = false;
            finish(cu_b, cu_u, fresh && (f.w & 2));
        }
    }
    /* the first unit began in another CTA's share and ends in this one: from which CTA on it is to be joined
     * (the last whose share begins at or before the unit) */
    if (tid == 0)
        a.desc[blockIdx.x] =
            join ? make_int4(b0_, u0_, (int)(((unit0_at + 1) * s_ncta - 1) / s_total), 0) : make_int4(-1, 0, 0, 0);
}

/* The pieces of units that more than one CTA's share holds, summed in the
 * CTAs' order: block i joins the unit whose last piece is CTA i's, a warp per
 * head. Few and small: its time is a launch's latency, part of which the
 * programmatic launch hides. */
constexpr int JN_THREADS = 256;
template <int HD, int MT>
__global__ void __launch_bounds__(JN_THREADS) paged_join_kernel(const __grid_constant__ AttendArgs a) {
    cudaGridDependencySynchronize();
    const int4 d = a.desc[blockIdx.x];
    if (d.x < 0) return;
    constexpr int HC = 8 * MT, PF = part_floats<HD, MT>(), NV = HD > 128 ? 2 : 1;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c1 = blockIdx.x;
    const int g = d.y / a.chunks, h0 = (d.y - g * a.chunks) * HC, nh = min(HC, a.group - h0);
    auto piece = [&](int c) { return a.part + ((size_t)2 * c + (c == d.z ? 1 : 0)) * PF; };
    for (int h = warp; h < nh; h += JN_THREADS / 32) {
        float M = -INFINITY;
        for (int k = d.z + lane; k <= c1; k += 32) M = fmaxf(M, piece(k)[HC * HD + h]);
        M = warp_max(M);
        const float base = M == -INFINITY ? 0.0f : M;
        float4 o[NV];
        float L = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; j++) o[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
        for (int k = d.z; k <= c1; k++) {
            const float *p = piece(k);
            const float f = exp2f(p[HC * HD + h] - base);
            L += f * p[HC * HD + HC + h];
#pragma unroll
            for (int j = 0; j < NV; j++) {
                const int e = 4 * lane + 128 * j;
                if (e < HD) {
                    const float4 t = *(const float4 *)(p + h * HD + e);
                    o[j].x += f * t.x;
                    o[j].y += f * t.y;
                    o[j].z += f * t.z;
                    o[j].w += f * t.w;
                }
            }
        }
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int e = 4 * lane + 128 * j;
            if (e < a.kv.hd) *(float4 *)(a.out + d.x * a.ldo + (size_t)(g * a.group + h0 + h) * a.kv.hd + e) = over(o[j], L);
        }
    }
}

}  // namespace kc
