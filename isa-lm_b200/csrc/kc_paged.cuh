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
#include <climits>
#include <cstdint>
#include <type_traits>

#include "kc_kernels.cuh"
#include "krafla_cuda.h"

namespace kc {

/* error bits of the serving operators' word */
enum { SE_HIST = 1, SE_BIAS = 2, SE_LEN = 4, SE_PAGE = 8, SE_ROW = 16 };

/* n / d for 0 <= n < 2^31 as the high half of n * mul, shifted: with 2^(s-1) < d <= 2^s, mul = 2^(31+s) / d rounded up
 * is off by less than 2^s / d / 2^31 of itself, which no such n turns into a quotient */
struct Divisor {
    unsigned mul = 0;
    int shift = 0;
    Divisor() = default;                               /* by 1 */
    explicit Divisor(int d) {
        int s = 0;
        while ((1ll << s) < d) s++;
        if (s) mul = (unsigned)(((1ull << (31 + s)) + (unsigned)d - 1) / (unsigned)d);
        shift = s - 1;
    }
    __device__ __forceinline__ int operator()(int n) const { return mul ? (int)(__umulhi((unsigned)n, mul) >> shift) : n; }
};

struct PagedKV {
    uint8_t *k, *v;
    float *kd, *vd;
    const int *table;
    int n_seqs, ld_table, n_pages, page, n_kv, hd;
    Divisor page_of;             /* p / page */
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
    int tasks;                   /* warps of a row */
    Divisor row_of;              /* warp / tasks */
    unsigned *err;
};

constexpr int AP_THREADS = 256;
/* heads that a group of lanes takes at once */
template <int NV>
constexpr int ap_heads() { return NV == 1 ? 4 : 2; }

/* The sum over the LPH lanes that hold a head's row. */
template <int LPH, class T>
__device__ __forceinline__ T head_sum(T v) {
#pragma unroll
    for (int o = LPH / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

/* 1 / sqrt(mean(x^2) + eps) of each of a lane's NH heads, in type T. The root
 * and the division are taken once for all of them: lane k of a group does head
 * k's and hands it round. */
template <class T, int LPH, int NV, int NH>
__device__ __forceinline__ void head_norms(const float (&x)[NH][NV][4], T (&inv)[NH], float eps, int hd) {
    T mine = (T)0;
#pragma unroll
    for (int k = 0; k < NH; k++) {
        T s = (T)0;
#pragma unroll
        for (int j = 0; j < NV; j++)
#pragma unroll
            for (int i = 0; i < 4; i++) s += (T)x[k][j][i] * (T)x[k][j][i];
        s = head_sum<LPH>(s);
        if (threadIdx.x % NH == k) mine = s;
    }
    if constexpr (sizeof(T) == 8) mine = 1.0 / sqrt(mine / (double)hd + (double)eps);
    else mine = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(mine, (float)hd), eps)));
#pragma unroll
    for (int k = 0; k < NH; k++) inv[k] = __shfl_sync(0xffffffffu, mine, k, LPH);
}

/* y = x inv w, then the rotation of adjacent pairs, of 4 * NV values of a head, in type T. */
template <class T, int NV>
__device__ __forceinline__ void norm_rope(float (&x)[NV][4], bool norm, T inv, const float4 (&w)[NV], const float2 (&cs)[NV],
                                          const float2 (&sn)[NV]) {
#pragma unroll
    for (int j = 0; j < NV; j++) {
        T a = (T)x[j][0], b = (T)x[j][1], e = (T)x[j][2], f = (T)x[j][3];
        if (norm) {
            a = a * inv * (T)w[j].x;
            b = b * inv * (T)w[j].y;
            e = e * inv * (T)w[j].z;
            f = f * inv * (T)w[j].w;
        }
        x[j][0] = (float)(a * (T)cs[j].x - b * (T)sn[j].x);
        x[j][1] = (float)(a * (T)sn[j].x + b * (T)cs[j].x);
        x[j][2] = (float)(e * (T)cs[j].y - f * (T)sn[j].y);
        x[j][3] = (float)(e * (T)sn[j].y + f * (T)cs[j].y);
    }
}

/* Measured: 4096 rows of 32 + 8 + 8 heads of 128 into an f16 cache 30.6 us a call in
 * a run of them (187 MB, floor 28.9 at a copy's rate), 34.6 us where the rows come
 * from memory; as many normed into an 8-bit cache 42.9 us (floor 27.6), the
 * difference mostly the conversions to 64 bits and back.
 *
 * A warp takes four heads (two wide ones) of one kind (queries, keys or values)
 * of a row for each of its groups of LPH lanes, 4 * NV values of a head a lane. Bound by
 * memory: every value is read once and written once, so all of a warp's heads
 * are requested before anything waits, and the row's place in the cache (three
 * dependent loads), its angles and the norm's weights are fetched once for them.
 *
 * K rows of an 8-bit cache are normed and rotated in 64 bits and rounded once,
 * so that which side of a step's border a value falls on does not depend on
 * the order of the norm's sum; queries and wider caches use 32 bits. */
template <int KV, int LPH, int NV>
__global__ void __launch_bounds__(AP_THREADS, KV == KC_Q8_0 ? (NV == 1 ? 4 : 3) : (NV == 1 ? 5 : 4)) append_kernel(const AppendArgs a) {
    launch_next();
    stream_order();
    constexpr int NH = ap_heads<NV>(), HW = NH * (32 / LPH);   /* heads per lane group and per warp */
    const int lane = threadIdx.x % LPH, sub = threadIdx.x % 32 / LPH, hd = a.kv.hd;
    const int tq = (a.n_heads + HW - 1) / HW, tk = (a.kv.n_kv + HW - 1) / HW;
    const int item = (int)(blockIdx.x * (AP_THREADS / 32) + threadIdx.x / 32), row = a.row_of(item), task = item - row * a.tasks;
    if (row >= a.rows) return;                         /* (whole warps) */
    const bool isq = task < tq, isv = task >= tq + tk;
    const int h0 = HW * (isq ? task : (isv ? task - tq - tk : task - tq)) + sub, nh = isq ? a.n_heads : a.kv.n_kv;
    const float *src = isq ? a.q + row * a.ldq : (isv ? a.v + row * a.ldv : a.k + row * a.ldk);
    const int seq = a.seqs ? a.seqs[row] : row, p = a.pos[row];
    if (seq < 0) return;                               /* padding */
    float x[NH][NV][4];
#pragma unroll
    for (int k = 0; k < NH; k++)
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int d = 4 * (lane + j * LPH), h = h0 + k * (32 / LPH);
            float4 t = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (h < nh && d < hd) t = load_once(src + (size_t)h * hd + d);
            x[k][j][0] = t.x; x[k][j][1] = t.y; x[k][j][2] = t.z; x[k][j][3] = t.w;
        }
    const int pi = p >= 0 ? a.kv.page_of(p) : 0, slot = p - pi * a.kv.page;
    bool ok = seq < a.kv.n_seqs && p >= 0 && p < a.n_pos && pi < a.kv.ld_table;
    int page = 0;
    if (ok) {
        page = a.kv.table[(size_t)seq * a.kv.ld_table + pi];
        ok = page >= 0 && page < a.kv.n_pages;
    }
    if (!ok) {
        if (threadIdx.x % 32 == 0) atomicOr(a.err, (unsigned)SE_ROW);
        return;
    }
    if (!isv) {
        const float *wt = isq ? a.q_norm : a.k_norm;
        float4 w[NV];
        float2 cs[NV], sn[NV];
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int d = 4 * (lane + j * LPH);
            cs[j] = sn[j] = make_float2(0.0f, 0.0f);
            w[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (d < hd) {
                cs[j] = *(const float2 *)(a.cos + (size_t)p * (hd / 2) + d / 2);
                sn[j] = *(const float2 *)(a.sin + (size_t)p * (hd / 2) + d / 2);
                if (wt) w[j] = *(const float4 *)(wt + d);
            }
        }
        auto turn = [&](auto one) {
            using T = decltype(one);
            T inv[NH];
            if (wt) head_norms<T, LPH, NV, NH>(x, inv, a.eps, hd);
#pragma unroll
            for (int k = 0; k < NH; k++) norm_rope<T, NV>(x[k], wt != nullptr, wt ? inv[k] : one, w, cs, sn);
        };
        if (KV == KC_Q8_0 && !isq) turn(1.0);
        else turn(1.0f);
    }
    if (isq) {
        float *dst = a.q_out + row * a.ldo;
#pragma unroll
        for (int k = 0; k < NH; k++)
#pragma unroll
            for (int j = 0; j < NV; j++) {
                const int d = 4 * (lane + j * LPH), h = h0 + k * (32 / LPH);
                if (h < nh && d < hd)
                    *(float4 *)(dst + (size_t)h * hd + d) = make_float4(x[k][j][0], x[k][j][1], x[k][j][2], x[k][j][3]);
            }
        return;
    }
    uint8_t *pool = isv ? a.kv.v : a.kv.k;
    const size_t r0 = (size_t)page * a.kv.n_kv * a.kv.page + slot;
    /* the single-scale row rule of the model's 8-bit cache (ops/ops.c:81-96), its two divisions as the norms' */
    float id[NH];
    if constexpr (KV == KC_Q8_0) {
        float mine = 0.0f;
#pragma unroll
        for (int k = 0; k < NH; k++) {
            float amax = 0.0f;
#pragma unroll
            for (int j = 0; j < NV; j++)               /* (values beyond the head are zero) */
                amax = fmaxf(amax, fmaxf(fmaxf(fabsf(x[k][j][0]), fabsf(x[k][j][1])), fmaxf(fabsf(x[k][j][2]), fabsf(x[k][j][3]))));
#pragma unroll
            for (int o = LPH / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
            if (threadIdx.x % NH == k) mine = amax;
        }
        const bool tiny = mine < 1e-30f;
        const float mid = tiny ? 0.0f : __fdiv_rn(127.0f, mine);
        const int h = h0 + lane * (32 / LPH);          /* lane k holds head k's */
        if (lane < NH && h < nh)
            (isv ? a.kv.vd : a.kv.kd)[r0 + (size_t)h * a.kv.page] = tiny ? 0.0f : __fdiv_rn(mine, 127.0f);
#pragma unroll
        for (int k = 0; k < NH; k++) id[k] = __shfl_sync(0xffffffffu, mid, k, LPH);
    }
#pragma unroll
    for (int k = 0; k < NH; k++) {
        const int h = h0 + k * (32 / LPH);
        const size_t r = r0 + (size_t)h * a.kv.page;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int d = 4 * (lane + j * LPH);
            if (h >= nh || d >= hd) continue;
            const float *y = x[k][j];
            if constexpr (KV == KC_F32) {
                ((float4 *)pool)[(r * hd + d) / 4] = make_float4(y[0], y[1], y[2], y[3]);
            } else if constexpr (KV == KC_F16) {
                __half2 lo = __floats2half2_rn(y[0], y[1]), hi = __floats2half2_rn(y[2], y[3]);
                ((uint2 *)pool)[(r * hd + d) / 4] = make_uint2(*(unsigned *)&lo, *(unsigned *)&hi);
            } else {
                /* rounded half away from zero: at most 127.5 and a rounding, never 128 */
                int q[4];
#pragma unroll
                for (int i = 0; i < 4; i++) q[i] = __float2int_rz(__fadd_rn(__fmul_rn(y[i], id[k]), copysignf(0.5f, y[i])));
                ((unsigned *)pool)[(r * hd + d) / 4] =
                    __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
            }
        }
    }
}

/* ------------------------------------------------------------ attention */

/* out = sum_t exp(s_t - m) v_t / sum_t exp(s_t - m), s_t = q . k_t * scale (or
 * softcap * tanh of that over softcap) for t in [max(0, len - window), len).
 *
 * Work is cut into quanta of AT_WARPS tiles of TP positions of one unit (a
 * sequence's KV head, or a chunk of 8 * MT of its query heads). All units in a
 * row, each unit_cost quanta's time for itself and one for each quantum, are
 * shared out evenly over the CTAs, so that ragged lengths leave none idle; a
 * CTA's share may begin and end inside a unit: it then leaves its piece in the
 * workspace, and the CTA that brings a unit's last missing piece joins them all,
 * in the CTAs' order, so that the result does not depend on who came last.
 * Within a quantum each warp has a tile, its own ring of shared-memory slots
 * (cp.async) and its own running softmax; the warps meet once per unit.
 *
 * Both products run on the tensor cores with the query heads as the 16-row
 * side: rows 0-7 hold the high halves of eight heads' values, rows 8-15 what
 * the high halves leave (two f16 of 11 bits each, or two tf32), so a product
 * keeps 22 bits of a 32-bit query or softmax weight, at no more instructions
 * than one f16 row block takes. The sums of a tile leave the tensor core once
 * per tile and are carried in f32. (Up to 16 query rows against rows that are
 * used once: a product of this shape has 4 operations a byte and wants warps
 * that load for themselves; mma.sync at its operands' rate is far from bounding
 * it, tcgen05's 128-row tiles would be 7/8 padding.)
 *
 * What bounds it: the cache's bytes, read once. 64 sequences of 2048..8192
 * positions (32 heads on 8, head 128, f16, 1.34 GB) 211 us in a long run, 6.4 TB/s,
 * what a copy reaches; 2 of 131072 177 us, 5.8 TB/s. Where the bytes are fewer the
 * warps' own work shows: splitting an f32 value takes four integer and float
 * instructions, an 8-bit one a fifth of a word's five, in chains that 12 warps an
 * SM do not hide (0.36 instructions issued a cycle; 64 of 4096, head 64, 8-bit:
 * 61 us at a floor of 44, 65 in a long run; 32 of 2048, head 64, f32: 52 at 41, in
 * a long run 56). Where more than 8 heads share a KV head, f32 and heads above 128
 * go over the rows once for every 8 (kc_serve.cu: the instances). Small calls are
 * bound by their chain of latencies: 128 positions, head 64, f16 4.3 us (a tile a
 * warp), f32 6.0 (two): launch, length, table, rows, products, the warps' meeting;
 * a joined unit 3 us more (of which its pieces' sums 1.5). */
constexpr int AT_WARPS = 4;
constexpr int AT_THREADS = AT_WARPS * 32;
/* Quanta of a unit that is not worth sharing out where every unit has a CTA of its own: of 5 quanta, 78 units 11.2 us
 * instead of 12.5, 8 units 9.9 instead of 9.1. */
constexpr int AT_SHORT = 5;
constexpr int AT_COMB = 4;                /* heads that the warps of a CTA put together at a time */

template <int KV>
constexpr int att_es() { return KV == KC_F32 ? 4 : (KV == KC_F16 ? 2 : 1); }
/* positions of a warp's tile: 32 * TM bytes of each dimension */
template <int KV, int TM>
constexpr int att_tp() { return 32 / att_es<KV>() * TM; }

struct AttendArgs {
    PagedKV kv;
    const float *q;
    float *out;
    long long ldq, ldo;
    const int *lens;
    int n_seqs, n_heads, group, chunks;   /* chunks: head chunks per KV head */
    int window;
    float scale, softcap, inv_softcap;
    int unit_cost;                        /* a unit's own time, in quanta */
    float join_cost;                      /* a piece's time in the joining, in quanta */
    unsigned long long grid_inv;          /* 2^64 / CTAs, rounded up */
    int near;                             /* a tile's pages lie within 32 entries of its table row */
    unsigned *count;                      /* [CTAs] pieces that have come, of the unit that ends there; 0 between calls */
    float *part;                          /* [2 * CTAs] pieces */
    unsigned *err;
};

/* One piece of a unit: 8 * MT heads' sums [HD], then their maxima, then their weights' sums. */
template <int HD, int MT>
constexpr int part_floats() { return 8 * MT * (HD + 2); }

__device__ __forceinline__ void cp_async16s(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src));
}
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
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
/* the product alone, without a sum to add it to */
__device__ __forceinline__ void mma_f16_first(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void mma_tf32_first(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
/* the same from four times `init`; rows 8-15 of A are zero */
__device__ __forceinline__ void mma_s8_first(int (&c)[4], unsigned a0, unsigned a2, unsigned b0, unsigned b1, int init) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %5}, {%7, %8}, {%9, %9, %9, %9};"
        : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3]) : "r"(a0), "r"(0), "r"(a2), "r"(b0), "r"(b1), "r"(init));
}
/* rows 8-15 of A are zero */
__device__ __forceinline__ void mma_s8(int (&c)[4], unsigned a0, unsigned a2, unsigned b0, unsigned b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %5}, {%7, %8}, {%0, %1, %2, %3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(0), "r"(a2), "r"(b0), "r"(b1));
}

__device__ __forceinline__ unsigned h2u(__half2 h) { return *(unsigned *)&h; }
/* a float as two tf32: the nearest above or below, and what it leaves (|.| <= 2^-10 of it, of which
 * 11 bits are kept); integer operations, since the conversion instruction runs at a fraction of their rate */
__device__ __forceinline__ void split_tf32(float a, unsigned &hi, unsigned &lo) {
    hi = __float_as_uint(a) & 0xffffe000u;
    lo = (__float_as_uint(a - __uint_as_float(hi)) + 0x1000u) & 0xffffe000u;
}
/* 2^x, 0 below 2^-126 (relative error 2^-22) */
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
/* two f32 at once */
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n add.rn.f32x2 z, x, y;\n mov.b64 {%0, %1}, z;\n}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("{\n .reg .b64 x, y, z, w;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mov.b64 z, {%6, %7};\n"
        " fma.rn.f32x2 w, x, y, z;\n mov.b64 {%0, %1}, w;\n}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 r;
    asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mul.rn.f32x2 z, x, y;\n mov.b64 {%0, %1}, z;\n}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
/* two floats as f16 pairs: the high parts, and what they leave */
__device__ __forceinline__ void split_f16(float2 a, unsigned &hi, unsigned &lo) {
    const __half2 h = __floats2half2_rn(a.x, a.y);
    const float2 r = fma2(__half22float2(h), make_float2(-1.0f, -1.0f), a);
    hi = h2u(h);
    lo = h2u(__floats2half2_rn(r.x, r.y));
}
/* rows 0-7 and 8-15 of a product together */
__device__ __forceinline__ float2 halves(const float (&d)[4]) { return add2(make_float2(d[0], d[1]), make_float2(d[2], d[3])); }

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

/* Shared memory: a ring of S slots for each warp (a tile's K rows, then its V
 * rows; on a boundary of 1024 bytes, so that a row's chunk is reached by an
 * exclusive or on the address), their 8-bit rows' scales, what each slot holds,
 * and finish's part. */
template <int HD, int TM>
constexpr int slot_bytes() { return 2 * 32 * TM * HD; }
template <int KV, int HD, int TM, int MT, int S>
constexpr int attend_smem() {
    return 1024 + AT_WARPS * (S * (slot_bytes<HD, TM>() + (KV == KC_Q8_0 ? 8 * att_tp<KV, TM>() : 0) + 16) +
                              AT_COMB * HD * 4 + 2 * 8 * MT * 4);
}

/* sum / weights; nothing attended gives zeros */
__device__ __forceinline__ float4 over(float4 o, float l) {
    const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
    return make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
}

/* The pieces of CTAs c0..c1 of one unit into the output, AT_THREADS / runs
 * times four outputs at a time: their parts of as many pieces as fit into the
 * ring's memory are copied there at once, so that they take one latency and few
 * instructions (which are fetched for the first time here); then every four
 * outputs are summed by `runs` neighbouring lanes, which meet in shuffles. */
template <int HD, int MT>
__device__ __noinline__ void join_pieces(const AttendArgs &a, int b, int u, int c0, int c1, unsigned char *mem, int bytes) {
    constexpr int HC = 8 * MT, PF = part_floats<HD, MT>(), ML = HC / 2;   /* 16-byte units of the maxima and sums */
    const int tid = threadIdx.x;
    const int g = u / a.chunks, h0 = (u - g * a.chunks) * HC, nh = min(HC, a.group - h0), outs = nh * (HD / 4);
    int runs = 1;
    while (2 * runs * outs <= AT_THREADS) runs *= 2;
    const int lots = AT_THREADS / runs, pitch = 16 * (lots + ML), fit = bytes / pitch, run = tid % runs;
    for (int i0 = 0; i0 < outs; i0 += lots) {
        const int idx = i0 + tid / runs, h = min(idx, outs - 1) / (HD / 4), e = 4 * (idx - h * (HD / 4));
        float M = -INFINITY, L = 0.0f;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int k0 = c0; k0 <= c1; k0 += fit) {
            const int n = min(fit, c1 - k0 + 1);
            const float *p = a.part + ((size_t)2 * k0 + (k0 == c0 ? 1 : 0)) * PF;
            uint32_t to = smem_u32(mem) + 16 * tid;
            for (int j = 0; j < n; j++) {
                if (tid < lots && i0 + tid < outs) cp_async16s(to, p + 4 * (i0 + tid));
                if (tid < ML) cp_async16s(to + 16 * lots, p + HC * HD + 4 * tid);
                p += (j == 0 && k0 == c0 ? 1 : 2) * PF;
                to += pitch;
            }
            cp_async_commit();
            cp_async_wait_all();
            __syncthreads();
            const unsigned char *at = mem + run * pitch, *end = mem + n * pitch;
            const float *ml = (const float *)(at + 16 * lots) + h;
            float mn = M;
            for (int j = run; j < n; j += runs) mn = fmaxf(mn, *(const float *)((const unsigned char *)ml + (j - run) * pitch));
            const float base = mn == -INFINITY ? 0.0f : mn, f0 = ex2(M - base);
            M = mn;
            L *= f0;
            o = make_float4(o.x * f0, o.y * f0, o.z * f0, o.w * f0);
#pragma unroll 4
            for (; at < end; at += runs * pitch) {
                ml = (const float *)(at + 16 * lots) + h;
                const float f = ex2(ml[0] - base);
                const float4 t = *(const float4 *)(at + 16 * (idx - i0));
                L += f * ml[HC];
                o.x += f * t.x;
                o.y += f * t.y;
                o.z += f * t.z;
                o.w += f * t.w;
            }
            __syncthreads();
        }
        for (int d = 1; d < runs; d *= 2) {
            const float m2 = __shfl_xor_sync(0xffffffffu, M, d), mn = fmaxf(M, m2), base = mn == -INFINITY ? 0.0f : mn;
            const float f1 = ex2(M - base), f2 = ex2(m2 - base);
            /* the lower run first, on both sides */
            auto both = [&](float v) { const float w = __shfl_xor_sync(0xffffffffu, v, d); return run & d ? f2 * w + f1 * v : f1 * v + f2 * w; };
            L = both(L);
            o = make_float4(both(o.x), both(o.y), both(o.z), both(o.w));
            M = mn;
        }
        if (idx < outs && run == 0 && e < a.kv.hd)
            *(float4 *)(a.out + b * a.ldo + (size_t)(g * a.group + h0 + h) * a.kv.hd + e) = over(o, L);
    }
}

template <int KV, int HD, int TM, int MT, int S, int OCC>
__global__ void __launch_bounds__(AT_THREADS, OCC) paged_attend_kernel(const __grid_constant__ AttendArgs a) {
    constexpr int ES = att_es<KV>(), TP = att_tp<KV, TM>(), QP = AT_WARPS * TP;
    constexpr int PITCH = HD * ES, CPR = PITCH / 16;   /* bytes and 16-byte chunks of a row */
    constexpr int NT = TP / 8;                         /* 8-position column blocks of the scores */
    constexpr int LK = TP > 32 ? TP / 32 : 1;          /* tile rows whose page a lane looks up */
    constexpr int RW = TP / LK;
    constexpr int SLOT = slot_bytes<HD, TM>(), VOFF = TP * PITCH, SCALES = KV == KC_Q8_0 ? 2 * TP : 0;
    constexpr int HC = 8 * MT;
    extern __shared__ __align__(128) unsigned char at_raw[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int r = lane >> 2, c = lane & 3;             /* fragment row (head) and column group */
    unsigned char *slots = at_raw + (-smem_u32(at_raw) & 1023u);
    const uint32_t ring_s = smem_u32(slots) + (uint32_t)(warp * S * SLOT);
    float *scl = (float *)(slots + AT_WARPS * S * SLOT) + warp * S * SCALES;   /* K's and V's row scales of each slot */
    int4 *info = (int4 *)(slots + AT_WARPS * S * (SLOT + SCALES * 4)) + warp * S;   /* what each slot holds */
    float *comb = (float *)(slots + AT_WARPS * S * (SLOT + SCALES * 4 + 16));  /* finish: the warps' sums */
    float *cml = comb + AT_WARPS * AT_COMB * HD;       /* and their maxima and weights' sums */
    const int U = a.kv.n_kv * a.chunks;                /* units per sequence */
    const int W = a.unit_cost;
    stream_order();

    /* ---- this CTA's share: [i chunk, (i + 1) chunk) of the units' times, laid end to end; every warp
     * finds it by itself, a run of sequences a lane ---- */
    int lb, first, len, lu, lq, nq;                    /* the loader's place: sequence, unit of it, quantum of that */
    long long ubase, chunk;                            /* where the loader's unit begins */
    int left;                                          /* time to the share's end */
    bool bad_;
    {
        const int per = (a.n_seqs + 31) / 32, b0 = min(lane * per, a.n_seqs), b1 = min(b0 + per, a.n_seqs);
        int most = 0, sum = 0;                         /* a unit's worth of the run's time (fewer than 2^31 in all) */
        bool none = false, far = (long long)a.n_seqs * U > gridDim.x, any_bad = false;
        for (int b = b0; b < b1; b++) {
            len = seq_span(a, b, first, bad_);
            const int t = len > 0 ? (len - first + QP - 1) / QP + W : 0;
            sum += t;
            most = max(most, t);
            none |= t == 0;
            far |= t > AT_SHORT + W;
            any_bad |= bad_;
        }
        if (any_bad && blockIdx.x == 0) atomicOr(a.err, (unsigned)SE_LEN);
        int pre = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, pre, o);
            if (lane >= o) pre += t;
        }
        const int all = __shfl_sync(0xffffffffu, pre, 31);
        pre -= sum;
        /* sequences without positions: zeros */
        if (__any_sync(0xffffffffu, none))
            for (int b = blockIdx.x; b < a.n_seqs; b += gridDim.x)
                if (seq_span(a, b, first, bad_) == 0)
                    for (int i = tid; i < a.n_heads * a.kv.hd; i += AT_THREADS) a.out[b * a.ldo + i] = 0.0f;
        if (!__any_sync(0xffffffffu, far)) {
            /* short sequences, a CTA for each unit: joining would take longer than it saved */
            lb = blockIdx.x / U;
            lu = blockIdx.x % U;
            if (lb >= a.n_seqs) return;
            len = seq_span(a, lb, first, bad_);
            nq = (len - first + QP - 1) / QP;
            lq = 0;
            left = nq;
            ubase = 0;
            chunk = 1ll << 40;
        } else {
            const long long total = (long long)all * U;
            /* total / CTAs rounded up: grid_inv is 2^64 / CTAs rounded up, so the product's high half is the
             * quotient or one more */
            long long q = (long long)__umul64hi((unsigned long long)total, a.grid_inv);
            q -= q * gridDim.x > total;
            /* n quanta in shares of c take c of them and the joining of n / c pieces: least at c = sqrt(n join_cost) */
            chunk = max(q + (q * gridDim.x < total), (long long)sqrtf((float)__reduce_max_sync(0xffffffffu, most) * a.join_cost));
            const long long lo = blockIdx.x * chunk, hi = min(lo + chunk, total);
            if (lo >= hi) return;
            /* the lane whose run holds lo, and the sequence in it */
            const unsigned at = __ballot_sync(0xffffffffu, lo >= (long long)pre * U && lo < ((long long)pre + sum) * U);
            const int own = __ffs(at) - 1;
            int b = __shfl_sync(0xffffffffu, b0, own), p = __shfl_sync(0xffffffffu, pre, own);
            for (;; b++) {
                len = seq_span(a, b, first, bad_);
                nq = (len - first + QP - 1) / QP;
                const int t = nq > 0 ? nq + W : 0;
                if (lo < ((long long)p + t) * U || b + 1 >= a.n_seqs) break;
                p += t;
            }
            lb = b;
            const long long rel = lo - (long long)p * U;
            lu = rel >> 31 ? (int)(rel / (nq + W)) : (int)((unsigned)rel / (unsigned)(nq + W));
            const int off = (int)(rel - (long long)lu * (nq + W));
            lq = max(0, off - W);
            ubase = lo - off;
            left = (int)min(hi - ubase, 1ll << 30) - W - lq;
        }
        if (left <= 0) return;                         /* (the same for the CTA's warps) */
    }
    const int b0_ = lb, u0_ = lu;
    const bool whole0 = lq == 0;                       /* the first unit begins in this share */
    const int nq0 = nq;
    const long long ubase0 = ubase;
    const int prow = lane & (RW - 1);
    int ql = nq - lq, p0 = first + (lq * AT_WARPS + warp) * TP, lg = lu / a.chunks;   /* quanta left, the tile's first position, KV head */
    /* 32 entries of the sequence's table row from tb0 on, an entry a lane; a tile's are among them unless
     * pages are so short that it may span more (a.near 0), where each row's entry is loaded */
    int tab = -1, tb0 = 0, tbn = 0;
    unsigned live[LK], row[LK];                        /* of the loader's tile: rows that are there, and where */
    bool full;                                         /* all of them */
    auto look = [&]() {
        const int n = len - p0;                        /* positions of the tile, 0 or fewer: none */
        full = false;
#pragma unroll
        for (int k = 0; k < LK; k++) live[k] = row[k] = 0u;
        if (n <= 0) return;
        if (a.near) {
            const int i0 = a.kv.page_of(p0);
            if (i0 < tb0 || p0 + min(n, TP) > tbn) {
                tb0 = i0;
                tbn = (int)min((long long)(tb0 + 32) * a.kv.page, (long long)INT_MAX);
                tab = tb0 + lane < a.kv.ld_table ? a.kv.table[(size_t)lb * a.kv.ld_table + tb0 + lane] : -1;
            }
        }
        full = true;
#pragma unroll
        for (int k = 0; k < LK; k++) {
            const int o = k * RW + prow, pi = a.kv.page_of(p0 + o);
            const bool in = o < n;
            int pg = __shfl_sync(0xffffffffu, tab, (pi - tb0) & 31);
            if (!a.near) pg = in ? a.kv.table[(size_t)lb * a.kv.ld_table + pi] : -1;
            const bool ok = in && (unsigned)pg < (unsigned)a.kv.n_pages;
            if (in && !ok) atomicOr(a.err, (unsigned)SE_PAGE);
            live[k] = __ballot_sync(0xffffffffu, ok) & (unsigned)((1ull << RW) - 1);
            full &= live[k] == (unsigned)((1ull << RW) - 1);
            if (ok) row[k] = ((unsigned)pg * a.kv.n_kv + lg) * a.kv.page + (p0 + o - pi * a.kv.page);
        }
    };
    enum { LAST_OF_UNIT = 1 << 28, LAST_OF_SHARE = 1 << 29 };
    /* Rows start at different bank groups, by an exclusive or of the 16-byte chunk's number with swz(row): for
     * row-per-lane reads of eight rows (ldmatrix, and f32 V) the row's low bits, or the next ones where two rows
     * share 128 bytes; for f32 K, read by four lanes a row and eight rows in turn, the low bits reversed. */
    constexpr int SWV = CPR >= 8 ? 0 : 1, SWK = KV == KC_F32 ? 2 : SWV;
    auto swz = [](int sw, int t) { return sw == 0 ? (t & 7) : (sw == 1 ? ((t >> 1) & 3) : (((t & 1) << 2) | ((t >> 1) & 3))); };
    /* a lane's chunk of the warp's e-th 512 bytes: row te + tl, te a constant of e whose bits tl has not */
    const int tl = CPR < 32 ? lane / CPR : 0, cl = lane % (CPR < 32 ? CPR : 32);
    auto copy_rows = [&](uint32_t sk) {
        constexpr int RE = CPR < 32 ? 32 / CPR : 1, WE = CPR > 32 ? CPR / 32 : 1;   /* rows per 512 bytes, or the other way round */
        const uint32_t tk = sk + tl * PITCH + ((cl ^ swz(SWK, tl)) << 4), tv = sk + VOFF + tl * PITCH + ((cl ^ swz(SWV, tl)) << 4);
        const unsigned rowb = (unsigned)a.kv.hd * ES;
        if (full) {
            const uint8_t *ks = a.kv.k + cl * 16, *vs = a.kv.v + cl * 16;
#pragma unroll
            for (int e = 0; e < TP * CPR / 32; e++) {
                const int te = e / WE * RE, ce = 32 * (e % WE), to = te * PITCH + ce * 16;
                const size_t off = (size_t)__shfl_sync(0xffffffffu, row[te / RW], (te + tl) & (RW - 1)) * rowb;
                if ((cl + ce) * 16 < (int)rowb) {      /* (the chunks behind a shorter head stay zero) */
                    cp_async16s((tk ^ (uint32_t)(swz(SWK, te) << 4)) + to, ks + off + ce * 16);
                    cp_async16s((tv ^ (uint32_t)(swz(SWV, te) << 4)) + to, vs + off + ce * 16);
                }
            }
        } else {
#pragma unroll 1
            for (int e = 0; e < TP * CPR / 32; e++) {
                const int te = e / WE * RE, ce = 32 * (e % WE), t = (te + tl) & (RW - 1), k = te / RW, to = te * PITCH + ce * 16;
                const unsigned rr = __shfl_sync(0xffffffffu, k ? row[LK - 1] : row[0], t);
                const bool lv = (((k ? live[LK - 1] : live[0]) >> t) & 1u) && (cl + ce) * 16 < (int)rowb;
                const size_t off = (size_t)rr * rowb + (lv ? (cl + ce) * 16 : 0);
                cp_async16z((tk ^ (uint32_t)(swz(SWK, te) << 4)) + to, a.kv.k + off, lv);
                cp_async16z((tv ^ (uint32_t)(swz(SWV, te) << 4)) + to, a.kv.v + off, lv);
            }
        }
    };
    if (a.kv.hd < HD) {
        for (int i = lane; i < S * SLOT / 16; i += 32) ((uint4 *)(slots + (size_t)warp * S * SLOT))[i] = make_uint4(0u, 0u, 0u, 0u);
        __syncwarp();
    }
    auto copy_scales = [&](float *dst, const float *src) {
#pragma unroll
        for (int k = 0; k < LK; k++) cp_async4z(smem_u32(dst + k * 32 + lane), src + row[k], (live[k] >> lane) & 1u);
    };
    int issued = 0;
    auto issue = [&](int stage) {
        issued++;
        if (live[0] | live[LK - 1]) {
            copy_rows(ring_s + stage * SLOT);
            if constexpr (KV == KC_Q8_0) {
                copy_scales(scl + stage * SCALES, a.kv.kd);
                copy_scales(scl + stage * SCALES + TP, a.kv.vd);
            }
        }
        if (lane == 0) {
            const int f = (ql == 1 ? LAST_OF_UNIT : 0) | (left <= (ql == 1 ? 1 + W : 1) ? LAST_OF_SHARE : 0);
            info[stage] = make_int4(lb, lu | f, (int)live[0], LK > 1 ? (int)live[LK - 1] : 0);
        }
    };
    auto advance = [&]() {
        left -= ql == 1 ? 1 + W : 1;
        if (left <= 0) return;
        if (--ql > 0) {
            p0 += QP;
        } else {
            ubase += nq + W;
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
                tbn = 0;                               /* another table row */
            }
            ql = nq;
            p0 = first + warp * TP;
            lg = lu / a.chunks;
        }
        look();
    };
    /* the lane's part of a unit's query rows, as loaded */
    float xq[MT][HD / 4];
    auto fetch_q = [&](int b, int u) {
        const int g = u / a.chunks, h0 = (u - g * a.chunks) * HC, nh = min(HC, a.group - h0);
        const float *qb = a.q + b * a.ldq + (size_t)(g * a.group + h0) * a.kv.hd;
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
            const bool on = mt * 8 + r < nh;
            const float *qh = qb + (size_t)(mt * 8 + r) * a.kv.hd;
#pragma unroll
            for (int j = 0; j < HD / 16; j++) {
                if constexpr (KV == KC_F16) {          /* dims 16 j + 2 c + {0, 1, 8, 9} */
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const int d = 16 * j + 8 * i + 2 * c;
                        float2 t = make_float2(0.0f, 0.0f);
                        if (on && d < a.kv.hd) t = *(const float2 *)(qh + d);
                        xq[mt][4 * j + 2 * i] = t.x;
                        xq[mt][4 * j + 2 * i + 1] = t.y;
                    }
                } else {                               /* dims 16 j + 4 c + {0, 1, 2, 3} */
                    const int d = 16 * j + 4 * c;
                    float4 t = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    if (on && d < a.kv.hd) t = *(const float4 *)(qh + d);
                    xq[mt][4 * j] = t.x; xq[mt][4 * j + 1] = t.y; xq[mt][4 * j + 2] = t.z; xq[mt][4 * j + 3] = t.w;
                }
            }
        }
    };
    fetch_q(lb, lu);
    look();

    /* ---- the compute side ---- */
    constexpr int QR = KV == KC_F32 ? HD / 8 * 4 : (KV == KC_F16 ? HD / 16 * 4 : HD / 32 * 2);
    unsigned qf[MT][QR];                               /* the query fragments */
    float qc[MT];                                      /* score of a raw product, times log2 e, or over the soft-cap */
    constexpr int NACC = HD / 4;
    float2 acc[MT][NACC / 2];                          /* see finish for which dimensions */
    float m[MT], l[MT];                                /* running maxima, and the lane's part of the weights' sums */
    const float LOG2E = 1.4426950408889634f;
    int cu_b = b0_, cu_u = u0_;                        /* the current unit */
    bool fresh = whole0;                               /* it begins in this share */

    /* the fragments of the query rows in xq */
    auto set_q = [&]() {
        /* qc is positive (its sign goes to the query): the largest product is the largest score, and one that is
         * masked away, -inf, stays so */
        const float post = fabsf(a.scale) * (a.softcap > 0.0f ? a.inv_softcap : LOG2E);
        const float sign = copysignf(1.0f, a.scale);
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
            const float *x = xq[mt];
            if constexpr (KV == KC_F32) {
#pragma unroll
                for (int i = 0; i < HD / 4; i++) split_tf32(x[i] * sign, qf[mt][2 * i], qf[mt][2 * i + 1]);
                qc[mt] = post;
            } else {
                float mx = 0.0f;                       /* of the head, whose values the four lanes of a row hold */
#pragma unroll
                for (int i = 0; i < HD / 4; i++) mx = fmaxf(mx, fabsf(x[i]));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                if constexpr (KV == KC_F16) {
                    /* the largest |q| of the head is brought to [2^12, 2^13), a power of two exactly, so
                     * that the low parts of all but vanishing values stay normal f16 */
                    int ex = (int)((__float_as_uint(mx) >> 23) & 255) - 127;
                    ex = min(max(ex, -100), 100);
                    const float up = sign * __uint_as_float((unsigned)(127 + 12 - ex) << 23);
                    qc[mt] = __uint_as_float((unsigned)(127 - 12 + ex) << 23) * post;
#pragma unroll
                    for (int i = 0; i < HD / 8; i++)
                        split_f16(make_float2(x[2 * i] * up, x[2 * i + 1] * up), qf[mt][2 * i], qf[mt][2 * i + 1]);
                } else {
                    /* the query head quantized as a cache row is (ops/ops.c:229-233) */
                    const bool tiny = mx < 1e-30f;
                    const float id = tiny ? 0.0f : sign * __fdiv_rn(127.0f, mx), qd = tiny ? 0.0f : __fdiv_rn(mx, 127.0f);
#pragma unroll
                    for (int j = 0; j < HD / 16; j++) {
                        /* x 127 / max rounded half away from zero: at most 127.5 and a rounding, never 128 */
                        int q[4];
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            q[i] = __float2int_rz(__fadd_rn(__fmul_rn(x[4 * j + i], id), copysignf(0.5f, sign * x[4 * j + i])));
                        const unsigned w = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
                        qf[mt][j] = w;
                    }
                    qc[mt] = qd * post;
                }
            }
            qc[mt] = fmaxf(qc[mt], 1.17549435e-38f);
        }
    };

    /* the scores of the tile of TP positions in ring slot `stage`: of head row r, positions 8 nt + 2 c and + 1 */
    float2 s[MT][NT];
    auto scores = [&](int stage) {
        const uint32_t sk = ring_s + stage * SLOT;
        if constexpr (KV == KC_F16) {
            float d[MT][NT][4];
            const uint32_t kb = sk + (lane & 7) * PITCH + (((lane >> 3) ^ (lane & 7)) << 4);
#pragma unroll
            for (int jj = 0; jj < HD / 32; jj++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    unsigned b[4];
                    ldsm4(b, (kb ^ (64 * jj)) + nt * 8 * PITCH);
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) {
                        const unsigned a0[4] = { qf[mt][8 * jj], qf[mt][8 * jj + 1], qf[mt][8 * jj + 2], qf[mt][8 * jj + 3] };
                        const unsigned a1[4] = { qf[mt][8 * jj + 4], qf[mt][8 * jj + 5], qf[mt][8 * jj + 6], qf[mt][8 * jj + 7] };
                        if (jj == 0) mma_f16_first(d[mt][nt], a0, b[0], b[1]);
                        else mma_f16(d[mt][nt], a0, b[0], b[1]);
                        mma_f16(d[mt][nt], a1, b[2], b[3]);
                    }
                }
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    s[mt][nt] = halves(d[mt][nt]);
                }
        } else if constexpr (KV == KC_F32) {
            float dh[MT][NT][4], dl[MT][NT][4];
            const uint32_t kb = sk + r * PITCH + ((c ^ swz(SWK, r)) << 4);
#pragma unroll
            for (int jj = 0; jj < HD / 16; jj++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    const float4 t = lds4((kb ^ (64 * jj)) + nt * 8 * PITCH);
                    unsigned h[4], w[4];
                    split_tf32(t.x, h[0], w[0]);
                    split_tf32(t.y, h[1], w[1]);
                    split_tf32(t.z, h[2], w[2]);
                    split_tf32(t.w, h[3], w[3]);
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) {
                        const unsigned a0[4] = { qf[mt][8 * jj], qf[mt][8 * jj + 1], qf[mt][8 * jj + 2], qf[mt][8 * jj + 3] };
                        const unsigned a1[4] = { qf[mt][8 * jj + 4], qf[mt][8 * jj + 5], qf[mt][8 * jj + 6], qf[mt][8 * jj + 7] };
                        if (jj == 0) {
                            mma_tf32_first(dh[mt][nt], a0, h[0], h[1]);
                            mma_tf32_first(dl[mt][nt], a0, w[0], w[1]);
                        } else {
                            mma_tf32(dh[mt][nt], a0, h[0], h[1]);
                            mma_tf32(dl[mt][nt], a0, w[0], w[1]);
                        }
                        mma_tf32(dh[mt][nt], a1, h[2], h[3]);
                        mma_tf32(dl[mt][nt], a1, w[2], w[3]);
                    }
                }
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    s[mt][nt] = add2(halves(dh[mt][nt]), halves(dl[mt][nt]));
                }
        } else {
            int d[MT][NT][4];                          /* from 1.5 * 2^23: the sums come out as its floats */
            const uint32_t kb = sk + (lane & 7) * PITCH + (((lane >> 3) ^ swz(SWK, lane & 7)) << 4);
#pragma unroll
            for (int jj = 0; jj < HD / 64; jj++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    unsigned b[4];
                    ldsm4(b, (kb ^ (64 * jj)) + nt * 8 * PITCH);
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) {
                        if (jj == 0) mma_s8_first(d[mt][nt], qf[mt][4 * jj], qf[mt][4 * jj + 1], b[0], b[1], 0x4b400000);
                        else mma_s8(d[mt][nt], qf[mt][4 * jj], qf[mt][4 * jj + 1], b[0], b[1]);
                        mma_s8(d[mt][nt], qf[mt][4 * jj + 2], qf[mt][4 * jj + 3], b[2], b[3]);
                    }
                }
            const float *kd = scl + stage * SCALES;
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                const float2 e = *(const float2 *)(kd + nt * 8 + 2 * c);
#pragma unroll
                for (int mt = 0; mt < MT; mt++) {
                    s[mt][nt] = mul2(add2(make_float2(__int_as_float(d[mt][nt][0]), __int_as_float(d[mt][nt][1])),
                                          make_float2(-12582912.0f, -12582912.0f)),
                                     e);
                }
            }
        }
    };
    /* soft-cap, mask, running softmax in base 2: the scores become weights. For f16 products they are then lifted
     * by a power of two that keeps the small ones normal f16 numbers: 2^15, and for 8-bit rows, whose scales join
     * the weights, over the next power of two above the tile's largest scale (back: what the tile's sums are
     * multiplied by). By a product, which is exact: added to the exponent it would take as many bits off the
     * exponent's fraction as it is large, 4 of 24 for 2^15 and up to 7 for the smallest scales. */
    constexpr float LIFT = KV == KC_F32 ? 1.0f : 32768.0f;
    float2 corr[MT];                                   /* what the sums so far are scaled by */
    float lift = LIFT, back = 1.0f;
    auto soften = [&](int stage, const unsigned (&live)[LK]) {
        if constexpr (KV == KC_Q8_0) {
            const float *vd = scl + stage * SCALES + TP;
            float top = fabsf(vd[lane]);
#pragma unroll
            for (int k = 1; k < LK; k++) top = fmaxf(top, fabsf(vd[k * 32 + lane]));
            top = warp_max(top);
            int ex = (int)((__float_as_uint(top) >> 23) & 255) - 126;
            ex = min(max(ex, -100), 100);
            lift = __uint_as_float((unsigned)(127 + 15 - ex) << 23);
            back = __uint_as_float((unsigned)(127 + ex) << 23);
        }
        bool all = true;
#pragma unroll
        for (int k = 0; k < LK; k++) all &= live[k] == (unsigned)((1ull << RW) - 1);
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
            float qm = qc[mt];
            if (a.softcap > 0.0f) {
                qm = a.softcap * LOG2E;
#pragma unroll
                for (int nt = 0; nt < NT; nt++) s[mt][nt] = make_float2(tanhf(s[mt][nt].x * qc[mt]), tanhf(s[mt][nt].y * qc[mt]));
            }
            if (!all) {
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    const unsigned here = live[nt * 8 / RW] >> ((nt * 8) % RW + 2 * c);
                    if (!(here & 1u)) s[mt][nt].x = -INFINITY;
                    if (!(here & 2u)) s[mt][nt].y = -INFINITY;
                }
            }
            float mx = fmaxf(s[mt][0].x, s[mt][0].y);
#pragma unroll
            for (int nt = 1; nt < NT; nt++) mx = fmaxf(mx, fmaxf(s[mt][nt].x, s[mt][nt].y));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const float mn = fmaxf(m[mt], mx * qm), base = mn == -INFINITY ? 0.0f : mn;
            const float cr = ex2(m[mt] - base);
            corr[mt] = make_float2(cr, cr);
            m[mt] = mn;
            float2 both = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                const float2 x = fma2(s[mt][nt], make_float2(qm, qm), make_float2(-base, -base));
                s[mt][nt] = make_float2(ex2(x.x), ex2(x.y));
                both = nt ? add2(both, s[mt][nt]) : s[mt][nt];
            }
            const float sum = both.x + both.y;
            l[mt] = l[mt] * cr + sum * LIFT;
        }
    };
    /* the weighted sum of V's rows */
    auto weigh = [&](int stage) {
        const uint32_t sv = ring_s + stage * SLOT + VOFF;
        if constexpr (KV == KC_F16) {
            constexpr int KS = TP / 16;
            unsigned w[MT][KS][4];
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
                    split_f16(mul2(s[mt][nt], make_float2(LIFT, LIFT)), w[mt][nt >> 1][2 * (nt & 1)], w[mt][nt >> 1][2 * (nt & 1) + 1]);
            const uint32_t vb = sv + (lane & 15) * PITCH + (((lane >> 4) ^ (lane & 7)) << 4);
#pragma unroll
            for (int jj = 0; jj < HD / 16; jj++) {
                float d[MT][2][4];
#pragma unroll
                for (int ks = 0; ks < KS; ks++) {
                    unsigned b[4];
                    ldsm4t(b, (vb ^ (32 * jj)) + ks * 16 * PITCH);
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) {
                        if (ks == 0) {
                            mma_f16_first(d[mt][0], w[mt][ks], b[0], b[1]);
                            mma_f16_first(d[mt][1], w[mt][ks], b[2], b[3]);
                        } else {
                            mma_f16(d[mt][0], w[mt][ks], b[0], b[1]);
                            mma_f16(d[mt][1], w[mt][ks], b[2], b[3]);
                        }
                    }
                }
#pragma unroll
                for (int mt = 0; mt < MT; mt++) {
                    acc[mt][2 * jj] = fma2(acc[mt][2 * jj], corr[mt], halves(d[mt][0]));
                    acc[mt][2 * jj + 1] = fma2(acc[mt][2 * jj + 1], corr[mt], halves(d[mt][1]));
                }
            }
        } else if constexpr (KV == KC_F32) {
            unsigned w[MT][NT][4];
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    split_tf32(s[mt][nt].x, w[mt][nt][0], w[mt][nt][1]);
                    split_tf32(s[mt][nt].y, w[mt][nt][2], w[mt][nt][3]);
                }
            const uint32_t v0 = sv + (2 * c) * PITCH + ((r ^ (2 * c)) << 4), v1 = sv + (2 * c + 1) * PITCH + ((r ^ (2 * c + 1)) << 4);
#pragma unroll
            for (int j = 0; j < HD / 32; j++) {
                float d[MT][4][4];
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    const float4 ya = lds4((v0 ^ (128 * j)) + nt * 8 * PITCH);
                    const float4 yb = lds4((v1 ^ (128 * j)) + nt * 8 * PITCH);
                    const float y0[4] = { ya.x, ya.y, ya.z, ya.w }, y1[4] = { yb.x, yb.y, yb.z, yb.w };
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        unsigned h0, h1, g0, g1;
                        split_tf32(y0[i], h0, g0);
                        split_tf32(y1[i], h1, g1);
#pragma unroll
                        for (int mt = 0; mt < MT; mt++) {
                            if (nt == 0) mma_tf32_first(d[mt][i], w[mt][nt], g0, g1);
                            else mma_tf32(d[mt][i], w[mt][nt], g0, g1);
                            mma_tf32(d[mt][i], w[mt][nt], h0, h1);
                        }
                    }
                }
#pragma unroll
                for (int mt = 0; mt < MT; mt++)
#pragma unroll
                    for (int i = 0; i < 4; i++) acc[mt][4 * j + i] = fma2(acc[mt][4 * j + i], corr[mt], halves(d[mt][i]));
            }
        } else {
            constexpr int KS = TP / 16;
            const float *vd = scl + stage * SCALES + TP;
            unsigned w[MT][KS][4];
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                const float2 e = mul2(*(const float2 *)(vd + nt * 8 + 2 * c), make_float2(lift, lift));
#pragma unroll
                for (int mt = 0; mt < MT; mt++)
                    split_f16(mul2(s[mt][nt], e), w[mt][nt >> 1][2 * (nt & 1)],
                              w[mt][nt >> 1][2 * (nt & 1) + 1]);
            }
            const uint32_t vb = sv + (lane & 15) * PITCH + (((lane >> 4) ^ swz(SWV, lane & 7)) << 4);
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
                for (int ks = 0; ks < KS; ks++) {
                    unsigned b[4];
                    ldsm4t(b, (vb ^ (32 * jj)) + ks * 16 * PITCH);
                    unsigned e0, o0, e1, o1;
                    bytes(b[0], e0, o0);
                    bytes(b[1], e1, o1);
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) {
                        if (ks == 0) {
                            mma_f16_first(d[mt][0], w[mt][ks], e0, e1);
                            mma_f16_first(d[mt][1], w[mt][ks], o0, o1);
                        } else {
                            mma_f16(d[mt][0], w[mt][ks], e0, e1);
                            mma_f16(d[mt][1], w[mt][ks], o0, o1);
                        }
                    }
                    bytes(b[2], e0, o0);
                    bytes(b[3], e1, o1);
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) {
                        if (ks == 0) {
                            mma_f16_first(d[mt][2], w[mt][ks], e0, e1);
                            mma_f16_first(d[mt][3], w[mt][ks], o0, o1);
                        } else {
                            mma_f16(d[mt][2], w[mt][ks], e0, e1);
                            mma_f16(d[mt][3], w[mt][ks], o0, o1);
                        }
                    }
                }
#pragma unroll
                for (int mt = 0; mt < MT; mt++)
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        acc[mt][4 * jj + k] = fma2(acc[mt][4 * jj + k], corr[mt], mul2(halves(d[mt][k]), make_float2(back, back)));
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
                    const float2 *o = &acc[mt][4 * j];
                    if constexpr (KV == KC_F32) {
                        /* o[i]: dims 32 j + 8 c + i and + 4 */
                        float *p = row + ((32 * j + 8 * c) ^ x);
                        *(float4 *)p = make_float4(o[0].x, o[1].x, o[2].x, o[3].x);
                        *(float4 *)(p + 4) = make_float4(o[0].y, o[1].y, o[2].y, o[3].y);
                    } else if constexpr (KV == KC_F16) {
#pragma unroll
                        for (int k = 0; k < 4; k++)    /* o[k]: dims 32 j + 8 k + 2 c and + 1 */
                            *(float2 *)(row + ((32 * j + 8 * k + 2 * c) ^ x)) = o[k];
                    } else {
#pragma unroll
                        for (int k = 0; k < 2; k++)    /* o[2 k], o[2 k + 1]: dims 32 j + 16 k + 4 c + {0, 2}, {1, 3} */
                            *(float4 *)(row + ((32 * j + 16 * k + 4 * c) ^ x)) =
                                make_float4(o[2 * k].x, o[2 * k + 1].x, o[2 * k].y, o[2 * k + 1].y);
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

    /* a piece is written: was it the unit's last missing one? (A unit that is not fresh is the share's first,
     * one that is left unfinished its last: at most two, and they are joined after the loop, which keeps the
     * loop's registers out of a call.) */
    __shared__ int s_join[2][4];
    if (tid < 2) s_join[tid][0] = 0;
    auto leave = [&](int b, int u) {
        if (tid != 0) return;
        __threadfence();                               /* finish's barrier is behind every thread's part of the piece */
        const long long x = (fresh ? ubase : ubase0) + W;
        const int c0 = (int)(x / chunk), c1 = (int)((x + (fresh ? nq : nq0) - 1) / chunk);
        const unsigned n = atomicAdd(a.count + c1, 1u);
        int *j = s_join[fresh];
        j[0] = n == (unsigned)(c1 - c0) ? c1 + 1 : 0;
        j[1] = c0;
        j[2] = b;
        j[3] = u;
        if (j[0]) a.count[c1] = 0u;
        __threadfence();
    };

    auto begin = [&]() {
        set_q();
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
            m[mt] = -INFINITY;
            l[mt] = 0.0f;
#pragma unroll
            for (int i = 0; i < NACC / 2; i++) acc[mt][i] = make_float2(0.0f, 0.0f);
        }
    };
    begin();
    /* the first S passes only load */
    for (int it = -S, stage = 0; it < issued; it++, stage = stage + 1 == S ? 0 : stage + 1) {
        int4 f = make_int4(cu_b, cu_u, 0, 0);
        /* lane 0 wrote what the slot holds when its copies were issued: with several slots a pass, and its barriers,
         * ago, with one slot at the end of the pass before */
        if constexpr (S == 1) __syncwarp();
        if (it >= 0) f = info[stage];
        const int fu = f.y & (LAST_OF_UNIT - 1);
        if (f.x != cu_b || fu != cu_u) {
            /* a new unit: its queries are on their way while the tile arrives */
            cu_b = f.x;
            cu_u = fu;
            fresh = true;
            fetch_q(cu_b, cu_u);
            begin();
        }
        const bool on = f.z | f.w;
        cp_async_wait_but<S - 1>();
        __syncwarp();
        if (on) {
            scores(stage);
            unsigned here[LK];
            here[0] = (unsigned)f.z;
            if constexpr (LK > 1) here[1] = (unsigned)f.w;
            soften(stage, here);
            weigh(stage);
        }
        __syncwarp();
        if (left > 0) {
            issue(stage);
            advance();
        }
        cp_async_commit();
        if (f.y & (LAST_OF_UNIT | LAST_OF_SHARE)) {
            const bool complete = fresh && (f.y & LAST_OF_UNIT);
            finish(cu_b, cu_u, complete);
            if (!complete) leave(cu_b, cu_u);
        }
    }
    /* not sooner: the next call's CTAs would crowd the SMs that still have room, and its few working ones share them */
    launch_next();
    __syncthreads();
    for (int k = 0; k < 2; k++)
        if (s_join[k][0]) {
            join_pieces<HD, MT>(a, s_join[k][2], s_join[k][3], s_join[k][1], s_join[k][0] - 1, slots, AT_WARPS * S * SLOT);
            __syncthreads();
        }
}

}  // namespace kc
