/* Serving several sequences: the C entries of the paged KV cache (rows of new
 * tokens, attention of one new token per sequence) and of the processing of a
 * batch's logits. Every argument that the host can see is checked before a
 * launch; what lies in device memory is checked by the kernels, which skip what
 * is out of range and flag it for the next kc_dev_sync. */
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <string>

#include "kc_internal.h"
#include "kc_logits.cuh"
#include "kc_paged.cuh"

namespace kc {

static int sv_cuda(cudaError_t e, const char *what) {
    if (e == cudaSuccess) return KC_OK;
    set_error(std::string(what) + ": " + cudaGetErrorString(e));
    (void)cudaGetLastError();
    if (e == cudaErrorMemoryAllocation) return KC_E_NOMEM;
    if (e == cudaErrorNoDevice || e == cudaErrorInsufficientDriver || e == cudaErrorNoKernelImageForDevice)
        return KC_E_ISA;
    return KC_E_IO;
}
#define SK(call, what)                                    \
    do {                                                  \
        const cudaError_t e_ = (call);                    \
        if (e_ != cudaSuccess) return sv_cuda(e_, what);  \
    } while (0)

static int refuse(const std::string &msg) {
    set_error(msg);
    return KC_E_SHAPE;
}

constexpr int SV_MAX_DEVICES = 64;

/* The serving kernels' error word, one per device, sticky until kc_dev_sync. */
static __device__ unsigned g_sv_err;
/* What is looked up at a device's first use may be looked up by several threads at once, with the same result: each
 * stores it whole, the pointer last, and whoever sees the pointer sees what was stored before it. */
static std::atomic<unsigned *> g_sv_err_ptr[SV_MAX_DEVICES];

struct ServeDev {
    int dev = 0, sms = 0;
    unsigned *err = nullptr;
};

/* The current device: its SMs and error word (looked up once per device). */
static int serve_device(ServeDev &d) {
    static std::atomic<int> sms[SV_MAX_DEVICES];
    SK(cudaGetDevice(&d.dev), "current device");
    if (d.dev < 0 || d.dev >= SV_MAX_DEVICES) return refuse("device index " + std::to_string(d.dev) + " beyond this library's table");
    d.err = g_sv_err_ptr[d.dev].load(std::memory_order_acquire);
    if (!d.err) {
        int major = 0, minor = 0, n = 0;
        SK(cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, d.dev), "device");
        SK(cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, d.dev), "device");
        if (major != 10 || minor != 0) {
            set_error("not an sm_100 device");
            return KC_E_ISA;
        }
        SK(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, d.dev), "device");
        void *p = nullptr;
        SK(cudaGetSymbolAddress(&p, g_sv_err), "error word");
        d.err = (unsigned *)p;
        sms[d.dev].store(n, std::memory_order_relaxed);
        g_sv_err_ptr[d.dev].store(d.err, std::memory_order_release);
    }
    d.sms = sms[d.dev].load(std::memory_order_relaxed);
    return KC_OK;
}

unsigned *serve_err_word(int dev) { return dev >= 0 && dev < SV_MAX_DEVICES ? g_sv_err_ptr[dev].load(std::memory_order_acquire) : nullptr; }

std::string serve_err_text(unsigned w) {
    std::string s;
    auto add = [&](unsigned bit, const char *t) {
        if (w & bit) s += std::string(s.empty() ? "" : ", ") + t;
    };
    add(SE_HIST, "a history length below 0 or beyond its rows");
    add(SE_BIAS, "bias offsets out of order or beyond the list");
    add(SE_LEN, "a sequence length below 0 or beyond its table row");
    add(SE_PAGE, "a page number outside the pool");
    add(SE_ROW, "a new row's sequence, position or page out of range");
    return s;
}

/* Device memory of the current device, aligned to `align` bytes. */
static int check_ptr(const void *p, int dev, size_t align, const char *name) {
    if (!p) return refuse(std::string(name) + " is NULL");
    if ((uintptr_t)p % align) return refuse(std::string(name) + " is not aligned to " + std::to_string(align) + " bytes");
    cudaPointerAttributes at;
    const cudaError_t e = cudaPointerGetAttributes(&at, p);
    if (e != cudaSuccess) return sv_cuda(e, name);
    if (at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged)
        return refuse(std::string(name) + " is not device memory");
    if (at.type == cudaMemoryTypeDevice && at.device != dev)
        return refuse(std::string(name) + " lies on device " + std::to_string(at.device) + ", not on the current device " +
                      std::to_string(dev));
    return KC_OK;
}
#define PTR(p, align)                                                   \
    do {                                                                \
        const int rc_ = check_ptr((const void *)(p), d.dev, align, #p); \
        if (rc_ != KC_OK) return rc_;                                   \
    } while (0)

/* The sizes of a cache, without its pointers. */
static int check_cache(const kc_paged_kv *kv) {
    if (!kv) return refuse("kv is NULL");
    if (kv->kv_type != KC_F32 && kv->kv_type != KC_F16 && kv->kv_type != KC_Q8_0)
        return refuse("kv_type must be KC_F32, KC_F16 or KC_Q8_0");
    if (kv->head_dim < 16 || kv->head_dim > 256 || kv->head_dim % 16)
        return refuse("head_dim must be a multiple of 16 from 16 to 256");
    if (kv->n_pages < 1 || kv->page_size < 1 || kv->n_kv_heads < 1 || kv->n_seqs < 1 || kv->ld_table < 1)
        return refuse("n_pages, page_size, n_kv_heads, n_seqs and ld_table must be at least 1");
    if ((double)kv->n_pages * kv->page_size * kv->n_kv_heads >= 4294967296.0)
        return refuse("the pool's rows (n_pages * page_size * n_kv_heads) must be fewer than 2^32");
    if ((double)kv->ld_table * kv->page_size > 2147483647.0 - 65536.0)
        return refuse("a table row (ld_table * page_size) must hold fewer than 2^31 - 2^16 positions");
    return KC_OK;
}

static int take_cache(const kc_paged_kv *kv, const ServeDev &d, PagedKV &o) {
    PTR(kv->k, 16);
    PTR(kv->v, 16);
    PTR(kv->table, 4);
    if (kv->kv_type == KC_Q8_0) {
        PTR(kv->kd, 4);
        PTR(kv->vd, 4);
    }
    o = PagedKV{ (uint8_t *)kv->k, (uint8_t *)kv->v, kv->kd, kv->vd, kv->table, kv->n_seqs, kv->ld_table, kv->n_pages,
                 kv->page_size, kv->n_kv_heads, kv->head_dim, Divisor(kv->page_size) };
    return KC_OK;
}

/* A launch that may begin while the stream's kernel before it ends (its CTAs wait in stream_order): in a run of
 * these operators the launch itself costs nothing then. */
template <class A>
static cudaError_t launch_after(void (*kernel)(const A), unsigned gx, unsigned gy, int threads, size_t smem, cudaStream_t st, const A &a) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(gx, gy);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

/* ------------------------------------------------------------ append */

template <int KV>
static cudaError_t launch_append(AppendArgs &a, cudaStream_t st) {
    const int hd = a.kv.hd, lph = hd <= 32 ? 8 : (hd <= 64 ? 16 : 32);
    const int hw = (hd <= 128 ? ap_heads<1>() : ap_heads<2>()) * (32 / lph);
    a.tasks = (a.n_heads + hw - 1) / hw + 2 * ((a.kv.n_kv + hw - 1) / hw);
    a.row_of = Divisor(a.tasks);
    const long long warps = (long long)a.rows * a.tasks;
    const unsigned grid = (unsigned)((warps + AP_THREADS / 32 - 1) / (AP_THREADS / 32));
    return launch_after(lph == 8 ? append_kernel<KV, 8, 1>
                                 : (lph == 16 ? append_kernel<KV, 16, 1> : (hd <= 128 ? append_kernel<KV, 32, 1> : append_kernel<KV, 32, 2>)),
                        grid, 1, AP_THREADS, 0, st, a);
}

/* ------------------------------------------------------------ attention */

/* A unit's own time beside its tiles', in quanta (queries, the warps' meeting, the output). */
constexpr int AT_UNIT_COST = 2;

/* The workspace: a counter for each CTA of any instance, zero between calls, and the pieces. */
constexpr int AT_MAX_CTAS = 2048;

/* One instance: its kernel, shared memory, and on each device the CTAs that fit. */
struct AttendVariant {
    void (*attend)(const AttendArgs);
    int smem, part, tile, heads;
    std::atomic<int> ctas[SV_MAX_DEVICES];             /* 0: not asked yet */
};

template <int KV, int HD, int TM, int MT, int S, int OCC>
static AttendVariant *variant() {
    static AttendVariant v{ paged_attend_kernel<KV, HD, TM, MT, S, OCC>, attend_smem<KV, HD, TM, MT, S>(), part_floats<HD, MT>(),
                            att_tp<KV, TM>(), 8 * MT, {} };
    return &v;
}

/* The instance for a cache and group: a template of positions per tile, heads
 * per chunk, ring slots and CTAs an SM. Two slots a warp are enough (a third only
 * puts more copies under way than the memory likes: 64 sequences of 2048..8192
 * positions, f16, head 128: 206 us with 16 KB a warp under way, 219 us with 24);
 * a third CTA an SM (12 warps instead of 8) pays where arithmetic or the short
 * sequences' own time fills the SM, above all at the clocks that a long run is
 * held to: the same 64 sequences 212 us instead of 224, 256 of 1..1000 100 instead
 * of 105, 64 of 4096, 8-bit, head 64, 66 instead of 71. Only the 8-bit cache of
 * head 128 has no registers for it to spare: 32 of 2048 37 us with two CTAs, 38.5
 * with three. A tile of head 256 is so large that two slots a warp leave room for
 * one CTA an SM, whose 4 warps wait for their own results; one slot lets two in:
 * 16 of 2048, f32, 85 us with two slots, 70 with one; f16 34 and 32, 8-bit (32 of
 * them) 44 and 38; 200 of 1..300, f16, 47 and 35. A sequence or two alone are cut
 * into as many pieces as there are CTAs, and half as many are better joined: one of
 * 32768, f16, 37 us with two slots, 43 with one, 8 heads to a KV head, f32, 71 and
 * 91; from 16 units on (4 of 8192: f32 84 and 69, f16 34 and 34) it is the other way. */
template <int KV>
static AttendVariant *variants_of(int hd, int group, long long units, int &mt) {
    if constexpr (KV != KC_F32) {
        /* more than 8 heads share a KV head: 16 at a time, so that the cache is read once */
        if (group > 8 && hd <= 128) {
            mt = 2;
            return hd <= 64 ? variant<KV, 64, 2, 2, 2, 2>() : variant<KV, 128, 1, 2, 2, 2>();
        }
    }
    mt = 1;
    if (hd <= 64) return variant<KV, 64, 2, 1, 2, 3>();
    if (hd <= 128) return variant<KV, 128, 1, 1, 2, KV == KC_Q8_0 ? 2 : 3>();
    return units <= 8 ? variant<KV, 256, 1, 1, 2, 1>() : variant<KV, 256, 1, 1, 1, 2>();
}

static int attend_variant(const kc_paged_kv *kv, int n_heads, int n_seqs, const ServeDev &d, AttendVariant *&v, int &chunks, int &ctas) {
    const int group = n_heads / kv->n_kv_heads;
    const long long units = (long long)n_seqs * kv->n_kv_heads * ((group + 7) / 8);
    int mt = 1;
    v = kv->kv_type == KC_F32 ? variants_of<KC_F32>(kv->head_dim, group, units, mt)
                              : (kv->kv_type == KC_F16 ? variants_of<KC_F16>(kv->head_dim, group, units, mt)
                                                       : variants_of<KC_Q8_0>(kv->head_dim, group, units, mt));
    chunks = (group + 8 * mt - 1) / (8 * mt);
    ctas = v->ctas[d.dev].load(std::memory_order_acquire);
    if (!ctas) {
        SK(cudaFuncSetAttribute((const void *)v->attend, cudaFuncAttributeMaxDynamicSharedMemorySize, v->smem), "attend");
        int n = 0;
        SK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, (const void *)v->attend, AT_THREADS, (size_t)v->smem), "attend");
        ctas = std::min(n * d.sms, AT_MAX_CTAS);
        if (ctas < 1) {
            set_error("attend: no CTA fits an SM");
            return KC_E_IO;
        }
        v->ctas[d.dev].store(ctas, std::memory_order_release);
    }
    return KC_OK;
}

static size_t ws_bytes(const AttendVariant *v, int ctas) {
    return sizeof(unsigned) * AT_MAX_CTAS + 2 * sizeof(float) * (size_t)v->part * (size_t)ctas;
}

}  // namespace kc

using namespace kc;

extern "C" int kc_paged_append_dev(const kc_paged_kv *kv, const kc_append_args *x, void *stream) {
    clear_error();
    int rc = check_cache(kv);
    if (rc != KC_OK) return rc;
    if (!x) return refuse("args is NULL");
    if (x->rows < 0 || x->n_heads < 1 || x->n_pos < 1) return refuse("rows must not be negative, n_heads and n_pos at least 1");
    const long long qd = (long long)x->n_heads * kv->head_dim, kd = (long long)kv->n_kv_heads * kv->head_dim;
    if (x->ldq % 4 || x->ldk % 4 || x->ldv % 4 || x->ldo % 4) return refuse("row strides must be multiples of 4 floats");
    if (x->rows > 1 && (x->ldq < qd || x->ldo < qd || x->ldk < kd || x->ldv < kd))
        return refuse("a row stride is shorter than its row");
    if (!x->q_norm != !x->k_norm) return refuse("q_norm and k_norm come together");
    if (!(x->eps >= 0.0f) || std::isinf(x->eps)) return refuse("eps must be finite and not negative");
    if ((double)x->rows * (x->n_heads + 2 * kv->n_kv_heads) > 2147483647.0 - 65536.0) return refuse("too many rows in one call");
    if (!x->seqs && x->rows > kv->n_seqs) return refuse("more rows than sequences, and no seqs");
    if (x->q == x->q_out && x->rows > 1 && x->ldq != x->ldo) return refuse("in place, but the row strides differ");
    ServeDev d;
    rc = serve_device(d);
    if (rc != KC_OK) return rc;
    if (x->rows == 0) return KC_OK;
    AppendArgs a{};
    rc = take_cache(kv, d, a.kv);
    if (rc != KC_OK) return rc;
    PTR(x->q, 16);
    PTR(x->k, 16);
    PTR(x->v, 16);
    PTR(x->q_out, 16);
    PTR(x->cos, 8);
    PTR(x->sin, 8);
    PTR(x->pos, 4);
    if (x->seqs) PTR(x->seqs, 4);
    if (x->q_norm) {
        PTR(x->q_norm, 16);
        PTR(x->k_norm, 16);
    }
    a.q = x->q; a.k = x->k; a.v = x->v; a.q_out = x->q_out;
    a.ldq = x->ldq; a.ldk = x->ldk; a.ldv = x->ldv; a.ldo = x->ldo;
    a.cos = x->cos; a.sin = x->sin; a.q_norm = x->q_norm; a.k_norm = x->k_norm; a.eps = x->eps;
    a.seqs = x->seqs; a.pos = x->pos; a.rows = x->rows; a.n_heads = x->n_heads; a.n_pos = x->n_pos;
    a.err = d.err;
    const cudaStream_t st = (cudaStream_t)stream;
    return sv_cuda(kv->kv_type == KC_F32 ? launch_append<KC_F32>(a, st)
                                         : (kv->kv_type == KC_F16 ? launch_append<KC_F16>(a, st) : launch_append<KC_Q8_0>(a, st)),
                   "append");
}

static int check_heads(const kc_paged_kv *kv, int n_heads) {
    if (n_heads < 1 || n_heads % kv->n_kv_heads) return refuse("n_heads must be a multiple of n_kv_heads");
    if (n_heads > 65536) return refuse("n_heads must be at most 65536");
    return KC_OK;
}

extern "C" int kc_paged_attend_ws(const kc_paged_kv *kv, int n_heads, size_t *bytes) {
    clear_error();
    int rc = check_cache(kv);
    if (rc == KC_OK) rc = check_heads(kv, n_heads);
    if (rc != KC_OK) return rc;
    if (!bytes) return refuse("bytes is NULL");
    ServeDev d;
    AttendVariant *v = nullptr;
    int chunks = 0, ctas = 0;
    rc = serve_device(d);
    size_t most = 0;
    for (int n : { 1, kv->n_seqs }) {                  /* calls of any number of sequences share it */
        if (rc == KC_OK) rc = attend_variant(kv, n_heads, n, d, v, chunks, ctas);
        if (rc != KC_OK) return rc;
        most = std::max(most, ws_bytes(v, ctas));
    }
    *bytes = most;
    return KC_OK;
}

extern "C" int kc_paged_attend_ws_init(void *ws, size_t bytes) {
    clear_error();
    ServeDev d;
    const int rc = serve_device(d);
    if (rc != KC_OK) return rc;
    PTR(ws, 16);
    if (bytes < sizeof(unsigned) * AT_MAX_CTAS) return refuse("workspace too small (kc_paged_attend_ws)");
    SK(cudaMemsetAsync(ws, 0, sizeof(unsigned) * AT_MAX_CTAS, nullptr), "workspace");
    return sv_cuda(cudaStreamSynchronize(nullptr), "workspace");
}

extern "C" int kc_paged_attend_dev(const kc_paged_kv *kv, const kc_attend_args *x, void *stream) {
    clear_error();
    int rc = check_cache(kv);
    if (rc != KC_OK) return rc;
    if (!x) return refuse("args is NULL");
    rc = check_heads(kv, x->n_heads);
    if (rc != KC_OK) return rc;
    if (x->n_seqs < 0 || x->n_seqs > kv->n_seqs) return refuse("n_seqs must be 0 to the cache's");
    const long long qd = (long long)x->n_heads * kv->head_dim;
    if (x->ldq % 4 || x->ldo % 4) return refuse("row strides must be multiples of 4 floats");
    if (x->n_seqs > 1 && (x->ldq < qd || x->ldo < qd)) return refuse("a row stride is shorter than its row");
    if (x->window < 0) return refuse("window must not be negative");
    if (!std::isfinite(x->scale) || !std::isfinite(x->softcap) || x->softcap < 0.0f)
        return refuse("scale and softcap must be finite, softcap not negative");
    ServeDev d;
    rc = serve_device(d);
    if (rc != KC_OK) return rc;
    if (x->n_seqs == 0) return KC_OK;
    AttendArgs a{};
    AttendVariant *v = nullptr;
    int ctas = 0;
    rc = attend_variant(kv, x->n_heads, x->n_seqs, d, v, a.chunks, ctas);
    if (rc != KC_OK) return rc;
    const double quanta = (double)x->n_seqs * ((double)kv->ld_table * kv->page_size / (AT_WARPS * v->tile) + 2 + AT_UNIT_COST);
    if (quanta >= 2147483648.0 || quanta * kv->n_kv_heads * a.chunks / ctas >= 1073741824.0)
        return refuse("n_seqs sequences of ld_table * page_size positions are too many for one call");
    if (x->ws_bytes < ws_bytes(v, ctas))
        return refuse("workspace of " + std::to_string(x->ws_bytes) + " bytes, " + std::to_string(ws_bytes(v, ctas)) +
                      " needed (kc_paged_attend_ws)");
    rc = take_cache(kv, d, a.kv);
    if (rc != KC_OK) return rc;
    PTR(x->q, 16);
    PTR(x->out, 16);
    PTR(x->lens, 4);
    PTR(x->ws, 16);
    a.q = x->q; a.out = x->out; a.ldq = x->ldq; a.ldo = x->ldo; a.lens = x->lens;
    a.n_seqs = x->n_seqs; a.n_heads = x->n_heads; a.group = x->n_heads / kv->n_kv_heads;
    a.window = x->window; a.scale = x->scale; a.softcap = x->softcap;
    a.inv_softcap = x->softcap > 0.0f ? 1.0f / x->softcap : 0.0f;
    a.near = (v->tile - 1) / kv->page_size + 2 <= 32;
    a.unit_cost = AT_UNIT_COST;
    /* measured: a piece of 16 heads of 128 (8 KB) is joined in about 0.28 of a quantum's time, one of 4 heads of 64 in
     * 0.035; one sequence of 8192 positions, 16 heads to a KV head, takes 53 us in the smallest shares, 25 us so
     * (27 with half or twice the cost) */
    a.join_cost = 1.4e-4f * (float)(std::min(a.group, v->heads) * kv->head_dim);
    a.grid_inv = ~0ull / (unsigned)ctas + 1;
    a.count = (unsigned *)x->ws;
    a.part = (float *)((char *)x->ws + sizeof(unsigned) * AT_MAX_CTAS);
    a.err = d.err;
    return sv_cuda(launch_after(v->attend, (unsigned)ctas, 1, AT_THREADS, (size_t)v->smem, (cudaStream_t)stream, a), "attend");
}

/* ------------------------------------------------------------ logits */

extern "C" int kc_logits_process_dev(const kc_logits_args *x, void *stream) {
    clear_error();
    if (!x) return refuse("args is NULL");
    if (x->rows < 0 || x->vocab < 1 || x->vocab > (1 << 27)) return refuse("rows must not be negative, vocab 1 to 2^27");
    if (x->rows > 1 && (x->ld_in < x->vocab || x->ld_out < x->vocab)) return refuse("a row stride is shorter than its row");
    if (x->in == x->out && x->rows > 1 && x->ld_in != x->ld_out) return refuse("in place, but the row strides differ");
    const bool pen = x->repeat || x->presence || x->frequency;
    if (x->history_cap < 0 || (x->history && x->rows > 1 && x->ld_history < x->history_cap))
        return refuse("history_cap must not be negative nor beyond ld_history");
    if (!x->history && x->history_cap > 0) return refuse("history is NULL");
    const bool bias = x->bias_off != nullptr;
    if (x->n_bias < 0 || (bias && x->n_bias > 0 && (!x->bias_ids || !x->bias_vals)))
        return refuse("biases need offsets, ids and values");
    if (!bias && (x->bias_ids || x->bias_vals)) return refuse("biases need offsets, ids and values");
    if (x->mask && x->rows > 1 && x->ld_mask < (x->vocab + 31) / 32) return refuse("a mask row is shorter than the vocabulary");
    ServeDev d;
    int rc = serve_device(d);
    if (rc != KC_OK) return rc;
    if (x->rows == 0) return KC_OK;
    PTR(x->in, 4);
    PTR(x->out, 4);
    if (x->history) PTR(x->history, 4);
    if (x->history_len) PTR(x->history_len, 4);
    if (x->repeat) PTR(x->repeat, 4);
    if (x->presence) PTR(x->presence, 4);
    if (x->frequency) PTR(x->frequency, 4);
    if (bias) {
        PTR(x->bias_off, 4);
        if (x->n_bias > 0) {
            PTR(x->bias_ids, 4);
            PTR(x->bias_vals, 4);
        }
    }
    if (x->mask) PTR(x->mask, 4);
    LogitsArgs a{};
    a.in = x->in; a.out = x->out; a.ld_in = x->ld_in; a.ld_out = x->ld_out; a.vocab = x->vocab;
    a.hist = x->history; a.hist_len = x->history_len; a.ld_hist = x->ld_history; a.hist_cap = x->history_cap;
    a.repeat = x->repeat; a.presence = x->presence; a.frequency = x->frequency;
    a.bias_off = x->bias_off; a.bias_ids = x->bias_ids; a.bias_vals = x->bias_vals; a.n_bias = x->n_bias;
    a.mask = x->mask; a.ld_mask = x->ld_mask;
    a.err = d.err;
    const bool hist = pen && x->history_cap > 0;
    const unsigned rows = (unsigned)x->rows, chunks = (unsigned)((x->vocab + 3 + LG_CHUNK - 1) / LG_CHUNK);
    const cudaStream_t st = (cudaStream_t)stream;
    if (hist && bias && (x->history_cap > 65535 || x->n_bias > 65534)) {
        /* beyond the 16 bits that a count and a bias share: one after the other */
        SK(launch_after(logits_kernel<true, false>, rows, chunks, LG_THREADS, 0, st, a), "logits");
        a.in = a.out;
        a.ld_in = a.ld_out;
        return sv_cuda(launch_after(logits_kernel<false, true>, rows, chunks, LG_THREADS, 0, st, a), "logits");
    }
    return sv_cuda(launch_after(hist ? (bias ? logits_kernel<true, true> : logits_kernel<true, false>)
                                     : (bias ? logits_kernel<false, true> : logits_kernel<false, false>),
                                rows, chunks, LG_THREADS, 0, st, a),
                   "logits");
}
