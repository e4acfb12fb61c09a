/* First calls of the serving entries from several threads at once, on the CPU
 * (tests/test_serving_first_use.py): kc_serve.cu compiled for the host under
 * ThreadSanitizer and linked with this stand-in for the CUDA runtime, which
 * answers every question as a B200 would and launches nothing. */
#include <cuda_runtime.h>

#include <cstdio>
#include <string>
#include <thread>
#include <vector>

#include "krafla_cuda.h"

namespace kc {
static thread_local std::string g_text;
void set_error(const std::string &s) { g_text = s; }
void clear_error() { g_text.clear(); }
unsigned *serve_err_word(int dev);
}  // namespace kc

extern "C" {
cudaError_t cudaGetDevice(int *d) { *d = 0; return cudaSuccess; }
cudaError_t cudaDeviceGetAttribute(int *v, cudaDeviceAttr a, int) {
    *v = a == cudaDevAttrComputeCapabilityMajor ? 10 : (a == cudaDevAttrComputeCapabilityMinor ? 0 : 148);
    return cudaSuccess;
}
cudaError_t cudaGetSymbolAddress(void **p, const void *) { static unsigned word; *p = &word; return cudaSuccess; }
cudaError_t cudaPointerGetAttributes(cudaPointerAttributes *a, const void *) {
    a->type = cudaMemoryTypeDevice;
    a->device = 0;
    return cudaSuccess;
}
cudaError_t cudaFuncSetAttribute(const void *, cudaFuncAttribute, int) { return cudaSuccess; }
cudaError_t cudaOccupancyMaxActiveBlocksPerMultiprocessor(int *n, const void *, int, size_t) { *n = 2; return cudaSuccess; }
cudaError_t cudaOccupancyMaxActiveBlocksPerMultiprocessorWithFlags(int *n, const void *, int, size_t, unsigned) {
    *n = 2;
    return cudaSuccess;
}
const char *cudaGetErrorString(cudaError_t) { return "error"; }
cudaError_t cudaGetLastError() { return cudaSuccess; }
cudaError_t cudaMemsetAsync(void *, int, size_t, cudaStream_t) { return cudaSuccess; }
cudaError_t cudaStreamSynchronize(cudaStream_t) { return cudaSuccess; }
cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t *, const void *, void **) { return cudaSuccess; }
cudaError_t cudaLaunchKernel(const void *, dim3, dim3, void **, size_t, cudaStream_t) { return cudaSuccess; }
/* what the compiler's own registration code calls */
void **__cudaRegisterFatBinary(void *) { static void *p; return &p; }
void __cudaRegisterFatBinaryEnd(void **) {}
void __cudaUnregisterFatBinary(void **) {}
void __cudaRegisterFunction(void **, const char *, char *, const char *, int, uint3 *, uint3 *, dim3 *, dim3 *, int *) {}
void __cudaRegisterVar(void **, char *, char *, const char *, int, size_t, int, int) {}
unsigned __cudaPushCallConfiguration(dim3, dim3, size_t, void *) { return 0; }
cudaError_t __cudaPopCallConfiguration(dim3 *, dim3 *, size_t *, void *) { return cudaSuccess; }
cudaError_t __cudaGetKernel(cudaKernel_t *, const void *) { return cudaSuccess; }
cudaError_t __cudaLaunchKernel(cudaKernel_t, dim3, dim3, void **, size_t, cudaStream_t) { return cudaSuccess; }
char __cudaInitModule(void **) { return 0; }
}

static int one(int i) {
    kc_paged_kv kv{};
    kv.n_seqs = 4; kv.ld_table = 8; kv.n_pages = 32; kv.page_size = 16; kv.n_kv_heads = 2; kv.head_dim = 64;
    const int types[3] = { KC_F32, KC_F16, KC_Q8_0 };
    kv.kv_type = types[i % 3];
    size_t n = 0;
    if (kc_paged_attend_ws(&kv, 4, &n) != KC_OK || n < 8192) return 1;
    /* addresses that nothing follows */
    void *p = (void *)4096;
    kv.k = kv.v = p;
    kv.kd = kv.vd = (float *)p;
    kv.table = (const int *)p;
    kc_attend_args a{};
    a.q = (const float *)p; a.out = (float *)p; a.ldq = a.ldo = 256; a.lens = (const int *)p;
    a.n_seqs = 4; a.n_heads = 4; a.scale = 1.0f; a.ws = p; a.ws_bytes = n;
    if (kc_paged_attend_dev(&kv, &a, nullptr) != KC_OK) return 2;
    return kc::serve_err_word(0) ? 0 : 3;
}

int main() {
    std::vector<std::thread> ts;
    std::vector<int> rc(12, -1);
    for (int i = 0; i < 12; i++) ts.emplace_back([&rc, i] { rc[i] = one(i); });
    for (auto &t : ts) t.join();
    for (int r : rc)
        if (r) {
            std::printf("status %d\n", r);
            return 1;
        }
    std::printf("ok\n");
    return 0;
}
