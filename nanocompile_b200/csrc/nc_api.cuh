// nc_api.cuh -- host-side helpers of the C entry points: errors, launches.
#pragma once

#include "../../include/nc_cuda.h"

#include <atomic>
#include <cstdint>
#include <cstdlib>

#include <cuda_runtime.h>

namespace nc {

// Records the message of nc_last_error on this thread and returns `code`.
__attribute__((visibility("hidden"), format(printf, 2, 3))) int32_t fail(int32_t code, const char *fmt, ...);

// Whether a bounded wait of the serving kernels has run out since the last call (nc_serving.cu).
__attribute__((visibility("hidden"))) int32_t prompt_fault(bool *fault);
// Their g_wait_cycles: each source file has its own.
__attribute__((visibility("hidden"))) int32_t set_prompt_wait_limit(long long cycles);
// The same of the adapters' kernels (nc_requests.cu).
__attribute__((visibility("hidden"))) int32_t requests_fault(const char **what);
__attribute__((visibility("hidden"))) int32_t set_requests_wait_limit(long long cycles);

#define CUDA_TRY(expr)                                                                           \
    do {                                                                                         \
        cudaError_t e_ = (expr);                                                                 \
        if (e_ != cudaSuccess)                                                                   \
            return nc::fail(NC_ERR_CUDA, "%s failed: %s (%s:%d)", #expr, cudaGetErrorString(e_), \
                            __FILE__, __LINE__);                                                 \
    } while (0)

#define NC_TRY(expr)                  \
    do {                              \
        int32_t s_ = (expr);          \
        if (s_ != NC_OK) return s_;   \
    } while (0)

// Every kernel of the step is launched with programmatic stream serialization (PDL): it may
// begin while its predecessor runs, prefetch immutable data (weights), and wait in-kernel for
// the predecessor's results.  NC_PDL=0 in the environment turns it off (for A/B timing).
inline bool pdl_enabled() {
    static const bool on = [] {
        const char *v = std::getenv("NC_PDL");
        return !(v && v[0] == '0');
    }();
    return on;
}

constexpr int64_t I32 = (int64_t(1) << 31) - 1;
// Whether an address or a number of bytes is no multiple of n, a power of two.
inline bool misaligned(const void *p, int64_t n) { return ((uintptr_t)p & (uintptr_t)(n - 1)) != 0; }
inline bool misaligned(int64_t v, int64_t n) { return (v & (n - 1)) != 0; }

inline int sm_count() {
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
        return 148;
    return sms > 0 ? sms : 148;
}

template <typename... KArgs, typename... Args>
cudaError_t launch_k(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}

template <typename K>
cudaError_t allow_smem(K kernel, size_t bytes) {
    if (bytes <= 48 * 1024) return cudaSuccess;
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
}

// Raises a kernel's limit of shared memory, once on each device (`allowed`: a bit for each).
template <typename K>
int32_t allow_smem_once(K kernel, size_t bytes, std::atomic<uint64_t> *allowed) {
    int device = 0;
    CUDA_TRY(cudaGetDevice(&device));
    if (device < 64 && (allowed->load(std::memory_order_relaxed) >> device & 1)) return NC_OK;
    CUDA_TRY(allow_smem(kernel, bytes));
    if (device < 64) allowed->fetch_or(uint64_t(1) << device, std::memory_order_relaxed);
    return NC_OK;
}

inline int32_t check_launch(const char *what) {
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return fail(NC_ERR_CUDA, "launching %s: %s", what, cudaGetErrorString(e));
    return NC_OK;
}

}  // namespace nc
