// k1_host.cuh -- host-side helpers shared by the C ABI's translation units: error
// reporting, launches, device queries, the tensor-map encoder.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <mutex>
#include <string>

#include "k1_logprob.h"

// Not part of the C ABI: one definition (k1_capi.cu) for all translation units.
#define K1_INTERNAL __attribute__((visibility("hidden")))
K1_INTERNAL int k1_host_fail(int code, const char* message);
// The wait status word and test knobs of k1_decode_capi.cu's kernels.
K1_INTERNAL cudaError_t k1_decode_wait_status(unsigned* bits);
#ifdef K1_WAIT_TEST
K1_INTERNAL cudaError_t k1_decode_set_withhold(long long withhold);
#endif

namespace {

constexpr int kMaxDevices = 64;

int fail(int code, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    return k1_host_fail(code, buf);
}

#ifndef K1_PDL
#define K1_PDL 1
#endif

// Launch with programmatic stream serialization (see pdl_wait / pdl_trigger): the grid
// may be scheduled while the previous kernel of the stream drains; it waits for that
// kernel's completion on the device before touching memory.
template <typename... KArgs, typename... Args>
cudaError_t launch(void (*kernel)(KArgs...), int64_t grid, int block, size_t smem,
                   cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3((unsigned)block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = K1_PDL ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

int check_launch(const char* what) {
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess)
        return fail(K1_ERR_CUDA, "%s: kernel launch failed: %s", what, cudaGetErrorString(e));
    return K1_OK;
}

int elem_size(int dtype) { return dtype == K1_DTYPE_F32 ? 4 : 2; }

int current_device(int* dev) {
    cudaError_t e = cudaGetDevice(dev);
    if (e != cudaSuccess) return fail(K1_ERR_CUDA, "cudaGetDevice: %s", cudaGetErrorString(e));
    if (*dev < 0 || *dev >= kMaxDevices) return fail(K1_ERR_CUDA, "device ordinal %d out of range", *dev);
    return K1_OK;
}

int sm_count(int dev, int* out) {
    static std::atomic<int> cache[kMaxDevices];
    int v = cache[dev].load(std::memory_order_relaxed);
    if (v == 0) {
        cudaError_t e = cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev);
        if (e != cudaSuccess)
            return fail(K1_ERR_CUDA, "cudaDeviceGetAttribute(SM count): %s", cudaGetErrorString(e));
        cache[dev].store(v, std::memory_order_relaxed);
    }
    *out = v;
    return K1_OK;
}

using TmapEncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                  const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// cuTensorMapEncodeTiled from the driver, looked up through the runtime (no link-time
// dependency on libcuda).
int tmap_encoder(TmapEncodeFn* out) {
    static std::once_flag once;
    static TmapEncodeFn fn = nullptr;
    std::call_once(once, [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) ==
                cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<TmapEncodeFn>(f);
    });
    if (!fn) return fail(K1_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    *out = fn;
    return K1_OK;
}

}  // namespace
