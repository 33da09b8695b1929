// k1_host.cuh -- host-side helpers shared by the C ABI's translation units: error
// reporting, launches, device queries, the tensor-map encoder.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <map>
#include <mutex>
#include <string>
#include <tuple>
#include <utility>

#include "k1_logprob.h"

// Not part of the C ABI: one definition (k1_capi.cu) for all translation units.
#define K1_INTERNAL __attribute__((visibility("hidden")))
K1_INTERNAL int k1_host_fail(int code, const char* message);
// The wait status word and test knobs of the other translation units' kernels.
K1_INTERNAL cudaError_t k1_decode_wait_status(unsigned* bits);
K1_INTERNAL cudaError_t k1_sandwich_wait_status(unsigned* bits);
#ifdef K1_WAIT_TEST
K1_INTERNAL cudaError_t k1_decode_set_withhold(long long withhold);
K1_INTERNAL cudaError_t k1_sandwich_set_withhold(long long withhold);
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

bool known_dtype(int d) { return d == K1_DTYPE_F32 || d == K1_DTYPE_F16 || d == K1_DTYPE_BF16; }

bool aligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

// Opt in to `smem` bytes of dynamic shared memory, once per device and kernel (the largest
// asked for so far).
template <typename Kernel>
int allow_smem(Kernel kernel, int dev, size_t smem) {
    static std::mutex mu;
    static std::map<std::pair<int, const void*>, size_t> cache;
    std::lock_guard<std::mutex> lock(mu);
    size_t& have = cache[std::make_pair(dev, reinterpret_cast<const void*>(kernel))];
    if (smem <= have) return K1_OK;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return fail(K1_ERR_CUDA, "cudaFuncSetAttribute(smem): %s", cudaGetErrorString(e));
    have = smem;
    return K1_OK;
}

// Blocks of `threads` threads and `smem` bytes of dynamic shared memory that an SM holds at once.
// Cached per device and launch shape.
template <typename Kernel>
int resident_blocks(Kernel kernel, int dev, int threads, size_t smem, int* out) {
    static std::mutex mu;
    static std::map<std::tuple<int, const void*, int, size_t>, int> cache;
    std::lock_guard<std::mutex> lock(mu);
    int& have = cache[std::make_tuple(dev, reinterpret_cast<const void*>(kernel), threads, smem)];
    if (have == 0) {
        cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&have, kernel, threads, smem);
        if (e != cudaSuccess || have < 1) {
            have = 0;
            return fail(K1_ERR_CUDA, "cudaOccupancyMaxActiveBlocksPerMultiprocessor: %s", cudaGetErrorString(e));
        }
    }
    *out = have;
    return K1_OK;
}

// `launch` with a cluster of `cluster` blocks along x.
template <typename... KArgs, typename... Args>
cudaError_t launch_cluster(void (*kernel)(KArgs...), dim3 grid, int block, size_t smem, int cluster,
                           cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)cluster;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = K1_PDL ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

int launched(const char* fn, cudaError_t e) {
    if (e != cudaSuccess) {
        cudaGetLastError();
        return fail(K1_ERR_CUDA, "%s: kernel launch failed: %s", fn, cudaGetErrorString(e));
    }
    return K1_OK;
}

}  // namespace
