// k1_decode_capi.cu -- extern "C" entry points of the decoding-step operators (declared in
// include/k1_logprob.h): residual RMS norm, 8-bit product, token sampling.  Argument
// validation, kernel choice, launches.
#include <algorithm>
#include <cmath>
#include <map>
#include <mutex>
#include <tuple>
#include <utility>

#include "k1_fp8_linear.cuh"
#include "k1_host.cuh"
#include "k1_norm.cuh"
#include "k1_sample.cuh"

cudaError_t k1_decode_wait_status(unsigned* bits) {
    unsigned zero = 0;
    cudaError_t e = cudaMemcpyFromSymbol(bits, k1::k1_ring_error, sizeof *bits);
    if (e == cudaSuccess) e = cudaMemcpyToSymbol(k1::k1_ring_error, &zero, sizeof zero);
    return e;
}

#ifdef K1_WAIT_TEST
cudaError_t k1_decode_set_withhold(long long withhold) {
    return cudaMemcpyToSymbol(k1::k1_test_withhold, &withhold, sizeof withhold);
}

// Host-side tests of the sampling kernel's arithmetic (the wait-timeout test library alone has
// them).  The words of a list of n weights, and the target at which `share` of its mass is reached.
extern "C" void k1_test_list(const float* w, int n, double share, uint64_t* words, uint64_t* target) {
    using namespace k1::sample;
    double mass = 0.0;
    for (int i = 0; i < n; ++i) mass += (double)w[i];
    const double unit = list_unit(mass);
    uint64_t all = 0;
    for (int i = 0; i < n; ++i) all += words[i] = weight_word(w[i], unit);
    *target = list_target(share * mass * unit, word_weight(all));
}

// The element that a lane with these eight weights draws.
extern "C" int k1_test_pick(const float* w, double cum, double target) {
    float v[8];
    for (int i = 0; i < 8; ++i) v[i] = w[i];
    return k1::sample::pick_element(v, cum, target);
}
#endif

namespace {

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

// ---------------------------------------------------------------------------------------
// Residual RMS norm
// ---------------------------------------------------------------------------------------
// Elements per piece (a 16-byte vector, 2 or 1), pieces per thread and threads of a row of
// `hidden` elements; nv is one of the kernel's instances (vectors: 1, 2, 4 or 8; others: 2, 4,
// 8 or 16).
struct NormShape {
    int e, nv, threads;
};

NormShape norm_shape(int hidden, int es, int e) {
    NormShape s;
    s.e = e;
    const int pieces = hidden / e;
    const bool vec = e * es == 16;
    s.nv = vec ? 1 : 2;
    if (vec)
        while (s.nv < 8 && pieces > 256 * s.nv && (s.nv < 2 || pieces > 512 * s.nv)) s.nv *= 2;
    else
        while (pieces > s.nv * k1::norm::kMaxSmall) s.nv *= 2;
    // whole groups of 128 threads, so that the columns of a scale are whole warps
    const int unit = vec ? 32 : 128;
    s.threads = std::max(unit, (pieces + s.nv - 1) / s.nv);
    s.threads = (s.threads + unit - 1) / unit * unit;
    return s;
}

// Blocks of a launch: as many as 2048 threads per SM make (registers, which may let fewer reside,
// are not counted), or the rows if there are fewer.
int64_t norm_grid(int64_t n, int threads, int sms, int most_per_sm) {
    const int per_sm = std::max(1, std::min(most_per_sm, 2048 / threads));
    return std::min<int64_t>(n, (int64_t)sms * per_sm);
}

template <typename T, int OUT, int E, int NV>
cudaError_t norm_launch1(const k1::norm::FwdParams& p, const NormShape& s, int64_t grid, cudaStream_t st) {
    return launch(k1::norm::k1_rmsnorm_kernel<T, E, NV, OUT>, grid, s.threads, 0, st, p);
}

template <typename T, int OUT>
cudaError_t norm_launch(const k1::norm::FwdParams& p, const NormShape& s, int64_t grid, cudaStream_t st) {
    constexpr int V = k1::DT<T>::kEPV;
    switch (s.e * 100 + s.nv) {
        case 102: return norm_launch1<T, OUT, 1, 2>(p, s, grid, st);
        case 104: return norm_launch1<T, OUT, 1, 4>(p, s, grid, st);
        case 108: return norm_launch1<T, OUT, 1, 8>(p, s, grid, st);
        case 116: return norm_launch1<T, OUT, 1, 16>(p, s, grid, st);
        case 202: return norm_launch1<T, OUT, 2, 2>(p, s, grid, st);
        case 204: return norm_launch1<T, OUT, 2, 4>(p, s, grid, st);
        case 208: return norm_launch1<T, OUT, 2, 8>(p, s, grid, st);
        case V * 100 + 1: return norm_launch1<T, OUT, V, 1>(p, s, grid, st);
        case V * 100 + 2: return norm_launch1<T, OUT, V, 2>(p, s, grid, st);
        case V * 100 + 4: return norm_launch1<T, OUT, V, 4>(p, s, grid, st);
        case 408:
            if constexpr (V == 4) return norm_launch1<T, OUT, 4, 8>(p, s, grid, st);
    }
    return cudaErrorInvalidValue;
}

template <typename T, int E, int NV>
cudaError_t norm_bwd_launch1(const k1::norm::BwdParams& p, const NormShape& s, int64_t grid, cudaStream_t st) {
    return launch(k1::norm::k1_rmsnorm_bwd_kernel<T, E, NV>, grid, s.threads, 0, st, p);
}

template <typename T>
cudaError_t norm_bwd_launch(const k1::norm::BwdParams& p, const NormShape& s, int64_t grid, cudaStream_t st) {
    constexpr int V = k1::DT<T>::kEPV;
    switch (s.e * 100 + s.nv) {
        case 102: return norm_bwd_launch1<T, 1, 2>(p, s, grid, st);
        case 104: return norm_bwd_launch1<T, 1, 4>(p, s, grid, st);
        case 108: return norm_bwd_launch1<T, 1, 8>(p, s, grid, st);
        case 116: return norm_bwd_launch1<T, 1, 16>(p, s, grid, st);
        case 202: return norm_bwd_launch1<T, 2, 2>(p, s, grid, st);
        case 204: return norm_bwd_launch1<T, 2, 4>(p, s, grid, st);
        case 208: return norm_bwd_launch1<T, 2, 8>(p, s, grid, st);
        case V * 100 + 1: return norm_bwd_launch1<T, V, 1>(p, s, grid, st);
        case V * 100 + 2: return norm_bwd_launch1<T, V, 2>(p, s, grid, st);
        case V * 100 + 4: return norm_bwd_launch1<T, V, 4>(p, s, grid, st);
        case 408:
            if constexpr (V == 4) return norm_bwd_launch1<T, 4, 8>(p, s, grid, st);
    }
    return cudaErrorInvalidValue;
}

int norm_check(const char* fn, int dtype, int weight_dtype, int64_t n_rows, int64_t hidden) {
    if (!known_dtype(dtype))
        return fail(K1_ERR_UNSUPPORTED_DTYPE, "%s: dtype must be bf16, fp16, or fp32", fn);
    if (weight_dtype != dtype && weight_dtype != K1_DTYPE_F32)
        return fail(K1_ERR_UNSUPPORTED_DTYPE, "%s: the weight must have the inputs' dtype or fp32", fn);
    if (n_rows < 0) return fail(K1_ERR_INVALID_ARGUMENT, "%s: n_rows must be >= 0", fn);
    if (hidden < 1 || hidden > k1::norm::kMaxHidden)
        return fail(K1_ERR_INVALID_ARGUMENT, "%s: hidden must be in [1, %d], got %lld", fn,
                    k1::norm::kMaxHidden, (long long)hidden);
    return K1_OK;
}

// The most of `bytes` at which every row of a matrix starts (NULL: no limit).
int rows_align(const void* p, int64_t stride, int64_t n, int es, int bytes) {
    if (!p) return bytes;
    const uintptr_t at = reinterpret_cast<uintptr_t>(p) | (n > 1 ? (uintptr_t)(stride * es) : 0);
    while (bytes > es && at % bytes != 0) bytes /= 2;
    return bytes;
}

// Elements per piece: a 16-byte vector, a pair, or one, by the width and every address.
int norm_piece(int64_t hidden, int es, int align) {
    if ((hidden * es) % 16 == 0 && align >= 16) return 16 / es;
    return hidden % 2 == 0 && align >= 2 * es ? 2 : 1;
}

// The backward's grid: every block writes a partial row of dw, so no more blocks than keep the
// loads going, and at least four rows each once every SM has a block.  Measured (bf16, us a
// training step of 16384 x 3584 with 3, 4, 6 blocks per SM): 189, 172, 184.
constexpr int kBwdBlocksPerSm = 4;

int64_t norm_bwd_grid(int64_t n, int threads, int sms) {
    return std::min(norm_grid(n, threads, sms, kBwdBlocksPerSm), std::max<int64_t>(sms, n / 4));
}

int norm_forward(const char* fn, int out, const void* x, int64_t x_stride, const void* r, int64_t r_stride,
                 const void* w, int weight_dtype, int dtype, int64_t n, int64_t hidden, float eps, void* s,
                 void* y, float* scales, float* rstd, cudaStream_t st) {
    const bool only = out == k1::norm::FP8_ONLY;
    int rc = norm_check(fn, dtype, only ? dtype : weight_dtype, n, hidden);
    if (rc) return rc;
    if (!only && (!(eps > 0.f) || !std::isfinite(eps)))
        return fail(K1_ERR_INVALID_ARGUMENT, "%s: eps must be positive and finite", fn);
    if (n == 0) return K1_OK;
    if (!x || !y || (!only && !w) || (r && !s) || (out != k1::norm::SAME && !scales))
        return fail(K1_ERR_INVALID_ARGUMENT, "%s: NULL pointer argument", fn);
    const int es = elem_size(dtype);
    if (n > 1 && (x_stride < 0 || (r && r_stride < 0)))
        return fail(K1_ERR_INVALID_ARGUMENT, "%s: strides must be >= 0", fn);
    if (!aligned(x, es) || !aligned(r, es) || !aligned(s, es) || (out == k1::norm::SAME && !aligned(y, es)) ||
        (w && !aligned(w, weight_dtype == K1_DTYPE_F32 ? 4 : es)))
        return fail(K1_ERR_INVALID_ARGUMENT, "%s: a pointer is not aligned to its element size", fn);
    int dev = 0, sms = 0;
    rc = current_device(&dev);
    if (!rc) rc = sm_count(dev, &sms);
    if (rc) return rc;
    // outputs are contiguous; a vector of the weight in fp32 is two or more
    int align = rows_align(x, x_stride, n, es, 16);
    align = rows_align(r, r_stride, n, es, align);
    align = rows_align(s, hidden, n, es, align);
    if (out == k1::norm::SAME) align = rows_align(y, hidden, n, es, align);
    const int e = std::min(norm_piece(hidden, es, align), !w || aligned(w, 16) ? 8 : aligned(w, 2 * es) ? 2 : 1);
    const NormShape sh = norm_shape((int)hidden, es,
                                    out != k1::norm::SAME && !aligned(y, e) ? 1 : e);
    k1::norm::FwdParams p = {};
    p.x = x;
    p.r = r;
    p.w = w;
    p.s = s;
    p.y = y;
    p.scales = scales;
    p.rstd = rstd;
    p.n = n;
    p.x_stride = x_stride;
    p.r_stride = r_stride;
    p.h = (int)hidden;
    p.w32 = weight_dtype == K1_DTYPE_F32;
    p.eps = eps;
    const int64_t grid = norm_grid(n, sh.threads, sms, 8);
    auto go = [&](auto tag) {
        using T = decltype(tag);
        if (out == k1::norm::SAME) return norm_launch<T, k1::norm::SAME>(p, sh, grid, st);
        if (out == k1::norm::FP8) return norm_launch<T, k1::norm::FP8>(p, sh, grid, st);
        return norm_launch<T, k1::norm::FP8_ONLY>(p, sh, grid, st);
    };
    return launched(fn, dtype == K1_DTYPE_BF16  ? go(__nv_bfloat16{})
                        : dtype == K1_DTYPE_F16 ? go(__half{})
                                                : go(float{}));
}

// ---------------------------------------------------------------------------------------
// 8-bit product
// ---------------------------------------------------------------------------------------
// Row-major 8-bit [rows, cols] matrix, rows `stride` bytes apart, read in boxes of
// box_rows x 128 with 128-byte swizzle; what lies beyond it reads as zero.
int make_tmap8(CUtensorMap* m, const void* base, int64_t rows, int64_t cols, int64_t stride, int box_rows,
               const char* what) {
    TmapEncodeFn enc = nullptr;
    int rc = tmap_encoder(&enc);
    if (rc) return rc;
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)stride};
    const cuuint32_t box[2] = {(cuuint32_t)k1::fp8::BK, (cuuint32_t)box_rows};
    const cuuint32_t es[2] = {1, 1};
    CUresult r = enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, es,
                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                     CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(K1_ERR_CUDA, "cuTensorMapEncodeTiled(%s) failed: %d", what, (int)r);
    return K1_OK;
}

// Largest inner dimension: the few-token kernel keeps its scales (up to 64 tokens) in shared
// memory beside the ring.
constexpr int64_t kMaxInner = 32768;

template <int TN, typename OutT>
int skinny(const char* fn, const k1::fp8::Params& p, const void* x, int64_t ldx, const void* w, int64_t ldw,
           int64_t inner, int sms, int dev, cudaStream_t st) {
    using S = k1::fp8::Skinny<TN>;
    CUtensorMap tx, tw;
    int rc = make_tmap8(&tx, x, p.m, inner, ldx, TN, "x");
    if (!rc) rc = make_tmap8(&tw, w, p.n, inner, ldw, k1::fp8::BM, "weight");
    if (rc) return rc;
    const int64_t tiles = (p.n + 127) / 128, tok = (p.m + TN - 1) / TN;
    // K is split over a cluster where a third of the SMs or more would stay without a block,
    // until all have one and while every part keeps two blocks of K.  Measured (us, bf16 out):
    // 100 x 3584 x 4096 in 64 / 128 / 256 parts - / 14.0 / 12.0; 200 x 3584 x 3584 in 112 / 224
    // 15.1 / 18.7; 936 x 800 x 1978 in 240 / 480 8.7 / 22.9.
    int split = 1;
    if (tiles * tok * 3 < 2 * sms)
        while (split < 8 && tiles * tok * split < sms && p.kb_total >= 4 * split) split *= 2;
    auto kern = k1::fp8::k1_fp8_skinny_kernel<TN, OutT>;
    const size_t smem = S::smem((p.kb_total + split - 1) / split);
    rc = allow_smem(kern, dev, smem);
    if (rc) return rc;
    const dim3 grid((unsigned)(tiles * tok * split));
    return launched(fn, launch_cluster(kern, grid, S::THREADS, smem, split, st, tx, tw, p, split));
}

// Pairs of the many-token kernel that can be resident at once; its persistent grid must not
// exceed them.  Cached per device.
template <typename Kernel>
int wide_pairs(Kernel kern, int dev, int* out) {
    static std::atomic<int> cache[kMaxDevices];
    int v = cache[dev].load(std::memory_order_relaxed);
    if (v == 0) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(2);
        cfg.blockDim = dim3(k1::fp8::Wide::THREADS);
        cfg.dynamicSmemBytes = k1::fp8::Wide::SMEM;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = 2;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        cudaError_t e = cudaOccupancyMaxActiveClusters(&v, kern, &cfg);
        if (e != cudaSuccess || v < 1)
            return fail(K1_ERR_CUDA, "cudaOccupancyMaxActiveClusters: %s (%d)", cudaGetErrorString(e), v);
        cache[dev].store(v, std::memory_order_relaxed);
    }
    *out = v;
    return K1_OK;
}

template <typename OutT>
int wide(const char* fn, k1::fp8::Params p, const void* x, int64_t ldx, const void* w, int64_t ldw,
         int64_t inner, int dev, cudaStream_t st) {
    using S = k1::fp8::Wide;
    CUtensorMap tx, tw;
    int rc = make_tmap8(&tx, x, p.m, inner, ldx, k1::fp8::BM, "x");
    if (!rc) rc = make_tmap8(&tw, w, p.n, inner, ldw, S::LOAD_N, "weight");
    if (rc) return rc;
    p.m_tiles = (int)((p.m + S::TM - 1) / S::TM);
    p.n_tiles = (int)((p.n + S::BN - 1) / S::BN);
    const bool aligned16 = ((reinterpret_cast<uintptr_t>(p.y) | (uintptr_t)(p.ldy * sizeof(OutT))) & 15) == 0;
    auto kern = aligned16 ? k1::fp8::k1_fp8_wide_kernel<OutT, true> : k1::fp8::k1_fp8_wide_kernel<OutT, false>;
    int pairs = 0;
    rc = allow_smem(kern, dev, S::SMEM);
    if (!rc) rc = wide_pairs(kern, dev, &pairs);
    if (rc) return rc;
    const dim3 grid((unsigned)(2 * std::min<int64_t>(pairs, (int64_t)p.m_tiles * p.n_tiles)));
    return launched(fn, launch_cluster(kern, grid, S::THREADS, (size_t)S::SMEM, 2, st, tx, tw, p));
}

// The kernel of a product: the tokens per block of the few-token kernel, or 0 for the many-token
// kernel.
int linear_kernel(int64_t m, int64_t n, int kb_total, int sms) {
    if (m <= 16) return 16;
    if (m <= 32) return 32;
    // The few-token kernel in blocks of 64 tokens (two blocks of threads per SM) or the
    // many-token kernel (a tile per two SMs), by their rounds times what a round takes: about
    // 4 + 0.65 us per block of K, and 10 + 0.6.  Measured (us, few / many): 936 x 800 x 1978
    // 8.7 / 17.2; 162 x 1328 x 12141 12.9 / 20.3; 142 x 4352 x 14269 41 / 33; 300 x 3584 x 8192
    // 34 / 26; 128 x 3584 x 32768 43 / 44; 2180 x 6160 x 3492 127 / 71.
    const int64_t few = (m + 63) / 64 * ((n + 127) / 128), many = (m + 255) / 256 * ((n + 255) / 256);
    const double few_us = (double)((few + 2 * sms - 1) / (2 * sms)) * (4.0 + 0.65 * kb_total);
    const double many_us = (double)((many + sms / 2 - 1) / (sms / 2)) * (10.0 + 0.6 * kb_total);
    return m <= 64 || few_us <= many_us ? 64 : 0;
}

template <typename OutT>
int linear(const char* fn, const k1::fp8::Params& p, const void* x, int64_t ldx, const void* w, int64_t ldw,
           int64_t inner, int sms, int dev, cudaStream_t st) {
    switch (linear_kernel(p.m, p.n, p.kb_total, sms)) {
        case 16: return skinny<16, OutT>(fn, p, x, ldx, w, ldw, inner, sms, dev, st);
        case 32: return skinny<32, OutT>(fn, p, x, ldx, w, ldw, inner, sms, dev, st);
        case 64: return skinny<64, OutT>(fn, p, x, ldx, w, ldw, inner, sms, dev, st);
        default: return wide<OutT>(fn, p, x, ldx, w, ldw, inner, dev, st);
    }
}

// ---------------------------------------------------------------------------------------
// Sampling
// ---------------------------------------------------------------------------------------
template <typename T, bool FILTER>
int sample_launch(const char* fn, k1::sample::Params p, int sms, int dev, cudaStream_t st) {
    using namespace k1::sample;
    constexpr int E = k1::DT<T>::kEPV;
    // Bytes of a row's part in one block: what lets two blocks with lists (113 KB each, 300 x
    // 70000 fp32, top-k 50: 75 us, 100 with one), or five without, share an SM (with lists, 512
    // rows of 152064 bf16, top-k 50: 157 us in four parts of 76 KB, 239 in eight of 38); a lone
    // block takes up to kLone; a row that is longer still stays in global memory.
    constexpr int64_t kShared = FILTER ? 113 * 1024 - (int64_t)smem_header<true>() : 48 * 1024;
    constexpr int64_t kLone = 184 * 1024, kLeast = 8 * 1024;
    const int64_t row_bytes = ((p.vocab + E - 1) / E + 1) * 16;  // one more for the shift
    // As few parts as fit where the rows fill the device 2.5 times or more, else a power of two
    // of them, whose shorter parts end a partial round sooner.  Measured (us, filters, 128256
    // wide, fewest / power of two): fp32 in 6 / 8, 567 rows 232 / 262, 150 rows 68 / 74, 64 rows
    // 88 / 84; bf16 in 3 / 4, 512 rows 131 / 138, 200 rows 218 / 214, 64 rows 97 / 82.
    const int fewest = (int)std::min<int64_t>((row_bytes + kShared - 1) / kShared, kMaxCluster);
    int cluster = 1;
    while (cluster < fewest) cluster *= 2;
    if (FILTER && p.n_rows * fewest >= 5 * sms) cluster = fewest;
    // few rows: more blocks per row, so that the SMs share the load
    while (cluster < kMaxCluster && p.n_rows * cluster < sms && row_bytes > 2 * cluster * kLeast) cluster *= 2;
    const int64_t vecs = (row_bytes / 16 + cluster - 1) / cluster;
    if (vecs > (int64_t)1 << 30) return fail(K1_ERR_INVALID_ARGUMENT, "%s: vocab too large", fn);
    p.cluster = cluster;
    p.slice_vecs = (int)vecs;
    const bool resident = vecs * 16 <= kLone;
    const size_t smem = smem_header<FILTER>() + (resident ? (size_t)vecs * 16 : 0);
    auto kern = resident ? k1_sample_kernel<T, true, FILTER> : k1_sample_kernel<T, false, FILTER>;
    int rc = allow_smem(kern, dev, smem);
    if (rc) return rc;
    const dim3 grid((unsigned)(p.n_rows * cluster));
    return launched(fn, launch_cluster(kern, grid, FILTER ? kFilterThreads : kPlainThreads, smem, cluster, st, p));
}

template <typename T>
int sample(const char* fn, const k1::sample::Params& p, int sms, int dev, cudaStream_t st) {
    // settings that may cut the distribution of some row (temperature 0 does)
    const bool filter = p.temperature || p.top_k || p.top_p || p.min_p || p.greedy0 || p.top_p0 < 1.f ||
                        (p.top_k0 > 0 && p.top_k0 < p.vocab) || p.min_p0 > 0.f;
    return filter ? sample_launch<T, true>(fn, p, sms, dev, st) : sample_launch<T, false>(fn, p, sms, dev, st);
}

}  // namespace

extern "C" {

#ifdef K1_WAIT_TEST
// Which kernel a product takes on a device of `sms` SMs, so that a test knows which one it tests.
int k1_test_linear_kernel(int64_t tokens, int64_t inner, int64_t outer, int sms) {
    return linear_kernel(tokens, outer, (int)((inner + 127) / 128), sms);
}
#endif

int k1_residual_rmsnorm(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride,
                        const void* weight, int weight_dtype, int dtype, int64_t n_rows, int64_t hidden,
                        float eps, void* stream_out, void* y, float* rstd, void* stream) {
    return norm_forward("k1_residual_rmsnorm", k1::norm::SAME, x, x_stride, residual, residual_stride, weight,
                        weight_dtype, dtype, n_rows, hidden, eps, stream_out, y, nullptr, rstd,
                        reinterpret_cast<cudaStream_t>(stream));
}

int k1_residual_rmsnorm_fp8(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride,
                            const void* weight, int weight_dtype, int dtype, int64_t n_rows, int64_t hidden,
                            float eps, void* stream_out, void* q, float* scales, void* stream) {
    return norm_forward("k1_residual_rmsnorm_fp8", k1::norm::FP8, x, x_stride, residual, residual_stride, weight,
                        weight_dtype, dtype, n_rows, hidden, eps, stream_out, q, scales, nullptr,
                        reinterpret_cast<cudaStream_t>(stream));
}

int k1_quantize_fp8_rows(const void* x, int64_t x_stride, int dtype, int64_t n_rows, int64_t hidden, void* q,
                         float* scales, void* stream) {
    return norm_forward("k1_quantize_fp8_rows", k1::norm::FP8_ONLY, x, x_stride, nullptr, 0, nullptr, dtype, dtype,
                        n_rows, hidden, 0.f, nullptr, q, scales, nullptr, reinterpret_cast<cudaStream_t>(stream));
}

int k1_quantize_fp8_blocks(const void* w, int64_t w_stride, int dtype, int64_t rows, int64_t cols, void* q,
                           float* scales, void* stream) {
    static const char* fn = "k1_quantize_fp8_blocks";
    if (!known_dtype(dtype))
        return fail(K1_ERR_UNSUPPORTED_DTYPE, "%s: dtype must be bf16, fp16, or fp32", fn);
    if (rows < 0 || cols < 1) return fail(K1_ERR_INVALID_ARGUMENT, "%s: rows must be >= 0 and cols >= 1", fn);
    if (rows > (int64_t)65535 * 128 || cols > (int64_t)65535 * 128)
        return fail(K1_ERR_INVALID_ARGUMENT, "%s: at most %lld rows and columns", fn, (long long)65535 * 128);
    if (rows == 0) return K1_OK;
    if (!w || !q || !scales) return fail(K1_ERR_INVALID_ARGUMENT, "%s: NULL pointer argument", fn);
    if (w_stride < 0) return fail(K1_ERR_INVALID_ARGUMENT, "%s: strides must be >= 0", fn);
    if (!aligned(w, elem_size(dtype)))
        return fail(K1_ERR_INVALID_ARGUMENT, "%s: a pointer is not aligned to its element size", fn);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((cols + 127) / 128), (unsigned)((rows + 127) / 128));
    cfg.blockDim = dim3(256);
    cfg.stream = reinterpret_cast<cudaStream_t>(stream);
    auto go = [&](auto tag) {
        using T = decltype(tag);
        return cudaLaunchKernelEx(&cfg, k1::norm::k1_quantize_blocks_kernel<T>, reinterpret_cast<const T*>(w),
                                  w_stride, rows, cols, reinterpret_cast<uint8_t*>(q), scales);
    };
    return launched(fn, dtype == K1_DTYPE_BF16  ? go(__nv_bfloat16{})
                        : dtype == K1_DTYPE_F16 ? go(__half{})
                                                : go(float{}));
}

size_t k1_residual_rmsnorm_workspace_bytes(int64_t n_rows, int64_t hidden, int device) {
    int sms = 0;
    if (n_rows < 0 || hidden < 1 || hidden > k1::norm::kMaxHidden || device < 0 || device >= kMaxDevices ||
        sm_count(device, &sms) != K1_OK)
        return 0;
    return (size_t)std::min<int64_t>(std::max<int64_t>(n_rows, 1), (int64_t)sms * kBwdBlocksPerSm) *
           (size_t)hidden * sizeof(float);
}

int k1_residual_rmsnorm_backward(const void* g_y, int64_t g_y_stride, const void* g_stream,
                                 int64_t g_stream_stride, const void* stream_in, int64_t stream_stride,
                                 const float* rstd, const void* weight, int weight_dtype, int dtype,
                                 int64_t n_rows, int64_t hidden, void* d_x, void* d_weight, void* workspace,
                                 size_t workspace_bytes, void* stream) {
    static const char* fn = "k1_residual_rmsnorm_backward";
    int rc = norm_check(fn, dtype, weight_dtype, n_rows, hidden);
    if (rc) return rc;
    const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const int es = elem_size(dtype), ws = elem_size(weight_dtype);
    if (n_rows == 0) {
        if (d_weight) {
            cudaError_t e = cudaMemsetAsync(d_weight, 0, (size_t)hidden * ws, st);
            if (e != cudaSuccess) return fail(K1_ERR_CUDA, "%s: %s", fn, cudaGetErrorString(e));
        }
        return K1_OK;
    }
    if (!g_y || !stream_in || !rstd || !weight)
        return fail(K1_ERR_INVALID_ARGUMENT, "%s: NULL pointer argument", fn);
    if (!d_x && !d_weight) return K1_OK;
    if (n_rows > 1 && (g_y_stride < 0 || stream_stride < 0 || (g_stream && g_stream_stride < 0)))
        return fail(K1_ERR_INVALID_ARGUMENT, "%s: strides must be >= 0", fn);
    if (!aligned(g_y, es) || !aligned(g_stream, es) || !aligned(stream_in, es) || !aligned(d_x, es) ||
        !aligned(weight, ws) || !aligned(d_weight, ws))
        return fail(K1_ERR_INVALID_ARGUMENT, "%s: a pointer is not aligned to its element size", fn);
    int dev = 0, sms = 0;
    rc = current_device(&dev);
    if (!rc) rc = sm_count(dev, &sms);
    if (rc) return rc;
    int align = rows_align(g_y, g_y_stride, n_rows, es, 16);
    align = rows_align(g_stream, g_stream_stride, n_rows, es, align);
    align = rows_align(stream_in, stream_stride, n_rows, es, align);
    align = rows_align(d_x, hidden, n_rows, es, align);
    const NormShape sh = norm_shape(
        (int)hidden, es, std::min(norm_piece(hidden, es, align), aligned(weight, 16) ? 8 : aligned(weight, 2 * es) ? 2 : 1));
    const int64_t grid = norm_bwd_grid(n_rows, sh.threads, sms);
    if (d_weight && (!workspace || !aligned(workspace, 16) ||
                     workspace_bytes < (size_t)grid * hidden * sizeof(float)))
        return fail(K1_ERR_WORKSPACE, "%s: the weight's gradient needs %zu bytes of 16-byte aligned workspace", fn,
                    k1_residual_rmsnorm_workspace_bytes(n_rows, hidden, dev));
    k1::norm::BwdParams p = {};
    p.gy = g_y;
    p.gs = g_stream;
    p.s = stream_in;
    p.rstd = rstd;
    p.w = weight;
    p.ds = d_x;
    p.dw = d_weight ? reinterpret_cast<float*>(workspace) : nullptr;
    p.n = n_rows;
    p.gy_stride = g_y_stride;
    p.gs_stride = g_stream_stride;
    p.s_stride = stream_stride;
    p.h = (int)hidden;
    p.w32 = weight_dtype == K1_DTYPE_F32;
    rc = launched(fn, dtype == K1_DTYPE_BF16  ? norm_bwd_launch<__nv_bfloat16>(p, sh, grid, st)
                      : dtype == K1_DTYPE_F16 ? norm_bwd_launch<__half>(p, sh, grid, st)
                                              : norm_bwd_launch<float>(p, sh, grid, st));
    if (rc || !d_weight) return rc;
    const int64_t blocks = (hidden + 31) / 32;
    auto sum = [&](auto tag) {
        using W = decltype(tag);
        return launch(k1::norm::k1_rmsnorm_dw_kernel<W>, blocks, 512, 0, st, (const float*)p.dw, (int)grid,
                      (int)hidden, reinterpret_cast<W*>(d_weight));
    };
    return launched(fn, weight_dtype == K1_DTYPE_BF16  ? sum(__nv_bfloat16{})
                        : weight_dtype == K1_DTYPE_F16 ? sum(__half{})
                                                       : sum(float{}));
}

int k1_fp8_linear(const void* x, int64_t x_stride, const float* x_scales, const void* weight,
                  int64_t weight_stride, const float* weight_scales, int64_t tokens, int64_t inner,
                  int64_t outer, void* y, int64_t y_stride, int out_dtype, void* stream) {
    static const char* fn = "k1_fp8_linear";
    if (!known_dtype(out_dtype))
        return fail(K1_ERR_UNSUPPORTED_DTYPE, "%s: the output's dtype must be bf16, fp16, or fp32", fn);
    if (tokens < 0 || outer < 0) return fail(K1_ERR_INVALID_ARGUMENT, "%s: tokens and outer must be >= 0", fn);
    if (inner < 16 || inner % 16 != 0 || inner > kMaxInner)
        return fail(K1_ERR_INVALID_ARGUMENT, "%s: inner must be a multiple of 16 in [16, %lld], got %lld", fn,
                    (long long)kMaxInner, (long long)inner);
    if (tokens > (int64_t)1 << 24 || outer > (int64_t)1 << 27 || (tokens + 63) / 64 * ((outer + 127) / 128) > (int64_t)1 << 28)
        return fail(K1_ERR_INVALID_ARGUMENT, "%s: tokens or outer too large", fn);
    if (tokens == 0 || outer == 0) return K1_OK;
    if (!x || !x_scales || !weight || !weight_scales || !y)
        return fail(K1_ERR_INVALID_ARGUMENT, "%s: NULL pointer argument", fn);
    if (!aligned(x, 16) || !aligned(weight, 16) || x_stride % 16 != 0 || weight_stride % 16 != 0 ||
        x_stride < inner || weight_stride < inner)
        return fail(K1_ERR_INVALID_ARGUMENT,
                    "%s: x and weight rows must start at multiples of 16 bytes and not overlap", fn);
    if (y_stride < outer) return fail(K1_ERR_INVALID_ARGUMENT, "%s: y_stride must be >= outer", fn);
    if (!aligned(y, elem_size(out_dtype)) || !aligned(x_scales, 4) || !aligned(weight_scales, 4))
        return fail(K1_ERR_INVALID_ARGUMENT, "%s: a pointer is not aligned to its element size", fn);
    int dev = 0, sms = 0;
    int rc = current_device(&dev);
    if (!rc) rc = sm_count(dev, &sms);
    if (rc) return rc;
    k1::fp8::Params p = {};
    p.xs = x_scales;
    p.ws = weight_scales;
    p.y = y;
    p.m = tokens;
    p.n = outer;
    p.ldy = y_stride;
    p.kb_total = (int)((inner + 127) / 128);
    const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    switch (out_dtype) {
        case K1_DTYPE_BF16:
            return linear<__nv_bfloat16>(fn, p, x, x_stride, weight, weight_stride, inner, sms, dev, st);
        case K1_DTYPE_F16:
            return linear<__half>(fn, p, x, x_stride, weight, weight_stride, inner, sms, dev, st);
        default:
            return linear<float>(fn, p, x, x_stride, weight, weight_stride, inner, sms, dev, st);
    }
}

int k1_sample_tokens(const void* logits, int dtype, int64_t n_rows, int64_t vocab, int64_t row_stride,
                     const float* u, const k1_sampling* s, int64_t* token, float* logprob,
                     float* kept_logprob, void* stream) {
    static const char* fn = "k1_sample_tokens";
    if (!known_dtype(dtype))
        return fail(K1_ERR_UNSUPPORTED_DTYPE, "%s: logits dtype must be bf16, fp16, or fp32", fn);
    if (n_rows < 0) return fail(K1_ERR_INVALID_ARGUMENT, "%s: n_rows must be >= 0", fn);
    if (vocab < 1 || vocab > INT32_MAX)
        return fail(K1_ERR_INVALID_ARGUMENT, "%s: vocab must be in [1, 2^31)", fn);
    if (n_rows > (INT32_MAX / k1::sample::kMaxCluster))
        return fail(K1_ERR_INVALID_ARGUMENT, "%s: too many rows", fn);
    if (!s) return fail(K1_ERR_INVALID_ARGUMENT, "%s: NULL settings", fn);
    if (!s->temperature_rows && !(s->temperature >= 0.0 && std::isfinite(s->temperature)))
        return fail(K1_ERR_INVALID_ARGUMENT, "%s: temperature must be finite and >= 0", fn);
    if (!s->top_p_rows && !(s->top_p >= 0.f))
        return fail(K1_ERR_INVALID_ARGUMENT, "%s: top_p must be >= 0", fn);
    if (!s->min_p_rows && !(s->min_p >= 0.f && s->min_p <= 1.f))
        return fail(K1_ERR_INVALID_ARGUMENT, "%s: min_p must be in [0, 1]", fn);
    if (n_rows == 0) return K1_OK;
    if (!logits || !u || !token || !logprob || !kept_logprob)
        return fail(K1_ERR_INVALID_ARGUMENT, "%s: NULL pointer argument", fn);
    if (n_rows > 1 && row_stride < 0) return fail(K1_ERR_INVALID_ARGUMENT, "%s: strides must be >= 0", fn);
    if (!aligned(logits, elem_size(dtype)))
        return fail(K1_ERR_INVALID_ARGUMENT, "%s: logits not aligned to its element size", fn);
    int dev = 0, sms = 0;
    int rc = current_device(&dev);
    if (!rc) rc = sm_count(dev, &sms);
    if (rc) return rc;
    k1::sample::Params p = {};
    p.logits = logits;
    p.n_rows = n_rows;
    p.vocab = vocab;
    p.row_stride = row_stride;
    p.u = u;
    p.temperature = s->temperature_rows;
    p.top_k = s->top_k_rows;
    p.top_p = s->top_p_rows;
    p.min_p = s->min_p_rows;
    p.greedy0 = s->temperature == 0.0;
    p.scale0 = p.greedy0 ? 1.f : (float)(1.0 / s->temperature);
    p.top_k0 = s->top_k;
    p.top_p0 = s->top_p;
    p.min_p0 = s->min_p;
    p.token = token;
    p.logprob = logprob;
    p.kept_logprob = kept_logprob;
    const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    switch (dtype) {
        case K1_DTYPE_BF16: return sample<__nv_bfloat16>(fn, p, sms, dev, st);
        case K1_DTYPE_F16: return sample<__half>(fn, p, sms, dev, st);
        default: return sample<float>(fn, p, sms, dev, st);
    }
}

}  // extern "C"
