// k1_sandwich_capi.cu -- extern "C" entry points of the norms around a block's end (declared in
// include/k1_logprob.h): argument validation, kernel choice, launches.
#include <algorithm>
#include <cmath>

#include "k1_norm_host.cuh"
#include "k1_sandwich.cuh"

cudaError_t k1_sandwich_wait_status(unsigned* bits) {
    unsigned zero = 0;
    cudaError_t e = cudaMemcpyFromSymbol(bits, k1::k1_ring_error, sizeof *bits);
    if (e == cudaSuccess) e = cudaMemcpyToSymbol(k1::k1_ring_error, &zero, sizeof zero);
    return e;
}

#ifdef K1_WAIT_TEST
cudaError_t k1_sandwich_set_withhold(long long withhold) {
    return cudaMemcpyToSymbol(k1::k1_test_withhold, &withhold, sizeof withhold);
}

// Not part of the product: see k1_test_lone.
extern "C" int k1_test_set_lone(long long row) {
    return cudaMemcpyToSymbol(k1::norm::k1_test_lone, &row, sizeof row) == cudaSuccess ? K1_OK : K1_ERR_CUDA;
}
#endif

namespace {

using k1::norm::GATE_COLUMN;
using k1::norm::GATE_FULL;
using k1::norm::GATE_NONE;
using k1::norm::GATE_TOKEN;

// The instance of a shape: f(E, NV) as integral constants.
template <typename T, typename F>
cudaError_t with_shape(const NormShape& s, F f) {
    constexpr int V = k1::DT<T>::kEPV;
    auto c = [](auto v) { return v; };
#define K1_SHAPE(e, nv) return f(c(std::integral_constant<int, e>{}), c(std::integral_constant<int, nv>{}))
    switch (s.e * 100 + s.nv) {
        case 102: K1_SHAPE(1, 2);
        case 104: K1_SHAPE(1, 4);
        case 108: K1_SHAPE(1, 8);
        case 116: K1_SHAPE(1, 16);
        case 202: K1_SHAPE(2, 2);
        case 204: K1_SHAPE(2, 4);
        case 208: K1_SHAPE(2, 8);
        case V * 100 + 1: K1_SHAPE(V, 1);
        case V * 100 + 2: K1_SHAPE(V, 2);
        case V * 100 + 4: K1_SHAPE(V, 4);
        case 408:
            if constexpr (V == 4) K1_SHAPE(4, 8);
    }
#undef K1_SHAPE
    return cudaErrorInvalidValue;
}

// The ring kernels' layout for rows of vectors of `inputs` tensors, or groups = 0 where they do not
// serve: few rows (their latency counts, and the ring's set-up), rows shorter than 512 bytes, rows of
// more than two vectors per thread, or of which a block cannot hold two.  one, two: threads of a block
// with one and two vectors each.
constexpr size_t kRingShared = 224 * 1024;
constexpr int kRingOne = 256;  // vectors of a row that get a thread each
k1::norm::Ring ring_of(int e, int64_t n, int64_t hidden, int es, int inputs, int one, int two, int sms) {
    k1::norm::Ring q = {};
    const int vecs = (int)(hidden / e);
    if (e * es != 16 || n <= sms || hidden * es < 512 || vecs > 1024) return q;
    q.e = e;
    q.nv = vecs <= kRingOne ? 1 : 2;
    q.threads = ((vecs + q.nv - 1) / q.nv + 31) / 32 * 32;
    q.inputs = inputs;
    q.slot = (int)((hidden * es + 127) / 128 * 128);
    q.groups = (int)std::min<int64_t>({k1::norm::kMaxRingGroups, (q.nv == 1 ? one : two) / q.threads, (n + sms - 1) / sms});
    for (; q.groups > 0; --q.groups)
        for (q.stages = k1::norm::kMaxRingStages; q.stages >= 2; --q.stages)
            if (ring_smem(q) <= kRingShared) return q;
    q.groups = 0;
    return q;
}

// The instance of a ring kernel: f(NV).
template <typename F>
cudaError_t with_ring(const k1::norm::Ring& q, F f) {
    if (q.nv == 1) return f(std::integral_constant<int, 1>{});
    return f(std::integral_constant<int, 2>{});
}

// Checks that forward and backward share.
int sandwich_check(const char* fn, int dtype, int weight_dtype, int64_t n_rows, int64_t hidden, int gate_kind,
                   float branch_scale, float residual_scale) {
    int rc = norm_check(fn, dtype, weight_dtype, n_rows, hidden);
    if (rc) return rc;
    if (gate_kind < GATE_NONE || gate_kind > GATE_FULL)
        return fail(K1_ERR_INVALID_ARGUMENT, "%s: gate_kind must be one of K1_GATE_*, got %d", fn, gate_kind);
    if (!std::isfinite(branch_scale) || !std::isfinite(residual_scale))
        return fail(K1_ERR_INVALID_ARGUMENT, "%s: branch_scale and residual_scale must be finite", fn);
    return K1_OK;
}

// Rows of the gate that vectors must fit, and weights' alignment.
int gate_align(const void* gate, int kind, int64_t stride, int64_t n, int es, int align) {
    return kind == GATE_FULL ? rows_align(gate, stride, n, es, align) : align;
}
int weights_piece(int es, std::initializer_list<const void*> weights) {
    int e = 8;
    for (const void* w : weights) e = std::min(e, !w || aligned(w, 16) ? 8 : aligned(w, 2 * es) ? 2 : 1);
    return e;
}

int sandwich_forward(const char* fn, int out, const void* x, int64_t x_stride, const void* r, int64_t r_stride,
                     const void* wp, const void* gate, int gate_kind, int64_t gate_stride, const void* w,
                     int weight_dtype, int dtype, int64_t n, int64_t hidden, float branch_scale, float residual_scale,
                     float eps, void* s, void* y, float* scales, float* rstd_post, float* rstd, cudaStream_t st) {
    int rc = sandwich_check(fn, dtype, weight_dtype, n, hidden, gate_kind, branch_scale, residual_scale);
    if (rc) return rc;
    if (!(eps > 0.f) || !std::isfinite(eps))
        return fail(K1_ERR_INVALID_ARGUMENT, "%s: eps must be positive and finite", fn);
    if (n == 0) return K1_OK;
    const bool same = out == k1::norm::SAME;
    if (!x || !r || !wp || !w || !s || !y || (gate_kind != GATE_NONE && !gate) || (!same && !scales))
        return fail(K1_ERR_INVALID_ARGUMENT, "%s: NULL pointer argument", fn);
    if (n > 1 && (x_stride < 0 || r_stride < 0 || (gate_kind >= GATE_TOKEN && gate_stride < 0)))
        return fail(K1_ERR_INVALID_ARGUMENT, "%s: strides must be >= 0", fn);
    const int es = elem_size(dtype), ws = elem_size(weight_dtype);
    const void* column = gate_kind == GATE_COLUMN ? gate : nullptr;
    if (!aligned(x, es) || !aligned(r, es) || !aligned(s, es) || (same && !aligned(y, es)) || !aligned(w, ws) ||
        !aligned(wp, ws) || !aligned(gate, column ? ws : es))
        return fail(K1_ERR_INVALID_ARGUMENT, "%s: a pointer is not aligned to its element size", fn);
    int dev = 0, sms = 0;
    rc = current_device(&dev);
    if (!rc) rc = sm_count(dev, &sms);
    if (rc) return rc;
    int align = rows_align(x, x_stride, n, es, 16);
    align = rows_align(r, r_stride, n, es, align);
    align = rows_align(s, hidden, n, es, align);
    align = gate_align(gate, gate_kind, gate_stride, n, es, align);
    if (same) align = rows_align(y, hidden, n, es, align);
    int e = std::min(norm_piece(hidden, es, align), weights_piece(es, {w, wp, column}));
    if (!same && !aligned(y, e)) e = 1;
    const NormShape sh = norm_shape((int)hidden, es, e);
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
    p.wp = wp;
    p.gate = gate;
    p.gate_stride = gate_kind >= GATE_TOKEN ? gate_stride : 0;
    p.gate_kind = gate_kind;
    p.branch_scale = branch_scale;
    p.residual_scale = residual_scale;
    p.rstd_post = rstd_post;
    // as many blocks as reside at once (or rows): a row costs the same everywhere, so a second round
    // of blocks would leave SMs idle
    auto go = [&](auto tag) {
        using T = decltype(tag);
        constexpr int V = k1::DT<T>::kEPV;
        const int inputs = gate_kind == GATE_FULL ? 3 : 2;
        const bool lng = hidden / V > k1::norm::kRingFwd<V, 2>;  // two such groups have more threads
        const k1::norm::Ring q = ring_of(sh.e, n, hidden, es, inputs, k1::norm::kRingFwd<V, 1>,
                                         lng ? k1::norm::kRingFwd<V, 2, true> : k1::norm::kRingFwd<V, 2>, sms);
        if (q.groups > 0)
            return with_ring(q, [&](auto NV) {
                auto kern = same ? k1::norm::k1_sandwich_ring_kernel<T, NV, k1::norm::SAME, false>
                                 : k1::norm::k1_sandwich_ring_kernel<T, NV, k1::norm::FP8, false>;
                if constexpr (NV == 2)
                    if (lng)
                        kern = same ? k1::norm::k1_sandwich_ring_kernel<T, NV, k1::norm::SAME, true>
                                    : k1::norm::k1_sandwich_ring_kernel<T, NV, k1::norm::FP8, true>;
                const int threads = q.groups * q.threads;
                const size_t smem = ring_smem(q);
                int per_sm = 0;
                if (allow_smem(kern, dev, smem) != K1_OK || resident_blocks(kern, dev, threads, smem, &per_sm) != K1_OK)
                    return cudaErrorInvalidValue;
                const int64_t grid = std::min<int64_t>((n + q.groups - 1) / q.groups, (int64_t)sms * per_sm);
                return launch(kern, grid, threads, smem, st, p, q);
            });
        return with_shape<T>(sh, [&](auto E, auto NV) {
            auto kern = same ? k1::norm::k1_rmsnorm_kernel<T, E, NV, k1::norm::SAME, true>
                             : k1::norm::k1_rmsnorm_kernel<T, E, NV, k1::norm::FP8, true>;
            int per_sm = 0;
            if (resident_blocks(kern, dev, sh.threads, 0, &per_sm) != K1_OK) return cudaErrorInvalidValue;
            return launch(kern, std::min<int64_t>(n, (int64_t)sms * per_sm), sh.threads, 0, st, p);
        });
    };
    return launched(fn, dtype == K1_DTYPE_BF16  ? go(__nv_bfloat16{})
                        : dtype == K1_DTYPE_F16 ? go(__half{})
                                                : go(float{}));
}

}  // namespace

extern "C" {

int k1_sandwich_rmsnorm(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride,
                        const void* post_weight, const void* gate, int gate_kind, int64_t gate_stride,
                        const void* weight, int weight_dtype, int dtype, int64_t n_rows, int64_t hidden,
                        float branch_scale, float residual_scale, float eps, void* stream_out, void* y,
                        float* rstd_post, float* rstd, void* stream) {
    return sandwich_forward("k1_sandwich_rmsnorm", k1::norm::SAME, x, x_stride, residual, residual_stride, post_weight,
                            gate, gate_kind, gate_stride, weight, weight_dtype, dtype, n_rows, hidden, branch_scale,
                            residual_scale, eps, stream_out, y, nullptr, rstd_post, rstd,
                            reinterpret_cast<cudaStream_t>(stream));
}

int k1_sandwich_rmsnorm_fp8(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride,
                            const void* post_weight, const void* gate, int gate_kind, int64_t gate_stride,
                            const void* weight, int weight_dtype, int dtype, int64_t n_rows, int64_t hidden,
                            float branch_scale, float residual_scale, float eps, void* stream_out, void* q,
                            float* scales, void* stream) {
    return sandwich_forward("k1_sandwich_rmsnorm_fp8", k1::norm::FP8, x, x_stride, residual, residual_stride,
                            post_weight, gate, gate_kind, gate_stride, weight, weight_dtype, dtype, n_rows, hidden,
                            branch_scale, residual_scale, eps, stream_out, q, scales, nullptr, nullptr,
                            reinterpret_cast<cudaStream_t>(stream));
}

size_t k1_sandwich_rmsnorm_workspace_bytes(int64_t n_rows, int64_t hidden, int device) {
    int sms = 0;
    if (n_rows < 0 || hidden < 1 || hidden > k1::norm::kMaxHidden || device < 0 || device >= kMaxDevices ||
        sm_count(device, &sms) != K1_OK)
        return 0;
    return (size_t)std::min<int64_t>(std::max<int64_t>(n_rows, 1), (int64_t)sms * kBwdBlocksPerSm) * (size_t)hidden *
           2 * sizeof(float);
}

int k1_sandwich_rmsnorm_backward(const void* g_y, int64_t g_y_stride, const void* g_stream, int64_t g_stream_stride,
                                 const void* stream_in, int64_t stream_stride, const void* x, int64_t x_stride,
                                 const void* post_weight, const void* gate, int gate_kind, int64_t gate_stride,
                                 const void* weight, int weight_dtype, int dtype, const float* rstd_post,
                                 const float* rstd, int64_t n_rows, int64_t hidden, float branch_scale,
                                 float residual_scale, void* d_x, void* d_residual, void* d_post_weight, void* d_gate,
                                 void* d_weight, void* workspace, size_t workspace_bytes, void* stream) {
    static const char* fn = "k1_sandwich_rmsnorm_backward";
    int rc = sandwich_check(fn, dtype, weight_dtype, n_rows, hidden, gate_kind, branch_scale, residual_scale);
    if (rc) return rc;
    const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const int es = elem_size(dtype), ws = elem_size(weight_dtype);
    if (gate_kind == GATE_NONE) d_gate = nullptr;
    void* d_column = gate_kind == GATE_COLUMN ? d_gate : nullptr;
    if (n_rows == 0) {
        for (void* d : {d_post_weight, d_column, d_weight}) {
            if (!d) continue;
            cudaError_t e = cudaMemsetAsync(d, 0, (size_t)hidden * ws, st);
            if (e != cudaSuccess) return fail(K1_ERR_CUDA, "%s: %s", fn, cudaGetErrorString(e));
        }
        return K1_OK;
    }
    if (!stream_in || !x || !rstd_post || !rstd || !post_weight || !weight || (gate_kind != GATE_NONE && !gate))
        return fail(K1_ERR_INVALID_ARGUMENT, "%s: NULL pointer argument", fn);
    if (!d_x && !d_residual && !d_post_weight && !d_gate && !d_weight) return K1_OK;
    if (n_rows > 1 && ((g_y && g_y_stride < 0) || (g_stream && g_stream_stride < 0) || stream_stride < 0 ||
                       x_stride < 0 || (gate_kind >= GATE_TOKEN && gate_stride < 0)))
        return fail(K1_ERR_INVALID_ARGUMENT, "%s: strides must be >= 0", fn);
    const void* column = gate_kind == GATE_COLUMN ? gate : nullptr;
    if (!aligned(g_y, es) || !aligned(g_stream, es) || !aligned(stream_in, es) || !aligned(x, es) ||
        !aligned(d_x, es) || !aligned(d_residual, es) || !aligned(weight, ws) || !aligned(post_weight, ws) ||
        !aligned(d_weight, ws) || !aligned(d_post_weight, ws) || !aligned(gate, column ? ws : es) ||
        !aligned(d_gate, column ? ws : es))
        return fail(K1_ERR_INVALID_ARGUMENT, "%s: a pointer is not aligned to its element size", fn);
    int dev = 0, sms = 0;
    rc = current_device(&dev);
    if (!rc) rc = sm_count(dev, &sms);
    if (rc) return rc;
    int align = rows_align(g_y, g_y_stride, n_rows, es, 16);
    align = rows_align(g_stream, g_stream_stride, n_rows, es, align);
    align = rows_align(stream_in, stream_stride, n_rows, es, align);
    align = rows_align(x, x_stride, n_rows, es, align);
    align = rows_align(d_x, hidden, n_rows, es, align);
    align = rows_align(d_residual, hidden, n_rows, es, align);
    align = gate_align(gate, gate_kind, gate_stride, n_rows, es, align);
    align = gate_align(d_gate, gate_kind, hidden, n_rows, es, align);
    const NormShape sh = norm_shape((int)hidden, es, std::min(norm_piece(hidden, es, align),
                                                              weights_piece(es, {weight, post_weight, column})));
    const int want = (d_weight ? 1 : 0) | (d_post_weight ? 2 : 0) | (d_column ? 4 : 0);
    if (want && (!workspace || !aligned(workspace, 16) ||
                 workspace_bytes < k1_sandwich_rmsnorm_workspace_bytes(n_rows, hidden, dev)))
        return fail(K1_ERR_WORKSPACE, "%s: the weights' gradients need %zu bytes of 16-byte aligned workspace", fn,
                    k1_sandwich_rmsnorm_workspace_bytes(n_rows, hidden, dev));
    k1::norm::SandwichBwdParams p = {};
    p.gy = g_y;
    p.gs = g_stream;
    p.s = stream_in;
    p.x = x;
    p.gate = gate;
    p.wp = post_weight;
    p.w = weight;
    p.rstd_post = rstd_post;
    p.rstd = rstd;
    p.dx = d_x;
    p.dr = d_residual;
    p.dgate = d_column ? nullptr : d_gate;
    p.sums = want ? reinterpret_cast<float*>(workspace) : nullptr;
    p.want = want;
    p.n = n_rows;
    p.gy_stride = g_y_stride;
    p.gs_stride = g_stream_stride;
    p.s_stride = stream_stride;
    p.x_stride = x_stride;
    p.gate_stride = gate_kind >= GATE_TOKEN ? gate_stride : 0;
    p.h = (int)hidden;
    p.w32 = weight_dtype == K1_DTYPE_F32;
    p.gate_kind = gate_kind;
    p.branch_scale = branch_scale;
    p.residual_scale = residual_scale;
    const size_t smem = (size_t)hidden * 8;
    int64_t grid = 0;  // resident blocks, as in the forward
    auto go = [&](auto tag) {
        using T = decltype(tag);
        constexpr int V = k1::DT<T>::kEPV;
        const int inputs = 2 + (g_y != nullptr) + (g_stream != nullptr) + (gate_kind == GATE_FULL);
        const k1::norm::Ring q = ring_of(sh.e, n_rows, hidden, es, inputs, k1::norm::kRingBwd<V, 1>,
                                         k1::norm::kRingBwd<V, 2>, sms);
        if (q.groups > 0)
            return with_ring(q, [&](auto NV) {
                const bool plain = g_y && g_stream && d_x && d_residual && gate_kind != GATE_FULL;
                auto kern = plain ? k1::norm::k1_sandwich_bwd_ring_kernel<T, NV, true>
                                  : k1::norm::k1_sandwich_bwd_ring_kernel<T, NV, false>;
                const int threads = q.groups * q.threads;
                const size_t ring = ring_smem(q);
                int per_sm = 0;
                if (allow_smem(kern, dev, ring) != K1_OK || resident_blocks(kern, dev, threads, ring, &per_sm) != K1_OK)
                    return cudaErrorInvalidValue;
                grid = std::min<int64_t>((n_rows + q.groups - 1) / q.groups,
                                         (int64_t)sms * std::min(per_sm, kBwdBlocksPerSm));
                return launch(kern, grid, threads, ring, st, p, q);
            });
        return with_shape<T>(sh, [&](auto E, auto NV) {
            auto kern = k1::norm::k1_sandwich_bwd_kernel<T, E, NV>;
            int per_sm = 0;
            if (allow_smem(kern, dev, smem) != K1_OK ||
                resident_blocks(kern, dev, sh.threads, smem, &per_sm) != K1_OK)
                return cudaErrorInvalidValue;
            grid = std::min<int64_t>(n_rows, (int64_t)sms * std::min(per_sm, kBwdBlocksPerSm));
            return launch(kern, grid, sh.threads, smem, st, p);
        });
    };
    rc = launched(fn, dtype == K1_DTYPE_BF16  ? go(__nv_bfloat16{})
                      : dtype == K1_DTYPE_F16 ? go(__half{})
                                              : go(float{}));
    if (rc || !want) return rc;
    auto sum = [&](auto tag) {
        using W = decltype(tag);
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)((hidden + 31) / 32), want & 6 ? 2 : 1);
        cfg.blockDim = dim3(1024);
        cfg.stream = st;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = K1_PDL ? 1 : 0;
        return cudaLaunchKernelEx(&cfg, k1::norm::k1_sandwich_dw_kernel<W>, (const float*)p.sums, (int)grid, (int)hidden,
                                  reinterpret_cast<W*>(d_weight), reinterpret_cast<W*>(d_post_weight),
                                  reinterpret_cast<W*>(d_column), reinterpret_cast<const W*>(post_weight),
                                  reinterpret_cast<const W*>(column));
    };
    return launched(fn, weight_dtype == K1_DTYPE_BF16  ? sum(__nv_bfloat16{})
                        : weight_dtype == K1_DTYPE_F16 ? sum(__half{})
                                                       : sum(float{}));
}

}  // extern "C"
