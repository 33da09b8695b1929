// k1_torch_binding.cpp -- the `kernel_opt._C` torch extension.
//
// Mirrors the reference binding (csrc/bindings.cpp:3-26): the same three functions with
// the same out-parameter signatures and the same TORCH_CHECK messages as the reference
// host dispatch (csrc/fused_logprob.cu:284-458), so `RuntimeError`s read the same.  The
// work itself goes through the C ABI of libk1_b200.so (include/k1_logprob.h); this file
// only turns tensors into pointers, strides and the current CUDA stream.
//
// Deliberate relaxations of the reference's checks:
//  * logits need unit stride on the vocab axis only; leading dims must collapse to at
//    most two stride levels (e.g. logits[:, :-1, :] of a [B, L, V] tensor);
//  * backward upstream gradients may be None (treated as zero);
//  * d_logits may have any layout of the same kind (and may alias logits).
#include <torch/extension.h>

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <algorithm>
#include <atomic>
#include <cstdlib>
#include <map>
#include <mutex>
#include <utility>
#include <vector>

#include "k1_logprob.h"

namespace {

struct Rows {
    int64_t n_rows = 0, vocab = 0, inner_rows = 1, inner_stride = 0, outer_stride = 0;
};

// Collapse the leading dims of x[..., V] (stride(-1) == 1) into the two-level layout of
// the C ABI.  Returns false when the leading dims need more than two stride levels.
bool rows_of(const at::Tensor& x, Rows& L) {
    const int64_t nd = x.dim();
    L.vocab = x.size(nd - 1);
    std::vector<std::pair<int64_t, int64_t>> dims;  // (size, stride) with size > 1
    int64_t n = 1;
    for (int64_t d = 0; d < nd - 1; ++d) {
        n *= x.size(d);
        if (x.size(d) != 1) dims.emplace_back(x.size(d), x.stride(d));
    }
    L.n_rows = n;
    // merge dims that are contiguous with respect to each other
    std::vector<std::pair<int64_t, int64_t>> m;
    for (auto& d : dims) {
        if (!m.empty() && m.back().second == d.first * d.second) {
            m.back().first *= d.first;
            m.back().second = d.second;
        } else {
            m.push_back(d);
        }
    }
    if (m.empty()) {
        L.inner_rows = 1;
        L.inner_stride = L.vocab;
        L.outer_stride = L.vocab;
        return true;
    }
    if (m.size() == 1) {
        L.inner_rows = m[0].first;
        L.inner_stride = m[0].second;
        L.outer_stride = m[0].first * m[0].second;
        return true;
    }
    if (m.size() == 2) {
        L.inner_rows = m[1].first;
        L.inner_stride = m[1].second;
        L.outer_stride = m[0].second;
        return true;
    }
    return false;
}

int dtype_code(const at::Tensor& x) {
    if (x.scalar_type() == at::kBFloat16) return K1_DTYPE_BF16;
    if (x.scalar_type() == at::kHalf) return K1_DTYPE_F16;
    if (x.scalar_type() == at::kFloat) return K1_DTYPE_F32;
    return -1;
}

void check_rc(int rc) {
    TORCH_CHECK(rc == K1_OK, k1_last_error());
}

// Opt-in check of the kernels' bounded waits (K1_CHECK_WAITS=1 in the environment, or
// _C.set_check_waits(True)).  A wait inside a kernel that runs out sets a device word and
// leaves NaN in the outputs it could not finish; with the check on, every compute call
// then synchronises its stream, reads and clears that word and raises.  Off by default
// (it synchronises); skipped while the current stream is being captured into a graph.
std::atomic<bool>& check_waits_flag() {
    static std::atomic<bool> flag{[] {
        const char* e = std::getenv("K1_CHECK_WAITS");
        return e != nullptr && e[0] != '\0' && e[0] != '0';
    }()};
    return flag;
}

void check_launch(int rc) {
    check_rc(rc);
    if (!check_waits_flag().load(std::memory_order_relaxed)) return;
    cudaStream_t s = at::cuda::getCurrentCUDAStream().stream();
    cudaStreamCaptureStatus cs = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(s, &cs) != cudaSuccess || cs != cudaStreamCaptureStatusNone) return;
    const cudaError_t e = cudaStreamSynchronize(s);
    TORCH_CHECK(e == cudaSuccess, "k1: ", cudaGetErrorString(e));
    unsigned v = 0;
    check_rc(k1_ring_status(&v));
    TORCH_CHECK(v == 0, "k1: a bounded wait inside a K1 kernel ran out (status ", v,
                "); the outputs it could not finish hold NaN");
}

Rows logits_rows(const at::Tensor& logits) {
    TORCH_CHECK(logits.dim() >= 1, "logits must have a vocab dimension");
    TORCH_CHECK(logits.size(-1) == 0 || logits.stride(-1) == 1 || logits.size(-1) == 1,
                "logits must be contiguous along the vocab dimension");
    Rows L;
    TORCH_CHECK(rows_of(logits, L),
                "logits must be contiguous, or a view whose leading dims collapse to two "
                "strided levels with unit vocab stride");
    return L;
}

// Persistent zero-initialised forward workspace, one per (device, stream); the kernels
// leave it zeroed after every call.  Never freed (kept alive until process exit).
void* forward_workspace(const at::Tensor& like, size_t* bytes) {
    static std::mutex mu;
    static auto* cache = new std::map<std::pair<int, cudaStream_t>, at::Tensor>();
    const int dev = like.get_device();
    cudaStream_t s = at::cuda::getCurrentCUDAStream(dev).stream();
    const size_t need = k1_forward_workspace_bytes(0, 0, 0, dev);
    TORCH_CHECK(need > 0, "k1: could not size the forward workspace: ", k1_last_error());
    std::lock_guard<std::mutex> lock(mu);
    auto key = std::make_pair(dev, s);
    auto it = cache->find(key);
    if (it == cache->end() || (size_t)it->second.numel() < need) {
        at::Tensor ws = at::zeros({(int64_t)need}, like.options().dtype(at::kByte));
        it = cache->insert_or_assign(key, ws).first;
    }
    *bytes = (size_t)it->second.numel();
    return it->second.data_ptr();
}

void check_fwd_common(const at::Tensor& logits, const at::Tensor& targets,
                      const at::Tensor& logprob, const at::Tensor& entropy,
                      const at::Tensor& lse_out, int64_t n_rows) {
    TORCH_CHECK(logits.is_cuda(), "logits must be CUDA");
    TORCH_CHECK(targets.is_cuda(), "targets must be CUDA");
    TORCH_CHECK(targets.scalar_type() == at::kLong, "targets must be int64");
    TORCH_CHECK(targets.is_contiguous(), "targets must be contiguous");
    TORCH_CHECK(logprob.scalar_type() == at::kFloat && entropy.scalar_type() == at::kFloat &&
                    lse_out.scalar_type() == at::kFloat,
                "outputs must be float32");
    TORCH_CHECK(logprob.is_contiguous() && entropy.is_contiguous() && lse_out.is_contiguous(),
                "outputs must be contiguous");
    TORCH_CHECK(logprob.is_cuda() && entropy.is_cuda() && lse_out.is_cuda(),
                "outputs must be CUDA");
    TORCH_CHECK(targets.get_device() == logits.get_device() &&
                    logprob.get_device() == logits.get_device() &&
                    entropy.get_device() == logits.get_device() &&
                    lse_out.get_device() == logits.get_device(),
                "all tensors must be on the same device");
    TORCH_CHECK(targets.numel() == n_rows, "targets numel must match leading dims of logits");
    TORCH_CHECK(logprob.numel() == n_rows && entropy.numel() == n_rows && lse_out.numel() == n_rows,
                "output tensor numels must equal leading-dim count");
}

// _C.fused_logprob_entropy_v1 (reference csrc/fused_logprob.cu:355-403)
void fused_logprob_entropy_v1(at::Tensor logits, at::Tensor targets, at::Tensor logprob,
                              at::Tensor entropy, at::Tensor lse_out) {
    const int dt = dtype_code(logits);
    TORCH_CHECK(dt >= 0, "logits dtype must be bf16, fp16, or fp32");
    Rows L = logits_rows(logits);
    check_fwd_common(logits, targets, logprob, entropy, lse_out, L.n_rows);
    if (L.n_rows == 0) return;
    c10::cuda::CUDAGuard guard(logits.device());
    size_t ws_bytes = 0;
    void* ws = forward_workspace(logits, &ws_bytes);
    check_launch(k1_fused_logprob_entropy_v1(
        logits.data_ptr(), dt, L.n_rows, L.vocab, L.inner_rows, L.inner_stride, L.outer_stride,
        targets.data_ptr<int64_t>(), logprob.data_ptr<float>(), entropy.data_ptr<float>(),
        lse_out.data_ptr<float>(), ws, ws_bytes, at::cuda::getCurrentCUDAStream().stream()));
}

// _C.fused_logprob_entropy_scaled: the forward on logits read as dtype(x * scale) (the
// GRPO temperature, scale = 1/T in fp32), in place of `logits.div_(T)` + K1 (reference
// python/kernel_opt/trainer.py:101-127).
void fused_logprob_entropy_scaled(at::Tensor logits, at::Tensor targets, at::Tensor logprob,
                                  at::Tensor entropy, at::Tensor lse_out, double scale) {
    const int dt = dtype_code(logits);
    TORCH_CHECK(dt >= 0, "logits dtype must be bf16, fp16, or fp32");
    Rows L = logits_rows(logits);
    check_fwd_common(logits, targets, logprob, entropy, lse_out, L.n_rows);
    if (L.n_rows == 0) return;
    c10::cuda::CUDAGuard guard(logits.device());
    size_t ws_bytes = 0;
    void* ws = forward_workspace(logits, &ws_bytes);
    check_launch(k1_fused_logprob_entropy_scaled(
        logits.data_ptr(), dt, L.n_rows, L.vocab, L.inner_rows, L.inner_stride, L.outer_stride,
        (float)scale, targets.data_ptr<int64_t>(), logprob.data_ptr<float>(),
        entropy.data_ptr<float>(), lse_out.data_ptr<float>(), ws, ws_bytes,
        at::cuda::getCurrentCUDAStream().stream()));
}

// _C.fused_logprob_entropy_naive (reference csrc/fused_logprob.cu:405-458)
void fused_logprob_entropy_naive(at::Tensor logits, at::Tensor targets, at::Tensor logprob,
                                 at::Tensor entropy, at::Tensor lse_out) {
    const int dt = dtype_code(logits);
    TORCH_CHECK(dt >= 0, "logits dtype must be bf16, fp16, or fp32");
    Rows L = logits_rows(logits);
    check_fwd_common(logits, targets, logprob, entropy, lse_out, L.n_rows);
    if (L.n_rows == 0) return;
    c10::cuda::CUDAGuard guard(logits.device());
    check_launch(k1_fused_logprob_entropy_naive(
        logits.data_ptr(), dt, L.n_rows, L.vocab, L.inner_rows, L.inner_stride, L.outer_stride,
        targets.data_ptr<int64_t>(), logprob.data_ptr<float>(), entropy.data_ptr<float>(),
        lse_out.data_ptr<float>(), at::cuda::getCurrentCUDAStream().stream()));
}

const float* opt_grad(const c10::optional<at::Tensor>& g, int64_t n_rows, const at::Tensor& like) {
    if (!g.has_value() || !g->defined()) return nullptr;
    TORCH_CHECK(g->scalar_type() == at::kFloat, "upstream gradients must be fp32");
    TORCH_CHECK(g->is_contiguous(), "upstream gradients must be contiguous");
    TORCH_CHECK(g->is_cuda() && g->get_device() == like.get_device(),
                "upstream gradients must be on the logits' device");
    TORCH_CHECK(g->numel() == n_rows, "leading-dim count mismatch");
    return g->data_ptr<float>();
}

void backward_common(const char* which, at::Tensor logits, at::Tensor targets, int64_t vocab_offset,
                     at::Tensor lse, at::Tensor entropy, c10::optional<at::Tensor> g_logp,
                     c10::optional<at::Tensor> g_ent, c10::optional<at::Tensor> g_lse,
                     at::Tensor d_logits, double scale = 1.0) {
    TORCH_CHECK(logits.is_cuda(), "logits must be contiguous CUDA");
    TORCH_CHECK(targets.scalar_type() == at::kLong, "targets must be int64");
    TORCH_CHECK(targets.is_contiguous() && targets.is_cuda(), "targets must be contiguous CUDA");
    TORCH_CHECK(lse.scalar_type() == at::kFloat && entropy.scalar_type() == at::kFloat,
                "saved lse / entropy must be fp32");
    TORCH_CHECK(lse.is_contiguous() && entropy.is_contiguous(), "saved lse / entropy must be contiguous");
    const int dt = dtype_code(logits);
    TORCH_CHECK(dt >= 0, "logits dtype must be bf16, fp16, or fp32");
    TORCH_CHECK(d_logits.scalar_type() == logits.scalar_type() && d_logits.sizes() == logits.sizes(),
                "d_logits must match logits dtype/shape");
    TORCH_CHECK(d_logits.is_cuda() && d_logits.get_device() == logits.get_device(),
                "d_logits must be on the logits' device");
    Rows L = logits_rows(logits);
    TORCH_CHECK(targets.numel() == L.n_rows && lse.numel() == L.n_rows && entropy.numel() == L.n_rows,
                "leading-dim count mismatch");
    const float* gl = opt_grad(g_logp, L.n_rows, logits);
    const float* ge = opt_grad(g_ent, L.n_rows, logits);
    const float* gs = opt_grad(g_lse, L.n_rows, logits);
    if (L.n_rows == 0) return;
    // logits and d_logits share one row grouping (inner_rows): try the grouping of each
    // tensor, view both as [n_rows / k, k, V] (no copy) and read their row strides.
    TORCH_CHECK(d_logits.size(-1) == 1 || d_logits.stride(-1) == 1,
                "d_logits must be contiguous along the vocab dimension");
    Rows D = logits_rows(d_logits);
    bool found = false;
    for (int64_t k : {L.inner_rows, D.inner_rows}) {
        if (k < 1 || L.n_rows % k != 0) continue;
        try {
            at::Tensor lv = logits.view({L.n_rows / k, k, L.vocab});
            at::Tensor dv = d_logits.view({L.n_rows / k, k, L.vocab});
            L.inner_rows = D.inner_rows = k;
            L.inner_stride = lv.stride(1);
            L.outer_stride = lv.stride(0);
            D.inner_stride = dv.stride(1);
            D.outer_stride = dv.stride(0);
            found = true;
            break;
        } catch (const c10::Error&) {
        }
    }
    TORCH_CHECK(found, "d_logits layout cannot be addressed with the logits' row grouping");
    c10::cuda::CUDAGuard guard(logits.device());
    cudaStream_t s = at::cuda::getCurrentCUDAStream().stream();
    int rc;
    if (which[0] == 'v' && scale != 1.0) {
        rc = k1_vocab_shard_scaled_backward(
            logits.data_ptr(), dt, L.n_rows, L.vocab, L.inner_rows, L.inner_stride, L.outer_stride,
            vocab_offset, (float)scale, targets.data_ptr<int64_t>(), lse.data_ptr<float>(),
            entropy.data_ptr<float>(), gl, ge, gs, d_logits.data_ptr(), D.inner_stride,
            D.outer_stride, s);
    } else if (which[0] == 'v') {
        rc = k1_vocab_shard_backward(logits.data_ptr(), dt, L.n_rows, L.vocab, L.inner_rows,
                                     L.inner_stride, L.outer_stride, vocab_offset,
                                     targets.data_ptr<int64_t>(), lse.data_ptr<float>(),
                                     entropy.data_ptr<float>(), gl, ge, gs, d_logits.data_ptr(),
                                     D.inner_stride, D.outer_stride, s);
    } else if (which[0] == 's') {
        rc = k1_fused_logprob_entropy_scaled_backward(
            logits.data_ptr(), dt, L.n_rows, L.vocab, L.inner_rows, L.inner_stride, L.outer_stride,
            (float)scale, targets.data_ptr<int64_t>(), lse.data_ptr<float>(),
            entropy.data_ptr<float>(), gl, ge, gs, d_logits.data_ptr(), D.inner_stride,
            D.outer_stride, s);
    } else {
        rc = k1_fused_logprob_entropy_v1_backward(
            logits.data_ptr(), dt, L.n_rows, L.vocab, L.inner_rows, L.inner_stride, L.outer_stride,
            targets.data_ptr<int64_t>(), lse.data_ptr<float>(), entropy.data_ptr<float>(), gl, ge,
            gs, d_logits.data_ptr(), D.inner_stride, D.outer_stride, s);
    }
    check_launch(rc);
}

// _C.fused_logprob_entropy_v1_backward (reference csrc/fused_logprob.cu:284-346)
void fused_logprob_entropy_v1_backward(at::Tensor logits, at::Tensor targets, at::Tensor lse,
                                       at::Tensor entropy, c10::optional<at::Tensor> g_logp,
                                       c10::optional<at::Tensor> g_ent,
                                       c10::optional<at::Tensor> g_lse, at::Tensor d_logits) {
    backward_common("b", logits, targets, 0, lse, entropy, g_logp, g_ent, g_lse, d_logits);
}

// _C.fused_logprob_entropy_scaled_backward: gradient w.r.t. the unscaled logits x,
// dtype(dtype(dL/dy) * scale) with y = dtype(x * scale).
void fused_logprob_entropy_scaled_backward(at::Tensor logits, at::Tensor targets, at::Tensor lse,
                                           at::Tensor entropy, c10::optional<at::Tensor> g_logp,
                                           c10::optional<at::Tensor> g_ent,
                                           c10::optional<at::Tensor> g_lse, at::Tensor d_logits,
                                           double scale) {
    backward_common("s", logits, targets, 0, lse, entropy, g_logp, g_ent, g_lse, d_logits, scale);
}

// Vocab-parallel step 1: partials [n_rows, 4] float64 (one k1_partial per row).
void vocab_shard_partials(at::Tensor logits, at::Tensor targets, int64_t vocab_offset,
                          at::Tensor partials) {
    const int dt = dtype_code(logits);
    TORCH_CHECK(dt >= 0, "logits dtype must be bf16, fp16, or fp32");
    TORCH_CHECK(logits.is_cuda() && targets.is_cuda() && partials.is_cuda(),
                "logits, targets and partials must be CUDA");
    TORCH_CHECK(targets.scalar_type() == at::kLong && targets.is_contiguous(),
                "targets must be contiguous int64");
    Rows L = logits_rows(logits);
    TORCH_CHECK(targets.numel() == L.n_rows, "targets numel must match leading dims of logits");
    TORCH_CHECK(partials.scalar_type() == at::kDouble && partials.is_contiguous() &&
                    partials.numel() == 4 * L.n_rows,
                "partials must be a contiguous float64 tensor of n_rows x 4");
    if (L.n_rows == 0) return;
    c10::cuda::CUDAGuard guard(logits.device());
    size_t ws_bytes = 0;
    void* ws = forward_workspace(logits, &ws_bytes);
    check_launch(k1_vocab_shard_partials(logits.data_ptr(), dt, L.n_rows, L.vocab, L.inner_rows,
                                     L.inner_stride, L.outer_stride, vocab_offset,
                                     targets.data_ptr<int64_t>(),
                                     reinterpret_cast<k1_partial*>(partials.data_ptr()), ws,
                                     ws_bytes, at::cuda::getCurrentCUDAStream().stream()));
}

// Vocab-parallel step 3: gathered [n_shards, n_rows, 4] float64 -> outputs.
void vocab_combine(at::Tensor gathered, int64_t n_shards, at::Tensor logprob, at::Tensor entropy,
                   at::Tensor lse_out) {
    TORCH_CHECK(gathered.is_cuda() && gathered.scalar_type() == at::kDouble &&
                    gathered.is_contiguous(),
                "gathered partials must be a contiguous CUDA float64 tensor");
    TORCH_CHECK(n_shards >= 1, "n_shards must be >= 1");
    const int64_t n_rows = logprob.numel();
    TORCH_CHECK(gathered.numel() == 4 * n_shards * n_rows,
                "gathered partials must hold n_shards x n_rows x 4 values");
    TORCH_CHECK(logprob.scalar_type() == at::kFloat && entropy.scalar_type() == at::kFloat &&
                    lse_out.scalar_type() == at::kFloat,
                "outputs must be float32");
    TORCH_CHECK(entropy.numel() == n_rows && lse_out.numel() == n_rows,
                "output tensor numels must equal leading-dim count");
    TORCH_CHECK(logprob.is_contiguous() && entropy.is_contiguous() && lse_out.is_contiguous(),
                "outputs must be contiguous");
    if (n_rows == 0) return;
    c10::cuda::CUDAGuard guard(gathered.device());
    check_launch(k1_vocab_combine(reinterpret_cast<const k1_partial*>(gathered.data_ptr()),
                              (int)n_shards, n_rows, logprob.data_ptr<float>(),
                              entropy.data_ptr<float>(), lse_out.data_ptr<float>(),
                              at::cuda::getCurrentCUDAStream().stream()));
}

// Vocab-parallel backward of one shard.
void vocab_shard_backward(at::Tensor logits, at::Tensor targets, int64_t vocab_offset,
                          at::Tensor lse, at::Tensor entropy, c10::optional<at::Tensor> g_logp,
                          c10::optional<at::Tensor> g_ent, c10::optional<at::Tensor> g_lse,
                          at::Tensor d_logits, double scale) {
    // scale != 1: the shard's logits are read as dtype(x * scale) (temperature folded in)
    backward_common("v", logits, targets, vocab_offset, lse, entropy, g_logp, g_ent, g_lse,
                    d_logits, scale);
}

// LM head fused with K1 on the tensor cores (bf16 hidden [N, H] and weight [V, H]).
void check_lm_head(const at::Tensor& hidden, const at::Tensor& weight, const at::Tensor& targets) {
    TORCH_CHECK(hidden.is_cuda() && weight.is_cuda() && targets.is_cuda(),
                "hidden, weight and targets must be CUDA");
    TORCH_CHECK(hidden.scalar_type() == at::kBFloat16 && weight.scalar_type() == at::kBFloat16,
                "the tensor-core LM head takes bf16 hidden and weight");
    TORCH_CHECK(hidden.dim() == 2 && weight.dim() == 2 && hidden.size(1) == weight.size(1),
                "hidden [N, H] and weight [V, H] expected");
    TORCH_CHECK(hidden.is_contiguous() && weight.is_contiguous(), "hidden and weight must be contiguous");
    TORCH_CHECK(targets.scalar_type() == at::kLong && targets.is_contiguous() &&
                    targets.numel() == hidden.size(0),
                "targets must be contiguous int64 with one entry per hidden row");
    TORCH_CHECK(hidden.get_device() == weight.get_device() && hidden.get_device() == targets.get_device(),
                "hidden, weight and targets must be on one device");
}

void lm_head_forward(at::Tensor hidden, at::Tensor weight, at::Tensor targets, at::Tensor logprob,
                     at::Tensor entropy, at::Tensor lse_out, double scale,
                     c10::optional<at::Tensor> logits_out) {
    check_lm_head(hidden, weight, targets);
    const int64_t N = hidden.size(0), H = hidden.size(1), V = weight.size(0);
    for (const at::Tensor* o : {&logprob, &entropy, &lse_out})
        TORCH_CHECK(o->scalar_type() == at::kFloat && o->is_contiguous() && o->numel() == N,
                    "outputs must be contiguous fp32 with one entry per row");
    void* zp = nullptr;
    int64_t zs = V;
    if (logits_out.has_value() && logits_out->defined()) {
        const at::Tensor& z = *logits_out;
        TORCH_CHECK(z.scalar_type() == at::kBFloat16 && z.dim() == 2 && z.size(0) == N &&
                        z.size(1) == V && z.stride(1) == 1,
                    "logits_out must be bf16 [N, V] with unit stride along V");
        zp = z.data_ptr();
        zs = z.stride(0);
    }
    if (N == 0) return;
    c10::cuda::CUDAGuard guard(hidden.device());
    const size_t ws_bytes = k1_lm_head_workspace_bytes(N, H, V, hidden.get_device());
    TORCH_CHECK(ws_bytes > 0, "k1: could not size the LM head workspace: ", k1_last_error());
    at::Tensor ws = at::empty({(int64_t)ws_bytes}, hidden.options().dtype(at::kByte));
    check_launch(k1_lm_head_forward(hidden.data_ptr(), weight.data_ptr(), N, H, V, (float)scale,
                                    targets.data_ptr<int64_t>(), logprob.data_ptr<float>(),
                                    entropy.data_ptr<float>(), lse_out.data_ptr<float>(), zp, zs,
                                    ws.data_ptr(), ws_bytes,
                                    at::cuda::getCurrentCUDAStream().stream()));
}

void lm_head_backward(at::Tensor hidden, at::Tensor weight, at::Tensor targets, at::Tensor lse,
                      at::Tensor entropy, c10::optional<at::Tensor> g_logp,
                      c10::optional<at::Tensor> g_ent, c10::optional<at::Tensor> g_lse,
                      at::Tensor d_logits, double scale) {
    check_lm_head(hidden, weight, targets);
    const int64_t N = hidden.size(0), H = hidden.size(1), V = weight.size(0);
    TORCH_CHECK(lse.scalar_type() == at::kFloat && entropy.scalar_type() == at::kFloat &&
                    lse.is_contiguous() && entropy.is_contiguous() && lse.numel() == N &&
                    entropy.numel() == N,
                "saved lse / entropy must be contiguous fp32 with one entry per row");
    TORCH_CHECK(d_logits.scalar_type() == at::kBFloat16 && d_logits.dim() == 2 &&
                    d_logits.size(0) == N && d_logits.size(1) == V && d_logits.stride(1) == 1,
                "d_logits must be bf16 [N, V] with unit stride along V");
    const float* gl = opt_grad(g_logp, N, hidden);
    const float* ge = opt_grad(g_ent, N, hidden);
    const float* gs = opt_grad(g_lse, N, hidden);
    if (N == 0) return;
    c10::cuda::CUDAGuard guard(hidden.device());
    check_launch(k1_lm_head_backward(hidden.data_ptr(), weight.data_ptr(), N, H, V, (float)scale,
                                     targets.data_ptr<int64_t>(), lse.data_ptr<float>(),
                                     entropy.data_ptr<float>(), gl, ge, gs, d_logits.data_ptr(),
                                     d_logits.stride(0), at::cuda::getCurrentCUDAStream().stream()));
}

// The LM head over a vocabulary shard (rows [vocab_offset, vocab_offset + weight.size(0)) of
// the full weight): per-row k1_partial of the shard, for the all-gather and vocab_combine.
void lm_head_shard_partials(at::Tensor hidden, at::Tensor weight, at::Tensor targets,
                            int64_t vocab_offset, at::Tensor partials, double scale,
                            c10::optional<at::Tensor> logits_out) {
    check_lm_head(hidden, weight, targets);
    const int64_t N = hidden.size(0), H = hidden.size(1), V = weight.size(0);
    TORCH_CHECK(partials.is_cuda() && partials.scalar_type() == at::kDouble &&
                    partials.is_contiguous() && partials.numel() == 4 * N,
                "partials must be a contiguous CUDA float64 tensor of n_rows x 4");
    void* zp = nullptr;
    int64_t zs = V;
    if (logits_out.has_value() && logits_out->defined()) {
        const at::Tensor& z = *logits_out;
        TORCH_CHECK(z.scalar_type() == at::kBFloat16 && z.dim() == 2 && z.size(0) == N &&
                        z.size(1) == V && z.stride(1) == 1,
                    "logits_out must be bf16 [N, V_shard] with unit stride along V");
        zp = z.data_ptr();
        zs = z.stride(0);
    }
    if (N == 0) return;
    c10::cuda::CUDAGuard guard(hidden.device());
    const size_t ws_bytes = k1_lm_head_workspace_bytes(N, H, V, hidden.get_device());
    TORCH_CHECK(ws_bytes > 0, "k1: could not size the LM head workspace: ", k1_last_error());
    at::Tensor ws = at::empty({(int64_t)ws_bytes}, hidden.options().dtype(at::kByte));
    check_launch(k1_lm_head_shard_partials(
        hidden.data_ptr(), weight.data_ptr(), N, H, V, vocab_offset, (float)scale,
        targets.data_ptr<int64_t>(), reinterpret_cast<k1_partial*>(partials.data_ptr()), zp, zs,
        ws.data_ptr(), ws_bytes, at::cuda::getCurrentCUDAStream().stream()));
}

void lm_head_shard_backward(at::Tensor hidden, at::Tensor weight, at::Tensor targets,
                            int64_t vocab_offset, at::Tensor lse, at::Tensor entropy,
                            c10::optional<at::Tensor> g_logp, c10::optional<at::Tensor> g_ent,
                            c10::optional<at::Tensor> g_lse, at::Tensor d_logits, double scale) {
    check_lm_head(hidden, weight, targets);
    const int64_t N = hidden.size(0), H = hidden.size(1), V = weight.size(0);
    TORCH_CHECK(lse.scalar_type() == at::kFloat && entropy.scalar_type() == at::kFloat &&
                    lse.is_contiguous() && entropy.is_contiguous() && lse.numel() == N &&
                    entropy.numel() == N,
                "saved lse / entropy must be contiguous fp32 with one entry per row");
    TORCH_CHECK(d_logits.scalar_type() == at::kBFloat16 && d_logits.dim() == 2 &&
                    d_logits.size(0) == N && d_logits.size(1) == V && d_logits.stride(1) == 1,
                "d_logits must be bf16 [N, V_shard] with unit stride along V");
    const float* gl = opt_grad(g_logp, N, hidden);
    const float* ge = opt_grad(g_ent, N, hidden);
    const float* gs = opt_grad(g_lse, N, hidden);
    if (N == 0) return;
    c10::cuda::CUDAGuard guard(hidden.device());
    check_launch(k1_lm_head_shard_backward(
        hidden.data_ptr(), weight.data_ptr(), N, H, V, vocab_offset, (float)scale,
        targets.data_ptr<int64_t>(), lse.data_ptr<float>(), entropy.data_ptr<float>(), gl, ge, gs,
        d_logits.data_ptr(), d_logits.stride(0), at::cuda::getCurrentCUDAStream().stream()));
}

// ---------------------------------------------------------------------------------------
// The tail of a decoding step: residual RMS norm, 8-bit product, token sampling
// ---------------------------------------------------------------------------------------
// [..., H] as [N, H] with unit stride inside a row; a view where the layout allows it.
at::Tensor rows2d(const at::Tensor& t) {
    TORCH_CHECK_VALUE(t.dim() >= 1, "a tensor with a hidden dimension is expected");
    at::Tensor r = t;
    if (t.dim() != 2) {
        const int64_t H = t.size(-1);
        r = t.reshape({H ? t.numel() / H : 0, H});
    }
    return r.stride(1) == 1 || r.size(1) == 1 ? r : r.contiguous();
}

int float_dtype(const at::Tensor& x, const char* what) {
    TORCH_CHECK_VALUE(x.is_cuda(), what, " must be a CUDA tensor");
    const int dt = dtype_code(x);
    TORCH_CHECK(dt >= 0, what, " dtype must be bf16, fp16, or fp32");
    return dt;
}

int norm_inputs(const at::Tensor& x, const at::Tensor& residual, const at::Tensor& weight, double eps) {
    const int dt = float_dtype(x, "x");
    if (residual.defined())
        TORCH_CHECK_VALUE(residual.sizes() == x.sizes() && residual.scalar_type() == x.scalar_type() &&
                              residual.device() == x.device(),
                          "residual must match x in shape, dtype and device, got ", residual.sizes(), " ",
                          residual.scalar_type(), " for ", x.sizes(), " ", x.scalar_type());
    TORCH_CHECK_VALUE(x.dim() >= 1 && weight.dim() == 1 && weight.size(0) == x.size(-1),
                      "weight must have one value per column of x, got ", weight.sizes(), " for ", x.sizes());
    TORCH_CHECK_VALUE(weight.device() == x.device(), "weight must be on x's device");
    TORCH_CHECK(weight.scalar_type() == x.scalar_type() || weight.scalar_type() == at::kFloat,
                "weight must have x's dtype or fp32");
    TORCH_CHECK_VALUE(eps > 0, "eps must be positive, got ", eps);
    return dt;
}

struct NormOut {
    at::Tensor y, stream, rstd, scales, weight;  // as rows [N, H]; stream is x without a residual
};

// The forward on rows; rstd only for a backward, scales only in 8 bits.
NormOut norm_run(const at::Tensor& x, const at::Tensor& residual, const at::Tensor& weight, double eps, bool fp8,
                 bool want_rstd) {
    const int dt = norm_inputs(x, residual, weight, eps);
    c10::cuda::CUDAGuard guard(x.device());
    const at::Tensor x2 = rows2d(x);
    const at::Tensor r2 = residual.defined() ? rows2d(residual) : at::Tensor();
    NormOut o;
    o.weight = weight.contiguous();
    const int64_t N = x2.size(0), H = x2.size(1);
    o.y = fp8 ? at::empty({N, H}, x.options().dtype(at::kFloat8_e4m3fn)) : at::empty({N, H}, x.options());
    o.stream = r2.defined() ? at::empty({N, H}, x.options()) : x2;
    void* r = r2.defined() ? r2.data_ptr() : nullptr;
    const int64_t rs = r2.defined() ? r2.stride(0) : 0;
    void* so = r2.defined() ? o.stream.data_ptr() : nullptr;
    cudaStream_t st = at::cuda::getCurrentCUDAStream().stream();
    if (fp8) {
        o.scales = at::empty({N, (H + 127) / 128}, x.options().dtype(at::kFloat));
        check_launch(k1_residual_rmsnorm_fp8(x2.data_ptr(), x2.stride(0), r, rs, o.weight.data_ptr(),
                                             dtype_code(weight), dt, N, H, (float)eps, so, o.y.data_ptr(),
                                             o.scales.data_ptr<float>(), st));
    } else {
        if (want_rstd) o.rstd = at::empty({N}, x.options().dtype(at::kFloat));
        check_launch(k1_residual_rmsnorm(x2.data_ptr(), x2.stride(0), r, rs, o.weight.data_ptr(), dtype_code(weight),
                                         dt, N, H, (float)eps, so, o.y.data_ptr(),
                                         want_rstd ? o.rstd.data_ptr<float>() : nullptr, st));
    }
    return o;
}

at::Tensor shaped(const at::Tensor& t, at::IntArrayRef sizes) { return t.sizes() == sizes ? t : t.view(sizes); }

// The differentiable norm: y alone without a residual, else y and the stream.
struct ResidualRmsnorm : public torch::autograd::Function<ResidualRmsnorm> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x,
                                                  const c10::optional<at::Tensor>& residual_,
                                                  const at::Tensor& weight, double eps) {
        const at::Tensor residual = residual_.has_value() ? *residual_ : at::Tensor();
        NormOut o = norm_run(x, residual, weight, eps, false, true);
        const at::Tensor y = shaped(o.y, x.sizes());
        const at::Tensor stream = residual.defined() ? shaped(o.stream, x.sizes()) : at::Tensor();
        // without a residual the stream is the caller's x: saved as the input it is
        ctx->save_for_backward({residual.defined() ? stream : x, o.rstd, weight});
        ctx->set_materialize_grads(false);
        ctx->saved_data["residual"] = residual.defined();
        if (residual.defined()) return {y, stream};
        return {y};
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                   torch::autograd::variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "the residual RMS norm has no second derivative");
        const auto saved = ctx->get_saved_variables();
        const at::Tensor &stream = saved[0], &rstd = saved[1], &weight = saved[2];
        // counted over the tensors that were given
        const bool has_r = ctx->saved_data["residual"].toBool();
        const bool need_x = ctx->needs_input_grad(0), need_r = has_r && ctx->needs_input_grad(1),
                   need_w = ctx->needs_input_grad(has_r ? 2 : 1);
        const at::Tensor g_y = grads[0];
        const at::Tensor g_s = grads.size() > 1 ? grads[1] : at::Tensor();
        const at::Tensor none;
        if (!g_y.defined())  // only the stream was used: the addition's own gradient
            return {need_x ? g_s : none, need_r ? g_s : none, none, none};
        c10::cuda::CUDAGuard guard(stream.device());
        const at::Tensor s2 = rows2d(stream), gy2 = rows2d(g_y);
        const at::Tensor gs2 = g_s.defined() ? rows2d(g_s) : at::Tensor();
        const at::Tensor w = weight.contiguous();
        const int64_t N = s2.size(0), H = s2.size(1);
        at::Tensor d, dw, ws;
        size_t ws_bytes = 0;
        if (need_x || need_r) d = at::empty({N, H}, stream.options());
        if (need_w) {
            dw = at::empty(weight.sizes(), weight.options());
            ws_bytes = k1_residual_rmsnorm_workspace_bytes(N, H, stream.get_device());
            ws = at::empty({(int64_t)ws_bytes}, stream.options().dtype(at::kByte));
        }
        check_launch(k1_residual_rmsnorm_backward(
            gy2.data_ptr(), gy2.stride(0), gs2.defined() ? gs2.data_ptr() : nullptr,
            gs2.defined() ? gs2.stride(0) : 0, s2.data_ptr(), s2.stride(0), rstd.data_ptr<float>(), w.data_ptr(),
            dtype_code(weight), dtype_code(stream), N, H, d.defined() ? d.data_ptr() : nullptr,
            dw.defined() ? dw.data_ptr() : nullptr, ws.defined() ? ws.data_ptr() : nullptr, ws_bytes,
            at::cuda::getCurrentCUDAStream().stream()));
        if (d.defined()) d = shaped(d, stream.sizes());
        return {need_x ? d : none, need_r ? d : none, dw, none};
    }
};

// (y, stream); differentiable in x, residual and weight.
std::tuple<at::Tensor, at::Tensor> residual_rmsnorm(const at::Tensor& x, const c10::optional<at::Tensor>& residual_,
                                                    const at::Tensor& weight, double eps) {
    const at::Tensor residual = residual_.has_value() ? *residual_ : at::Tensor();
    // a tangent would be lost where the node is not entered
    for (const at::Tensor* t : {&x, &residual, &weight})
        TORCH_CHECK(!t->defined() || !t->_fw_grad(/*level=*/0).defined(),
                    "the residual RMS norm does not support forward AD: it has no jvp");
    if (at::GradMode::is_enabled() &&
        (x.requires_grad() || weight.requires_grad() || (residual.defined() && residual.requires_grad()))) {
        norm_inputs(x, residual, weight, eps);
        auto out = ResidualRmsnorm::apply(x, residual_, weight, eps);
        return {out[0], residual.defined() ? out[1] : x};
    }
    NormOut o = norm_run(x, residual, weight, eps, false, false);
    return {shaped(o.y, x.sizes()), residual.defined() ? shaped(o.stream, x.sizes()) : x};
}

// Sizes of x with the last one replaced.
at::Tensor lead_shaped(const at::Tensor& t, const at::Tensor& x) {
    if (x.dim() == 2) return t;
    std::vector<int64_t> sizes(x.sizes().begin(), x.sizes().end());
    sizes.back() = t.size(1);
    return t.view(sizes);
}

// (q, scales, stream)
std::tuple<at::Tensor, at::Tensor, at::Tensor> residual_rmsnorm_fp8(const at::Tensor& x,
                                                                    const c10::optional<at::Tensor>& residual_,
                                                                    const at::Tensor& weight, double eps) {
    const at::Tensor residual = residual_.has_value() ? *residual_ : at::Tensor();
    NormOut o = norm_run(x, residual, weight, eps, true, false);
    return {lead_shaped(o.y, x), lead_shaped(o.scales, x), residual.defined() ? lead_shaped(o.stream, x) : x};
}

// (q, scales): rows in 8 bits, one scale per row and 128 columns
std::tuple<at::Tensor, at::Tensor> quantize_fp8_rows(const at::Tensor& x) {
    const int dt = float_dtype(x, "x");
    c10::cuda::CUDAGuard guard(x.device());
    const at::Tensor x2 = rows2d(x);
    const int64_t N = x2.size(0), H = x2.size(1);
    at::Tensor q = at::empty({N, H}, x.options().dtype(at::kFloat8_e4m3fn));
    at::Tensor scales = at::empty({N, (H + 127) / 128}, x.options().dtype(at::kFloat));
    check_launch(k1_quantize_fp8_rows(x2.data_ptr(), x2.stride(0), dt, N, H, q.data_ptr(), scales.data_ptr<float>(),
                                      at::cuda::getCurrentCUDAStream().stream()));
    return {lead_shaped(q, x), lead_shaped(scales, x)};
}

// (q, scales): a weight in 8 bits, one scale per block of 128 x 128
std::tuple<at::Tensor, at::Tensor> quantize_fp8_blocks(const at::Tensor& w) {
    const int dt = float_dtype(w, "weight");
    TORCH_CHECK_VALUE(w.dim() == 2, "weight must be [O, H]");
    c10::cuda::CUDAGuard guard(w.device());
    const at::Tensor w2 = rows2d(w);
    const int64_t N = w2.size(0), H = w2.size(1);
    at::Tensor q = at::empty({N, H}, w.options().dtype(at::kFloat8_e4m3fn));
    at::Tensor scales = at::empty({(N + 127) / 128, (H + 127) / 128}, w.options().dtype(at::kFloat));
    check_launch(k1_quantize_fp8_blocks(w2.data_ptr(), w2.stride(0), dt, N, H, q.data_ptr(),
                                        scales.data_ptr<float>(), at::cuda::getCurrentCUDAStream().stream()));
    return {q, scales};
}

// Whether a and b, both [M, N] of one type with unit stride along N, are the same elements.
bool same_rows(const at::Tensor& a, const at::Tensor& b) {
    return a.data_ptr() == b.data_ptr() && (a.size(0) == 1 || a.stride(0) == b.stride(0));
}

// Whether they share memory.  Column blocks of one buffer lie between each other's rows, so the rows' own
// ranges count, not the tensors'; b's rows do not overlap (stride(0) >= N).
bool rows_meet(const at::Tensor& a, const at::Tensor& b) {
    const int64_t M = a.size(0), es = a.element_size(), width = a.size(1) * es;
    const auto start = [](const at::Tensor& t) { return (int64_t)reinterpret_cast<uintptr_t>(t.data_ptr()); };
    const int64_t sa = M > 1 ? a.stride(0) * es : 0, sb = M > 1 ? b.stride(0) * es : width;
    const int64_t a0 = start(a), b0 = start(b);
    if (a0 + (M - 1) * sa + width <= b0 || b0 + (M - 1) * sb + width <= a0) return false;
    for (int64_t i = 0; i < M; ++i) {
        const int64_t at = a0 + i * sa - b0;  // the first row of b that ends behind it
        const int64_t j = at < width ? 0 : (at - width) / sb + 1;
        if (j < M && j * sb < at + width) return true;
    }
    return false;
}

at::Tensor fp8_linear(const at::Tensor& x, const at::Tensor& x_scales, const at::Tensor& weight,
                      const at::Tensor& weight_scales, at::ScalarType out_dtype, const c10::optional<at::Tensor>& out,
                      const c10::optional<at::Tensor>& bias_, const c10::optional<std::string>& activation,
                      const c10::optional<at::Tensor>& residual_) {
    TORCH_CHECK_VALUE(x.is_cuda() && weight.is_cuda(), "x and weight must be CUDA tensors");
    TORCH_CHECK(x.scalar_type() == at::kFloat8_e4m3fn && weight.scalar_type() == at::kFloat8_e4m3fn,
                "x and weight must be float8_e4m3fn");
    TORCH_CHECK(x.dim() >= 1 && weight.dim() == 2 && x.size(-1) == weight.size(1),
                "x [N, H] and weight [O, H] expected");
    TORCH_CHECK_VALUE(x_scales.dim() == x.dim() && x_scales.sizes().slice(0, x.dim() - 1) == x.sizes().slice(0, x.dim() - 1),
                      "x_scales must have x's leading dimensions, got ", x_scales.sizes(), " for ", x.sizes());
    for (const at::Tensor* t : {&x_scales, &weight_scales, &weight})
        TORCH_CHECK(t->device() == x.device(), "all tensors must be on the same device");
    c10::cuda::CUDAGuard guard(x.device());
    const at::Tensor x2 = rows2d(x), w2 = rows2d(weight);
    const int64_t M = x2.size(0), K = x2.size(1), N = w2.size(0), KB = (K + 127) / 128;
    TORCH_CHECK(x_scales.scalar_type() == at::kFloat && x_scales.size(-1) == KB,
                "x_scales must be fp32 [N, ceil(H / 128)]");
    TORCH_CHECK(weight_scales.scalar_type() == at::kFloat && weight_scales.dim() == 2 &&
                    weight_scales.size(0) == (N + 127) / 128 && weight_scales.size(1) == KB,
                "weight_scales must be fp32 [ceil(O / 128), ceil(H / 128)]");
    const at::Tensor xs = x_scales.contiguous(), ws = weight_scales.contiguous();
    at::Tensor y;
    if (out.has_value()) {
        y = *out;
        TORCH_CHECK(y.dim() == 2 && y.size(0) == M && y.size(1) == N && (N <= 1 || y.stride(1) == 1) &&
                        y.device() == x.device(),
                    "the output must be [N, O] on x's device, contiguous along the last dimension");
        TORCH_CHECK(dtype_code(y) >= 0, "the output's dtype must be bf16, fp16, or fp32");
    } else {
        TORCH_CHECK_VALUE(out_dtype == at::kBFloat16 || out_dtype == at::kHalf || out_dtype == at::kFloat,
                          "out_dtype must be bf16, fp16, or fp32, got ", out_dtype);
        y = at::empty({M, N}, x.options().dtype(out_dtype));
    }
    int act = K1_ACT_NONE;
    if (activation.has_value()) {
        static const char* const names[] = {"none", "relu", "silu", "gelu", "gelu_tanh"};
        for (act = K1_ACT_GELU_TANH; act > K1_ACT_NONE && *activation != names[act]; --act) {}
        TORCH_CHECK_VALUE(act != K1_ACT_NONE, "activation must be None, 'relu', 'silu', 'gelu' or 'gelu_tanh', got '",
                          *activation, "'");
    }
    at::Tensor bias, residual;
    if (bias_.has_value()) {
        TORCH_CHECK_VALUE(bias_->dim() == 1 && bias_->size(0) == N && bias_->device() == x.device(),
                          "bias must be [O] on x's device, got ", bias_->sizes());
        TORCH_CHECK(bias_->scalar_type() == y.scalar_type() || bias_->scalar_type() == at::kFloat,
                    "bias must have the output's dtype or fp32");
        bias = bias_->contiguous();
    }
    if (residual_.has_value()) {
        TORCH_CHECK_VALUE(residual_->dim() == x.dim() && residual_->size(-1) == N &&
                              residual_->sizes().slice(0, x.dim() - 1) == x.sizes().slice(0, x.dim() - 1) &&
                              residual_->device() == x.device(),
                          "residual must be shaped like the product, on x's device, got ", residual_->sizes());
        TORCH_CHECK(residual_->scalar_type() == y.scalar_type(), "residual must have the output's dtype");
        residual = rows2d(*residual_);
        // broadcast rows (and what torch lets overlap) are laid out
        if (M > 1 && residual.stride(0) < N) residual = residual.contiguous();
        if (out.has_value() && M > 0 && N > 0)
            TORCH_CHECK_VALUE(same_rows(y, residual) || !rows_meet(y, residual),
                              "residual must be the output itself or lie apart from it");
    }
    check_launch(k1_fp8_linear_epilogue(
        x2.data_ptr(), M > 1 ? x2.stride(0) : K, xs.data_ptr<float>(), w2.data_ptr(), N > 1 ? w2.stride(0) : K,
        ws.data_ptr<float>(), M, K, N, bias.defined() ? bias.data_ptr() : nullptr,
        bias.defined() ? dtype_code(bias) : K1_DTYPE_F32, act, residual.defined() ? residual.data_ptr() : nullptr,
        residual.defined() && M > 1 ? residual.stride(0) : N, y.data_ptr(), M > 1 ? y.stride(0) : N, dtype_code(y),
        at::cuda::getCurrentCUDAStream().stream()));
    return out.has_value() ? y : lead_shaped(y, x);
}

// A sampling setting: a number, or a tensor with one entry per row (kept alive in `rows`).
template <typename V>
const V* setting(const pybind11::object& v, at::ScalarType type, const at::Tensor& u, const char* what, double* number,
                 at::Tensor& rows) {
    if (!THPVariable_Check(v.ptr())) {
        *number = v.cast<double>();
        return nullptr;
    }
    const at::Tensor& t = THPVariable_Unpack(v.ptr());
    TORCH_CHECK_VALUE(t.dim() == 0 || t.sizes() == u.sizes(), what,
                      " must be a number or a tensor shaped like the rows ", u.sizes(), ", got ", t.sizes());
    // 64-bit whole numbers are cut to 32 bits as numbers are, not to their low halves
    const bool wide = type == at::kInt && t.scalar_type() == at::kLong;
    rows = (wide ? t.clamp(0, INT32_MAX) : t).to(u.device(), type).expand(u.sizes()).contiguous();
    return rows.const_data_ptr<V>();
}

// (token, logprob, kept_logprob), each shaped like u
std::tuple<at::Tensor, at::Tensor, at::Tensor> sample_tokens(const at::Tensor& logits, const at::Tensor& u,
                                                             const pybind11::object& temperature,
                                                             const pybind11::object& top_k,
                                                             const pybind11::object& top_p,
                                                             const pybind11::object& min_p) {
    const int dt = float_dtype(logits, "logits");
    TORCH_CHECK_VALUE(logits.dim() >= 1 && u.sizes() == logits.sizes().slice(0, logits.dim() - 1),
                      "u must be shaped like the rows of logits ", logits.sizes(), ", got ", u.sizes());
    TORCH_CHECK_VALUE(u.device() == logits.device(), "u must be on the logits' device");
    c10::cuda::CUDAGuard guard(logits.device());
    const int64_t N = u.numel(), V = logits.size(-1);
    at::Tensor x = logits.dim() == 2 ? logits : logits.reshape({N, V});
    if (x.stride(1) != 1 && V > 1) x = x.contiguous();
    const at::Tensor uu = u.to(at::kFloat).contiguous();
    k1_sampling s = {};
    at::Tensor t_rows, k_rows, p_rows, q_rows;
    double k = 0, p = 1, q = 0;
    s.temperature_rows = setting<float>(temperature, at::kFloat, u, "temperature", &s.temperature, t_rows);
    s.top_k_rows = setting<int>(top_k, at::kInt, u, "top_k", &k, k_rows);
    s.top_p_rows = setting<float>(top_p, at::kFloat, u, "top_p", &p, p_rows);
    s.min_p_rows = setting<float>(min_p, at::kFloat, u, "min_p", &q, q_rows);
    TORCH_CHECK_VALUE(k == k, "top_k must be a whole number, got nan");
    s.top_k = (int)std::min(std::max(k, 0.0), (double)INT32_MAX);
    s.top_p = (float)p;
    s.min_p = (float)q;
    at::Tensor token = at::empty(u.sizes(), logits.options().dtype(at::kLong));
    at::Tensor logprob = at::empty(u.sizes(), logits.options().dtype(at::kFloat));
    at::Tensor kept = at::empty(u.sizes(), logits.options().dtype(at::kFloat));
    check_launch(k1_sample_tokens(x.data_ptr(), dt, N, V, x.stride(0), uu.data_ptr<float>(), &s,
                                  token.data_ptr<int64_t>(), logprob.data_ptr<float>(), kept.data_ptr<float>(),
                                  at::cuda::getCurrentCUDAStream().stream()));
    return {token, logprob, kept};
}

// ---------------------------------------------------------------------------------------
// The norms around a block's end
// ---------------------------------------------------------------------------------------
// The arguments as rows (those of the gate where it has rows) and what kind of gate it is.
struct Sandwich {
    at::Tensor x, residual, post_weight, weight, gate;
    int kind = K1_GATE_NONE;
    int64_t gate_stride = 0;
    int dt = 0;
    const void* gate_ptr() const { return kind == K1_GATE_NONE ? nullptr : gate.data_ptr(); }
};

Sandwich sandwich_inputs(const at::Tensor& x, const at::Tensor& residual, const at::Tensor& post_weight,
                         const at::Tensor& weight, const at::Tensor& gate, double eps) {
    Sandwich a;
    TORCH_CHECK_VALUE(residual.defined(), "a residual is expected");
    a.dt = norm_inputs(x, residual, weight, eps);
    TORCH_CHECK_VALUE(post_weight.sizes() == weight.sizes() && post_weight.scalar_type() == weight.scalar_type() &&
                          post_weight.device() == x.device(),
                      "post_weight must match weight in shape, dtype and device, got ", post_weight.sizes(), " ",
                      post_weight.scalar_type(), " for ", weight.sizes(), " ", weight.scalar_type());
    if (gate.defined()) {
        TORCH_CHECK_VALUE(gate.device() == x.device(), "gate must be on x's device");
        const int64_t H = x.size(-1);
        const bool rows = gate.dim() == x.dim() && gate.sizes().slice(0, x.dim() - 1) == x.sizes().slice(0, x.dim() - 1);
        // a gate [H] beside a single row [H] may be either: its type says which (column where both fit)
        const bool element = x.dim() == 1 && gate.scalar_type() != weight.scalar_type() &&
                             gate.scalar_type() == x.scalar_type();
        if (gate.dim() == 1 && gate.size(0) == H && !element) {
            a.kind = K1_GATE_COLUMN;
            TORCH_CHECK(gate.scalar_type() == weight.scalar_type(), "a gate per column must have the weights' dtype");
        } else {
            TORCH_CHECK_VALUE(rows && (gate.size(-1) == H || gate.size(-1) == 1),
                              "gate must be [H], or shaped like x with H or 1 columns, got ", gate.sizes(), " for ",
                              x.sizes());
            a.kind = gate.size(-1) == H ? K1_GATE_FULL : K1_GATE_TOKEN;
            TORCH_CHECK(gate.scalar_type() == x.scalar_type(), "a gate with rows must have x's dtype");
        }
    }
    return a;
}

// Rows of the arguments; on x's device.
void sandwich_rows(Sandwich& a, const at::Tensor& x, const at::Tensor& residual, const at::Tensor& post_weight,
                   const at::Tensor& weight, const at::Tensor& gate) {
    a.x = rows2d(x);
    if (residual.defined()) a.residual = rows2d(residual);
    a.post_weight = post_weight.contiguous();
    a.weight = weight.contiguous();
    if (a.kind == K1_GATE_COLUMN) {
        a.gate = gate.contiguous();
    } else if (a.kind != K1_GATE_NONE) {
        a.gate = rows2d(gate);
        a.gate_stride = a.gate.stride(0);
    }
}

struct SandwichRmsnorm : public torch::autograd::Function<SandwichRmsnorm> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x,
                                                  const at::Tensor& residual, const at::Tensor& post_weight,
                                                  const at::Tensor& weight, const c10::optional<at::Tensor>& gate_,
                                                  double branch_scale, double residual_scale, double eps, bool want) {
        const at::Tensor gate = gate_.has_value() ? *gate_ : at::Tensor();
        c10::cuda::CUDAGuard guard(x.device());
        Sandwich a = sandwich_inputs(x, residual, post_weight, weight, gate, eps);
        sandwich_rows(a, x, residual, post_weight, weight, gate);
        const int64_t N = a.x.size(0), H = a.x.size(1);
        at::Tensor y = at::empty({N, H}, x.options()), stream = at::empty({N, H}, x.options()), r1, r2;
        if (want) {
            r1 = at::empty({N}, x.options().dtype(at::kFloat));
            r2 = at::empty({N}, x.options().dtype(at::kFloat));
        }
        check_launch(k1_sandwich_rmsnorm(a.x.data_ptr(), a.x.stride(0), a.residual.data_ptr(), a.residual.stride(0),
                                         a.post_weight.data_ptr(), a.gate_ptr(), a.kind, a.gate_stride,
                                         a.weight.data_ptr(), dtype_code(weight), a.dt, N, H, (float)branch_scale,
                                         (float)residual_scale, (float)eps, stream.data_ptr(), y.data_ptr(),
                                         want ? r1.data_ptr<float>() : nullptr, want ? r2.data_ptr<float>() : nullptr,
                                         at::cuda::getCurrentCUDAStream().stream()));
        y = shaped(y, x.sizes());
        stream = shaped(stream, x.sizes());
        if (want) {
            ctx->save_for_backward({stream, x, r1, r2, post_weight, weight, gate});
            ctx->set_materialize_grads(false);
            ctx->saved_data["kind"] = (int64_t)a.kind;
            ctx->saved_data["branch_scale"] = branch_scale;
            ctx->saved_data["residual_scale"] = residual_scale;
        }
        return {y, stream};
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                   torch::autograd::variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "the sandwich RMS norm has no second derivative");
        const at::Tensor none;
        const at::Tensor &g_y = grads[0], &g_s = grads[1];
        torch::autograd::variable_list out(9);
        if (!g_y.defined() && !g_s.defined()) return out;
        const auto saved = ctx->get_saved_variables();
        const at::Tensor &stream = saved[0], &x = saved[1], &r1 = saved[2], &r2 = saved[3], &post_weight = saved[4],
                         &weight = saved[5], &gate = saved[6];
        c10::cuda::CUDAGuard guard(stream.device());
        Sandwich a;
        a.kind = (int)ctx->saved_data["kind"].toInt();
        sandwich_rows(a, x, none, post_weight, weight, gate);
        const at::Tensor s2 = rows2d(stream), gy2 = g_y.defined() ? rows2d(g_y) : none,
                         gs2 = g_s.defined() ? rows2d(g_s) : none;
        const int64_t N = s2.size(0), H = s2.size(1);
        // counted over the tensors that were given
        if (ctx->needs_input_grad(0)) out[0] = at::empty({N, H}, stream.options());
        if (ctx->needs_input_grad(1)) out[1] = at::empty({N, H}, stream.options());
        if (ctx->needs_input_grad(2)) out[2] = at::empty(post_weight.sizes(), post_weight.options());
        if (ctx->needs_input_grad(3)) out[3] = at::empty(weight.sizes(), weight.options());
        if (gate.defined() && ctx->needs_input_grad(4)) out[4] = at::empty(gate.sizes(), gate.options());
        size_t ws_bytes = 0;
        at::Tensor ws;
        if (out[2].defined() || out[3].defined() || (out[4].defined() && a.kind == K1_GATE_COLUMN)) {
            ws_bytes = k1_sandwich_rmsnorm_workspace_bytes(N, H, stream.get_device());
            ws = at::empty({(int64_t)ws_bytes}, stream.options().dtype(at::kByte));
        }
        const auto ptr = [](const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
        const auto step = [](const at::Tensor& t) { return t.defined() ? t.stride(0) : 0; };
        check_launch(k1_sandwich_rmsnorm_backward(
            ptr(gy2), step(gy2), ptr(gs2), step(gs2), s2.data_ptr(), s2.stride(0), a.x.data_ptr(), a.x.stride(0),
            a.post_weight.data_ptr(), a.gate_ptr(), a.kind, a.gate_stride, a.weight.data_ptr(), dtype_code(weight),
            dtype_code(stream), r1.data_ptr<float>(), r2.data_ptr<float>(), N, H,
            (float)ctx->saved_data["branch_scale"].toDouble(), (float)ctx->saved_data["residual_scale"].toDouble(),
            ptr(out[0]), ptr(out[1]), ptr(out[2]), ptr(out[4]), ptr(out[3]), ptr(ws), ws_bytes,
            at::cuda::getCurrentCUDAStream().stream()));
        for (int i : {0, 1})
            if (out[i].defined()) out[i] = shaped(out[i], stream.sizes());
        return out;
    }
};

// (y, stream); differentiable in x, residual, both weights and the gate.
std::tuple<at::Tensor, at::Tensor> sandwich_rmsnorm(const at::Tensor& x, const at::Tensor& residual,
                                                    const at::Tensor& post_weight, const at::Tensor& weight,
                                                    const c10::optional<at::Tensor>& gate_, double branch_scale,
                                                    double residual_scale, double eps) {
    const at::Tensor gate = gate_.has_value() ? *gate_ : at::Tensor();
    sandwich_inputs(x, residual, post_weight, weight, gate, eps);
    bool want = false;
    for (const at::Tensor* t : {&x, &residual, &post_weight, &weight, &gate}) {
        if (!t->defined()) continue;
        TORCH_CHECK(!t->_fw_grad(/*level=*/0).defined(),
                    "the sandwich RMS norm does not support forward AD: it has no jvp");
        want |= t->requires_grad();
    }
    want &= at::GradMode::is_enabled();
    auto out = SandwichRmsnorm::apply(x, residual, post_weight, weight, gate_, branch_scale, residual_scale, eps, want);
    return {out[0], out[1]};
}

// (q, scales, stream)
std::tuple<at::Tensor, at::Tensor, at::Tensor> sandwich_rmsnorm_fp8(const at::Tensor& x, const at::Tensor& residual,
                                                                    const at::Tensor& post_weight,
                                                                    const at::Tensor& weight,
                                                                    const c10::optional<at::Tensor>& gate_,
                                                                    double branch_scale, double residual_scale,
                                                                    double eps) {
    const at::Tensor gate = gate_.has_value() ? *gate_ : at::Tensor();
    Sandwich a = sandwich_inputs(x, residual, post_weight, weight, gate, eps);
    c10::cuda::CUDAGuard guard(x.device());
    sandwich_rows(a, x, residual, post_weight, weight, gate);
    const int64_t N = a.x.size(0), H = a.x.size(1);
    at::Tensor q = at::empty({N, H}, x.options().dtype(at::kFloat8_e4m3fn)), stream = at::empty({N, H}, x.options());
    at::Tensor scales = at::empty({N, (H + 127) / 128}, x.options().dtype(at::kFloat));
    check_launch(k1_sandwich_rmsnorm_fp8(a.x.data_ptr(), a.x.stride(0), a.residual.data_ptr(), a.residual.stride(0),
                                         a.post_weight.data_ptr(), a.gate_ptr(), a.kind, a.gate_stride,
                                         a.weight.data_ptr(), dtype_code(weight), a.dt, N, H, (float)branch_scale,
                                         (float)residual_scale, (float)eps, stream.data_ptr(), q.data_ptr(),
                                         scales.data_ptr<float>(), at::cuda::getCurrentCUDAStream().stream()));
    return {lead_shaped(q, x), lead_shaped(scales, x), lead_shaped(stream, x)};
}

// ---------------------------------------------------------------------------------------
// Log-probabilities of given tokens and of the most likely ones
// ---------------------------------------------------------------------------------------
struct ScoreOut {
    at::Tensor logprobs, entropy, lse, top_ids, top, rest;  // rest: of lse, for a backward
};

// The rows of logits; without any, a grouping that the C ABI takes.
Rows score_rows(const at::Tensor& logits) {
    Rows L = logits_rows(logits);
    if (L.n_rows == 0) L.inner_rows = 1;
    return L;
}

// ids: [..., K] (K = 1 for a target), undefined: none.
ScoreOut score_run(const at::Tensor& logits, const at::Tensor& ids, int64_t k, double temperature, bool want_rest) {
    const Rows L = score_rows(logits);
    c10::cuda::CUDAGuard guard(logits.device());
    const auto lead = logits.sizes().slice(0, logits.dim() - 1);
    const auto f32 = logits.options().dtype(at::kFloat);
    ScoreOut o;
    o.entropy = at::empty(lead, f32);
    o.lse = at::empty(lead, f32);
    if (want_rest) o.rest = at::empty(lead, f32);
    if (k > 0) {
        std::vector<int64_t> wide(lead.begin(), lead.end());
        wide.push_back(k);
        o.top_ids = at::empty(wide, logits.options().dtype(at::kLong));
        o.top = at::empty(wide, f32);
    }
    const int64_t n_ids = ids.defined() ? ids.size(-1) : 0;
    if (ids.defined()) o.logprobs = at::empty(ids.sizes(), f32);
    const auto ptr = [](const at::Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; };
    check_launch(k1_token_logprobs(
        logits.data_ptr(), dtype_code(logits), L.n_rows, L.vocab, L.inner_rows, L.inner_stride, L.outer_stride,
        temperature, ids.defined() ? ids.data_ptr<int64_t>() : nullptr, n_ids, ptr(o.logprobs), k,
        k > 0 ? o.top_ids.data_ptr<int64_t>() : nullptr, ptr(o.top), o.entropy.data_ptr<float>(), o.lse.data_ptr<float>(),
        ptr(o.rest), at::cuda::getCurrentCUDAStream().stream()));
    return o;
}

struct TokenLogprobs : public torch::autograd::Function<TokenLogprobs> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& logits,
                                                  const c10::optional<at::Tensor>& ids_, int64_t k,
                                                  double temperature) {
        const at::Tensor ids = ids_.has_value() ? *ids_ : at::Tensor();
        ScoreOut o = score_run(logits, ids, k, temperature, true);
        ctx->save_for_backward({logits, ids, o.entropy, o.lse, o.top_ids, o.rest});
        ctx->saved_data["temperature"] = temperature;
        ctx->set_materialize_grads(false);
        torch::autograd::variable_list out = {o.entropy, o.lse};
        if (ids.defined()) out.push_back(o.logprobs);
        if (k > 0) {
            ctx->mark_non_differentiable({o.top_ids});
            out.push_back(o.top_ids);
            out.push_back(o.top);
        }
        return out;
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                   torch::autograd::variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "the log-probabilities have no second derivative");
        const auto saved = ctx->get_saved_variables();
        const at::Tensor &logits = saved[0], &ids = saved[1], &entropy = saved[2], &lse = saved[3], &top_ids = saved[4],
                         &rest = saved[5];
        const at::Tensor none;
        const Rows L = score_rows(logits);
        c10::cuda::CUDAGuard guard(logits.device());
        const auto ready = [](const at::Tensor& g) { return g.defined() ? g.to(at::kFloat).contiguous() : g; };
        const at::Tensor g_ent = ready(grads[0]), g_lse = ready(grads[1]), g_ids = ids.defined() ? ready(grads[2]) : none,
                         g_top = top_ids.defined() ? ready(grads.back()) : none;
        if (!g_ent.defined() && !g_lse.defined() && !g_top.defined() && !g_ids.defined()) return {none, none, none, none};
        const auto ptr = [](const at::Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; };
        at::Tensor d = at::empty(logits.sizes(), logits.options());
        check_launch(k1_token_logprobs_backward(
            logits.data_ptr(), dtype_code(logits), L.n_rows, L.vocab, L.inner_rows, L.inner_stride, L.outer_stride,
            ctx->saved_data["temperature"].toDouble(), ids.defined() ? ids.data_ptr<int64_t>() : nullptr,
            ids.defined() ? ids.size(-1) : 0, ptr(g_ids), top_ids.defined() ? top_ids.data_ptr<int64_t>() : nullptr,
            top_ids.defined() ? top_ids.size(-1) : 0, ptr(g_top), lse.data_ptr<float>(), ptr(rest),
            entropy.data_ptr<float>(), ptr(g_ent), ptr(g_lse), d.data_ptr(), L.vocab,
            at::cuda::getCurrentCUDAStream().stream()));
        return {d, none, none, none};
    }
};

ScoreOut score(const at::Tensor& logits, const at::Tensor& ids_, int64_t k, double temperature) {
    TORCH_CHECK(!logits._fw_grad(/*level=*/0).defined(),
                "the log-probabilities do not support forward AD: they have no jvp");
    const at::Tensor ids = ids_.defined() ? ids_.contiguous() : ids_;
    if (!at::GradMode::is_enabled() || !logits.requires_grad()) return score_run(logits, ids, k, temperature, false);
    auto out = TokenLogprobs::apply(logits, ids.defined() ? c10::optional<at::Tensor>(ids) : c10::nullopt, k, temperature);
    const size_t at = ids.defined() ? 3 : 2;
    return {ids.defined() ? out[2] : at::Tensor(), out[0], out[1], k > 0 ? out[at] : at::Tensor(),
            k > 0 ? out[at + 1] : at::Tensor()};
}

void score_tokens(const at::Tensor& ids, const at::Tensor& logits, const char* what) {
    TORCH_CHECK_VALUE(ids.device() == logits.device(), what, " must be on the logits' device");
    TORCH_CHECK(ids.scalar_type() == at::kLong, what, " must be int64");
}

// (logprob or None, entropy, lse, top_ids, top_logprobs)
std::tuple<c10::optional<at::Tensor>, at::Tensor, at::Tensor, at::Tensor, at::Tensor> top_logprobs(
    const at::Tensor& logits, const c10::optional<at::Tensor>& targets, int64_t k, double temperature) {
    float_dtype(logits, "logits");
    TORCH_CHECK_VALUE(logits.dim() >= 1, "logits must have a vocab dimension");
    TORCH_CHECK_VALUE(k >= 1, "k must be at least 1, got ", k);
    at::Tensor ids;
    if (targets.has_value()) {
        TORCH_CHECK_VALUE(targets->sizes() == logits.sizes().slice(0, logits.dim() - 1),
                          "targets must be shaped like the rows of logits ", logits.sizes(), ", got ", targets->sizes());
        score_tokens(*targets, logits, "targets");
        ids = targets->unsqueeze(-1);
    }
    ScoreOut o = score(logits, ids, k, temperature);
    return {ids.defined() ? c10::optional<at::Tensor>(o.logprobs.squeeze(-1)) : c10::nullopt, o.entropy, o.lse, o.top_ids,
            o.top};
}

// (logprobs, entropy, lse)
std::tuple<at::Tensor, at::Tensor, at::Tensor> token_logprobs(const at::Tensor& logits, const at::Tensor& ids,
                                                              double temperature) {
    float_dtype(logits, "logits");
    TORCH_CHECK_VALUE(logits.dim() >= 1 && ids.dim() == logits.dim() &&
                          ids.sizes().slice(0, ids.dim() - 1) == logits.sizes().slice(0, logits.dim() - 1),
                      "token_ids must be [..., K] with the leading dimensions of logits ", logits.sizes(), ", got ",
                      ids.sizes());
    score_tokens(ids, logits, "token_ids");
    ScoreOut o = score(logits, ids, 0, temperature);
    return {o.logprobs, o.entropy, o.lse};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.def("fused_logprob_entropy_naive", &fused_logprob_entropy_naive,
          "Forward, one thread per row in fp64 (correctness anchor).");
    m.def("fused_logprob_entropy_v1", &fused_logprob_entropy_v1,
          "Forward: one streaming pass, split evenly over all SMs.");
    m.def("fused_logprob_entropy_v1_backward", &fused_logprob_entropy_v1_backward,
          "Backward: streaming, recomputes softmax from the saved lse.", pybind11::arg("logits"),
          pybind11::arg("targets"), pybind11::arg("lse"), pybind11::arg("entropy"),
          pybind11::arg("g_logp"), pybind11::arg("g_ent"), pybind11::arg("g_lse"),
          pybind11::arg("d_logits"));
    m.def("fused_logprob_entropy_scaled", &fused_logprob_entropy_scaled,
          "Forward on logits read as dtype(x * scale) (temperature folded in).",
          pybind11::arg("logits"), pybind11::arg("targets"), pybind11::arg("logprob"),
          pybind11::arg("entropy"), pybind11::arg("lse_out"), pybind11::arg("scale"));
    m.def("fused_logprob_entropy_scaled_backward", &fused_logprob_entropy_scaled_backward,
          "Backward of the scaled forward, gradient w.r.t. the unscaled logits.",
          pybind11::arg("logits"), pybind11::arg("targets"), pybind11::arg("lse"),
          pybind11::arg("entropy"), pybind11::arg("g_logp"), pybind11::arg("g_ent"),
          pybind11::arg("g_lse"), pybind11::arg("d_logits"), pybind11::arg("scale"));
    m.def("vocab_shard_partials", &vocab_shard_partials,
          "Vocab-parallel: per-row partial state of a vocabulary shard.");
    m.def("vocab_combine", &vocab_combine, "Vocab-parallel: merge gathered shard partials.");
    m.def("vocab_shard_backward", &vocab_shard_backward,
          "Vocab-parallel: backward of a shard (scale != 1: logits read as dtype(x * scale)).",
          pybind11::arg("logits"), pybind11::arg("targets"), pybind11::arg("vocab_offset"),
          pybind11::arg("lse"), pybind11::arg("entropy"), pybind11::arg("g_logp"),
          pybind11::arg("g_ent"), pybind11::arg("g_lse"), pybind11::arg("d_logits"),
          pybind11::arg("scale") = 1.0);
    m.def("lm_head_forward", &lm_head_forward,
          "LM head fused with K1 on the tensor cores: per-row logprob / entropy / lse of "
          "bf16(hidden weight^T) read as bf16(z * scale); optionally also writes z.",
          pybind11::arg("hidden"), pybind11::arg("weight"), pybind11::arg("targets"),
          pybind11::arg("logprob"), pybind11::arg("entropy"), pybind11::arg("lse_out"),
          pybind11::arg("scale"), pybind11::arg("logits_out") = pybind11::none());
    m.def("lm_head_backward", &lm_head_backward,
          "Recomputes the LM head's logits on the tensor cores and writes K1's gradient "
          "w.r.t. them (the scaled backward's rounding).",
          pybind11::arg("hidden"), pybind11::arg("weight"), pybind11::arg("targets"),
          pybind11::arg("lse"), pybind11::arg("entropy"), pybind11::arg("g_logp"),
          pybind11::arg("g_ent"), pybind11::arg("g_lse"), pybind11::arg("d_logits"),
          pybind11::arg("scale"));
    m.def("lm_head_shard_partials", &lm_head_shard_partials,
          "Vocab-parallel LM head: per-row partial state of this rank's weight shard, from "
          "the tensor-core kernel's epilogue.",
          pybind11::arg("hidden"), pybind11::arg("weight"), pybind11::arg("targets"),
          pybind11::arg("vocab_offset"), pybind11::arg("partials"), pybind11::arg("scale"),
          pybind11::arg("logits_out") = pybind11::none());
    m.def("lm_head_shard_backward", &lm_head_shard_backward,
          "Vocab-parallel LM head: K1's gradient w.r.t. this shard's logits, recomputed on "
          "the tensor cores, from the combined lse / entropy.",
          pybind11::arg("hidden"), pybind11::arg("weight"), pybind11::arg("targets"),
          pybind11::arg("vocab_offset"), pybind11::arg("lse"), pybind11::arg("entropy"),
          pybind11::arg("g_logp"), pybind11::arg("g_ent"), pybind11::arg("g_lse"),
          pybind11::arg("d_logits"), pybind11::arg("scale"));
    m.def("residual_rmsnorm", &residual_rmsnorm,
          "stream = x + residual, y = its RMS norm times the weight: (y, stream), differentiable.",
          pybind11::arg("x"), pybind11::arg("residual"), pybind11::arg("weight"), pybind11::arg("eps"));
    m.def("residual_rmsnorm_fp8", &residual_rmsnorm_fp8,
          "residual_rmsnorm with y in 8 bits, one scale per row and 128 columns: (q, scales, stream).",
          pybind11::arg("x"), pybind11::arg("residual"), pybind11::arg("weight"), pybind11::arg("eps"));
    m.def("quantize_fp8_rows", &quantize_fp8_rows, "Rows in 8 bits: (q, scales [N, ceil(H / 128)]).",
          pybind11::arg("x"));
    m.def("quantize_fp8_blocks", &quantize_fp8_blocks,
          "A weight in 8 bits: (q, scales [ceil(O / 128), ceil(H / 128)]).", pybind11::arg("weight"));
    m.def("fp8_linear", &fp8_linear,
          "y = act(x weight^T + bias) + residual of 8-bit operands with a scale per block of 128.",
          pybind11::arg("x"), pybind11::arg("x_scales"), pybind11::arg("weight"),
          pybind11::arg("weight_scales"), pybind11::arg("out_dtype"), pybind11::arg("out"),
          pybind11::arg("bias") = pybind11::none(), pybind11::arg("activation") = pybind11::none(),
          pybind11::arg("residual") = pybind11::none());
    m.def("sample_tokens", &sample_tokens,
          "One token per row from given uniform numbers: (token, logprob, kept_logprob).",
          pybind11::arg("logits"), pybind11::arg("u"), pybind11::arg("temperature"), pybind11::arg("top_k"),
          pybind11::arg("top_p"), pybind11::arg("min_p"));
    m.def("sandwich_rmsnorm", &sandwich_rmsnorm,
          "stream = residual_scale residual + branch_scale gate norm(x) post_weight, y = its RMS norm times the "
          "weight: (y, stream), differentiable.",
          pybind11::arg("x"), pybind11::arg("residual"), pybind11::arg("post_weight"), pybind11::arg("weight"),
          pybind11::arg("gate"), pybind11::arg("branch_scale"), pybind11::arg("residual_scale"), pybind11::arg("eps"));
    m.def("sandwich_rmsnorm_fp8", &sandwich_rmsnorm_fp8,
          "sandwich_rmsnorm with y in 8 bits, one scale per row and 128 columns: (q, scales, stream).",
          pybind11::arg("x"), pybind11::arg("residual"), pybind11::arg("post_weight"), pybind11::arg("weight"),
          pybind11::arg("gate"), pybind11::arg("branch_scale"), pybind11::arg("residual_scale"), pybind11::arg("eps"));
    m.def("top_logprobs", &top_logprobs,
          "The k most likely tokens with their log-probabilities, the target's, entropy and lse; differentiable.",
          pybind11::arg("logits"), pybind11::arg("targets"), pybind11::arg("k"), pybind11::arg("temperature"));
    m.def("token_logprobs", &token_logprobs,
          "Log-probabilities of K given tokens per row, entropy and lse; differentiable.", pybind11::arg("logits"),
          pybind11::arg("token_ids"), pybind11::arg("temperature"));
    m.def("abi_version", &k1_abi_version, "C ABI version of the loaded libk1_b200.so.");
    m.def(
        "ring_status",
        []() {
            unsigned v = 0;
            check_rc(k1_ring_status(&v));
            return v;
        },
        "Read and clear the bulk-copy ring's timeout word of the current device (0 = ok).");
    m.def(
        "set_check_waits", [](bool on) { check_waits_flag().store(on); },
        "Raise after any K1 call whose kernel's bounded wait ran out (synchronises each call).");
    m.def(
        "check_waits", []() { return check_waits_flag().load(); },
        "Whether K1 calls check the kernels' bounded waits (K1_CHECK_WAITS / set_check_waits).");
}
