// k1_score_capi.cu -- extern "C" entry points of the log-probabilities of given tokens and of the
// most likely ones (declared in include/k1_logprob.h): argument validation, work split, launches.
#include <algorithm>
#include <cmath>

#include "k1_host.cuh"
#include "k1_score.cuh"

namespace {

// The factor of the logits, or 0.  The bounds keep masked values (at most -1e38) at probability 0.
float score_scale(double temperature) {
    return temperature >= 1e-30 && temperature <= 1e30 ? (float)(1.0 / temperature) : 0.f;
}

int score_check(const char* fn, const void* logits, int dtype, int64_t n_rows, int64_t vocab, int64_t inner_rows,
                int64_t inner_stride, int64_t outer_stride, double temperature, int64_t n_ids, int64_t k) {
    if (!known_dtype(dtype))
        return fail(K1_ERR_UNSUPPORTED_DTYPE, "%s: logits dtype must be bf16, fp16, or fp32", fn);
    if (n_rows < 0 || n_rows > (int64_t)1 << 27)
        return fail(K1_ERR_INVALID_ARGUMENT, "%s: n_rows must be in [0, 2^27], got %lld", fn, (long long)n_rows);
    if (vocab < 1 || vocab >= (int64_t)1 << 30)
        return fail(K1_ERR_INVALID_ARGUMENT, "%s: vocab must be in [1, 2^30), got %lld", fn, (long long)vocab);
    if (inner_rows < 1 || n_rows % inner_rows != 0)
        return fail(K1_ERR_INVALID_ARGUMENT, "%s: inner_rows (%lld) must be >= 1 and divide n_rows (%lld)", fn,
                    (long long)inner_rows, (long long)n_rows);
    if (inner_stride < 0 || outer_stride < 0)
        return fail(K1_ERR_INVALID_ARGUMENT, "%s: strides must be >= 0", fn);
    if (!(score_scale(temperature) > 0.f))
        return fail(K1_ERR_INVALID_ARGUMENT, "%s: temperature must be in [1e-30, 1e30], got %g", fn, temperature);
    if (n_ids < 0 || n_ids > k1::score::kMaxIds)
        return fail(K1_ERR_INVALID_ARGUMENT, "%s: the tokens per row must be at most %d, got %lld", fn,
                    k1::score::kMaxIds, (long long)n_ids);
    if (k < 0 || k > k1::score::kMaxTop || k > vocab)
        return fail(K1_ERR_INVALID_ARGUMENT, "%s: k must be at most %d and the vocabulary (%lld), got %lld", fn,
                    k1::score::kMaxTop, (long long)vocab, (long long)k);
    if (n_rows > 0 && logits == nullptr) return fail(K1_ERR_INVALID_ARGUMENT, "%s: logits is NULL", fn);
    if (!aligned(logits, elem_size(dtype)))
        return fail(K1_ERR_INVALID_ARGUMENT, "%s: logits not aligned to its element size", fn);
    return K1_OK;
}

template <typename T, int TH, int U, int MINB, bool TOP>
int score_launch(const char* fn, k1::score::FwdParams p, int64_t n_rows, int sms, int dev, cudaStream_t st) {
    using namespace k1::score;
    constexpr int E = k1::DT<T>::kEPV;
    constexpr int chunk = U * TH;
    const int64_t vecs = (p.vocab + E - 1) / E + 1;  // one more where a row starts inside a vector
    int cluster = 1;
    while (cluster < kMaxCluster && n_rows * cluster < 2 * sms && vecs >= 2 * cluster * chunk) cluster *= 2;
    p.cluster = cluster;
    p.slice = (int)((vecs + cluster - 1) / cluster);
    const int chunks = (p.slice + chunk - 1) / chunk;
    p.group_chunks = (chunks + kMaxGroups - 1) / kMaxGroups;
    p.groups = (chunks + p.group_chunks - 1) / p.group_chunks;
    auto kern = k1_score_kernel<T, TH, U, MINB, TOP>;
    const size_t smem = fwd_smem<TH, TOP>(cluster, p.groups);
    int rc = allow_smem(kern, dev, smem);
    if (rc) return rc;
    return launched(fn, launch_cluster(kern, dim3((unsigned)(n_rows * cluster)), TH, smem, cluster, st, p));
}

// Threads of a row's block (the same with and without a list, so that both give the same bits).
int score_threads(int64_t n_rows, int sms) { return n_rows >= 6 * sms ? 128 : 256; }

template <typename T>
int score_forward(const char* fn, const k1::score::FwdParams& p, int64_t n_rows, int sms, int dev, cudaStream_t st) {
    if (score_threads(n_rows, sms) == 128)
        return p.k > 0 ? score_launch<T, 128, 4, 7, true>(fn, p, n_rows, sms, dev, st)
                       : score_launch<T, 128, 4, 7, false>(fn, p, n_rows, sms, dev, st);
    return p.k > 0 ? score_launch<T, 256, 4, 4, true>(fn, p, n_rows, sms, dev, st)
                   : score_launch<T, 256, 4, 4, false>(fn, p, n_rows, sms, dev, st);
}

template <typename T>
int score_backward(const char* fn, k1::score::BwdParams p, int64_t n_rows, int sms, int dev, cudaStream_t st) {
    using namespace k1::score;
    constexpr int E = k1::DT<T>::kEPV;
    constexpr int chunk = UB * kBwdThreads;
    const int64_t vecs = (p.vocab + E - 1) / E + 1;
    int64_t parts = 1;
    while (n_rows * parts < 2 * sms && vecs >= 2 * parts * chunk) parts *= 2;
    p.parts = (int)parts;
    p.slice = (int)((vecs + parts - 1) / parts);
    const size_t smem = (size_t)(p.n_ids + p.k) * 12;
    return launched(fn, launch(k1_score_bwd_kernel<T>, n_rows * parts, kBwdThreads, smem, st, p));
}

}  // namespace

extern "C" {

#ifdef K1_WAIT_TEST
// Not part of the product: the threads of a row's block, for tests that mean one kernel of them.
int k1_test_score_threads(int64_t n_rows, int sms) { return score_threads(n_rows, sms); }
#endif

int k1_token_logprobs(const void* logits, int dtype, int64_t n_rows, int64_t vocab, int64_t inner_rows,
                      int64_t inner_stride, int64_t outer_stride, double temperature, const int64_t* token_ids,
                      int64_t n_ids, float* logprobs, int64_t k, int64_t* top_ids, float* top_logprobs,
                      float* entropy, float* lse, float* lse_rest, void* stream) {
    const char* fn = "k1_token_logprobs";
    int rc = score_check(fn, logits, dtype, n_rows, vocab, inner_rows, inner_stride, outer_stride, temperature, n_ids, k);
    if (rc) return rc;
    if (n_rows == 0) return K1_OK;
    if (!entropy || !lse || (n_ids > 0 && (!token_ids || !logprobs)) || (k > 0 && (!top_ids || !top_logprobs)))
        return fail(K1_ERR_INVALID_ARGUMENT, "%s: NULL token or output pointer", fn);
    int dev = 0, sms = 0;
    rc = current_device(&dev);
    if (!rc) rc = sm_count(dev, &sms);
    if (rc) return rc;
    k1::score::FwdParams p = {};
    p.logits = logits;
    p.lay = k1::RowLayout{inner_rows, inner_stride, outer_stride};
    p.vocab = vocab;
    p.scale = score_scale(temperature);
    p.ids = token_ids;
    p.n_ids = (int)n_ids;
    p.logprobs = logprobs;
    p.k = (int)k;
    p.top_ids = top_ids;
    p.top_logprobs = top_logprobs;
    p.entropy = entropy;
    p.lse = lse;
    p.lse_rest = lse_rest;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    switch (dtype) {
        case K1_DTYPE_BF16: return score_forward<__nv_bfloat16>(fn, p, n_rows, sms, dev, st);
        case K1_DTYPE_F16: return score_forward<__half>(fn, p, n_rows, sms, dev, st);
        default: return score_forward<float>(fn, p, n_rows, sms, dev, st);
    }
}

int k1_token_logprobs_backward(const void* logits, int dtype, int64_t n_rows, int64_t vocab, int64_t inner_rows,
                               int64_t inner_stride, int64_t outer_stride, double temperature,
                               const int64_t* token_ids, int64_t n_ids, const float* g_logprobs,
                               const int64_t* top_ids, int64_t k, const float* g_top, const float* lse,
                               const float* lse_rest, const float* entropy, const float* g_entropy,
                               const float* g_lse, void* d_logits, int64_t d_stride, void* stream) {
    const char* fn = "k1_token_logprobs_backward";
    int rc = score_check(fn, logits, dtype, n_rows, vocab, inner_rows, inner_stride, outer_stride, temperature, n_ids, k);
    if (rc) return rc;
    if (d_stride < vocab && n_rows > 1) return fail(K1_ERR_INVALID_ARGUMENT, "%s: d_stride must be >= vocab", fn);
    if (n_rows == 0) return K1_OK;
    if (!lse || !entropy || !d_logits || (g_logprobs && n_ids > 0 && !token_ids) || (g_top && k > 0 && !top_ids))
        return fail(K1_ERR_INVALID_ARGUMENT, "%s: NULL token, saved or output pointer", fn);
    if (!aligned(d_logits, elem_size(dtype)))
        return fail(K1_ERR_INVALID_ARGUMENT, "%s: d_logits not aligned to its element size", fn);
    if (d_logits == logits) return fail(K1_ERR_INVALID_ARGUMENT, "%s: d_logits must not be logits", fn);
    int dev = 0, sms = 0;
    rc = current_device(&dev);
    if (!rc) rc = sm_count(dev, &sms);
    if (rc) return rc;
    k1::score::BwdParams p = {};
    p.logits = logits;
    p.lay = k1::RowLayout{inner_rows, inner_stride, outer_stride};
    p.vocab = vocab;
    p.scale = score_scale(temperature);
    p.ids = token_ids;
    p.g_ids = g_logprobs;
    p.n_ids = g_logprobs ? (int)n_ids : 0;
    p.top_ids = top_ids;
    p.g_top = g_top;
    p.k = g_top ? (int)k : 0;
    p.lse = lse;
    p.lse_rest = lse_rest;
    p.entropy = entropy;
    p.g_entropy = g_entropy;
    p.g_lse = g_lse;
    p.d = d_logits;
    p.d_stride = d_stride;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    switch (dtype) {
        case K1_DTYPE_BF16: return score_backward<__nv_bfloat16>(fn, p, n_rows, sms, dev, st);
        case K1_DTYPE_F16: return score_backward<__half>(fn, p, n_rows, sms, dev, st);
        default: return score_backward<float>(fn, p, n_rows, sms, dev, st);
    }
}

}  // extern "C"
