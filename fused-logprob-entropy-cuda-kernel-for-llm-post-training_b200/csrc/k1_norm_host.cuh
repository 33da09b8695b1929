// k1_norm_host.cuh -- host-side work split and checks shared by the norms' entry points.
#pragma once

#include <algorithm>

#include "k1_host.cuh"
#include "k1_norm.cuh"

namespace {

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

}  // namespace
