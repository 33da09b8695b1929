// k1_norm.cuh -- residual addition + root-mean-square norm, with its gradient, and with an
// output in 8 bits (e4m3, one fp32 scale per row and 128 columns).
//
//   s = T(x + r)                         the residual stream, as stored (T: the tensors' type)
//   R = 1 / sqrt(mean(s^2) + eps)        one per row, fp32
//   y = T(s R w)                         or, in 8 bits, q = e4m3(y / a), a = max |y| / 448
//   ds = R (t - s R c) + gs,  t = gy w,  c = mean(t s R);      dx = dr = T(ds)
//   dw = sum over rows of gy s R
//
// The norm reads the stream as it is stored, so the forward, the backward (which keeps only
// s and R) and the next layer all see the same numbers.  Sums, R and dw are fp32; y (and ds)
// is rounded once.  The 8-bit output is rounded once too, from fp32: in bf16 (values and weight)
// from the exact quotient, since R cancels in y / a and s w has 16 bits; in fp16 and fp32 the product
// is rounded to 24 bits first, so a value that lies that close to a midpoint may land one step off.
//
// One block of threads owns a row at a time and keeps it in registers between the sum of
// squares and the output, so every tensor crosses HBM once: 4 N H elements forward (x, r, s,
// y), 4 N H backward (gy, gs, s, ds).  Both are bound by that traffic.  Blocks are
// persistent, as many as 2048 threads per SM make (four per SM at most in the backward).  Registers
// may let fewer reside at a time: with 8-bit output 8192 x 3584 bf16 runs its 8 blocks per SM in two
// rounds of 4.  A thread keeps the same columns for every row, which lets the backward add up its
// columns of dw in registers and write one partial row per block; a second kernel adds the blocks'
// partials in block order (no atomics, so dw does not depend on timing).
//
// Measured on B200: 16384 x 3584 bf16 training step 168 to 174 us (940 MB, 5.4 to 5.6 TB/s), 8192 x
// 3584 bf16 with 8-bit output 43 us, one row 2.8 us of device time; rows of odd width move single
// elements and take 2 to 4 times their bytes' time (4096 x 3585 bf16 forward 55 us, with 8-bit output
// 74; its bytes 18).
#pragma once

#include <type_traits>

#include "k1_common.cuh"

namespace k1 {
namespace norm {

// Threads of a block: rows of vectors need at most 512; rows of smaller pieces get more
// threads rather than more registers.
constexpr int kMaxThreads = 512;
constexpr int kMaxSmall = 1024;
template <int E>
constexpr int kThreads = E >= 4 ? kMaxThreads : kMaxSmall;
constexpr int kMaxHidden = 16384;
constexpr int kFp8Block = 128;       // columns that share a scale
constexpr float kFp8Max = 448.f;     // largest finite e4m3
constexpr float kAmaxFloor = 1e-30f; // a block of zeros gets a finite scale and zeros

// e4m3 (round to nearest even, saturating; NaN stays NaN) of (a, b), a in the low byte.
__device__ __forceinline__ uint32_t e4m3x2(float a, float b) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
    return r;
}

// A thread's piece of a row: E consecutive elements, kept as loaded and converted to fp32
// where they are used: a 16-byte vector, two elements (rows of an even width that no vector
// divides) or one.
template <typename T, int E>
struct Piece;

template <typename T>
struct Piece<T, DT<T>::kEPV> {
    static constexpr int E = DT<T>::kEPV;
    uint4 v;
    // not .nc: the stream may be written over x or the residual
    __device__ __forceinline__ void load(const T* p) { v = ld_stream(p); }
    __device__ __forceinline__ void load_cached(const T* p) { v = __ldg(reinterpret_cast<const uint4*>(p)); }
    __device__ __forceinline__ void store(T* p) const { stg_stream(p, v); }
    __device__ __forceinline__ void zero() { v = make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ void get(float (&f)[E]) const {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(w[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 t = DT<T>::to_f2(w[i]);
                f[2 * i] = t.x;
                f[2 * i + 1] = t.y;
            }
        }
    }
    __device__ __forceinline__ void set(const float (&f)[E]) {
        if constexpr (sizeof(T) == 4) {
            v = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                           __float_as_uint(f[3]));
        } else {
            v = make_uint4(DT<T>::from_f2(make_float2(f[0], f[1])),
                           DT<T>::from_f2(make_float2(f[2], f[3])),
                           DT<T>::from_f2(make_float2(f[4 % E], f[5 % E])),
                           DT<T>::from_f2(make_float2(f[6 % E], f[7 % E])));
        }
    }
};

template <typename T>
struct Piece<T, 2> {
    using V = std::conditional_t<sizeof(T) == 4, float2, uint32_t>;
    V v;
    __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const V*>(p); }
    __device__ __forceinline__ void load_cached(const T* p) { v = *reinterpret_cast<const V*>(p); }
    __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<V*>(p) = v; }
    __device__ __forceinline__ void zero() { v = V{}; }
    __device__ __forceinline__ void get(float (&f)[2]) const {
        float2 t;
        if constexpr (sizeof(T) == 4)
            t = v;
        else
            t = DT<T>::to_f2(v);
        f[0] = t.x;
        f[1] = t.y;
    }
    __device__ __forceinline__ void set(const float (&f)[2]) {
        if constexpr (sizeof(T) == 4)
            v = make_float2(f[0], f[1]);
        else
            v = DT<T>::from_f2(make_float2(f[0], f[1]));
    }
};

template <typename T>
struct Piece<T, 1> {
    T v;
    __device__ __forceinline__ void load(const T* p) { v = *p; }
    __device__ __forceinline__ void load_cached(const T* p) { v = *p; }
    __device__ __forceinline__ void store(T* p) const { *p = v; }
    __device__ __forceinline__ void zero() { DT<T>::store1(&v, 0.f); }
    __device__ __forceinline__ void get(float (&f)[1]) const { f[0] = DT<T>::load1(&v); }
    __device__ __forceinline__ void set(const float (&f)[1]) { DT<T>::store1(&v, f[0]); }
};

// The weight's columns, fp32 or T (w32 is uniform over the launch).  Read through L1: a
// block reads the same columns for every row.
template <typename T, int E>
__device__ __forceinline__ void load_weight(const void* w, bool w32, int col, float (&f)[E]) {
    if (w32) {
        const float* p = reinterpret_cast<const float*>(w) + col;
        if constexpr (E >= 4) {
#pragma unroll
            for (int i = 0; i < E; i += 4) {
                const float4 t = __ldg(reinterpret_cast<const float4*>(p + i));
                f[i] = t.x;
                f[i + 1] = t.y;
                f[i + 2] = t.z;
                f[i + 3] = t.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < E; ++i) f[i] = __ldg(p + i);
        }
    } else {
        Piece<T, E> t;
        t.load_cached(reinterpret_cast<const T*>(w) + col);
        t.get(f);
    }
}

// The 8-bit values of a block whose largest magnitude is m: 448 y / m, as n / step with
// n = 7/8 y and step = m / 512 = 7/8 m / 448.  7/8 y takes three more bits than y and the step
// none, so for products of two bf16 numbers nothing is rounded before the quotient, and a value
// that lies midway between two of e4m3's (1e-4 of them do) is seen as that; y / (m / 448), with
// m / 448 rounded, moves some of them.
//
// The quotient of many values by one step: a product with the reciprocal and one Newton step on
// its residual.  The bare product would move the midway values again, and a division for each
// element costs 7 us of 42 at 8192 x 3584.
struct Quotient {
    float inv, step;
    __device__ __forceinline__ explicit Quotient(float d) : Quotient(d, 1.f / d) {}
    __device__ __forceinline__ Quotient(float d, float one_over_d) {
        inv = one_over_d;
        step = inv == 0.f ? 0.f : d;  // infinite: finite values give 0, not 0 x inf
    }
    __device__ __forceinline__ float operator()(float n) const {
        const float q = n * inv;
        return fmaf(fmaf(-q, step, n), inv, q);
    }
};

// Sum over the block, the same value (and order) in every thread.  scratch: 32 floats, not
// reused before the next __syncthreads of the caller's loop (two alternate buffers).
__device__ __forceinline__ float block_sum(float v, float* scratch) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    const int warps = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    float s = 0.f;
    for (int i = 0; i < warps; ++i) s += scratch[i];
    return s;
}

enum Out : int { SAME = 0, FP8 = 1, FP8_ONLY = 2 };  // FP8_ONLY: no norm, the 8-bit output of x

struct FwdParams {
    const void* x;
    const void* r;  // NULL: no residual (the stream is x; nothing is written to s)
    const void* w;
    void* s;
    void* y;        // T (SAME) or e4m3 (FP8)
    float* scales;  // FP8: [n, ceil(h / 128)]
    float* rstd;    // may be NULL
    int64_t n, x_stride, r_stride;
    int h, w32;
    float eps;
    // POST: the norm after the block, its gate and the scales of both terms
    const void* wp;
    const void* gate;
    int64_t gate_stride;
    int gate_kind;
    float branch_scale, residual_scale;
    float* rstd_post;  // may be NULL
};

// The gate of the branch: none, one per column (the weights' type), one per row, or one per
// element (the tensors' type).
enum Gate : int { GATE_NONE = 0, GATE_COLUMN = 1, GATE_TOKEN = 2, GATE_FULL = 3 };

// The gate's values for a piece; `token` is the row's.
template <typename T, int E>
__device__ __forceinline__ void load_gate(const void* gate, int kind, int64_t row_at, float token, bool w32, int col,
                                          float (&f)[E]) {
    if (kind == GATE_COLUMN) {
        load_weight<T, E>(gate, w32, col, f);
    } else if (kind == GATE_FULL) {
        Piece<T, E> t;
        t.load(reinterpret_cast<const T*>(gate) + row_at + col);
        t.get(f);
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) f[i] = token;
    }
}

// NV pieces per thread: piece j of thread t starts at column (j * threads + t) * E.  Rows of few
// small pieces per thread keep to 32 registers, so that two blocks of 1024 threads share an SM
// (4096 x 3585 bf16, us: forward 62 -> 55, with 8-bit output 93 -> 74).
//
// POST: x goes through a norm of its own first, s = T(residual_scale r + branch_scale gate (x R1 wp)).
template <typename T, int E, int NV, int OUT, bool POST = false>
__global__ void __launch_bounds__(kThreads<E>, E < 4 && E * NV <= 4 ? 2 : 1) k1_rmsnorm_kernel(FwdParams p) {
    using P = Piece<T, E>;
    constexpr bool VEC = E >= 4;
    __shared__ float scratch[POST ? 4 : 2][32];
    __shared__ float wmax[(!VEC && OUT != SAME) ? NV : 1][kMaxSmall / 32];
    pdl_wait();
    pdl_trigger();
    const int threads = blockDim.x, tid = threadIdx.x;
    const int n_blocks = (p.h + kFp8Block - 1) / kFp8Block;
    int flip = 0;
    for (int64_t row = blockIdx.x; row < p.n; row += gridDim.x, flip ^= 1) {
        P s[NV];
        const T* x = reinterpret_cast<const T*>(p.x) + row * p.x_stride;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int col = (j * threads + tid) * E;
            if (col < p.h)
                s[j].load(x + col);
            else
                s[j].zero();
        }
        if (OUT != FP8_ONLY && p.r) {
            const T* r = reinterpret_cast<const T*>(p.r) + row * p.r_stride;
            P q[NV];
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int col = (j * threads + tid) * E;
                if (col < p.h)
                    q[j].load(r + col);
                else
                    q[j].zero();
            }
            float scale = 1.f, token = 1.f;
            int64_t gate_row = 0;
            if constexpr (POST) {
                float sum = 0.f;
#pragma unroll
                for (int j = 0; j < NV; ++j) {
                    float a[E];
                    s[j].get(a);
#pragma unroll
                    for (int i = 0; i < E; ++i) sum = fmaf(a[i], a[i], sum);
                }
                gate_row = row * p.gate_stride;
                if (p.gate_kind == GATE_TOKEN) token = DT<T>::load1(reinterpret_cast<const T*>(p.gate) + gate_row);
                sum = block_sum(sum, scratch[2 + flip]);
                scale = rsqrtf(sum / (float)p.h + p.eps);
                if (p.rstd_post && tid == 0) p.rstd_post[row] = scale;
            }
            T* so = reinterpret_cast<T*>(p.s) + row * p.h;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int col = (j * threads + tid) * E;
                float a[E], b[E];
                s[j].get(a);
                q[j].get(b);
                if constexpr (POST) {
                    if (col < p.h) {
                        float wp[E], gate[E];
                        load_weight<T, E>(p.wp, p.w32, col, wp);
                        load_gate<T, E>(p.gate, p.gate_kind, gate_row, token, p.w32, col, gate);
#pragma unroll
                        for (int i = 0; i < E; ++i) {
                            a[i] = a[i] * scale * wp[i] * (gate[i] * p.branch_scale);
                            b[i] *= p.residual_scale;
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < E; ++i) a[i] += b[i];
                s[j].set(a);
                if (col < p.h) s[j].store(so + col);
            }
        }
        float rstd = 1.f;
        // 8 bits: the quotients' numerators are 7/8 y / 2^k, 2^k <= R < 2^(k + 1), so that no bits
        // are lost to R (it cancels in y / amax) and the range is still y's
        float unit = 0.875f, rest = 1.f, least = kAmaxFloor;
        if constexpr (OUT != FP8_ONLY) {
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                float a[E];
                s[j].get(a);
#pragma unroll
                for (int i = 0; i < E; ++i) sum = fmaf(a[i], a[i], sum);
            }
            sum = block_sum(sum, scratch[flip]);
            rstd = rsqrtf(sum / (float)p.h + p.eps);
            if (p.rstd && tid == 0) p.rstd[row] = rstd;
            if constexpr (OUT == FP8) {
                const uint32_t bits = __float_as_uint(rstd);
                unit *= rstd == rstd ? __uint_as_float(bits & 0x7f800000u) : rstd;
                rest = __uint_as_float((bits & 0x007fffffu) | 0x3f800000u) * (8.f / 7.f);
                least = kAmaxFloor / rest;
            }
        }
        if constexpr (OUT == SAME) {
            T* y = reinterpret_cast<T*>(p.y) + row * p.h;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int col = (j * threads + tid) * E;
                if (col >= p.h) break;
                float a[E], w[E];
                s[j].get(a);
                load_weight<T, E>(p.w, p.w32, col, w);
#pragma unroll
                for (int i = 0; i < E; ++i) a[i] = a[i] * rstd * w[i];
                P o;
                o.set(a);
                o.store(y + col);
            }
        } else {
            // 128 columns are 128 / E consecutive threads' pieces: 16 lanes (16-bit types),
            // a warp (fp32), or two or four warps (pairs, single elements)
            uint8_t* y = reinterpret_cast<uint8_t*>(p.y) + row * (int64_t)p.h;
            float a[NV][E];
            auto step_of = [&](float& m) {  // m: the largest numerator (FP8) or value
                m = fmax_nan(m, least);
                return OUT == FP8 ? m / kFp8Max : m * (1.f / 512.f);
            };
            if constexpr (!VEC) __syncthreads();  // wmax of the previous row has been read
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int col = (j * threads + tid) * E;
                s[j].get(a[j]);
                float m = 0.f;
                if (col < p.h) {
                    if constexpr (OUT == FP8) {
                        float w[E];
                        load_weight<T, E>(p.w, p.w32, col, w);
#pragma unroll
                        for (int i = 0; i < E; ++i) a[j][i] = a[j][i] * unit * w[i];
                    }
#pragma unroll
                    for (int i = 0; i < E; ++i) m = fmax_nan(m, fabsf(a[j][i]));
                    if constexpr (OUT == FP8_ONLY) {
#pragma unroll
                        for (int i = 0; i < E; ++i) a[j][i] *= unit;
                    }
                }
                constexpr int LANES = kFp8Block / E < 32 ? kFp8Block / E : 32;
#pragma unroll
                for (int o = LANES / 2; o > 0; o >>= 1)
                    m = fmax_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
                if constexpr (VEC) {
                    if (col < p.h) {
                        const float step = step_of(m);
                        const Quotient to(step);
                        auto quo = [&](int i) { return to(a[j][i]); };
                        uint32_t q[(E + 3) / 4];
#pragma unroll
                        for (int i = 0; i < E; i += 4)
                            q[i / 4] = e4m3x2(quo(i), quo(i + 1)) | (e4m3x2(quo(i + 2), quo(i + 3)) << 16);
                        if constexpr (E == 8)
                            *reinterpret_cast<uint2*>(y + col) = make_uint2(q[0], q[(E + 3) / 4 - 1]);
                        else
                            *reinterpret_cast<uint32_t*>(y + col) = q[0];
                        if ((tid & (LANES - 1)) == 0)
                            p.scales[row * n_blocks + col / kFp8Block] = OUT == FP8 ? step * rest : m / kFp8Max;
                    }
                } else {
                    if ((tid & 31) == 0) wmax[j][tid >> 5] = m;
                }
            }
            if constexpr (!VEC) {
                // a thread for each scale: its step and the step's reciprocal go where its
                // warps' maxima were
                constexpr int W = kFp8Block / E / 32;  // warps that share a scale
                const int per = threads * E / kFp8Block;
                __syncthreads();
                if (tid < NV * per && tid < n_blocks) {
                    float* g = &wmax[tid / per][tid % per * W];
                    float m = g[0];
#pragma unroll
                    for (int i = 1; i < W; ++i) m = fmax_nan(m, g[i]);
                    const float step = step_of(m);
                    g[0] = step;
                    g[1] = 1.f / step;
                    p.scales[row * n_blocks + tid] = OUT == FP8 ? step * rest : m / kFp8Max;
                }
                __syncthreads();
#pragma unroll
                for (int j = 0; j < NV; ++j) {
                    const int col = (j * threads + tid) * E;
                    if (col >= p.h) break;
                    const float* g = wmax[j] + ((tid >> 5) & ~(W - 1));
                    const Quotient to(g[0], g[1]);
                    const uint32_t q = e4m3x2(to(a[j][0]), to(a[j][E - 1]));
                    if constexpr (E == 2)
                        *reinterpret_cast<uint16_t*>(y + col) = (uint16_t)q;
                    else
                        y[col] = (uint8_t)q;
                }
            }
        }
    }
}

struct BwdParams {
    const void* gy;
    const void* gs;  // NULL: no gradient of the stream
    const void* s;
    const float* rstd;
    const void* w;
    void* ds;      // NULL: not wanted
    float* dw;     // partials [gridDim.x, h]; NULL: not wanted
    int64_t n, gy_stride, gs_stride, s_stride;
    int h, w32;
};

template <typename T, int E, int NV>
__global__ void __launch_bounds__(kThreads<E>) k1_rmsnorm_bwd_kernel(BwdParams p) {
    using P = Piece<T, E>;
    __shared__ float scratch[2][32];
    pdl_wait();
    pdl_trigger();
    const int threads = blockDim.x, tid = threadIdx.x;
    float dw[NV][E];
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < E; ++i) dw[j][i] = 0.f;
    int flip = 0;
    for (int64_t row = blockIdx.x; row < p.n; row += gridDim.x, flip ^= 1) {
        const T* gy = reinterpret_cast<const T*>(p.gy) + row * p.gy_stride;
        const T* sp = reinterpret_cast<const T*>(p.s) + row * p.s_stride;
        const T* gs = p.gs ? reinterpret_cast<const T*>(p.gs) + row * p.gs_stride : nullptr;
        P g[NV], s[NV], u[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int col = (j * threads + tid) * E;
            if (col < p.h) {
                g[j].load(gy + col);
                s[j].load(sp + col);
                if (gs)
                    u[j].load(gs + col);
                else
                    u[j].zero();
            } else {
                g[j].zero();
                s[j].zero();
                u[j].zero();
            }
        }
        const float rstd = p.rstd[row];
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int col = (j * threads + tid) * E;
            if (col >= p.h) break;
            float a[E], b[E], w[E];
            g[j].get(a);
            s[j].get(b);
            load_weight<T, E>(p.w, p.w32, col, w);
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const float n = b[i] * rstd;
                sum = fmaf(a[i] * w[i], n, sum);
                dw[j][i] = fmaf(a[i], n, dw[j][i]);
            }
        }
        if (p.ds) {
            const float c = block_sum(sum, scratch[flip]) / (float)p.h;
            T* ds = reinterpret_cast<T*>(p.ds) + row * p.h;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int col = (j * threads + tid) * E;
                if (col >= p.h) break;
                float a[E], b[E], t[E], w[E];
                g[j].get(a);
                s[j].get(b);
                u[j].get(t);
                load_weight<T, E>(p.w, p.w32, col, w);
#pragma unroll
                for (int i = 0; i < E; ++i)
                    t[i] = fmaf(rstd, fmaf(-(b[i] * rstd), c, a[i] * w[i]), t[i]);
                P o;
                o.set(t);
                o.store(ds + col);
            }
        }
    }
    if (p.dw) {
        float* out = p.dw + (int64_t)blockIdx.x * p.h;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int col = (j * threads + tid) * E;
            if (col >= p.h) break;
#pragma unroll
            for (int i = 0; i < E; ++i) out[col + i] = dw[j][i];
        }
    }
}

// dw[col] = sum over the blocks' partials, in a fixed order: 32 columns per block, the
// partial rows dealt to 16 warps, the warps' sums added in warp order.
template <typename W>
__global__ void __launch_bounds__(512) k1_rmsnorm_dw_kernel(const float* part, int parts, int h, W* dw) {
    __shared__ float sums[16][33];
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int col = blockIdx.x * 32 + lane;
    float v = 0.f;
    if (col < h) {
#pragma unroll 8
        for (int i = warp; i < parts; i += 16) v += part[(int64_t)i * h + col];
    }
    sums[warp][lane] = v;
    __syncthreads();
    if (warp == 0 && col < h) {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) t += sums[i][lane];
        DT<W>::store1(dw + col, t);
    }
}

// ------------------------------------------------------------------------------------
// Weights in 8 bits: one scale per block of 128 x 128 (done once per weight, not in a step)
// ------------------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(256) k1_quantize_blocks_kernel(const T* w, int64_t stride, int64_t rows,
                                                                 int64_t cols, uint8_t* q, float* scales) {
    __shared__ float wmax[8];
    pdl_wait();
    pdl_trigger();
    const int64_t c0 = (int64_t)blockIdx.x * kFp8Block, r0 = (int64_t)blockIdx.y * kFp8Block;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float v[16][4];  // rows warp + 8 i, columns lane + 32 k
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int64_t r = r0 + warp + 8 * i;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int64_t c = c0 + lane + 32 * k;
            v[i][k] = (r < rows && c < cols) ? DT<T>::load1(w + r * stride + c) : 0.f;
            m = fmax_nan(m, fabsf(v[i][k]));
        }
    }
    m = warp_max_nan(m);
    if (lane == 0) wmax[warp] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmax_nan(m, wmax[i]);
    m = fmax_nan(m, kAmaxFloor);
    const Quotient to(m * (1.f / 512.f));
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int64_t r = r0 + warp + 8 * i;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int64_t c = c0 + lane + 32 * k;
            if (r < rows && c < cols) q[r * cols + c] = (uint8_t)e4m3x2(to(0.875f * v[i][k]), 0.f);
        }
    }
    if (threadIdx.x == 0) scales[(int64_t)blockIdx.y * gridDim.x + blockIdx.x] = m / kFp8Max;
}

}  // namespace norm
}  // namespace k1
