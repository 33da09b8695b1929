// k1_sandwich.cuh -- gradient of the norms around a block's end: the norm of the block's output,
// its gate and scales, the residual addition, and the norm in front of the next block.
//
//   R1 = 1 / sqrt(mean(x^2) + eps),  m = x R1,  b = m wp gate
//   s = T(rs r + bs b)                            the residual stream, as stored
//   R2 = 1 / sqrt(mean(s^2) + eps),  n = s R2,  y = T(n w)
//   (the forward is k1_rmsnorm_kernel with POST: k1_norm.cuh)
//
//   ds = R2 (gy w - n c2) + gs,  c2 = mean(gy w n);      dr = T(rs ds),  dw = sum over rows of gy n
//   u = bs ds;  dgate = u m wp (summed over rows, or over the row, where the gate is broadcast)
//   t = u gate wp,  c1 = mean(t m);  dx = T(R1 (t - m c1)),  dwp = sum over rows of u gate m
//
// ds stays in fp32 from the stream's gradient to the branch's.  Layout as in the norm's own backward:
// a block of threads owns a row at a time, a thread the same columns for every row.  Sums over rows
// (up to three per column) are kept in shared memory, where only their thread touches them, and
// written as one partial row per block; a second kernel adds the blocks' partials in block order.
// Bound by traffic: gy, gs, s, x in, dr, dx out (and a gate per element in, its gradient out).
#pragma once

#include "k1_norm.cuh"

namespace k1 {
namespace norm {

struct SandwichBwdParams {
    const void* gy;  // NULL: none
    const void* gs;  // NULL: none
    const void* s;
    const void* x;
    const void* gate;
    const void* wp;
    const void* w;
    const float* rstd_post;
    const float* rstd;
    void* dx;        // outputs that are NULL are not wanted
    void* dr;
    void* dgate;     // per row or per element; per column it is a partial sum
    float* sums;     // [3][gridDim.x][h]: dw, dwp, dgate per column; NULL: none is wanted
    int want;        // bits: 1 dw, 2 dwp, 4 dgate per column
    int64_t n, gy_stride, gs_stride, s_stride, x_stride, gate_stride;
    int h, w32, gate_kind;
    float branch_scale, residual_scale;
};

// Two sums over the block at once (see block_sum).
__device__ __forceinline__ float2 block_sum2(float2 v, float2* scratch) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
        v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
    const int warps = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    float2 s = make_float2(0.f, 0.f);
    for (int i = 0; i < warps; ++i) {
        s.x += scratch[i].x;
        s.y += scratch[i].y;
    }
    return s;
}

// Adds v to E consecutive sums of this thread.
template <int E>
__device__ __forceinline__ void add_to(float* at, const float (&v)[E]) {
    if constexpr (E >= 4) {
#pragma unroll
        for (int i = 0; i < E; i += 4) {
            float4 t = *reinterpret_cast<float4*>(at + i);
            t.x += v[i];
            t.y += v[i + 1];
            t.z += v[i + 2];
            t.w += v[i + 3];
            *reinterpret_cast<float4*>(at + i) = t;
        }
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) at[i] += v[i];
    }
}

template <typename T, int E, int NV>
__global__ void __launch_bounds__(kThreads<E>) k1_sandwich_bwd_kernel(SandwichBwdParams p) {
    using P = Piece<T, E>;
    // the tensors of the second phase are loaded with the first's where registers allow
    constexpr bool EARLY = E * NV <= (E >= 4 ? 16 : 4);
    __shared__ float scratch[2][32];
    __shared__ float2 scratch2[2][32];
    extern __shared__ __align__(16) float sums[];  // [3][h]
    pdl_wait();
    pdl_trigger();
    const int threads = blockDim.x, tid = threadIdx.x, h = p.h;
    for (int i = tid; i < 3 * h; i += threads) sums[i] = 0.f;
    __syncthreads();
    int flip = 0;
    for (int64_t row = blockIdx.x; row < p.n; row += gridDim.x, flip ^= 1) {
        const T* gy = p.gy ? reinterpret_cast<const T*>(p.gy) + row * p.gy_stride : nullptr;
        const T* gs = p.gs ? reinterpret_cast<const T*>(p.gs) + row * p.gs_stride : nullptr;
        const T* sp = reinterpret_cast<const T*>(p.s) + row * p.s_stride;
        const T* xp = reinterpret_cast<const T*>(p.x) + row * p.x_stride;
        P g[NV], s[NV], u[EARLY ? NV : 1], x[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int col = (j * threads + tid) * E;
            g[j].zero();
            s[j].zero();
            if (col < h) {
                if (gy) g[j].load(gy + col);
                s[j].load(sp + col);
            }
        }
        if constexpr (EARLY) {
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int col = (j * threads + tid) * E;
                u[j].zero();
                x[j].zero();
                if (col < h) {
                    if (gs) u[j].load(gs + col);
                    x[j].load(xp + col);
                }
            }
        }
        const float r1 = p.rstd_post[row], r2 = p.rstd[row];
        const int64_t gate_row = row * p.gate_stride;
        const float token =
            p.gate_kind == GATE_TOKEN ? DT<T>::load1(reinterpret_cast<const T*>(p.gate) + gate_row) : 1.f;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int col = (j * threads + tid) * E;
            if (col >= h) break;
            float a[E], b[E], w[E];
            g[j].get(a);
            s[j].get(b);
            load_weight<T, E>(p.w, p.w32, col, w);
#pragma unroll
            for (int i = 0; i < E; ++i) {
                b[i] *= r2;
                sum = fmaf(a[i] * w[i], b[i], sum);
                b[i] *= a[i];
            }
            if (p.want & 1) add_to<E>(sums + col, b);
        }
        const float c2 = block_sum(sum, scratch[flip]) / (float)h;
        float2 dots = make_float2(0.f, 0.f);
        float t[NV][E];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int col = (j * threads + tid) * E;
            if (col >= h) break;
            float a[E], b[E], w[E];
            g[j].get(a);
            s[j].get(b);
            load_weight<T, E>(p.w, p.w32, col, w);
            float e[E];
            {
                P q;
                if constexpr (EARLY) {
                    q = u[j];
                } else {
                    q.zero();
                    if (gs) q.load(gs + col);
                    x[j].load(xp + col);
                }
                q.get(e);
            }
#pragma unroll
            for (int i = 0; i < E; ++i) a[i] = fmaf(r2, fmaf(-(b[i] * r2), c2, a[i] * w[i]), e[i]);
            if (p.dr) {
#pragma unroll
                for (int i = 0; i < E; ++i) b[i] = p.residual_scale * a[i];
                P o;
                o.set(b);
                o.store(reinterpret_cast<T*>(p.dr) + row * h + col);
            }
            float gate[E];
            load_gate<T, E>(p.gate, p.gate_kind, gate_row, token, p.w32, col, gate);
            load_weight<T, E>(p.wp, p.w32, col, w);
            x[j].get(b);
#pragma unroll
            for (int i = 0; i < E; ++i) {
                a[i] *= p.branch_scale;
                b[i] *= r1;
                e[i] = a[i] * b[i] * w[i];          // dgate
                a[i] *= gate[i];
                t[j][i] = a[i] * w[i];
                a[i] *= b[i];                       // dwp
                dots.x = fmaf(t[j][i], b[i], dots.x);
                dots.y += e[i];
            }
            if (p.want & 2) add_to<E>(sums + h + col, a);
            if (p.want & 4) add_to<E>(sums + 2 * h + col, e);
            if (p.dgate && p.gate_kind == GATE_FULL) {
                P o;
                o.set(e);
                o.store(reinterpret_cast<T*>(p.dgate) + row * h + col);
            }
        }
        const bool by_token = p.dgate && p.gate_kind == GATE_TOKEN;
        if (p.dx || by_token) {
            dots = block_sum2(dots, scratch2[flip]);
            if (by_token && tid == 0) DT<T>::store1(reinterpret_cast<T*>(p.dgate) + row, dots.y);
            const float c1 = dots.x / (float)h;
            if (p.dx) {
#pragma unroll
                for (int j = 0; j < NV; ++j) {
                    const int col = (j * threads + tid) * E;
                    if (col >= h) break;
                    float b[E];
                    x[j].get(b);
#pragma unroll
                    for (int i = 0; i < E; ++i) b[i] = r1 * fmaf(-(b[i] * r1), c1, t[j][i]);
                    P o;
                    o.set(b);
                    o.store(reinterpret_cast<T*>(p.dx) + row * h + col);
                }
            }
        }
    }
    if (p.sums) {
        __syncthreads();
        for (int k = 0; k < 3; ++k) {
            if (!(p.want >> k & 1)) continue;
            float* out = p.sums + ((int64_t)k * gridDim.x + blockIdx.x) * h;
            for (int i = tid; i < h; i += threads) out[i] = sums[k * h + i];
        }
    }
}

// The blocks' partial sums of dw, dwp and dgate (blockIdx.y), added in a fixed order as in
// k1_rmsnorm_dw_kernel.
template <typename W>
__global__ void __launch_bounds__(512) k1_sandwich_dw_kernel(const float* part, int parts, int h, W* dw, W* dwp, W* dg) {
    __shared__ float sums[16][33];
    W* out = blockIdx.y == 0 ? dw : blockIdx.y == 1 ? dwp : dg;
    pdl_wait();
    pdl_trigger();
    if (!out) return;
    part += (int64_t)blockIdx.y * parts * h;
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
        DT<W>::store1(out + col, t);
    }
}

}  // namespace norm
}  // namespace k1
