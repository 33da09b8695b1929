// k1_sandwich.cuh -- the norms around a block's end: the norm of the block's output, its gate and
// scales, the residual addition, and the norm in front of the next block; and their gradient.
//
//   R1 = 1 / sqrt(mean(x^2) + eps),  m = x R1,  b = m wp gate
//   s = T(rs r + bs b)                            the residual stream, as stored
//   R2 = 1 / sqrt(mean(s^2) + eps),  n = s R2,  y = T(n w)
//   (k1_sandwich_ring_kernel below for many rows of whole vectors, else k1_rmsnorm_kernel with POST:
//   k1_norm.cuh)
//
//   ds = R2 (gy w - n c2) + gs,  c2 = mean(gy w n);      dr = T(rs ds),  dw = sum over rows of gy n
//   u = bs ds;  dgate = u m wp (summed over rows, or over the row, where the gate is broadcast)
//   t = u gate wp,  c1 = mean(t m);  dx = T(R1 (t - m c1)),  dwp = sum over rows of u gate m
//
// ds stays in fp32 from the stream's gradient to the branch's.  Sums over rows are two per column whatever
// the gate, since dwp and a column gate's gradient are multiples of one.
//
// k1_sandwich_bwd_kernel, for few rows and for widths without whole vectors: layout as in the norm's own
// backward, a block of threads owns a row at a time, a thread the same columns for every row.  The
// sums over rows are kept in shared memory, where only their thread touches them, and written as one partial
// row per block; a second kernel adds the blocks' partials in block order.
// Bound by traffic: gy, gs, s, x in, dr, dx out (and a gate per element in, its gradient out).
#pragma once

#include "k1_norm.cuh"
#include "k1_sync.cuh"

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
    float* sums;     // [2][gridDim.x][h]: dw, and what dwp and a column gate's are multiples of
    int want;        // bits: 1 dw, 2 dwp, 4 dgate per column; 0: sums is NULL
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
    extern __shared__ __align__(16) float sums[];  // [2][h]
    pdl_wait();
    pdl_trigger();
    const int threads = blockDim.x, tid = threadIdx.x, h = p.h;
    for (int i = tid; i < 2 * h; i += threads) sums[i] = 0.f;
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
                t[j][i] = a[i] * gate[i] * w[i];
                a[i] *= p.gate_kind == GATE_COLUMN ? b[i] : gate[i] * b[i];
                dots.x = fmaf(t[j][i], b[i], dots.x);
                dots.y += e[i];
            }
            if (p.want & 6) add_to<E>(sums + h + col, a);
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
        for (int k = 0; k < 2; ++k) {
            if (!(p.want & (k == 0 ? 1 : 6))) continue;
            float* out = p.sums + ((int64_t)k * gridDim.x + blockIdx.x) * h;
            for (int i = tid; i < h; i += threads) out[i] = sums[k * h + i];
        }
    }
}

// ------------------------------------------------------------------------------------
// Rows of vectors, many of them: loads by bulk copies
// ------------------------------------------------------------------------------------
// The kernels above and in k1_norm.cuh load a row, reduce it twice and store it, and nothing is in flight
// meanwhile but other blocks' loads, of which registers allow two or three blocks per SM (75 us
// forward and 128 backward at 8192 x 3584 bf16; the bytes alone take 36 and 55, these kernels 39 and 68,
// and 53 forward with 8-bit output).  Here a block is a few groups of threads, each with rows and a ring
// of stages of its own: a stage holds one row of every input, a bulk copy each, counted on the stage's
// mbarrier.  When a group has read a stage (which the row's second reduction, a barrier of the group,
// tells), one thread orders the group's next row into it.  So 112 to 168 KB per SM are in flight
// whatever the groups wait for (bf16, forward with two inputs and backward with four; 96 forward at 2048, and 60
// and 120 at 256, the shortest rows).  Columns are summed in pairs, so a row's last bits may differ from those
// of the other kernels, which keep the order of the norms without POST (from the stored stream on their
// y is the residual norm's): one by one the sums would cost the packed arithmetic.  Sums over rows stay
// in registers and are added over the groups, in their order, at the end; the weights are in shared
// memory too, as fp32, and not in registers.
//
// Every wait is bounded; one that runs out, be it for one thread of a group alone, sets bit 0 of the wait
// status word.  That thread brings NaN into the sums over the row and over its columns: from there on the
// group's rows are NaN (backward without a gradient of y: dx, a gate's per row, and the columns of the threads
// that saw nothing land).  A block leaves only when the copies that it ordered have landed.
struct Ring {
    int groups, threads;  // groups per block, threads per group
    int e, nv;            // elements of a vector, vectors per thread
    int stages;           // per group
    int slot;             // bytes of one input's row in a stage (a multiple of 128)
    int inputs;           // of the stage
};

constexpr int kMaxRingGroups = 15;  // a named barrier each
constexpr int kMaxRingStages = 4;
// Threads of a block: what registers allow (a thread holds E NV columns, and backward 2 E NV sums).
// Forward, rows of which that many threads hold one only (LONG) have 1024 for two, which is worth the
// 64 registers: 3584 x 8192 bf16 46 to 44 us and 58 to 51 with 8-bit output; at 7168 x 4096 44 instead of 42.6.
template <int E, int NV, bool LONG = false>
constexpr int kRingFwd = LONG ? 1024 : E * NV >= 16 ? 896 : 960;
template <int E, int NV>
constexpr int kRingBwd = E * NV >= 16 ? 512 : 896;

struct RingSmem {
    uint64_t full[kMaxRingGroups * kMaxRingStages];
    float scratch[kMaxRingGroups][2][16];
};
constexpr size_t ring_smem(const Ring& q) {
    return sizeof(RingSmem) + 128 + (size_t)q.groups * q.stages * q.slot * q.inputs + (size_t)q.threads * q.nv * q.e * 8;
}

// 16 bytes of shared memory by address (addresses of 32 bits: generic pointers would cost these
// kernels a fifth of their instructions).
__device__ __forceinline__ uint4 lds16(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
    return v;
}
__device__ __forceinline__ void sts16(uint32_t at, uint4 v) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

#ifdef K1_WAIT_TEST
// Test only: one thread of block 0's first group takes the group's row of this number, and all after it,
// for rows whose wait ran out; the others see them land.  -1: off.
static __device__ long long k1_test_lone = -1;
#endif

// One group's view of its ring (shared-memory addresses).
struct RingGroup {
    uint32_t rings;    // all groups' stages
    uint32_t stages;   // this group's
    uint32_t full;
    uint32_t scratch;
    int t, id, stage_bytes, slots;
    int at;            // the current row's stage, and
    uint32_t parity;   // the parity of its use
    int failed;        // the row whose wait ran out
    bool ok;
    __device__ __forceinline__ void init(unsigned char* raw, const Ring& q) {
        RingSmem* sm = reinterpret_cast<RingSmem*>(raw);
        rings = (ring::saddr(raw) + (uint32_t)sizeof(RingSmem) + 127u) & ~127u;
        id = threadIdx.x / q.threads;
        t = threadIdx.x - id * q.threads;
        slots = q.stages;
        stage_bytes = q.slot * q.inputs;
        stages = rings + id * slots * stage_bytes;
        full = ring::saddr(sm->full + id * slots);
        scratch = ring::saddr(sm->scratch[id][0]);
        at = 0;
        parity = 0;
        failed = 0;
        ok = true;
        for (int i = threadIdx.x; i < kMaxRingGroups * 32; i += blockDim.x) sm->scratch[0][0][i] = 0.f;
        if (threadIdx.x == 0) {
            for (int i = 0; i < q.groups * slots; ++i) ring::bar_init(&sm->full[i], 1);
            ring::fence_init();
        }
        __syncthreads();
    }
    __device__ __forceinline__ bool wait_for(int slot, uint32_t parity_) const {
        for (int i = 0; i < ring::kMaxTries; ++i)
            if (ring::try_wait_at(full + slot * 8, parity_)) return true;
        atomicOr(&k1_ring_error, 1u);
        return false;
    }
    // The current stage holds row i of the group (or the wait ran out, now or before).
    __device__ __forceinline__ uint32_t wait(int i) {
        if (ok && !(ok = wait_for(at, parity))) failed = i;
#ifdef K1_WAIT_TEST
        if (ok && k1_test_lone == i && blockIdx.x == 0 && threadIdx.x == 5) {
            ok = false;
            failed = i;
            atomicOr(&k1_ring_error, 1u);
        }
#endif
        return stages + at * stage_bytes;
    }
    __device__ __forceinline__ void next() {
        if (++at == slots) {
            at = 0;
            parity ^= 1u;
        }
    }
    // The thread that orders, before it leaves: the copies that it has not seen land.
    __device__ __forceinline__ void drain(int rows) const {
        if (ok) return;
        for (int i = failed; i < min(rows, failed + slots); ++i) wait_for(i % slots, (uint32_t)(i / slots) & 1u);
    }
    // The sum over the group (what lies behind the last warp is 0).  Two buffers: `second` is the
    // caller's second sum of a row.
    __device__ __forceinline__ float sum(float v, int threads, bool second) const {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        const uint32_t to = scratch + (second ? 64 : 0);
        if ((t & 31) == 0) asm volatile("st.shared.f32 [%0], %1;" ::"r"(to + (t >> 5) * 4), "f"(v) : "memory");
        asm volatile("bar.sync %0, %1;" ::"r"(1 + id), "r"(threads) : "memory");
        auto four = [&](uint32_t from) {
            const uint4 a = lds16(from), b = lds16(from + 16);
            return add2(add2(make_float2(__uint_as_float(a.x), __uint_as_float(a.y)),
                             make_float2(__uint_as_float(a.z), __uint_as_float(a.w))),
                        add2(make_float2(__uint_as_float(b.x), __uint_as_float(b.y)),
                             make_float2(__uint_as_float(b.z), __uint_as_float(b.w))));
        };
        float2 s = four(to);
        if (threads > 256) s = add2(s, four(to + 32));
        return s.x + s.y;
    }
};

// Orders row i of the group, of every input that is not NULL, into a stage.
template <int N>
__device__ __forceinline__ void order_row(const RingGroup& g, const Ring& q, int i, int stage,
                                          const void* const (&rows)[N], int bytes) {
#ifdef K1_WAIT_TEST
    if (blockIdx.x == 0 && k1_test_withhold >= 0 && i >= k1_test_withhold) return;  // test only
#endif
    const uint32_t bar = g.full + stage * 8;
    uint32_t to = g.stages + stage * g.stage_bytes;
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(q.inputs * bytes) : "memory");
#pragma unroll
    for (int k = 0; k < N; ++k)
        if (rows[k]) {
            asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(to),
                         "l"(rows[k]), "r"(bytes), "r"(bar)
                         : "memory");
            to += q.slot;
        }
}

// Vectors as pairs of fp32 numbers: instructions are what these kernels run out of first (22 per element
// forward and 34 backward, counting all that a row costs; with generic addresses, single conversions and
// every option tested per row it was 48 and 86, and bound by that).
template <typename T>
struct Vec {
    static constexpr int E = DT<T>::kEPV, N = E / 2;
    __device__ static __forceinline__ uint4 at(uint32_t p) { return lds16(p); }
    __device__ static __forceinline__ void get(uint4 v, float2 (&f)[N]) {
        if constexpr (sizeof(T) == 4) {
            f[0] = make_float2(__uint_as_float(v.x), __uint_as_float(v.y));
            f[1] = make_float2(__uint_as_float(v.z), __uint_as_float(v.w));
        } else {
            f[0] = DT<T>::to_f2(v.x);
            f[1] = DT<T>::to_f2(v.y);
            f[2 % N] = DT<T>::to_f2(v.z);
            f[3 % N] = DT<T>::to_f2(v.w);
        }
    }
    __device__ static __forceinline__ uint4 put(const float2 (&f)[N]) {
        if constexpr (sizeof(T) == 4)
            return make_uint4(__float_as_uint(f[0].x), __float_as_uint(f[0].y), __float_as_uint(f[1].x),
                              __float_as_uint(f[1].y));
        else
            return make_uint4(DT<T>::from_f2(f[0]), DT<T>::from_f2(f[1]), DT<T>::from_f2(f[2 % N]),
                              DT<T>::from_f2(f[3 % N]));
    }
};

// A thread's columns of a weight as fp32 pairs (0 beyond the last column).
template <typename T, int NV, int N>
__device__ __forceinline__ void hold_weight(const void* w, bool w32, int t, int threads, int h, float2 (&f)[NV][N]) {
    constexpr int E = 2 * N;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int col = (j * threads + t) * E;
        float v[E];
#pragma unroll
        for (int k = 0; k < E; ++k) v[k] = 0.f;
        if (col < h) load_weight<T, E>(w, w32, col, v);
#pragma unroll
        for (int k = 0; k < N; ++k) f[j][k] = make_float2(v[2 * k], v[2 * k + 1]);
    }
}

// The weight w, and f = branch_scale post_weight (times a gate per column), as fp32 in shared memory.  A
// thread's 2 NV H pieces of 16 bytes (H to a vector) lie side by side, in an order that differs between
// the threads of an eighth of a warp, so that they meet no bank twice.
template <typename T, int NV>
struct Weights {
    static constexpr int E = DT<T>::kEPV, N = E / 2, H = E / 4, PIECES = 2 * NV * H;
    static_assert((PIECES & (PIECES - 1)) == 0 && PIECES <= 8, "pieces are told apart by exclusive or");
    uint32_t at;
    __device__ __forceinline__ uint32_t piece(int which, int j, int b) const { return at ^ (((which * NV + j) * H + b) * 16); }
    template <typename P>
    __device__ __forceinline__ void init(const RingGroup& g, const Ring& q, const P& p) {
        const int t = g.t;
        at = g.rings + q.groups * q.stages * g.stage_bytes + (uint32_t)((t * PIECES + (t * PIECES / 8 & (PIECES - 1))) * 16);
        if (g.id == 0) {
            float2 w[NV][N], f[NV][N], c[NV][N];
            hold_weight<T, NV, N>(p.w, p.w32, t, q.threads, p.h, w);
            hold_weight<T, NV, N>(p.wp, p.w32, t, q.threads, p.h, f);
            if (p.gate_kind == GATE_COLUMN) hold_weight<T, NV, N>(p.gate, p.w32, t, q.threads, p.h, c);
#pragma unroll
            for (int j = 0; j < NV; ++j) {
#pragma unroll
                for (int k = 0; k < N; ++k) {
                    f[j][k] = mul2(f[j][k], splat(p.branch_scale));
                    if (p.gate_kind == GATE_COLUMN) f[j][k] = mul2(f[j][k], c[j][k]);
                }
#pragma unroll
                for (int b = 0; b < H; ++b) {
                    auto keep = [&](int which, float2 lo, float2 hi) {
                        sts16(piece(which, j, b), make_uint4(__float_as_uint(lo.x), __float_as_uint(lo.y),
                                                             __float_as_uint(hi.x), __float_as_uint(hi.y)));
                    };
                    keep(0, w[j][2 * b], w[j][2 * b + 1]);
                    keep(1, f[j][2 * b], f[j][2 * b + 1]);
                }
            }
        }
        __syncthreads();
    }
    // w (0) or f (1) of the thread's vector j
    __device__ __forceinline__ void get(int which, int j, float2 (&v)[N]) const {
#pragma unroll
        for (int b = 0; b < H; ++b) {
            const uint4 u = lds16(piece(which, j, b));
            v[2 * b] = make_float2(__uint_as_float(u.x), __uint_as_float(u.y));
            v[2 * b + 1] = make_float2(__uint_as_float(u.z), __uint_as_float(u.w));
        }
    }
};

template <typename T, int NV, int OUT, bool LONG>
__global__ void __launch_bounds__(kRingFwd<DT<T>::kEPV, NV, LONG>, 1) k1_sandwich_ring_kernel(FwdParams p, Ring q) {
    using V = Vec<T>;
    constexpr int E = V::E, N = V::N;
    extern __shared__ __align__(16) unsigned char raw[];
    RingGroup g;
    g.init(raw, q);
    pdl_wait();
    pdl_trigger();
    const int t = g.t, threads = q.threads, h = p.h, bytes = h * (int)sizeof(T);
    const int64_t step = (int64_t)gridDim.x * q.groups, first = (int64_t)blockIdx.x * q.groups + g.id;
    const int rows = first < p.n ? (int)((p.n - 1 - first) / step + 1) : 0;
    const int n_blocks = (h + kFp8Block - 1) / kFp8Block;
    const T* gates = p.gate_kind == GATE_FULL ? reinterpret_cast<const T*>(p.gate) : nullptr;
    auto order = [&](int i, int stage) {
        const int64_t row = first + i * step;
        const void* from[3] = {reinterpret_cast<const T*>(p.x) + row * p.x_stride,
                               reinterpret_cast<const T*>(p.r) + row * p.r_stride,
                               gates ? gates + row * p.gate_stride : nullptr};
        order_row(g, q, i, stage, from, bytes);
    };
    if (t == 0)
        for (int i = 0; i < min(rows, q.stages); ++i) order(i, i);
    Weights<T, NV> weights;
    weights.init(g, q, p);
    const float2 rs = splat(p.residual_scale);
    const float inv_h = 1.f / (float)h;
    // a row's gate is loaded while the row before it is worked on
    auto gate_of = [&](int i) {
        return p.gate_kind == GATE_TOKEN && i < rows
                   ? DT<T>::load1(reinterpret_cast<const T*>(p.gate) + (first + i * step) * p.gate_stride) : 1.f;
    };
    float token_next = gate_of(0);
    int64_t at_row = first * h + t * E;  // the thread's place in the outputs
    for (int i = 0; i < rows; ++i, g.next(), at_row += step * h) {
        const int64_t row = first + i * step;
        const float token = token_next;
        token_next = gate_of(i + 1);
        const uint32_t in = g.wait(i) + t * 16;
        float2 x[NV][N], two = splat(0.f);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            if ((j * threads + t) * E >= h) break;
            V::get(V::at(in + j * threads * 16), x[j]);
#pragma unroll
            for (int k = 0; k < N; ++k) two = fma2(x[j][k], x[j][k], two);
        }
        if (!g.ok) two.x = __int_as_float(0x7fc00000);  // one thread's wait ran out: the row is lost to all
        float sum = g.sum(two.x + two.y, threads, false);
        const float r1 = rsqrtf(fmaf(sum, inv_h, p.eps));
        if (p.rstd_post && t == 0) p.rstd_post[row] = r1;
        const float2 k1 = splat(r1 * token);
        two = splat(0.f);
        T* so = reinterpret_cast<T*>(p.s) + at_row;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int col = (j * threads + t) * E;
            if (col >= h) break;
            const uint32_t at = in + j * threads * 16;
            float2 b[N];
            V::get(V::at(at + q.slot), b);
            if (gates) {
                float2 c[N];
                V::get(V::at(at + 2 * q.slot), c);
#pragma unroll
                for (int k = 0; k < N; ++k) x[j][k] = mul2(x[j][k], c[k]);
            }
            float2 f[N];
            weights.get(1, j, f);
#pragma unroll
            for (int k = 0; k < N; ++k) x[j][k] = fma2(mul2(x[j][k], k1), f[k], mul2(b[k], rs));
            const uint4 s = V::put(x[j]);
            stg_stream(so + j * threads * E, s);
            V::get(s, x[j]);  // the stream as stored
#pragma unroll
            for (int k = 0; k < N; ++k) two = fma2(x[j][k], x[j][k], two);
        }
        sum = g.sum(two.x + two.y, threads, true);  // after it nobody reads the stage
        if (t == 0 && g.ok && i + q.stages < rows) order(i + q.stages, g.at);
        const float r2 = rsqrtf(fmaf(sum, inv_h, p.eps));
        if (p.rstd && t == 0) p.rstd[row] = r2;
        if constexpr (OUT == SAME) {
            T* y = reinterpret_cast<T*>(p.y) + at_row;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int col = (j * threads + t) * E;
                if (col >= h) break;
                float2 w[N];
                weights.get(0, j, w);
#pragma unroll
                for (int k = 0; k < N; ++k) x[j][k] = mul2(mul2(x[j][k], splat(r2)), w[k]);
                stg_stream(y + j * threads * E, V::put(x[j]));
            }
        } else {
            // as in k1_rmsnorm_kernel, which has the reasons; the largest value is taken before the factor 7/8,
            // so that its part in 512 needs no division, and its reciprocal may be rough (the quotient's
            // Newton step makes up for it; the step is at least 1e-33 and at most 1e36)
            const uint32_t bits = __float_as_uint(r2);
            const float unit = r2 == r2 ? __uint_as_float(bits & 0x7f800000u) : r2;
            const float rest = __uint_as_float((bits & 0x007fffffu) | 0x3f800000u) * (8.f / 7.f);
            const float least = kAmaxFloor * (8.f / 7.f) / rest;
            constexpr int LANES = kFp8Block / E;
            uint8_t* y = reinterpret_cast<uint8_t*>(p.y) + at_row;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int col = (j * threads + t) * E;
                float2 (&a)[N] = x[j];
                float m = 0.f;
                if (col < h) {
                    float2 w[N];
                    weights.get(0, j, w);
#pragma unroll
                    for (int k = 0; k < N; ++k) {
                        a[k] = mul2(mul2(a[k], splat(unit)), w[k]);
                        m = fmax_nan(m, fmax_nan(fabsf(a[k].x), fabsf(a[k].y)));
                    }
                }
#pragma unroll
                for (int o = LANES / 2; o > 0; o >>= 1) m = fmax_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
                if (col < h) {
                    const float d = fmax_nan(m, least) * (1.f / 512.f);
                    float inv;
                    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(d));
                    const Quotient to(d, inv);
                    uint32_t v[N];
#pragma unroll
                    for (int k = 0; k < N; ++k) {  // Quotient's steps, in pairs
                        const float2 n = mul2(a[k], splat(0.875f));
                        const float2 c = mul2(n, splat(to.inv));
                        const float2 e = fma2(fma2(make_float2(-c.x, -c.y), splat(to.step), n), splat(to.inv), c);
                        v[k] = e4m3x2(e.x, e.y);
                    }
                    if constexpr (E == 8)
                        *reinterpret_cast<uint2*>(y + j * threads * E) =
                            make_uint2(v[0] | (v[1] << 16), v[2 % N] | (v[3 % N] << 16));
                    else
                        *reinterpret_cast<uint32_t*>(y + j * threads * E) = v[0] | (v[1] << 16);
                    if ((t & (LANES - 1)) == 0) p.scales[row * n_blocks + col / kFp8Block] = d * rest;
                }
            }
        }
    }
    if (t == 0) g.drain(rows);
}

// Per row and column: ds as in the header; with m = x R1 and f = bs wp (gate per column, where there
// is one),
//   t = ds f gate (per row or element), dot = sum t m;  dx = R1 (t - m dot / h)
//   A = sum over rows of ds m gate (per row or element), of which dwp and a column gate's gradient are
//   multiples: bs gate A and bs wp A.
// So two sums per column whatever the gate.  PLAIN: both gradients come in, both go out, and the gate
// is not per element, so that a training step's rows test for none of it.
template <typename T, int NV, bool PLAIN>
__global__ void __launch_bounds__(kRingBwd<DT<T>::kEPV, NV>, 1) k1_sandwich_bwd_ring_kernel(SandwichBwdParams p, Ring q) {
    using V = Vec<T>;
    constexpr int E = V::E, N = V::N;
    extern __shared__ __align__(16) unsigned char raw[];
    RingGroup g;
    g.init(raw, q);
    pdl_wait();
    pdl_trigger();
    const int t = g.t, threads = q.threads, h = p.h, bytes = h * (int)sizeof(T);
    const int64_t step = (int64_t)gridDim.x * q.groups, first = (int64_t)blockIdx.x * q.groups + g.id;
    const int rows = first < p.n ? (int)((p.n - 1 - first) / step + 1) : 0;
    const bool has_gy = PLAIN || p.gy, has_gs = PLAIN || p.gs;
    const T* gates = !PLAIN && p.gate_kind == GATE_FULL ? reinterpret_cast<const T*>(p.gate) : nullptr;
    // the inputs' places in a stage: s, x, then those of gy, gs and the gate that there are
    const int at_gs = q.slot * (2 + has_gy), at_gate = at_gs + q.slot * has_gs;
    auto order = [&](int i, int stage) {
        const int64_t row = first + i * step;
        const void* from[5] = {reinterpret_cast<const T*>(p.s) + row * p.s_stride,
                               reinterpret_cast<const T*>(p.x) + row * p.x_stride,
                               has_gy ? reinterpret_cast<const T*>(p.gy) + row * p.gy_stride : nullptr,
                               has_gs ? reinterpret_cast<const T*>(p.gs) + row * p.gs_stride : nullptr,
                               gates ? gates + row * p.gate_stride : nullptr};
        order_row(g, q, i, stage, from, bytes);
    };
    if (t == 0)
        for (int i = 0; i < min(rows, q.stages); ++i) order(i, i);
    Weights<T, NV> weights;
    weights.init(g, q, p);
    float2 dw[NV][N], A[NV][N];
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int k = 0; k < N; ++k) dw[j][k] = A[j][k] = splat(0.f);
    const float inv_h = 1.f / (float)h;
    // a row's own values are loaded while the row before it is worked on
    float next_r1 = 0.f, next_r2 = 0.f, next_token = 1.f;
    auto fetch = [&](int i) {
        if (i >= rows) return;
        const int64_t row = first + i * step;
        next_r1 = p.rstd_post[row];
        next_r2 = p.rstd[row];
        if (p.gate_kind == GATE_TOKEN) next_token = DT<T>::load1(reinterpret_cast<const T*>(p.gate) + row * p.gate_stride);
    };
    fetch(0);
    int64_t at_row = first * h + t * E;  // the thread's place in the outputs
    for (int i = 0; i < rows; ++i, g.next(), at_row += step * h) {
        const float r1 = next_r1, token = next_token;
        float r2 = next_r2;
        fetch(i + 1);
        const uint32_t in = g.wait(i) + t * 16;
        if (!g.ok) r2 = __int_as_float(0x7fc00000);
        float c2 = 0.f;
        if (has_gy) {
            float2 sum = splat(0.f);
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                if ((j * threads + t) * E >= h) break;
                const uint32_t at = in + j * threads * 16;
                float2 a[N], b[N], w[N];
                V::get(V::at(at + 2 * q.slot), a);
                V::get(V::at(at), b);
                weights.get(0, j, w);
#pragma unroll
                for (int k = 0; k < N; ++k) {
                    a[k] = mul2(a[k], b[k]);
                    sum = fma2(a[k], w[k], sum);
                    dw[j][k] = fma2(a[k], splat(r2), dw[j][k]);
                }
            }
            c2 = g.sum((sum.x + sum.y) * r2, threads, false) * inv_h;
        }
        float2 dots = splat(0.f);
        const float2 minus = splat(-r2 * r2 * c2);
        float2 u[NV][N];
        uint4 x[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            if ((j * threads + t) * E >= h) break;
            const uint32_t at = in + j * threads * 16;
            float2 ds[N], a[N], b[N];
            if (has_gs) {
                V::get(V::at(at + at_gs), ds);
            } else {
#pragma unroll
                for (int k = 0; k < N; ++k) ds[k] = splat(0.f);
            }
            if (has_gy) {
                V::get(V::at(at), a);
#pragma unroll
                for (int k = 0; k < N; ++k) ds[k] = fma2(a[k], minus, ds[k]);
                V::get(V::at(at + 2 * q.slot), a);
                weights.get(0, j, b);
#pragma unroll
                for (int k = 0; k < N; ++k) ds[k] = fma2(mul2(a[k], b[k]), splat(r2), ds[k]);
            } else if (!g.ok) {
#pragma unroll
                for (int k = 0; k < N; ++k) ds[k] = splat(r2);
            }
            if (PLAIN || p.dr) {
#pragma unroll
                for (int k = 0; k < N; ++k) a[k] = mul2(ds[k], splat(p.residual_scale));
                stg_stream(reinterpret_cast<T*>(p.dr) + at_row + j * threads * E, V::put(a));
            }
            x[j] = V::at(at + q.slot);
            V::get(x[j], a);
            weights.get(1, j, b);
#pragma unroll
            for (int k = 0; k < N; ++k) {
                a[k] = mul2(a[k], splat(r1));  // m
                u[j][k] = mul2(ds[k], b[k]);
                ds[k] = mul2(ds[k], a[k]);     // ds m
            }
            if (gates) {  // a gate per element: its gradient, and the products with it
                V::get(V::at(at + at_gate), b);
                float2 c[N];
#pragma unroll
                for (int k = 0; k < N; ++k) {
                    c[k] = mul2(u[j][k], a[k]);
                    u[j][k] = mul2(u[j][k], b[k]);
                    ds[k] = mul2(ds[k], b[k]);
                }
                if (p.dgate) stg_stream(reinterpret_cast<T*>(p.dgate) + at_row + j * threads * E, V::put(c));
            }
#pragma unroll
            for (int k = 0; k < N; ++k) {
                dots = fma2(u[j][k], a[k], dots);
                A[j][k] = fma2(ds[k], splat(token), A[j][k]);
            }
        }
        const float dot = g.sum(dots.x + dots.y, threads, has_gy || (i & 1));  // after it nobody reads the stage
        if (t == 0 && g.ok && i + q.stages < rows) order(i + q.stages, g.at);
        if (p.dgate && p.gate_kind == GATE_TOKEN && t == 0)
            DT<T>::store1(reinterpret_cast<T*>(p.dgate) + first + i * step, dot);
        if (PLAIN || p.dx) {
            const float2 c1 = splat(-r1 * dot * inv_h);
            const float2 k1 = splat(r1 * token);
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                if ((j * threads + t) * E >= h) break;
                float2 a[N];
                V::get(x[j], a);
#pragma unroll
                for (int k = 0; k < N; ++k) a[k] = mul2(fma2(a[k], c1, u[j][k]), k1);
                stg_stream(reinterpret_cast<T*>(p.dx) + at_row + j * threads * E, V::put(a));
            }
        }
    }
    if (t == 0) g.drain(rows);
    if (!p.sums) return;
    // the groups' sums, added in their order; the rings have room for one of them from each group
    float* part = reinterpret_cast<float*>(raw + (g.rings - ring::saddr(raw)));
    auto add = [&](int k, bool wanted, const float2 (&v)[NV][N], float factor) {
        if (!wanted) return;
        __syncthreads();
        if (g.id > 0) {
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int col = (j * threads + t) * E;
                if (col >= h) break;
#pragma unroll
                for (int c = 0; c < N; ++c) *reinterpret_cast<float2*>(part + (g.id - 1) * h + col + 2 * c) = v[j][c];
            }
        }
        __syncthreads();
        if (g.id > 0) return;
        float* out = p.sums + ((int64_t)k * gridDim.x + blockIdx.x) * h;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int col = (j * threads + t) * E;
            if (col >= h) break;
#pragma unroll
            for (int c = 0; c < N; ++c) {
                float2 s = v[j][c];
                for (int o = 0; o < q.groups - 1; ++o) s = add2(s, *reinterpret_cast<const float2*>(part + o * h + col + 2 * c));
                *reinterpret_cast<float2*>(out + col + 2 * c) = mul2(s, splat(factor));
            }
        }
    };
    add(0, p.want & 1, dw, 1.f);
    add(1, p.want & 6, A, p.branch_scale);
}

// The blocks' partial sums (blockIdx.y: of dw, or of A), added in a fixed order as in
// k1_rmsnorm_dw_kernel, by 32 warps so that one batch of loads covers them.  A gives dwp (times a gate per
// column) and that gate's gradient (times wp).
template <typename W>
__global__ void __launch_bounds__(1024) k1_sandwich_dw_kernel(const float* part, int parts, int h, W* dw, W* dwp, W* dg,
                                                             const W* wp, const W* gate) {
    __shared__ float sums[32][33];
    pdl_wait();
    pdl_trigger();
    part += (int64_t)blockIdx.y * parts * h;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int col = blockIdx.x * 32 + lane;
    float v = 0.f;
    if (col < h) {
#pragma unroll 8
        for (int i = warp; i < parts; i += 32) v += part[(int64_t)i * h + col];
    }
    sums[warp][lane] = v;
    __syncthreads();
    if (warp == 0 && col < h) {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) t += sums[i][lane];
        if (blockIdx.y == 0) {
            if (dw) DT<W>::store1(dw + col, t);
        } else {
            if (dwp) DT<W>::store1(dwp + col, gate ? t * DT<W>::load1(gate + col) : t);
            if (dg) DT<W>::store1(dg + col, t * DT<W>::load1(wp + col));
        }
    }
}

}  // namespace norm
}  // namespace k1
