// k1_score.cuh -- log-probabilities of given tokens and of the k most likely ones, with entropy
// and log-sum-exp, in one pass over the logits, and their gradient.
//
//   y_i = s x_i (s = 1/T in fp32; y is not rounded),  l = log sum exp y_i,  log p_i = y_i - l
//   H = -sum p_i log p_i
//   the k most likely: larger x first, the lowest index first among equals
//   dL/dx_i = s ( G_i + p_i (g_l - sum of all g_j - g_H (log p_i + H)) ),  G_i: the sum of the
//   upstream gradients of the entries of row's lists that name token i
//
// A row is read once as 16-byte vectors from its own 16-byte boundary (the first and last vector
// may be partly outside the row: those are put together from single elements).  A block of
// threads owns a row, or a part of one where there are few rows; the parts' blocks are a cluster
// and meet in the first one's shared memory.  Sums run as in k1_common.cuh (the maximum's own
// terms counted apart, so that a near-one-hot row's entropy keeps its precision), on x itself
// with the factor s log2 e in the exponent, so a temperature costs no instruction.
//
// The k most likely cost almost nothing while streaming: each thread stores the maximum of every
// group of its vectors (one chunk's 8 usually), which the sums need anyway.  Then
//   T0, the k-th largest of the threads' maxima cut to 16 bits, is a bound that at least k
//   elements reach, and usually few more;
//   the groups that reach T0 are read again (from L2, some k x 64 bytes) and their elements that
//   do go to a list of 64-bit keys (value, then lowest index), each key's rank in the list is its
//   place.
// Where that overflows (many equal values, masks that leave fewer than k, rows whose large values
// lie in few threads' columns) the block finds the k-th largest value by histograms of 8 bits a
// pass and takes the equal ones in index order.  Either way the result is exact.
//
// Forward and backward are bound by traffic where rows are many and wide; small calls by latency, and
// lists by the chain of short phases behind a row's last load.  Measured on B200 (us, with the call):
// 2048 x 151936 bf16, 32 given tokens, forward 108 (5.8 TB/s) and backward 211 (5.9 TB/s), 323 to 335
// together; 1024 x 128256 bf16 top 8 with gradient 149 to 153; 512 x 152064 bf16 top 20 38 to 39 (32 without a
// list, its bytes 24); 1023 x 50257 fp16 top 64 32 to 33 (22 without, 16); one row of 151936 top 20 11.
//
// Two ways are slow, and right.  A list where a mask leaves fewer than k in a block's part takes the exact
// selection: 512 x 152064 bf16 with 50 tokens left 480.  The backward stores single elements where a row of the
// gradient starts at another place of a 16-byte vector than its logits (a window of a wider head, odd
// vocabularies): 1024 x 50257 of 50304 columns 162, all columns of 50257 45.
#pragma once

#include <cstddef>
#include <type_traits>

#include "k1_common.cuh"
#include "k1_sync.cuh"

namespace k1 {
namespace score {

constexpr int kMaxGroups = 32;   // maxima per thread
constexpr int kKeys = 256;       // maxima that the bound is found among
constexpr int kCand = 512;       // entries of the list
constexpr int kMaxTop = 128;     // largest k
constexpr int kMaxIds = 1024;    // given tokens per row
constexpr int kMaxCluster = 8;

// Values at or below this count as masked (p = 0); 16-bit types: as the type rounds it.  pad: what
// stands for elements outside the row.
template <typename T>
struct Floor;
template <>
struct Floor<__nv_bfloat16> {
    static constexpr uint32_t pad = 0xFE96FE96u;  // -9.97e37, both halves
    static constexpr float value = -9.969209968386869e37f;
};
template <>
struct Floor<__half> {
    static constexpr uint32_t pad = 0xFC00FC00u;  // -inf, both halves
    static constexpr float value = -1.0e38f;      // fp16's own values lie above
};
template <>
struct Floor<float> {
    static constexpr uint32_t pad = 0xFE967699u;  // -1e38
    static constexpr float value = -1.0e38f;
};

// Differences of values that fp32 has no number for are held to this in sums: of a masked value and a maximum
// above 2.4e38, say, whose weight, 0, times an infinity would be NaN.
constexpr float kFar = -3.0e38f;

struct FwdParams {
    const void* logits;
    RowLayout lay;
    int64_t vocab;
    float scale;
    const int64_t* ids;  // [n, n_ids]
    int n_ids;
    float* logprobs;     // [n, n_ids]
    int k;
    int64_t* top_ids;    // [n, k]
    float* top_logprobs; // [n, k]
    float* entropy;
    float* lse;
    float* lse_rest;     // lse before its rounding, less lse; may be NULL
    int cluster;         // blocks per row
    int slice;           // vectors per block
    int groups;          // groups per thread
    int group_chunks;    // chunks per group
};

// One thread's sums, relative to its warp's maximum m (as k1_common.cuh's FwdState, which has each
// thread's own; c = s log2 e is the exponent's factor, t a sum of e d in x, not y).  A warp's chunk whose
// values all lie below m, which nearly all chunks but a row's first do, needs neither the maximum's
// terms told apart nor the reference moved: 5.5 instructions per element instead of 7.9 (2048 x 151936
// bf16, with the next chunk's loads in flight: 122 -> 108 us).
struct State {
    float m, np;
    float2 zs, ms, t;
    __device__ __forceinline__ void init() {
        m = -3.402823466e38f;
        np = 0.f;
        zs = ms = t = splat(0.f);
    }
    __device__ __forceinline__ float2 at_max() const { return make_float2(np - ms.x, np - ms.y); }
    __device__ __forceinline__ void rescale(float mc, float c) {
        const float mn = fmax_nan(m, mc);
        const float dl = m - mn;
        const bool moved = !(dl == 0.f);
        const float s = moved ? ex2(dl * c) : 1.f;
        const float2 z = add2(zs, at_max());
        t = fma2(splat(dl * s), z, mul2(t, splat(s)));
        if (moved) {
            zs = mul2(z, splat(s));
            ms = splat(0.f);
            np = 0.f;
        }
        m = mn;
    }
    template <bool BELOW>
    __device__ __forceinline__ void accum(float2 d, float2 c2) {
        const float2 a = mul2(d, c2);
        const float2 e = make_float2(ex2(a.x), ex2(a.y));
        if constexpr (BELOW) {
            zs = add2(zs, e);
        } else {
            const float2 nz = make_float2(not_zero(d.x), not_zero(d.y));
            zs = fma2(e, nz, zs);
            ms = add2(ms, nz);
        }
        t = fma2(e, d, t);
    }
    __device__ __forceinline__ double z64() const {
        const float2 c = at_max();
        return ((double)c.x + (double)c.y) + ((double)zs.x + (double)zs.y);
    }
    __device__ __forceinline__ double t64() const { return (double)t.x + (double)t.y; }
};

// The largest of a warp's values, NaN where there is one.
__device__ __forceinline__ float warp_max(float v) {
    float m;
    asm("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
    return m;
}

template <typename T, int N, bool BELOW>
__device__ __forceinline__ void add_words(const uint32_t (&w)[4 * N], State& st, float c) {
    const float2 c2 = splat(c);
    const float nm = -st.m;
#pragma unroll
    for (int i = 0; i < 4 * N; ++i) {
        if constexpr (std::is_same<T, __nv_bfloat16>::value) {
            st.accum<BELOW>(bf16x2_minus(w[i], nm), c2);
        } else if constexpr (sizeof(T) == 2) {  // -inf stays outside fp16's range, so that -65504 is a value like others
            const float2 d = f16x2_minus(w[i], nm);
            st.accum<BELOW>(make_float2(fmax_nan(d.x, Floor<T>::value), fmax_nan(d.y, Floor<T>::value)), c2);
        } else if (i % 2 == 0) {
            st.accum<BELOW>(add2(make_float2(__uint_as_float(w[i]), __uint_as_float(w[i + 1])), splat(nm)), c2);
        }
    }
    if constexpr (!BELOW) st.np += sizeof(T) == 2 ? (float)(4 * N) : (float)(2 * N);
}

// Adds a chunk of N vectors per lane to a warp's states; returns the lane's maximum (of the values as
// clamped).
template <typename T, int N>
__device__ __forceinline__ float add_chunk(const uint4 (&v)[N], State& st, float c) {
    uint32_t w[4 * N];
#pragma unroll
    for (int u = 0; u < N; ++u) {
        w[4 * u] = v[u].x;
        w[4 * u + 1] = v[u].y;
        w[4 * u + 2] = v[u].z;
        w[4 * u + 3] = v[u].w;
    }
    float mc;
    if constexpr (sizeof(T) == 2) {
        uint32_t mx[4 * N];
#pragma unroll
        for (int i = 0; i < 4 * N; ++i) {
            if constexpr (std::is_same<T, __nv_bfloat16>::value) w[i] = DT<T>::max2(w[i], Floor<T>::pad);
            mx[i] = w[i];
        }
#pragma unroll
        for (int s = 2 * N; s >= 1; s >>= 1)
#pragma unroll
            for (int i = 0; i < s; ++i) mx[i] = DT<T>::max2(mx[i], mx[i + s]);
        const float2 mf = DT<T>::to_f2(mx[0]);
        mc = fmax_nan(mf.x, mf.y);
    } else {
        float mx[4 * N];
#pragma unroll
        for (int i = 0; i < 4 * N; ++i) {
            mx[i] = fmax_nan(__uint_as_float(w[i]), Floor<T>::value);
            w[i] = __float_as_uint(mx[i]);
        }
#pragma unroll
        for (int s = 2 * N; s >= 1; s >>= 1)
#pragma unroll
            for (int i = 0; i < s; ++i) mx[i] = fmax_nan(mx[i], mx[i + s]);
        mc = mx[0];
    }
    const float wm = warp_max(mc);
    if (wm < st.m) {  // the same in all lanes
        add_words<T, N, true>(w, st, c);
    } else {
        st.rescale(wm, c);
        add_words<T, N, false>(w, st, c);
    }
    return mc;
}

// A row as vectors from the 16-byte boundary at or before its first element: vector j holds
// elements j E - shift ... ; whole vectors are [lo, hi), all that touch the row [0, n).
template <typename T>
struct Row {
    static constexpr int E = DT<T>::kEPV;
    const T* p;
    const uint4* base;
    int shift, lo, hi, n;
    int64_t vocab;
    __device__ __forceinline__ Row(const T* row, int64_t v) {
        p = row;
        vocab = v;
        shift = (int)((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T));
        base = reinterpret_cast<const uint4*>(row - shift);
        lo = shift ? 1 : 0;
        hi = (int)((shift + v) / E);
        n = (int)((shift + v + E - 1) / E);
    }
    // element i of vector j
    __device__ __forceinline__ int64_t at(int j, int i) const { return (int64_t)j * E + i - shift; }
    __device__ __forceinline__ bool inside(int64_t e) const { return (uint64_t)e < (uint64_t)vocab; }
    // a vector that is partly outside the row, put together from its elements (rare)
    __device__ __noinline__ uint4 partial(int j) const {
        uint32_t w[4];
        const uint32_t pad = Floor<T>::pad;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = pad;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const int64_t e = at(j, i);
            if (inside(e)) {
                if constexpr (sizeof(T) == 2) {
                    const uint32_t b = *reinterpret_cast<const uint16_t*>(p + e);
                    w[i / 2] = i & 1 ? (w[i / 2] & 0xffffu) | (b << 16) : (w[i / 2] & 0xffff0000u) | b;
                } else {
                    w[i] = *reinterpret_cast<const uint32_t*>(p + e);
                }
            }
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    // vectors j, j + step, ... below `end`; what lies beyond reads as padding
    template <int N>
    __device__ __forceinline__ void load(uint4 (&v)[N], int j, int step, int end) const {
        const uint32_t pad = Floor<T>::pad;
        const int to = min(end, hi);
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const int a = j + u * step;
            v[u] = a >= lo && a < to ? ldg_stream(base + a) : make_uint4(pad, pad, pad, pad);
        }
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const int a = j + u * step;
            if (a < end && (a < lo || a >= hi)) v[u] = partial(a);
        }
    }
};

// A thread's sum of e d once more, relative to the part's maximum and with differences held to kFar: for logits
// beyond 1e31, where a difference (or an earlier reference's) was beyond fp32 and the sum is NaN.  Out of the
// way of all others: held in the loop itself, lists took 1 % longer.
template <typename T, int TH>
__device__ __noinline__ double far_sum(const T* p, int64_t vocab, int j0, int j1, float m, float c) {
    constexpr int E = DT<T>::kEPV;
    const Row<T> row(p, vocab);
    double t = 0.0;
    for (int j = j0 + threadIdx.x; j < j1; j += TH)
        for (int i = 0; i < E; ++i) {
            const int64_t e = row.at(j, i);
            if (!row.inside(e)) continue;
            const float d = fmax_nan(fmax_nan(DT<T>::load1(p + e), Floor<T>::value) - m, kFar);
            t += (double)ex2(d * c) * (double)d;
        }
    return t;
}

template <typename T>
__device__ __forceinline__ void unpack(uint4 v, float (&f)[DT<T>::kEPV]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) {
            f[i] = __uint_as_float(w[i]);
        } else {
            const float2 t = DT<T>::to_f2(w[i]);
            f[2 * i] = t.x;
            f[2 * i + 1] = t.y;
        }
    }
}

// Keys in the values' order (-0 as 0), and back.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t u = __float_as_uint(x + 0.f);
    return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
// Larger is earlier in the list: the larger value, then the lower index.
__device__ __forceinline__ uint64_t entry_of(float x, int64_t e) {
    return ((uint64_t)key_of(x) << 32) | (uint32_t)~(uint32_t)e;
}

// Shared memory is kept small: what it leaves is L1, through which the loads in flight go (with 26
// instead of 24 KB per block, 182 instead of 168 per SM, 1024 x 128256 bf16 with gradient took 165 us
// instead of 151; with all of it as shared memory, 2048 x 151936 took 372 instead of 323).
template <int TH>
struct FwdSums {
    static constexpr int W = TH / 32;
    double wz[W], wt[W];
    unsigned wmax[W];         // keys of the warps' maxima
};
// Only where a list is wanted; behind it the groups' maxima, [groups][TH], as the upper 16 bits of keys.
struct FwdList {
    int n_cand;
    unsigned bound;           // T0's key, its upper 16 bits
    unsigned prefix, need, scan[8];
    int n_list;
    uint16_t keys[kKeys];
    uint16_t list[kCand];
    union {
        uint64_t cand[kCand];
        unsigned hist[256];   // while the list is empty
    };
};
// Of a cluster's first block, written by all: their sums and their lists.
struct Meet {
    RowPartial part[kMaxCluster];
    int n[kMaxCluster];
    uint64_t list[kMaxCluster][kMaxTop];  // only where a list is wanted
};
template <int TH, bool TOP>
constexpr size_t fwd_smem(int cluster, int groups) {
    return sizeof(FwdSums<TH>) + (cluster > 1 ? (TOP ? sizeof(Meet) : offsetof(Meet, list)) : 0) +
           (TOP ? sizeof(FwdList) + (size_t)groups * TH * 2 : 0);
}

// The block's list by exact selection: the kk-th largest key by histograms, what lies above it,
// and the first ones in index order among what equals it.
template <typename T, int TH>
__device__ __noinline__ void select_exact(const Row<T>& row, int j0, int j1, int kk, FwdList& sm) {
    constexpr int E = DT<T>::kEPV;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    auto each = [&](int j, auto&& f) {
        uint4 v[1];
        row.template load<1>(v, j, 0, j1);
        float x[E];
        unpack<T>(v[0], x);
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const int64_t e = row.at(j, i);
            if (j < j1 && row.inside(e)) f(x[i], e);
        }
    };
    unsigned prefix = 0, mask = 0, need = (unsigned)kk;
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = tid; i < 256; i += TH) sm.hist[i] = 0;
        __syncthreads();
        unsigned bin = 0, run = 0;  // equal values in a row are counted together
        for (int j = j0 + tid; j < j1; j += TH)
            each(j, [&](float x, int64_t) {
                const unsigned k = key_of(x);
                if ((k & mask) != prefix) return;
                const unsigned b = (k >> shift) & 255u;
                if (b != bin) {
                    if (run) atomicAdd(&sm.hist[bin], run);
                    bin = b;
                    run = 0;
                }
                ++run;
            });
        if (run) atomicAdd(&sm.hist[bin], run);
        __syncthreads();
        if (tid == 0) {
            unsigned sum = 0;
            int b = 255;
            while (b > 0 && sum + sm.hist[b] < need) sum += sm.hist[b--];
            sm.prefix = prefix | ((unsigned)b << shift);
            sm.need = need - sum;
        }
        __syncthreads();
        prefix = sm.prefix;
        need = sm.need;
        mask |= 255u << shift;
    }
    const int above = kk - (int)need;
    if (tid == 0) sm.n_cand = 0;
    __syncthreads();
    for (int j = j0 + tid; j < j1; j += TH)
        each(j, [&](float x, int64_t e) {
            if (key_of(x) > prefix) sm.cand[atomicAdd(&sm.n_cand, 1)] = entry_of(x, e);
        });
    unsigned found = 0;
    for (int jb = j0; jb < j1 && found < need; jb += TH) {
        const int j = jb + tid;
        unsigned n = 0;
        each(j, [&](float x, int64_t) { n += key_of(x) == prefix; });
        unsigned upto = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned a = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += a;
        }
        __syncthreads();
        if (lane == 31) sm.scan[warp] = upto;
        __syncthreads();
        unsigned at = found + upto - n;
        for (int w = 0; w < TH / 32; ++w) {
            if (w < warp) at += sm.scan[w];
            found += sm.scan[w];
        }
        if (n && at < need)
            each(j, [&](float x, int64_t e) {
                if (key_of(x) == prefix && at < need) sm.cand[above + at++] = entry_of(x, e);
            });
    }
    __syncthreads();
    if (tid == 0) sm.n_cand = kk;
    __syncthreads();
}

// T0: a bound that kk of the threads' maxima reach and, to 16 bits, no more than their equals do (one
// warp).
template <int TH>
__device__ __forceinline__ void find_bound(int kk, FwdList& sm) {
    const int lane = threadIdx.x & 31;
    unsigned mine[kKeys / 32], top = 0, low = 0xffffu;
#pragma unroll
    for (int i = 0; i < kKeys / 32; ++i) {
        mine[i] = sm.keys[lane + 32 * i];
        top = max(top, mine[i]);
        low = min(low, mine[i]);
    }
    top = __reduce_max_sync(0xffffffffu, top);
    low = __reduce_min_sync(0xffffffffu, low);
    // bit by bit below the common prefix of all keys
    unsigned t = top;
    if (top != low) {
        int b = 31 - __clz((int)(top ^ low));
        t = top & ~((2u << b) - 1u);
        for (; b >= 0; --b) {
            const unsigned next = t | (1u << b);
            unsigned n = 0;
#pragma unroll
            for (int i = 0; i < kKeys / 32; ++i) n += mine[i] >= next;
            n = __reduce_add_sync(0xffffffffu, n);
            if (n >= (unsigned)kk) t = next;
            if (n == (unsigned)kk) break;
        }
    }
    if (lane == 0) sm.bound = t;
}

// The elements of the part that reach T0 go to sm.cand: their groups are listed, and the groups'
// vectors read again, dealt to all threads (lists that overflow are left to select_exact: n_cand says
// so).  Up to four loads per thread are in flight at once: with each warp reading its own threads'
// groups one after the other, k = 64 of 50264 took 11300 cycles here.
template <typename T, int TH, int U>
__device__ __forceinline__ void gather(const Row<T>& row, int j0, int j1, unsigned thread_key, const FwdParams& p,
                                       const uint16_t* gmax, unsigned bound, FwdList& sm) {
    constexpr int E = DT<T>::kEPV, B = 4;
    const int tid = threadIdx.x;
    const float t0 = value_of(bound << 16);
    if (bound != 0) {
        if (thread_key >= bound) {
            unsigned mine = 0;  // this thread's groups
#pragma unroll 4
            for (int g = 0; g < p.groups; ++g) mine |= (gmax[g * TH + tid] >= bound ? 1u : 0u) << g;
            int at = atomicAdd(&sm.n_list, __popc(mine));
            for (; mine; mine &= mine - 1, ++at)
                if (at < kCand) sm.list[at] = (uint16_t)((__ffs((int)mine) - 1) * TH + tid);
        }
        __syncthreads();
    }
    const int per = p.group_chunks * U;
    const int n_list = bound != 0 ? sm.n_list : 0;
    const int tasks = bound == 0 ? j1 - j0 : n_list <= kCand ? n_list * per : 0;
    if (n_list > kCand && tid == 0) sm.n_cand = kCand + 1;
    for (int i = tid; i < tasks; i += B * TH) {
        uint4 v[B];
        int j[B];
#pragma unroll
        for (int q = 0; q < B; ++q) {
            const int task = i + q * TH;
            j[q] = j1;
            if (task < tasks) {
                if (bound == 0) {
                    j[q] = j0 + task;
                } else {
                    const int entry = sm.list[task / per];
                    j[q] = j0 + (entry / TH * per + task % per) * TH + entry % TH;
                }
            }
        }
        // whole vectors first, all in flight together; the row's first and last are put together after
#pragma unroll
        for (int q = 0; q < B; ++q) {
            v[q] = make_uint4(0, 0, 0, 0);
            if (j[q] < j1 && j[q] >= row.lo && j[q] < row.hi) v[q] = ldg_stream(row.base + j[q]);
        }
#pragma unroll
        for (int q = 0; q < B; ++q)
            if (j[q] < j1 && (j[q] < row.lo || j[q] >= row.hi)) v[q] = row.partial(j[q]);
#pragma unroll
        for (int q = 0; q < B; ++q) {
            if (j[q] >= j1) continue;
            float x[E];
            unpack<T>(v[q], x);
            unsigned hit = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) hit |= (bound == 0 || x[e] >= t0 ? 1u : 0u) << e;
            if (j[q] < row.lo || j[q] >= row.hi)
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (!row.inside(row.at(j[q], e))) hit &= ~(1u << e);
            if (hit) {
                int at = atomicAdd(&sm.n_cand, __popc(hit));
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (hit >> e & 1) {
                        if (at < kCand) sm.cand[at] = entry_of(x[e], row.at(j[q], e));
                        ++at;
                    }
            }
        }
    }
}

// How many of n keys are larger.
__device__ __forceinline__ int rank_among(const uint64_t* keys, int n, uint64_t key) {
    int rank = 0;
#pragma unroll 8
    for (int q = 0; q < n; ++q) rank += keys[q] > key;
    return rank;
}

// Stores into another block's shared memory.
__device__ __forceinline__ void st_cluster64(uint32_t addr, uint64_t v) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}
__device__ __forceinline__ void st_cluster32(uint32_t addr, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

template <typename T, int TH, int U, int MINB, bool TOP>
__global__ void __launch_bounds__(TH, MINB) k1_score_kernel(FwdParams p) {
    extern __shared__ __align__(16) unsigned char raw[];
    FwdSums<TH>& sums = *reinterpret_cast<FwdSums<TH>*>(raw);
    Meet& meet = *reinterpret_cast<Meet*>(raw + sizeof(FwdSums<TH>));  // only in a cluster
    FwdList& sm = *reinterpret_cast<FwdList*>(raw + sizeof(FwdSums<TH>) + (p.cluster > 1 ? sizeof(Meet) : 0));
    uint16_t* gmax = reinterpret_cast<uint16_t*>(&sm + 1);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = p.cluster > 1 ? (int)ring::cluster_rank() : 0;
    const int64_t r = p.cluster > 1 ? blockIdx.x / p.cluster : blockIdx.x;
    if (p.cluster > 1) ring::cluster_arrive();
    pdl_wait();
    pdl_trigger();
    const Row<T> row(reinterpret_cast<const T*>(p.logits) + p.lay.offset(r), p.vocab);
    const int j0 = min(row.n, rank * p.slice), j1 = min(row.n, j0 + p.slice);
    const float c = p.scale * kLog2e;

    const int64_t id = rank == 0 && tid < p.n_ids ? p.ids[r * p.n_ids + tid] : -1;

    State st;
    st.init();
    unsigned own = 0, odd = 0;  // keys of the thread's maximum, and of that of its groups of odd number
    auto key16 = [](float m) { return key_of(m) >> 16; };
    {
        int g = 0, left = p.group_chunks;
        float gm = -INFINITY;
        uint4 next[U];
        auto fetch = [&](int j) {
            if (j >= row.lo && j + U * TH <= min(j1, row.hi)) {
#pragma unroll
                for (int u = 0; u < U; ++u) next[u] = ldg_stream(row.base + j + tid + u * TH);
            } else if (j < j1) {
                row.template load<U>(next, j + tid, TH, j1);
            }
        };
        fetch(j0);
        for (int j = j0; j < j1; j += U * TH) {
            uint4 v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) v[u] = next[u];
            fetch(j + U * TH);  // in flight while this chunk is added
            const float mc = add_chunk<T, U>(v, st, c);
            if constexpr (TOP) {
                gm = fmax_nan(gm, mc);
                if (--left == 0 || j + U * TH >= j1) {
                    const unsigned key = key16(gm);
                    gmax[g * TH + tid] = (uint16_t)key;
                    own = max(own, key);
                    if (g & 1) odd = max(odd, key);
                    ++g;
                    left = p.group_chunks;
                    gm = -INFINITY;
                }
            }
        }
        if constexpr (TOP) {
            for (; g < p.groups; ++g) gmax[g * TH + tid] = 0;
            // one key per thread, or two where that makes too few; what is masked bounds nothing
            auto real = [&](unsigned key) { return key > key16(Floor<T>::value) ? (uint16_t)key : (uint16_t)0; };
            if constexpr (TH < kKeys) {
                unsigned even = 0;
                for (int q = 0; q < p.groups; q += 2) even = max(even, (unsigned)gmax[q * TH + tid]);
                sm.keys[tid] = real(even);
                sm.keys[TH + tid] = real(odd);
            } else {
                sm.keys[tid] = real(own);
            }
        }
    }

    // the given token's logit, in flight until the row's values are written
    const float xid = row.inside(id) ? DT<T>::load1(row.p + id) : 0.f;

    // the block's sums, relative to its maximum; one warp looks for the bound meanwhile
    const bool empty = st.m <= Floor<T>::value;
    if (lane == 0) sums.wmax[warp] = key_of(empty ? -INFINITY : st.m);
    if (TOP && tid == 0) sm.n_cand = sm.n_list = 0;
    __syncthreads();
    RowPartial part;
    {
        unsigned m = sums.wmax[0];
#pragma unroll
        for (int i = 1; i < TH / 32; ++i) m = max(m, sums.wmax[i]);
        part.m = value_of(m);
        double z = 0.0, t = 0.0;
        if (!empty) {
            const float dm = fmax_nan(st.m - part.m, kFar);
            const double f = dm == 0.f ? 1.f : ex2(dm * c);
            z = f * st.z64();
            t = f * st.t64() + f * (double)dm * st.z64();
        }
        z = warp_sum(z);
        t = warp_sum(t);
        if (lane == 0) {
            sums.wz[warp] = z;
            sums.wt[warp] = t;
        }
    }
    // elements of the part, and the entries wanted of it
    const int64_t elements = max((int64_t)0, min(row.vocab, row.at(j1, 0)) - max((int64_t)0, row.at(j0, 0)));
    const int kk = (int)min((int64_t)p.k, elements);
    if constexpr (TOP)
        if (warp == 0) find_bound<TH>(kk, sm);
    __syncthreads();
    part.z = part.t = 0.0;
#pragma unroll
    for (int i = 0; i < TH / 32; ++i) {
        part.z += sums.wz[i];
        part.t += sums.wt[i];
    }
    part.pad = 0.f;
    if constexpr (!std::is_same<T, __half>::value) {  // whose values lie close enough
        if (isnan(part.t) && part.m - part.m == 0.f) {  // uniform
            const double t = warp_sum(far_sum<T, TH>(row.p, p.vocab, j0, j1, part.m, c));
            __syncthreads();
            if (lane == 0) sums.wt[warp] = t;
            __syncthreads();
            part.t = 0.0;
            for (int i = 0; i < TH / 32; ++i) part.t += sums.wt[i];
        }
    }
    // a NaN or +inf somewhere: no list either, what cannot be ordered must not reach one
    const bool sound = part.m < INFINITY;
    const double s = (double)p.scale;
    // log-probabilities are s (x - m) - log Z: beside s m, which a low temperature makes large, log Z would be lost
    double log_z = p.cluster > 1 ? 0.0 : log(part.z);
    int n = 0;
    if constexpr (TOP) {
        if (sound && kk > 0) {
            const unsigned bound = sm.bound;
            const bool all = bound == 0 && elements > kCand;
            if (!all) gather<T, TH, U>(row, j0, j1, own, p, gmax, bound, sm);
            __syncthreads();
            n = sm.n_cand;
            if (all || n > kCand) {  // uniform
                __syncthreads();
                select_exact<T, TH>(row, j0, j1, kk, sm);
                n = kk;
            }
        }
    }

    auto logprob = [&](float x) { return (float)(s * ((double)x - (double)part.m) - log_z); };
    auto emit = [&](int place, uint64_t key) {
        p.top_ids[r * p.k + place] = (int64_t)(uint32_t)~(uint32_t)key;
        p.top_logprobs[r * p.k + place] = logprob(value_of((uint32_t)(key >> 32)));
    };
    if (p.cluster == 1) {
        if constexpr (TOP)
            for (int i = tid; i < n; i += TH) {
                const uint64_t key = sm.cand[i];
                const int place = rank_among(sm.cand, n, key);
                if (place < kk) emit(place, key);
            }
    } else {
        // every block writes its sums and its list, sorted, into the first one's shared memory
        ring::cluster_wait();  // which runs by now
        const uint32_t to = ring::mapa(ring::saddr(&meet), 0);
        const uint32_t base = ring::saddr(&meet);
        if constexpr (TOP)
            for (int i = tid; i < n; i += TH) {
                const uint64_t key = sm.cand[i];
                const int place = rank_among(sm.cand, n, key);
                if (place < kk) st_cluster64(to + (ring::saddr(&meet.list[rank][place]) - base), key);
            }
        if (tid == 0) {
            st_cluster64(to + (ring::saddr(&meet.part[rank].z) - base), (uint64_t)__double_as_longlong(part.z));
            st_cluster64(to + (ring::saddr(&meet.part[rank].t) - base), (uint64_t)__double_as_longlong(part.t));
            st_cluster32(to + (ring::saddr(&meet.part[rank].m) - base), __float_as_uint(part.m));
            st_cluster32(to + (ring::saddr(&meet.n[rank]) - base), sound ? (uint32_t)kk : 0u);
        }
        ring::cluster_sync();
        if (rank != 0) return;
        float M = meet.part[0].m;
        int total = meet.n[0];
        for (int q = 1; q < p.cluster; ++q) {
            M = fmax_nan(M, meet.part[q].m);
            total += meet.n[q];
        }
        part.z = part.t = 0.0;
        for (int q = 0; q < p.cluster; ++q) {
            const float m = meet.part[q].m;
            if (m != -INFINITY) {
                const float dm = fmax_nan(m - M, kFar);
                const double f = dm == 0.f ? 1.f : ex2(dm * c);
                part.z += f * meet.part[q].z;
                part.t += f * meet.part[q].t + f * (double)dm * meet.part[q].z;
            }
        }
        part.m = M;
        log_z = log(part.z);
        if constexpr (TOP) {
            if (M < INFINITY)
                for (int i = tid; i < p.cluster * p.k; i += TH) {
                    const int q = i / p.k, at = i - q * p.k;
                    if (at >= meet.n[q]) continue;
                    const uint64_t key = meet.list[q][at];
                    int place = 0;
                    for (int o = 0; o < p.cluster; ++o) {
                        // entries of list o before this one: counted, or by bisection of long lists
                        if (p.k <= 32) {
                            place += rank_among(meet.list[o], meet.n[o], key);
                        } else {
                            int lo = 0, hi = meet.n[o];
                            while (lo < hi) {
                                const int mid = (lo + hi) >> 1;
                                if (meet.list[o][mid] > key)
                                    lo = mid + 1;
                                else
                                    hi = mid;
                            }
                            place += lo;
                        }
                    }
                    if (place < p.k) emit(place, key);
                }
        }
    }

    // the row's values
    const bool none = part.m == -INFINITY;  // nothing above the floor
    const double l = s * (double)part.m + log_z;
    const bool fine = !none && part.m < INFINITY && l - l == 0.0;
    if (tid == 0) {
        p.lse[r] = fine ? (float)l : none ? -INFINITY : NAN;
        if (p.lse_rest) p.lse_rest[r] = fine ? (float)(l - (double)(float)l) : 0.f;
        p.entropy[r] = fine ? (float)(log_z - s * part.t / part.z) : NAN;
    }
    if (tid < p.n_ids) p.logprobs[r * p.n_ids + tid] = fine ? logprob(xid) : NAN;
    for (int i = tid + TH; i < p.n_ids; i += TH) {
        const int64_t e = p.ids[r * p.n_ids + i];
        const float x = row.inside(e) ? DT<T>::load1(row.p + e) : 0.f;
        p.logprobs[r * p.n_ids + i] = fine ? logprob(x) : NAN;
    }
    if constexpr (TOP) {
        if (fine) return;
        __syncthreads();  // in place of what the block may have written
        for (int i = tid; i < p.k; i += TH) {
            p.top_ids[r * p.k + i] = -1;
            p.top_logprobs[r * p.k + i] = NAN;
        }
    }
}

// ------------------------------------------------------------------------------------
// Backward
// ------------------------------------------------------------------------------------
struct BwdParams {
    const void* logits;
    RowLayout lay;
    int64_t vocab;
    float scale;
    const int64_t* ids;      // [n, n_ids]
    const float* g_ids;      // [n, n_ids], NULL: none
    const int64_t* top_ids;  // [n, k]
    const float* g_top;      // [n, k], NULL: none
    int n_ids, k;            // 0 without gradient
    const float* lse;
    const float* lse_rest;   // NULL: 0
    const float* entropy;
    const float* g_entropy;  // NULL: none
    const float* g_lse;      // NULL: none
    void* d;                 // rows d_stride elements apart
    int64_t d_stride;
    int parts;               // blocks per row
    int slice;               // vectors per block
};

// A log-probability whose weight is 0 in fp32, whatever lse_rest (at most 64 where it matters) adds.
constexpr float kNoWeight = -1024.f;

constexpr int kBwdThreads = 256;
constexpr int UB = 4;

// From this |lse| on, the values next to a row's maximum m lie 2^-24 |m| s >= 128 or more below it: their
// weight is 0 in fp32, and those equal to m share it all.  lse and lse_rest together then no longer hold log Z, but
// they hold m (log Z is at most 21, less than half of fp32's spacing at s m), and the entropy is log Z.
constexpr float kOnlyMax = 2147483648.f;  // 2^31

// dL/dx of a vector of logits that no list names.
struct BwdRow {
    float s, nl, nr, c0, ge;  // s, -lse, -lse_rest log2 e, s (g_lse - sum g - g_H (H - lse_rest)), s g_H
};
template <typename T>
__device__ __forceinline__ uint4 grad_vector(uint4 v, const BwdRow& q) {
    constexpr int E = DT<T>::kEPV;
    float x[E];
    unpack<T>(v, x);
    float2 g[E / 2];
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
        // d = s x - lse is rounded by 2^-24 of itself; lse's own rounding, which at a low temperature is
        // many times that, is made good in the exponent and in c0
        float2 d = fma2(make_float2(x[2 * i], x[2 * i + 1]), splat(q.s), splat(q.nl));
        // far below the maximum the weight is 0; d stays small, so that its product with s g_H is finite
        d = make_float2(fmax_nan(d.x, kNoWeight), fmax_nan(d.y, kNoWeight));
        const float2 a = fma2(d, splat(kLog2e), splat(q.nr));
        g[i] = mul2(make_float2(ex2(a.x), ex2(a.y)), fma2(d, splat(-q.ge), splat(q.c0)));
    }
    if constexpr (sizeof(T) == 4)
        return make_uint4(__float_as_uint(g[0].x), __float_as_uint(g[0].y), __float_as_uint(g[1].x),
                          __float_as_uint(g[1].y));
    else
        return make_uint4(DT<T>::from_f2(g[0]), DT<T>::from_f2(g[1]), DT<T>::from_f2(g[2 % (E / 2)]),
                          DT<T>::from_f2(g[3 % (E / 2)]));
}

// Such a row's maximum, and vectors [j0, j1) of its gradient (each element as one: such rows are rare).
__device__ __forceinline__ float only_max_of(float lse, float rest, float scale) {
    return (float)(((double)lse + (double)rest) / (double)scale);
}
template <typename T>
__device__ __noinline__ void grad_only_max(const T* p, int64_t vocab, T* out, int j0, int j1, float m, float equal) {
    constexpr int E = DT<T>::kEPV;
    const Row<T> row(p, vocab);
    for (int j = j0 + threadIdx.x; j < j1; j += kBwdThreads) {
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const int64_t e = row.at(j, i);
            if (row.inside(e)) DT<T>::store1(out + e, DT<T>::load1(p + e) == m ? equal : 0.f);
        }
    }
}

constexpr int kBwdBlocks = 4;

template <typename T>
__global__ void __launch_bounds__(kBwdThreads, kBwdBlocks) k1_score_bwd_kernel(BwdParams p) {
    constexpr int E = DT<T>::kEPV, TH = kBwdThreads;
    __shared__ double wsum[TH / 32];
    extern __shared__ __align__(16) unsigned char raw[];
    int64_t* ids = reinterpret_cast<int64_t*>(raw);
    float* gs = reinterpret_cast<float*>(ids + p.n_ids + p.k);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t r = blockIdx.x / p.parts;
    const int rank = (int)(blockIdx.x - r * p.parts);
    pdl_wait();
    pdl_trigger();
    const Row<T> row(reinterpret_cast<const T*>(p.logits) + p.lay.offset(r), p.vocab);
    T* out = reinterpret_cast<T*>(p.d) + r * p.d_stride;
    const int j0 = min(row.n, rank * p.slice), j1 = min(row.n, j0 + p.slice);
    const int n = p.n_ids + p.k;
    const bool same = ((reinterpret_cast<uintptr_t>(out) ^ reinterpret_cast<uintptr_t>(row.p)) & 15u) == 0;
    // a whole chunk inside the row, stored as vectors (uniform)
    auto whole = [&](int j) { return same && j >= row.lo && j + UB * TH <= min(j1, row.hi); };
    uint4 v[UB];
    auto fetch = [&](int j) {
        if (whole(j)) {
#pragma unroll
            for (int u = 0; u < UB; ++u) v[u] = ldg_stream(row.base + j + tid + u * TH);
        }
    };
    fetch(j0);
    const float ge = p.g_entropy ? p.g_entropy[r] : 0.f, gl = p.g_lse ? p.g_lse[r] : 0.f;
    double sum = 0.0;
    bool any = ge != 0.f || gl != 0.f;  // true for a NaN
    for (int i = tid; i < n; i += TH) {
        const bool given = i < p.n_ids;
        ids[i] = given ? p.ids[r * p.n_ids + i] : p.top_ids[r * p.k + i - p.n_ids];
        const float g = given ? p.g_ids[r * p.n_ids + i] : p.g_top[r * p.k + i - p.n_ids];
        gs[i] = g;
        sum += (double)g;
        any |= g != 0.f;
    }
    sum = warp_sum(sum);
    if (lane == 0) wsum[warp] = sum;
    any = __syncthreads_or(any);
    sum = 0.0;
#pragma unroll
    for (int i = 0; i < TH / 32; ++i) sum += wsum[i];
    const float lse = p.lse[r], h = p.entropy[r];
    BwdRow q;
    q.s = p.scale;
    const float rest = p.lse_rest ? p.lse_rest[r] : 0.f;
    q.nr = -rest * kLog2e;
    q.nl = lse - lse == 0.f ? -lse : NAN;  // a row without a distribution
    q.ge = p.scale * ge;
    // entropy: only where it has a gradient, so that a row without one needs no finite entropy
    const double c0 = (double)gl - sum - (ge != 0.f ? (double)ge * ((double)h - (double)rest) : 0.0);
    q.c0 = (float)((double)p.scale * c0);
    uint4* ov = reinterpret_cast<uint4*>(out - row.shift);
    auto store = [&](int j, uint4 v) {
        if (same && j >= row.lo && j < row.hi) {
            stg_stream(ov + j, v);
        } else {
            float x[E];
            unpack<T>(v, x);
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const int64_t e = row.at(j, i);
                if (row.inside(e)) DT<T>::store1(out + e, x[i]);
            }
        }
    };
    if (!any) {  // nothing asked of this row (a padded position): zeros whatever it holds
        for (int j = j0 + tid; j < j1; j += TH) store(j, make_uint4(0, 0, 0, 0));
        return;
    }
    const bool only_max = fabsf(lse) >= kOnlyMax && lse - lse == 0.f;  // a low temperature
    if (only_max)
        grad_only_max<T>(row.p, p.vocab, out, j0, j1, only_max_of(lse, rest, p.scale),
                         (float)((double)p.scale * exp(-(double)h) * ((double)gl - sum)));
    for (int j = only_max ? j1 : j0; j < j1; j += UB * TH) {
        if (whole(j)) {
            uint4 o[UB];
#pragma unroll
            for (int u = 0; u < UB; ++u) o[u] = v[u];
            fetch(j + UB * TH);
#pragma unroll
            for (int u = 0; u < UB; ++u) stg_stream(ov + j + tid + u * TH, grad_vector<T>(o[u], q));
        } else {
            uint4 o[UB];
            row.template load<UB>(o, j + tid, TH, j1);
            fetch(j + UB * TH);
#pragma unroll
            for (int u = 0; u < UB; ++u)
                if (j + tid + u * TH < j1) store(j + tid + u * TH, grad_vector<T>(o[u], q));
        }
    }
    __syncthreads();  // the named tokens' own gradients replace what the block wrote there
    const int64_t e0 = row.at(j0, 0), e1 = row.at(j1, 0);
    for (int i = tid; i < n; i += TH) {
        const int64_t e = ids[i];
        if (!row.inside(e) || e < e0 || e >= e1) continue;
        // a token named more than once is written by its first entry, with all entries' gradients
        double mine = 0.0, others = 0.0;
        bool first = true;
        for (int o = 0; o < n; ++o) {
            const bool eq = ids[o] == e;
            if (eq && o < i) first = false;
            (eq ? mine : others) += (double)gs[o];
        }
        if (!first) continue;
        const float x = DT<T>::load1(row.p + e);
        const double lp = !only_max ? (double)p.scale * (double)x - ((double)-q.nl + (double)rest)
                          : x == only_max_of(lse, rest, p.scale) ? -(double)h
                                                                 : -INFINITY;
        const double pr = exp(lp);
        double g = mine * -expm1(lp) + pr * ((double)gl - others);
        if (ge != 0.f && pr > 0.0) g -= (double)ge * pr * (lp + (double)h);
        DT<T>::store1(out + e, (float)((double)p.scale * g));
    }
}

}  // namespace score
}  // namespace k1
