// k1_sample.cuh -- one token per row of logits from a given uniform number, with
// temperature, top-k, top-p and min-p, and the token's log-probability.
//
//   y_i = x_i * s (s = 1/T in fp32),  m = max y,  w_i = exp(y_i - m) in fp32;  S = sum w
//   order: y downwards, the lowest index first among equals
//   top-k  keeps the first k;  top-p, of those (mass Z), the shortest prefix with mass >=
//   p Z;  min-p keeps w_i >= min_p;  the first one always stays
//   token: the first kept index, in index order, at which the kept mass up to it exceeds u C
//   (C: the kept mass);  logprob = y - m - log S,  kept logprob = y - m - log C
//
// Sums of weights decide which token is drawn, so they are taken far beyond fp32, whatever the
// weights' sizes: a weight is split into three parts, two of which add exactly in fp32, and goes
// to fp64 once per 16-byte vector (Mass).  What is left depends on how a row is cut, at about 1e-13
// of S; a list's sums (below) are within 2^-40 of its mass.  So the same row gives the same token at
// any address and in any batch unless u (or top-p) lies within about 1e-12 of a boundary.
//
// A cluster of 1 to 8 blocks owns a row: every block holds its part of the row in shared
// memory, so the logits cross HBM once whatever the filters ask for, and all later passes
// (weights, histograms, thresholds) run from there.  The blocks push maxima, sums and
// thresholds into each other's shared memory.  Two to five blocks per SM: one row's passes
// run while another row's loads are in flight.  (Rows too long for a cluster's shared memory
// are read again from global memory in each pass.)
//
//   whole rows (no filter)  load + max, sum, draw.
//   short lists             Each thread keeps the maxima of four groups of its elements.  A
//                           histogram of those maxima gives a bound that at least K elements
//                           reach, and few more; the pass that sums the weights puts them
//                           into a list, and the row's first block applies the filters to it
//                           (thresholds by histograms of the list's keys).  Serves top-k up
//                           to kListK and every top-p whose nucleus lies within the list.
//   selection               Otherwise the threshold is found by histograms over all elements:
//                           bins of equal width in y (counts for top-k, masses for top-p,
//                           the latter in steps of 2^-12 of the bin's middle weight, so only
//                           a guide), then the bin's exact limits and its elements as a
//                           list, and again inside the bin while it has too many.
//
// Measured on B200 (us; bf16, N(0, 3^2) with half of the rows peaked, unless noted): no
// filter, 512 x 152064 82 (1.89 TB/s; its bytes alone 24) and 1 x 151936 7.5; 512 x 152064 top-k 50
// 164, top-k 1000 233, top-p 0.9 553; 567 x 128256 fp32 top-k 40 top-p 0.82 235; 64 x 128256
// fp32 with mixed settings 61; 128 x 50257 fp16 top-p 0.95 59.  Without a filter the time goes to
// instructions, about 24 per element by the counters, most of them for the weights (expf, the exact
// split, conversions), and to the exchanges; loading alone takes 30 us of the 82.  With filters the
// chain of short phases in each block is the limit: two blocks per SM cannot hide all of it.
//
// A row that holds a NaN or +inf, or nothing above -inf, has no distribution: token -1 and
// NaN log-probabilities.  So does one whose own settings mean nothing (a temperature that is negative
// or not finite, a negative top-p, a min-p outside [0, 1], a NaN); as numbers for all rows they are
// refused.
#pragma once

#include "k1_common.cuh"
#include "k1_sample_math.cuh"
#include "k1_sync.cuh"

#include <type_traits>

namespace k1 {
namespace sample {

// Threads per block.  With filters the passes after the first are many and short, so a block
// brings more threads; without, a thread's fixed work (the exchanges) counts, and fewer
// threads win.  Measured (512 rows of 152064 bf16, no filter, us; threads x blocks per SM, KB of
// a row per block): 256 x 5, 38 KB 82; 128 x 10, 19 KB 90; 512 x 2, 76 KB 97; 256 x 4, 76 KB 106.
constexpr int kFilterThreads = 512, kFilterBlocks = 2;
constexpr int kPlainThreads = 256, kPlainBlocks = 5;
constexpr int kMaxWarps = 16;
constexpr int THREADS = kFilterThreads;  // of the code that only filters use
constexpr int NB = THREADS;        // histogram bins, one per thread
constexpr int NG = 4;              // groups of elements per thread
constexpr int kListCap = 2048;     // entries of the list
constexpr int kListK = 1024;       // largest top-k that tries the list
constexpr int kNucleusK = 384;     // groups that a list for top-p asks for
constexpr int kMaxCluster = 8;

struct Params {
    const void* logits;
    int64_t n_rows, vocab, row_stride;
    const float* u;
    // per row, or one value for all rows (pointer NULL)
    const float* temperature;
    const int* top_k;
    const float* top_p;
    const float* min_p;
    float scale0;      // fp32(1 / temperature), 1 at temperature 0
    bool greedy0;      // temperature 0
    float top_p0, min_p0;
    int top_k0;
    int64_t* token;
    float* logprob;
    float* kept_logprob;
    int cluster;       // blocks per row
    int slice_vecs;    // 16-byte vectors per block (of the row widened to vector boundaries)
};

// One block's contribution to an exchange between the blocks of a row.
struct Xch {
    double a, b;
    float lo, hi;
    unsigned n, pad;
};

// What every row needs of shared memory, and what only filters need.
struct Smem {
    Xch slot[2][kMaxCluster];  // every block's contribution, written by its owner
    double wsum[kMaxWarps];    // the warps' parts of an exchange
    double wsum_b[kMaxWarps];
    unsigned wn[kMaxWarps];
    float wlo[kMaxWarps], whi[kMaxWarps];
    double logs[2];            // of the whole and the kept mass
};
struct FilterSmem : Smem {
    uint64_t list[kListCap];
    uint64_t sums[NB];    // histogram of the list
    unsigned hist[NB];    // histogram of the block's elements
    double wscan[kMaxWarps];
    uint64_t wsum64[kMaxWarps];
    uint64_t few_key[32], few_word[32];  // kFew
    unsigned few_n;
    uint64_t entry;       // block-wide values
    uint64_t above;
    unsigned found;
    unsigned list_n;
    int pick;
    float tau;            // the threshold, told by the block that finds it
    int told;
    int64_t ilim;
};

template <bool FILTER>
__host__ __device__ constexpr size_t smem_header() {
    return ((FILTER ? sizeof(FilterSmem) : sizeof(Smem)) + 15) & ~(size_t)15;
}

// ------------------------------------------------------------------------------------
// A row's part in one block
// ------------------------------------------------------------------------------------
// The row is widened to 16-byte boundaries: virtual index v = i + shift, shift = elements
// between the boundary at or below the row's start and the start.  Elements outside the row
// read as -inf, which no pass counts.
template <typename T>
__device__ __noinline__ uint4 load_edge(const T* row, int64_t i0, int64_t vocab) {
    constexpr int E = DT<T>::kEPV;
    uint4 v;
    T* e = reinterpret_cast<T*>(&v);
#pragma unroll
    for (int k = 0; k < E; ++k) {
        const int64_t i = i0 + k;
        if (i >= 0 && i < vocab)
            e[k] = row[i];
        else
            DT<T>::store1(e + k, -INFINITY);
    }
    return v;
}

template <typename T, bool RES>
struct Slice {
    static constexpr int E = DT<T>::kEPV;
    const T* row;
    const uint4* base;  // the boundary at or below the block's first element (vectors in
                        // [whole0, whole1) alone may be read through it)
    uint4* buf;         // RES: the slice in shared memory
    int64_t vocab;
    int64_t i0;         // index of the first vector's first element (negative: before the row)
    int nvec;           // the block's vectors
    int whole0, whole1; // those that lie inside the row
    int w0, w1;         // the warp's vectors: contiguous, lanes interleaved

    __device__ __forceinline__ void init(const T* r, int64_t v, int64_t vec0, int slice_vecs) {
        row = r;
        vocab = v;
        const int shift = (int)((reinterpret_cast<uintptr_t>(r) & 15) / sizeof(T));
        i0 = vec0 * E - shift;
        base = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(r) & ~(uintptr_t)15) + vec0;
        const int64_t left = v - i0;  // elements from the first vector to the row's end
        nvec = left <= 0 ? 0 : (int)min((int64_t)slice_vecs, (left + E - 1) / E);
        whole0 = i0 < 0 ? 1 : 0;
        whole1 = left <= 0 ? 0 : (int)min((int64_t)nvec, left / E);
    }
    __device__ __forceinline__ uint4 load_global(int j) const {
        if (j >= whole0 && j < whole1) return ldg_stream(base + j);
        return load_edge<T>(row, i0 + (int64_t)j * E, vocab);
    }
    __device__ __forceinline__ uint4 vec(int j) const {
        if constexpr (RES)
            return buf[j];
        else
            return load_global(j);
    }
    __device__ __forceinline__ int64_t index(int j, int e) const { return i0 + (int64_t)j * E + e; }
};

// y = x * s, rounded.  A packed product (mul2) whose use is a sum or a difference is carried out
// together with it, y never being rounded: the largest element's y - m is then that rounding's error
// instead of 0, and equal y fall into different bins.  An fma whose addend is -0 (which the compiler
// does not know: s is a number it has not seen) is the rounded product and joins nothing.  (Single
// products, __fmul_rn, do as well: 512 x 152064 bf16 83.8 us, 82.3 so.)
template <typename T>
__device__ __forceinline__ void unpack(uint4 v, float s, float (&y)[DT<T>::kEPV]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    const float2 zero = splat(__fmul_rn(s, -0.f));
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            const float2 f = fma2(make_float2(__uint_as_float(w[i]), __uint_as_float(w[i + 1])), splat(s), zero);
            y[i] = f.x;
            y[i + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = fma2(DT<T>::to_f2(w[i]), splat(s), zero);
            y[2 * i] = f.x;
            y[2 * i + 1] = f.y;
        }
    }
}

// Largest element of a set of vectors (NaN if it holds one), in the elements' type: two
// 16-bit elements per instruction.
template <typename T>
struct Peak {
    uint32_t v = sizeof(T) == 4                  ? 0xff800000u
                 : std::is_same_v<T, __half>     ? 0xfc00fc00u
                                                 : 0xff80ff80u;
    __device__ __forceinline__ void add(uint4 x) {
        if constexpr (sizeof(T) == 4)
            v = __float_as_uint(fmax_nan(
                __uint_as_float(v), fmax_nan(fmax_nan(__uint_as_float(x.x), __uint_as_float(x.y)),
                                             fmax_nan(__uint_as_float(x.z), __uint_as_float(x.w)))));
        else
            v = DT<T>::max2(v, DT<T>::max2(DT<T>::max2(x.x, x.y), DT<T>::max2(x.z, x.w)));
    }
    __device__ __forceinline__ float value() const {
        if constexpr (sizeof(T) == 4) {
            return __uint_as_float(v);
        } else {
            const float2 f = DT<T>::to_f2(v);
            return fmax_nan(f.x, f.y);
        }
    }
};
template <typename T>
__device__ __forceinline__ float vec_max(uint4 v) {
    Peak<T> p;
    p.add(v);
    return p.value();
}

// Running sum of weights in [0, 1], two per instruction.  Adding a weight to a sum that is kept
// above 2^10 rounds it to a multiple of 2^-13; how much went in is the sum's difference, and what
// did not, at most 2^-14, is added in the same way to a sum above 2^-9: multiples of 2^-32.  Both
// are exact for as many vectors as they run before they go to fp64.  What is left then, at most
// 2^-33 of a weight, is added in fp32 over four vectors: 2^-50 lost of them at most, whatever the
// weights' sizes.  (Sent to fp64 after every vector, the small parts cost 512 rows of 152064 bf16
// 85 us instead of 81.)
struct Mass {
    static constexpr float kHigh = 0x1p10f, kMid = 0x1.8p-9f;
    float2 hi = make_float2(kHigh, kHigh), mid = make_float2(kMid, kMid), lo = make_float2(0.f, 0.f);
    double sum = 0.0;
    int vectors = 0;
    template <int E>
    __device__ __forceinline__ void add(const float (&w)[E]) {
        // adds x to s and leaves in x what s did not take
        auto take = [](float2& s, float2& x) {
            const float2 t = add2(s, x);
            x = diff2(x, diff2(t, s));
            s = t;
        };
#pragma unroll
        for (int i = 0; i < E; i += 2) {
            float2 x = make_float2(w[i], w[i + 1]);
            take(hi, x);
            take(mid, x);
            lo = add2(lo, x);
        }
        if ((++vectors & 3) == 0) {  // 16 weights per half: mid has moved by 2^-10 at most
            sum += small();
            mid = splat(kMid);
            lo = splat(0.f);
            if (vectors == 256) {  // 1024 weights per half: hi is 2^11 at most
                sum += high();
                hi = splat(kHigh);
                vectors = 0;
            }
        }
    }
    __device__ __forceinline__ double small() const {
        return (double)((mid.x - kMid) + (mid.y - kMid)) + (double)(lo.x + lo.y);
    }
    __device__ __forceinline__ double high() const { return (double)(hi.x - kHigh) + (double)(hi.y - kHigh); }
    __device__ __forceinline__ double total() const { return sum + (small() + high()); }
};

// Order-preserving key of a float (larger value, larger key; -0 and +0 are one).
__device__ __forceinline__ uint32_t key_of(float y) {
    const uint32_t b = __float_as_uint(y + 0.f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

// Below m - kFloor a weight is 0 in fp32, so such elements are neither drawn nor counted.
constexpr float kFloor = 104.f;

// Monotone bins of an interval of y that ends at `top`: of equal width in y (the first
// level: it spreads the elements), or of equal width in the float's key (the levels inside a
// bin: integers, so the interval's ends always fall into different bins).
struct Bins {
    float top, per_unit;
    uint32_t key_top;
    int shift;  // < 0: equal width in y
    __device__ __forceinline__ static Bins linear(float top, float bottom) {
        // an empty range gives +inf: the cap keeps 0 * per_unit a number
        return Bins{top, fminf((float)NB / (top - bottom), 1e30f), 0u, -1};
    }
    __device__ __forceinline__ static Bins keys(float top, float bottom) {
        const uint32_t range = key_of(top) - key_of(bottom);
        return Bins{top, 0.f, key_of(top), max(0, 32 - __clz(range) - 9)};  // NB = 2^9
    }
    // equal width: the bin is this, rounded to the nearest whole number
    __device__ __forceinline__ float place(float y) const {
        return fminf((top - y) * per_unit, (float)(NB - 1));
    }
    __device__ __forceinline__ int of(float y) const {
        return shift < 0 ? __float2int_rn(place(y)) : (int)((key_top - key_of(y)) >> shift);
    }
    // the y that weights of bin b are taken relative to: its middle (equal width), or its top
    __device__ __forceinline__ float base_of(int b) const {
        return shift < 0 ? top - (float)b / per_unit : value_of(key_top - ((uint32_t)b << shift));
    }
};
static_assert(NB == 512, "Bins::keys takes 9 bits");

// ------------------------------------------------------------------------------------
// The blocks of a row
// ------------------------------------------------------------------------------------
template <typename V>
__device__ __forceinline__ V warp_add(V v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// What an exchange carries.
enum Carry : int { A = 1, B = 2, N = 4, RANGE = 8 };

struct Joined {
    double a, b;
    double before;      // sum of a over the blocks of lower rank
    unsigned n;
    unsigned n_before;
    float lo, hi;
};

// Adds a, b, n and joins lo (min) and hi (max, NaN survives) over all threads of all blocks of
// the row, in a fixed order; every thread gets the result.  The warps' parts of a and n stay
// in sm.wsum and sm.wn.  Each block writes its contribution into every block's shared memory,
// so that after one cluster barrier all are at hand.  `phase` alternates between calls: a block
// may write its next contribution while another still reads the last one, and the barrier in
// between keeps it from getting further ahead.
template <int WHAT, int WARPS>
__device__ __forceinline__ Joined exchange(Smem& sm, int& phase, int cluster, int rank, double a, double b,
                                           unsigned n, float lo, float hi) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (WHAT & A) a = warp_add(a);
    if (WHAT & B) b = warp_add(b);
    if (WHAT & N) n = __reduce_add_sync(0xffffffffu, n);
    if (WHAT & RANGE) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = warp_max_nan(hi);
    }
    if (lane == 0) {
        if (WHAT & A) sm.wsum[warp] = a;
        if (WHAT & B) sm.wsum_b[warp] = b;
        if (WHAT & N) sm.wn[warp] = n;
        if (WHAT & RANGE) {
            sm.wlo[warp] = lo;
            sm.whi[warp] = hi;
        }
    }
    __syncthreads();
    if (warp == 0) {
        const int i = lane & (WARPS - 1);  // every WARPS lanes hold all parts
        if (WHAT & A) a = sm.wsum[i];
        if (WHAT & B) b = sm.wsum_b[i];
        if (WHAT & N) n = sm.wn[i];
        if (WHAT & RANGE) {
            lo = sm.wlo[i];
            hi = sm.whi[i];
        }
#pragma unroll
        for (int o = WARPS / 2; o > 0; o >>= 1) {
            if (WHAT & A) a += __shfl_xor_sync(0xffffffffu, a, o);
            if (WHAT & B) b += __shfl_xor_sync(0xffffffffu, b, o);
            if (WHAT & N) n += __shfl_xor_sync(0xffffffffu, n, o);
            if (WHAT & RANGE) {
                lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
                hi = fmax_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
            }
        }
        if (lane < cluster) {
            const uint32_t to = ring::mapa(ring::saddr(&sm.slot[phase][rank]), lane);
            if (WHAT & A)
                asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(to), "d"(a) : "memory");
            if (WHAT & B)
                asm volatile("st.shared::cluster.f64 [%0 + 8], %1;" ::"r"(to), "d"(b) : "memory");
            if (WHAT & RANGE)
                asm volatile("st.shared::cluster.v2.f32 [%0 + 16], {%1, %2};" ::"r"(to), "f"(lo), "f"(hi)
                             : "memory");
            if (WHAT & N) asm volatile("st.shared::cluster.u32 [%0 + 24], %1;" ::"r"(to), "r"(n) : "memory");
        }
    }
    ring::cluster_sync();
    Joined t = {0.0, 0.0, 0.0, 0, 0, INFINITY, -INFINITY};
#pragma unroll 4
    for (int r = 0; r < cluster; ++r) {
        const Xch& x = sm.slot[phase][r];
        if (r == rank) {
            t.before = t.a;
            t.n_before = t.n;
        }
        if (WHAT & A) t.a += x.a;
        if (WHAT & B) t.b += x.b;
        if (WHAT & N) t.n += x.n;
        if (WHAT & RANGE) {
            t.lo = fminf(t.lo, x.lo);
            t.hi = fmax_nan(t.hi, x.hi);
        }
    }
    phase ^= 1;
    return t;
}

// Adds the blocks' histograms: thread b returns bin b of the row.  A block may write its
// histogram again after the next exchange.
__device__ __forceinline__ unsigned row_bin(FilterSmem& sm, int cluster) {
    ring::cluster_sync();
    unsigned v = 0;
    const uint32_t a = ring::saddr(&sm.hist[threadIdx.x]);
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r) {
        if (r < cluster) {
            unsigned x;
            asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(x) : "r"(ring::mapa(a, r)) : "memory");
            v += x;
        }
    }
    return v;
}

// Inclusive prefix sum over the block's threads.
template <typename V>
__device__ __forceinline__ V block_scan(V v, V* warp_sums) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const V t = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += t;
    }
    __syncthreads();
    if (lane == 31) warp_sums[warp] = v;
    __syncthreads();
    V base = 0;
#pragma unroll
    for (int i = 0; i < THREADS / 32 - 1; ++i) base += i < warp ? warp_sums[i] : V(0);
    return base + v;
}

// The first bin whose prefix (thread b's, growing with b) reaches what is asked for; the last
// one if none does.
__device__ __forceinline__ int first_bin(bool reached) { return min(__syncthreads_count(!reached), NB - 1); }

// ------------------------------------------------------------------------------------
// The list: entries of the row (key of y, ~index), in the row's first block
// ------------------------------------------------------------------------------------
constexpr int PER = kListCap / THREADS;  // entries per thread
static_assert(PER == 4, "block sums of a list's words add four");

__device__ __forceinline__ uint64_t entry(float y, int64_t index) {
    return ((uint64_t)key_of(y) << 32) | (uint32_t)~(uint32_t)index;
}
__device__ __forceinline__ float entry_value(uint64_t e) { return value_of((uint32_t)(e >> 32)); }
__device__ __forceinline__ int64_t entry_index(uint64_t e) { return (int64_t)(uint32_t)~(uint32_t)e; }

// The elements of vector j that `hits` marks, one bit each, into this block's own list, one
// atomic per warp (whose lanes all call) and round; entries past the list's end are only
// counted.  f(y) for each.
template <int E, typename F>
__device__ __forceinline__ void append(FilterSmem& sm, unsigned hits, const float (&y)[E], int64_t index, F f) {
    const unsigned lane = threadIdx.x & 31;
    for (unsigned some; (some = __ballot_sync(0xffffffffu, hits != 0)) != 0; hits &= hits - 1) {
        unsigned pos = 0;
        if (lane == 0) pos = atomicAdd(&sm.list_n, (unsigned)__popc(some));
        pos = __shfl_sync(0xffffffffu, pos, 0) + __popc(some & ((1u << lane) - 1));
        if (hits) {
            const int at = __ffs(hits) - 1;
            float v = 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) v = at == e ? y[e] : v;
            if (pos < (unsigned)kListCap) sm.list[pos] = entry(v, index + at);
            f(v);
        }
    }
}

// The blocks' lists (n_before entries in lower ranks, kListCap in all at most) joined in the
// first block.
__device__ __forceinline__ void join_lists(FilterSmem& sm, int rank, unsigned n_before) {
    if (rank > 0) {
        const uint32_t to = ring::mapa(ring::saddr(&sm.list[0]), 0) + n_before * 8;
        for (unsigned i = threadIdx.x; i < sm.list_n; i += THREADS)
            asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(to + i * 8), "l"(sm.list[i]) : "memory");
    }
    ring::cluster_sync();
}

// One thread tells every block of the row the threshold; they read it after a cluster barrier.
__device__ __forceinline__ void tell(FilterSmem& sm, int cluster, float tau, int64_t ilim) {
    for (int r = 0; r < cluster; ++r) {
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(ring::mapa(ring::saddr(&sm.tau), r)), "f"(tau)
                     : "memory");
        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(ring::mapa(ring::saddr(&sm.told), r)), "r"(1)
                     : "memory");
        asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(ring::mapa(ring::saddr(&sm.ilim), r)), "l"(ilim)
                     : "memory");
    }
}

__device__ __forceinline__ uint64_t block_sum64(FilterSmem& sm, uint64_t v) {
    v = warp_add(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sm.wsum64[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0;
    for (int i = 0; i < kFilterThreads / 32; ++i) v += sm.wsum64[i];
    return v;
}

// Of the block's entries (PER to a thread, distinct keys, a word of 0 for none), largest key
// first: the key at which the weight added up so far first reaches `target`; the entries' keys
// lie in [lo, hi].  `lo`, which keeps them all, where none does (a target of 0 or more than their
// whole weight).  Each round adds the words up in 512 bins of the remaining key range and keeps
// the crossing bin, until that holds few entries: one round for spread keys; kRounds leave one key
// to a bin.
constexpr int kFew = 32;           // one to a lane
constexpr int kRounds = (64 + 8) / 9;
__device__ __forceinline__ uint64_t select_entry(FilterSmem& sm, const uint64_t (&key)[PER],
                                                 const uint64_t (&word)[PER], uint64_t lo, uint64_t hi,
                                                 uint64_t target) {
    uint64_t above = 0;
    const uint64_t none = lo;
    for (int round = 0; round < kRounds; ++round) {
        const int shift = max(0, 64 - __clzll((long long)(hi - lo)) - 9);
        sm.sums[threadIdx.x] = 0;
        if (threadIdx.x == 0) {
            sm.found = 0;
            sm.entry = none;
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < PER; ++r)
            if (word[r] && key[r] >= lo && key[r] <= hi)
                atomicAdd(reinterpret_cast<unsigned long long*>(&sm.sums[(hi - key[r]) >> shift]),
                          (unsigned long long)word[r]);
        __syncthreads();
        const uint64_t mine = sm.sums[threadIdx.x];
        const uint64_t upto = block_scan(mine, sm.wsum64);
        // the one bin that holds entries and crosses
        const uint64_t before = above + word_weight(upto - mine);
        if (mine && before < target && above + word_weight(upto) >= target) {
            sm.pick = threadIdx.x;
            sm.above = before;
            sm.found = (unsigned)(mine & ((1u << kCountBits) - 1));
        }
        __syncthreads();
        if (sm.found == 0) break;  // none crosses
        const uint64_t top = hi - ((uint64_t)sm.pick << shift);
        const uint64_t bottom = top - (((uint64_t)1 << shift) - 1);
        lo = bottom > top || bottom < lo ? lo : bottom;
        hi = top;
        above = sm.above;
        if (sm.found <= kFew) break;
        __syncthreads();
    }
    // the bin's entries, one to a lane, against one another
#pragma unroll
    for (int r = 0; r < PER; ++r)
        if (word[r] && key[r] >= lo && key[r] <= hi) {
            const unsigned i = atomicAdd(&sm.few_n, 1u);
            if (i < kFew) {
                sm.few_key[i] = key[r];
                sm.few_word[i] = word_weight(word[r]);
            }
        }
    __syncthreads();
    if (threadIdx.x < 32) {
        const unsigned n = min(sm.found, (unsigned)kFew), lane = threadIdx.x;
        const uint64_t k = lane < n ? sm.few_key[lane] : 0, w = lane < n ? sm.few_word[lane] : 0;
        uint64_t before = above;
        for (unsigned i = 0; i < n; ++i) before += sm.few_key[i] > k ? sm.few_word[i] : 0;
        if (w && before < target && before + w >= target) sm.entry = k;
    }
    __syncthreads();
    const uint64_t e = sm.entry;
    if (threadIdx.x == 0) sm.few_n = 0;
    __syncthreads();
    return e;
}

// ------------------------------------------------------------------------------------
// The kernel
// ------------------------------------------------------------------------------------
// What is kept so far: y above tau, and y equal to tau up to index ilim.
struct Keep {
    float tau;
    int64_t ilim;
    float min_p;  // a weight's lower limit, 0: off
    // Whether y >= tau is kept (of equals, those up to ilim).
    template <typename SL>
    __device__ __forceinline__ bool allows(float y, const SL& sl, int j, int e) const {
        return y != tau || sl.index(j, e) <= ilim;
    }
};

template <typename T, bool RES, int TH>
struct Row {
    static constexpr int E = DT<T>::kEPV;
    static constexpr int WARPS = TH / 32;
    Slice<T, RES> sl;
    float s, m;
    int cluster, rank, phase;

    // f(j, y): every vector of the warp's part, lanes interleaved
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        for (int j = sl.w0 + (threadIdx.x & 31); j < sl.w1; j += 32) {
            float y[E];
            unpack<T>(sl.vec(j), s, y);
            f(j, y);
        }
    }

    // The same with all lanes of a warp at every step, for what they do together, and the
    // vector as it is; past the part's end it holds -inf.
    template <typename F>
    __device__ __forceinline__ void each_vector(F f) const {
        constexpr uint32_t kNone = sizeof(T) == 4 ? 0xff800000u
                                   : std::is_same_v<T, __half> ? 0xfc00fc00u : 0xff80ff80u;
        for (int j0 = sl.w0; j0 < sl.w1; j0 += 32) {
            const int j = j0 + (threadIdx.x & 31);
            f(j, j < sl.w1 ? sl.vec(j) : make_uint4(kNone, kNone, kNone, kNone));
        }
    }

    // The weights of vector j that are kept (ALL: all of them).
    template <bool ALL>
    __device__ __forceinline__ void weights(const Keep& k, int j, const float (&y)[E], float (&w)[E]) const {
#pragma unroll
        for (int e = 0; e < E; e += 2) {
            const float2 d = add2(make_float2(y[e], y[e + 1]), splat(-m));
            w[e] = expf(d.x);
            w[e + 1] = expf(d.y);
        }
        if (!ALL) {
            bool tie = false;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                tie |= y[e] == k.tau;
                if (!(y[e] >= k.tau && w[e] >= k.min_p)) w[e] = 0.f;
            }
            if (tie) {  // rare: the threshold itself, kept up to an index
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (y[e] == k.tau && sl.index(j, e) > k.ilim) w[e] = 0.f;
            }
        }
    }

    // Mass of what is kept over the row; the warps' parts stay in sm.wsum.
    template <bool ALL>
    __device__ __forceinline__ Joined kept_mass(Smem& sm, const Keep& k) {
        Mass mass;
        each([&](int j, float (&y)[E]) {
            float w[E];
            weights<ALL>(k, j, y, w);
            mass.add(w);
        });
        return exchange<A, WARPS>(sm, phase, cluster, rank, mass.total(), 0.0, 0, 0.f, 0.f);
    }

    // The token at mass `target` of what is kept, in index order: the block, then its warp's
    // part, then the vector and the element whose prefix first exceeds the target (where
    // rounding leaves none, the last with any mass).  Follows the kept_mass that gave `c`,
    // whose parts in sm.wsum it reads.
    template <bool ALL>
    __device__ __forceinline__ void draw(Smem& sm, const Keep& k, const Joined& c, double target, double sum,
                                         const Params& p, int64_t row) const {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        const double end = rank + 1 < cluster ? c.before + sm.slot[phase ^ 1][rank].a : c.a;
        const double blk = sm.slot[phase ^ 1][rank].a;
        if (!(blk > 0.0) || target < c.before || !(target < end || !(end < c.a))) return;
        // the logarithms while the others look for the element
        if (lane == 0 && warp < 2) sm.logs[warp] = log(warp == 0 ? sum : c.a);
        int part = 0;
        double base = c.before, run = c.before;
#pragma unroll
        for (int i = 0; i < WARPS; ++i) {
            const double w = sm.wsum[i];
            if (w > 0.0 && !(run > target)) {
                part = i;
                base = run;
                run += w;
            }
        }
        const int per = (sl.nvec + WARPS - 1) / WARPS;
        const int j1 = min(sl.nvec, (part + 1) * per);
        for (int j0 = part * per; j0 < j1; j0 += TH) {
            const int j = j0 + threadIdx.x;
            float y[E], w[E];
            double mass = 0.0;
            if (j < j1) {
                unpack<T>(sl.vec(j), s, y);
                weights<ALL>(k, j, y, w);
#pragma unroll
                for (int e = 0; e < E; ++e) mass += (double)w[e];
            }
            double incl = mass;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double t = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += t;
            }
            __syncthreads();  // sm.wsum and sm.wsum_b have been read
            if (lane == 31) sm.wsum_b[warp] = incl;
            __syncthreads();
            double before = base, all = base;
            int last = 0;  // the last warp with any mass
#pragma unroll
            for (int i = 0; i < WARPS; ++i) {
                const double w = sm.wsum_b[i];
                if (i == warp) before = all;
                if (w > 0.0) last = i;
                all += w;
            }
            const bool crossed = all > target;
            // one warp holds it: the first whose end exceeds the target; until one does, the
            // last with any mass stands in (and is written over)
            const double wend = before + __shfl_sync(0xffffffffu, incl, 31);
            if (all > base && (crossed ? wend > target && !(before > target) : warp == last)) {
                const unsigned over = __ballot_sync(0xffffffffu, mass > 0.0 && before + incl > target);
                const unsigned some = __ballot_sync(0xffffffffu, mass > 0.0);
                const int at = over ? __ffs(over) - 1 : 31 - __clz(some);
                if (lane == at) {
                    const int el = pick_element(w, before + incl - mass, over ? target : INFINITY);
                    float d = 0.f;
#pragma unroll
                    for (int e = 0; e < E; ++e) d = e == el ? y[e] - m : d;
                    p.token[row] = sl.index(j, el);
                    p.logprob[row] = (float)((double)d - sm.logs[0]);
                    p.kept_logprob[row] = (float)((double)d - sm.logs[1]);
                }
            }
            if (crossed) return;
            base = all;
        }
    }
};

// FILTER: top-k, top-p or min-p may be in use (else rows draw from the whole distribution,
// and the kernel needs no list or histogram).
template <typename T, bool RES, bool FILTER>
__global__ void __launch_bounds__(FILTER ? kFilterThreads : kPlainThreads, FILTER ? kFilterBlocks : kPlainBlocks)
    k1_sample_kernel(Params p) {
    constexpr int E = DT<T>::kEPV;
    constexpr int TH = FILTER ? kFilterThreads : kPlainThreads;
    constexpr int WARPS = TH / 32;
    using SM = std::conditional_t<FILTER, FilterSmem, Smem>;
    extern __shared__ __align__(16) unsigned char sp_raw[];
    SM& sm = *reinterpret_cast<SM*>(sp_raw);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int cluster = p.cluster;
    const int rank = blockIdx.x % cluster;
    const int64_t row = blockIdx.x / cluster;
    const bool leader = rank == 0;
    ring::cluster_arrive();  // this block has started: the others may write its shared memory
    pdl_wait();
    pdl_trigger();

    Row<T, RES, TH> R;
    R.cluster = cluster;
    R.rank = rank;
    R.phase = 0;
    Slice<T, RES>& sl = R.sl;
    sl.buf = reinterpret_cast<uint4*>(sp_raw + smem_header<FILTER>());
    sl.init(reinterpret_cast<const T*>(p.logits) + row * p.row_stride, p.vocab, (int64_t)rank * p.slice_vecs,
            p.slice_vecs);
    const int per_warp = (sl.nvec + WARPS - 1) / WARPS;
    sl.w0 = min(sl.nvec, warp * per_warp);
    sl.w1 = min(sl.nvec, sl.w0 + per_warp);

    // ---- load; the maxima of this thread's NG groups of vectors ----
    Peak<T> peak[NG];
    if constexpr (FILTER) {
        sm.hist[threadIdx.x] = 0;
        if (threadIdx.x == 0) {
            sm.list_n = 0;
            sm.few_n = 0;
            sm.told = 0;
        }
    }
    auto load = [&](auto get) {
        int j = sl.w0 + lane;
        for (; j + 32 * (NG - 1) < sl.w1; j += 32 * NG) {
            uint4 v[NG];
#pragma unroll
            for (int q = 0; q < NG; ++q) v[q] = get(j + 32 * q);
#pragma unroll
            for (int q = 0; q < NG; ++q) {
                if constexpr (RES) sl.buf[j + 32 * q] = v[q];
                peak[q].add(v[q]);
            }
        }
#pragma unroll
        for (int q = 0; q < NG; ++q)
            if (j + 32 * q < sl.w1) {
                const uint4 v = get(j + 32 * q);
                if constexpr (RES) sl.buf[j + 32 * q] = v;
                peak[q].add(v);
            }
    };
    if (sl.w0 >= sl.whole0 && sl.w1 <= sl.whole1)  // the warp's part lies inside the row
        load([&](int j) { return ldg_stream(sl.base + j); });
    else
        load([&](int j) { return sl.load_global(j); });
    // the row's temperature
    const float temp = p.temperature ? p.temperature[row] : 1.f;
    const bool greedy = p.temperature ? temp == 0.f : p.greedy0;
    R.s = !p.temperature ? p.scale0 : greedy ? 1.f : (float)(1.0 / (double)temp);
    float g[NG], hi = -INFINITY, lo = INFINITY;
#pragma unroll
    for (int q = 0; q < NG; ++q) {
        g[q] = __fmul_rn(peak[q].value(), R.s);
        hi = fmax_nan(hi, g[q]);
        if (FILTER && g[q] > -INFINITY) lo = fminf(lo, g[q]);
    }
    ring::cluster_wait();  // every block of the row has started; the loads lay between
    const Joined range = exchange<RANGE, WARPS>(sm, R.phase, cluster, rank, 0.0, 0.0, 0, lo, hi);
    const float m = range.hi;
    R.m = m;
    // NaN, +inf, or nothing above -inf; or a setting of the row's own that means nothing
    bool none = !(m > -INFINITY && m < INFINITY) || !(temp >= 0.f && R.s > 0.f);
    if constexpr (FILTER) {
        if (p.top_p) none |= !(p.top_p[row] >= 0.f);
        if (p.min_p) none |= !(p.min_p[row] >= 0.f && p.min_p[row] <= 1.f);
    }
    if (none) {
        if (leader && threadIdx.x == 0) {
            p.token[row] = -1;
            p.logprob[row] = p.kept_logprob[row] = __int_as_float(0x7fc00000);
        }
        return;
    }
    const double u = (double)p.u[row];

    if constexpr (!FILTER) {
        const Keep keep = {-INFINITY, 0, 0.f};
        const Joined S = R.template kept_mass<true>(sm, keep);
        R.template draw<true>(sm, keep, S, u * S.a, S.a, p, row);
    } else {
        int top_k = greedy ? 1 : p.top_k ? p.top_k[row] : p.top_k0;
        if (top_k <= 0 || top_k >= p.vocab) top_k = 0;
        const float top_p = greedy ? 1.f : p.top_p ? p.top_p[row] : p.top_p0;
        const bool use_p = top_p < 1.f;
        const float min_p = greedy ? 0.f : p.min_p ? p.min_p[row] : p.min_p0;
        const float floor = m - kFloor;

        // ---- a bound for a short list ----
        // What at least `want` elements reach (about; whether so many do is seen from their
        // number): the bin of the groups' maxima in which their count gets that far.  Twice
        // the groups' range, so that the elements below the lowest of them spread too.
        const bool try_list = top_k ? top_k <= min(kListK, cluster * THREADS) : use_p;
        const unsigned want = top_k ? top_k : kNucleusK;
        Bins bins = Bins::linear(m, fmaxf(m - 2.f * (m - range.lo), floor));
        float least = INFINITY;
        if (try_list) {
#pragma unroll
            for (int q = 0; q < NG; ++q)
                if (g[q] >= floor) atomicAdd(&sm.hist[bins.of(g[q])], 1u);
            const unsigned upto = block_scan(row_bin(sm, cluster), sm.wn);
            const int b = first_bin(upto >= want);
            least = b == NB - 1 ? floor : fmaxf(floor, m - ((float)b + 0.5f) / bins.per_unit);
        }

        // ---- the whole mass, and the list ----
        Keep keep = {-INFINITY, 0, 0.f};
        Joined whole;
        if (try_list) {
            Mass mass;
            double listed = 0.0;
            unsigned n = 0;
            R.each_vector([&](int j, uint4 v) {
                float y[E], w[E];
                unpack<T>(v, R.s, y);
                R.template weights<true>(keep, j, y, w);
                mass.add(w);
                float top = y[0];
#pragma unroll
                for (int e = 1; e < E; ++e) top = fmaxf(top, y[e]);
                if (!__any_sync(0xffffffffu, top >= least)) return;
                unsigned hits = 0;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    hits |= y[e] >= least ? 1u << e : 0u;
                    listed += y[e] >= least ? (double)w[e] : 0.0;
                }
                n += __popc(hits);
                append(sm, hits, y, sl.index(j, 0), [](float) {});
            });
            whole = exchange<A | B | N, WARPS>(sm, R.phase, cluster, rank, mass.total(), listed, n, 0.f, 0.f);
        } else {
            whole = R.template kept_mass<true>(sm, keep);
        }
        const double S = whole.a;

        if (!top_k && !use_p && !(min_p > 0.f)) {
            R.template draw<true>(sm, keep, whole, u * S, S, p, row);
            return;
        }

        // ---- a short list ----
        if (try_list) {
            if (whole.n <= (unsigned)kListCap &&
                (top_k ? whole.n >= want || least == floor : whole.b >= (double)top_p * S)) {
                join_lists(sm, rank, whole.n_before);
                if (!leader) return;
                const int count = (int)whole.n;
                const double unit = list_unit(whole.b);
                uint64_t e[PER], word[PER];
                float w[PER];
                uint64_t part = 0;
#pragma unroll
                for (int r = 0; r < PER; ++r) {
                    const int i = r * THREADS + threadIdx.x;
                    e[r] = i < count ? sm.list[i] : 0;
                    w[r] = i < count ? expf(entry_value(e[r]) - m) : 0.f;
                    word[r] = i < count ? weight_word(w[r], unit) : 0;
                    part += word[r];
                }
                const uint64_t top = entry(m, 0), bottom = entry(least, 0xffffffffll);
                uint64_t cut = bottom;  // the last entry kept
                if (top_k && top_k < count) {
                    uint64_t one[PER];
#pragma unroll
                    for (int r = 0; r < PER; ++r) one[r] = word[r] ? count_word() : 0;
                    cut = select_entry(sm, e, one, bottom, top, (uint64_t)top_k);
                    part = 0;
#pragma unroll
                    for (int r = 0; r < PER; ++r) {
                        if (e[r] < cut) word[r] = 0;
                        part += word[r];
                    }
                }
                if (use_p) {
                    // of the whole mass without top-k: the list holds that share, up to the
                    // words' rounding
                    const uint64_t all = word_weight(block_sum64(sm, part));
                    const double Z = top_k ? (double)all : S * unit;
                    cut = select_entry(sm, e, word, cut, top, list_target((double)top_p * Z, all));
                }
                part = 0;
#pragma unroll
                for (int r = 0; r < PER; ++r) {
                    if (e[r] < cut || w[r] < min_p) word[r] = 0;
                    part += word[r];
                }
                // the draw: the same over the kept indices, the lowest first
                const uint64_t C = word_weight(block_sum64(sm, part));
                uint64_t id[PER];
#pragma unroll
                for (int r = 0; r < PER; ++r) id[r] = e[r] & 0xffffffffu;
                const uint64_t at = select_entry(sm, id, word, (uint64_t)(uint32_t)~(uint32_t)(p.vocab - 1),
                                                 0xffffffffu, min(C, (uint64_t)(u * (double)C) + 1));
#pragma unroll
                for (int r = 0; r < PER; ++r)
                    if (word[r] && id[r] == at) {
                        const double d = (double)(entry_value(e[r]) - m);
                        p.token[row] = entry_index(e[r]);
                        p.logprob[row] = (float)(d - log(S));
                        p.kept_logprob[row] = (float)(d - log((double)C / unit));
                    }
                return;
            }
        }

        // ---- selection over all elements: top-k, then top-p ----
        double Z = S;
        for (int what = 0; what < 2; ++what) {
            const bool by_mass = what == 1;
            if (!(by_mass ? use_p : top_k > 0)) continue;
            const double target = by_mass ? (double)top_p * Z : (double)top_k;
            // the crossing element (the last one kept) lies in y of [ylo, yhi]; `above` is
            // what is placed before that interval
            float ylo = fmaxf(floor, keep.tau), yhi = m;
            if (by_mass) {
                // elements whose weight is below (1 - p) Z / V have less than (1 - p) Z
                // together, so the crossing lies above them (half a unit of y to spare)
                ylo = fmaxf(ylo, m + logf((float)((1.0 - (double)top_p) * Z / (double)p.vocab)) - 0.5f);
                bins = Bins::linear(m, ylo);
            }
            double above = 0.0;
            for (;;) {
                // histogram of the interval: counts, or weights relative to one of the bin's
                // in steps of 2^-12 (larger ones for vocabularies above 2^18, so that a bin
                // that holds every element fits 32 bits: a bin of equal width spans less than
                // 0.21 units of y, so no weight is above 1.12 of its middle's)
                const float step = by_mass ? fminf(4096.f, 1073741824.f / (float)p.vocab) : 1.f;
                sm.hist[threadIdx.x] = 0;
                if (threadIdx.x == 0) sm.list_n = 0;
                __syncthreads();
                const bool tied = keep.tau > -INFINITY;  // some of the equals at tau are out
                if (bins.shift < 0) {
                    // Adding 1.5 2^23 rounds to a whole number and leaves it in the low bits.
                    // The fast exponential has a guide's precision.
                    constexpr float kWhole = 12582912.f;
                    const float to_log2 = kLog2e / bins.per_unit;
                    R.each([&](int j, float (&y)[E]) {
#pragma unroll
                        for (int e = 0; e < E; ++e) {
                            if (!(y[e] >= ylo && y[e] <= yhi)) continue;
                            if (tied && !keep.allows(y[e], sl, j, e)) continue;
                            const float at = bins.place(y[e]), whole = at + kWhole;
                            const unsigned b = __float_as_uint(whole) & (NB - 1);
                            unsigned v = 1;
                            if (by_mass)
                                v = __float_as_uint(fmaf(ex2(((whole - kWhole) - at) * to_log2), step, 8388608.f)) &
                                    0x7fffffu;
                            atomicAdd(&sm.hist[b], v);
                        }
                    });
                } else {
                    R.each([&](int j, float (&y)[E]) {
#pragma unroll
                        for (int e = 0; e < E; ++e) {
                            if (!(y[e] >= ylo && y[e] <= yhi)) continue;
                            if (tied && !keep.allows(y[e], sl, j, e)) continue;
                            const int b = bins.of(y[e]);
                            atomicAdd(&sm.hist[b], by_mass ? (unsigned)(__expf(y[e] - bins.base_of(b)) * step) : 1u);
                        }
                    });
                }
                double part = (double)row_bin(sm, cluster);
                if (by_mass) part *= exp((double)bins.base_of(threadIdx.x) - (double)m) / (double)step;
                const double upto = above + block_scan(part, sm.wscan);
                if (!by_mass && __syncthreads_or(threadIdx.x == NB - 1 && upto < target))
                    break;  // fewer elements than top-k asks for: all stay
                int b = first_bin(upto >= target);
                // the bin's exact limits, its elements into the list; a neighbour's if the
                // rounded masses misled
                Joined t;
                for (int tries = 0; tries < 2 * NB; ++tries) {
                    Mass over;
                    double in = 0.0;
                    unsigned n_over = 0, n_in = 0;
                    float lo = INFINITY, hi = -INFINITY;
                    const float fb = (float)b;
                    R.each_vector([&](int j, uint4 x) {
                        float y[E], w[E];
                        unpack<T>(x, R.s, y);
                        unsigned inside = 0;  // the vector's elements in the bin
                        if (bins.shift < 0) {
                            constexpr float kWhole = 12582912.f;
#pragma unroll
                            for (int e = 0; e < E; ++e) {
                                const float whole = bins.place(y[e]) + kWhole - kWhole;
                                // past yhi or ylo: no bin (the interval is the first one)
                                const bool here = y[e] >= ylo;
                                inside |= here && whole == fb ? 1u << e : 0u;
                                w[e] = here && whole < fb ? y[e] : -INFINITY;
                            }
                        } else {
#pragma unroll
                            for (int e = 0; e < E; ++e) {
                                const bool here = y[e] >= ylo && y[e] <= yhi;
                                const int q = here ? bins.of(y[e]) : NB;
                                inside |= q == b ? 1u << e : 0u;
                                w[e] = q < b ? y[e] : -INFINITY;
                            }
                        }
                        if (tied) {
#pragma unroll
                            for (int e = 0; e < E; ++e)
                                if (!keep.allows(y[e], sl, j, e)) {
                                    w[e] = -INFINITY;
                                    inside &= ~(1u << e);
                                }
                        }
                        if (by_mass) {
#pragma unroll
                            for (int e = 0; e < E; e += 2) {
                                const float2 d = add2(make_float2(w[e], w[e + 1]), splat(-m));
                                w[e] = expf(d.x);
                                w[e + 1] = expf(d.y);
                            }
                            over.add(w);
                        } else {
#pragma unroll
                            for (int e = 0; e < E; ++e) n_over += w[e] > -INFINITY;
                        }
                        n_in += __popc(inside);
                        append(sm, inside, y, sl.index(j, 0), [&](float v) {
                            lo = fminf(lo, v);
                            hi = fmaxf(hi, v);
                            if (by_mass) in += (double)expf(v - m);
                        });
                    });
                    t = exchange<A | B | N | RANGE, WARPS>(sm, R.phase, cluster, rank,
                                                    by_mass ? over.total() : (double)n_over,
                                                    by_mass ? in : (double)n_in, n_in, lo, hi);
                    const int b0 = b;
                    if (t.a > 0.0 && above + t.a >= target && b > 0)
                        --b;
                    else if ((t.n == 0 || above + t.a + t.b < target) && b < NB - 1)
                        ++b;
                    if (b == b0) break;
                    if (threadIdx.x == 0) sm.list_n = 0;
                    __syncthreads();
                }
                if (t.n == 0) break;  // not reached: the interval holds the crossing element
                above += t.a;
                ylo = t.lo;
                yhi = t.hi;
                if (t.n <= (unsigned)kListCap) {
                    // the crossing element by rank in the list
                    join_lists(sm, rank, t.n_before);
                    if (leader) {
                        const int count = (int)t.n;
                        const double unit = by_mass ? list_unit(t.b) : 1.0;
                        uint64_t e[PER], word[PER];
#pragma unroll
                        for (int r = 0; r < PER; ++r) {
                            const int i = r * THREADS + threadIdx.x;
                            e[r] = i < count ? sm.list[i] : 0;
                            word[r] = i >= count ? 0
                                      : by_mass  ? weight_word(expf(entry_value(e[r]) - m), unit)
                                                 : count_word();
                        }
                        const uint64_t all = word_weight(block_sum64(sm, word[0] + word[1] + word[2] + word[3]));
                        const uint64_t at = select_entry(sm, e, word, entry(ylo, 0xffffffffll), entry(yhi, 0),
                                                         list_target((target - above) * unit, all));
                        if (threadIdx.x == 0) tell(sm, cluster, entry_value(at), entry_index(at));
                    }
                    ring::cluster_sync();
                    break;
                }
                if (ylo == yhi) {
                    // all equal: the nth of them in index order
                    const double each_one = by_mass ? (double)expf(ylo - m) : 1.0;
                    const int64_t nth =
                        (int64_t)fmin(fmax(ceil((target - above) / each_one), 1.0), (double)t.n);
                    unsigned n = 0;
                    R.each([&](int j, float (&y)[E]) {
#pragma unroll
                        for (int e = 0; e < E; ++e)
                            if (y[e] == ylo && keep.allows(y[e], sl, j, e)) ++n;
                    });
                    const Joined o = exchange<N, WARPS>(sm, R.phase, cluster, rank, 0.0, 0.0, n, 0.f, 0.f);
                    int64_t run = o.n_before;
                    for (int i = 0; i < warp; ++i) run += sm.wn[i];
                    if (run < nth && nth <= run + (int64_t)sm.wn[warp]) {
                        for (int j0 = sl.w0; j0 < sl.w1; j0 += 32) {
                            const int j = j0 + lane;
                            unsigned k = 0;
                            float y[E];
                            if (j < sl.w1) {
                                unpack<T>(sl.vec(j), R.s, y);
#pragma unroll
                                for (int e = 0; e < E; ++e)
                                    if (y[e] == ylo && keep.allows(y[e], sl, j, e)) ++k;
                            }
                            unsigned incl = k;
#pragma unroll
                            for (int o2 = 1; o2 < 32; o2 <<= 1) {
                                const unsigned x = __shfl_up_sync(0xffffffffu, incl, o2);
                                if (lane >= o2) incl += x;
                            }
                            int64_t at = run + incl - k;
                            if (k > 0 && at < nth && nth <= at + k) {
#pragma unroll
                                for (int e = 0; e < E; ++e)
                                    if (y[e] == ylo && keep.allows(y[e], sl, j, e) && ++at == nth)
                                        tell(sm, cluster, ylo, sl.index(j, e));
                            }
                            run += __shfl_sync(0xffffffffu, incl, 31);
                        }
                    }
                    ring::cluster_sync();
                    break;
                }
                bins = Bins::keys(yhi, ylo);
            }
            if (sm.told) {
                keep.tau = sm.tau;
                keep.ilim = sm.ilim;
            }
            if (!by_mass && use_p) Z = R.template kept_mass<false>(sm, keep).a;
        }
        keep.min_p = min_p;
        const Joined C = R.template kept_mass<false>(sm, keep);
        R.template draw<false>(sm, keep, C, u * C.a, S, p, row);
    }
}

}  // namespace sample
}  // namespace k1
