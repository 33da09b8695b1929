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
// Sums of weights decide which token is drawn, so they must not depend on how a row is cut:
// a weight is split into a multiple of 2^-13, whose fp32 sums are exact, and a rest that
// goes to fp64 once per 16-byte vector.  The error of S is then about 1e-11 of it.
//
// A cluster of 1 to 8 blocks owns a row: every block holds its part of the row in shared
// memory, so the logits cross HBM once whatever the filters ask for, and all later passes
// (weights, histograms, thresholds) run from there.  The blocks exchange maxima, sums and
// histograms through distributed shared memory.  Two blocks per SM: one row's passes run
// while another row's loads are in flight.  (Rows too long for a cluster's shared memory
// are read again from global memory in each pass.)
//
//   whole rows (no filter)  load + max, sum, draw.
//   short lists             Each thread keeps the maxima of four groups of its elements.  A
//                           histogram of those maxima gives a bound that at least K elements
//                           reach, and few more; only groups that reach it are read again,
//                           and their elements go to a list in the first block, which sorts
//                           it and applies the filters.  Serves top-k up to kListK and every
//                           top-p whose nucleus lies within the list.
//   selection               Otherwise the threshold is found by histograms over all elements:
//                           bins of equal width in y (counts for top-k, masses for top-p,
//                           the latter rounded to 2^-14 of the bin's largest weight, so
//                           only a guide), then the bin's exact limits, and again inside it
//                           until its elements fit the list or are all equal.
//
// A row that holds a NaN or +inf, or nothing above -inf, has no distribution: token -1 and
// NaN log-probabilities.
#pragma once

#include "k1_common.cuh"
#include "k1_sync.cuh"

namespace k1 {
namespace sample {

constexpr int THREADS = 512;
constexpr int WARPS = THREADS / 32;
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
    double temperature0;
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

struct Smem {
    uint64_t list[kListCap];
    double scan[kListCap];
    unsigned hist[NB];
    Xch slot[2];
    Xch all;              // the exchange's result
    double before;        // sum of `a` over the blocks of lower rank
    unsigned n_before;    // sum of `n` over the blocks of lower rank
    double wsum[WARPS];
    double wsum_b[WARPS];
    unsigned wn[WARPS];
    float wlo[WARPS], whi[WARPS];
    unsigned list_n;
    int pick;             // a block-wide choice
    int64_t ilim;
    float tau;
};

// ------------------------------------------------------------------------------------
// A row's part in one block
// ------------------------------------------------------------------------------------
// The row is widened to 16-byte boundaries: virtual index v = i + shift, shift = elements
// between the boundary at or below the row's start and the start.  Elements outside the row
// read as -inf, which no pass counts.
template <typename T, bool RES>
struct Slice {
    static constexpr int E = DT<T>::kEPV;
    const T* row;
    uint4* buf;        // RES: the slice in shared memory
    int64_t vocab;
    int shift;
    int64_t vec0;      // the block's first vector
    int nvec;          // its vectors
    int w0, w1;        // the warp's vectors: contiguous, lanes interleaved

    __device__ __forceinline__ uint4 load_global(int64_t vec) const {
        const int64_t i0 = vec * E - shift;
        if (i0 >= 0 && i0 + E <= vocab) return ldg_stream(row + i0);
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
    __device__ __forceinline__ uint4 vec(int j) const {
        if constexpr (RES)
            return buf[j];
        else
            return load_global(vec0 + j);
    }
    __device__ __forceinline__ int64_t index(int j, int e) const { return (vec0 + j) * E + e - shift; }
};

template <typename T>
__device__ __forceinline__ void unpack(uint4 v, float s, float (&y)[DT<T>::kEPV]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) {
            y[i] = __uint_as_float(w[i]) * s;
        } else {
            const float2 f = DT<T>::to_f2(w[i]);
            y[2 * i] = f.x * s;
            y[2 * i + 1] = f.y * s;
        }
    }
}

// Largest element of a vector (NaN if it holds one).
template <typename T>
__device__ __forceinline__ float vec_max(uint4 v) {
    if constexpr (sizeof(T) == 4) {
        return fmax_nan(fmax_nan(__uint_as_float(v.x), __uint_as_float(v.y)),
                        fmax_nan(__uint_as_float(v.z), __uint_as_float(v.w)));
    } else {
        const float2 f = DT<T>::to_f2(DT<T>::max2(DT<T>::max2(v.x, v.y), DT<T>::max2(v.z, v.w)));
        return fmax_nan(f.x, f.y);
    }
}

// Exact running sum of weights in [0, 1]: multiples of 2^-13 add exactly in fp32 (up to 2^11
// per thread and fold), the rests of one vector go to fp64.
struct Mass {
    float hi = 0.f;
    double sum = 0.0;
    int folds = 0;
    template <int E>
    __device__ __forceinline__ void add(const float (&w)[E]) {
        float lo = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const float h = __fadd_rn(__fadd_rn(w[i], 1536.f), -1536.f);
            hi += h;
            lo += w[i] - h;
        }
        sum += (double)lo;
        if (++folds == 128) {
            sum += (double)hi;
            hi = 0.f;
            folds = 0;
        }
    }
    __device__ __forceinline__ double total() const { return sum + (double)hi; }
};

// Order-preserving key of a float (larger value, larger key).
__device__ __forceinline__ uint32_t key_of(float y) {
    const uint32_t b = __float_as_uint(y);
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
    __device__ __forceinline__ int of(float y) const {
        return shift < 0 ? (int)fminf((top - y) * per_unit, (float)(NB - 1))
                         : (int)((key_top - key_of(y)) >> shift);
    }
    // the largest y of bin b (up to rounding)
    __device__ __forceinline__ float top_of(int b) const {
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

__device__ __forceinline__ void ld_remote(Xch* dst, const Xch* slot, int rank) {
    const uint32_t a = ring::mapa(ring::saddr(slot), rank);
    uint64_t w[sizeof(Xch) / 8];
#pragma unroll
    for (int i = 0; i < (int)(sizeof(Xch) / 8); ++i)
        asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(w[i]) : "r"(a + 8 * i) : "memory");
    memcpy(dst, w, sizeof(Xch));
}

// Adds a, b, n and joins lo (min), hi (max) over all threads of all blocks of the row;
// the result is in sm.all (and sm.before, sm.n_before) for every thread on return.  NaN in
// hi survives.  Sums run in a fixed order.  `phase` alternates between calls, so that a
// block may write its next contribution while another still reads the last one.
__device__ __forceinline__ void exchange(Smem& sm, int& phase, int cluster, int rank, double a, double b,
                                         unsigned n, float lo, float hi) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    a = warp_add(a);
    b = warp_add(b);
    n = warp_add(n);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = warp_max_nan(hi);
    if (lane == 0) {
        sm.wsum[warp] = a;
        sm.wsum_b[warp] = b;
        sm.wn[warp] = n;
        sm.wlo[warp] = lo;
        sm.whi[warp] = hi;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        Xch x = {0.0, 0.0, INFINITY, -INFINITY, 0, 0};
        for (int i = 0; i < WARPS; ++i) {
            x.a += sm.wsum[i];
            x.b += sm.wsum_b[i];
            x.n += sm.wn[i];
            x.lo = fminf(x.lo, sm.wlo[i]);
            x.hi = fmax_nan(x.hi, sm.whi[i]);
        }
        sm.slot[phase] = x;
    }
    ring::cluster_sync();
    if (threadIdx.x == 0) {
        Xch t = {0.0, 0.0, INFINITY, -INFINITY, 0, 0};
        Xch x[kMaxCluster];
#pragma unroll
        for (int r = 0; r < kMaxCluster; ++r)
            if (r < cluster) ld_remote(&x[r], &sm.slot[phase], r);
#pragma unroll
        for (int r = 0; r < kMaxCluster; ++r) {
            if (r < cluster) {
                if (r == rank) {
                    sm.before = t.a;
                    sm.n_before = t.n;
                }
                t.a += x[r].a;
                t.b += x[r].b;
                t.n += x[r].n;
                t.lo = fminf(t.lo, x[r].lo);
                t.hi = fmax_nan(t.hi, x[r].hi);
            }
        }
        sm.all = t;
    }
    __syncthreads();
    phase ^= 1;
}

// Adds the blocks' histograms: thread b returns bin b of the row.  Ends with no block still
// reading another's.
__device__ __forceinline__ unsigned row_bin(Smem& sm, int cluster) {
    ring::cluster_sync();
    unsigned v = 0;
    const uint32_t a = ring::saddr(&sm.hist[threadIdx.x]);
    for (int r = 0; r < cluster; ++r) {
        unsigned x;
        asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(x) : "r"(ring::mapa(a, r)) : "memory");
        v += x;
    }
    ring::cluster_sync();
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
    for (int i = 0; i < warp; ++i) base += warp_sums[i];
    return base + v;
}

// The first thread whose (inclusive, nondecreasing) prefix satisfies `hit`; the last thread
// if none does.
__device__ __forceinline__ int first_thread(Smem& sm, bool hit) {
    if (threadIdx.x == 0) sm.pick = NB - 1;
    __syncthreads();
    if (hit) atomicMin(&sm.pick, (int)threadIdx.x);
    __syncthreads();
    const int v = sm.pick;
    __syncthreads();
    return v;
}

// Append to the list in the row's first block.
__device__ __forceinline__ void append(Smem& sm, float y, int64_t index) {
    const uint32_t cnt = ring::mapa(ring::saddr(&sm.list_n), 0);
    unsigned pos;
    asm volatile("atom.relaxed.cluster.shared::cluster.add.u32 %0, [%1], 1;" : "=r"(pos) : "r"(cnt) : "memory");
    if (pos < (unsigned)kListCap) {
        const uint64_t k = ((uint64_t)key_of(y) << 32) | (uint32_t)~(uint32_t)index;
        asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(ring::mapa(ring::saddr(&sm.list[0]), 0) + pos * 8),
                     "l"(k)
                     : "memory");
    }
}

// Bitonic sort of keys[0, n), n <= kListCap, largest first (this block's threads).
__device__ __forceinline__ void sort_list(uint64_t* keys, int n) {
    int size = 2;
    while (size < n) size <<= 1;
    for (int i = n + threadIdx.x; i < size; i += THREADS) keys[i] = 0;
    __syncthreads();
    for (int k = 2; k <= size; k <<= 1) {
        for (int j = k >> 1; j > 0; j >>= 1) {
            for (int t = threadIdx.x; t < size / 2; t += THREADS) {
                const int i = ((t & ~(j - 1)) << 1) | (t & (j - 1));
                const uint64_t a = keys[i], b = keys[i + j];
                if ((a < b) == ((i & k) == 0)) {
                    keys[i] = b;
                    keys[i + j] = a;
                }
            }
            __syncthreads();
        }
    }
}

// scan[i] = sum of weight(i') for i' <= i < n, in fp64 (this block's threads).
template <typename F>
__device__ __forceinline__ void scan_list(Smem& sm, int n, F weight) {
    double base = 0.0;
    for (int i0 = 0; i0 < n; i0 += THREADS) {
        const int i = i0 + threadIdx.x;
        const double v = block_scan(i < n ? weight(i) : 0.0, sm.wsum) + base;
        if (i < n) sm.scan[i] = v;
        __syncthreads();
        base = sm.scan[min(n, i0 + THREADS) - 1];
    }
    __syncthreads();
}

// The first i in [0, n) with test(i) (a test that stays true once true); n - 1 if none.
template <typename F>
__device__ __forceinline__ int first_in_list(Smem& sm, int n, F test) {
    if (threadIdx.x == 0) sm.pick = n - 1;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += THREADS)
        if (test(i)) {
            atomicMin(&sm.pick, i);
            break;
        }
    __syncthreads();
    const int v = sm.pick;
    __syncthreads();
    return v;
}

// ------------------------------------------------------------------------------------
// The kernel
// ------------------------------------------------------------------------------------
// What is kept so far: y above tau, and y equal to tau up to index ilim.
struct Keep {
    float tau;
    int64_t ilim;
    float min_p;  // a weight's lower limit, 0: off
    __device__ __forceinline__ bool ranked(float y, int64_t i) const {
        return y > tau || (y == tau && i <= ilim);
    }
    __device__ __forceinline__ bool holds(float y, float w, int64_t i) const {
        return w >= min_p && ranked(y, i);
    }
};

template <typename T, bool RES>
struct Row {
    static constexpr int E = DT<T>::kEPV;
    Smem& sm;
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

    // Mass of what is kept (`all`: of everything) over the row; the warps' parts stay in
    // sm.wsum, the lower ranks' in sm.before.
    __device__ __forceinline__ double kept_mass(const Keep& k, bool all) {
        Mass mass;
        each([&](int j, float (&y)[E]) {
            float w[E];
#pragma unroll
            for (int e = 0; e < E; ++e) {
                w[e] = expf(y[e] - m);
                if (!all && !k.holds(y[e], w[e], sl.index(j, e))) w[e] = 0.f;
            }
            mass.add(w);
        });
        exchange(sm, phase, cluster, rank, mass.total(), 0.0, 0, 0.f, 0.f);
        return sm.all.a;
    }

    // The token at mass `target` of what is kept, in index order, found by the warp that
    // holds it.  Follows kept_mass (whose partial sums it reads) directly.
    __device__ __forceinline__ void draw(const Keep& k, bool all, double target, double total, double sum,
                                         const Params& p, int64_t row) {
        // the block, then the warp, whose prefix first exceeds the target; the last one with
        // any mass if rounding leaves none
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        double base = sm.before, blk = 0.0;
        for (int i = 0; i < WARPS; ++i) blk += sm.wsum[i];  // as exchange added them
        if (blk <= 0.0) return;
        const bool last_block = !(base + blk < total);
        if (target < base || !(target < base + blk || last_block)) return;
        int pick = -1;
        double pick_base = base, run = base;
        for (int i = 0; i < WARPS; ++i) {
            const double w = sm.wsum[i];
            if (w > 0.0) {
                pick = i;
                pick_base = run;
                run += w;
                if (run > target) break;
            }
        }
        if (warp != pick) return;
        run = pick_base;
        int64_t found = -1;
        float yf = 0.f;
        for (int j0 = sl.w0; j0 < sl.w1; j0 += 32) {
            const int j = j0 + lane;
            float y[E], w[E];
            double mass = 0.0;
            if (j < sl.w1) {
                unpack<T>(sl.vec(j), s, y);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    w[e] = expf(y[e] - m);
                    if (!all && !k.holds(y[e], w[e], sl.index(j, e))) w[e] = 0.f;
                    mass += (double)w[e];
                }
            }
            double incl = mass;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double t = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += t;
            }
            const bool over = mass > 0.0 && run + incl > target;
            const unsigned any = __ballot_sync(0xffffffffu, over);
            const unsigned some = __ballot_sync(0xffffffffu, mass > 0.0);
            // the crossing lane; without one, the last lane with mass holds the candidate
            const int at = any ? __ffs(any) - 1 : some ? 31 - __clz(some) : -1;
            if (at == lane) {
                double c = run + incl - mass;
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (w[e] > 0.f && !(any && c > target)) {
                        c += (double)w[e];
                        found = sl.index(j, e);
                        yf = y[e];
                    }
            }
            if (at >= 0) {
                found = __shfl_sync(0xffffffffu, found, at);
                yf = __shfl_sync(0xffffffffu, yf, at);
            }
            if (any) break;
            run += __shfl_sync(0xffffffffu, incl, 31);
        }
        if (lane == 0) {
            p.token[row] = found;
            p.logprob[row] = (float)((double)(yf - m) - log(sum));
            p.kept_logprob[row] = (float)((double)(yf - m) - log(total));
        }
    }
};

template <typename T, bool RES>
__global__ void __launch_bounds__(THREADS, 2) k1_sample_kernel(Params p) {
    constexpr int E = DT<T>::kEPV;
    extern __shared__ __align__(16) unsigned char sp_raw[];
    Smem& sm = *reinterpret_cast<Smem*>(sp_raw);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int cluster = p.cluster;
    const int rank = blockIdx.x % cluster;
    const int64_t row = blockIdx.x / cluster;
    const bool leader = rank == 0;
    pdl_wait();
    pdl_trigger();

    // the row's settings
    const double temp = p.temperature ? (double)p.temperature[row] : p.temperature0;
    const bool greedy = temp == 0.0;
    int top_k = greedy ? 1 : p.top_k ? p.top_k[row] : p.top_k0;
    if (top_k <= 0 || top_k >= p.vocab) top_k = 0;
    const float top_p = greedy ? 1.f : p.top_p ? p.top_p[row] : p.top_p0;
    const bool use_p = top_p < 1.f;
    const float min_p = greedy ? 0.f : fminf(p.min_p ? p.min_p[row] : p.min_p0, 1.f);

    Row<T, RES> R{sm};
    R.cluster = cluster;
    R.rank = rank;
    R.phase = 0;
    R.s = greedy ? 1.f : (float)(1.0 / temp);
    Slice<T, RES>& sl = R.sl;
    sl.row = reinterpret_cast<const T*>(p.logits) + row * p.row_stride;
    sl.buf = reinterpret_cast<uint4*>(sp_raw + ((sizeof(Smem) + 15) & ~(size_t)15));
    sl.vocab = p.vocab;
    sl.shift = (int)((reinterpret_cast<uintptr_t>(sl.row) & 15) / sizeof(T));
    sl.vec0 = (int64_t)rank * p.slice_vecs;
    const int64_t row_vecs = (p.vocab + sl.shift + E - 1) / E;
    sl.nvec = (int)max((int64_t)0, min((int64_t)p.slice_vecs, row_vecs - sl.vec0));
    const int per_warp = (sl.nvec + WARPS - 1) / WARPS;
    sl.w0 = min(sl.nvec, warp * per_warp);
    sl.w1 = min(sl.nvec, sl.w0 + per_warp);

    // ---- load; the maxima of this thread's NG groups of vectors ----
    float g[NG];
#pragma unroll
    for (int q = 0; q < NG; ++q) g[q] = -INFINITY;
    sm.hist[threadIdx.x] = 0;
    if (threadIdx.x == 0) sm.list_n = 0;
    for (int j = sl.w0 + lane; j < sl.w1; j += 32 * NG) {
        uint4 v[NG];
#pragma unroll
        for (int q = 0; q < NG; ++q)
            if (j + 32 * q < sl.w1) v[q] = sl.load_global(sl.vec0 + j + 32 * q);
#pragma unroll
        for (int q = 0; q < NG; ++q)
            if (j + 32 * q < sl.w1) {
                if constexpr (RES) sl.buf[j + 32 * q] = v[q];
                g[q] = fmax_nan(g[q], vec_max<T>(v[q]));
            }
    }
    {
        float hi = -INFINITY, lo = INFINITY;
#pragma unroll
        for (int q = 0; q < NG; ++q) {
            g[q] *= R.s;
            hi = fmax_nan(hi, g[q]);
            if (g[q] > -INFINITY) lo = fminf(lo, g[q]);
        }
        exchange(sm, R.phase, cluster, rank, 0.0, 0.0, 0, lo, hi);
    }
    const float m = sm.all.hi;
    const float floor = m - kFloor;
    R.m = m;
    // NaN, +inf, or nothing above -inf; or a temperature that is negative or no number
    if (!(m > -INFINITY && m < INFINITY) || !(temp >= 0.0 && R.s > 0.f)) {
        if (leader && threadIdx.x == 0) {
            p.token[row] = -1;
            p.logprob[row] = p.kept_logprob[row] = __int_as_float(0x7fc00000);
        }
        ring::cluster_sync();  // no block leaves while its shared memory may be read
        return;
    }

    // ---- the whole mass ----
    const bool try_list = top_k ? top_k <= min(kListK, cluster * THREADS) : use_p;
    Bins bins = Bins::linear(m, fmaxf(sm.all.lo, floor));
    if (try_list) {
#pragma unroll
        for (int q = 0; q < NG; ++q)
            if (g[q] >= floor) atomicAdd(&sm.hist[bins.of(g[q])], 1u);
    }
    Keep keep = {-INFINITY, 0, 0.f};
    const double S = R.kept_mass(keep, true);
    const double u = (double)p.u[row];

    if (!top_k && !use_p && !(min_p > 0.f)) {
        R.draw(keep, true, u * S, S, S, p, row);
        ring::cluster_sync();
        return;
    }

    // ---- a short list ----
    if (try_list) {
        const unsigned want = top_k ? top_k : kNucleusK;
        const unsigned upto = block_scan(row_bin(sm, cluster), sm.wn);
        const int b = first_thread(sm, upto >= want);
        double mass = 0.0;
        unsigned n = 0;
#pragma unroll
        for (int q = 0; q < NG; ++q) {
            if (!(g[q] >= floor && bins.of(g[q]) <= b)) continue;
            for (int j = sl.w0 + lane + 32 * q; j < sl.w1; j += 32 * NG) {
                float y[E];
                unpack<T>(sl.vec(j), R.s, y);
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (y[e] >= floor && bins.of(y[e]) <= b) {
                        mass += (double)expf(y[e] - m);
                        append(sm, y[e], sl.index(j, e));
                        ++n;
                    }
            }
        }
        exchange(sm, R.phase, cluster, rank, mass, 0.0, n, 0.f, 0.f);
        const int count = (int)sm.all.n;
        if (count <= kListCap && (top_k || sm.all.a >= (double)top_p * S)) {
            if (leader) {
                sort_list(sm.list, count);
                auto weight = [&](int i) { return (double)expf(value_of((uint32_t)(sm.list[i] >> 32)) - m); };
                scan_list(sm, count, weight);
                int kept = top_k ? min(top_k, count) : count;
                if (use_p) {
                    const double target = (double)top_p * (top_k ? sm.scan[kept - 1] : S);
                    kept = first_in_list(sm, kept, [&](int i) { return sm.scan[i] >= target; }) + 1;
                }
                if (min_p > 0.f) {
                    const int lowest = first_in_list(sm, kept, [&](int i) { return weight(i) < (double)min_p; });
                    if (weight(lowest) < (double)min_p) kept = max(1, lowest);
                    __syncthreads();
                }
                // index order: keys (~index, value) sorted largest first
                for (int i = threadIdx.x; i < kept; i += THREADS)
                    sm.list[i] = (sm.list[i] << 32) | (sm.list[i] >> 32);
                __syncthreads();
                sort_list(sm.list, kept);
                scan_list(sm, kept, [&](int i) { return (double)expf(value_of((uint32_t)sm.list[i]) - m); });
                const double C = sm.scan[kept - 1], target = u * C;
                const int at = first_in_list(sm, kept, [&](int i) { return sm.scan[i] > target; });
                if (threadIdx.x == 0) {
                    const double d = (double)(value_of((uint32_t)sm.list[at]) - m);
                    p.token[row] = (int64_t)(uint32_t)~(uint32_t)(sm.list[at] >> 32);
                    p.logprob[row] = (float)(d - log(S));
                    p.kept_logprob[row] = (float)(d - log(C));
                }
            }
            ring::cluster_sync();
            return;
        }
    }

    // ---- selection over all elements: top-k, then top-p ----
    double Z = S;
    for (int what = 0; what < 2; ++what) {
        const bool by_mass = what == 1;
        if (!(by_mass ? use_p : top_k > 0)) continue;
        const double target = by_mass ? (double)top_p * Z : (double)top_k;
        // the crossing element (the last one kept) lies in y of [ylo, yhi]; `above` is what
        // is ranked before that interval
        float ylo = floor, yhi = m;
        double above = 0.0;
        for (;;) {
            // histogram of the interval: counts, or weights relative to the bin's largest
            // one in steps of 2^-14 (larger ones for vocabularies above 2^18, so that a bin
            // that holds every element fits 32 bits)
            const float step = by_mass ? fminf(16384.f, 4294967040.f / (float)p.vocab) : 1.f;
            sm.hist[threadIdx.x] = 0;
            __syncthreads();
            R.each([&](int j, float (&y)[E]) {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    if (!(y[e] >= ylo && y[e] <= yhi && keep.ranked(y[e], sl.index(j, e)))) continue;
                    const int b = bins.of(y[e]);
                    unsigned v = 1;
                    if (by_mass) v = (unsigned)(fminf(expf(y[e] - bins.top_of(b)), 1.f) * step);
                    if (v) atomicAdd(&sm.hist[b], v);
                }
            });
            __syncthreads();
            double part = (double)row_bin(sm, cluster);
            if (by_mass) part *= exp((double)bins.top_of(threadIdx.x) - (double)m) / (double)step;
            const double upto = above + block_scan(part, sm.wsum);
            if (!by_mass && __syncthreads_or(threadIdx.x == NB - 1 && upto < target)) {
                break;  // fewer elements than top-k asks for: all stay
            }
            int b = first_thread(sm, upto >= target);
            // the bin's exact limits; a neighbour's if the rounded masses misled
            for (int tries = 0; tries < 2 * NB; ++tries) {
                Mass over, in;
                unsigned n_over = 0, n_in = 0;
                float lo = INFINITY, hi = -INFINITY;
                R.each([&](int j, float (&y)[E]) {
                    float wo[E], wi[E];
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        wo[e] = wi[e] = 0.f;
                        if (!(y[e] >= ylo && y[e] <= yhi && keep.ranked(y[e], sl.index(j, e)))) continue;
                        const int q = bins.of(y[e]);
                        if (q > b) continue;
                        const float w = by_mass ? expf(y[e] - m) : 0.f;
                        if (q < b) {
                            wo[e] = w;
                            ++n_over;
                        } else {
                            wi[e] = w;
                            ++n_in;
                            lo = fminf(lo, y[e]);
                            hi = fmaxf(hi, y[e]);
                        }
                    }
                    if (by_mass) {
                        over.add(wo);
                        in.add(wi);
                    }
                });
                exchange(sm, R.phase, cluster, rank, by_mass ? over.total() : (double)n_over,
                         by_mass ? in.total() : (double)n_in, n_in, lo, hi);
                if (sm.all.a > 0.0 && above + sm.all.a >= target && b > 0)
                    --b;
                else if ((sm.all.n == 0 || above + sm.all.a + sm.all.b < target) && b < NB - 1)
                    ++b;
                else
                    break;
            }
            const Xch x = sm.all;
            above += x.a;
            ylo = x.lo;
            yhi = x.hi;
            const unsigned n_in = x.n;
            if (n_in == 0) break;  // not reached: the interval holds the crossing element
            if (n_in <= (unsigned)kListCap) {
                // the rest in the list: the crossing element by rank
                if (leader && threadIdx.x == 0) sm.list_n = 0;
                ring::cluster_sync();
                R.each([&](int j, float (&y)[E]) {
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const int64_t i = sl.index(j, e);
                        if (y[e] >= ylo && y[e] <= yhi && keep.ranked(y[e], i))
                            append(sm, y[e], i);
                    }
                });
                ring::cluster_sync();
                if (leader) {
                    sort_list(sm.list, (int)n_in);
                    scan_list(sm, (int)n_in, [&](int i) {
                        return by_mass ? (double)expf(value_of((uint32_t)(sm.list[i] >> 32)) - m) : 1.0;
                    });
                    const int at = first_in_list(sm, (int)n_in, [&](int i) { return above + sm.scan[i] >= target; });
                    if (threadIdx.x == 0) {
                        sm.tau = value_of((uint32_t)(sm.list[at] >> 32));
                        sm.ilim = (int64_t)(uint32_t)~(uint32_t)sm.list[at];
                    }
                }
                ring::cluster_sync();
                uint32_t tb;
                uint64_t ib;
                asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(tb) : "r"(ring::mapa(ring::saddr(&sm.tau), 0)) : "memory");
                asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(ib) : "r"(ring::mapa(ring::saddr(&sm.ilim), 0)) : "memory");
                keep.tau = __uint_as_float(tb);
                keep.ilim = (int64_t)ib;
                ring::cluster_sync();
                break;
            }
            if (ylo == yhi) {
                // all equal: the q-th of them in index order
                const double each_one = by_mass ? (double)expf(ylo - m) : 1.0;
                double q = ceil((target - above) / each_one);
                q = fmin(fmax(q, 1.0), (double)n_in);
                const int64_t nth = (int64_t)q;
                unsigned n = 0;
                R.each([&](int j, float (&y)[E]) {
#pragma unroll
                    for (int e = 0; e < E; ++e)
                        if (y[e] == ylo && keep.ranked(y[e], sl.index(j, e))) ++n;
                });
                exchange(sm, R.phase, cluster, rank, 0.0, 0.0, n, 0.f, 0.f);
                // per warp counts are in sm.wn (exchange's own scratch), in index order
                int64_t run = sm.n_before;
                for (int i = 0; i < warp; ++i) run += sm.wn[i];
                const int64_t have = sm.wn[warp];
                if (leader && threadIdx.x == 0) sm.ilim = -1;
                ring::cluster_sync();
                if (run < nth && nth <= run + have) {
                    for (int j0 = sl.w0; j0 < sl.w1; j0 += 32) {
                        const int j = j0 + lane;
                        unsigned k = 0;
                        float y[E];
                        if (j < sl.w1) {
                            unpack<T>(sl.vec(j), R.s, y);
#pragma unroll
                            for (int e = 0; e < E; ++e)
                                if (y[e] == ylo && keep.ranked(y[e], sl.index(j, e))) ++k;
                        }
                        unsigned incl = k;
#pragma unroll
                        for (int o = 1; o < 32; o <<= 1) {
                            const unsigned t = __shfl_up_sync(0xffffffffu, incl, o);
                            if (lane >= o) incl += t;
                        }
                        int64_t at = run + incl - k;
                        if (k > 0 && at < nth && nth <= at + k) {
                            for (int e = 0; e < E; ++e)
                                if (y[e] == ylo && keep.ranked(y[e], sl.index(j, e)) && ++at == nth) {
                                    const int64_t idx = sl.index(j, e);
                                    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(
                                                     ring::mapa(ring::saddr(&sm.ilim), 0)),
                                                 "l"(idx)
                                                 : "memory");
                                }
                        }
                        run += __shfl_sync(0xffffffffu, incl, 31);
                    }
                }
                ring::cluster_sync();
                uint64_t ib;
                asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(ib) : "r"(ring::mapa(ring::saddr(&sm.ilim), 0)) : "memory");
                keep.tau = ylo;
                keep.ilim = (int64_t)ib;
                ring::cluster_sync();
                break;
            }
            bins = Bins::keys(yhi, ylo);
        }
        if (!by_mass && use_p) {
            Z = R.kept_mass(keep, false);
            bins = Bins::linear(m, fmaxf(keep.tau, floor));
        }
    }
    keep.min_p = min_p > 0.f ? min_p : 0.f;
    const double C = R.kept_mass(keep, false);
    R.draw(keep, false, u * C, C, S, p, row);
    ring::cluster_sync();
}

}  // namespace sample
}  // namespace k1
