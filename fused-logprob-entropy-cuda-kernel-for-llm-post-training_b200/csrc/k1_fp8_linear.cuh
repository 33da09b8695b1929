// k1_fp8_linear.cuh -- matrix product of 8-bit (e4m3) operands with a scale for each block
// of 128: y[m, n] = sum over blocks b of K  xs[m, b] ws[n / 128, b] (xq[m, b] . wq[n, b]).
//
// Both kernels run the block products on the tensor cores (tcgen05.mma kind::f8f6f4, fp32
// sums of one 128-wide block in TMEM, four MMAs of K = 32) from tiles that TMA stages in a
// ring of shared memory (128-byte swizzle: one block of K is one swizzle row), and add the
// blocks in fp32 registers: the epilogue warps read a finished block from TMEM, scale it and
// accumulate it while the tensor cores compute the next one into another TMEM buffer.  The
// scales are any fp32 values, so they cannot be folded into the tensor cores' own
// (power-of-two) scaling.
//
// Few tokens (k1_fp8_skinny_kernel): the bytes of the weight are the work.  The weight's 128
// rows are the MMA's M and the tokens (padded to 16, 32 or 64) its N, so no tensor work is
// spent on rows that are not there.  Blocks of threads are small enough for two or three per
// SM, which keeps the weight stream going while one of them starts or ends; K is split over
// a cluster of up to 8 when the weight has too few rows to fill the SMs, and the parts are
// added through distributed shared memory in rank order (no atomics).
//
// Many tokens (k1_fp8_wide_kernel): 128 tokens x 256 rows of the weight per tile, one
// persistent block per SM.  A thread owns one token and 128 columns (one block of weight
// rows, so its scale is one product per block), 128 accumulators in registers.
//
// Every mbarrier wait is bounded; one that runs out sets bit 4 of the wait status word, and
// the outputs that could not be finished are NaN.
#pragma once

#include "k1_common.cuh"
#include "k1_tc.cuh"

namespace k1 {
namespace fp8 {

using namespace tc;

constexpr int BK = 128;       // one scale block of K: 128 bytes, one swizzle row
constexpr int UK = 32;        // K per tcgen05.mma (kind::f8f6f4)
constexpr int BM = 128;       // TMEM lanes
constexpr int kAbortBit = 16;

// Instruction descriptor, kind::f8f6f4: D fp32 (bits 4-5 = 1), A and B e4m3 (bits 7-9 and
// 10-12 = 0), both K-major, N >> 3 at bits 17-22, M >> 4 at bits 24-28.
template <int N>
constexpr uint32_t kIdesc = (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);

template <int N>
__device__ __forceinline__ void umma8(uint32_t tmem_d, uint64_t da, uint64_t db, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
        "l"(da), "l"(db), "r"(kIdesc<N>), "r"(acc));
}

template <int COLS>
__device__ __forceinline__ void tmem_alloc(uint32_t* slot) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     ring::saddr(slot)),
                 "r"(COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
template <int COLS>
__device__ __forceinline__ void tmem_free(uint32_t tmem) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(COLS)
                 : "memory");
}

__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, volatile int* abort) {
    for (int i = 0; i < ring::kMaxTries; ++i) {
        if (ring::try_wait(bar, parity)) return true;
        if (*abort) return false;
    }
    atomicOr(&k1_ring_error, (unsigned)kAbortBit);
    *abort = 1;
    return false;
}

// 16 consecutive fp32 columns of this thread's TMEM lane (warp-collective).
template <int OFF, int N>
__device__ __forceinline__ void tmem_ld16_async(uint32_t taddr, uint32_t (&r)[N]) {
    static_assert(OFF + 16 <= N, "destination too small");
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[OFF + 0]), "=r"(r[OFF + 1]), "=r"(r[OFF + 2]), "=r"(r[OFF + 3]), "=r"(r[OFF + 4]),
          "=r"(r[OFF + 5]), "=r"(r[OFF + 6]), "=r"(r[OFF + 7]), "=r"(r[OFF + 8]), "=r"(r[OFF + 9]),
          "=r"(r[OFF + 10]), "=r"(r[OFF + 11]), "=r"(r[OFF + 12]), "=r"(r[OFF + 13]),
          "=r"(r[OFF + 14]), "=r"(r[OFF + 15])
        : "r"(taddr));
}

struct Params {
    const float* xs;  // [m, kb_total]
    const float* ws;  // [ceil(n / 128), kb_total]
    void* y;          // [m] rows of ldy elements
    int64_t m, n, ldy;
    int kb_total;     // ceil(k / 128)
    int m_blocks, n_tiles;
};

// ------------------------------------------------------------------------------------
// Few tokens
// ------------------------------------------------------------------------------------
template <int TN>
struct Skinny {
    static constexpr int W_BYTES = BM * BK;           // 16 KB
    static constexpr int X_BYTES = TN * BK;
    static constexpr int STAGE = W_BYTES + X_BYTES;
    static constexpr int STAGES = 4;
    static constexpr int NBUF = TN <= 32 ? 4 : 2;     // TMEM buffers
    static constexpr int COLS = NBUF * TN;            // 64, 128, 128
    static constexpr int THREADS = 192;
    static constexpr int RING = STAGES * STAGE;
    // ring (1024-byte aligned), barriers, scales [blocks of this CTA][TN]
    static constexpr size_t smem(int kb) { return 1024 + RING + 256 + (size_t)kb * TN * 4; }
};

template <int TN, typename OutT>
__global__ void __launch_bounds__(192)
    k1_fp8_skinny_kernel(const __grid_constant__ CUtensorMap tmap_x,
                         const __grid_constant__ CUtensorMap tmap_w, Params p, int split) {
    using S = Skinny<TN>;
    extern __shared__ __align__(16) unsigned char sk_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>(
        (reinterpret_cast<uintptr_t>(sk_raw) + 1023) & ~(uintptr_t)1023);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::RING);
    uint64_t* empty = full + S::STAGES;
    uint64_t* tfull = empty + S::STAGES;
    uint64_t* tempty = tfull + S::NBUF;
    uint64_t* drain = tempty + S::NBUF;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
    volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
    float* scales = reinterpret_cast<float*>(smem + S::RING + 256);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = split > 1 ? (int)ring::cluster_rank() : 0;
    const int tile = blockIdx.x / split;  // 128 rows of the weight
    const int tok0 = blockIdx.y * TN;
    const int kb0 = (int)((int64_t)rank * p.kb_total / split);
    const int kb1 = (int)((int64_t)(rank + 1) * p.kb_total / split);
    if (threadIdx.x == 0) {
        for (int s = 0; s < S::STAGES; ++s) {
            ring::bar_init(&full[s], 1);
            ring::bar_init(&empty[s], 1);
        }
        for (int a = 0; a < S::NBUF; ++a) {
            ring::bar_init(&tfull[a], 1);
            ring::bar_init(&tempty[a], 128);
        }
        ring::bar_init(drain, 1);
        *abort = 0;
        ring::fence_init();
        prefetch_tmap(&tmap_x);
        prefetch_tmap(&tmap_w);
    }
    if (warp == 1) tmem_alloc<S::COLS>(tmem_slot);
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_wait();
    pdl_trigger();

    if (warp == 0) {
        if (lane == 0) {
            bool ok = true;
            int issued = 0;
            for (int kb = kb0; kb < kb1; ++kb, ++issued) {
                const int s = issued % S::STAGES;
                if (!wait(&empty[s], ((issued / S::STAGES) & 1) ^ 1u, abort)) {
                    ok = false;
                    break;
                }
#ifdef K1_WAIT_TEST
                if (blockIdx.x == 0 && blockIdx.y == 0 && (long long)issued == k1_test_withhold) {
                    ok = false;  // test only: block 0 issues nothing more
                    break;
                }
#endif
                unsigned char* st = smem + s * S::STAGE;
                ring::arrive_expect(&full[s], S::STAGE);
                tma_load_2d(st, &tmap_w, kb * BK, tile * BM, &full[s]);
                tma_load_2d(st + S::W_BYTES, &tmap_x, kb * BK, tok0, &full[s]);
            }
            if (!ok)  // stopping early: wait (bounded) for the copies in flight
                for (int i = issued > S::STAGES ? issued - S::STAGES : 0; i < issued; ++i)
                    ring::wait(&full[i % S::STAGES], (i / S::STAGES) & 1);
        }
        __syncwarp();
        if (split > 1) asm volatile("bar.arrive 2, 160;" ::: "memory");  // no copy is in flight
    } else if (warp == 1) {
        if (lane == 0) {
            const uint32_t base = ring::saddr(smem);
            for (int i = 0; i < kb1 - kb0; ++i) {
                const int s = i % S::STAGES, a = i % S::NBUF;
                if (!wait(&tempty[a], ((i / S::NBUF) & 1) ^ 1u, abort)) break;
                if (!wait(&full[s], (i / S::STAGES) & 1, abort)) break;
                tc_fence_after();
                const uint64_t dw = smem_desc(base + s * S::STAGE);
                const uint64_t dx = smem_desc(base + s * S::STAGE + S::W_BYTES);
#pragma unroll
                for (int k = 0; k < BK / UK; ++k)  // +32 bytes per K slice: +2 in >> 4 units
                    umma8<TN>(tmem + (uint32_t)(a * TN), dw + 2 * k, dx + 2 * k, k > 0 ? 1u : 0u);
                umma_commit(&empty[s]);
                umma_commit(&tfull[a]);
            }
            umma_commit(drain);  // every MMA issued has completed before the TMEM is freed
            ring::wait(drain, 0);
        }
    } else {
        // each thread owns one row of the weight (a TMEM lane) and all TN tokens
        const int t = threadIdx.x - 64;
        const int quarter = warp & 3;
        const int row = quarter * 32 + lane;
        const uint32_t tlane = tmem + ((uint32_t)(quarter * 32) << 16);
        const int nkb = kb1 - kb0;
        const float* ws = p.ws + (int64_t)tile * p.kb_total + kb0;
        for (int i = t; i < nkb * TN; i += 128) {
            const int tok = i / nkb, kb = i - tok * nkb;
            const int64_t m = tok0 + tok;
            scales[kb * TN + tok] =
                m < p.m ? __ldg(p.xs + m * p.kb_total + kb0 + kb) * __ldg(ws + kb) : 0.f;
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");
        float acc[TN];
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[j] = 0.f;
        for (int i = 0; i < nkb; ++i) {
            const int a = i % S::NBUF;
            // warp-uniform: the TMEM loads below are warp-collective
            if (!__all_sync(0xffffffffu, wait(&tfull[a], (i / S::NBUF) & 1, abort))) {
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[j] = __int_as_float(0x7fc00000);
                break;
            }
            tc_fence_after();
            uint32_t r[TN];
            tmem_ld16_async<0>(tlane + (uint32_t)(a * TN), r);
            if constexpr (TN >= 32) tmem_ld16_async<16 % TN>(tlane + (uint32_t)(a * TN + 16), r);
            if constexpr (TN >= 64) {
                tmem_ld16_async<32 % TN>(tlane + (uint32_t)(a * TN + 32), r);
                tmem_ld16_async<48 % TN>(tlane + (uint32_t)(a * TN + 48), r);
            }
            tmem_wait();
            tc_fence_before();
            ring::arrive(&tempty[a]);
            const float4* sc = reinterpret_cast<const float4*>(scales + i * TN);
#pragma unroll
            for (int j = 0; j < TN; j += 4) {
                const float4 f = sc[j / 4];
                acc[j] = fmaf(__uint_as_float(r[j]), f.x, acc[j]);
                acc[j + 1] = fmaf(__uint_as_float(r[j + 1]), f.y, acc[j + 1]);
                acc[j + 2] = fmaf(__uint_as_float(r[j + 2]), f.z, acc[j + 2]);
                acc[j + 3] = fmaf(__uint_as_float(r[j + 3]), f.w, acc[j + 3]);
            }
        }
        const int64_t col = (int64_t)tile * BM + row;
        OutT* y = reinterpret_cast<OutT*>(p.y);
        if (split == 1) {
            if (col < p.n)
#pragma unroll
                for (int j = 0; j < TN; ++j)
                    if (tok0 + j < p.m) DT<OutT>::store1(y + (tok0 + j) * p.ldy + col, acc[j]);
        } else {
            // the ring is done with: every stage was consumed before the last block's sums (or,
            // after a wait that ran out, the producer has waited for its copies)
            asm volatile("bar.sync 2, 160;" ::: "memory");
            float* part = reinterpret_cast<float*>(smem);
#pragma unroll
            for (int j = 0; j < TN; ++j) part[j * BM + row] = acc[j];
        }
    }
    __syncwarp();
    tc_fence_before();
    if (split > 1) {
        ring::cluster_sync();  // every rank's part is in its shared memory
        if (warp >= 2) {
            // rank r finishes tokens r, r + split, ...: the parts added in rank order
            const int row = (warp & 3) * 32 + lane;
            const int64_t col = (int64_t)tile * BM + row;
            const uint32_t mine = ring::saddr(smem) + (uint32_t)row * 4;
            for (int j = rank; j < TN; j += split) {
                float v = 0.f;
                for (int r = 0; r < split; ++r) {
                    float f;
                    asm volatile("ld.shared::cluster.f32 %0, [%1];"
                                 : "=f"(f)
                                 : "r"(ring::mapa(mine + (uint32_t)j * BM * 4, r)));
                    v += f;
                }
                if (col < p.n && tok0 + j < p.m)
                    DT<OutT>::store1(reinterpret_cast<OutT*>(p.y) + (tok0 + j) * p.ldy + col, v);
            }
        }
        ring::cluster_sync();  // no rank leaves while its part may be read
    } else {
        __syncthreads();
    }
    tc_fence_after();
    __syncwarp();
    if (warp == 1) tmem_free<S::COLS>(tmem);
}

// ------------------------------------------------------------------------------------
// Many tokens
// ------------------------------------------------------------------------------------
struct Wide {
    static constexpr int BN = 256;
    static constexpr int X_BYTES = BM * BK;  // 16 KB
    static constexpr int W_BYTES = BN * BK;  // 32 KB
    static constexpr int STAGE = X_BYTES + W_BYTES;
    static constexpr int STAGES = 4;
    static constexpr int NBUF = 2;
    static constexpr int COLS = NBUF * BN;   // 512: all of TMEM
    static constexpr int EPI_WARPS = 8;
    static constexpr int THREADS = (2 + EPI_WARPS) * 32;
    static constexpr int GROUP_M = 16;       // token blocks that share the weight tiles in L2
    static constexpr int SMEM = 1024 + STAGES * STAGE + 256;
};

// Tiles in groups of GROUP_M token blocks, token block fastest.
__device__ __forceinline__ void wide_tile(const Params& p, int u, int& mb, int& nt) {
    const int per_group = Wide::GROUP_M * p.n_tiles;
    const int g = u / per_group, r = u - g * per_group;
    const int rows = min(Wide::GROUP_M, p.m_blocks - g * Wide::GROUP_M);
    nt = r / rows;
    mb = g * Wide::GROUP_M + (r - nt * rows);
}

// 32 columns of one row, `valid` of them.
template <typename OutT>
__device__ __forceinline__ void store_row32(OutT* dst, const float* v, int valid, bool vec) {
    if (vec && valid >= 32) {
        if constexpr (sizeof(OutT) == 4) {
#pragma unroll
            for (int i = 0; i < 32; i += 4)
                *reinterpret_cast<float4*>(dst + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        } else {
#pragma unroll
            for (int i = 0; i < 32; i += 8)
                *reinterpret_cast<uint4*>(dst + i) =
                    make_uint4(DT<OutT>::from_f2(make_float2(v[i], v[i + 1])),
                               DT<OutT>::from_f2(make_float2(v[i + 2], v[i + 3])),
                               DT<OutT>::from_f2(make_float2(v[i + 4], v[i + 5])),
                               DT<OutT>::from_f2(make_float2(v[i + 6], v[i + 7])));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 32; ++i)
            if (i < valid) DT<OutT>::store1(dst + i, v[i]);
    }
}

template <typename OutT>
__global__ void __launch_bounds__(Wide::THREADS, 1)
    k1_fp8_wide_kernel(const __grid_constant__ CUtensorMap tmap_x,
                       const __grid_constant__ CUtensorMap tmap_w, Params p) {
    using S = Wide;
    extern __shared__ __align__(16) unsigned char wd_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>(
        (reinterpret_cast<uintptr_t>(wd_raw) + 1023) & ~(uintptr_t)1023);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::STAGES * S::STAGE);
    uint64_t* empty = full + S::STAGES;
    uint64_t* tfull = empty + S::STAGES;
    uint64_t* tempty = tfull + S::NBUF;
    uint64_t* drain = tempty + S::NBUF;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
    volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int units = p.m_blocks * p.n_tiles;
    if (threadIdx.x == 0) {
        for (int s = 0; s < S::STAGES; ++s) {
            ring::bar_init(&full[s], 1);
            ring::bar_init(&empty[s], 1);
        }
        for (int a = 0; a < S::NBUF; ++a) {
            ring::bar_init(&tfull[a], 1);
            ring::bar_init(&tempty[a], S::EPI_WARPS * 32);
        }
        ring::bar_init(drain, 1);
        *abort = 0;
        ring::fence_init();
        prefetch_tmap(&tmap_x);
        prefetch_tmap(&tmap_w);
    }
    if (warp == 1) tmem_alloc<S::COLS>(tmem_slot);
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_wait();
    pdl_trigger();

    if (warp == 0) {
        if (lane == 0) {
            bool ok = true;
            uint32_t issued = 0;
            for (int u = blockIdx.x; ok && u < units; u += gridDim.x) {
                int mb, nt;
                wide_tile(p, u, mb, nt);
                for (int kb = 0; kb < p.kb_total; ++kb, ++issued) {
                    const int s = issued % S::STAGES;
                    if (!wait(&empty[s], ((issued / S::STAGES) & 1) ^ 1u, abort)) {
                        ok = false;
                        break;
                    }
#ifdef K1_WAIT_TEST
                    if (blockIdx.x == 0 && (long long)issued == k1_test_withhold) {
                        ok = false;  // test only: block 0 issues nothing more
                        break;
                    }
#endif
                    unsigned char* st = smem + s * S::STAGE;
                    ring::arrive_expect(&full[s], S::STAGE);
                    tma_load_2d(st, &tmap_x, kb * BK, mb * BM, &full[s]);
                    tma_load_2d(st + S::X_BYTES, &tmap_w, kb * BK, nt * S::BN, &full[s]);
                }
            }
            if (!ok)
                for (uint32_t i = issued > S::STAGES ? issued - S::STAGES : 0; i < issued; ++i)
                    ring::wait(&full[i % S::STAGES], (i / S::STAGES) & 1);
        }
    } else if (warp == 1) {
        if (lane == 0) {
            const uint32_t base = ring::saddr(smem);
            uint32_t i = 0;
            bool ok = true;
            for (int u = blockIdx.x; ok && u < units; u += gridDim.x) {
                for (int kb = 0; kb < p.kb_total; ++kb, ++i) {
                    const int s = i % S::STAGES, a = i % S::NBUF;
                    if (!wait(&tempty[a], ((i / S::NBUF) & 1) ^ 1u, abort) ||
                        !wait(&full[s], (i / S::STAGES) & 1, abort)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint64_t dx = smem_desc(base + s * S::STAGE);
                    const uint64_t dw = smem_desc(base + s * S::STAGE + S::X_BYTES);
#pragma unroll
                    for (int k = 0; k < BK / UK; ++k)
                        umma8<S::BN>(tmem + (uint32_t)(a * S::BN), dx + 2 * k, dw + 2 * k,
                                     k > 0 ? 1u : 0u);
                    umma_commit(&empty[s]);
                    umma_commit(&tfull[a]);
                }
            }
            umma_commit(drain);
            ring::wait(drain, 0);
        }
    } else {
        const int quarter = warp & 3;          // TMEM lanes 32 quarter ...: tokens
        const int half = (warp - 2) >> 2;      // 128 columns: one block of weight rows
        const uint32_t tlane = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(half * 128);
        const bool vec = (p.ldy * sizeof(OutT)) % 16 == 0 && reinterpret_cast<uintptr_t>(p.y) % 16 == 0;
        uint32_t i = 0;
        bool ok = true;
        for (int u = blockIdx.x; u < units; u += gridDim.x) {
            int mb, nt;
            wide_tile(p, u, mb, nt);
            const int64_t row = (int64_t)mb * BM + quarter * 32 + lane;
            const int64_t col0 = (int64_t)nt * S::BN + half * 128;
            const bool live = row < p.m && col0 < p.n;
            const float* xs = p.xs + (live ? row : 0) * p.kb_total;
            const float* ws = p.ws + (live ? col0 / 128 : 0) * p.kb_total;
            float acc[128];
#pragma unroll
            for (int j = 0; j < 128; ++j) acc[j] = 0.f;
            for (int kb = 0; kb < p.kb_total; ++kb, ++i) {
                const int a = i % S::NBUF;
                const float f = __ldg(xs + kb) * __ldg(ws + kb);
                if (ok && !__all_sync(0xffffffffu, wait(&tfull[a], (i / S::NBUF) & 1, abort)))
                    ok = false;
                if (!ok) break;
                tc_fence_after();
#pragma unroll
                for (int c = 0; c < 128; c += 32) {
                    uint32_t r[32];
                    tmem_ld32_async<0>(tlane + (uint32_t)(a * S::BN + c), r);
                    tmem_wait();
#pragma unroll
                    for (int j = 0; j < 32; ++j)
                        acc[c + j] = fmaf(__uint_as_float(r[j]), f, acc[c + j]);
                }
                tc_fence_before();
                ring::arrive(&tempty[a]);
            }
            if (!ok)  // a wait ran out: this tile and the block's later ones are NaN
#pragma unroll
                for (int j = 0; j < 128; ++j) acc[j] = __int_as_float(0x7fc00000);
            if (live) {
                OutT* y = reinterpret_cast<OutT*>(p.y) + row * p.ldy + col0;
#pragma unroll
                for (int c = 0; c < 128; c += 32) {
                    const int64_t left = p.n - col0 - c;
                    if (left > 0) store_row32<OutT>(y + c, acc + c, left < 32 ? (int)left : 32, vec);
                }
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    __syncwarp();
    if (warp == 1) tmem_free<S::COLS>(tmem);
}

}  // namespace fp8
}  // namespace k1
