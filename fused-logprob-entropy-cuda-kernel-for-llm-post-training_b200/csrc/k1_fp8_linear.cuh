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
// Many tokens (k1_fp8_wide_kernel): 256 tokens x 256 rows of the weight per tile and pair of
// CTAs, persistent.  A thread owns one token and 128 columns (one block of weight rows, so its
// scale is one product per block), 128 accumulators in registers; it loads the next 32
// columns from TMEM while it adds the last.
//
// Measured on B200: 1 x 3584 x 152064 83 us (the weight's bytes at 6.6 TB/s, the measured copy
// rate), 64 x 3584 x 128256 101 to 103 us (4.6 to 4.7 TB/s: the last round of blocks and the 64-column epilogue
// between loads), 2048 x 3584 x 32768 285 to 295 us (1.63 to 1.69 PFLOP/s: adding the blocks in
// fp32 takes about 40 us of it that the tensor cores do not hide, and a block of K's
// handshakes, tile copies and operand reads fill what the MMAs leave of shared memory's
// bandwidth).
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

// Bounded wait on the barrier at a shared-memory address.
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, volatile int* abort) {
    for (int i = 0; i < ring::kMaxTries; ++i) {
        if (ring::try_wait_at(bar, parity)) return true;
        if (*abort) return false;
    }
    atomicOr(&k1_ring_error, (unsigned)kAbortBit);
    *abort = 1;
    return false;
}

// The same for a converged warp, true where all lanes saw the phase complete: lanes whose limit ran
// out and lanes whose poll came after the completion must not part before the warp's next elect or
// TMEM load.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort) {
    return __all_sync(0xffffffffu, wait(bar, parity, abort));
}

// A place in a ring of N slots and the parity of its current round.
template <int N>
struct Place {
    uint32_t slot = 0, parity = 0;
    __device__ __forceinline__ void next() {
        if (++slot == N) {
            slot = 0;
            parity ^= 1u;
        }
    }
};

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

// Wait for this thread's TMEM loads; tied to the registers of one, so that nothing that reads
// them is moved ahead of the wait.
__device__ __forceinline__ void tmem_wait_on(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]),
                   "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]),
                   "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]),
                   "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]),
                   "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_wait_on(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]),
                   "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]),
                   "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}

// Asynchronous copy of 4 bytes into shared memory (zeros where not live).
__device__ __forceinline__ void copy4(uint32_t dst, const float* src, bool live) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(live ? 4 : 0)
                 : "memory");
}

struct Params {
    const float* xs;  // [m, kb_total]
    const float* ws;  // [ceil(n / 128), kb_total]
    void* y;          // [m] rows of ldy elements
    int64_t m, n, ldy;
    int kb_total;     // ceil(k / 128)
    int m_tiles, n_tiles;  // many tokens: tiles of 256 x 256
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
    static constexpr int GROUPS = TN <= 32 ? 1 : TN / 32;  // epilogue groups of 4 warps
    static constexpr int CW = TN / GROUPS;                 // tokens per group: 16 or 32
    static constexpr int THREADS = 64 + GROUPS * 128;
    static constexpr int RING = STAGES * STAGE;
    // ring (1024-byte aligned), barriers, scales [blocks of this CTA][TN]
    static constexpr size_t smem(int kb) { return 1024 + RING + 256 + (size_t)kb * TN * 4; }
};

// Two consecutive 16-bit elements in one store.
template <typename OutT>
__device__ __forceinline__ void store_pair(OutT* dst, float a, float b) {
    if constexpr (sizeof(OutT) == 2) *reinterpret_cast<uint32_t*>(dst) = DT<OutT>::from_f2(make_float2(a, b));
}

template <int TN, typename OutT>
__global__ void __launch_bounds__(Skinny<TN>::THREADS, TN <= 32 ? 3 : 2)
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
    // token blocks of one tile (128 rows of the weight) run side by side: the weight comes from
    // HBM once and from L2 for the others
    const int tok_blocks = (int)((p.m + TN - 1) / TN);
    const int tile = (int)(blockIdx.x / split) / tok_blocks;
    const int tok0 = ((int)(blockIdx.x / split) - tile * tok_blocks) * TN;
    const int kb0 = (int)((int64_t)rank * p.kb_total / split);
    const int kb1 = (int)((int64_t)(rank + 1) * p.kb_total / split);
    if (threadIdx.x == 0) {
        for (int s = 0; s < S::STAGES; ++s) {
            ring::bar_init(&full[s], 1);
            ring::bar_init(&empty[s], 1);
        }
        for (int a = 0; a < S::NBUF; ++a) {
            ring::bar_init(&tfull[a], 1);
            ring::bar_init(&tempty[a], 4 * S::GROUPS);  // one arrival per epilogue warp
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

    // shared-memory addresses
    const uint32_t a_ring = ring::saddr(smem), a_full = ring::saddr(full), a_empty = ring::saddr(empty),
                   a_tfull = ring::saddr(tfull), a_tempty = ring::saddr(tempty);
    // One elected lane walks the producer's loop, and one the issuer's: it waits and issues.  (A whole
    // warp that elects a lane at every block of K would have to vote on each bounded wait, so that
    // its lanes stop together: 64 x 3584 x 128256 102.5 us with one lane, 104.6 with votes.)
    if (warp == 0) {
        if (ring::elect_one()) {
            Place<S::STAGES> at;
            bool ok = true;
            int issued = 0;
            for (int kb = kb0; kb < kb1; ++kb, ++issued, at.next()) {
                if (!wait(a_empty + at.slot * 8, at.parity ^ 1u, abort)) {
                    ok = false;
                    break;
                }
#ifdef K1_WAIT_TEST
                if (blockIdx.x == 0 && (long long)issued == k1_test_withhold) {
                    ok = false;  // test only: block 0 issues nothing more
                    break;
                }
#endif
                const uint32_t st = a_ring + at.slot * S::STAGE, bar = a_full + at.slot * 8;
                ring::arrive_expect(&full[at.slot], S::STAGE);
                tma_load_2d_at(st, &tmap_w, kb * BK, tile * BM, bar);
                tma_load_2d_at(st + S::W_BYTES, &tmap_x, kb * BK, tok0, bar);
            }
            if (!ok)  // stopping early: wait (bounded) for the copies in flight
                for (int i = issued > S::STAGES ? issued - S::STAGES : 0; i < issued; ++i)
                    ring::wait(&full[i % S::STAGES], (i / S::STAGES) & 1);
        }
        __syncwarp();
        if (split > 1)  // no copy is in flight
            asm volatile("bar.arrive 2, %0;" ::"n"(S::GROUPS * 128 + 32) : "memory");
    } else if (warp == 1) {
        if (ring::elect_one()) {
            Place<S::STAGES> at;
            Place<S::NBUF> acc;
            const uint64_t dw0 = smem_desc(a_ring), dx0 = smem_desc(a_ring + S::W_BYTES);
            // both barriers of the next block are tested together, while this one's MMAs run
            bool freed = true, there = false;
            for (int i = 0; i < kb1 - kb0; ++i) {
                if (!freed && !wait(a_tempty + acc.slot * 8, acc.parity ^ 1u, abort)) break;
                if (!there && !wait(a_full + at.slot * 8, at.parity, abort)) break;
                tc_fence_after();
                const uint64_t dw = dw0 + at.slot * (S::STAGE >> 4), dx = dx0 + at.slot * (S::STAGE >> 4);
                const uint32_t d = tmem + acc.slot * TN;
#pragma unroll
                for (int k = 0; k < BK / UK; ++k)  // +32 bytes per K slice: +2 in >> 4 units
                    umma8<TN>(d, dw + 2 * k, dx + 2 * k, k > 0 ? 1u : 0u);
                umma_commit_at(a_empty + at.slot * 8);
                umma_commit_at(a_tfull + acc.slot * 8);
                at.next();
                acc.next();
                there = ring::test_at(a_full + at.slot * 8, at.parity);
                freed = ring::test_at(a_tempty + acc.slot * 8, acc.parity ^ 1u);
            }
            umma_commit(drain);  // every MMA issued has completed before the TMEM is freed
            ring::wait(drain, 0);
        }
    } else {
        // each thread owns one row of the weight (a TMEM lane) and its group's tokens
        constexpr int CW = S::CW, EPI = S::GROUPS * 128;
        const int t = threadIdx.x - 64;
        const int quarter = warp & 3;
        const int row = quarter * 32 + lane;
        const int j0 = (t >> 7) * CW;  // the group's first token in the block
        const uint32_t tlane = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)j0;
        const int nkb = kb1 - kb0;
        const float* ws = p.ws + (int64_t)tile * p.kb_total + kb0;
        {
            // a thread's token is fixed (TN divides the threads); eight loads in flight
            const int64_t m = tok0 + t % TN;
            const float* xs = p.xs + (m < p.m ? m : 0) * p.kb_total + kb0;
            constexpr int STEP = EPI / TN;
            for (int kb = t / TN; kb < nkb; kb += 8 * STEP) {
                float f[8];
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    f[q] = kb + q * STEP < nkb ? __ldg(xs + kb + q * STEP) * __ldg(ws + kb + q * STEP) : 0.f;
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    if (kb + q * STEP < nkb) scales[(kb + q * STEP) * TN + t % TN] = m < p.m ? f[q] : 0.f;
            }
        }
        asm volatile("bar.sync 1, %0;" ::"n"(EPI) : "memory");
        float acc[CW];
#pragma unroll
        for (int j = 0; j < CW; ++j) acc[j] = 0.f;
        Place<S::NBUF> buf;
        for (int i = 0; i < nkb; ++i, buf.next()) {
            const uint32_t a = buf.slot;
            // warp-uniform: the TMEM loads below are warp-collective
            if (!warp_wait(a_tfull + a * 8, buf.parity, abort)) {
#pragma unroll
                for (int j = 0; j < CW; ++j) acc[j] = __int_as_float(0x7fc00000);
                break;
            }
            tc_fence_after();
            const float4* sc = reinterpret_cast<const float4*>(scales + i * TN + j0);
            uint32_t r[CW];
            if constexpr (CW == 32)
                tmem_ld32_async<0>(tlane + a * TN, r);
            else
                tmem_ld16_async<0>(tlane + a * TN, r);
            tmem_wait_on(r);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) ring::arrive_at(a_tempty + a * 8);
#pragma unroll
            for (int j = 0; j < CW; j += 4) {
                const float4 f = sc[j / 4];
                acc[j] = fmaf(__uint_as_float(r[j]), f.x, acc[j]);
                acc[j + 1] = fmaf(__uint_as_float(r[j + 1]), f.y, acc[j + 1]);
                acc[j + 2] = fmaf(__uint_as_float(r[j + 2]), f.z, acc[j + 2]);
                acc[j + 3] = fmaf(__uint_as_float(r[j + 3]), f.w, acc[j + 3]);
            }
        }
        const int64_t col = (int64_t)tile * BM + row;
        const int tok = tok0 + j0;
        OutT* y = reinterpret_cast<OutT*>(p.y);
        if (split == 1) {
            // 16-bit outputs: two lanes trade, so that each stores two columns of one of two
            // tokens in one word
            const bool paired = sizeof(OutT) == 2 && (p.ldy & 1) == 0 &&
                                (reinterpret_cast<uintptr_t>(y) & 3) == 0 && ((p.n & 1) == 0);
            if (paired) {
                const bool odd = lane & 1;
#pragma unroll
                for (int j = 0; j < CW; j += 2) {
                    const float got = __shfl_xor_sync(0xffffffffu, odd ? acc[j] : acc[j + 1], 1);
                    const int tj = tok + j + odd;
                    if (col < p.n && tj < p.m)
                        store_pair(y + (int64_t)tj * p.ldy + (col - odd), odd ? got : acc[j], odd ? acc[j + 1] : got);
                }
            } else if (col < p.n) {
#pragma unroll
                for (int j = 0; j < CW; ++j)
                    if (tok + j < p.m) DT<OutT>::store1(y + (int64_t)(tok + j) * p.ldy + col, acc[j]);
            }
        } else {
            // the ring is done with: every stage was consumed before the last block's sums (or,
            // after a wait that ran out, the producer has waited for its copies)
            asm volatile("bar.sync 2, %0;" ::"n"(EPI + 32) : "memory");
            float* part = reinterpret_cast<float*>(smem);
#pragma unroll
            for (int j = 0; j < CW; ++j) part[(j0 + j) * BM + row] = acc[j];
        }
    }
    __syncwarp();
    tc_fence_before();
    if (split > 1) {
        ring::cluster_sync();  // every rank's part is in its shared memory
        if (warp >= 2) {
            // rank r finishes tokens r, r + split, ... (dealt to its groups): the parts added in
            // rank order
            const int row = (warp & 3) * 32 + lane;
            const int64_t col = (int64_t)tile * BM + row;
            const uint32_t mine = ring::saddr(smem) + (uint32_t)row * 4;
            for (int j = rank + split * ((warp - 2) >> 2); j < TN; j += split * S::GROUPS) {
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
// A pair of CTAs (two SMs) computes 256 tokens x 256 weight rows with cta_group::2 MMAs: each
// CTA stages its 128 tokens and its 128 of the weight rows and keeps the sums of its tokens.
// One CTA alone with 128 x 256 moves 1.5 times the bytes through its shared memory (48 KB in
// by TMA and 48 KB out to the tensor cores per 512 cycles of MMA, at 128 bytes per cycle).
struct Wide {
    static constexpr int BN = 256;
    static constexpr int TM = 2 * BM;              // tokens per tile
    static constexpr int LOAD_N = BN / 2;          // weight rows per CTA
    static constexpr int X_BYTES = BM * BK;        // 16 KB
    static constexpr int W_BYTES = LOAD_N * BK;    // 16 KB
    static constexpr int STAGE = X_BYTES + W_BYTES;
    static constexpr int STAGES = 6;
    static constexpr int NBUF = 2;
    static constexpr int COLS = NBUF * BN;         // 512: all of TMEM
    static constexpr int EPI_WARPS = 8;
    static constexpr int CPT = BN * 4 / EPI_WARPS; // columns per thread: 128
    static constexpr int THREADS = (4 + EPI_WARPS) * 32;
    // Registers: 384 threads start with 168 each; the first warpgroup goes down to 40 and the
    // other two up to 232 (128 x 40 + 256 x 232 = 384 x 168).
    static constexpr int REGS_DOWN = 40, REGS_UP = 232;
    static constexpr int SB = 32;                  // blocks of K per chunk of token scales
    static constexpr int SROW = BM + 1;            // its row pitch: stores along K meet no bank twice
    static constexpr int S_BYTES = SB * SROW * 4 + SB * 8;  // and the two weight blocks' scales
    static constexpr int GROUP_M = 8;              // token tiles that share the weight tiles in L2
    static constexpr int SMEM = 1024 + STAGES * STAGE + 2 * S_BYTES + 256;
    static constexpr uint32_t IDESC =
        (1u << 4) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(TM >> 4) << 24);
};
static_assert(Wide::SMEM <= 227 * 1024, "shared memory of one block");

// Tiles in groups of GROUP_M token tiles, token tile fastest.
__device__ __forceinline__ void wide_tile(const Params& p, int u, int& mt, int& nt) {
    const int per_group = Wide::GROUP_M * p.n_tiles;
    const int g = u / per_group, r = u - g * per_group;
    const int rows = min(Wide::GROUP_M, p.m_tiles - g * Wide::GROUP_M);
    nt = r / rows;
    mt = g * Wide::GROUP_M + (r - nt * rows);
}

// Transposes 32 x 32 values across a warp: lane l's v[i] becomes lane i's v[l].
__device__ __forceinline__ void warp_transpose(float (&v)[32]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
        const bool up = lane & d;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            if (i & d) continue;
            // the half of each pair that belongs to the other lane
            const float other = __shfl_xor_sync(0xffffffffu, up ? v[i] : v[i + d], d);
            if (up)
                v[i] = other;
            else
                v[i + d] = other;
        }
    }
}

// 32 columns of one row that starts at a multiple of 16 bytes (32 with align32), `valid` of
// them.
template <typename OutT>
__device__ __forceinline__ void store_row32(OutT* dst, const float2* v, int valid, bool align32) {
    if (valid >= 32) {
        constexpr int E = 16 / sizeof(OutT);  // elements of a vector
#pragma unroll
        for (int i = 0; i < 32; i += 2 * E) {
            uint4 w[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float2* s = v + (i + h * E) / 2;
                if constexpr (sizeof(OutT) == 4)
                    w[h] = make_uint4(__float_as_uint(s[0].x), __float_as_uint(s[0].y), __float_as_uint(s[1].x),
                                      __float_as_uint(s[1].y));
                else
                    w[h] = make_uint4(DT<OutT>::from_f2(s[0]), DT<OutT>::from_f2(s[1]),
                                      DT<OutT>::from_f2(s[2 % (E / 2)]), DT<OutT>::from_f2(s[3 % (E / 2)]));
            }
            if (align32) {
                stg32(dst + i, w[0], w[1]);
            } else {
                stg_stream(dst + i, w[0]);
                stg_stream(dst + i + E, w[1]);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if (2 * i < valid) DT<OutT>::store1(dst + 2 * i, v[i].x);
            if (2 * i + 1 < valid) DT<OutT>::store1(dst + 2 * i + 1, v[i].y);
        }
    }
}

// ALIGNED: the output's rows start at multiples of 16 bytes.
template <typename OutT, bool ALIGNED>
__global__ void __launch_bounds__(Wide::THREADS, 1)
    k1_fp8_wide_kernel(const __grid_constant__ CUtensorMap tmap_x,
                       const __grid_constant__ CUtensorMap tmap_w, Params p) {
    using S = Wide;
    extern __shared__ __align__(16) unsigned char wd_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>(
        (reinterpret_cast<uintptr_t>(wd_raw) + 1023) & ~(uintptr_t)1023);
    float* scales = reinterpret_cast<float*>(smem + S::STAGES * S::STAGE);  // two chunks
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::STAGES * S::STAGE + 2 * S::S_BYTES);
    uint64_t* empty = full + S::STAGES;
    uint64_t* tfull = empty + S::STAGES;
    uint64_t* tempty = tfull + S::NBUF;
    uint64_t* sfull = tempty + S::NBUF;
    uint64_t* sempty = sfull + 2;
    uint64_t* drain = sempty + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
    volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = ring::cluster_rank();  // 0: issues the pair's MMAs
    const bool leader = rank == 0;
    const int units = p.m_tiles * p.n_tiles;
    const int first = blockIdx.x >> 1, step = gridDim.x >> 1;
    if (threadIdx.x == 0) {
        for (int s = 0; s < S::STAGES; ++s) {
            ring::bar_init(&full[s], 2);  // both producers arrive at the leader's
            ring::bar_init(&empty[s], 1);
        }
        for (int a = 0; a < S::NBUF; ++a) {
            ring::bar_init(&tfull[a], 1);
            ring::bar_init(&tempty[a], 2 * S::EPI_WARPS);  // at the leader's, one per warp of both
        }
        for (int a = 0; a < 2; ++a) {
            ring::bar_init(&sfull[a], 1);
            ring::bar_init(&sempty[a], S::EPI_WARPS);
        }
        ring::bar_init(drain, 1);
        *abort = 0;
        ring::fence_init();
        prefetch_tmap(&tmap_x);
        prefetch_tmap(&tmap_w);
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         ring::saddr(tmem_slot)),
                     "r"(S::COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    __syncwarp();
    tc_fence_before();
    ring::cluster_sync();  // both CTAs' barriers are initialised before any remote arrival
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_wait();
    pdl_trigger();

    // shared-memory addresses
    const uint32_t a_ring = ring::saddr(smem), a_full = ring::saddr(full), a_empty = ring::saddr(empty),
                   a_tfull = ring::saddr(tfull), a_tempty = ring::saddr(tempty), a_sfull = ring::saddr(sfull),
                   a_sempty = ring::saddr(sempty), a_scales = ring::saddr(scales);

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::REGS_DOWN));
        if (warp == 0) {
            // ---------------- TMA producer (each CTA's own tiles) ----------------
            Place<S::STAGES> at;
            bool ok = true;
            uint32_t issued = 0;
            const uint32_t cl_full = ring::mapa(a_full, 0);  // the leader's barriers
            if (ring::elect_one()) {
                for (int u = first; ok && u < units; u += step) {
                    int mt, nt;
                    wide_tile(p, u, mt, nt);
                    const int row_x = mt * S::TM + (int)rank * BM;
                    const int row_w = nt * S::BN + (int)rank * S::LOAD_N;
                    for (int kb = 0; kb < p.kb_total; ++kb, ++issued, at.next()) {
                        if (!wait(a_empty + at.slot * 8, at.parity ^ 1u, abort)) {
                            ok = false;
                            break;
                        }
#ifdef K1_WAIT_TEST
                        if (blockIdx.x == 0 && (long long)issued == k1_test_withhold) {
                            ok = false;  // test only: block 0 issues nothing more
                            break;
                        }
#endif
                        const uint32_t st = a_ring + at.slot * S::STAGE, cl = cl_full + at.slot * 8;
                        tma_load_2d_pair_at(st, &tmap_x, kb * BK, row_x, cl);
                        tma_load_2d_pair_at(st + S::X_BYTES, &tmap_w, kb * BK, row_w, cl);
                        if (leader)
                            ring::arrive_expect(&full[at.slot], 2 * S::STAGE);
                        else
                            ring::arrive_remote(cl);
                    }
                }
                // Stopping early: wait (bounded) for the copies in flight.  They are counted on the
                // leader's barriers, which the other CTA cannot wait on: it stays about a millisecond,
                // a hundred times what a tile takes, before it lets its shared memory go.
                if (!ok && leader)
                    for (uint32_t i = issued > S::STAGES ? issued - S::STAGES : 0; i < issued; ++i)
                        ring::wait(&full[i % S::STAGES], (i / S::STAGES) & 1);
                else if (!ok)
                    for (long long i = 0, t = clock64(); i < 1000 && clock64() - t < 2000000; ++i) __nanosleep(2000);
            }
        } else if (warp == 1) {
            // ---------------- MMA issuer (the leader, for both) ----------------
            if (leader && ring::elect_one()) {
                Place<S::STAGES> at;
                Place<S::NBUF> acc;
                bool ok = true;
                const uint64_t dx0 = smem_desc(a_ring), dw0 = smem_desc(a_ring + S::X_BYTES);
                // both barriers of the next block are tested together, while this one's MMAs run
                bool freed = true, there = false;
                for (int u = first; ok && u < units; u += step) {
                    for (int kb = 0; kb < p.kb_total; ++kb) {
                        if ((!freed && !wait(a_tempty + acc.slot * 8, acc.parity ^ 1u, abort)) ||
                            (!there && !wait(a_full + at.slot * 8, at.parity, abort))) {
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                        const uint64_t dx = dx0 + at.slot * (S::STAGE >> 4), dw = dw0 + at.slot * (S::STAGE >> 4);
                        const uint32_t d = tmem + acc.slot * S::BN;
#pragma unroll
                        for (int k = 0; k < BK / UK; ++k)
                            asm volatile(
                                "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                                "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
                                "l"(dx + 2 * k), "l"(dw + 2 * k), "r"(S::IDESC), "r"(k > 0 ? 1u : 0u));
                        umma_commit_pair_at(a_empty + at.slot * 8);
                        umma_commit_pair_at(a_tfull + acc.slot * 8);
                        at.next();
                        acc.next();
                        there = ring::test_at(a_full + at.slot * 8, at.parity);
                        freed = ring::test_at(a_tempty + acc.slot * 8, acc.parity ^ 1u);
                    }
                }
                umma_commit_pair(drain);  // every MMA issued has completed before the TMEM is freed
                ring::wait(drain, 0);
            }
        } else if (warp == 2) {
            // ---------------- scales: tokens transposed, [K block][token], and weight ----------------
            // Straight from global memory the epilogue's 32 lanes (32 tokens) would read 32
            // rows for one block of K: 32 wavefronts per load instead of one.
            Place<2> at;
            bool ok = true;
            for (int u = first; ok && u < units; u += step) {
                int mt, nt;
                wide_tile(p, u, mt, nt);
                const int64_t m0 = (int64_t)mt * S::TM + (int64_t)rank * BM;
                const int rows = (int)max((int64_t)0, min((int64_t)BM, p.m - m0));
                const int64_t nb = (int64_t)nt * 2, nb_last = (p.n - 1) / 128;
                for (int k0 = 0; k0 < p.kb_total; k0 += S::SB, at.next()) {
                    if (!warp_wait(a_sempty + at.slot * 8, at.parity ^ 1u, abort)) {
                        ok = false;
                        break;
                    }
                    // asynchronous copies: all of a chunk in flight at once
                    const bool in = k0 + lane < p.kb_total;
                    const float* src = p.xs + (in ? m0 * p.kb_total + k0 + lane : 0);
                    const uint32_t chunk = a_scales + at.slot * S::S_BYTES;
                    const uint32_t dst = chunk + lane * (S::SROW * 4);
#pragma unroll 8
                    for (int r = 0; r < BM; ++r) {
                        const bool live = in && r < rows;
                        copy4(dst + r * 4, live ? src + (int64_t)r * p.kb_total : p.xs, live);
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        copy4(chunk + (S::SB * S::SROW + 2 * lane + h) * 4,
                              p.ws + (in ? min(nb + h, nb_last) * p.kb_total + k0 + lane : 0), in);
                    asm volatile("cp.async.wait_all;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) ring::arrive_at(a_sfull + at.slot * 8);
                }
            }
        }
    } else {
        // ---------------- epilogue (each CTA's own 128 tokens) ----------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(S::REGS_UP));
        constexpr int CPT = S::CPT;
        const int quarter = warp & 3;          // TMEM lanes 32 quarter ...: tokens
        const int part = (warp - 4) >> 2;      // CPT columns: one block of weight rows
        const int rloc = quarter * 32 + lane;
        const uint32_t tlane = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(part * CPT);
        const bool align32 =
            ((reinterpret_cast<uintptr_t>(p.y) | (uintptr_t)(p.ldy * sizeof(OutT))) & 31) == 0;
        const uint32_t cl_tempty = ring::mapa(a_tempty, 0);  // the leader's barriers
        static_assert(CPT == 128 && S::NBUF == 2, "four loads of 32 columns per block of K");
        uint32_t buf = 0, parity = 0;
        Place<2> chunk;
        bool ok = true;
        for (int u = first; u < units; u += step) {
            int mt, nt;
            wide_tile(p, u, mt, nt);
            const int64_t row = (int64_t)mt * S::TM + (int64_t)rank * BM + rloc;
            const int64_t col0 = (int64_t)nt * S::BN + part * CPT;
            float2 acc[CPT / 2];
#pragma unroll
            for (int j = 0; j < CPT / 2; ++j) acc[j] = make_float2(0.f, 0.f);
            uint32_t ra[32], rb[32];
            auto add = [&](int c0, const uint32_t (&r)[32], float2 g) {
#pragma unroll
                for (int j = 0; j < 32; j += 2)
                    acc[(c0 + j) / 2] =
                        fma2(make_float2(__uint_as_float(r[j]), __uint_as_float(r[j + 1])), g, acc[(c0 + j) / 2]);
            };
            for (int k0 = 0; ok && k0 < p.kb_total; k0 += S::SB, chunk.next()) {
                // warp-uniform: the TMEM loads are warp-collective
                ok = warp_wait(a_sfull + chunk.slot * 8, chunk.parity, abort);
                if (!ok) break;
                const float* sx = scales + chunk.slot * (S::S_BYTES / 4) + rloc;
                const float* sw = scales + chunk.slot * (S::S_BYTES / 4) + S::SB * S::SROW + part;
                const int n = min(S::SB, p.kb_total - k0);
                for (int kc = 0; kc < n; ++kc) {
                    const float2 f = splat(sx[kc * S::SROW] * sw[2 * kc]);
                    if (!warp_wait(a_tfull + buf * 8, parity, abort)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    // the next 32 columns are loaded while the last ones are added
                    const uint32_t t = tlane + buf * S::BN;
                    tmem_ld32_async<0>(t, ra);
                    tmem_wait_on(ra);
                    tmem_ld32_async<0>(t + 32, rb);
                    add(0, ra, f);
                    tmem_wait_on(rb);
                    tmem_ld32_async<0>(t + 64, ra);
                    add(32, rb, f);
                    tmem_wait_on(ra);
                    tmem_ld32_async<0>(t + 96, rb);
                    add(64, ra, f);
                    tmem_wait_on(rb);
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) ring::arrive_remote(cl_tempty + buf * 8);
                    buf ^= 1u;
                    parity ^= buf ^ 1u;
                    add(96, rb, f);
                }
                __syncwarp();
                if (lane == 0) ring::arrive_at(a_sempty + chunk.slot * 8);
            }
            if (!ok) {  // a wait ran out: this tile and the CTA's later ones are NaN
#pragma unroll
                for (int j = 0; j < CPT / 2; ++j) acc[j] = splat(__int_as_float(0x7fc00000));
            }
            if constexpr (ALIGNED) {
                if (row < p.m) {
                    OutT* y = reinterpret_cast<OutT*>(p.y) + row * p.ldy + col0;
#pragma unroll
                    for (int c0 = 0; c0 < CPT; c0 += 32) {
                        const int64_t left = p.n - col0 - c0;
                        if (left > 0) store_row32<OutT>(y + c0, acc + c0 / 2, left < 32 ? (int)left : 32, align32);
                    }
                }
            } else {
                // rows that start anywhere: turned across the warp, so that its lanes store
                // consecutive columns of one row (element by element of its own row, a warp's
                // store would touch 32 rows)
                const int64_t row0 = row - lane;
                const int rows = (int)max((int64_t)0, min((int64_t)32, p.m - row0));
#pragma unroll
                for (int c0 = 0; c0 < CPT; c0 += 32) {
                    float v[32];
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        v[i] = acc[(c0 + i) / 2].x;
                        v[i + 1] = acc[(c0 + i) / 2].y;
                    }
                    warp_transpose(v);
                    const int64_t col = col0 + c0 + lane;
                    OutT* y = reinterpret_cast<OutT*>(p.y) + row0 * p.ldy + col;
                    if (col < p.n) {
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (i < rows) DT<OutT>::store1(y + (int64_t)i * p.ldy, v[i]);
                    }
                }
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    ring::cluster_sync();  // neither CTA leaves while the pair's MMAs or arrivals may touch it
    tc_fence_after();
    __syncwarp();
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::COLS)
                     : "memory");
}

}  // namespace fp8
}  // namespace k1
