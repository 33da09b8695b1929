// k1_sync.cuh -- mbarriers with bounded waits, bulk copies and thread-block clusters,
// shared by the kernels that stage data in shared memory.
//
// Every wait is bounded (kMaxTries polls with a suspend hint, a few seconds in all).  One
// that runs out sets a bit of k1_ring_error, which k1_ring_status reports.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

// Polls of a bounded mbarrier wait before it gives up (each poll suspends for at most
// kSuspendHintNs).  The wait-timeout test library is built with a small value.
#ifndef K1_RING_MAX_TRIES
#define K1_RING_MAX_TRIES 4096
#endif

namespace k1 {

// One word per translation unit; k1_ring_status reads (and clears) all of them.
static __device__ unsigned k1_ring_error;

#ifdef K1_WAIT_TEST
// Test-only knob (compiled into the wait-timeout test library only): block 0's producer
// issues no copy from its chunk number k1_test_withhold on, so the consumers' waits for
// that chunk run out.  -1: off.
static __device__ long long k1_test_withhold = -1;
#endif

namespace ring {

constexpr int kMaxTries = K1_RING_MAX_TRIES;  // x up to 1 ms suspend hint per poll
constexpr uint32_t kSuspendHintNs = 1000000;

__device__ __forceinline__ uint32_t saddr(const void* p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void bar_init(uint64_t* b, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(saddr(b)), "r"(count) : "memory");
}
__device__ __forceinline__ void fence_init() {
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}
__device__ __forceinline__ void arrive_expect(uint64_t* b, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(saddr(b)),
                 "r"(bytes)
                 : "memory");
}
__device__ __forceinline__ void arrive(uint64_t* b) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(saddr(b)) : "memory");
}
__device__ __forceinline__ bool try_wait(uint64_t* b, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(saddr(b)), "r"(parity), "r"(kSuspendHintNs)
        : "memory");
    return ok != 0;
}
// Bounded wait for the phase of parity `parity`; false (and the error word set) if it
// did not complete in time.
__device__ __forceinline__ bool wait(uint64_t* b, uint32_t parity) {
    for (int i = 0; i < kMaxTries; ++i)
        if (try_wait(b, parity)) return true;
    atomicOr(&k1_ring_error, 1u);
    return false;
}
// The same on the barrier's shared-memory address, for loops that keep addresses rather than
// pointers (a pointer into shared memory is converted at every use).
__device__ __forceinline__ void arrive_at(uint32_t b) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(b) : "memory");
}
__device__ __forceinline__ bool try_wait_at(uint32_t b, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(b), "r"(parity), "r"(kSuspendHintNs)
        : "memory");
    return ok != 0;
}
// Whether the phase has completed, without waiting for it.
__device__ __forceinline__ bool test_at(uint32_t b, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(b), "r"(parity)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ void bulk_g2s(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::
            "r"(saddr(dst)),
        "l"(src), "r"(bytes), "r"(saddr(bar))
        : "memory");
}

// One lane of a converged warp (the same one at every call).  The compiler knows a branch on
// it to be taken by one thread, so what it guards can use uniform registers; after a branch
// on the lane's number, tcgen05 and TMA instructions cost several times the issue cycles.
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile(
        "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(one)
        :
        : "memory");
    return one != 0;
}

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// The shared::cluster address of `saddr` (a shared::cta address) in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t mapa(uint32_t saddr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
    return r;
}
// Every thread of both CTAs (per-thread form: the warps need not be converged).
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// Its two halves, for work that lies between them.
__device__ __forceinline__ void cluster_arrive() {
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}
// Arrive on an mbarrier of another CTA of the cluster (address from mapa).  The default
// (CTA-scope) semantics: a release at cluster scope here would make the arriving thread
// wait for its own bulk copies in flight, which serialises the producer.
__device__ __forceinline__ void arrive_remote(uint32_t cl_addr) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cl_addr) : "memory");
}

}  // namespace ring
}  // namespace k1
