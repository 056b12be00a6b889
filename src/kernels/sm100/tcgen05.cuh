// Fifth-generation tensor cores for a pair of CTAs: matrix instructions that one thread issues for both SMs (cta_group::2), their operands in
// shared memory, their accumulators in tensor memory, and the barriers between the CTAs of the pair.
#pragma once

#include "kernels/sm100/sync.cuh"
#include "kernels/sm100/tma.cuh"

#include <cuda.h>

#include <cstdint>

namespace b200ccl::dev {

__device__ __forceinline__ unsigned cluster_rank() {
    unsigned r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// Barrier of all threads of the cluster; what they stored before it is visible after it.
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
}

// ---- barriers -------------------------------------------------------------------------------------------
__device__ __forceinline__ void mbar_arrive(unsigned bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// The barrier at the same place in CTA `rank` of the cluster. What this thread's CTA stored to its shared memory, and this thread has seen, is visible to
// who waits there; nothing else is ordered, because a release of everything at cluster scope waits for this thread's accesses to global memory too.
__device__ __forceinline__ void mbar_arrive_at(unsigned bar, unsigned rank) {
    asm volatile(
        "{\n .reg .b32 remote;\n mapa.shared::cluster.u32 remote, %0, %1;\n fence.release.sync_restrict::shared::cta.cluster;\n"
        " mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [remote];\n}\n" ::"r"(bar),
        "r"(rank)
        : "memory");
}
// kCluster: threads of the other CTA arrive at the barrier too (mbar_arrive_at); otherwise this CTA's threads, its copies and products.
template <bool kCluster>
__device__ __forceinline__ bool phase_over(unsigned bar, unsigned parity) {
    unsigned done;
    if constexpr (kCluster) {
        asm volatile(
            "{\n .reg .pred p;\n mbarrier.try_wait.parity.relaxed.cluster.shared::cta.b64 p, [%1], %2, 1000;\n selp.u32 %0, 1, 0, p;\n"
            " fence.acquire.sync_restrict::shared::cluster.cluster;\n}\n"
            : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    } else {
        asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 1000;\n selp.u32 %0, 1, 0, p;\n}\n"
                     : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    }
    return done != 0u;
}
// A word at this place in CTA `rank` of the cluster.
__device__ __forceinline__ void store_word_at(unsigned where, unsigned rank, unsigned v) {
    asm volatile("{\n .reg .b32 remote;\n mapa.shared::cluster.u32 remote, %0, %1;\n st.shared::cluster.u32 [remote], %2;\n}\n" ::"r"(where), "r"(rank), "r"(v) : "memory");
}
// Waits for the phase of parity `parity`, for `limit` ns (and a few polls) at most; false then, and in every later wait of the CTA (`failed`, shared).
template <bool kCluster = false>
__device__ __forceinline__ bool wait_phase(unsigned bar, unsigned parity, volatile unsigned* failed, unsigned long long limit) {
    if (phase_over<kCluster>(bar, parity)) return true;
    unsigned long long t0 = 0;
    const unsigned between = limit != 0ull ? 15u : 0u;  // polls without a look at the clock
    for (unsigned polls = 1;; ++polls) {
        if (phase_over<kCluster>(bar, parity)) return true;
        if ((polls & between) != 0u) continue;
        const unsigned long long now = global_timer_ns();
        if (t0 == 0) t0 = now;
        if (*failed != 0u) return false;
        if (now - t0 >= limit) {
            *failed = 1u;
            return false;
        }
    }
}

// ---- copies ---------------------------------------------------------------------------------------------
// A box of a three-dimensional tensor map, from this GPU's own memory; x times the element's size is a multiple of 16 bytes.
__device__ __forceinline__ void tma_load_box(unsigned dst, const CUtensorMap* map, int x, int y, int z, unsigned bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst), "l"(map),
        "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}
// A box of shared memory to a three-dimensional tensor map of this GPU's own memory, in the thread's bulk async-group; no coordinate is negative.
__device__ __forceinline__ void tma_store_box(const CUtensorMap* map, unsigned src, int x, int y, int z) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(map), "r"(x), "r"(y), "r"(z), "r"(src) : "memory");
}
__device__ __forceinline__ void tma_prefetch_map(const CUtensorMap* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}
// Orders this thread's stores to shared memory before what the tensor cores read of it after the next barrier.
__device__ __forceinline__ void fence_shared_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// ---- tensor memory --------------------------------------------------------------------------------------
// One warp of each CTA of the pair. `where`: shared memory that receives the address.
__device__ __forceinline__ void tmem_alloc_pair(unsigned where, unsigned columns) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(where), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free_pair(unsigned address, unsigned columns) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(address), "r"(columns) : "memory");
}
// 32 columns of the warp's 32 lanes: thread i receives lane i. A warp reaches the lanes 32 * (warp % 4) and on.
__device__ __forceinline__ void tmem_load32(unsigned address, float (&f)[32]) {
    unsigned* r = reinterpret_cast<unsigned*>(f);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,"
        "%27,%28,%29,%30,%31}, [%32];\n"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
          "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(address)
        : "memory");
}
__device__ __forceinline__ void tcgen05_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tcgen05_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// ---- matrix instructions --------------------------------------------------------------------------------
// An operand whose rows run along the product's summed axis (row k holds neighbouring m or n): blocks of 64 elements (128 bytes, swizzled) by rows of the
// summed axis; eight rows are 1024 bytes, the next 64 elements `block_bytes` further.
__device__ __forceinline__ std::uint64_t operand_by_rows(unsigned address, unsigned block_bytes) {
    std::uint64_t d = (address >> 4) & 0x3fffu;
    d |= (std::uint64_t)((block_bytes >> 4) & 0x3fffu) << 16;  // from 64 elements to the next 64
    d |= (std::uint64_t)(1024u >> 4) << 32;                    // from eight rows to the next eight
    d |= 1ull << 46;                                           // version of sm_100
    d |= 2ull << 61;                                           // 128-byte swizzle
    return d;
}
// An operand whose rows lie along m or n and hold 64 neighbouring elements of the summed axis (128 bytes, swizzled): eight rows are 1024 bytes.
// The next 16 elements of the summed axis are 32 bytes further.
__device__ __forceinline__ std::uint64_t operand_by_columns(unsigned address) {
    std::uint64_t d = (address >> 4) & 0x3fffu;
    d |= 1ull << 16;                          // not looked at: a row of the tile is one swizzled row
    d |= (std::uint64_t)(1024u >> 4) << 32;   // from eight rows to the next eight
    d |= 1ull << 46;                          // version of sm_100
    d |= 2ull << 61;                          // 128-byte swizzle
    return d;
}
// 16-bit operands, each by rows or not, 32-bit accumulators.
__host__ __device__ constexpr unsigned product_shape(unsigned m, unsigned n, bool bf16, bool a_by_rows, bool b_by_rows) {
    return 1u << 4 | (bf16 ? 1u : 0u) << 7 | (bf16 ? 1u : 0u) << 10 | (a_by_rows ? 1u : 0u) << 15 | (b_by_rows ? 1u : 0u) << 16 | n / 8u << 17 | m / 16u << 24;
}
__host__ __device__ constexpr unsigned product_by_rows(unsigned m, unsigned n, bool bf16) { return product_shape(m, n, bf16, true, true); }
// 16 rows of both operands, in both CTAs of the pair; one thread of the first CTA.
__device__ __forceinline__ void mma_pair(unsigned accumulators, std::uint64_t a, std::uint64_t b, unsigned shape, bool add) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(accumulators), "l"(a), "l"(b),
        "r"(shape), "r"(add ? 1u : 0u)
        : "memory");
}
// Arrives at the barrier at this place in both CTAs once the products issued so far by this thread are done.
__device__ __forceinline__ void commit_pair(unsigned bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((unsigned short)3)
                 : "memory");
}

}  // namespace b200ccl::dev
