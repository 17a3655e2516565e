/**
 * Tensor memory, tensor-core products and tiled copies of sm_100a, as the instructions of the PTX manual: mbarriers with waits that
 * end, 2-D tensor-map loads into swizzled shared memory, tcgen05 allocation, products, commits and loads.
 */
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <cstdint>

namespace dccl {

__device__ __forceinline__ uint32_t shared_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

/* ---- mbarriers ---- */

__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t arrivals) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(arrivals) : "memory"); }
__device__ __forceinline__ void bar_init_fence() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
__device__ __forceinline__ void bar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    return done != 0;
}

constexpr long long kWaitClocks = 1ll << 34;     // about nine seconds: what a wait inside one CTA never takes

constexpr long long kLandClocks = 1ll << 24;     // about nine milliseconds: a thousand times what a copy takes

/** Waits for the phase of this parity. False after nine seconds, or once another wait of the CTA gave up (`failed`, in shared memory). */
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile int* failed) {
    if (bar_try(bar, parity)) return true;
    const long long start = clock64();
    while (!bar_try(bar, parity)) {
        if (*failed) return false;
        if (clock64() - start > kWaitClocks) { *failed = 1; return false; }
    }
    return true;
}

/** The same for a whole warp, which goes on as one. */
__device__ __forceinline__ bool bar_wait_warp(uint32_t bar, uint32_t parity, volatile int* failed) { return __all_sync(0xffffffffu, bar_wait(bar, parity, failed)); }

/* ---- tensor-map loads ---- */

/** One box into shared memory; the barrier counts its bytes, those outside of the tensor (zeros) among them. x * element size is a
 *  multiple of 16. */
__device__ __forceinline__ void load_box(uint32_t to, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(to), "l"(map), "r"(x), "r"(y), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }

/* ---- tensor memory ---- */

__device__ __forceinline__ void tmem_alloc(uint32_t to_shared, uint32_t columns) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(to_shared), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t columns) { asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(columns)); }
__device__ __forceinline__ void tc_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

/** 32 columns of this warp's 32 lanes: lane l gets row l. Complete after tmem_wait(). */
__device__ __forceinline__ void tmem_load32(uint32_t (&r)[32], uint32_t addr) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                 "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
                   "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                   "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(addr));
}
__device__ __forceinline__ void tmem_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

/* ---- products ---- */

/**
 * Matrix descriptor of a tile in shared memory with the 128-byte swizzle, 1024-byte aligned.
 * K-major (a row holds 64 consecutive k): groups of eight rows are 1024 bytes apart, `lead` is not used.
 * MN-major (a row holds 64 consecutive m or n of one k): groups of eight k are 1024 bytes apart, `lead` bytes lie between blocks of 64 m or n.
 */
__device__ __forceinline__ uint64_t tile_descriptor(uint32_t addr, uint32_t lead) {
    return (uint64_t)((addr & 0x3ffff) >> 4) | (uint64_t)((lead >> 4) & 0x3fff) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
/** Instruction descriptor of a 16-bit product with fp32 sums: types 0 f16, 1 bf16. */
__host__ __device__ constexpr uint32_t product_descriptor(int type, bool a_mn_major, bool b_mn_major, int m, int n) {
    return 1u << 4 | (uint32_t)type << 7 | (uint32_t)type << 10 | (uint32_t)a_mn_major << 15 | (uint32_t)b_mn_major << 16 | (uint32_t)(n >> 3) << 17 | (uint32_t)(m >> 4) << 24;
}
/** D (+)= A B^T over 16 k, by one thread. */
__device__ __forceinline__ void product(uint32_t d, uint64_t a, uint64_t b, uint32_t desc, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(desc), "r"((int)add)
                 : "memory");
}
/** One arrival on the barrier when this thread's products so far are done. */
__device__ __forceinline__ void commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

/* ---- pairs of CTAs: a cluster of two whose tensor cores work on one product of 256 rows, each CTA's memory holding its 128 rows of A and of the
 *      sums, and half of B. The CTA of rank 0 leads: it issues the products, which read both CTAs' shared memory at the same offsets. ---- */

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
/** This shared address in the CTA of that rank. */
__device__ __forceinline__ uint32_t in_cta(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void bar_arrive_remote(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
/** load_box into this CTA, its bytes counted by a barrier of either. */
__device__ __forceinline__ void pair_load_box(uint32_t to, const CUtensorMap* map, int x, int y, uint32_t cluster_bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];" ::"r"(to), "l"(map), "r"(x), "r"(y),
                 "r"(cluster_bar)
                 : "memory");
}
__device__ __forceinline__ void pair_tmem_alloc(uint32_t to_shared, uint32_t columns) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(to_shared), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void pair_tmem_free(uint32_t addr, uint32_t columns) { asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(columns)); }
__device__ __forceinline__ void pair_product(uint32_t d, uint64_t a, uint64_t b, uint32_t desc, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(desc), "r"((int)add)
                 : "memory");
}
/** One arrival on the barrier at this offset in both CTAs when the leader's products so far are done. */
__device__ __forceinline__ void pair_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3) : "memory");
}

} // namespace dccl
