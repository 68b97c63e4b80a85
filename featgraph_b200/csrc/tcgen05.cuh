// Thin wrappers of the sm_100a instructions the grouped product is built from: mbarriers with bounded waits, TMA tile
// loads, tcgen05 products with their accumulators in tensor memory.
#pragma once
#include <cuda.h>

#include "common.cuh"

namespace fg {

__device__ __forceinline__ uint32_t smem_address(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void barrier_init(uint32_t bar, uint32_t arrivals) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(arrivals));
}
__device__ __forceinline__ void barrier_init_fence() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
__device__ __forceinline__ void barrier_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void barrier_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
template <bool CLUSTER>
__device__ __forceinline__ bool barrier_try(uint32_t bar, uint32_t parity) {
    uint32_t done;
    if (CLUSTER)  // arrivals may come from the other block of a pair
        asm volatile(
            "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n selp.b32 %0, 1, 0, p;\n}"
            : "=r"(done)
            : "r"(bar), "r"(parity)
            : "memory");
    else
        asm volatile(
            "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.b32 %0, 1, 0, p;\n}"
            : "=r"(done)
            : "r"(bar), "r"(parity)
            : "memory");
    return done != 0;
}

// Every wait ends: after about four seconds (at 2 GHz) it raises the block's `stop` word and gives up, and so does every
// other wait of the block that sees the word.  `ignore_stop`: the last waits for copies in flight.
constexpr long long kWaitClocks = 8ll << 30;
template <bool CLUSTER = false>
__device__ __forceinline__ bool barrier_wait(uint32_t bar, uint32_t parity, volatile int* stop, bool ignore_stop = false) {
    if (barrier_try<CLUSTER>(bar, parity)) return true;
    const long long start = clock64();
    while (!barrier_try<CLUSTER>(bar, parity)) {
        if ((*stop && !ignore_stop) || clock64() - start > kWaitClocks) {
            *stop = 1;
            return false;
        }
    }
    return true;
}

// ---- pairs of blocks (clusters of two) ----
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Arrives at block `rank`'s barrier of the same address.  With RELEASE, what this thread wrote before is seen by who waits
// there, which takes over a thousand cycles; without, the arrival alone is (tensor memory has been read).
template <bool RELEASE>
__device__ __forceinline__ void barrier_arrive_at(uint32_t bar, uint32_t rank) {
    if (RELEASE)
        asm volatile(
            "{\n .reg .b32 r;\n mapa.shared::cluster.u32 r, %0, %1;\n mbarrier.arrive.release.cluster.shared::cluster.b64 _, [r];\n}" ::"r"(bar),
            "r"(rank)
            : "memory");
    else
        asm volatile("{\n .reg .b32 r;\n mapa.shared::cluster.u32 r, %0, %1;\n mbarrier.arrive.shared::cluster.b64 _, [r];\n}" ::"r"(bar), "r"(rank)
                     : "memory");
}

// Tile loads into this block's shared memory.  In a pair both blocks' loads count on the first one's barrier (the second
// block's bit of a cluster address cleared).
template <int BLOCKS>
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    if (BLOCKS == 2)
        asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
                     "l"(map), "r"(x), "r"(y), "r"(bar & 0xfeffffffu)
                     : "memory");
    else
        asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
                     "l"(map), "r"(x), "r"(y), "r"(bar)
                     : "memory");
}
template <int BLOCKS>
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    if (BLOCKS == 2)
        asm volatile(
            "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
            "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar & 0xfeffffffu)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
            "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
            : "memory");
}
// Consecutive bytes (addresses and size on the 16-byte grid).
__device__ __forceinline__ void bulk_load(uint32_t dst, uint64_t src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }

// True in one lane of the (converged) warp, the same every time.  Copies and products are issued under it: their operands
// sit in uniform registers, and only under elect.sync does the compiler know that one thread is left.  Under
// `lane == 0` it wraps each of them in a loop over the active lanes.
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.b32 %0, 1, 0, p;\n}" : "=r"(one));
    return one != 0;
}

// ---- tensor memory ----
// (a pair allocates, multiplies and frees together: cta_group::2)
template <int BLOCKS>
__device__ __forceinline__ void tmem_alloc(uint32_t slot, uint32_t columns) {
    if (BLOCKS == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    } else {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
}
template <int BLOCKS>
__device__ __forceinline__ void tmem_free(uint32_t address, uint32_t columns) {
    if (BLOCKS == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(address), "r"(columns));
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(address), "r"(columns));
}
__device__ __forceinline__ void tcgen05_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tcgen05_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 32 lanes (this warp's quarter) x 16 or 32 columns: thread = lane, register = column.
template <int N>
__device__ __forceinline__ void tmem_load(uint32_t address, uint32_t (&r)[N]);
template <>
__device__ __forceinline__ void tmem_load<16>(uint32_t address, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(address));
}
template <>
__device__ __forceinline__ void tmem_load<32>(uint32_t address, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(address));
}
__device__ __forceinline__ void tmem_load_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// ---- products ----
// Shared-memory operand descriptor, 128-byte swizzle: address and strides in 16-byte units.  Rows of 128 bytes along the
// inner axis of the product ("K-major"): `stride` is the distance of two groups of 8 rows.  Rows of 128 bytes along the
// operand's own axis ("MN-major", one row for each step of the inner axis): `stride` is the distance of two groups of 8
// inner steps, `lead` that of two 128-byte columns.
__device__ __forceinline__ uint64_t operand_descriptor(uint32_t address, uint32_t lead, uint32_t stride) {
    return (uint64_t)((address & 0x3ffffu) >> 4) | ((uint64_t)(lead >> 4) << 16) | ((uint64_t)(stride >> 4) << 32) | (1ull << 46) |
           (2ull << 61);
}
// Instruction descriptor: 32-bit sums; format 0 = fp16 or e4m3, 1 = bf16; *_mn: that operand is MN-major.
__host__ __device__ constexpr uint32_t product_descriptor(uint32_t format, bool a_mn, bool b_mn, uint32_t m, uint32_t n) {
    return (1u << 4) | (format << 7) | (format << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) | ((n >> 3) << 17) | ((m >> 4) << 24);
}
#define FG_PRODUCT(group, kind)                                                                                                       \
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::" group ".kind::" kind " [%0], %1, %2, %3, p;\n}" ::"r"( \
                     acc),                                                                                                           \
                 "l"(a), "l"(b), "r"(descriptor), "r"((uint32_t)add)                                                                 \
                 : "memory")
template <int BLOCKS, bool EIGHT>
__device__ __forceinline__ void product_step(uint32_t acc, uint64_t a, uint64_t b, uint32_t descriptor, bool add) {
    if (BLOCKS == 2) {
        if (EIGHT) FG_PRODUCT("2", "f8f6f4");
        else FG_PRODUCT("2", "f16");
    } else {
        if (EIGHT) FG_PRODUCT("1", "f8f6f4");
        else FG_PRODUCT("1", "f16");
    }
}
#undef FG_PRODUCT
// Arrives at `bar` (of both blocks of a pair) when all products issued so far by this thread are done.
template <int BLOCKS>
__device__ __forceinline__ void product_commit(uint32_t bar) {
    if (BLOCKS == 2)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3)
                     : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

}  // namespace fg
