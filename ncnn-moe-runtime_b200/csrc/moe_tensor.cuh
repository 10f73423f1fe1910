// Building blocks of kernels that feed the fifth-generation tensor cores: mbarriers with bounded waits, tile copies by the
// copy engine, products into tensor memory and reads from it.
#pragma once

#include <cuda.h>

#include "moe_common.cuh"

namespace moe {

constexpr uint32_t kSpinLimit = 1u << 18; // looks at a barrier before a wait gives up: one that fails is held for 4 us, so a second

// ---- mbarriers, tensor memory, descriptors ---------------------------------------------

__device__ __forceinline__ void barrier_init(uint32_t barrier, uint32_t arrivals)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(barrier), "r"(arrivals) : "memory");
}
// makes the initialised barriers known to the copy engine and the other CTAs
__device__ __forceinline__ void barrier_init_fence()
{
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}
__device__ __forceinline__ void barrier_arrive(uint32_t barrier)
{
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(barrier) : "memory");
}
__device__ __forceinline__ uint32_t cta_in_cluster()
{
    uint32_t rank;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    return rank;
}
__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void barrier_expect_bytes(uint32_t barrier, uint32_t bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(barrier), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool barrier_test(uint32_t barrier, uint32_t parity)
{
    uint32_t done;
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        "selp.u32 %0, 1, 0, p;\n"
        "}\n"
        : "=r"(done)
        : "r"(barrier), "r"(parity)
        : "memory");
    return done != 0;
}
// Bounded.  A wait that runs out marks the CTA as stalled; every role then leaves its loop.  The first look is apart from the
// loop: most waits find their phase complete, and a look costs 16 cycles where the loop takes 85.
__device__ __forceinline__ bool barrier_wait(uint32_t barrier, uint32_t parity, volatile uint32_t* stalled, uint32_t limit = kSpinLimit)
{
    if (barrier_test(barrier, parity))
        return true;
#pragma unroll 1
    for (uint32_t spin = 0; spin < limit; ++spin)
    {
        if (barrier_test(barrier, parity))
            return true;
        if ((spin & 255u) == 255u && *stalled != 0u)
            return false;
    }
    *stalled = 1u;
    return false;
}
// The same for a whole warp, which stays together.
__device__ __forceinline__ bool barrier_wait_warp(uint32_t barrier, uint32_t parity, volatile uint32_t* stalled, uint32_t limit = kSpinLimit)
{
    if (__all_sync(kFullMask, barrier_test(barrier, parity)))
        return true;
#pragma unroll 1
    for (uint32_t spin = 0; spin < limit; ++spin)
    {
        if (__all_sync(kFullMask, barrier_test(barrier, parity)))
            return true;
        if ((spin & 255u) == 255u && __any_sync(kFullMask, *stalled != 0u))
            return false;
    }
    *stalled = 1u;
    return false;
}

__device__ __forceinline__ void copy_tile(uint32_t destination, const CUtensorMap* map, uint32_t column, uint32_t row, uint32_t barrier)
{
    asm volatile("cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(destination), "l"(map), "r"(column), "r"(row),
                 "r"(barrier)
                 : "memory");
}

// four bytes, or zeros
__device__ __forceinline__ void copy_word(uint32_t destination, const float* source, bool valid)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(destination), "l"(__cvta_generic_to_global(source)), "r"(valid ? 4u : 0u) : "memory");
}

// A tile in shared memory as the copy engine leaves it: rows of 128 bytes, swizzled in groups of eight rows (1024 bytes
// from group to group).  A step of 32 columns moves the start by 32 bytes.
__device__ __forceinline__ uint64_t tile_descriptor(uint32_t address)
{
    return static_cast<uint64_t>((address & 0x3FFFFu) >> 4) | (1ull << 16) | (static_cast<uint64_t>(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// e4m3 by e4m3 into fp32, both operands with adjacent columns: `tall` lanes by `wide` columns
__device__ __forceinline__ constexpr uint32_t product_descriptor(uint32_t tall, uint32_t wide)
{
    return (1u << 4) | ((wide >> 3) << 17) | ((tall >> 4) << 24);
}
__device__ __forceinline__ void issue_product(uint32_t accumulator, uint64_t tall, uint64_t wide, uint32_t descriptor, bool accumulate)
{
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.u32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
        "}\n" ::"r"(accumulator),
        "l"(tall), "l"(wide), "r"(descriptor), "r"(accumulate ? 1u : 0u)
        : "memory");
}
// arrives at the barrier once the products issued so far are done
__device__ __forceinline__ void commit_products(uint32_t barrier)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(barrier) : "memory");
}

template<int kCount>
__device__ __forceinline__ void load_accumulator(uint32_t (&t)[kCount], uint32_t address);
template<>
__device__ __forceinline__ void load_accumulator<16>(uint32_t (&t)[16], uint32_t address)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(t[0]), "=r"(t[1]), "=r"(t[2]), "=r"(t[3]), "=r"(t[4]), "=r"(t[5]), "=r"(t[6]), "=r"(t[7]), "=r"(t[8]), "=r"(t[9]), "=r"(t[10]),
                   "=r"(t[11]), "=r"(t[12]), "=r"(t[13]), "=r"(t[14]), "=r"(t[15])
                 : "r"(address));
}
template<>
__device__ __forceinline__ void load_accumulator<32>(uint32_t (&t)[32], uint32_t address)
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(t[0]), "=r"(t[1]), "=r"(t[2]), "=r"(t[3]), "=r"(t[4]), "=r"(t[5]), "=r"(t[6]), "=r"(t[7]), "=r"(t[8]), "=r"(t[9]), "=r"(t[10]), "=r"(t[11]),
          "=r"(t[12]), "=r"(t[13]), "=r"(t[14]), "=r"(t[15]), "=r"(t[16]), "=r"(t[17]), "=r"(t[18]), "=r"(t[19]), "=r"(t[20]), "=r"(t[21]), "=r"(t[22]),
          "=r"(t[23]), "=r"(t[24]), "=r"(t[25]), "=r"(t[26]), "=r"(t[27]), "=r"(t[28]), "=r"(t[29]), "=r"(t[30]), "=r"(t[31])
        : "r"(address));
}
// The registers go through the wait, so that nothing that uses them moves in front of it.
template<int kCount>
__device__ __forceinline__ void wait_accumulator(uint32_t (&t)[kCount]);
template<>
__device__ __forceinline__ void wait_accumulator<16>(uint32_t (&t)[16])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(t[0]), "+r"(t[1]), "+r"(t[2]), "+r"(t[3]), "+r"(t[4]), "+r"(t[5]), "+r"(t[6]), "+r"(t[7]), "+r"(t[8]), "+r"(t[9]), "+r"(t[10]),
                   "+r"(t[11]), "+r"(t[12]), "+r"(t[13]), "+r"(t[14]), "+r"(t[15])::"memory");
}
template<>
__device__ __forceinline__ void wait_accumulator<32>(uint32_t (&t)[32])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(t[0]), "+r"(t[1]), "+r"(t[2]), "+r"(t[3]), "+r"(t[4]), "+r"(t[5]), "+r"(t[6]), "+r"(t[7]), "+r"(t[8]), "+r"(t[9]), "+r"(t[10]), "+r"(t[11]),
                   "+r"(t[12]), "+r"(t[13]), "+r"(t[14]), "+r"(t[15]), "+r"(t[16]), "+r"(t[17]), "+r"(t[18]), "+r"(t[19]), "+r"(t[20]), "+r"(t[21]), "+r"(t[22]),
                   "+r"(t[23]), "+r"(t[24]), "+r"(t[25]), "+r"(t[26]), "+r"(t[27]), "+r"(t[28]), "+r"(t[29]), "+r"(t[30]), "+r"(t[31])::"memory");
}
// One thread of a whole warp.  Not a comparison of the lane: behind that the compiler feeds every instruction of the tensor
// cores and the copy engine through code for several lanes (a block of 128 columns took about 1000 cycles to issue).
__device__ __forceinline__ bool elect_one()
{
    uint32_t elected;
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "elect.sync _|p, 0xFFFFFFFF;\n"
        "selp.u32 %0, 1, 0, p;\n"
        "}\n"
        : "=r"(elected));
    return elected != 0u;
}

// A position in a ring of `size` slots: its slot and the parity of the phase that it is in.
struct Cursor
{
    uint32_t slot = 0;
    uint32_t parity = 0;
    __device__ __forceinline__ void advance(uint32_t size)
    {
        if (++slot == size)
        {
            slot = 0;
            parity ^= 1u;
        }
    }
};

// Columns of tensor memory for the CTA; whole warps.
__device__ __forceinline__ void allocate_memory(uint32_t base_address, uint32_t columns)
{
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(base_address), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void free_memory(uint32_t base, uint32_t columns)
{
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(columns) : "memory");
}
__device__ __forceinline__ void memory_fence_before()
{
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void memory_fence_after()
{
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
// All threads of the CTA, with what they did to tensor memory.
__device__ __forceinline__ void memory_sync()
{
    __syncwarp();
    memory_fence_before();
    __syncthreads();
    memory_fence_after();
}

} // namespace moe
