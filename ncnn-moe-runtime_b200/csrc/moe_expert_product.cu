// The experts' matrix products in e4m3 with a scale for each block of 128:
//   out[r, n] = sum_b scales[b, r] * weight_scales[e, n / 128, b] * sum_{k in b} values[r, k] * weights[e, n, k]
//
// The weights are the tall operand: a tile is 128 outputs (the 128 lanes of the accumulator in tensor memory) by kTokens
// rows (its columns), so that a few rows of a decode step do not fill a tile of 128 rows with padding, and a tile's outputs
// lie in one block of the weights' scales.  Per block of 128 columns the tensor cores compute the inner sum into a fresh
// accumulator, four instructions of 32 columns each, and the epilogue warps add it to their registers times the product of
// the two scales: one fused multiply-add per element of the tile and block, with a factor that all 128 lanes share per
// column.
//
// Roles of a CTA, which stays for all its tiles: a thread that requests tiles of both operands from the copy engine, a
// thread that issues the products, a warp that multiplies the scales, four or eight warps that scale, sum and store.  They
// pass a ring of operand stages, two to four accumulators and a ring of scales to each other through mbarriers, so that the
// copies, the products and the sums of different blocks, and of different tiles, overlap.

#include <cuda.h>

#include "moe_common.cuh"
#include "moe_internal.h"

namespace moe {

namespace {

constexpr uint32_t kOutputs = 128;      // outputs of a tile
constexpr uint32_t kBlockBytes = MOE_EXPERT_BLOCK;
constexpr uint32_t kWeightTile = kOutputs * kBlockBytes;
constexpr uint32_t kScaleSlots = 8;     // blocks of scales in flight
constexpr uint32_t kGroupTiles = 16;    // row tiles that share a weight tile before the next one is taken
constexpr uint32_t kSpinLimit = 1u << 20;
constexpr uint32_t kRoleThreads = 128;  // one warp for the copies, one for the products, one for the scales, one for tensor memory

template<int kTokens>
struct Shape
{
    static constexpr uint32_t kStageBytes = kWeightTile + kTokens * kBlockBytes;
    static constexpr uint32_t kStages = kTokens <= 16 ? 10u : kTokens <= 32 ? 9u : kTokens <= 64 ? 8u : kTokens <= 128 ? 6u : 4u;
    static constexpr uint32_t kAccumulators = kTokens <= 128 ? 4u : 2u;
    static constexpr uint32_t kMemoryColumns = kTokens * kAccumulators < 32 ? 32u : kTokens * kAccumulators;
    static constexpr uint32_t kSumWarps = kTokens <= 64 ? 4u : 8u;
    static constexpr uint32_t kThreads = kRoleThreads + 32u * kSumWarps;
    static constexpr uint32_t kColumns = kTokens / (kSumWarps / 4u);      // columns of the tile that a warp sums
    static constexpr uint32_t kChunk = kColumns < 32u ? kColumns : 32u;   // columns read from tensor memory at once
    static constexpr uint32_t kScaleBytes = kScaleSlots * kTokens * 4u;
    static constexpr uint32_t kBarriers = 2u * kStages + 2u * kAccumulators + 2u * kScaleSlots;
    static constexpr uint32_t kFixedBytes = kStages * kStageBytes + kScaleBytes + kBarriers * 8u + 64u;
};

// ---- mbarriers, tensor memory, descriptors ---------------------------------------------

__device__ __forceinline__ void barrier_init(uint32_t barrier, uint32_t arrivals)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(barrier), "r"(arrivals) : "memory");
}
__device__ __forceinline__ void barrier_arrive(uint32_t barrier)
{
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(barrier) : "memory");
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
// Bounded.  A wait that runs out marks the CTA as stalled; every role then leaves its loop.
__device__ __forceinline__ bool barrier_wait(uint32_t barrier, uint32_t parity, volatile uint32_t* stalled)
{
    for (uint32_t spin = 0; spin < kSpinLimit; ++spin)
    {
        if (barrier_test(barrier, parity))
            return true;
        if ((spin & 255u) == 255u && *stalled != 0u)
            return false;
    }
    *stalled = 1u;
    return false;
}

__device__ __forceinline__ void copy_tile(uint32_t destination, const CUtensorMap* map, uint32_t column, uint32_t row, uint32_t barrier)
{
    asm volatile("cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(destination), "l"(map),
                 "r"(column), "r"(row), "r"(barrier)
                 : "memory");
}
// A tile in shared memory as the copy engine leaves it: rows of 128 bytes, swizzled in groups of eight rows (1024 bytes
// from group to group).  A step of 32 columns moves the start by 32 bytes.
__device__ __forceinline__ uint64_t tile_descriptor(uint32_t address)
{
    return static_cast<uint64_t>((address & 0x3FFFFu) >> 4) | (1ull << 16) | (static_cast<uint64_t>(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// e4m3 by e4m3 into fp32, both operands with adjacent columns, 128 x kTokens
template<int kTokens>
__device__ __forceinline__ constexpr uint32_t product_descriptor()
{
    return (1u << 4) | (static_cast<uint32_t>(kTokens >> 3) << 17) | ((kOutputs >> 4) << 24);
}
__device__ __forceinline__ void issue_product(uint32_t accumulator, uint64_t weights, uint64_t rows, uint32_t descriptor, bool accumulate)
{
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.u32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
        "}\n" ::"r"(accumulator),
        "l"(weights), "l"(rows), "r"(descriptor), "r"(accumulate ? 1u : 0u)
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
// two sums at once: sum += part * factor
__device__ __forceinline__ void add_scaled_pair(uint64_t& sum, uint32_t part_low, uint32_t part_high, uint64_t factors)
{
    asm("{\n"
        ".reg .b64 part;\n"
        "mov.b64 part, {%1, %2};\n"
        "fma.rn.f32x2 %0, part, %3, %0;\n"
        "}\n"
        : "+l"(sum)
        : "r"(part_low), "r"(part_high), "l"(factors));
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

// ---- tiles ------------------------------------------------------------------------------

struct Tile
{
    uint32_t expert;
    uint32_t first_row;
    uint32_t rows;
    uint32_t output_block;
};

// The tile-th tile of the call.  first_tile: [experts + 1] tiles before each expert's.  Within an expert, groups of row tiles
// share a weight tile before the next weight tile is taken: a wave of CTAs then reads a few of both from L2.
template<int kTokens>
__device__ __forceinline__ Tile find_tile(const ProductArgs& a, const uint32_t* first_tile, uint32_t tile, uint32_t output_blocks)
{
    Tile found;
    uint32_t low = 0, high = a.expert_count;
    while (high - low > 1u)
    {
        const uint32_t middle = (low + high) / 2u;
        if (first_tile[middle] <= tile)
            low = middle;
        else
            high = middle;
    }
    found.expert = low;
    const uint32_t begin = a.expert_offsets != nullptr ? a.expert_offsets[low] : 0u;
    const uint32_t end = a.expert_offsets != nullptr ? a.expert_offsets[low + 1u] : a.rows;
    const uint32_t row_tiles = (end - begin + kTokens - 1u) / kTokens;
    const uint32_t local = tile - first_tile[low];
    const uint32_t group = local / (kGroupTiles * output_blocks);
    const uint32_t in_group = local - group * kGroupTiles * output_blocks;
    const uint32_t width = min(kGroupTiles, row_tiles - group * kGroupTiles);
    found.output_block = in_group / width;
    const uint32_t row_tile = group * kGroupTiles + in_group - found.output_block * width;
    found.first_row = begin + row_tile * kTokens;
    found.rows = min(static_cast<uint32_t>(kTokens), end - found.first_row);
    return found;
}

// Tiles before every expert's, by all threads; returns false when the offsets descend or exceed the rows.
template<int kTokens>
__device__ __forceinline__ bool count_tiles(const ProductArgs& a, uint32_t* first_tile, uint32_t output_blocks)
{
    __shared__ uint32_t warp_totals[32];
    const uint32_t threads = Shape<kTokens>::kThreads;
    const uint32_t per = (a.expert_count + threads - 1u) / threads;
    const uint32_t begin = min(a.expert_count, threadIdx.x * per), end = min(a.expert_count, begin + per);
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    bool good = true;
    uint32_t mine = 0;
    for (uint32_t e = begin; e < end; ++e)
    {
        const uint32_t first = a.expert_offsets != nullptr ? a.expert_offsets[e] : 0u;
        const uint32_t last = a.expert_offsets != nullptr ? a.expert_offsets[e + 1u] : a.rows;
        good = good && first <= last && last <= a.rows;
        mine += (last - first + kTokens - 1u) / kTokens * output_blocks;
    }
    uint32_t before = mine;
#pragma unroll
    for (int offset = 1; offset < 32; offset <<= 1)
    {
        const uint32_t other = __shfl_up_sync(kFullMask, before, offset);
        before += lane >= static_cast<uint32_t>(offset) ? other : 0u;
    }
    if (lane == 31u)
        warp_totals[warp] = before;
    before -= mine;
    good = __syncthreads_and(good) != 0;
    if (!good)
        return false;
    for (uint32_t w = 0; w < warp; ++w)
        before += warp_totals[w];
    for (uint32_t e = begin; e < end; ++e)
    {
        const uint32_t first = a.expert_offsets != nullptr ? a.expert_offsets[e] : 0u;
        const uint32_t last = a.expert_offsets != nullptr ? a.expert_offsets[e + 1u] : a.rows;
        first_tile[e] = before;
        before += (last - first + kTokens - 1u) / kTokens * output_blocks;
    }
    if (end == a.expert_count && begin < end)
        first_tile[a.expert_count] = before;
    return true;
}

// ---- the kernel -------------------------------------------------------------------------

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

template<int kTokens, typename Out>
__global__ void __launch_bounds__(Shape<kTokens>::kThreads, 1)
    expert_product_kernel(const ProductArgs a, const __grid_constant__ CUtensorMap weight_map, const __grid_constant__ CUtensorMap row_map)
{
    using S = Shape<kTokens>;
    extern __shared__ unsigned char shared_raw[];
    __shared__ uint32_t memory_base_shared;
    __shared__ volatile uint32_t stalled;
    unsigned char* const shared = shared_raw + ((1024u - (shared_address(shared_raw) & 1023u)) & 1023u);
    const uint32_t stages = shared_address(shared);
    const uint32_t scale_slots = stages + S::kStages * S::kStageBytes;
    const uint32_t full = scale_slots + S::kScaleBytes;
    const uint32_t empty = full + 8u * S::kStages;
    const uint32_t sum_full = empty + 8u * S::kStages;
    const uint32_t sum_empty = sum_full + 8u * S::kAccumulators;
    const uint32_t scale_full = sum_empty + 8u * S::kAccumulators;
    const uint32_t scale_empty = scale_full + 8u * kScaleSlots;
    uint32_t* const first_tile = reinterpret_cast<uint32_t*>(shared + S::kStages * S::kStageBytes + S::kScaleBytes + 8u * S::kBarriers);
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;

    if (threadIdx.x == 0)
    {
        for (uint32_t i = 0; i < S::kStages; ++i)
        {
            barrier_init(full + 8u * i, 1u);
            barrier_init(empty + 8u * i, 1u);
        }
        for (uint32_t i = 0; i < S::kAccumulators; ++i)
        {
            barrier_init(sum_full + 8u * i, 1u);
            barrier_init(sum_empty + 8u * i, S::kSumWarps);
        }
        for (uint32_t i = 0; i < kScaleSlots; ++i)
        {
            barrier_init(scale_full + 8u * i, 1u);
            barrier_init(scale_empty + 8u * i, S::kSumWarps);
        }
        stalled = 0u;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 3u)
    {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(shared_address(&memory_base_shared)), "r"(S::kMemoryColumns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t memory_base = memory_base_shared;

    wait_for_previous_kernel();
    const uint32_t blocks = (a.columns + MOE_EXPERT_BLOCK - 1u) / MOE_EXPERT_BLOCK;
    const uint32_t output_blocks = (a.outputs + kOutputs - 1u) / kOutputs;
    const bool good = count_tiles<kTokens>(a, first_tile, output_blocks);
    __syncthreads();
    const uint32_t tiles = good ? first_tile[a.expert_count] : 0u;
    if (!good && threadIdx.x == 0)
        atomicOr(a.flags, MOE_EXPERT_FLAG_OFFSETS);

    if (warp == 0u)
    {
        if (elect_one())
        {
            Cursor cursor;
            uint32_t issued = 0;
            for (uint32_t t = blockIdx.x; t < tiles && stalled == 0u; t += gridDim.x)
            {
                const Tile tile = find_tile<kTokens>(a, first_tile, t, output_blocks);
                const uint32_t weight_row = tile.expert * a.outputs + tile.output_block * kOutputs;
                for (uint32_t block = 0; block < blocks; ++block)
                {
                    if (!barrier_wait(empty + 8u * cursor.slot, cursor.parity ^ 1u, &stalled))
                        break;
                    const uint32_t stage = stages + cursor.slot * S::kStageBytes;
                    const uint32_t barrier = full + 8u * cursor.slot;
                    barrier_expect_bytes(barrier, S::kStageBytes);
                    copy_tile(stage, &weight_map, block * kBlockBytes, weight_row, barrier);
                    copy_tile(stage + kWeightTile, &row_map, block * kBlockBytes, tile.first_row, barrier);
                    cursor.advance(S::kStages);
                    ++issued;
                }
            }
            // no copy may land after the CTA has left: the last ones are waited for, in the order of their requests
            for (uint32_t back = min(issued, S::kStages); back > 0u; --back)
            {
                const uint32_t slot = (cursor.slot + S::kStages - back) % S::kStages;
                const uint32_t parity = slot < cursor.slot ? cursor.parity : cursor.parity ^ 1u;
                for (uint32_t spin = 0; spin < kSpinLimit && !barrier_test(full + 8u * slot, parity); ++spin)
                    ;
            }
        }
    }
    else if (warp == 1u)
    {
        if (elect_one())
        {
            Cursor cursor, sum;
            bool running = true;
            bool any = false;
            for (uint32_t t = blockIdx.x; t < tiles && running; t += gridDim.x)
            {
                for (uint32_t block = 0; block < blocks; ++block)
                {
                    running = barrier_wait(sum_empty + 8u * sum.slot, sum.parity ^ 1u, &stalled) && barrier_wait(full + 8u * cursor.slot, cursor.parity, &stalled);
                    if (!running)
                        break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t stage = stages + cursor.slot * S::kStageBytes;
                    const uint64_t weights = tile_descriptor(stage), rows = tile_descriptor(stage + kWeightTile);
                    // what lies behind the last column is zero: whole steps of it are left out
                    const uint32_t steps = min(4u, (a.columns - block * MOE_EXPERT_BLOCK + 31u) / 32u);
                    for (uint32_t step = 0; step < steps; ++step)
                        issue_product(memory_base + sum.slot * kTokens, weights + 2u * step, rows + 2u * step, product_descriptor<kTokens>(), step != 0u);
                    commit_products(empty + 8u * cursor.slot);
                    commit_products(sum_full + 8u * sum.slot);
                    any = true;
                    cursor.advance(S::kStages);
                    sum.advance(S::kAccumulators);
                }
            }
            // tensor memory is given back below: the last product must be done, also when somebody stalled
            if (any)
            {
                const uint32_t slot = sum.slot == 0u ? S::kAccumulators - 1u : sum.slot - 1u;
                const uint32_t parity = sum.slot == 0u ? sum.parity ^ 1u : sum.parity;
                for (uint32_t spin = 0; spin < kSpinLimit && !barrier_test(sum_full + 8u * slot, parity); ++spin)
                    ;
            }
        }
    }
    else if (warp == 2u)
    {
        // The products of the scales, four blocks ahead of the ring in registers.
        constexpr uint32_t kPerLane = (kTokens + 31u) / 32u;
        constexpr uint32_t kAhead = 4;
        Cursor cursor;
        bool running = true;
        for (uint32_t t = blockIdx.x; t < tiles && running; t += gridDim.x)
        {
            const Tile tile = find_tile<kTokens>(a, first_tile, t, output_blocks);
            const float* weight_scales = a.weight_scales + (static_cast<size_t>(tile.expert) * output_blocks + tile.output_block) * blocks;
            const float* scales = a.scales + tile.first_row;
            float next[kAhead][kPerLane], next_weight[kAhead];
            const auto load = [&](uint32_t first) {
#pragma unroll
                for (uint32_t i = 0; i < kAhead; ++i)
                {
                    const uint32_t block = first + i;
                    next_weight[i] = block < blocks ? weight_scales[block] : 0.0f;
#pragma unroll
                    for (uint32_t j = 0; j < kPerLane; ++j)
                    {
                        const uint32_t row = lane + 32u * j;
                        next[i][j] = block < blocks && row < tile.rows ? scales[static_cast<size_t>(block) * a.rows + row] : 0.0f;
                    }
                }
            };
            load(0u);
            for (uint32_t first = 0; first < blocks && running; first += kAhead)
            {
                float now[kAhead][kPerLane];
#pragma unroll
                for (uint32_t i = 0; i < kAhead; ++i)
#pragma unroll
                    for (uint32_t j = 0; j < kPerLane; ++j)
                        now[i][j] = next[i][j] * next_weight[i];
                if (first + kAhead < blocks)
                    load(first + kAhead);
#pragma unroll
                for (uint32_t i = 0; i < kAhead; ++i)
                {
                    if (first + i >= blocks || !running)
                        break;
                    running = __all_sync(kFullMask, barrier_wait(scale_empty + 8u * cursor.slot, cursor.parity ^ 1u, &stalled)) != 0;
                    if (!running)
                        break;
                    const uint32_t slot = scale_slots + cursor.slot * kTokens * 4u;
#pragma unroll
                    for (uint32_t j = 0; j < kPerLane; ++j)
                        if (kTokens >= 32 || lane < kTokens)
                            asm volatile("st.shared.f32 [%0], %1;" ::"r"(slot + 4u * (lane + 32u * j)), "f"(now[i][j]) : "memory");
                    __syncwarp();
                    if (lane == 0u)
                        barrier_arrive(scale_full + 8u * cursor.slot);
                    cursor.advance(kScaleSlots);
                }
            }
        }
    }
    else if (warp >= 4u)
    {
        const uint32_t quarter = warp & 3u;                                // lanes of tensor memory that this warp can read
        const uint32_t first_column = (warp - 4u) / 4u * S::kColumns;      // columns of the tile that it sums
        const uint32_t memory = memory_base + (quarter << 21) + first_column;
        Cursor sum, scale;
        bool running = true;
        for (uint32_t t = blockIdx.x; t < tiles && running; t += gridDim.x)
        {
            uint64_t sums[S::kColumns / 2];
#pragma unroll
            for (uint32_t i = 0; i < S::kColumns / 2; ++i)
                sums[i] = 0ull;
            for (uint32_t block = 0; block < blocks; ++block)
            {
                running = __all_sync(kFullMask, barrier_wait(scale_full + 8u * scale.slot, scale.parity, &stalled) &&
                                                    barrier_wait(sum_full + 8u * sum.slot, sum.parity, &stalled)) != 0;
                if (!running)
                    break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t factors = scale_slots + (scale.slot * kTokens + first_column) * 4u;
                const uint32_t source = memory + sum.slot * kTokens;
                // the next chunk is on its way while this one is summed
                constexpr uint32_t kChunks = S::kColumns / S::kChunk;
                uint32_t part[2][S::kChunk];
                load_accumulator<S::kChunk>(part[0], source);
#pragma unroll
                for (uint32_t chunk = 0; chunk < kChunks; ++chunk)
                {
                    wait_accumulator<S::kChunk>(part[chunk & 1u]);
                    if (chunk + 1u < kChunks)
                        load_accumulator<S::kChunk>(part[(chunk + 1u) & 1u], source + (chunk + 1u) * S::kChunk);
#pragma unroll
                    for (uint32_t i = 0; i < S::kChunk; i += 4u)
                    {
                        const ulonglong2 factor = load_shared_2x64(factors + (chunk * S::kChunk + i) * 4u);
                        const uint32_t(&p)[S::kChunk] = part[chunk & 1u];
                        add_scaled_pair(sums[(chunk * S::kChunk + i) / 2u], p[i], p[i + 1u], factor.x);
                        add_scaled_pair(sums[(chunk * S::kChunk + i) / 2u + 1u], p[i + 2u], p[i + 3u], factor.y);
                    }
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0u)
                {
                    barrier_arrive(sum_empty + 8u * sum.slot);
                    barrier_arrive(scale_empty + 8u * scale.slot);
                }
                sum.advance(S::kAccumulators);
                scale.advance(kScaleSlots);
            }
            if (!running)
                break;
            const Tile tile = find_tile<kTokens>(a, first_tile, t, output_blocks);
            const uint32_t output = tile.output_block * kOutputs + quarter * 32u + lane;
            if (output < a.outputs)
            {
                Out* target = static_cast<Out*>(a.out) + static_cast<size_t>(tile.first_row + first_column) * a.out_stride + output;
#pragma unroll
                for (uint32_t i = 0; i < S::kColumns; ++i)
                {
                    if (first_column + i < tile.rows)
                    {
                        const float value = __uint_as_float(static_cast<uint32_t>(sums[i / 2u] >> (32u * (i & 1u))));
                        if constexpr (sizeof(Out) == 4)
                            target[static_cast<size_t>(i) * a.out_stride] = value;
                        else
                            target[static_cast<size_t>(i) * a.out_stride] = __float2bfloat16_rn(value);
                    }
                }
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (warp == 3u)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(memory_base), "r"(S::kMemoryColumns) : "memory");
    if (threadIdx.x == 0 && stalled != 0u)
        atomicOr(a.flags, MOE_EXPERT_FLAG_STALLED);
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                 CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_function()
{
    static const EncodeTiled function = [] {
        void* entry = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &entry, 12000, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess)
            entry = nullptr;
        return reinterpret_cast<EncodeTiled>(entry);
    }();
    return function;
}

// Rows of `columns` bytes, read in boxes of `box_rows` rows by 128 columns; zeros behind the last column and row.
bool encode_rows(CUtensorMap* map, const uint8_t* base, uint32_t columns, uint64_t rows, uint32_t box_rows)
{
    const cuuint64_t extent[2] = {columns, rows};
    const cuuint64_t stride[1] = {columns};
    const cuuint32_t box[2] = {kBlockBytes, box_rows};
    const cuuint32_t step[2] = {1, 1};
    const EncodeTiled encode = encode_function();
    return encode != nullptr && encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(base), extent, stride, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                       CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template<int kTokens, typename Out>
cudaError_t launch_tiles(const ProductArgs& a, int sm_count, cudaStream_t stream)
{
    using S = Shape<kTokens>;
    CUtensorMap weight_map, row_map;
    if (!encode_rows(&weight_map, a.weights, a.columns, static_cast<uint64_t>(a.expert_count) * a.outputs, kOutputs) ||
        !encode_rows(&row_map, a.values, a.columns, a.rows, kTokens))
        return cudaErrorInvalidValue;
    const uint64_t row_tiles = (static_cast<uint64_t>(a.rows) + kTokens - 1u) / kTokens + (a.expert_count < a.rows ? a.expert_count : a.rows) - 1u;
    const uint64_t tiles = row_tiles * ((a.outputs + kOutputs - 1u) / kOutputs);
    const size_t shared_bytes = 1024u + S::kFixedBytes + sizeof(uint32_t) * (static_cast<size_t>(a.expert_count) + 1u);
    static SharedOptIn opt_in;
    if (cudaError_t status = opt_in_shared(opt_in, expert_product_kernel<kTokens, Out>, shared_bytes))
        return status;
    const uint32_t grid = static_cast<uint32_t>(tiles < static_cast<uint64_t>(sm_count) ? tiles : static_cast<uint64_t>(sm_count));
    return launch_following(expert_product_kernel<kTokens, Out>, grid, S::kThreads, shared_bytes, stream, a, weight_map, row_map);
}

template<typename Out>
cudaError_t launch_product(const ProductArgs& a, int sm_count, cudaStream_t stream)
{
    const uint32_t per_expert = (a.rows + a.expert_count - 1u) / a.expert_count;
    if (per_expert <= 16u)
        return launch_tiles<16, Out>(a, sm_count, stream);
    if (per_expert <= 32u)
        return launch_tiles<32, Out>(a, sm_count, stream);
    if (per_expert <= 64u)
        return launch_tiles<64, Out>(a, sm_count, stream);
    return launch_tiles<128, Out>(a, sm_count, stream);
}

} // namespace

cudaError_t launch_expert_product(const ProductArgs& args, int out_dtype, int sm_count, cudaStream_t stream)
{
    return out_dtype == MOE_DTYPE_F32 ? launch_product<float>(args, sm_count, stream) : launch_product<__nv_bfloat16>(args, sm_count, stream);
}

} // namespace moe
