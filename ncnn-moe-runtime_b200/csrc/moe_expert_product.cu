// The experts' matrix products in e4m3 with a scale for each block of 128:
//   out[r, n] = sum_b scales[b, r] * weight_scales[e, n / 128, b] * sum_{k in b} values[r, k] * weights[e, n, k]
//
// Per block of 128 columns the tensor cores compute the inner sums of a tile into a fresh accumulator in tensor memory, four
// instructions of 32 columns each; other warps read it out and add it to their registers times the product of the two scales,
// itself rounded to fp32, one fused multiply-add per element of the tile and block.  Two kernels:
//   few rows an expert   a tile is 128 outputs (the 128 lanes of an accumulator) by 16, 32 or 64 rows (its columns): the rows of
//                        a decode step do not fill a tile of 128 with padding.  Bound by the weights from HBM.
//   many rows            a tile is 128 rows by 256 outputs: a thread sums for one row, so that a block's factor is one register.
//                        Bound by the weights, or by what eight warps can take out of tensor memory and sum: with 128 sums a thread no
//                        others fit beside them to cover the waits (4096^3: tensor pipe 50 %, issue slots 49 %).
// Roles of a CTA, which stays for all its tiles: a thread that requests tiles of both operands from the copy engine, threads
// that issue the products, warps that scale, sum and store.  They pass a ring of operand stages and a few accumulators to each
// other through mbarriers, so that copies, products and sums of different blocks, and of different tiles, overlap.

#include "moe_internal.h"
#include "moe_tensor.cuh"

namespace moe {

namespace {

constexpr uint32_t kBlockBytes = MOE_EXPERT_BLOCK;
constexpr uint32_t kLanes = 128;        // of an accumulator
constexpr uint32_t kTallTile = kLanes * kBlockBytes;
constexpr uint32_t kGroupTiles = 16;    // row tiles that share a weight tile before the next one is taken
constexpr uint32_t kRoleThreads = 128;  // four warps that copy and issue; those that sum come behind them

// ---- tiles ------------------------------------------------------------------------------

struct Tile
{
    uint32_t expert;
    uint32_t first_row;
    uint32_t rows;
    uint32_t output_tile;
};

// The tile-th tile of the call.  first_tile: [experts + 1] tiles before each expert's.  Within an expert, groups of row tiles
// share a weight tile before the next weight tile is taken: a wave of CTAs then reads a few of both from L2.
template<uint32_t kRows>
__device__ __forceinline__ Tile find_tile(const ProductArgs& a, const uint32_t* first_tile, uint32_t tile, uint32_t output_tiles)
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
    const uint32_t row_tiles = (end - begin + kRows - 1u) / kRows;
    const uint32_t local = tile - first_tile[low];
    const uint32_t group = local / (kGroupTiles * output_tiles);
    const uint32_t in_group = local - group * kGroupTiles * output_tiles;
    const uint32_t width = min(kGroupTiles, row_tiles - group * kGroupTiles);
    found.output_tile = in_group / width;
    const uint32_t row_tile = group * kGroupTiles + in_group - found.output_tile * width;
    found.first_row = begin + row_tile * kRows;
    found.rows = min(kRows, end - found.first_row);
    return found;
}

// Tiles before every expert's, by all threads; returns false when the offsets descend or exceed the rows.
template<uint32_t kRows>
__device__ __forceinline__ bool count_tiles(const ProductArgs& a, uint32_t* first_tile, uint32_t output_tiles)
{
    __shared__ uint32_t warp_totals[32];
    const uint32_t per = (a.expert_count + blockDim.x - 1u) / blockDim.x;
    const uint32_t begin = min(a.expert_count, threadIdx.x * per), end = min(a.expert_count, begin + per);
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    bool good = true;
    uint32_t mine = 0;
    for (uint32_t e = begin; e < end; ++e)
    {
        const uint32_t first = a.expert_offsets != nullptr ? a.expert_offsets[e] : 0u;
        const uint32_t last = a.expert_offsets != nullptr ? a.expert_offsets[e + 1u] : a.rows;
        good = good && first <= last && last <= a.rows;
        mine += (last - first + kRows - 1u) / kRows * output_tiles;
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
        before += (last - first + kRows - 1u) / kRows * output_tiles;
    }
    if (end == a.expert_count && begin < end)
        first_tile[a.expert_count] = before;
    return true;
}

// ---- roles that both kernels have ----------------------------------------------------------

// No copy may land after the CTA has left: the last ones are waited for, in the order of their requests.
__device__ __forceinline__ void wait_for_copies(uint32_t full, const Cursor& cursor, uint32_t stages, uint32_t issued)
{
    for (uint32_t back = min(issued, stages); back > 0u; --back)
    {
        const uint32_t slot = (cursor.slot + stages - back) % stages;
        const uint32_t parity = slot < cursor.slot ? cursor.parity : cursor.parity ^ 1u;
        for (uint32_t spin = 0; spin < kSpinLimit && !barrier_test(full + 8u * slot, parity); ++spin)
            ;
    }
}

struct ProductRings
{
    uint32_t stages; // operand tiles: the tall one (lanes), then the wide one (columns)
    uint32_t full;
    uint32_t empty;
    uint32_t sum_full;
    uint32_t sum_empty;
};

// Issues the products of `count` blocks in a row, the first of them block `block` of its tile.  One thread.
template<uint32_t kStages, uint32_t kStageBytes, uint32_t kAccumulators, uint32_t kWide>
__device__ __forceinline__ void issue_products(const ProductRings& rings, uint32_t memory_base, uint32_t count, uint32_t block, uint32_t columns, volatile uint32_t* stalled)
{
    constexpr uint32_t kDescriptor = product_descriptor(kLanes, kWide);
    const uint32_t blocks = (columns + MOE_EXPERT_BLOCK - 1u) / MOE_EXPERT_BLOCK;
    const uint32_t last_steps = (columns - (blocks - 1u) * MOE_EXPERT_BLOCK + 31u) / 32u;
    Cursor cursor, sum;
    uint32_t done = 0;
    for (; done < count; ++done)
    {
        if (!barrier_wait(rings.sum_empty + 8u * sum.slot, sum.parity ^ 1u, stalled) || !barrier_wait(rings.full + 8u * cursor.slot, cursor.parity, stalled))
            break;
        memory_fence_after();
        const uint32_t stage = rings.stages + cursor.slot * kStageBytes;
        const uint64_t tall = tile_descriptor(stage), wide = tile_descriptor(stage + kTallTile);
        // what lies behind the last column is zero: whole steps of it are left out
        const uint32_t steps = ++block == blocks ? last_steps : 4u;
        block = block == blocks ? 0u : block;
#pragma unroll
        for (uint32_t step = 0; step < 4u; ++step)
            if (step < steps)
                issue_product(memory_base + sum.slot * kWide, tall + 2u * step, wide + 2u * step, kDescriptor, step != 0u);
        commit_products(rings.empty + 8u * cursor.slot);
        commit_products(rings.sum_full + 8u * sum.slot);
        cursor.advance(kStages);
        sum.advance(kAccumulators);
    }
    // tensor memory is given back at the end: the last product must be done, also when somebody stalled
    if (done > 0u)
    {
        const uint32_t slot = sum.slot == 0u ? kAccumulators - 1u : sum.slot - 1u;
        const uint32_t parity = sum.slot == 0u ? sum.parity ^ 1u : sum.parity;
        for (uint32_t spin = 0; spin < kSpinLimit && !barrier_test(rings.sum_full + 8u * slot, parity); ++spin)
            ;
    }
}

// ---- few rows an expert ----------------------------------------------------------------------

constexpr uint32_t kScaleGroup = 4; // blocks whose scales are passed on together
constexpr uint32_t kScaleSlots = 2; // groups of scales that wait for the sums
constexpr uint32_t kMostParts = 8;  // CTAs that share a tile
constexpr uint32_t kLeastPart = 4;  // blocks of each of them

template<int kTokens>
struct FewShape
{
    static constexpr uint32_t kStageBytes = kTallTile + kTokens * kBlockBytes;
    static constexpr uint32_t kStages = kTokens <= 16 ? 10u : kTokens <= 32 ? 9u : 8u;
    static constexpr uint32_t kAccumulators = 4;
    static constexpr uint32_t kMemoryColumns = kTokens * kAccumulators;
    static constexpr uint32_t kSumWarps = 4;
    static constexpr uint32_t kThreads = kRoleThreads + 32u * kSumWarps;
    static constexpr uint32_t kChunk = kTokens < 32 ? kTokens : 32; // columns read from tensor memory at once
    static constexpr uint32_t kScaleBytes = kScaleSlots * kScaleGroup * kTokens * 4u;
    static constexpr uint32_t kRawGroupBytes = kScaleGroup * kTokens * 4u + 128u; // scales of a group as they were copied, the weights' behind the rows'
    static constexpr uint32_t kBarriers = 2u * kStages + 2u * kAccumulators + 2u * kScaleSlots;
    static constexpr uint32_t kFixedBytes = kStages * kStageBytes + kScaleBytes + 2u * kRawGroupBytes + kBarriers * 8u + 64u;
};

// four floats in another CTA's shared memory
__device__ __forceinline__ float4 load_shared_of_cta(uint32_t address, uint32_t cta)
{
    float4 value;
    asm volatile(
        "{\n"
        ".reg .u32 remote;\n"
        "mapa.shared::cluster.u32 remote, %4, %5;\n"
        "ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [remote];\n"
        "}\n"
        : "=f"(value.x), "=f"(value.y), "=f"(value.z), "=f"(value.w)
        : "r"(address), "r"(cta)
        : "memory");
    return value;
}
__device__ __forceinline__ void store_output(float* target, float value)
{
    *target = value;
}
__device__ __forceinline__ void store_output(__nv_bfloat16* target, float value)
{
    *target = __float2bfloat16_rn(value);
}

template<int kTokens, typename Out>
__global__ void __launch_bounds__(FewShape<kTokens>::kThreads, 1)
    expert_product_few_kernel(const ProductArgs a, const __grid_constant__ CUtensorMap weight_map, const __grid_constant__ CUtensorMap row_map, const uint32_t split)
{
    using S = FewShape<kTokens>;
    extern __shared__ unsigned char shared_raw[];
    __shared__ uint32_t memory_base_shared;
    __shared__ volatile uint32_t stalled;
    unsigned char* const shared = shared_raw + ((1024u - (shared_address(shared_raw) & 1023u)) & 1023u);
    ProductRings rings;
    rings.stages = shared_address(shared);
    const uint32_t scale_slots = rings.stages + S::kStages * S::kStageBytes;
    rings.full = scale_slots + S::kScaleBytes + 2u * S::kRawGroupBytes;
    rings.empty = rings.full + 8u * S::kStages;
    rings.sum_full = rings.empty + 8u * S::kStages;
    rings.sum_empty = rings.sum_full + 8u * S::kAccumulators;
    const uint32_t scale_full = rings.sum_empty + 8u * S::kAccumulators;
    const uint32_t scale_empty = scale_full + 8u * kScaleSlots;
    uint32_t* const first_tile = reinterpret_cast<uint32_t*>(shared + S::kStages * S::kStageBytes + S::kScaleBytes + 2u * S::kRawGroupBytes + 8u * S::kBarriers);
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;

    if (threadIdx.x == 0)
    {
        for (uint32_t i = 0; i < S::kStages; ++i)
        {
            barrier_init(rings.full + 8u * i, 1u);
            barrier_init(rings.empty + 8u * i, 1u);
        }
        for (uint32_t i = 0; i < S::kAccumulators; ++i)
        {
            barrier_init(rings.sum_full + 8u * i, 1u);
            barrier_init(rings.sum_empty + 8u * i, S::kSumWarps);
        }
        for (uint32_t i = 0; i < kScaleSlots; ++i)
        {
            barrier_init(scale_full + 8u * i, 1u);
            barrier_init(scale_empty + 8u * i, S::kSumWarps);
        }
        stalled = 0u;
        barrier_init_fence();
    }
    if (warp == 3u)
        allocate_memory(shared_address(&memory_base_shared), S::kMemoryColumns);
    memory_sync();
    const uint32_t memory_base = memory_base_shared;

    wait_for_previous_kernel();
    // The next kernel may begin, up to its own wait: a layer of one token 20.0 -> 17.9 us, of 1024 tokens 91.3 -> 88.8.
    grid_dependency_release();
    const uint32_t blocks = (a.columns + MOE_EXPERT_BLOCK - 1u) / MOE_EXPERT_BLOCK;
    const uint32_t output_tiles = (a.outputs + kLanes - 1u) / kLanes; // blocks of the weights' scales, too
    const bool good = count_tiles<kTokens>(a, first_tile, output_tiles);
    __syncthreads();
    const uint32_t tiles = good ? first_tile[a.expert_count] : 0u;
    if (!good && threadIdx.x == 0)
        atomicOr(a.flags, MOE_EXPERT_FLAG_OFFSETS);
    // With a split, a cluster has one tile and each of its CTAs a part of the columns.
    const uint32_t cta = split > 1u ? cta_in_cluster() : 0u;
    const uint32_t first = blockIdx.x / split, stride = gridDim.x / split;
    const uint32_t begin = blocks * cta / split, end = blocks * (cta + 1u) / split;

    if (warp == 0u)
    {
        if (elect_one())
        {
            Cursor cursor;
            uint32_t issued = 0;
            for (uint32_t t = first; t < tiles && stalled == 0u; t += stride)
            {
                const Tile tile = find_tile<kTokens>(a, first_tile, t, output_tiles);
                // past an expert's last output lie the next one's weights, and zeros behind the last row: neither is stored
                const uint32_t weight_row = tile.expert * a.outputs + tile.output_tile * kLanes;
                for (uint32_t block = begin; block < end; ++block)
                {
                    if (!barrier_wait(rings.empty + 8u * cursor.slot, cursor.parity ^ 1u, &stalled))
                        break;
                    const uint32_t stage = rings.stages + cursor.slot * S::kStageBytes;
                    const uint32_t barrier = rings.full + 8u * cursor.slot;
                    barrier_expect_bytes(barrier, S::kStageBytes);
                    copy_tile(stage, &weight_map, block * kBlockBytes, weight_row, barrier);
                    copy_tile(stage + kTallTile, &row_map, block * kBlockBytes, tile.first_row, barrier);
                    cursor.advance(S::kStages);
                    ++issued;
                }
            }
            wait_for_copies(rings.full, cursor, S::kStages, issued);
        }
    }
    else if (warp == 1u)
    {
        if (elect_one())
            issue_products<S::kStages, S::kStageBytes, S::kAccumulators, kTokens>(
                rings, memory_base, first < tiles ? ((tiles - first - 1u) / stride + 1u) * (end - begin) : 0u, begin, a.columns, &stalled);
    }
    else if (warp == 2u)
    {
        // The products of the scales, up to four blocks of a tile at a time: the scales of the group behind this one are on their
        // way (also those of the next tile) while this group's are multiplied.
        constexpr uint32_t kPerLane = (kTokens + 31u) / 32u;
        const uint32_t raw_slots = scale_slots + S::kScaleBytes;
        uint32_t ahead_tile = begin < end ? first : tiles, ahead_slot = 0, ahead_left = 0; // its blocks that are left
        const float* ahead_scales = nullptr;
        const float* ahead_weights = nullptr;
        uint32_t ahead_rows = 0;
        const auto request = [&]() {
            if (ahead_tile < tiles)
            {
                if (ahead_left == 0u)
                {
                    const Tile tile = find_tile<kTokens>(a, first_tile, ahead_tile, output_tiles);
                    ahead_weights = a.weight_scales + (static_cast<size_t>(tile.expert) * output_tiles + tile.output_tile) * blocks + begin;
                    ahead_scales = a.scales + static_cast<size_t>(begin) * a.rows + tile.first_row;
                    ahead_rows = tile.rows;
                    ahead_left = end - begin;
                }
                const uint32_t raw = raw_slots + ahead_slot * S::kRawGroupBytes + 4u * lane;
                const uint32_t count = min(kScaleGroup, ahead_left);
#pragma unroll
                for (uint32_t i = 0; i < kScaleGroup; ++i)
                {
                    if (i < count)
                    {
#pragma unroll
                        for (uint32_t j = 0; j < kPerLane; ++j)
                        {
                            const uint32_t row = lane + 32u * j;
                            if (kTokens >= 32 || lane < kTokens)
                                copy_word(raw + (i * kTokens + 32u * j) * 4u, ahead_scales + (row < ahead_rows ? row : 0u), row < ahead_rows);
                        }
                        ahead_scales += a.rows;
                    }
                }
                if (lane < count)
                    copy_word(raw + kScaleGroup * kTokens * 4u, ahead_weights + lane, true);
                ahead_weights += count;
                ahead_left -= count;
                if (ahead_left == 0u)
                    ahead_tile += stride;
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            ahead_slot ^= 1u;
        };
        Cursor cursor;
        uint32_t raw_slot = 0;
        request();
        bool running = true;
        for (uint32_t t = first; t < tiles && running; t += stride)
        {
            for (uint32_t block = begin; block < end; block += kScaleGroup)
            {
                request();
                asm volatile("cp.async.wait_group 1;" ::: "memory");
                __syncwarp(); // the weights' scales are other lanes' copies
                running = barrier_wait_warp(scale_empty + 8u * cursor.slot, cursor.parity ^ 1u, &stalled);
                if (!running)
                    break;
                const uint32_t raw = raw_slots + raw_slot * S::kRawGroupBytes;
                const uint32_t slot = scale_slots + cursor.slot * kScaleGroup * kTokens * 4u + 4u * lane;
                // (blocks behind the last one: what an earlier group left there, which nobody reads)
                const uint4 weights = load_shared_16(raw + kScaleGroup * kTokens * 4u);
                const float weight[kScaleGroup] = {__uint_as_float(weights.x), __uint_as_float(weights.y), __uint_as_float(weights.z), __uint_as_float(weights.w)};
    #pragma unroll
                for (uint32_t i = 0; i < kScaleGroup; ++i)
                {
    #pragma unroll
                    for (uint32_t j = 0; j < kPerLane; ++j)
                        if (kTokens >= 32 || lane < kTokens)
                            asm volatile("st.shared.f32 [%0], %1;" ::"r"(slot + (i * kTokens + 32u * j) * 4u),
                                         "f"(__uint_as_float(load_shared_32(raw + (i * kTokens + 32u * j + lane) * 4u)) * weight[i])
                                         : "memory");
                }
                __syncwarp();
                if (lane == 0u)
                    barrier_arrive(scale_full + 8u * cursor.slot);
                cursor.advance(kScaleSlots);
                raw_slot ^= 1u;
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    }
    else if (warp >= 4u)
    {
        const uint32_t quarter = warp & 3u; // lanes of tensor memory that this warp can read
        const uint32_t memory = memory_base + (quarter << 21);
        const uint32_t tile_lane = quarter * 32u + lane;
        Cursor sum, scale;
        bool running = true;
        for (uint32_t t = first; t < tiles && running; t += stride)
        {
            float sums[kTokens];
#pragma unroll
            for (uint32_t i = 0; i < kTokens; ++i)
                sums[i] = 0.0f;
            for (uint32_t block = begin; block < end; ++block)
            {
                const uint32_t in_group = (block - begin) % kScaleGroup;
                running = (in_group != 0u || barrier_wait_warp(scale_full + 8u * scale.slot, scale.parity, &stalled)) &&
                          barrier_wait_warp(rings.sum_full + 8u * sum.slot, sum.parity, &stalled);
                if (!running)
                    break;
                memory_fence_after();
                const uint32_t factors = scale_slots + (scale.slot * kScaleGroup + in_group) * kTokens * 4u;
                const uint32_t source = memory + sum.slot * kTokens;
                // at most two chunks, on their way together
                constexpr uint32_t kChunks = kTokens / S::kChunk;
                static_assert(kChunks <= 2u, "an accumulator is read with two requests");
                uint32_t part[kChunks][S::kChunk];
#pragma unroll
                for (uint32_t chunk = 0; chunk < kChunks; ++chunk)
                    load_accumulator<S::kChunk>(part[chunk], source + chunk * S::kChunk);
#pragma unroll
                for (uint32_t chunk = 0; chunk < kChunks; ++chunk)
                    wait_accumulator<S::kChunk>(part[chunk]);
                // all of it is in registers: the accumulator may be written again
                memory_fence_before();
                __syncwarp();
                if (lane == 0u)
                    barrier_arrive(rings.sum_empty + 8u * sum.slot);
#pragma unroll
                for (uint32_t i = 0; i < kTokens; i += 4u)
                {
                    const uint4 factor = load_shared_16(factors + i * 4u);
                    const uint32_t* p = part[i / S::kChunk] + i % S::kChunk;
                    sums[i] = fmaf(__uint_as_float(p[0]), __uint_as_float(factor.x), sums[i]);
                    sums[i + 1u] = fmaf(__uint_as_float(p[1]), __uint_as_float(factor.y), sums[i + 1u]);
                    sums[i + 2u] = fmaf(__uint_as_float(p[2]), __uint_as_float(factor.z), sums[i + 2u]);
                    sums[i + 3u] = fmaf(__uint_as_float(p[3]), __uint_as_float(factor.w), sums[i + 3u]);
                }
                sum.advance(S::kAccumulators);
                if (in_group + 1u == kScaleGroup || block + 1u == end)
                {
                    __syncwarp();
                    if (lane == 0u)
                        barrier_arrive(scale_empty + 8u * scale.slot);
                    scale.advance(kScaleSlots);
                }
            }
            if (!running)
                break;
            if (split > 1u)
            {
                // the cluster's parts are added below; the stages are free: the last product that read them is done
#pragma unroll
                for (uint32_t i = 0; i < kTokens; ++i)
                    asm volatile("st.shared.f32 [%0], %1;" ::"r"(rings.stages + (i * kLanes + tile_lane) * 4u), "f"(sums[i]) : "memory");
                break;
            }
            const Tile tile = find_tile<kTokens>(a, first_tile, t, output_tiles);
            const uint32_t output = tile.output_tile * kLanes + tile_lane;
            if (output < a.outputs)
            {
                Out* target = static_cast<Out*>(a.out) + static_cast<size_t>(tile.first_row) * a.out_stride + output;
#pragma unroll
                for (uint32_t i = 0; i < kTokens; ++i)
                    if (i < tile.rows)
                        store_output(target + static_cast<size_t>(i) * a.out_stride, sums[i]);
            }
        }
    }
    memory_sync();
    if (warp == 3u)
        free_memory(memory_base, S::kMemoryColumns);
    if (threadIdx.x == 0 && stalled != 0u)
        atomicOr(a.flags, MOE_EXPERT_FLAG_STALLED);
    if (split > 1u)
    {
        // Each CTA adds the parts of some of the rows, in the order of the columns: a warp a row, four outputs a lane, all parts
        // requested before the first is added.
        cluster_sync();
        if (first < tiles)
        {
            const Tile tile = find_tile<kTokens>(a, first_tile, first, output_tiles);
            const uint32_t output = tile.output_tile * kLanes + 4u * lane;
            for (uint32_t i = cta + split * warp; i < tile.rows; i += split * (S::kThreads / 32u))
            {
                float4 parts[kMostParts];
#pragma unroll
                for (uint32_t part = 0; part < kMostParts; ++part)
                    if (part < split)
                        parts[part] = load_shared_of_cta(rings.stages + (i * kLanes + 4u * lane) * 4u, part);
                float total[4] = {parts[0].x, parts[0].y, parts[0].z, parts[0].w};
#pragma unroll
                for (uint32_t part = 1; part < kMostParts; ++part)
                {
                    if (part < split)
                    {
                        total[0] += parts[part].x;
                        total[1] += parts[part].y;
                        total[2] += parts[part].z;
                        total[3] += parts[part].w;
                    }
                }
                Out* target = static_cast<Out*>(a.out) + static_cast<size_t>(tile.first_row + i) * a.out_stride + output;
#pragma unroll
                for (uint32_t j = 0; j < 4u; ++j)
                    if (output + j < a.outputs)
                        store_output(target + j, total[j]);
            }
        }
        __syncwarp();
        cluster_sync(); // nobody leaves while its part is read
    }
}

// ---- many rows an expert ---------------------------------------------------------------------

constexpr uint32_t kTileOutputs = 256;

struct ManyShape
{
    static constexpr uint32_t kStageBytes = kTallTile + kTileOutputs * kBlockBytes;
    static constexpr uint32_t kStages = 4;
    static constexpr uint32_t kAccumulators = 2;
    static constexpr uint32_t kMemoryColumns = kTileOutputs * kAccumulators;
    static constexpr uint32_t kSumWarps = 8;
    static constexpr uint32_t kThreads = kRoleThreads + 32u * kSumWarps;
    static constexpr uint32_t kColumns = kTileOutputs / 2u; // outputs that a warp sums: one block of the weights' scales
    static constexpr uint32_t kChunk = 32;
    static constexpr uint32_t kBarriers = 2u * kStages + 2u * kAccumulators;
    static constexpr uint32_t kTurnStride = 17; // words of a row that a warp turns around, one of them so that columns lie in different banks
    static constexpr uint32_t kTurnBytes = 32u * kTurnStride * 4u;
    static constexpr uint32_t kFixedBytes = kStages * kStageBytes + kBarriers * 8u + kSumWarps * kTurnBytes + 64u;
    // 128 sums in a thread: the warps that sum take registers over from the other roles.  Launched with 168 a thread:
    // 128 * 40 + 256 * 232 = 384 * 168.
    static constexpr uint32_t kRoleRegisters = 40;
    static constexpr uint32_t kSumRegisters = 232;
};

// 32 bytes of outputs of one row, as they are stored.
__device__ __forceinline__ void pack_outputs(uint32_t (&words)[8], const float (&values)[8])
{
#pragma unroll
    for (int i = 0; i < 8; ++i)
        words[i] = __float_as_uint(values[i]);
}
__device__ __forceinline__ void pack_outputs(uint32_t (&words)[8], const float (&values)[16])
{
#pragma unroll
    for (int i = 0; i < 8; ++i)
    {
        const __nv_bfloat162 pair = __floats2bfloat162_rn(values[2 * i], values[2 * i + 1]);
        words[i] = *reinterpret_cast<const uint32_t*>(&pair);
    }
}

// Four lanes that follow each other, with four pieces each: lane j of them gets piece j of each one, in their order.
__device__ __forceinline__ void exchange_of_four(uint32_t (&words)[4][8], uint32_t lane)
{
#pragma unroll
    for (uint32_t bit = 1; bit < 4u; bit <<= 1)
    {
        const bool upper = (lane & bit) != 0u;
#pragma unroll
        for (uint32_t v = 0; v < 4u; ++v)
        {
            if ((v & bit) != 0u)
                continue;
#pragma unroll
            for (uint32_t i = 0; i < 8u; ++i)
            {
                const uint32_t other = __shfl_xor_sync(kFullMask, upper ? words[v][i] : words[v | bit][i], bit);
                words[v][i] = upper ? other : words[v][i];
                words[v | bit][i] = upper ? words[v | bit][i] : other;
            }
        }
    }
}

// Outputs that a lane stores at once as one vector, or two of 16 bytes.
template<typename Out>
constexpr uint32_t kStoreVector = 32u / sizeof(Out);

// Rows of outputs start and end at multiples of kAlignment bytes: 32, 16, or (1) anywhere.
template<typename Out, uint32_t kAlignment>
__global__ void __launch_bounds__(ManyShape::kThreads, 1)
    expert_product_many_kernel(const ProductArgs a, const __grid_constant__ CUtensorMap weight_map, const __grid_constant__ CUtensorMap row_map)
{
    using S = ManyShape;
    extern __shared__ unsigned char shared_raw[];
    __shared__ uint32_t memory_base_shared;
    __shared__ volatile uint32_t stalled;
    unsigned char* const shared = shared_raw + ((1024u - (shared_address(shared_raw) & 1023u)) & 1023u);
    ProductRings rings;
    rings.stages = shared_address(shared);
    rings.full = rings.stages + S::kStages * S::kStageBytes;
    rings.empty = rings.full + 8u * S::kStages;
    rings.sum_full = rings.empty + 8u * S::kStages;
    rings.sum_empty = rings.sum_full + 8u * S::kAccumulators;
    uint32_t* const first_tile = reinterpret_cast<uint32_t*>(shared + S::kStages * S::kStageBytes + 8u * S::kBarriers + S::kSumWarps * S::kTurnBytes);
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;

    if (threadIdx.x == 0)
    {
        for (uint32_t i = 0; i < S::kStages; ++i)
        {
            barrier_init(rings.full + 8u * i, 1u);
            barrier_init(rings.empty + 8u * i, 1u);
        }
        for (uint32_t i = 0; i < S::kAccumulators; ++i)
        {
            barrier_init(rings.sum_full + 8u * i, 1u);
            barrier_init(rings.sum_empty + 8u * i, S::kSumWarps);
        }
        stalled = 0u;
        barrier_init_fence();
    }
    __syncwarp();
    if (warp == 3u)
        allocate_memory(shared_address(&memory_base_shared), S::kMemoryColumns);
    memory_sync();
    const uint32_t memory_base = memory_base_shared;

    wait_for_previous_kernel();
    grid_dependency_release();
    const uint32_t blocks = (a.columns + MOE_EXPERT_BLOCK - 1u) / MOE_EXPERT_BLOCK;
    const uint32_t output_blocks = (a.outputs + MOE_EXPERT_BLOCK - 1u) / MOE_EXPERT_BLOCK;
    const uint32_t output_tiles = (a.outputs + kTileOutputs - 1u) / kTileOutputs;
    const bool good = count_tiles<kLanes>(a, first_tile, output_tiles);
    __syncthreads();
    const uint32_t tiles = good ? first_tile[a.expert_count] : 0u;
    if (!good && threadIdx.x == 0)
        atomicOr(a.flags, MOE_EXPERT_FLAG_OFFSETS);

    if (warp < 4u)
    {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::kRoleRegisters));
        if (warp == 0u)
        {
            if (elect_one())
            {
                Cursor cursor;
                uint32_t issued = 0;
                for (uint32_t t = blockIdx.x; t < tiles && stalled == 0u; t += gridDim.x)
                {
                    const Tile tile = find_tile<kLanes>(a, first_tile, t, output_tiles);
                    // what lies past an expert's rows or outputs belongs to the next one, or is zero: it is not stored
                    const uint32_t weight_row = tile.expert * a.outputs + tile.output_tile * kTileOutputs;
                    for (uint32_t block = 0; block < blocks; ++block)
                    {
                        if (!barrier_wait(rings.empty + 8u * cursor.slot, cursor.parity ^ 1u, &stalled))
                            break;
                        const uint32_t stage = rings.stages + cursor.slot * S::kStageBytes;
                        const uint32_t barrier = rings.full + 8u * cursor.slot;
                        barrier_expect_bytes(barrier, S::kStageBytes);
                        copy_tile(stage, &row_map, block * kBlockBytes, tile.first_row, barrier);
                        copy_tile(stage + kTallTile, &weight_map, block * kBlockBytes, weight_row, barrier);
                        cursor.advance(S::kStages);
                        ++issued;
                    }
                }
                wait_for_copies(rings.full, cursor, S::kStages, issued);
            }
        }
        else if (warp == 1u)
        {
            if (elect_one())
                issue_products<S::kStages, S::kStageBytes, S::kAccumulators, kTileOutputs>(
                    rings, memory_base, blockIdx.x < tiles ? ((tiles - blockIdx.x - 1u) / gridDim.x + 1u) * blocks : 0u, 0u, a.columns, &stalled);
        }
    }
    else
    {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(S::kSumRegisters));
        const uint32_t quarter = warp & 3u;      // lanes of tensor memory that this warp can read
        const uint32_t half = (warp - 4u) / 4u;  // of the tile's outputs
        const uint32_t memory = memory_base + (quarter << 21) + half * S::kColumns;
        const uint32_t row = quarter * 32u + lane; // of a tile
        // The scales are read two blocks ahead, across tiles.  The loads stand outside of any condition (behind the last tile they
        // read the first scales of all): a value that is merged with another one behind a branch is waited for there.
        uint32_t ahead_tile = blockIdx.x, ahead_block = 0;
        const float* ahead_scales = nullptr;
        const float* ahead_weights = nullptr;
        float next_scale[2], next_weight[2];
        Tile next_tile = {}; // whose first blocks were requested last
        const auto request = [&]() {
            if (ahead_block == 0u)
            {
                ahead_scales = a.scales;
                ahead_weights = a.weight_scales;
                if (ahead_tile < tiles)
                {
                    next_tile = find_tile<kLanes>(a, first_tile, ahead_tile, output_tiles);
                    // (an odd number of blocks: the second half of the last tile has no scales, and is not stored)
                    const uint32_t output_block = min(next_tile.output_tile * 2u + half, output_blocks - 1u);
                    ahead_weights += (static_cast<size_t>(next_tile.expert) * output_blocks + output_block) * blocks;
                    ahead_scales += next_tile.first_row + (row < next_tile.rows ? row : 0u);
                }
            }
            const bool second = ahead_block + 1u < blocks;
            next_scale[0] = ahead_scales[0];
            next_weight[0] = ahead_weights[0];
            next_scale[1] = ahead_scales[second ? a.rows : 0u];
            next_weight[1] = ahead_weights[second ? 1u : 0u];
            ahead_scales += 2u * static_cast<size_t>(a.rows);
            ahead_weights += 2u;
            ahead_block += 2u;
            if (ahead_block >= blocks)
            {
                ahead_block = 0;
                ahead_tile += gridDim.x;
            }
        };
        if (blockIdx.x < tiles)
            request();
        Cursor sum;
        bool running = true;
        for (uint32_t t = blockIdx.x; t < tiles && running; t += gridDim.x)
        {
            const Tile tile = next_tile;
            // a warp whose 32 rows are not the expert's only passes the accumulators on
            const bool idle = quarter * 32u >= tile.rows;
            float sums[S::kColumns];
#pragma unroll
            for (uint32_t i = 0; i < S::kColumns; ++i)
                sums[i] = 0.0f;
            for (uint32_t block = 0; block < blocks && running; block += 2u)
            {
                const float factors[2] = {next_scale[0] * next_weight[0], next_scale[1] * next_weight[1]};
                request();
#pragma unroll
                for (uint32_t of_two = 0; of_two < 2u; ++of_two)
                {
                    if (block + of_two >= blocks)
                        break;
                    running = barrier_wait_warp(rings.sum_full + 8u * sum.slot, sum.parity, &stalled);
                    if (!running)
                        break;
                    if (idle)
                    {
                        if (lane == 0u)
                            barrier_arrive(rings.sum_empty + 8u * sum.slot);
                        sum.advance(S::kAccumulators);
                        continue;
                    }
                    memory_fence_after();
                    const uint32_t source = memory + sum.slot * kTileOutputs;
                    const float factor = factors[of_two];
                    // Two chunks are on their way at a time, and the next two are requested as these are summed: while products
                    // run, tensor memory serves half as much to warps with one request outstanding.  (Single adds: the pairs of
                    // fma.f32x2 would have to be moved together first.)
                    constexpr uint32_t kChunks = S::kColumns / S::kChunk;
                    uint32_t part[2][S::kChunk];
                    load_accumulator<S::kChunk>(part[0], source);
                    load_accumulator<S::kChunk>(part[1], source + S::kChunk);
#pragma unroll
                    for (uint32_t chunk = 0; chunk < kChunks; ++chunk)
                    {
                        if (chunk % 2u == 0u)
                        {
                            wait_accumulator<S::kChunk>(part[0]);
                            wait_accumulator<S::kChunk>(part[1]);
                            if (chunk + 2u >= kChunks)
                            {
                                // all of it is in registers: the accumulator may be written again
                                memory_fence_before();
                                __syncwarp();
                                if (lane == 0u)
                                    barrier_arrive(rings.sum_empty + 8u * sum.slot);
                            }
                        }
#pragma unroll
                        for (uint32_t i = 0; i < S::kChunk; ++i)
                            sums[chunk * S::kChunk + i] = fmaf(__uint_as_float(part[chunk & 1u][i]), factor, sums[chunk * S::kChunk + i]);
                        if (chunk + 2u < kChunks)
                            load_accumulator<S::kChunk>(part[chunk & 1u], source + (chunk + 2u) * S::kChunk);
                    }
                    sum.advance(S::kAccumulators);
                }
            }
            if (!running)
                break;
            const uint32_t output = tile.output_tile * kTileOutputs + half * S::kColumns;
            if (idle || output >= a.outputs)
                continue;
            // Whole lines of 128 bytes, since the stores of all CTAs fall together: four lanes exchange what they have of four rows, and
            // each stores 32 bytes of every one of them.  4096 x 4096 x 4096 to bf16 74 us, each lane 32 bytes of its own row 76,
            // without storing 68; to fp32 80 and 85.
            constexpr uint32_t kVector = kStoreVector<Out>;
            const uint32_t count = min(S::kColumns, a.outputs - output);
            if constexpr (kAlignment >= 16u)
            {
                const uint32_t first_row = quarter * 32u + (lane & ~3u);
                Out* const target = static_cast<Out*>(a.out) + static_cast<size_t>(tile.first_row + first_row) * a.out_stride + output + (lane & 3u) * kVector;
#pragma unroll
                for (uint32_t i = 0; i < S::kColumns; i += 4u * kVector)
                {
                    uint32_t words[4][8];
#pragma unroll
                    for (uint32_t v = 0; v < 4u; ++v)
                    {
                        float values[kVector];
#pragma unroll
                        for (uint32_t j = 0; j < kVector; ++j)
                            values[j] = sums[i + v * kVector + j];
                        pack_outputs(words[v], values);
                    }
                    exchange_of_four(words, lane);
#pragma unroll
                    for (uint32_t r = 0; r < 4u; ++r)
                    {
                        const uint32_t(&w)[8] = words[r];
                        const uint32_t column = i + (lane & 3u) * kVector;
                        Out* const place = target + r * a.out_stride + i;
                        if (first_row + r >= tile.rows || column >= count)
                            continue;
                        if constexpr (kAlignment == 32u)
                        {
                            asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(place), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]),
                                         "r"(w[6]), "r"(w[7])
                                         : "memory");
                        }
                        else
                        {
                            *reinterpret_cast<uint4*>(place) = make_uint4(w[0], w[1], w[2], w[3]);
                            if (column + kVector <= count)
                                *reinterpret_cast<uint4*>(place + kVector / 2u) = make_uint4(w[4], w[5], w[6], w[7]);
                        }
                    }
                }
            }
            else
            {
                // Rows that start anywhere: the warp turns 64 bytes of its 32 rows around in shared memory and stores neighbouring
                // outputs side by side (4096 x 4096 x 4095 to bf16 92 us, each
                // lane those of its row 234; 128 experts of 120 rows x 768 x 2467 to fp32 114 and 268).
                constexpr uint32_t kPass = 64u / sizeof(Out);   // outputs
                constexpr uint32_t kAtOnce = 32u / kPass;       // rows
                unsigned char* const turn = shared + S::kStages * S::kStageBytes + 8u * S::kBarriers + (warp - 4u) * S::kTurnBytes;
                const uint32_t column = lane % kPass;
                const uint32_t end = min(32u, tile.rows - quarter * 32u);
                Out* const target = static_cast<Out*>(a.out) + static_cast<size_t>(tile.first_row + quarter * 32u) * a.out_stride + output + column;
#pragma unroll
                for (uint32_t i = 0; i < S::kColumns; i += kPass)
                {
                    if (i >= count)
                        break;
                    uint32_t words[2][8];
#pragma unroll
                    for (uint32_t v = 0; v < 2u; ++v)
                    {
                        float values[kVector];
#pragma unroll
                        for (uint32_t j = 0; j < kVector; ++j)
                            values[j] = sums[i + v * kVector + j];
                        pack_outputs(words[v], values);
                    }
                    __syncwarp();
#pragma unroll
                    for (uint32_t j = 0; j < 16u; ++j)
                        reinterpret_cast<uint32_t*>(turn)[lane * S::kTurnStride + j] = words[j / 8u][j % 8u];
                    __syncwarp();
#pragma unroll 8
                    for (uint32_t first = 0; first < end; first += kAtOnce)
                    {
                        const uint32_t r = first + lane / kPass;
                        const Out value = reinterpret_cast<const Out*>(turn + r * S::kTurnStride * 4u)[column];
                        if (r < end && i + column < count)
                            target[static_cast<size_t>(r) * a.out_stride + i] = value;
                    }
                }
            }
        }
    }
    memory_sync();
    if (warp == 3u)
        free_memory(memory_base, S::kMemoryColumns);
    if (threadIdx.x == 0 && stalled != 0u)
        atomicOr(a.flags, MOE_EXPERT_FLAG_STALLED);
}

// ---- launches -------------------------------------------------------------------------------

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                 CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_function()
{
    static std::atomic<EncodeTiled> found{nullptr};
    return found_once(found, [] {
        void* entry = nullptr;
        cudaDriverEntryPointQueryResult result;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &entry, 12000, cudaEnableDefault, &result) != cudaSuccess || result != cudaDriverEntryPointSuccess)
            entry = nullptr;
        return reinterpret_cast<EncodeTiled>(entry);
    });
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

template<typename... Parameters>
cudaError_t launch_tiles(void (*kernel)(ProductArgs, CUtensorMap, CUtensorMap, Parameters...), SharedOptIn& opt_in, const ProductArgs& a, uint32_t row_box, uint32_t weight_box,
                         uint64_t ctas, uint32_t cluster, uint32_t threads, size_t fixed_bytes, cudaStream_t stream, Parameters... more)
{
    CUtensorMap weight_map, row_map;
    if (!encode_rows(&weight_map, a.weights, a.columns, static_cast<uint64_t>(a.expert_count) * a.outputs, weight_box) ||
        !encode_rows(&row_map, a.values, a.columns, a.rows, row_box))
        return cudaErrorInvalidValue;
    const size_t shared_bytes = 1024u + fixed_bytes + sizeof(uint32_t) * (static_cast<size_t>(a.expert_count) + 1u);
    if (cudaError_t status = opt_in_shared(opt_in, kernel, shared_bytes))
        return status;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(static_cast<uint32_t>(ctas), 1, 1);
    config.blockDim = dim3(threads, 1, 1);
    config.dynamicSmemBytes = shared_bytes;
    config.stream = stream;
    cudaLaunchAttribute attributes[2] = {follow_closely(), {}};
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim.x = cluster;
    attributes[1].val.clusterDim.y = 1;
    attributes[1].val.clusterDim.z = 1;
    config.attrs = attributes;
    config.numAttrs = cluster > 1u ? 2 : 1;
    return cudaLaunchKernelEx(&config, kernel, a, weight_map, row_map, more...);
}

// The most tiles that any offsets give.
uint64_t most_tiles(const ProductArgs& a, uint32_t tile_rows, uint32_t tile_outputs)
{
    const uint64_t row_tiles = (static_cast<uint64_t>(a.rows) + tile_rows - 1u) / tile_rows + (a.expert_count < a.rows ? a.expert_count : a.rows) - 1u;
    return row_tiles * ((a.outputs + tile_outputs - 1u) / tile_outputs);
}

template<int kTokens, typename Out>
cudaError_t launch_few(const ProductArgs& a, int sm_count, cudaStream_t stream)
{
    using S = FewShape<kTokens>;
    static SharedOptIn opt_in;
    const uint64_t tiles = most_tiles(a, kTokens, kLanes), most = static_cast<uint64_t>(sm_count);
    const uint32_t blocks = (a.columns + MOE_EXPERT_BLOCK - 1u) / MOE_EXPERT_BLOCK;
    // Parts of one row x 4096 x 4096 (32 tiles): 1 10.2 us, 2 8.2, 4 6.9; 64 rows x 1024 x 4096 (8 tiles) 14.7, 10.6, 8.3, 8 parts
    // 7.7.  More than eight clusters of eight CTAs are not resident together (16 of them 14.3 us, as 32 of four 8.4).
    uint32_t split = 1;
    while (split < kMostParts && tiles * split * 2u <= (split * 2u == 8u ? 64u : most) && blocks >= split * 2u * kLeastPart)
        split *= 2u;
    return launch_tiles(expert_product_few_kernel<kTokens, Out>, opt_in, a, kTokens, kLanes, (tiles < most ? tiles * split : most), split, S::kThreads, S::kFixedBytes, stream, split);
}
template<typename Out, uint32_t kAlignment>
cudaError_t launch_many(const ProductArgs& a, int sm_count, cudaStream_t stream)
{
    using S = ManyShape;
    static SharedOptIn opt_in;
    const uint64_t tiles = most_tiles(a, kLanes, kTileOutputs), most = static_cast<uint64_t>(sm_count);
    return launch_tiles(expert_product_many_kernel<Out, kAlignment>, opt_in, a, kLanes, kTileOutputs, tiles < most ? tiles : most, 1u, S::kThreads, S::kFixedBytes, stream);
}

// Experts are taken to have equal numbers of rows.  Up to 32 a tile of as many rows wastes least (64 experts of 32 rows x
// 4096 x 4096: 32-row tiles 172 us, 64-row tiles 204, 128 x 256 tiles 187).  Above that the tiles' rates decide: a block of 64
// rows by 128 outputs takes three fifths of the time of one of 128 by 256, so the smaller ones win while they are one wave (one
// expert of 256 rows: 15.5 against 21.8 us) and lose from two on (512 rows: 27.0 against 22.2).  All of that at 4096 columns: with few,
// the rule is up to 1.5 times off (128 experts of 24 rows x 256 x 512: 12.9 us, tiles of 128 x 256 8.7).
template<typename Out>
cudaError_t launch_product(const ProductArgs& a, int sm_count, cudaStream_t stream)
{
    const uint64_t active = a.expert_count < a.rows ? a.expert_count : a.rows;
    const uint64_t rows = (a.rows + active - 1u) / active; // of an expert
    if (rows <= 16u)
        return launch_few<16, Out>(a, sm_count, stream);
    if (rows <= 32u)
        return launch_few<32, Out>(a, sm_count, stream);
    const auto waves = [&](uint64_t tile_rows, uint64_t tile_outputs) {
        const uint64_t tiles = active * ((rows + tile_rows - 1u) / tile_rows) * ((a.outputs + tile_outputs - 1u) / tile_outputs);
        return (tiles + sm_count - 1u) / sm_count;
    };
    if (waves(64u, kLanes) * 3u <= waves(kLanes, kTileOutputs) * 5u)
        return launch_few<64, Out>(a, sm_count, stream);
    // Where rows of outputs start and end decides how they are stored: 4096 x 4096 to bf16 74 us at multiples of 32 bytes (outputs 4096),
    // 78 of 16 (4088; 92 if they were turned around), 93 anywhere (4095).
    const uint64_t places = reinterpret_cast<uintptr_t>(a.out) | a.out_stride * sizeof(Out) | a.outputs * sizeof(Out);
    if (places % 32u == 0u)
        return launch_many<Out, 32u>(a, sm_count, stream);
    return places % 16u == 0u ? launch_many<Out, 16u>(a, sm_count, stream) : launch_many<Out, 1u>(a, sm_count, stream);
}

} // namespace

cudaError_t launch_expert_product(const ProductArgs& args, int out_dtype, int sm_count, cudaStream_t stream)
{
    return out_dtype == MOE_DTYPE_F32 ? launch_product<float>(args, sm_count, stream) : launch_product<__nv_bfloat16>(args, sm_count, stream);
}

} // namespace moe
