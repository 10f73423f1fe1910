// Rows to 8-bit blocks before the experts' products, and the routed rows back to
// their tokens behind them.

#include <cuda_fp8.h>

#include <type_traits>

#include "moe_common.cuh"
#include "moe_internal.h"

namespace moe {

namespace {

// ---- eight values of a row as floats ----------------------------------------------

// Eight values as they lie in memory: one 16-byte vector of bf16, two of fp32.
template<typename T>
struct Eight
{
    static constexpr int kVectors = sizeof(T) * 8 / 16;
    uint4 raw[kVectors];

    __device__ __forceinline__ void load(const T* source)
    {
#pragma unroll
        for (int i = 0; i < kVectors; ++i)
            raw[i] = *(reinterpret_cast<const uint4*>(source) + i);
    }
    // any alignment, the first `count` values; zeros behind them
    __device__ __forceinline__ void load_scalars(const T* source, uint32_t count)
    {
        T part[8] = {};
        for (uint32_t i = 0; i < 8u; ++i)
            if (i < count)
                part[i] = source[i];
        memcpy(raw, part, sizeof(part));
    }
    __device__ __forceinline__ void clear()
    {
#pragma unroll
        for (int i = 0; i < kVectors; ++i)
            raw[i] = make_uint4(0u, 0u, 0u, 0u);
    }
    __device__ __forceinline__ void unpack(float (&x)[8]) const
    {
        if constexpr (sizeof(T) == 4)
        {
#pragma unroll
            for (int i = 0; i < 2; ++i)
            {
                x[4 * i] = __uint_as_float(raw[i].x);
                x[4 * i + 1] = __uint_as_float(raw[i].y);
                x[4 * i + 2] = __uint_as_float(raw[i].z);
                x[4 * i + 3] = __uint_as_float(raw[i].w);
            }
        }
        else
        {
            const uint32_t words[4] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
            {
                x[2 * i] = __uint_as_float(words[i] << 16);
                x[2 * i + 1] = __uint_as_float(words[i] & 0xFFFF0000u);
            }
        }
    }
};

// ---- quantisation -------------------------------------------------------------------
//
// scale = max |x| / 448 over a block of 128 columns, value = e4m3(x / scale).  Sixteen lanes own a block, eight values each, so
// that a bf16 row is read in 16-byte vectors; a warp takes 1024 columns of a row (or 256: quantize_steps) and has all their loads in
// flight before the first maximum.  Large calls are bound by instructions before memory (16384 gated bf16 rows x 4096: 82 us,
// 4.1 TB/s, 72 % of the issue slots), so what belongs to a block is done once for the four blocks of a half warp: their maxima are
// reduced side by side until a lane has one of them, and it divides and inverts that one.

constexpr int kQuantizeThreads = 128;
constexpr float kE4m3Max = 448.0f;

__device__ __forceinline__ uint32_t to_e4m3_pair(float low, float high)
{
    return __nv_cvt_float2_to_fp8x2(make_float2(low, high), __NV_SATFINITE, __NV_E4M3);
}

__device__ __forceinline__ float approximate_reciprocal(float x)
{
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// a / b with r = 1 / b rounded to nearest, corrected once with the remainder: the exact quotient times 1 + e, |e| < 2^-45,
// rounded (the reciprocal and the first product are off by 2^-24 each; the correction multiplies that error with 2^-24, and a
// remainder of up to 25 bits is rounded itself).
__device__ __forceinline__ float divide_once(float a, float b, float r)
{
    const float q = __fmul_rn(a, r);
    return __fmaf_rn(__fmaf_rn(-q, b, a), r, q);
}

// gate / below * up where the short way below does not hold: infinities and NaN, and gates from -41 down.  From -88.7 down the
// denominator has left fp32, and the quotient is gate * exp(gate): in two halves.  Apart, since inlined it costs the common way a third.
__device__ __noinline__ float silu_gate_apart(float gate, float below, float up)
{
    if (gate < 0.0f && below == INFINITY)
    {
        const float half = expf(0.5f * gate);
        return gate * half * up * half;
    }
    return __fmul_rn(__fdiv_rn(gate, below), up);
}

// gate / (1 + exp(-gate)) * up; the quotient within a unit in the last place
__device__ __forceinline__ float silu_gate(float gate, float up)
{
    const float below = 1.0f + expf(-gate);
    // (from 2^126 on the reciprocal leaves the normal numbers; an infinity has no remainder)
    if (below < 0x1p60f && gate < INFINITY)
        return __fmul_rn(divide_once(gate, below, approximate_reciprocal(below)), up);
    return silu_gate_apart(gate, below, up);
}

// Whether one correction decides e4m3's rounding as the correctly rounded quotient does.  They differ only where the quotient
// is within 2^-45 of the middle between two fp32 numbers one of which is a tie of e4m3, a number of five bits: X / S = (m 2^20 +- 1)
// 2^k (1 + e) with mantissas X, S of 24 bits and m of five.  Then X 2^j - S (m 2^20 +- 1) is a whole number of at most 16, so S is
// within 16 of a multiple of 2^20.
__device__ __forceinline__ bool correction_decides(float scale)
{
    return ((__float_as_uint(scale) + 32u) & 0xFFFFFu) > 64u;
}

// The maximum of each of a half warp's four values over its lanes: the lane `sub` gets that of value sub / 4.
__device__ __forceinline__ float reduce_blocks(const float (&top)[4], uint32_t sub)
{
    const bool upper = (sub & 8u) != 0u;
    float a = upper ? top[2] : top[0], b = upper ? top[3] : top[1];
    a = fmaxf(a, __shfl_xor_sync(kFullMask, upper ? top[0] : top[2], 8));
    b = fmaxf(b, __shfl_xor_sync(kFullMask, upper ? top[1] : top[3], 8));
    const bool odd = (sub & 4u) != 0u;
    float c = odd ? b : a;
    c = fmaxf(c, __shfl_xor_sync(kFullMask, odd ? a : b, 4));
    c = fmaxf(c, __shfl_xor_sync(kFullMask, c, 2));
    return fmaxf(c, __shfl_xor_sync(kFullMask, c, 1));
}

// Large gated calls of bf16 rows keep eight blocks on an SM (64 registers; 16384 rows x 4096 82 us, with the seven of 71 registers 90).
template<typename T, bool kGate, int kSteps>
constexpr int kQuantizeBlocks = kGate && sizeof(T) == 2u && kSteps == 4 ? 8 : 0;

template<typename T, bool kGate, bool kVector, int kSteps>
__global__ void __launch_bounds__(kQuantizeThreads, kQuantizeBlocks<T, kGate, kSteps>) quantize_rows_kernel(const QuantizeArgs a)
{
    wait_for_previous_kernel();
    const uint32_t lane = threadIdx.x & 31u;
    const uint32_t half = lane >> 4, sub = lane & 15u;
    const uint32_t pieces = (a.columns + MOE_QUANTIZE_ITEM * kSteps - 1u) / (MOE_QUANTIZE_ITEM * kSteps);
    const uint64_t items = static_cast<uint64_t>(a.rows) * pieces;
    const uint64_t stride = static_cast<uint64_t>(gridDim.x) * (kQuantizeThreads / 32);
    for (uint64_t item = static_cast<uint64_t>(blockIdx.x) * (kQuantizeThreads / 32) + (threadIdx.x >> 5); item < items; item += stride)
    {
        const uint32_t row = static_cast<uint32_t>(item / pieces);
        const uint32_t first = static_cast<uint32_t>(item - static_cast<uint64_t>(row) * pieces) * (MOE_QUANTIZE_ITEM * kSteps);
        uint32_t source_row = row;
        bool valid = true;
        if (a.route_token != nullptr)
        {
            source_row = a.route_token[row];
            valid = source_row < a.source_rows;
            if (!valid && lane == 0)
                atomicOr(a.flags, MOE_EXPERT_FLAG_TOKEN_RANGE);
        }
        const T* source = static_cast<const T*>(a.source) + static_cast<size_t>(valid ? source_row : 0u) * a.row_stride;
        Eight<T> gate[kSteps];
        Eight<T> up[kGate ? kSteps : 1];
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
        {
            const uint32_t column = first + 256u * s + 128u * half + 8u * sub;
            const uint32_t count = valid && column < a.columns ? min(8u, a.columns - column) : 0u;
            gate[s].clear();
            if constexpr (kGate)
                up[s].clear();
            if (count == 0u)
                continue;
            if constexpr (kVector)
            {
                gate[s].load(source + column);
                if constexpr (kGate)
                    up[s].load(source + a.columns + column);
            }
            else
            {
                gate[s].load_scalars(source + column, count);
                if constexpr (kGate)
                    up[s].load_scalars(source + a.columns + column, count);
            }
        }
        grid_dependency_release(); // the next kernel may take its places on the SMs, behind these loads
        float x[kSteps][8];
        float top[kSteps];
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
        {
            gate[s].unpack(x[s]);
            if constexpr (kGate)
            {
                float y[8];
                up[s].unpack(y);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    x[s][i] = silu_gate(x[s][i], y[i]);
            }
            top[s] = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                top[s] = fmaxf(top[s], fabsf(x[s][i]));
        }
        // the block that this lane divides for: all of its half warp's lanes for the one, or four lanes for each of four
        static_assert(kSteps == 1 || kSteps == 4, "a lane divides for one block");
        float largest;
        if constexpr (kSteps == 4)
        {
            largest = reduce_blocks(top, sub);
        }
        else
        {
            largest = top[0];
#pragma unroll
            for (int offset = 8; offset > 0; offset >>= 1)
                largest = fmaxf(largest, __shfl_xor_sync(kFullMask, largest, offset));
        }
        constexpr uint32_t kSharers = 16u / kSteps;
        const float scale = __fdiv_rn(largest, kE4m3Max);
        {
            const uint32_t block_begin = first + 256u * (sub / kSharers) + 128u * half;
            if (sub % kSharers == 0u && block_begin < a.columns)
                a.scales[static_cast<size_t>(block_begin / MOE_EXPERT_BLOCK) * a.rows + row] = scale;
        }
        // A block of zeros, or one whose scale underflows, is divided by one: zeros, and NaN where there is one.
        const float divisor = scale == 0.0f ? 1.0f : scale;
        const float reciprocal = __frcp_rn(divisor);
        // Quotients round as the division's: ties in e4m3 are common among bf16 rows and hang on the last bit.  (In this range the
        // remainders are exact as above; a dividend too small for that gives a quotient far below e4m3's smallest.)
        const bool short_way = __all_sync(kFullMask, scale == 0.0f || (scale >= 0x1p-24f && scale < 0x1p25f && correction_decides(scale)));
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
        {
            const uint32_t column = first + 256u * s + 128u * half + 8u * sub;
            const float by = __shfl_sync(kFullMask, divisor, 16u * half + kSharers * s), inverse = __shfl_sync(kFullMask, reciprocal, 16u * half + kSharers * s);
            if (short_way)
            {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    x[s][i] = divide_once(x[s][i], by, inverse);
            }
            else
            {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    x[s][i] = __fdiv_rn(x[s][i], by);
            }
            if (column >= a.columns)
                continue;
            uint32_t packed[2];
            packed[0] = to_e4m3_pair(x[s][0], x[s][1]) | (to_e4m3_pair(x[s][2], x[s][3]) << 16);
            packed[1] = to_e4m3_pair(x[s][4], x[s][5]) | (to_e4m3_pair(x[s][6], x[s][7]) << 16);
            uint8_t* target = a.values + static_cast<size_t>(row) * a.columns + column;
            if constexpr (kVector)
                *reinterpret_cast<uint2*>(target) = make_uint2(packed[0], packed[1]);
            else
                for (uint32_t i = 0; i < min(8u, a.columns - column); ++i)
                    target[i] = static_cast<uint8_t>(packed[i >> 2] >> (8u * (i & 3u)));
        }
    }
}

// Rows that were quantised once, copied to every route that names them: a byte a value from L2 and to HBM.  A warp copies a row,
// 4 KiB in flight, and marks what it writes as not to be kept in L2, where the rows are that it reads (4096 rows x 4096 to 32768
// routes: both passes 35 us, 45 without the mark; the product behind it gains too, 132 -> 127 us for both calls).  The scales,
// which lie block by block, follow in a loop of their own.
constexpr int kSpreadThreads = 256;
__global__ void __launch_bounds__(kSpreadThreads) spread_rows_kernel(const QuantizeArgs a, const uint8_t* values, const float* scales)
{
    wait_for_previous_kernel();
    const uint32_t lane = threadIdx.x & 31u;
    const uint32_t warps = gridDim.x * (kSpreadThreads / 32);
    const uint32_t vectors = a.columns / 16u;
    for (uint32_t route = blockIdx.x * (kSpreadThreads / 32) + (threadIdx.x >> 5); route < a.rows; route += warps)
    {
        const uint32_t token = a.route_token[route];
        const bool valid = token < a.source_rows;
        if (!valid && lane == 0)
            atomicOr(a.flags, MOE_EXPERT_FLAG_TOKEN_RANGE);
        const uint4* source = reinterpret_cast<const uint4*>(values + static_cast<size_t>(valid ? token : 0u) * a.columns);
        uint4* target = reinterpret_cast<uint4*>(a.values + static_cast<size_t>(route) * a.columns);
        for (uint32_t first = lane; first < vectors; first += 256u)
        {
            uint4 part[8];
#pragma unroll
            for (uint32_t i = 0; i < 8u; ++i)
                part[i] = valid && first + 32u * i < vectors ? source[first + 32u * i] : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
            for (uint32_t i = 0; i < 8u; ++i)
                if (first + 32u * i < vectors)
                    __stcs(&target[first + 32u * i], part[i]);
        }
    }
    const uint32_t blocks = (a.columns + MOE_EXPERT_BLOCK - 1u) / MOE_EXPERT_BLOCK;
    const uint32_t threads = gridDim.x * kSpreadThreads;
    for (uint32_t route = blockIdx.x * kSpreadThreads + threadIdx.x; route < a.rows; route += threads)
    {
        const uint32_t token = a.route_token[route];
        const bool valid = token < a.source_rows;
#pragma unroll 8
        for (uint32_t block = 0; block < blocks; ++block)
            a.scales[static_cast<size_t>(block) * a.rows + route] = valid ? scales[static_cast<size_t>(block) * a.source_rows + token] : 0.0f;
    }
}

template<typename T, int kSteps>
cudaError_t launch_quantize_steps(const QuantizeArgs& a, bool gate, cudaStream_t stream)
{
    const bool vector = quantize_in_vectors(a, sizeof(T));
    const uint64_t items = static_cast<uint64_t>(a.rows) * ((a.columns + MOE_QUANTIZE_ITEM * kSteps - 1u) / (MOE_QUANTIZE_ITEM * kSteps));
    const uint64_t blocks = (items + kQuantizeThreads / 32 - 1) / (kQuantizeThreads / 32);
    const uint32_t grid = static_cast<uint32_t>(blocks < 148u * 16u ? blocks : 148u * 16u);
    auto kernel = gate ? (vector ? quantize_rows_kernel<T, true, true, kSteps> : quantize_rows_kernel<T, true, false, kSteps>)
                       : (vector ? quantize_rows_kernel<T, false, true, kSteps> : quantize_rows_kernel<T, false, false, kSteps>);
    return launch_following(kernel, grid, kQuantizeThreads, 0, stream, a);
}
template<typename T>
cudaError_t launch_quantize(const QuantizeArgs& a, bool gate, cudaStream_t stream)
{
    return quantize_steps(a, sizeof(T), gate) == 4u ? launch_quantize_steps<T, 4>(a, gate, stream) : launch_quantize_steps<T, 1>(a, gate, stream);
}

// ---- combine --------------------------------------------------------------------------
//
// A token's routes lie in the blocks of its experts.  HBM bound: every routed row is read once, every token written once.
// Many routes: one kernel notes for every (token, rank) the route that holds it, the next sums a token's rows with one CTA and
// leaves the notes at zero for the next call.  Few routes: each CTA looks through all of them for those of its token, which
// is cheaper than a second launch (128 tokens x 8 routes x 4096 3.8 against 4.9 us; 256 tokens x 4 5.5 against 4.8).  Either way
// a CTA first has the list of its token's routes and weights, ranks ascending, in shared memory; then a thread adds 16 bytes of
// up to eight rows at a time; rows are read once and marked so.  32768 bf16 rows x 4096 to 4096 tokens: 52 us (5.8 TB/s), without
// the mark 56.

constexpr int kCombineThreads = 256;
constexpr uint32_t kCombineFew = 1024;     // routes that every CTA looks through itself
constexpr uint32_t kCombineFewTokens = 128;
constexpr uint32_t kCombineFewRanks = 64;

__global__ void __launch_bounds__(256) combine_slots_kernel(const CombineArgs a)
{
    grid_dependency_release(); // the kernel that sums is on the SMs, waiting, when this one ends
    wait_for_previous_kernel();
    for (uint64_t i = static_cast<uint64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < a.route_count; i += static_cast<uint64_t>(gridDim.x) * blockDim.x)
    {
        const uint32_t token = a.route_token[i], rank = a.route_rank[i];
        if (token < a.token_count && rank < a.top_k)
            atomicMax(&a.slots[static_cast<size_t>(token) * a.top_k + rank], static_cast<uint32_t>(i) + 1u);
        else
            atomicOr(a.flags, MOE_EXPERT_FLAG_TOKEN_RANGE);
    }
}

__device__ __forceinline__ void narrow(float* target, const float (&x)[4])
{
    *reinterpret_cast<float4*>(target) = make_float4(x[0], x[1], x[2], x[3]);
}
__device__ __forceinline__ void narrow(__nv_bfloat16* target, const float (&x)[8])
{
    uint32_t words[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
    {
        const __nv_bfloat162 pair = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        memcpy(&words[i], &pair, 4);
    }
    *reinterpret_cast<uint4*>(target) = make_uint4(words[0], words[1], words[2], words[3]);
}
__device__ __forceinline__ void narrow(float* target, const float (&x)[1])
{
    *target = x[0];
}
__device__ __forceinline__ void narrow(__nv_bfloat16* target, const float (&x)[1])
{
    *target = __float2bfloat16_rn(x[0]);
}
// sum += weight * row
__device__ __forceinline__ void add_weighted(float (&sum)[4], const uint4& row, float weight)
{
    sum[0] = fmaf(weight, __uint_as_float(row.x), sum[0]);
    sum[1] = fmaf(weight, __uint_as_float(row.y), sum[1]);
    sum[2] = fmaf(weight, __uint_as_float(row.z), sum[2]);
    sum[3] = fmaf(weight, __uint_as_float(row.w), sum[3]);
}
__device__ __forceinline__ void add_weighted(float (&sum)[8], const uint4& row, float weight)
{
    const uint32_t words[4] = {row.x, row.y, row.z, row.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
    {
        sum[2 * i] = fmaf(weight, __uint_as_float(words[i] << 16), sum[2 * i]);
        sum[2 * i + 1] = fmaf(weight, __uint_as_float(words[i] & 0xFFFF0000u), sum[2 * i + 1]);
    }
}
__device__ __forceinline__ void add_weighted(float (&sum)[1], float row, float weight)
{
    sum[0] = fmaf(weight, row, sum[0]);
}
__device__ __forceinline__ void add_weighted(float (&sum)[1], __nv_bfloat16 row, float weight)
{
    sum[0] = fmaf(weight, __bfloat162float(row), sum[0]);
}

// Columns [begin, end) of a token: base plus the listed rows, in their order.  kWidth values of a thread at a time: 16 bytes, or
// one where a row does not start at a multiple of 16.
template<typename T, bool kVector>
__device__ __forceinline__ void sum_token(const CombineArgs& a, uint32_t token, const uint2* list, uint32_t count, uint32_t begin, uint32_t end)
{
    using Load = std::conditional_t<kVector, uint4, T>;
    constexpr uint32_t kWidth = kVector ? 16u / sizeof(T) : 1u;
    constexpr uint32_t kRows = 8; // in flight
    const T* rows = static_cast<const T*>(a.route_rows);
    for (uint32_t column = begin + threadIdx.x * kWidth; column < end; column += kCombineThreads * kWidth)
    {
        float sum[kWidth] = {};
        if (a.base != nullptr)
            add_weighted(sum, *reinterpret_cast<const Load*>(static_cast<const T*>(a.base) + static_cast<size_t>(token) * a.columns + column), 1.0f);
        for (uint32_t first = 0; first < count; first += kRows)
        {
            Load part[kRows];
#pragma unroll
            for (uint32_t i = 0; i < kRows; ++i)
                if (first + i < count)
                    part[i] = __ldcs(reinterpret_cast<const Load*>(rows + static_cast<size_t>(list[first + i].x) * a.row_stride + column));
#pragma unroll
            for (uint32_t i = 0; i < kRows; ++i)
                if (first + i < count)
                    add_weighted(sum, part[i], __uint_as_float(list[first + i].y));
        }
        narrow(static_cast<T*>(a.out) + static_cast<size_t>(token) * a.columns + column, sum);
    }
}

// Packs the routes noted in slots[0 .. top_k) (0: none), which may be global or shared memory, with their weights.  A note that is
// no route of the call is not followed.  One warp; returns their number.
__device__ __forceinline__ uint32_t list_routes(const CombineArgs& a, const uint32_t* slots, uint2* list)
{
    const uint32_t lane = threadIdx.x & 31u;
    uint32_t count = 0;
    for (uint32_t first = 0; first < a.top_k; first += 32u)
    {
        const uint32_t slot = first + lane < a.top_k ? slots[first + lane] : 0u;
        const bool noted = slot - 1u < a.route_count;
        const unsigned taken = __ballot_sync(kFullMask, noted);
        if (noted)
            list[count + __popc(taken & ((1u << lane) - 1u))] = make_uint2(slot - 1u, __float_as_uint(a.route_weight[slot - 1u]));
        count += __popc(taken);
    }
    return count;
}

template<typename T, bool kVector>
__global__ void __launch_bounds__(kCombineThreads) combine_routes_kernel(const CombineArgs a)
{
    extern __shared__ __align__(16) unsigned char shared_raw[];
    uint2* list = reinterpret_cast<uint2*>(shared_raw); // [top_k]
    __shared__ uint32_t count_shared;
    wait_for_previous_kernel();
    for (uint32_t token = blockIdx.x; token < a.token_count; token += gridDim.x)
    {
        uint32_t* slots = a.slots + static_cast<size_t>(token) * a.top_k;
        if (threadIdx.x < 32u)
        {
            const uint32_t count = list_routes(a, slots, list);
            if (threadIdx.x == 0)
                count_shared = count;
            __syncwarp();
            for (uint32_t rank = threadIdx.x; rank < a.top_k; rank += 32u)
                slots[rank] = 0u;
        }
        __syncthreads();
        sum_token<T, kVector>(a, token, list, count_shared, 0u, a.columns);
        __syncthreads();
    }
}

// A CTA for `piece` columns of a token; it looks through all routes.
template<typename T, bool kVector>
__global__ void __launch_bounds__(kCombineThreads) combine_few_kernel(const CombineArgs a, uint32_t pieces, uint32_t piece)
{
    __shared__ uint32_t slots[kCombineFewRanks];
    __shared__ uint2 list[kCombineFewRanks];
    __shared__ uint32_t count_shared;
    wait_for_previous_kernel();
    const uint32_t token = blockIdx.x / pieces;
    const uint32_t begin = (blockIdx.x - token * pieces) * piece;
    for (uint32_t rank = threadIdx.x; rank < a.top_k; rank += kCombineThreads)
        slots[rank] = 0u;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < a.route_count; i += kCombineThreads)
    {
        const uint32_t of = a.route_token[i], rank = a.route_rank[i];
        if (of == token && rank < a.top_k)
            atomicMax(&slots[rank], i + 1u);
        if (blockIdx.x == 0 && (of >= a.token_count || rank >= a.top_k))
            atomicOr(a.flags, MOE_EXPERT_FLAG_TOKEN_RANGE);
    }
    __syncthreads();
    if (threadIdx.x < 32u)
    {
        const uint32_t count = list_routes(a, slots, list);
        if (threadIdx.x == 0)
            count_shared = count;
    }
    __syncthreads();
    sum_token<T, kVector>(a, token, list, count_shared, begin, min(a.columns, begin + piece));
}

template<typename T>
cudaError_t launch_combine(const CombineArgs& a, cudaStream_t stream)
{
    constexpr uint32_t kWidth = 16u / sizeof(T);
    const uintptr_t bases = reinterpret_cast<uintptr_t>(a.route_rows) | reinterpret_cast<uintptr_t>(a.base) | reinterpret_cast<uintptr_t>(a.out);
    const bool vector = a.columns % kWidth == 0u && a.row_stride % kWidth == 0u && bases % 16u == 0u;
    if (combine_few(a.route_count, a.token_count, a.top_k))
    {
        // pieces of what a CTA's threads take at once, fewer when that gives more CTAs than are resident
        const uint32_t step = kCombineThreads * (vector ? kWidth : 1u);
        uint32_t pieces = (a.columns + step - 1u) / step;
        while (pieces > 1u && static_cast<uint64_t>(pieces) * a.token_count > 148u * 8u)
            pieces = (pieces + 1u) / 2u;
        const uint32_t piece = ((a.columns + pieces - 1u) / pieces + step - 1u) / step * step;
        auto kernel = vector ? combine_few_kernel<T, true> : combine_few_kernel<T, false>;
        return launch_following(kernel, pieces * a.token_count, kCombineThreads, 0, stream, a, pieces, piece);
    }
    const uint32_t blocks = (a.route_count + 255u) / 256u;
    if (blocks > 0u)
        if (cudaError_t status = launch_following(combine_slots_kernel, blocks < 592u ? blocks : 592u, 256u, 0, stream, a))
            return status;
    auto kernel = vector ? combine_routes_kernel<T, true> : combine_routes_kernel<T, false>;
    return launch_following(kernel, a.token_count < 148u * 8u ? a.token_count : 148u * 8u, kCombineThreads, sizeof(uint2) * a.top_k, stream, a);
}

} // namespace

cudaError_t launch_quantize_rows(const QuantizeArgs& args, int dtype, int activation, uint8_t* once, cudaStream_t stream)
{
    const bool gate = activation == MOE_ACTIVATION_SILU_GATE;
    if (once != nullptr)
    {
        // every source row once, then a copy for each route
        QuantizeArgs rows = args;
        rows.route_token = nullptr;
        rows.rows = args.source_rows;
        rows.values = once;
        rows.scales = reinterpret_cast<float*>(once + (static_cast<size_t>(args.source_rows) * args.columns + 15u) / 16u * 16u);
        const cudaError_t status = dtype == MOE_DTYPE_F32 ? launch_quantize<float>(rows, gate, stream) : launch_quantize<__nv_bfloat16>(rows, gate, stream);
        if (status != cudaSuccess)
            return status;
        const uint32_t blocks = (args.rows + kSpreadThreads / 32 - 1) / (kSpreadThreads / 32);
        return launch_following(spread_rows_kernel, blocks < 148u * 32u ? blocks : 148u * 32u, kSpreadThreads, 0, stream, args, rows.values, rows.scales);
    }
    return dtype == MOE_DTYPE_F32 ? launch_quantize<float>(args, gate, stream) : launch_quantize<__nv_bfloat16>(args, gate, stream);
}

bool combine_few(uint32_t route_count, uint32_t token_count, uint32_t top_k)
{
    return route_count <= kCombineFew && token_count <= kCombineFewTokens && top_k <= kCombineFewRanks;
}

cudaError_t launch_combine_routes(const CombineArgs& args, int dtype, cudaStream_t stream)
{
    return dtype == MOE_DTYPE_F32 ? launch_combine<float>(args, stream) : launch_combine<__nv_bfloat16>(args, stream);
}

} // namespace moe
