// Rows to 8-bit blocks before the experts' products, and the routed rows back to
// their tokens behind them.

#include <cuda_fp8.h>

#include "moe_common.cuh"
#include "moe_internal.h"

namespace moe {

namespace {

// ---- eight values of a row as floats ----------------------------------------------

template<typename T>
__device__ __forceinline__ float widen(T value);
template<>
__device__ __forceinline__ float widen<float>(float value)
{
    return value;
}
template<>
__device__ __forceinline__ float widen<__nv_bfloat16>(__nv_bfloat16 value)
{
    return __bfloat162float(value);
}

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
// scale = max |x| / 448 over a block of 128 columns, value = e4m3(x / scale): memory bound (the rows in, a byte a value
// out).  Sixteen lanes own a block, eight values each, so that a bf16 row is read in 16-byte vectors; a warp takes 1024
// columns of a row and has all their loads in flight before the first maximum.

constexpr int kQuantizeThreads = 256;
constexpr int kQuantizeSteps = 4;                               // blocks of 128 a half warp takes from one item
constexpr uint32_t kQuantizeItem = 256u * kQuantizeSteps;       // columns of an item
constexpr float kE4m3Max = 448.0f;

__device__ __forceinline__ uint32_t to_e4m3_pair(float low, float high)
{
    return __nv_cvt_float2_to_fp8x2(make_float2(low, high), __NV_SATFINITE, __NV_E4M3);
}

__device__ __forceinline__ float silu_gate(float gate, float up)
{
    return __fmul_rn(__fdiv_rn(gate, 1.0f + expf(-gate)), up);
}

template<typename T, bool kGate, bool kVector>
__global__ void __launch_bounds__(kQuantizeThreads) quantize_rows_kernel(const QuantizeArgs a)
{
    wait_for_previous_kernel();
    const uint32_t lane = threadIdx.x & 31u;
    const uint32_t half = lane >> 4, sub = lane & 15u;
    const uint32_t pieces = (a.columns + kQuantizeItem - 1u) / kQuantizeItem;
    const uint64_t items = static_cast<uint64_t>(a.rows) * pieces;
    const uint64_t stride = static_cast<uint64_t>(gridDim.x) * (kQuantizeThreads / 32);
    for (uint64_t item = static_cast<uint64_t>(blockIdx.x) * (kQuantizeThreads / 32) + (threadIdx.x >> 5); item < items; item += stride)
    {
        const uint32_t row = static_cast<uint32_t>(item / pieces);
        const uint32_t first = static_cast<uint32_t>(item - static_cast<uint64_t>(row) * pieces) * kQuantizeItem;
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
        Eight<T> gate[kQuantizeSteps];
        Eight<T> up[kGate ? kQuantizeSteps : 1];
#pragma unroll
        for (int s = 0; s < kQuantizeSteps; ++s)
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
#pragma unroll
        for (int s = 0; s < kQuantizeSteps; ++s)
        {
            const uint32_t block_begin = first + 256u * s + 128u * half;
            const uint32_t column = block_begin + 8u * sub;
            float x[8];
            gate[s].unpack(x);
            if constexpr (kGate)
            {
                float y[8];
                up[s].unpack(y);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    x[i] = silu_gate(x[i], y[i]);
            }
            float top = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                top = fmaxf(top, fabsf(x[i]));
#pragma unroll
            for (int offset = 8; offset > 0; offset >>= 1)
                top = fmaxf(top, __shfl_xor_sync(kFullMask, top, offset));
            const float scale = __fdiv_rn(top, kE4m3Max);
            // A block of zeros, or one whose scale underflows, converts as it is: zeros, and NaN where there is one.
            // Quotients are the division's: ties in e4m3 are common among bf16 rows and hang on the last bit.  divide_by
            // needs a fifth of its instructions; a dividend below its range gives a quotient far below e4m3's smallest.
            if (scale >= 0x1p-24f && scale < 0x1p25f)
            {
                const float reciprocal = __frcp_rn(scale);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    x[i] = divide_by(x[i], scale, reciprocal);
            }
            else if (scale > 0.0f)
            {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    x[i] = __fdiv_rn(x[i], scale);
            }
            if (block_begin >= a.columns)
                continue;
            if (sub == 0u)
                a.scales[static_cast<size_t>(block_begin / MOE_EXPERT_BLOCK) * a.rows + row] = scale;
            if (column >= a.columns)
                continue;
            uint32_t packed[2];
            packed[0] = to_e4m3_pair(x[0], x[1]) | (to_e4m3_pair(x[2], x[3]) << 16);
            packed[1] = to_e4m3_pair(x[4], x[5]) | (to_e4m3_pair(x[6], x[7]) << 16);
            uint8_t* target = a.values + static_cast<size_t>(row) * a.columns + column;
            if constexpr (kVector)
                *reinterpret_cast<uint2*>(target) = make_uint2(packed[0], packed[1]);
            else
                for (uint32_t i = 0; i < min(8u, a.columns - column); ++i)
                    target[i] = static_cast<uint8_t>(packed[i >> 2] >> (8u * (i & 3u)));
        }
    }
}

template<typename T>
cudaError_t launch_quantize(const QuantizeArgs& a, bool gate, cudaStream_t stream)
{
    const uintptr_t bases = reinterpret_cast<uintptr_t>(a.source);
    const bool vector = a.columns % 8u == 0u && bases % 16u == 0u && a.row_stride * sizeof(T) % 16u == 0u && reinterpret_cast<uintptr_t>(a.values) % 8u == 0u;
    const uint64_t items = static_cast<uint64_t>(a.rows) * ((a.columns + kQuantizeItem - 1u) / kQuantizeItem);
    const uint64_t blocks = (items + kQuantizeThreads / 32 - 1) / (kQuantizeThreads / 32);
    const uint32_t grid = static_cast<uint32_t>(blocks < 148u * 8u ? blocks : 148u * 8u);
    auto kernel = gate ? (vector ? quantize_rows_kernel<T, true, true> : quantize_rows_kernel<T, true, false>)
                       : (vector ? quantize_rows_kernel<T, false, true> : quantize_rows_kernel<T, false, false>);
    return launch_following(kernel, grid, kQuantizeThreads, 0, stream, a);
}

// ---- combine --------------------------------------------------------------------------
//
// A token's routes lie in the blocks of its experts.  The first kernel notes for every (token, rank) the route that holds
// it, the second sums a token's rows with one CTA, ranks ascending, and leaves the notes at zero for the next call.

constexpr int kCombineThreads = 256;

__global__ void __launch_bounds__(256) combine_slots_kernel(const CombineArgs a)
{
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

template<typename T>
__device__ __forceinline__ void store_narrow(T* target, float value);
template<>
__device__ __forceinline__ void store_narrow<float>(float* target, float value)
{
    *target = value;
}
template<>
__device__ __forceinline__ void store_narrow<__nv_bfloat16>(__nv_bfloat16* target, float value)
{
    *target = __float2bfloat16_rn(value);
}

template<typename T>
__global__ void __launch_bounds__(kCombineThreads) combine_routes_kernel(const CombineArgs a)
{
    wait_for_previous_kernel();
    for (uint32_t token = blockIdx.x; token < a.token_count; token += gridDim.x)
    {
        uint32_t* slots = a.slots + static_cast<size_t>(token) * a.top_k;
        for (uint32_t column = threadIdx.x; column < a.columns; column += kCombineThreads)
        {
            float sum = a.base != nullptr ? widen(static_cast<const T*>(a.base)[static_cast<size_t>(token) * a.columns + column]) : 0.0f;
            for (uint32_t rank = 0; rank < a.top_k; ++rank)
            {
                const uint32_t slot = slots[rank];
                if (slot != 0u)
                    sum = fmaf(a.route_weight[slot - 1u], widen(static_cast<const T*>(a.route_rows)[static_cast<size_t>(slot - 1u) * a.row_stride + column]), sum);
            }
            store_narrow(static_cast<T*>(a.out) + static_cast<size_t>(token) * a.columns + column, sum);
        }
        __syncthreads();
        for (uint32_t rank = threadIdx.x; rank < a.top_k; rank += kCombineThreads)
            slots[rank] = 0u;
    }
}

} // namespace

cudaError_t launch_quantize_rows(const QuantizeArgs& args, int dtype, int activation, cudaStream_t stream)
{
    const bool gate = activation == MOE_ACTIVATION_SILU_GATE;
    return dtype == MOE_DTYPE_F32 ? launch_quantize<float>(args, gate, stream) : launch_quantize<__nv_bfloat16>(args, gate, stream);
}

cudaError_t launch_combine_routes(const CombineArgs& args, int dtype, cudaStream_t stream)
{
    if (args.route_count > 0)
    {
        const uint64_t blocks = (static_cast<uint64_t>(args.route_count) + 255u) / 256u;
        if (cudaError_t status = launch_following(combine_slots_kernel, static_cast<uint32_t>(blocks < 592u ? blocks : 592u), 256u, 0, stream, args))
            return status;
    }
    const uint32_t grid = args.token_count < 148u * 8u ? args.token_count : 148u * 8u;
    return dtype == MOE_DTYPE_F32 ? launch_following(combine_routes_kernel<float>, grid, kCombineThreads, 0, stream, args)
                                  : launch_following(combine_routes_kernel<__nv_bfloat16>, grid, kCombineThreads, 0, stream, args);
}

} // namespace moe
