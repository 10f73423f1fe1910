// The experts' matrix products in e4m3 with a scale for each block of 128:
//   out[r, n] = sum_b scales[b, r] * weight_scales[e, n / 128, b] * sum_{k in b} values[r, k] * weights[e, n, k]

#include <cuda_fp8.h>

#include "moe_common.cuh"
#include "moe_internal.h"

namespace moe {

namespace {

constexpr uint32_t kTile = 64;
constexpr uint32_t kStep = 32; // columns of a step; a quarter of a scale's block

__device__ __forceinline__ float from_e4m3(uint8_t value)
{
    __nv_fp8_e4m3 x;
    x.__x = value;
    return static_cast<float>(x);
}

// One CTA per 64 outputs of one expert; it walks the expert's rows 64 at a time.
template<typename Out>
__global__ void __launch_bounds__(256) expert_product_kernel(const ProductArgs a)
{
    wait_for_previous_kernel();
    __shared__ float rows_shared[kStep][kTile + 1];
    __shared__ float weights_shared[kStep][kTile + 1];
    const uint32_t expert = blockIdx.y;
    const uint32_t blocks = (a.columns + MOE_EXPERT_BLOCK - 1u) / MOE_EXPERT_BLOCK;
    uint32_t begin = 0, end = a.rows;
    if (a.expert_offsets != nullptr)
    {
        bool good = true;
        for (uint32_t e = threadIdx.x; e < a.expert_count; e += blockDim.x)
            good = good && a.expert_offsets[e] <= a.expert_offsets[e + 1] && a.expert_offsets[e + 1] <= a.rows;
        if (!__syncthreads_and(good))
        {
            if (threadIdx.x == 0)
                atomicOr(a.flags, MOE_EXPERT_FLAG_OFFSETS);
            return;
        }
        begin = a.expert_offsets[expert];
        end = a.expert_offsets[expert + 1];
    }
    const uint32_t first_output = blockIdx.x * kTile;
    const uint8_t* weights = a.weights + static_cast<size_t>(expert) * a.outputs * a.columns;
    const uint32_t tx = threadIdx.x & 15u, ty = threadIdx.x >> 4;
    for (uint32_t first_row = begin; first_row < end; first_row += kTile)
    {
        float total[4][4] = {};
        float part[4][4] = {};
        for (uint32_t k = 0; k < a.columns; k += kStep)
        {
            for (uint32_t i = threadIdx.x; i < kTile * kStep; i += 256u)
            {
                const uint32_t c = i % kStep, r = i / kStep;
                const bool column_ok = k + c < a.columns;
                rows_shared[c][r] = column_ok && first_row + r < end ? from_e4m3(a.values[static_cast<size_t>(first_row + r) * a.columns + k + c]) : 0.0f;
                weights_shared[c][r] = column_ok && first_output + r < a.outputs ? from_e4m3(weights[static_cast<size_t>(first_output + r) * a.columns + k + c]) : 0.0f;
            }
            __syncthreads();
            for (uint32_t c = 0; c < kStep; ++c)
            {
                float x[4], w[4];
                for (int i = 0; i < 4; ++i)
                {
                    x[i] = rows_shared[c][ty * 4 + i];
                    w[i] = weights_shared[c][tx * 4 + i];
                }
                for (int i = 0; i < 4; ++i)
                    for (int j = 0; j < 4; ++j)
                        part[i][j] = fmaf(x[i], w[j], part[i][j]);
            }
            __syncthreads();
            if ((k + kStep) % MOE_EXPERT_BLOCK == 0u || k + kStep >= a.columns)
            {
                const uint32_t block = k / MOE_EXPERT_BLOCK;
                const float weight_scale =
                    a.weight_scales[(static_cast<size_t>(expert) * ((a.outputs + MOE_EXPERT_BLOCK - 1u) / MOE_EXPERT_BLOCK) + first_output / MOE_EXPERT_BLOCK) * blocks + block];
                for (int i = 0; i < 4; ++i)
                {
                    const uint32_t row = first_row + ty * 4 + i;
                    const float scale = row < end ? a.scales[static_cast<size_t>(block) * a.rows + row] * weight_scale : 0.0f;
                    for (int j = 0; j < 4; ++j)
                    {
                        total[i][j] = fmaf(part[i][j], scale, total[i][j]);
                        part[i][j] = 0.0f;
                    }
                }
            }
        }
        for (int i = 0; i < 4; ++i)
        {
            const uint32_t row = first_row + ty * 4 + i;
            for (int j = 0; j < 4; ++j)
            {
                const uint32_t output = first_output + tx * 4 + j;
                if (row < end && output < a.outputs)
                {
                    Out* target = static_cast<Out*>(a.out) + static_cast<size_t>(row) * a.out_stride + output;
                    if constexpr (sizeof(Out) == 4)
                        *target = total[i][j];
                    else
                        *target = __float2bfloat16_rn(total[i][j]);
                }
            }
        }
    }
}

} // namespace

cudaError_t launch_expert_product(const ProductArgs& args, int out_dtype, cudaStream_t stream)
{
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((args.outputs + kTile - 1u) / kTile, args.expert_count, 1);
    config.blockDim = dim3(256, 1, 1);
    config.stream = stream;
    cudaLaunchAttribute attribute = follow_closely();
    config.attrs = &attribute;
    config.numAttrs = 1;
    return out_dtype == MOE_DTYPE_F32 ? cudaLaunchKernelEx(&config, expert_product_kernel<float>, args)
                                      : cudaLaunchKernelEx(&config, expert_product_kernel<__nv_bfloat16>, args);
}

} // namespace moe
