// Balance of the experts: tokens per expert, mean router probabilities, the balance
// loss and its gradient with respect to the router logits.
//
// p_e = s_e / S, S = sum of the scores s over the experts (softmax: S = 1 after the usual shift by the maximum).
// L = coefficient * sum_e f_e P_e with f_e = E c_e / (k n), P_e = sum_t p_te / n.  With g_e = coefficient f_e / n:
//   softmax                 dL/dx_e = p_e (g_e - sum_j g_j p_j)
//   sigmoid, sqrt-softplus  dL/dx_e = s'(x_e) / S (g_e - sum_j g_j p_j)
// The p sum to one, so a constant may be taken off every g without changing the difference.  g_e is built from the
// integer E c_e - sum_j c_j: for experts that are nearly balanced the difference of the plain terms would lose its leading
// digits.

#include "moe_common.cuh"
#include "moe_internal.h"

namespace moe {

namespace {

constexpr int kBalanceThreads = 256;
constexpr int kBalanceWarps = kBalanceThreads / 32;

__device__ __forceinline__ float warp_sum(float v)
{
#pragma unroll
    for (int offset = 16; offset > 0; offset >>= 1)
        v += __shfl_xor_sync(kFullMask, v, offset);
    return v;
}
__device__ __forceinline__ float warp_max(float v)
{
#pragma unroll
    for (int offset = 16; offset > 0; offset >>= 1)
        v = fmaxf(v, __shfl_xor_sync(kFullMask, v, offset));
    return v;
}

// 1 / (1 + exp(-x)) without overflow, and 1 minus it without cancellation.
__device__ __forceinline__ void sigmoid_both(float x, float& value, float& rest)
{
    const float t = expf(-fabsf(x));
    const float large = __fdiv_rn(1.0f, 1.0f + t);
    const float small = t * large;
    value = x >= 0.0f ? large : small;
    rest = x >= 0.0f ? small : large;
    if (x != x)
        value = rest = x;
}
// sqrt(log(1 + exp(x))); far below zero it is exp(x / 2), and its derivative half of that
__device__ __forceinline__ float sqrt_softplus(float x)
{
    if (x < -20.0f)
        return expf(0.5f * x);
    return __fsqrt_rn(fmaxf(x, 0.0f) + log1pf(expf(-fabsf(x))));
}

__device__ __forceinline__ float score_of(float x, int function)
{
    if (function == MOE_ROUTER_SQRT_SOFTPLUS)
        return sqrt_softplus(x);
    float value, rest;
    sigmoid_both(x, value, rest);
    return value;
}
__device__ __forceinline__ float score_slope(float x, float score, int function)
{
    if (function == MOE_ROUTER_SQRT_SOFTPLUS && x < -20.0f)
        return 0.5f * score;
    float value, rest;
    sigmoid_both(x, value, rest);
    return function == MOE_ROUTER_SQRT_SOFTPLUS ? __fdiv_rn(value, 2.0f * score) : value * rest;
}

// Writes a token's scores to `row` and returns the factor that makes them sum to one (0 when they are all zero).  One warp.
__device__ __forceinline__ float score_row(const float* logits, uint32_t experts, int function, float* row)
{
    const uint32_t lane = threadIdx.x & 31u;
    float peak = 0.0f;
    if (function == MOE_ROUTER_SOFTMAX)
    {
        peak = -INFINITY;
        for (uint32_t e = lane; e < experts; e += 32u)
            peak = fmaxf(peak, logits[e]);
        peak = warp_max(peak);
    }
    float total = 0.0f;
    for (uint32_t e = lane; e < experts; e += 32u)
    {
        const float score = function == MOE_ROUTER_SOFTMAX ? expf(logits[e] - peak) : score_of(logits[e], function);
        row[e] = score;
        total += score;
    }
    total = warp_sum(total);
    return total == 0.0f ? 0.0f : __fdiv_rn(1.0f, total);
}

// Sums over a block's tokens: [block][expert] probabilities and counted routes, [block] counted tokens.
__global__ void __launch_bounds__(kBalanceThreads) balance_partial_kernel(const BalanceArgs a)
{
    wait_for_previous_kernel();
    extern __shared__ __align__(16) unsigned char shared_raw[];
    const uint32_t experts = a.expert_count;
    const uint32_t warps = blockDim.x / 32u;
    float* rows = reinterpret_cast<float*>(shared_raw);        // [warps][experts]
    float* sums = rows + static_cast<size_t>(warps) * experts; // [warps][experts]
    uint32_t* routed = reinterpret_cast<uint32_t*>(sums + static_cast<size_t>(warps) * experts); // [experts]
    uint32_t* offsets = routed + experts;                                                        // [experts + 1]
    __shared__ uint32_t counted;
    if (threadIdx.x == 0)
        counted = 0u;
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const uint64_t most_routes = static_cast<uint64_t>(a.token_count) * a.top_k;
    bool good = true;
    for (uint32_t e = threadIdx.x; e <= experts; e += blockDim.x)
    {
        const uint32_t offset = a.expert_offsets[e];
        offsets[e] = offset;
        good = good && offset <= most_routes && (e == 0u || a.expert_offsets[e - 1u] <= offset);
    }
    for (uint32_t e = threadIdx.x; e < experts; e += blockDim.x)
        routed[e] = 0u;
    good = __syncthreads_and(good) != 0;
    if (!good && threadIdx.x == 0)
        atomicOr(a.flags, MOE_EXPERT_FLAG_OFFSETS);

    // routes of counted tokens by expert: whole numbers, so the order of the atomics does not matter
    if (good)
    {
        for (uint64_t route = offsets[0] + static_cast<uint64_t>(blockIdx.x) * blockDim.x + threadIdx.x; route < offsets[experts];
             route += static_cast<uint64_t>(gridDim.x) * blockDim.x)
        {
            const uint32_t token = a.route_token[route];
            if (token >= a.token_count)
            {
                atomicOr(a.flags, MOE_EXPERT_FLAG_TOKEN_RANGE);
                continue;
            }
            if (a.token_mask != nullptr && a.token_mask[token] == 0)
                continue;
            uint32_t low = 0, high = experts; // the last expert whose range begins at or before the route
            while (high - low > 1u)
            {
                const uint32_t middle = (low + high) / 2u;
                if (offsets[middle] <= route)
                    low = middle;
                else
                    high = middle;
            }
            atomicAdd(&routed[low], 1u);
        }
    }

    float* row = rows + static_cast<size_t>(warp) * experts;
    float* sum = sums + static_cast<size_t>(warp) * experts;
    for (uint32_t e = lane; e < experts; e += 32u)
        sum[e] = 0.0f;
    uint32_t mine = 0;
    for (uint64_t token = static_cast<uint64_t>(blockIdx.x) * warps + warp; token < a.token_count; token += static_cast<uint64_t>(gridDim.x) * warps)
    {
        if (a.token_mask != nullptr && a.token_mask[token] == 0)
            continue;
        ++mine;
        const float factor = score_row(a.logits + token * experts, experts, a.score_function, row);
        for (uint32_t e = lane; e < experts; e += 32u)
            sum[e] += row[e] * factor;
    }
    if (lane == 0)
        atomicAdd(&counted, mine);
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < experts; e += blockDim.x)
    {
        float total = 0.0f;
        for (uint32_t w = 0; w < warps; ++w)
            total += sums[static_cast<size_t>(w) * experts + e];
        a.partial_sums[static_cast<size_t>(blockIdx.x) * experts + e] = total;
        a.partial_counts[static_cast<size_t>(blockIdx.x) * (experts + 1u) + e] = routed[e];
    }
    if (threadIdx.x == 0)
        a.partial_counts[static_cast<size_t>(blockIdx.x) * (experts + 1u) + experts] = counted;
}

// The blocks' sums in block order, then the loss.
__global__ void __launch_bounds__(1024) balance_reduce_kernel(const BalanceArgs a, uint32_t blocks)
{
    wait_for_previous_kernel();
    const uint32_t experts = a.expert_count;
    __shared__ uint32_t counted_shared;
    __shared__ float warp_totals[32];
    if (threadIdx.x == 0)
    {
        uint32_t counted = 0;
        for (uint32_t b = 0; b < blocks; ++b)
            counted += a.partial_counts[static_cast<size_t>(b) * (experts + 1u) + experts];
        counted_shared = counted;
        a.expert_tokens[experts] = counted;
    }
    __syncthreads();
    const float tokens = static_cast<float>(max(counted_shared, 1u));
    float weighted = 0.0f;
    for (uint32_t e = threadIdx.x; e < experts; e += blockDim.x)
    {
        float sum = 0.0f;
        uint32_t count = 0;
        for (uint32_t b = 0; b < blocks; ++b)
        {
            sum += a.partial_sums[static_cast<size_t>(b) * experts + e];
            count += a.partial_counts[static_cast<size_t>(b) * (experts + 1u) + e];
        }
        const float probability = __fdiv_rn(sum, tokens);
        a.expert_tokens[e] = count;
        a.expert_probability[e] = probability;
        weighted += static_cast<float>(count) * probability;
    }
    weighted = warp_sum(weighted);
    if ((threadIdx.x & 31u) == 0u)
        warp_totals[threadIdx.x >> 5] = weighted;
    __syncthreads();
    if (threadIdx.x < 32u)
    {
        const float total = warp_sum(warp_totals[threadIdx.x]);
        if (threadIdx.x == 0)
            *a.loss = a.coefficient * (total * __fdiv_rn(static_cast<float>(experts), static_cast<float>(a.top_k) * tokens));
    }
}

__global__ void __launch_bounds__(kBalanceThreads) balance_backward_kernel(const BalanceArgs a, const uint32_t* expert_tokens, const float* loss_gradient, float* gradient)
{
    wait_for_previous_kernel();
    extern __shared__ __align__(16) unsigned char shared_raw[];
    const uint32_t experts = a.expert_count;
    const uint32_t warps = blockDim.x / 32u;
    float* shares = reinterpret_cast<float*>(shared_raw); // [experts]: g
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    float* row = shares + static_cast<size_t>(warp + 1u) * experts;
    __shared__ unsigned long long routes_shared;
    if (threadIdx.x == 0)
        routes_shared = 0ull;
    __syncthreads();
    unsigned long long mine = 0;
    for (uint32_t e = threadIdx.x; e < experts; e += blockDim.x)
        mine += expert_tokens[e];
    atomicAdd(&routes_shared, mine);
    __syncthreads();
    const double counted = static_cast<double>(max(expert_tokens[experts], 1u));
    const double unit = static_cast<double>(a.coefficient) * (loss_gradient != nullptr ? static_cast<double>(*loss_gradient) : 1.0) / (static_cast<double>(a.top_k) * counted * counted);
    for (uint32_t e = threadIdx.x; e < experts; e += blockDim.x)
        shares[e] = static_cast<float>(unit * static_cast<double>(static_cast<long long>(experts) * static_cast<long long>(expert_tokens[e]) - static_cast<long long>(routes_shared)));
    __syncthreads();
    for (uint64_t token = static_cast<uint64_t>(blockIdx.x) * warps + warp; token < a.token_count; token += static_cast<uint64_t>(gridDim.x) * warps)
    {
        float* target = gradient + token * experts;
        if (a.token_mask != nullptr && a.token_mask[token] == 0)
        {
            for (uint32_t e = lane; e < experts; e += 32u)
                target[e] = 0.0f;
            continue;
        }
        const float* logits = a.logits + token * experts;
        const float factor = score_row(logits, experts, a.score_function, row);
        float mean = 0.0f;
        for (uint32_t e = lane; e < experts; e += 32u)
            mean += shares[e] * (row[e] * factor);
        mean = warp_sum(mean);
        for (uint32_t e = lane; e < experts; e += 32u)
        {
            const float slope = a.score_function == MOE_ROUTER_SOFTMAX ? row[e] : score_slope(logits[e], row[e], a.score_function);
            target[e] = factor == 0.0f ? 0.0f : slope * factor * (shares[e] - mean);
        }
    }
}

uint32_t warps_for(uint32_t experts)
{
    return experts <= 1024u ? kBalanceWarps : kBalanceWarps / 2;
}

} // namespace

uint32_t balance_blocks(uint32_t token_count, uint32_t experts)
{
    const uint32_t wanted = (token_count + warps_for(experts) - 1u) / warps_for(experts);
    return wanted < MOE_BALANCE_MAX_BLOCKS ? (wanted > 0u ? wanted : 1u) : MOE_BALANCE_MAX_BLOCKS;
}

cudaError_t launch_balance_loss(const BalanceArgs& args, cudaStream_t stream)
{
    const uint32_t blocks = balance_blocks(args.token_count, args.expert_count);
    const uint32_t warps = warps_for(args.expert_count);
    const size_t shared_bytes = sizeof(float) * (2u * warps + 2u) * args.expert_count + sizeof(uint32_t);
    static SharedOptIn opt_in;
    if (shared_bytes > 48u * 1024u)
        if (cudaError_t status = opt_in_shared(opt_in, balance_partial_kernel, shared_bytes))
            return status;
    if (cudaError_t status = launch_following(balance_partial_kernel, blocks, warps * 32u, shared_bytes, stream, args))
        return status;
    return launch_following(balance_reduce_kernel, 1u, 1024u, 0, stream, args, blocks);
}

cudaError_t launch_balance_loss_backward(const BalanceArgs& args, const uint32_t* expert_tokens, const float* loss_gradient, float* gradient, cudaStream_t stream)
{
    const uint32_t blocks = balance_blocks(args.token_count, args.expert_count);
    const uint32_t warps = warps_for(args.expert_count);
    const size_t shared_bytes = sizeof(float) * (warps + 1u) * args.expert_count;
    static SharedOptIn opt_in;
    if (shared_bytes > 48u * 1024u)
        if (cudaError_t status = opt_in_shared(opt_in, balance_backward_kernel, shared_bytes))
            return status;
    return launch_following(balance_backward_kernel, blocks, warps * 32u, shared_bytes, stream, args, expert_tokens, loss_gradient, gradient);
}

} // namespace moe
