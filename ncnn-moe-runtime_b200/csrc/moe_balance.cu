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
//
// A warp takes a token: 65536 x 256 with softmax 24 us for the loss, about five of them for its second launch, and 24 us for the
// gradient (5.6 TB/s).  Bound by instruction issue (71 % of the slots): exponentials, and sums across lanes.

#include "moe_common.cuh"
#include "moe_internal.h"

namespace moe {

namespace {

constexpr uint32_t kRegisterExperts = 1024; // up to here a lane holds a row's scores in registers
// Threads of a block by the scores a lane holds; rows in shared memory (kPer 0) need 8 bytes a warp and expert.
template<int kPer>
constexpr int kThreadsFor = kPer == 0 ? 128 : 512;
// One wave of blocks: with twice as many, the second half waits for registers (32768 x 512, loss 22.9 against 25.6 us, gradient
// 25.8 against 28.2; with half as many 65536 x 256 24.4 and 26.9, 24.1 and 29.3).  Rows in shared memory: as many as the scratch of
// the loss has room for (8192 x 2000 73 us, half as many 128); the gradient has none.
template<int kPer>
constexpr uint32_t kMostBlocks = kPer >= 16 ? 148u : MOE_BALANCE_MAX_BLOCKS;
template<int kPer>
constexpr uint32_t kMostBackwardBlocks = kPer == 0 ? 148u * 16u : kMostBlocks<kPer>;

__device__ __forceinline__ float warp_sum(float v)
{
#pragma unroll
    for (int offset = 16; offset > 0; offset >>= 1)
        v += __shfl_xor_sync(kFullMask, v, offset);
    return v;
}
// two sums side by side
__device__ __forceinline__ void warp_sum_both(float& v, float& w)
{
#pragma unroll
    for (int offset = 16; offset > 0; offset >>= 1)
    {
        v += __shfl_xor_sync(kFullMask, v, offset);
        w += __shfl_xor_sync(kFullMask, w, offset);
    }
}
__device__ __forceinline__ float warp_max(float v)
{
#pragma unroll
    for (int offset = 16; offset > 0; offset >>= 1)
        v = fmaxf(v, __shfl_xor_sync(kFullMask, v, offset));
    return v;
}

// 1 / x within a unit in the last place; 0 from 2^126 on
__device__ __forceinline__ float reciprocal(float x)
{
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// sqrt(log(1 + exp(x))); far below zero it is exp(x / 2), and its derivative half of that
__device__ __forceinline__ float sqrt_softplus(float x)
{
    if (x < -20.0f)
        return expf(0.5f * x);
    return __fsqrt_rn(fmaxf(x, 0.0f) + log1pf(expf(-fabsf(x))));
}

// A score.  Softmax: exp(x - peak).  A sigmoid below 2^-126 is 0 here; tokens with no larger one are taken again (tiny_scores).
template<int kFunction>
__device__ __forceinline__ float score_of(float x, float peak)
{
    if constexpr (kFunction == MOE_ROUTER_SOFTMAX)
        return expf(x - peak);
    else if constexpr (kFunction == MOE_ROUTER_SIGMOID)
        return reciprocal(1.0f + expf(-x));
    else
        return sqrt_softplus(x);
}
// A score and its derivative: softmax the score itself (the rest of the formula is the same for all), sigmoid s (1 - s), the
// smaller of the two factors without cancellation, sqrt-softplus sigmoid / (2 s).
template<int kFunction>
__device__ __forceinline__ void slope_of(float x, float peak, float& score, float& slope)
{
    if constexpr (kFunction == MOE_ROUTER_SOFTMAX)
    {
        score = slope = expf(x - peak);
    }
    else
    {
        const float t = expf(-fabsf(x));
        const float large = reciprocal(1.0f + t), small = t * large;
        if constexpr (kFunction == MOE_ROUTER_SIGMOID)
        {
            score = x >= 0.0f ? large : small;
            slope = large * small;
        }
        else
        {
            score = sqrt_softplus(x);
            slope = x < -20.0f ? 0.5f * score : __fdividef(x >= 0.0f ? large : small, 2.0f * score); // score in [2^-15, 2^64]
        }
    }
}

__device__ __forceinline__ bool token_counts(const BalanceArgs& a, uint64_t token)
{
    return a.token_mask == nullptr || a.token_mask[token] != 0;
}
// A lane's part of a token's logits: every 32nd.  The next token's are on their way while one is worked on (65536 x 256,
// gradient, 24.1 against 26.1 us; 32768 x 512 25.8 against 34.4).  kFull: 32 * kPer experts, so that every lane has kPer of them.
template<int kPer, bool kFull>
struct LaneRow
{
    float x[kPer];
    bool counts;

    __device__ __forceinline__ void load(const BalanceArgs& a, uint64_t token, uint32_t lane)
    {
        const bool there = token < a.token_count;
        const float* logits = a.logits + (there ? token : 0u) * a.expert_count;
        counts = there && token_counts(a, token);
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            x[i] = kFull ? logits[lane + 32u * i] : there && lane + 32u * i < a.expert_count ? logits[lane + 32u * i] : 0.0f;
    }
};

// Scores that sum to less than this are tiny for all experts: sigmoid is exp(x) there, sqrt-softplus exp(x / 2), to all digits.
// They may be subnormal or lost and the reciprocal of their sum infinite, so such a token is taken again relative to its largest
// logit, as softmax is, unless its scores are zeros in fp32.
constexpr float kTinyScores = 0x1p-60f;
template<int kFunction>
__device__ __forceinline__ bool tiny_scores(float total)
{
    return kFunction != MOE_ROUTER_SOFTMAX && total < kTinyScores;
}
template<int kFunction>
__device__ __forceinline__ float tiny_score(float x, float peak)
{
    return expf((kFunction == MOE_ROUTER_SQRT_SOFTPLUS ? 0.5f : 1.0f) * (x - peak));
}
template<int kFunction>
__device__ __forceinline__ bool zero_scores(float peak)
{
    return tiny_score<kFunction>(peak, 0.0f) == 0.0f;
}
// a tiny score's derivative over the score
template<int kFunction>
constexpr float kTinySlope = kFunction == MOE_ROUTER_SQRT_SOFTPLUS ? 0.5f : 1.0f;
// the largest of a token's logits; a warp
__device__ __forceinline__ float largest_logit(const float* logits, uint32_t experts)
{
    float peak = -INFINITY;
    for (uint32_t e = threadIdx.x & 31u; e < experts; e += 32u)
        peak = fmaxf(peak, logits[e]);
    return warp_max(peak);
}

// ---- forward ------------------------------------------------------------------------------

// Routes of counted tokens by expert, this block's share of them: whole numbers, so the order of the atomics does not matter.
// offsets, routed: shared.  All threads; ends with a barrier before the offsets are read, not behind the counts.
__device__ __forceinline__ void count_routes(const BalanceArgs& a, uint32_t* offsets, uint32_t* routed)
{
    const uint32_t experts = a.expert_count;
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
    if (!good)
    {
        if (threadIdx.x == 0)
            atomicOr(a.flags, MOE_EXPERT_FLAG_OFFSETS);
        return;
    }
    // a warp has 32 routes in a row, which mostly belong to one expert: one addition for all of them
    const uint32_t lane = threadIdx.x & 31u;
    const uint64_t stride = static_cast<uint64_t>(gridDim.x) * blockDim.x;
    const uint64_t end = offsets[experts];
    for (uint64_t base = offsets[0] + static_cast<uint64_t>(blockIdx.x) * blockDim.x + (threadIdx.x & ~31u); base < end; base += stride)
    {
        const uint64_t route = base + lane;
        const uint32_t token = route < end ? a.route_token[route] : 0u;
        bool valid = route < end && token < a.token_count;
        if (route < end && !valid)
            atomicOr(a.flags, MOE_EXPERT_FLAG_TOKEN_RANGE);
        valid = valid && token_counts(a, token);
        uint32_t low = 0, high = experts; // the last expert whose range begins at or before the route
        while (high - low > 1u)
        {
            const uint32_t middle = (low + high) / 2u;
            if (offsets[middle] <= route)
                low = middle;
            else
                high = middle;
        }
        const uint32_t expert = __shfl_sync(kFullMask, low, 0);
        const unsigned votes = __ballot_sync(kFullMask, valid);
        if (__all_sync(kFullMask, low == expert || !valid))
        {
            if (lane == 0)
                atomicAdd(&routed[expert], static_cast<uint32_t>(__popc(votes)));
        }
        else if (valid)
        {
            atomicAdd(&routed[low], 1u);
        }
    }
}

// The loss from every expert's sum and count; all threads of a block, expert e by the threads that hold it.
struct LossParts
{
    uint32_t counted;
    float weighted; // this thread's share of sum c_e P_e
};
__device__ __forceinline__ void store_expert(const BalanceArgs& a, LossParts& parts, uint32_t expert, float sum, uint32_t count)
{
    const float probability = __fdiv_rn(sum, static_cast<float>(max(parts.counted, 1u)));
    a.expert_tokens[expert] = count;
    a.expert_probability[expert] = probability;
    parts.weighted += static_cast<float>(count) * probability;
}
__device__ __forceinline__ void store_loss(const BalanceArgs& a, const LossParts& parts)
{
    __shared__ float warp_totals[32];
    const float weighted = warp_sum(parts.weighted);
    if ((threadIdx.x & 31u) == 0u)
        warp_totals[threadIdx.x >> 5] = weighted;
    __syncthreads();
    if (threadIdx.x < 32u)
    {
        const float total = warp_sum(threadIdx.x < blockDim.x / 32u ? warp_totals[threadIdx.x] : 0.0f);
        if (threadIdx.x == 0)
        {
            const float tokens = static_cast<float>(max(parts.counted, 1u));
            *a.loss = a.coefficient * (total * __fdiv_rn(static_cast<float>(a.expert_count), static_cast<float>(a.top_k) * tokens));
            a.expert_tokens[a.expert_count] = parts.counted;
        }
    }
}

// Sums over a block's tokens.  A warp per token: a lane has every 32nd expert, the scores and their sums over the tokens in
// registers (kPer of each; kPer 0: in shared memory).  The blocks' sums go to scratch, or, where one block has all tokens,
// straight into the results.
template<int kFunction, int kPer, bool kFull>
__global__ void __launch_bounds__(kThreadsFor<kPer>) balance_partial_kernel(const BalanceArgs a)
{
    extern __shared__ __align__(16) unsigned char shared_raw[];
    const uint32_t experts = a.expert_count;
    const uint32_t warps = blockDim.x / 32u;
    uint32_t* offsets = reinterpret_cast<uint32_t*>(shared_raw); // [experts + 1]
    uint32_t* routed = offsets + experts + 1u;                   // [experts]
    float* sums = reinterpret_cast<float*>(routed + experts);    // [warps][experts]
    __shared__ uint32_t counted_shared;
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    if (threadIdx.x == 0)
        counted_shared = 0u;
    wait_for_previous_kernel();
    const uint64_t first = static_cast<uint64_t>(blockIdx.x) * warps + warp, stride = static_cast<uint64_t>(gridDim.x) * warps;
    LaneRow<kPer == 0 ? 1 : kPer, kFull> next;
    if constexpr (kPer > 0)
        next.load(a, first, lane);
    count_routes(a, offsets, routed);

    uint32_t counted = 0;
    float* const sum_row = sums + static_cast<size_t>(warp) * experts;
    if constexpr (kPer > 0)
    {
        float sum[kPer];
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            sum[i] = 0.0f;
        for (uint64_t token = first; token < a.token_count; token += stride)
        {
            const LaneRow<kPer, kFull> row = next;
            next.load(a, token + stride, lane);
            if (!row.counts)
                continue;
            ++counted;
            float x[kPer];
            float peak = -INFINITY;
            if constexpr (kFunction == MOE_ROUTER_SOFTMAX)
            {
#pragma unroll
                for (int i = 0; i < kPer; ++i)
                    if (kFull || lane + 32u * i < experts)
                        peak = fmaxf(peak, row.x[i]);
                peak = warp_max(peak);
            }
            float total = 0.0f;
#pragma unroll
            for (int i = 0; i < kPer; ++i)
            {
                x[i] = score_of<kFunction>(row.x[i], peak);
                if (!kFull && lane + 32u * i >= experts)
                    x[i] = 0.0f;
                total += x[i];
            }
            total = warp_sum(total);
            if (tiny_scores<kFunction>(total))
            {
                const float* logits = a.logits + token * experts;
                peak = largest_logit(logits, experts);
                total = 0.0f;
#pragma unroll
                for (int i = 0; i < kPer; ++i)
                {
                    x[i] = lane + 32u * i < experts && !zero_scores<kFunction>(peak) ? tiny_score<kFunction>(logits[lane + 32u * i], peak) : 0.0f;
                    total += x[i];
                }
                total = warp_sum(total);
            }
            const float factor = total == 0.0f ? 0.0f : reciprocal(total);
#pragma unroll
            for (int i = 0; i < kPer; ++i)
                sum[i] = fmaf(x[i], factor, sum[i]);
        }
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            if (lane + 32u * i < experts)
                sum_row[lane + 32u * i] = sum[i];
    }
    else
    {
        float* const row = sums + static_cast<size_t>(warps + warp) * experts; // [warps][experts] behind the sums
        for (uint32_t e = lane; e < experts; e += 32u)
            sum_row[e] = 0.0f;
        for (uint64_t token = first; token < a.token_count; token += stride)
        {
            if (!token_counts(a, token))
                continue;
            ++counted;
            const float* logits = a.logits + token * experts;
            float peak = kFunction == MOE_ROUTER_SOFTMAX ? largest_logit(logits, experts) : 0.0f;
            float total = 0.0f;
            for (uint32_t e = lane; e < experts; e += 32u)
            {
                row[e] = score_of<kFunction>(logits[e], peak);
                total += row[e];
            }
            total = warp_sum(total);
            if (tiny_scores<kFunction>(total))
            {
                peak = largest_logit(logits, experts);
                total = 0.0f;
                for (uint32_t e = lane; e < experts; e += 32u)
                {
                    row[e] = zero_scores<kFunction>(peak) ? 0.0f : tiny_score<kFunction>(logits[e], peak);
                    total += row[e];
                }
                total = warp_sum(total);
            }
            const float factor = total == 0.0f ? 0.0f : reciprocal(total);
            for (uint32_t e = lane; e < experts; e += 32u)
                sum_row[e] = fmaf(row[e], factor, sum_row[e]);
        }
    }
    if (lane == 0 && counted > 0u)
        atomicAdd(&counted_shared, counted);
    __syncthreads();
    LossParts parts = {counted_shared, 0.0f};
    const bool alone = gridDim.x == 1u;
    for (uint32_t e = threadIdx.x; e < experts; e += blockDim.x)
    {
        float total = 0.0f;
        for (uint32_t w = 0; w < warps; ++w)
            total += sums[static_cast<size_t>(w) * experts + e];
        if (alone)
        {
            store_expert(a, parts, e, total, routed[e]);
        }
        else
        {
            a.partial_sums[static_cast<size_t>(blockIdx.x) * experts + e] = total;
            a.partial_counts[static_cast<size_t>(blockIdx.x) * (experts + 1u) + e] = routed[e];
        }
    }
    if (alone)
        store_loss(a, parts);
    else if (threadIdx.x == 0)
        a.partial_counts[static_cast<size_t>(blockIdx.x) * (experts + 1u) + experts] = parts.counted;
}

// The blocks' sums, 32 experts a CTA: a warp adds every 32nd block, then the warps' sums are added in their order.  The CTA that
// finishes last adds the loss from all experts, in their order.
__global__ void __launch_bounds__(1024) balance_reduce_kernel(const BalanceArgs a, uint32_t blocks)
{
    __shared__ float sums[32][33];
    __shared__ uint32_t routes[32][33];
    __shared__ uint32_t counted_shared, last_shared;
    const uint32_t experts = a.expert_count;
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const uint32_t e = blockIdx.x * 32u + lane;
    if (threadIdx.x == 0)
        counted_shared = 0u;
    wait_for_previous_kernel();
    __syncthreads();
    if (threadIdx.x < blocks)
        atomicAdd(&counted_shared, a.partial_counts[static_cast<size_t>(threadIdx.x) * (experts + 1u) + experts]);
    float sum = 0.0f;
    uint32_t count = 0;
#pragma unroll 10
    for (uint32_t b = warp; b < blocks; b += 32u)
    {
        sum += e < experts ? a.partial_sums[static_cast<size_t>(b) * experts + e] : 0.0f;
        count += e < experts ? a.partial_counts[static_cast<size_t>(b) * (experts + 1u) + e] : 0u;
    }
    sums[warp][lane] = sum;
    routes[warp][lane] = count;
    __syncthreads();
    LossParts parts = {counted_shared, 0.0f};
    if (warp == 0u)
    {
        if (e < experts)
        {
            float total = 0.0f;
            uint32_t all = 0;
            for (uint32_t w = 0; w < 32u; ++w)
            {
                total += sums[w][lane];
                all += routes[w][lane];
            }
            store_expert(a, parts, e, total, all);
        }
        const float weighted = warp_sum(parts.weighted);
        if (lane == 0)
        {
            a.partial_loss[blockIdx.x] = weighted;
            __threadfence();
            last_shared = atomicAdd(a.reduce_done, 1u) == gridDim.x - 1u ? 1u : 0u;
        }
    }
    __syncthreads();
    if (last_shared == 0u)
        return;
    __threadfence();
    parts.weighted = threadIdx.x < gridDim.x ? a.partial_loss[threadIdx.x] : 0.0f;
    if (threadIdx.x == 0)
        *a.reduce_done = 0u;
    store_loss(a, parts);
}

// ---- backward -----------------------------------------------------------------------------

template<int kFunction, int kPer, bool kFull>
__global__ void __launch_bounds__(kThreadsFor<kPer>) balance_backward_kernel(const BalanceArgs a, const uint32_t* expert_tokens, const float* loss_gradient, float* gradient)
{
    extern __shared__ __align__(16) unsigned char shared_raw[];
    const uint32_t experts = a.expert_count;
    const uint32_t warps = blockDim.x / 32u;
    float* shares = reinterpret_cast<float*>(shared_raw); // [experts]: g, without a constant that does not matter
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    __shared__ unsigned long long routes_shared;
    if (threadIdx.x == 0)
        routes_shared = 0ull;
    wait_for_previous_kernel();
    __syncthreads();
    unsigned long long mine = 0;
    for (uint32_t e = threadIdx.x; e < experts; e += blockDim.x)
        mine += expert_tokens[e];
#pragma unroll
    for (int offset = 16; offset > 0; offset >>= 1)
        mine += __shfl_xor_sync(kFullMask, mine, offset);
    if (lane == 0)
        atomicAdd(&routes_shared, mine);
    __syncthreads();
    const double counted = static_cast<double>(max(expert_tokens[experts], 1u));
    const double unit = static_cast<double>(a.coefficient) * (loss_gradient != nullptr ? static_cast<double>(*loss_gradient) : 1.0) / (static_cast<double>(a.top_k) * counted * counted);
    for (uint32_t e = threadIdx.x; e < experts; e += blockDim.x)
        shares[e] = static_cast<float>(unit * static_cast<double>(static_cast<long long>(experts) * static_cast<long long>(expert_tokens[e]) - static_cast<long long>(routes_shared)));
    __syncthreads();
    const uint64_t first = static_cast<uint64_t>(blockIdx.x) * warps + warp, stride = static_cast<uint64_t>(gridDim.x) * warps;
    if constexpr (kPer > 0)
    {
        LaneRow<kPer, kFull> next;
        next.load(a, first, lane);
        float share[kPer];
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            share[i] = kFull || lane + 32u * i < experts ? shares[lane + 32u * i] : 0.0f;
        for (uint64_t token = first; token < a.token_count; token += stride)
        {
            const LaneRow<kPer, kFull> row = next;
            next.load(a, token + stride, lane);
            float* target = gradient + token * experts;
            float slope[kPer];
            if (!row.counts)
            {
#pragma unroll
                for (int i = 0; i < kPer; ++i)
                    if (kFull || lane + 32u * i < experts)
                        target[lane + 32u * i] = 0.0f;
                continue;
            }
            float peak = -INFINITY;
            if constexpr (kFunction == MOE_ROUTER_SOFTMAX)
            {
#pragma unroll
                for (int i = 0; i < kPer; ++i)
                    if (kFull || lane + 32u * i < experts)
                        peak = fmaxf(peak, row.x[i]);
                peak = warp_max(peak);
            }
            float total = 0.0f, mean = 0.0f;
#pragma unroll
            for (int i = 0; i < kPer; ++i)
            {
                float score;
                slope_of<kFunction>(row.x[i], peak, score, slope[i]);
                if (!kFull && lane + 32u * i >= experts)
                    score = 0.0f;
                total += score;
                mean = fmaf(share[i], score, mean);
            }
            warp_sum_both(total, mean);
            if (tiny_scores<kFunction>(total))
            {
                const float* logits = a.logits + token * experts;
                peak = largest_logit(logits, experts);
                total = mean = 0.0f;
#pragma unroll
                for (int i = 0; i < kPer; ++i)
                {
                    const float score = lane + 32u * i < experts && !zero_scores<kFunction>(peak) ? tiny_score<kFunction>(logits[lane + 32u * i], peak) : 0.0f;
                    slope[i] = kTinySlope<kFunction> * score;
                    total += score;
                    mean = fmaf(share[i], score, mean);
                }
                warp_sum_both(total, mean);
            }
            const float factor = total == 0.0f ? 0.0f : reciprocal(total);
            mean *= factor;
#pragma unroll
            for (int i = 0; i < kPer; ++i)
                if (kFull || lane + 32u * i < experts)
                    target[lane + 32u * i] = slope[i] * factor * (share[i] - mean);
        }
    }
    else
    {
        for (uint64_t token = first; token < a.token_count; token += stride)
        {
            float* target = gradient + token * experts;
            if (!token_counts(a, token))
            {
                for (uint32_t e = lane; e < experts; e += 32u)
                    target[e] = 0.0f;
                continue;
            }
            const float* logits = a.logits + token * experts;
            float peak = kFunction == MOE_ROUTER_SOFTMAX ? largest_logit(logits, experts) : 0.0f;
            float total = 0.0f, mean = 0.0f;
            for (uint32_t e = lane; e < experts; e += 32u)
            {
                const float score = score_of<kFunction>(logits[e], peak);
                total += score;
                mean = fmaf(shares[e], score, mean);
            }
            warp_sum_both(total, mean);
            const bool tiny = tiny_scores<kFunction>(total);
            if (tiny)
            {
                peak = largest_logit(logits, experts);
                total = mean = 0.0f;
                for (uint32_t e = lane; e < experts; e += 32u)
                {
                    const float score = zero_scores<kFunction>(peak) ? 0.0f : tiny_score<kFunction>(logits[e], peak);
                    total += score;
                    mean = fmaf(shares[e], score, mean);
                }
                warp_sum_both(total, mean);
            }
            const float factor = total == 0.0f ? 0.0f : reciprocal(total);
            mean *= factor;
            for (uint32_t e = lane; e < experts; e += 32u)
            {
                float score, slope;
                slope_of<kFunction>(logits[e], peak, score, slope);
                if (tiny)
                    slope = zero_scores<kFunction>(peak) ? 0.0f : kTinySlope<kFunction> * tiny_score<kFunction>(logits[e], peak);
                target[e] = slope * factor * (shares[e] - mean);
            }
        }
    }
}

// ---- launches -----------------------------------------------------------------------------

template<int kFunction, int kPer, bool kFull>
cudaError_t launch_forward(const BalanceArgs& a, cudaStream_t stream)
{
    constexpr uint32_t warps = kThreadsFor<kPer> / 32;
    // one block alone (and no second launch) for up to four tokens a warp: 64 x 256 5.0 against 7.1 us, 128 x 256 7.7 against 7.2
    const uint32_t blocks = a.token_count <= 4u * warps ? 1u : balance_blocks(a.token_count, warps, kMostBlocks<kPer>);
    const size_t shared_bytes = sizeof(uint32_t) * (2u * a.expert_count + 1u) + sizeof(float) * (kPer > 0 ? 1u : 2u) * warps * a.expert_count;
    static SharedOptIn opt_in;
    if (shared_bytes > 48u * 1024u)
        if (cudaError_t status = opt_in_shared(opt_in, balance_partial_kernel<kFunction, kPer, kFull>, shared_bytes))
            return status;
    if (cudaError_t status = launch_following(balance_partial_kernel<kFunction, kPer, kFull>, blocks, warps * 32u, shared_bytes, stream, a))
        return status;
    return blocks == 1u ? cudaSuccess : launch_following(balance_reduce_kernel, (a.expert_count + 31u) / 32u, 1024u, 0, stream, a, blocks);
}

struct BackwardArgs
{
    const uint32_t* expert_tokens;
    const float* loss_gradient;
    float* gradient;
};
template<int kFunction, int kPer, bool kFull>
cudaError_t launch_backward(const BalanceArgs& a, const BackwardArgs& b, cudaStream_t stream)
{
    constexpr uint32_t warps = kThreadsFor<kPer> / 32;
    return launch_following(balance_backward_kernel<kFunction, kPer, kFull>, balance_blocks(a.token_count, warps, kMostBackwardBlocks<kPer>), warps * 32u, sizeof(float) * a.expert_count, stream, a,
                            b.expert_tokens, b.loss_gradient, b.gradient);
}

template<int kFunction, int kPer, bool kFull>
cudaError_t launch(const BalanceArgs& a, const BackwardArgs* b, cudaStream_t stream)
{
    return b != nullptr ? launch_backward<kFunction, kPer, kFull>(a, *b, stream) : launch_forward<kFunction, kPer, kFull>(a, stream);
}
// Experts that fill their lanes need no predicates (65536 x 256 softmax, loss 24.0 against 27.1
// us; 32768 x 1024 38.7 against 45.0).
template<int kFunction, int kPer>
cudaError_t launch(const BalanceArgs& a, const BackwardArgs* b, cudaStream_t stream)
{
    return a.expert_count == 32u * kPer ? launch<kFunction, kPer, true>(a, b, stream) : launch<kFunction, kPer, false>(a, b, stream);
}
template<int kFunction>
cudaError_t launch_for_experts(const BalanceArgs& a, const BackwardArgs* b, cudaStream_t stream)
{
    if (a.expert_count <= 64u)
        return launch<kFunction, 2>(a, b, stream);
    if (a.expert_count <= 128u)
        return launch<kFunction, 4>(a, b, stream);
    if (a.expert_count <= 256u)
        return launch<kFunction, 8>(a, b, stream);
    if (a.expert_count <= 512u)
        return launch<kFunction, 16>(a, b, stream);
    if (a.expert_count <= kRegisterExperts)
        return launch<kFunction, 32>(a, b, stream);
    return launch<kFunction, 0, false>(a, b, stream);
}
cudaError_t launch_balance(const BalanceArgs& a, const BackwardArgs* b, cudaStream_t stream)
{
    switch (a.score_function)
    {
    case MOE_ROUTER_SOFTMAX: return launch_for_experts<MOE_ROUTER_SOFTMAX>(a, b, stream);
    case MOE_ROUTER_SIGMOID: return launch_for_experts<MOE_ROUTER_SIGMOID>(a, b, stream);
    default: return launch_for_experts<MOE_ROUTER_SQRT_SOFTPLUS>(a, b, stream);
    }
}

} // namespace

cudaError_t launch_balance_loss(const BalanceArgs& args, cudaStream_t stream)
{
    return launch_balance(args, nullptr, stream);
}

cudaError_t launch_balance_loss_backward(const BalanceArgs& args, const uint32_t* expert_tokens, const float* loss_gradient, float* gradient, cudaStream_t stream)
{
    const BackwardArgs backward = {expert_tokens, loss_gradient, gradient};
    return launch_balance(args, &backward, stream);
}

} // namespace moe
