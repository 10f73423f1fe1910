// The bounded waits of the expert products (ncnn-moe-runtime_b200/csrc/moe_tensor.cuh) on barriers that nobody arrives at.
#include "../../ncnn-moe-runtime_b200/csrc/moe_tensor.cuh"

namespace {

// results: what a thread's wait said that ran out after `limit` looks, the CTA's mark behind it, what a warp's wait with 64 times
// the limit said, which the mark ends, what a warp's wait said that ran out itself, its mark, and two waits for a barrier that is complete
__global__ void wait_in_vain(uint32_t limit, int* results)
{
    __shared__ __align__(8) unsigned long long barriers[2];
    __shared__ volatile uint32_t stalled, other;
    const uint32_t never = static_cast<uint32_t>(__cvta_generic_to_shared(&barriers[0])), done = static_cast<uint32_t>(__cvta_generic_to_shared(&barriers[1]));
    if (threadIdx.x == 0)
    {
        moe::barrier_init(never, 1u);
        moe::barrier_init(done, 1u);
        moe::barrier_init_fence();
        stalled = other = 0u;
        moe::barrier_arrive(done);
    }
    __syncthreads();
    if (threadIdx.x == 0)
        results[0] = moe::barrier_wait(never, 0u, &stalled, limit);
    if (threadIdx.x >= 32u)
    {
        const bool said = moe::barrier_wait_warp(never, 0u, &stalled, 64u * limit);
        if (threadIdx.x == 32u)
            results[2] = said;
    }
    __syncthreads();
    if (threadIdx.x < 32u)
    {
        const bool said = moe::barrier_wait_warp(never, 0u, &other, limit);
        const bool completed = moe::barrier_wait_warp(done, 0u, &other, limit);
        if (threadIdx.x == 0)
        {
            results[1] = static_cast<int>(stalled);
            results[3] = said;
            results[4] = static_cast<int>(other);
            results[5] = completed;
            results[6] = moe::barrier_wait(done, 0u, &other, limit);
        }
    }
}

} // namespace

// results: seven host ints; microseconds: how long the kernel took.
extern "C" int test_waits(uint32_t limit, int* results, float* microseconds)
{
    int* device = nullptr;
    cudaEvent_t begin, end;
    cudaError_t status = cudaMalloc(reinterpret_cast<void**>(&device), 7 * sizeof(int));
    if (status != cudaSuccess)
        return status;
    cudaEventCreate(&begin);
    cudaEventCreate(&end);
    status = cudaMemset(device, 0xFF, 7 * sizeof(int));
    if (status == cudaSuccess)
    {
        cudaEventRecord(begin);
        wait_in_vain<<<1, 64>>>(limit, device);
        cudaEventRecord(end);
        status = cudaMemcpy(results, device, 7 * sizeof(int), cudaMemcpyDeviceToHost);
    }
    if (status == cudaSuccess)
        status = cudaEventElapsedTime(microseconds, begin, end);
    *microseconds *= 1000.0f;
    cudaEventDestroy(begin);
    cudaEventDestroy(end);
    cudaFree(device);
    return status;
}
