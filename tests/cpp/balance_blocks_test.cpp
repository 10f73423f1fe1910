// Host-only check of the balance kernels' grids (balance_blocks of ncnn-moe-runtime_b200/csrc/moe_internal.h): up to the largest
// token count there is a block for every token, or as many as there may be.  No CUDA call is made.
#include <cstdio>

#include "../../ncnn-moe-runtime_b200/csrc/moe_internal.h"

int main()
{
    int failures = 0;
    for (uint32_t warps : {4u, 16u})
        for (uint32_t most : {148u, MOE_BALANCE_MAX_BLOCKS})
            for (uint32_t tokens : {1u, 3u, 4u, 5u, 16u, 17u, 2368u, 4737u, 65536u, 0x7FFFFFFFu, 0xFFFFFFF0u, 0xFFFFFFF1u, 0xFFFFFFFFu})
            {
                const uint32_t blocks = moe::balance_blocks(tokens, warps, most);
                const bool all = static_cast<uint64_t>(blocks) * warps >= tokens && (blocks == 1u || static_cast<uint64_t>(blocks - 1u) * warps < tokens);
                if (blocks == 0u || blocks > most || (!all && blocks != most))
                {
                    std::printf("%u tokens, %u warps, %u at most: %u\n", tokens, warps, most, blocks);
                    ++failures;
                }
            }
    return failures == 0 ? 0 : 1;
}
