// Host-only check of how the quantisation divides its work (quantize_steps of ncnn-moe-runtime_b200/csrc/moe_internal.h): rows that leave
// most of a wide item empty, and small calls, take the narrow one.  No CUDA call is made; the pointers are never followed.
#include <cstdio>

#include "../../ncnn-moe-runtime_b200/csrc/moe_internal.h"

static int failures = 0;

static void expect(uint32_t steps, uint32_t rows, uint32_t columns, size_t element, bool gate, size_t source = 256)
{
    const size_t stride = static_cast<size_t>(columns) * (gate ? 2u : 1u);
    const moe::QuantizeArgs args = {reinterpret_cast<void*>(source), rows, rows, columns, stride, nullptr, reinterpret_cast<uint8_t*>(256), reinterpret_cast<float*>(64), nullptr};
    const uint32_t got = moe::quantize_steps(args, element, gate);
    if (got != steps)
    {
        std::printf("%u rows x %u, %zu bytes, gate %d: %u steps\n", rows, columns, element, gate, got);
        ++failures;
    }
}

int main()
{
    for (size_t element : {2u, 4u})
        for (bool gate : {false, true})
        {
            for (uint32_t columns : {1u, 128u, 256u, 512u})
                expect(1, 1u << 26 >> 9, columns, element, gate); // short rows, however many
            expect(4, 8192, 4096, element, gate);
            expect(4, 11650, 2880, element, gate);
            expect(1, 128, 2880, element, gate);
            expect(1, 1, 4096, element, gate);
            expect(1, 1536, 4095, element, gate);           // not in vectors
            expect(1, 1536, 4096, element, gate, 258);
            expect(4, 8194, 4095, element, gate);
            expect(4, 0x7FFFFFFFu, 0x7FFFFFFFu - 1023u, element, gate); // no product wraps
        }
    expect(1, 768, 4096, 2, false);
    expect(4, 1024, 4096, 2, false);
    expect(1, 18724, 1792, 2, false);
    expect(4, 5825, 5760, 2, false);
    expect(4, 18724, 1792, 2, true);
    expect(1, 1024, 4096, 2, true);
    expect(4, 1300, 4096, 2, true);
    expect(4, 32513, 1032, 4, false);
    expect(1, 32513, 1032, 2, false);
    expect(1, 2048, 4096, 4, true);
    return failures == 0 ? 0 : 1;
}
