// Host-only check of the scratch that captured graphs may hold (grow_kept of ncnn-moe-runtime_b200/csrc/moe_internal.h): it does
// not grow inside a capture, it is published behind its clearing alone, and what it replaces is kept.  The runtime calls are
// replaced by the fakes below; no CUDA library is linked and no memory of a device is touched.
#include <cstdio>
#include <string>

#include "../../ncnn-moe-runtime_b200/csrc/moe_internal.h"

static std::string calls;              // m allocated, c cleared, f freed, e error taken back
static bool capturing = false;
static bool refuse_clearing = false;
static size_t most_bytes = ~size_t(0); // an allocation beyond it fails
static cudaError_t query_status = cudaSuccess;
static size_t allocated_bytes = 0, cleared_bytes = 0;
static size_t next_address = 0x1000;

extern "C" cudaError_t CUDARTAPI cudaStreamIsCapturing(cudaStream_t, cudaStreamCaptureStatus* status)
{
    *status = capturing ? cudaStreamCaptureStatusActive : cudaStreamCaptureStatusNone;
    return query_status;
}
extern "C" cudaError_t CUDARTAPI cudaMalloc(void** pointer, size_t bytes)
{
    calls += 'm';
    if (bytes > most_bytes)
        return cudaErrorMemoryAllocation;
    allocated_bytes = bytes;
    *pointer = reinterpret_cast<void*>(next_address += 0x1000);
    return cudaSuccess;
}
extern "C" cudaError_t CUDARTAPI cudaMemsetAsync(void*, int value, size_t bytes, cudaStream_t)
{
    calls += 'c';
    cleared_bytes = value == 0 ? bytes : 0;
    return refuse_clearing ? cudaErrorInvalidValue : cudaSuccess;
}
extern "C" cudaError_t CUDARTAPI cudaFree(void*)
{
    calls += 'f';
    return cudaSuccess;
}
extern "C" cudaError_t CUDARTAPI cudaGetLastError()
{
    calls += 'e';
    return cudaSuccess;
}

static int failures = 0;
#define EXPECT(condition)                                       \
    do                                                          \
    {                                                           \
        if (!(condition))                                       \
        {                                                       \
            std::printf("line %d: %s (%s)\n", __LINE__, #condition, calls.c_str()); \
            ++failures;                                         \
        }                                                       \
    } while (0)

int main()
{
    std::vector<void*> kept;
    uint32_t* pointer = nullptr;
    size_t capacity = 0;
    const auto grow = [&](size_t wanted, bool cleared) {
        calls.clear();
        return moe::grow_kept(kept, pointer, capacity, wanted, nullptr, cleared);
    };
    EXPECT(grow(0, true) == cudaSuccess && calls.empty() && pointer == nullptr);

    // nothing is allocated, recorded or published inside a capture
    capturing = true;
    EXPECT(grow(100, true) == cudaErrorStreamCaptureUnsupported && calls.empty() && pointer == nullptr && capacity == 0);
    EXPECT(grow(100, false) == cudaErrorStreamCaptureUnsupported && calls.empty() && capacity == 0);
    capturing = false;
    query_status = cudaErrorStreamCaptureImplicit; // the legacy stream while another one captures
    EXPECT(grow(100, true) == cudaErrorStreamCaptureImplicit && calls.empty() && capacity == 0);
    query_status = cudaSuccess;

    // a clearing that was refused: the next call starts again
    refuse_clearing = true;
    EXPECT(grow(100, true) == cudaErrorInvalidValue && calls == "mcf" && pointer == nullptr && capacity == 0);
    refuse_clearing = false;
    EXPECT(grow(100, true) == cudaSuccess && calls == "mc" && pointer != nullptr && capacity == 100 && allocated_bytes == 400 && cleared_bytes == 400);
    uint32_t* const first = pointer;

    // enough is there, inside a capture too
    capturing = true;
    EXPECT(grow(100, true) == cudaSuccess && calls.empty() && pointer == first);
    EXPECT(grow(101, true) == cudaErrorStreamCaptureUnsupported && calls.empty() && pointer == first && capacity == 100);
    capturing = false;

    // a clearing that was refused leaves what was there
    refuse_clearing = true;
    EXPECT(grow(101, true) == cudaErrorInvalidValue && calls == "mcf" && pointer == first && capacity == 100 && kept.empty());
    refuse_clearing = false;

    // at least doubled, all of it cleared, and the old one kept
    EXPECT(grow(101, true) == cudaSuccess && capacity == 200 && cleared_bytes == 800 && pointer != first && kept.size() == 1 && kept[0] == first);

    // without memory for twice as much: what is wanted, or an error that the next launch of the caller does not meet again
    most_bytes = 4 * 250;
    EXPECT(grow(250, false) == cudaSuccess && calls == "mm" && capacity == 250 && kept.size() == 2);
    uint32_t* const last = pointer;
    EXPECT(grow(251, true) == cudaErrorMemoryAllocation && calls == "mme" && capacity == 250 && pointer == last && kept.size() == 2);
    if (failures == 0)
        std::puts("kept scratch ok");
    return failures == 0 ? 0 : 1;
}
