// Host-only check of functions that are looked up at run time (found_once of ncnn-moe-runtime_b200/csrc/moe_internal.h): a look-up
// that failed is made again by the next call.  No CUDA call is made.
#include <cstdio>

#include "../../ncnn-moe-runtime_b200/csrc/moe_internal.h"

static int answer(int x)
{
    return x + 1;
}

int main()
{
    using Function = int (*)(int);
    std::atomic<Function> found{nullptr};
    int asked = 0;
    const auto failing = [&]() -> Function { ++asked; return nullptr; };
    const auto answering = [&]() -> Function { ++asked; return answer; };
    bool good = moe::found_once(found, failing) == nullptr && asked == 1;
    good = good && moe::found_once(found, failing) == nullptr && asked == 2;
    good = good && moe::found_once(found, answering) == answer && asked == 3;
    good = good && moe::found_once(found, failing) == answer && asked == 3; // remembered
    std::puts(good ? "look-up ok" : "look-up: a failure was remembered, or a success was not");
    return good ? 0 : 1;
}
