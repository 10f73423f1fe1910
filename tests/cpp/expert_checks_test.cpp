// Host-only checks of the arguments of the expert products, the combine and the balance loss
// (ncnn-moe-runtime_b200/csrc/moe_internal.h): what is refused, and that what is documented passes.  No CUDA call is made;
// the pointers are numbers that are never followed.
#include <cmath>
#include <cstdio>

#include "../../ncnn-moe-runtime_b200/csrc/moe_internal.h"

namespace {

int failures = 0;

void expect(const char* what, const char* text, bool refused)
{
    if ((text != nullptr) != refused)
    {
        std::printf("%s: %s\n", what, text != nullptr ? text : "accepted");
        ++failures;
    }
}

template<typename T>
T* at(size_t address)
{
    return reinterpret_cast<T*>(address);
}

} // namespace

int main()
{
    using namespace moe;
    {
        const QuantizeArgs good = {at<void>(256), 4, 8, 200, 400, at<uint32_t>(64), at<uint8_t>(128), at<float>(64), at<uint32_t>(4)};
        const auto check = [&](const char* what, bool refused, int dtype, int activation, auto change) {
            QuantizeArgs args = good;
            change(args);
            expect(what, check_quantize(args, dtype, activation), refused);
        };
        check("quantize", false, MOE_DTYPE_BF16, MOE_ACTIVATION_SILU_GATE, [](QuantizeArgs&) {});
        check("quantize fp32", false, MOE_DTYPE_F32, MOE_ACTIVATION_NONE, [](QuantizeArgs&) {});
        check("quantize dtype", true, 2, MOE_ACTIVATION_NONE, [](QuantizeArgs&) {});
        check("quantize activation", true, MOE_DTYPE_F32, 2, [](QuantizeArgs&) {});
        check("quantize stride", true, MOE_DTYPE_F32, MOE_ACTIVATION_SILU_GATE, [](QuantizeArgs& a) { a.row_stride = 399; });
        check("quantize stride, plain", false, MOE_DTYPE_F32, MOE_ACTIVATION_NONE, [](QuantizeArgs& a) { a.row_stride = 200; });
        check("quantize no rows", false, MOE_DTYPE_F32, MOE_ACTIVATION_NONE, [](QuantizeArgs& a) { a.rows = 0; a.source = nullptr; a.values = nullptr; });
        check("quantize no source rows", false, MOE_DTYPE_F32, MOE_ACTIVATION_NONE, [](QuantizeArgs& a) { a.source_rows = 0; a.source = nullptr; });
        check("quantize rows", true, MOE_DTYPE_F32, MOE_ACTIVATION_NONE, [](QuantizeArgs& a) { a.rows = 0x80000000u; });
        check("quantize null source", true, MOE_DTYPE_F32, MOE_ACTIVATION_NONE, [](QuantizeArgs& a) { a.source = nullptr; });
        check("quantize null scales", true, MOE_DTYPE_F32, MOE_ACTIVATION_NONE, [](QuantizeArgs& a) { a.scales = nullptr; });
        check("quantize alignment", true, MOE_DTYPE_F32, MOE_ACTIVATION_NONE, [](QuantizeArgs& a) { a.source = at<void>(258); });
        check("quantize alignment bf16", false, MOE_DTYPE_BF16, MOE_ACTIVATION_NONE, [](QuantizeArgs& a) { a.source = at<void>(258); });
    }
    {
        // rows that are quantised once: four routes a row, 2^25 values, 16-byte vectors, scratch that stays in L2
        const auto once = [](uint32_t source_rows, uint32_t rows, uint32_t columns, size_t values) {
            const QuantizeArgs args = {at<void>(256), source_rows, rows, columns, columns, at<uint32_t>(64), at<uint8_t>(values), at<float>(64), at<uint32_t>(4)};
            return quantize_once_bytes(args);
        };
        if (once(4096, 32768, 4096, 256) != 4096u * 4096u + 4u * 4096u * 32u || once(1000, 33000, 1040, 256) != 1000u * 1040u + 4u * 1000u * 9u || once(4096, 16383, 4096, 256) != 0 ||
            once(1000, 32000, 1040, 256) != 0 || once(1000, 33000, 1032, 256) != 0 || once(1000, 33000, 1040, 264) != 0 || once(16384, 65536, 4096, 256) != 0 || once(0, 32768, 4096, 256) != 0)
        {
            std::printf("quantize_once_bytes\n");
            ++failures;
        }
    }
    {
        const ProductArgs good = {at<uint8_t>(256), at<float>(64), 10, 144, at<uint8_t>(512), at<float>(64), 4, 77, at<uint32_t>(64), at<void>(64), 80, at<uint32_t>(4)};
        const auto check = [&](const char* what, bool refused, int dtype, auto change) {
            ProductArgs args = good;
            change(args);
            expect(what, check_product(args, dtype), refused);
        };
        check("product", false, MOE_DTYPE_BF16, [](ProductArgs&) {});
        check("product out dtype", true, 7, [](ProductArgs&) {});
        check("product no experts", true, MOE_DTYPE_F32, [](ProductArgs& a) { a.expert_count = 0; });
        check("product most experts", false, MOE_DTYPE_F32, [](ProductArgs& a) { a.expert_count = 4096; });
        check("product too many experts", true, MOE_DTYPE_F32, [](ProductArgs& a) { a.expert_count = 4097; });
        check("product offsets missing", true, MOE_DTYPE_F32, [](ProductArgs& a) { a.expert_offsets = nullptr; });
        check("product dense", false, MOE_DTYPE_F32, [](ProductArgs& a) { a.expert_offsets = nullptr; a.expert_count = 1; });
        check("product columns", true, MOE_DTYPE_F32, [](ProductArgs& a) { a.columns = 136; });
        check("product no columns", true, MOE_DTYPE_F32, [](ProductArgs& a) { a.columns = 0; });
        check("product no outputs", true, MOE_DTYPE_F32, [](ProductArgs& a) { a.outputs = 0; });
        check("product weight rows", true, MOE_DTYPE_F32, [](ProductArgs& a) { a.outputs = 1u << 30; a.out_stride = 1u << 30; });
        check("product rows", true, MOE_DTYPE_F32, [](ProductArgs& a) { a.rows = 0x80000000u; });
        check("product stride", true, MOE_DTYPE_F32, [](ProductArgs& a) { a.out_stride = 76; });
        check("product no rows", false, MOE_DTYPE_F32, [](ProductArgs& a) { a.rows = 0; a.values = nullptr; a.out = nullptr; });
        check("product null out", true, MOE_DTYPE_F32, [](ProductArgs& a) { a.out = nullptr; });
        check("product values alignment", true, MOE_DTYPE_F32, [](ProductArgs& a) { a.values = at<uint8_t>(264); });
        check("product weights alignment", true, MOE_DTYPE_F32, [](ProductArgs& a) { a.weights = at<uint8_t>(520); });
        check("product out alignment", true, MOE_DTYPE_F32, [](ProductArgs& a) { a.out = at<void>(66); });
        check("product out alignment bf16", false, MOE_DTYPE_BF16, [](ProductArgs& a) { a.out = at<void>(66); });
    }
    {
        const CombineArgs good = {at<void>(256), 50, 50, at<uint32_t>(64), at<uint32_t>(64), at<float>(64), 12, 6, 2, nullptr, at<void>(64), nullptr, at<uint32_t>(4)};
        const auto check = [&](const char* what, bool refused, int dtype, auto change) {
            CombineArgs args = good;
            change(args);
            expect(what, check_combine(args, dtype), refused);
        };
        check("combine", false, MOE_DTYPE_BF16, [](CombineArgs&) {});
        check("combine dtype", true, -1, [](CombineArgs&) {});
        check("combine stride", true, MOE_DTYPE_F32, [](CombineArgs& a) { a.row_stride = 49; });
        check("combine no tokens", false, MOE_DTYPE_F32, [](CombineArgs& a) { a.token_count = 0; a.out = nullptr; });
        check("combine no routes", false, MOE_DTYPE_F32, [](CombineArgs& a) { a.route_count = 0; a.route_rows = nullptr; a.route_token = nullptr; });
        check("combine top_k", true, MOE_DTYPE_F32, [](CombineArgs& a) { a.top_k = 0; });
        check("combine largest top_k", false, MOE_DTYPE_F32, [](CombineArgs& a) { a.top_k = 4096; });
        check("combine too large top_k", true, MOE_DTYPE_F32, [](CombineArgs& a) { a.top_k = 4097; });
        check("combine null out", true, MOE_DTYPE_F32, [](CombineArgs& a) { a.out = nullptr; });
        check("combine null ranks", true, MOE_DTYPE_F32, [](CombineArgs& a) { a.route_rank = nullptr; });
        check("combine base alignment", true, MOE_DTYPE_F32, [](CombineArgs& a) { a.base = at<void>(66); });
        check("combine tokens", true, MOE_DTYPE_F32, [](CombineArgs& a) { a.token_count = 0x80000000u; });
    }
    {
        BalanceArgs args = {};
        expect("balance", check_balance(args), false);
        args.logits = at<float>(66);
        expect("balance logits alignment", check_balance(args), true);
        args.logits = at<float>(64);
        args.expert_tokens = at<uint32_t>(65);
        expect("balance tokens alignment", check_balance(args), true);
        args.expert_tokens = nullptr;
        args.score_function = 3;
        expect("balance score", check_balance(args), true);
        args.score_function = MOE_ROUTER_SQRT_SOFTPLUS;
        args.coefficient = NAN;
        expect("balance coefficient nan", check_balance(args), true);
        args.coefficient = INFINITY;
        expect("balance coefficient inf", check_balance(args), true);
    }
    return failures == 0 ? 0 : 1;
}
