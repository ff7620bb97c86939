// Shapes that the C++ host mirror has to refuse before the C ABI's ints cut them off.  No GPU is needed; the exit code counts what
// is not refused.
#include <cstdio>
#include <functional>

#include "ironmlx_b200.hpp"

using namespace ironmlx;

static int wrong = 0;
static void refused(const char* what, const std::function<void()>& call) {
    try {
        call();
    } catch (const Error& e) {
        if (e.code == IMX_ERR_INVALID) return;
    }
    std::printf("not refused: %s\n", what);
    ++wrong;
}

int main() {
    void* p = (void*)4096;
    const int64_t wrap = (int64_t)1 << 32;
    auto bf16 = [&](std::vector<int64_t> shape) { return Array(p, std::move(shape), Dtype::Bfloat16); };
    Array y = bf16({wrap, 64}), h = y;
    // with 2^32 rows an int would say none: nothing to do, and no error
    refused("a norm of 2^32 rows", [&] { RMSNorm{bf16({64}), 1e-6f}.forward_residual(bf16({wrap, 64}), nullptr, &h, &y, nullptr, nullptr); });
    refused("a product of 2^32 rows", [&] { ops::mxfp8_matmul(bf16({wrap, 16}), bf16({wrap, 2}), bf16({64, 16}), bf16({64, 2}), y); });
    refused("a product over 2^32 values", [&] { Array few = bf16({4, 64}); ops::mxfp8_matmul(bf16({4, wrap / 4 + 16}), bf16({4, wrap / 32 + 2}), bf16({64, wrap / 4 + 16}), bf16({64, wrap / 32 + 2}), few); });
    refused("adapters beside 2^32 rows", [&] { LowRankAdapters{bf16({2, 8, 64}), bf16({2, 64, 8}), std::nullopt}.add(y, bf16({wrap, 64}), bf16({wrap})); });
    refused("adapters of a rank above 2^32", [&] { Array few = bf16({0, 64}); LowRankAdapters{bf16({2, wrap + 8, 64}), bf16({2, 64, wrap + 8}), std::nullopt}.add(few, bf16({0, 64}), bf16({0})); });
    QuantizedLinear proj{};
    proj.weight = bf16({64, 16});
    proj.scales = bf16({64, 2});
    proj.biases = bf16({64, 2});
    proj.mode = "mxfp8";
    refused("8-bit rows and a weight with biases", [&] { Array none = bf16({0, 64}); proj.forward_rows(bf16({0, 16}), bf16({0, 2}), none); });
    return wrong;
}
