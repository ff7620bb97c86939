// The operators around the quantized projections through the C++ host mirror.  "refuse": shapes that do not match (no GPU);
// "run": whole numbers whose results are known.  The exit code counts what is wrong.
#include <cstdio>
#include <cstring>
#include <functional>

#include "ironmlx_b200.hpp"

using namespace ironmlx;

static int wrong = 0;
static void expect(bool ok, const char* what) {
    if (ok) return;
    std::printf("wrong: %s\n", what);
    ++wrong;
}

static void refused(const char* what, const std::function<void()>& call) {
    try {
        call();
        expect(false, what);
    } catch (const Error& e) {
        expect(e.code == IMX_ERR_INVALID, what);
    }
}

static Array bf16(void* p, std::vector<int64_t> shape) { return Array(p, std::move(shape), Dtype::Bfloat16); }

static int refuse() {
    void* p = (void*)4096;
    Array rows(p, {4, 16}, Dtype::Bfloat16), scales(p, {4, 2}, Dtype::Bfloat16), w(p, {8, 16}, Dtype::Bfloat16), ws(p, {8, 2}, Dtype::Bfloat16);
    Array y = bf16(p, {4, 8}), short_w(p, {8, 8}, Dtype::Bfloat16), few_ws(p, {7, 2}, Dtype::Bfloat16), y3 = bf16(p, {3, 8}), none(p, {4, 0}, Dtype::Bfloat16);
    refused("a weight of another length", [&] { ops::mxfp8_matmul(rows, scales, short_w, ws, y); });
    refused("scales of fewer outputs", [&] { ops::mxfp8_matmul(rows, scales, w, few_ws, y); });
    refused("y of fewer rows", [&] { ops::mxfp8_matmul(rows, scales, w, ws, y3); });
    refused("rows without values", [&] { ops::mxfp8_matmul(rows, none, w, ws, y); });
    Array x = bf16(p, {4, 64}), ids(p, {4}, Dtype::Bfloat16), b = bf16(p, {2, 8, 8});
    refused("adapters of two ranks", [&] { LowRankAdapters{bf16(p, {2, 16, 64}), b, std::nullopt}.add(y, x, ids); });
    refused("fewer of one matrix", [&] { LowRankAdapters{bf16(p, {1, 8, 64}), b, std::nullopt}.add(y, x, ids); });
    refused("y of fewer rows", [&] { LowRankAdapters{bf16(p, {2, 8, 64}), b, std::nullopt}.add(y3, x, ids); });
    RMSNorm norm{bf16(p, {64}), 1e-6f};
    Array h = bf16(p, {4, 32});
    refused("h of another size", [&] { norm.forward_residual(x, nullptr, &h, &x, nullptr, nullptr); });
    return wrong;
}

template <class T>
static T* device(const std::vector<T>& v) {
    T* p = nullptr;
    check_cuda(cudaMalloc((void**)&p, v.size() * sizeof(T)));
    check_cuda(cudaMemcpy(p, v.data(), v.size() * sizeof(T), cudaMemcpyHostToDevice));
    return p;
}

static int run() {
    const int m = 5, in = 64, out = 96, rank = 8;
    const uint16_t one = 0x3f80, two = 0x4000;
    Array x = bf16(device(std::vector<uint16_t>(m * in, one)), {m, in}), residual = bf16(device(std::vector<uint16_t>(m * in, one)), {m, in});
    Array h = bf16(device(std::vector<uint16_t>(m * in)), {m, in}), n = bf16(device(std::vector<uint16_t>(m * in)), {m, in});
    Array q(device(std::vector<uint32_t>(m * in / 4)), {m, in / 4}, Dtype::Bfloat16), qs(device(std::vector<uint8_t>(m * in / 32)), {m, in / 32}, Dtype::Bfloat16);
    RMSNorm norm{bf16(device(std::vector<uint16_t>(in, one)), {in}), 0.f};
    norm.forward_residual(x, &residual, &h, &n, &q, &qs);                // h = 2, the norm 1
    QuantizedLinear proj{};
    proj.weight = Array(device(std::vector<uint32_t>(out * in / 4, 0x38383838u)), {out, in / 4}, Dtype::Bfloat16);       // 1
    proj.scales = Array(device(std::vector<uint8_t>(out * in / 32, 127)), {out, in / 32}, Dtype::Bfloat16);
    proj.mode = "mxfp8";
    Array y = bf16(device(std::vector<uint16_t>(m * out)), {m, out});
    proj.forward_rows(q, qs, y);                                         // 64
    LowRankAdapters ad{bf16(device(std::vector<uint16_t>(2 * rank * in, one)), {2, rank, in}),
                       bf16(device(std::vector<uint16_t>(2 * out * rank, 0x3b00)), {2, out, rank}),                       // 2^-9
                       Array(device(std::vector<float>{2.f, 4.f}), {2}, Dtype::Bfloat16)};
    ad.add(y, n, Array(device(std::vector<int32_t>{0, 1, -1, 0, 2}), {m}, Dtype::Bfloat16));                              // + 2, 4, 0, 2, 0
    std::vector<uint16_t> got(m * out), hs(m * in);
    check_cuda(cudaDeviceSynchronize());
    check_cuda(cudaMemcpy(got.data(), y.ptr, got.size() * 2, cudaMemcpyDeviceToHost));
    check_cuda(cudaMemcpy(hs.data(), h.ptr, hs.size() * 2, cudaMemcpyDeviceToHost));
    for (uint16_t v : hs) expect(v == two, "h");
    const float want[m] = {66.f, 68.f, 64.f, 66.f, 64.f};
    for (int i = 0; i < m * out; ++i) {
        uint32_t bits;
        std::memcpy(&bits, &want[i / out], 4);
        expect(got[i] == (uint16_t)(bits >> 16), "y");
    }
    return wrong;
}

int main(int argc, char** argv) {
    if (argc != 2) return 99;
    return std::strcmp(argv[1], "run") == 0 ? run() : refuse();
}
