// The operators around the quantized projections through the C++ host mirror, their first calls of the process captured: whole
// numbers whose results are known.  The exit code counts what is wrong.
#include <cstdio>

#include "ironmlx_b200.hpp"

using namespace ironmlx;

template <class T>
static void* device(const std::vector<T>& v) {
    void* p = nullptr;
    check_cuda(cudaMalloc(&p, v.size() * sizeof(T)));
    check_cuda(cudaMemcpy(p, v.data(), v.size() * sizeof(T), cudaMemcpyHostToDevice));
    return p;
}

static int run() {
    const int m = 200, in = 64, out = 96, rank = 8;
    const uint16_t one = 0x3f80;
    const Array x(device(std::vector<uint16_t>(m * in, one)), {m, in}, Dtype::Bfloat16), residual(device(std::vector<uint16_t>(m * in, one)), {m, in}, Dtype::Bfloat16);
    Array h(device(std::vector<uint16_t>(m * in)), {m, in}, Dtype::Bfloat16), n(device(std::vector<uint16_t>(m * in)), {m, in}, Dtype::Bfloat16);
    Array q(device(std::vector<uint32_t>(m * in / 4)), {m, in / 4}, Dtype::Uint32), qs(device(std::vector<uint8_t>(m * in / 32)), {m, in / 32}, Dtype::Uint8);
    Array y(device(std::vector<uint16_t>(m * out)), {m, out}, Dtype::Bfloat16);
    const RMSNorm norm{Array(device(std::vector<uint16_t>(in, one)), {in}, Dtype::Bfloat16), 0.f};
    QuantizedLinear proj{};
    proj.weight = Array(device(std::vector<uint32_t>(out * in / 4, 0x38383838u)), {out, in / 4}, Dtype::Uint32);         // 1
    proj.scales = Array(device(std::vector<uint8_t>(out * in / 32, 127)), {out, in / 32}, Dtype::Uint8);
    proj.mode = "mxfp8";
    const LowRankAdapters ad{Array(device(std::vector<uint16_t>(2 * rank * in, one)), {2, rank, in}, Dtype::Bfloat16),
                             Array(device(std::vector<uint16_t>(2 * out * rank, 0x3b00)), {2, out, rank}, Dtype::Bfloat16),       // 2^-9
                             Array(device(std::vector<float>{2.f, 4.f}), {2}, Dtype::Float32)};
    std::vector<int32_t> which(m);
    for (int i = 0; i < m; ++i) which[i] = i % 3 - 1;
    const Array ids(device(which), {m}, Dtype::Int32);
    cudaStream_t stream;
    cudaGraph_t graph;
    cudaGraphExec_t exec;
    check_cuda(cudaStreamCreate(&stream));
    check_cuda(cudaDeviceSynchronize());
    check_cuda(cudaStreamBeginCapture(stream, cudaStreamCaptureModeGlobal));
    norm.forward_residual(x, &residual, &h, &n, &q, &qs, stream);        // h = 2, the norm 1
    proj.forward_rows(q, qs, y, stream);                                 // 64
    ad.add(y, n, ids, stream);                                           // + 0, 2, 4
    check_cuda(cudaStreamEndCapture(stream, &graph));
    check_cuda(cudaGraphInstantiate(&exec, graph, 0));
    int wrong = 0;
    for (int replay = 0; replay < 2; ++replay) {
        check_cuda(cudaGraphLaunch(exec, stream));
        ops::check_status(stream);
        std::vector<uint16_t> got(m * out);
        check_cuda(cudaMemcpy(got.data(), y.ptr, got.size() * 2, cudaMemcpyDeviceToHost));
        const uint16_t want[3] = {0x4280, 0x4284, 0x4288};               // 64, 66, 68
        for (int i = 0; i < m * out; ++i) wrong += got[i] != want[i / out % 3];
    }
    return wrong == 0 ? 0 : 1;
}

int main() {
    try {
        return run();
    } catch (const Error& e) {
        std::printf("failed: %s\n", e.what());
        return 98;
    }
}
