// y = dequantize(x_q) . dequantize(w)^T with both operands in mxfp8 (e4m3 codes, one power of two for 32 values):
//   y[m, n] = bf16( sum over the blocks g of 2^(sx + sw - 254) * sum over k in g of qx * qw )
// One thread an output, fp32 sums.
#include <cuda_fp8.h>

#include "internal.h"

namespace imx {

namespace {

constexpr size_t kStatusBytes = 256;

// NaN (0x7f, 0xff; 255) stays NaN
__device__ __forceinline__ float e4m3_value(uint32_t c) { return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)c, __NV_E4M3))); }
__device__ __forceinline__ float scale_value(uint32_t s) { return s == 255u ? __uint_as_float(0x7fc00000u) : ue8m0_to_f32(s); }

__global__ void __launch_bounds__(256)
mxfp8_mm_kernel(const uint8_t* __restrict__ xq, const uint8_t* __restrict__ xs, int m, const uint8_t* __restrict__ wq,
                const uint8_t* __restrict__ ws, int n_out, int in, __nv_bfloat16* __restrict__ y) {
    const int n = blockIdx.x * 32 + (threadIdx.x & 31), row = blockIdx.y * 8 + (threadIdx.x >> 5);
    if (n >= n_out || row >= m) return;
    const uint8_t* a = xq + (size_t)row * in;
    const uint8_t* b = wq + (size_t)n * in;
    float acc = 0.f;
    for (int g = 0; g < in / 32; ++g) {
        float part = 0.f;
        for (int k = 0; k < 32; k += 4) {
            const uint32_t ca = *reinterpret_cast<const uint32_t*>(a + g * 32 + k), cb = *reinterpret_cast<const uint32_t*>(b + g * 32 + k);
#pragma unroll
            for (int i = 0; i < 32; i += 8) part = fmaf(e4m3_value((ca >> i) & 255u), e4m3_value((cb >> i) & 255u), part);
        }
        acc += part * (scale_value(xs[(size_t)row * (in / 32) + g]) * scale_value(ws[(size_t)n * (in / 32) + g]));
    }
    y[(size_t)row * n_out + n] = __float2bfloat16_rn(acc);
}

}  // namespace

}  // namespace imx

using namespace imx;

extern "C" {

int imx_mxfp8_matmul_scratch_bytes(int m, int n_out, int in, size_t* bytes) {
    IMX_REQUIRE(bytes != nullptr && m >= 0 && n_out > 0 && in > 0 && in % 32 == 0, "mxfp8_matmul_scratch_bytes: bad arguments");
    *bytes = kStatusBytes;
    return IMX_OK;
}

int imx_mxfp8_matmul(const void* x_q, const void* x_scales, int m, const imx_qtensor* w, int n_out, int in, void* y,
                     void* scratch, size_t scratch_bytes, void* stream) {
    IMX_REQUIRE(m >= 0 && n_out > 0 && in > 0 && in % 32 == 0,
                "mxfp8_matmul: sizes (%d rows, %d -> %d) must be positive, the input dimension a multiple of 32", m, in, n_out);
    if (m == 0) return IMX_OK;
    IMX_REQUIRE(x_q && x_scales && w && w->w && w->scales && y, "mxfp8_matmul: rows, weight and their scales, and y are required");
    IMX_REQUIRE(w->biases == nullptr, "mxfp8_matmul: an mxfp8 weight has no biases");
    IMX_REQUIRE((uintptr_t)x_q % 16 == 0 && (uintptr_t)w->w % 16 == 0, "mxfp8_matmul: rows and weight must be 16-byte aligned");
    IMX_REQUIRE((uintptr_t)y % 2 == 0, "mxfp8_matmul: y must be aligned to its bf16 values");
    if (scratch == nullptr || (uintptr_t)scratch % 256 != 0 || scratch_bytes < kStatusBytes) {
        set_error("mxfp8_matmul: 256-byte aligned scratch of %zu bytes needed, %zu given", kStatusBytes, scratch_bytes);
        return IMX_ERR_WORKSPACE;
    }
    const size_t yb = (size_t)m * n_out * 2, xb = (size_t)m * in, wb = (size_t)n_out * in;
    IMX_REQUIRE(!overlap(y, yb, x_q, xb) && !overlap(y, yb, x_scales, xb / 32) && !overlap(y, yb, w->w, wb) &&
                !overlap(y, yb, w->scales, wb / 32) && !overlap(y, yb, scratch, kStatusBytes), "mxfp8_matmul: y overlaps another array");
    mxfp8_mm_kernel<<<dim3((unsigned)ceil_div(n_out, 32), (unsigned)ceil_div(m, 8)), 256, 0, (cudaStream_t)stream>>>(
        (const uint8_t*)x_q, (const uint8_t*)x_scales, m, (const uint8_t*)w->w, (const uint8_t*)w->scales, n_out, in,
        (__nv_bfloat16*)y); IMX_LAUNCHED();
    IMX_CHECK_CUDA(cudaGetLastError());
    return IMX_OK;
}

}  // extern "C"
