// Low-rank adapters of many requests beside a shared projection: row t with the adapter j = ids[t] gets
//   out[t] = bf16( y[t] + scale[j] * (x[t] . a[j]^T) . b[j]^T ),   a[j]: [rank, in], b[j]: [n_out, rank]
// and a row whose id is outside [0, count) gets out[t] = y[t].
// One CTA a row: a warp per value of the low-rank row (fp32), then a thread per output.
#include "internal.h"

namespace imx {

namespace {

constexpr int kMaxRank = 256;

__global__ void __launch_bounds__(256)
low_rank_kernel(const __nv_bfloat16* y, const __nv_bfloat16* __restrict__ x, int in, const __nv_bfloat16* __restrict__ a,
                const __nv_bfloat16* __restrict__ b, const float* __restrict__ scale, int count, int rank,
                const int32_t* __restrict__ ids, int n_out, __nv_bfloat16* out) {
    __shared__ float s_low[kMaxRank];
    const size_t row = blockIdx.x;
    const int id = ids[row], warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const bool has = id >= 0 && id < count;
    if (has) {
        const float sc = scale != nullptr ? scale[id] : 1.f;
        for (int r = warp; r < rank; r += 8) {
            const __nv_bfloat16* ar = a + ((size_t)id * rank + r) * in;
            float acc = 0.f;
            for (int k = lane; k < in; k += 32) acc = fmaf(__bfloat162float(x[row * in + k]), __bfloat162float(ar[k]), acc);
            acc = warp_sum(acc);
            if (lane == 0) s_low[r] = acc * sc;
        }
    }
    __syncthreads();
    for (int n = threadIdx.x; n < n_out; n += 256) {
        const size_t at = row * n_out + n;
        __nv_bfloat16 o = y[at];
        if (has) {
            const __nv_bfloat16* br = b + ((size_t)id * n_out + n) * rank;
            float acc = 0.f;
            for (int r = 0; r < rank; ++r) acc = fmaf(s_low[r], __bfloat162float(br[r]), acc);
            o = __float2bfloat16_rn(__bfloat162float(o) + acc);
        }
        out[at] = o;
    }
}

}  // namespace

}  // namespace imx

using namespace imx;

extern "C" {

int imx_low_rank_scratch_bytes(int n_rows, int in, int n_out, int count, int rank, size_t* bytes) {
    IMX_REQUIRE(bytes != nullptr && n_rows >= 0 && in > 0 && n_out > 0 && count > 0 && rank > 0 && rank <= kMaxRank,
                "low_rank_scratch_bytes: bad arguments");
    *bytes = 256;
    return IMX_OK;
}

int imx_low_rank_add(const void* y, const void* x, int n_rows, int in, const imx_adapters* ad, const int32_t* ids, int n_out,
                     void* out, void* scratch, size_t scratch_bytes, void* stream) {
    IMX_REQUIRE(n_rows >= 0 && n_out > 0 && in > 0 && in % 8 == 0,
                "low_rank_add: sizes (%d rows, %d -> %d) must be positive, the input dimension a multiple of 8", n_rows, in, n_out);
    if (n_rows == 0) return IMX_OK;
    IMX_REQUIRE(y && x && ad && ids && out, "low_rank_add: y, x, adapters, ids and out are required");
    IMX_REQUIRE(ad->a && ad->b && ad->count > 0, "low_rank_add: at least one adapter is required");
    IMX_REQUIRE(ad->rank > 0 && ad->rank % 8 == 0 && ad->rank <= kMaxRank,
                "low_rank_add: the rank (%d) must be a multiple of 8, at most %d", ad->rank, kMaxRank);
    IMX_REQUIRE((((uintptr_t)x | (uintptr_t)ad->a | (uintptr_t)ad->b) % 16) == 0, "low_rank_add: x, a and b must be 16-byte aligned");
    IMX_REQUIRE((((uintptr_t)ids | (uintptr_t)ad->scale) % 4) == 0, "low_rank_add: ids and scale must be aligned to their values");
    IMX_REQUIRE((((uintptr_t)y | (uintptr_t)out) % 2) == 0, "low_rank_add: y and out must be aligned to their bf16 values");
    if (scratch == nullptr || (uintptr_t)scratch % 256 != 0 || scratch_bytes < 256) {
        set_error("low_rank_add: 256-byte aligned scratch of %zu bytes needed, %zu given", (size_t)256, scratch_bytes);
        return IMX_ERR_WORKSPACE;
    }
    const size_t ob = (size_t)n_rows * n_out * 2;
    IMX_REQUIRE(out == y || !overlap(out, ob, y, ob), "low_rank_add: out overlaps y without being it");
    IMX_REQUIRE(!overlap(out, ob, x, (size_t)n_rows * in * 2) && !overlap(out, ob, ids, (size_t)n_rows * 4) &&
                !overlap(out, ob, ad->a, (size_t)ad->count * ad->rank * in * 2) &&
                !overlap(out, ob, ad->b, (size_t)ad->count * ad->rank * n_out * 2) &&
                (ad->scale == nullptr || !overlap(out, ob, ad->scale, (size_t)ad->count * 4)), "low_rank_add: out overlaps another array");
    low_rank_kernel<<<n_rows, 256, 0, (cudaStream_t)stream>>>((const __nv_bfloat16*)y, (const __nv_bfloat16*)x, in,
                                                              (const __nv_bfloat16*)ad->a, (const __nv_bfloat16*)ad->b, ad->scale,
                                                              ad->count, ad->rank, ids, n_out, (__nv_bfloat16*)out); IMX_LAUNCHED();
    IMX_CHECK_CUDA(cudaGetLastError());
    return IMX_OK;
}

}  // extern "C"
