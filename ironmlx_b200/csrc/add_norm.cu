// The residual's addition, RMSNorm and the next projection's rows in 8 bits (mlx/src/model/qwen35.rs:262-273 around
// fast::rms_norm, mlx/src/fast.rs:37-49), one pass over the data:
//   v = x + residual              fp32; h = bf16(v)
//   u = v * inv * w               fp32, inv = rsqrt(mean(v^2) + eps); y = bf16(u)
//   q = e4m3(u / 2^e)             e per 32 values: the smallest power of two with amax / 2^e <= 448 (imx_quantize's rule)
//
// Bound by memory for many rows, by latency for few: 8192 rows of 2048 with a residual and all outputs take 29 us (152 MB at
// 5.2 TB/s, 80% of the copy bandwidth), 777 rows of 5120 in bf16 5.6 us, 64 rows of 2048 2.6 us.  A row's values stay in the
// registers of its threads between the sum of squares and the outputs (NV pieces of eight values a thread), so that everything is
// read and written once.  Four neighbouring lanes hold the 32 values of a scale: two shuffles give the maximum.  Codes and scales
// are those that the formula has for v: squares are summed in 64 bits where codes leave, and what fp32 leaves uncertain after that
// is computed in 64 bits (1.5 of the 29 us).
#include <cuda_fp8.h>

#include "internal.h"

namespace imx {

namespace {

constexpr int kMaxRow = 32768;
// Threads a CTA may have with NV pieces a thread: what leaves a thread the registers to hold them.
constexpr int max_threads(int nv) { return nv <= 2 ? 1024 : 512; }

struct NormOut {
    __nv_bfloat16* h;
    __nv_bfloat16* y;
    uint8_t* q;
    uint8_t* scales;
};

// Biased exponent of the scale of 32 values: e + 127, e the smallest integer in [-127, 127] with amax / 448 <= 2^e
// (an infinity among them: 255, which is NaN).
__device__ __forceinline__ uint32_t scale_code(float amax) {
    const uint32_t b = __float_as_uint(__fdiv_rn(amax, 448.f));
    const uint32_t exp = b >> 23, man = b & 0x7fffffu;
    if (exp == 0) return man <= 0x400000u ? 0u : 1u;             // up to 2^-127, up to 2^-126
    return exp + (man != 0 ? 1u : 0u);
}

// 1 / sqrt(a) as hi + lo: a Newton step from rsqrtf, what it leaves kept apart.
__device__ __forceinline__ void inverse_root(double a, float& hi, float& lo) {
    const float f = (float)a, r = rsqrtf(f), t = f * r;
    const float e = fmaf(-t, r, 1.f) - (fmaf(f, r, -t) + (float)(a - (double)f) * r) * r;       // 1 - a r^2
    hi = r;
    lo = f > 0.f && f < INFINITY ? 0.5f * r * e : 0.f;
}
// Codes of values that fp32's roundings (two of v * inv * w, a's and rsqrtf's: under 2^-21) could have put on the other side of the
// middle between two codes, normal numbers or not: those of the value a little larger and a little smaller differ.  They are
// decided with what the roundings left out: one value in 50000, so that it costs next to nothing.  (Told by the mantissa's bits,
// and below 2^-6 by the value, 8192 rows of 2048 took 27.0 us, so 25.5.)
constexpr float kAround = 0x1p-20f;
__device__ __forceinline__ uint32_t codes2(float a, float b) { return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3); }     // NaN stays NaN
// v * inv * w * up for the conversion: what 64 bits round is 2^-45 of it, and so it is the middle itself if it is that near;
// else cut off to fp32 with a last bit that keeps it off the middle (whose bit is 0) on its side.
__device__ __forceinline__ float decided(float v, float inv, float inv_lo, float w, float up) {
    const double d = (double)v * ((double)inv + (double)inv_lo) * (double)w * (double)up;
    const float f = (float)d;
    if (fabs(d - (double)f) <= fabs(d) * 0x1p-42) return f;
    return __uint_as_float(__float_as_uint(__double2float_rz(d)) | 1u);
}

// T threads a row (a multiple of 32), blockDim.x / T rows a CTA.
template <int NV>
__global__ void __launch_bounds__(max_threads(NV), NV == 4 ? 2 : 1)         // (64 registers: with 66 8192 rows of 2048 take 29.9 us)
add_rms_norm_kernel(const __nv_bfloat16* x, const __nv_bfloat16* residual, int n, int H, const __nv_bfloat16* w, float eps,
                    const NormOut out, int T, double per_value) {
    __shared__ double s_part[32];
    const int row_in = threadIdx.x / T, t = threadIdx.x - row_in * T;
    const long row = (long)blockIdx.x * (blockDim.x / T) + row_in;
    const int pieces = row < n ? H / 8 : 0;
    const size_t base = (size_t)row * H;
    float v[NV][8];
    float ss = 0.f;
    uint4 a[NV], b[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int p = t + i * T;
        if (p < pieces) {
            a[i] = *reinterpret_cast<const uint4*>(x + base + (size_t)p * 8);
            if (residual != nullptr) b[i] = *reinterpret_cast<const uint4*>(residual + base + (size_t)p * 8);
        }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if (t + i * T < pieces) {
            const __nv_bfloat162* pa = reinterpret_cast<const __nv_bfloat162*>(&a[i]);
            const __nv_bfloat162* pb = reinterpret_cast<const __nv_bfloat162*>(&b[i]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float2 f = __bfloat1622float2(pa[j]);
                if (residual != nullptr) {
                    const float2 g = __bfloat1622float2(pb[j]);
                    f.x += g.x;
                    f.y += g.y;
                }
                v[i][2 * j] = f.x;
                v[i][2 * j + 1] = f.y;
            }
        }
    }
    // In 64 bits from the squares on where codes leave: sums of a thread's 32 in fp32 would put some 6 of 17 million on the other
    // side of a middle (8192 rows of 2048, mxfp8 alone: 25.4 instead of 24.4 us; with what fp32 rounds away added up, 25.8).
    double sum = 0.;
    if (out.q != nullptr) {
        double part[2] = {};                  // (two chains: with one 8192 rows take 2% longer)
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (t + i * T < pieces)
#pragma unroll
                for (int j = 0; j < 8; ++j) part[j % 2] = fma((double)v[i][j], (double)v[i][j], part[j % 2]);
        sum = part[0] + part[1];
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (t + i * T < pieces)
#pragma unroll
                for (int j = 0; j < 8; ++j) ss = fmaf(v[i][j], v[i][j], ss);
        sum = ss;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (T > 32) {
        if ((threadIdx.x & 31) == 0) s_part[threadIdx.x >> 5] = sum;
        __syncthreads();
        sum = 0.;
        for (int i = 0; i < T / 32; ++i) sum += s_part[row_in * (T / 32) + i];
    }
    float inv, inv_lo;
    inverse_root(fma(sum, per_value, (double)eps), inv, inv_lo);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int p = t + i * T;
        // whole quads of lanes are in or out where a scale is wanted (H a multiple of 32)
        const unsigned active = __ballot_sync(0xffffffffu, p < pieces);
        if (p >= pieces) continue;
        const size_t at = base + (size_t)p * 8;
        if (out.h != nullptr) {
            __nv_bfloat162 o[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = __floats2bfloat162_rn(v[i][2 * j], v[i][2 * j + 1]);
            *reinterpret_cast<uint4*>(out.h + at) = *reinterpret_cast<const uint4*>(o);
        }
        float u[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] = v[i][j] * inv;
        if (w != nullptr) {
            const uint4 wv = __ldg(reinterpret_cast<const uint4*>(w + (size_t)p * 8));
            const __nv_bfloat162* pw = reinterpret_cast<const __nv_bfloat162*>(&wv);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 f = __bfloat1622float2(pw[j]);
                u[2 * j] *= f.x;
                u[2 * j + 1] *= f.y;
            }
        }
        if (out.y != nullptr) {
            __nv_bfloat162 o[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = __floats2bfloat162_rn(u[2 * j], u[2 * j + 1]);
            *reinterpret_cast<uint4*>(out.y + at) = *reinterpret_cast<const uint4*>(o);
        }
        if (out.q != nullptr) {
            float amax = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(u[j]));
            amax = fmaxf(amax, __shfl_xor_sync(active, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(active, amax, 2));
            uint32_t code = scale_code(amax);
            float up = __uint_as_float((254u - code) << 23);               // 2^-e
            const float above = up * (1.f + kAround), below = up * (1.f - kAround);
            // (amax next to 448, 1.75 * 2^8, times a power of two, by eight units of the last place: its scale is uncertain too)
            const bool at_border = (__float_as_uint(amax) & 0x7fffffu) - 0x5ffff8u <= 16u;
            uint32_t c[4], differ = at_border;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                c[j] = codes2(u[2 * j] * above, u[2 * j + 1] * above);
                differ |= c[j] ^ codes2(u[2 * j] * below, u[2 * j + 1] * below);
            }
            if (differ != 0) {
                if (at_border) {                                           // (the same in the quad)
                    const float border = __uint_as_float((__float_as_uint(amax) & 0x7f800000u) | 0x600000u);
                    const double root = (double)inv + (double)inv_lo, most = (double)border * (1. + 0x1p-42);      // (nearer it is the border itself)
                    bool over = false;
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        over = over || fabs((double)v[i][j] * (w == nullptr ? 1. : (double)__bfloat162float(w[(size_t)p * 8 + j]))) * root > most;
                    code = scale_code(border) + (__any_sync(0xfu << (threadIdx.x & 28), over) ? 1u : 0u);
                    up = __uint_as_float((254u - code) << 23);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const size_t k = (size_t)p * 8 + 2 * j;
                    const float w0 = w == nullptr ? 1.f : __bfloat162float(w[k]), w1 = w == nullptr ? 1.f : __bfloat162float(w[k + 1]);
                    c[j] = codes2(decided(v[i][2 * j], inv, inv_lo, w0, up), decided(v[i][2 * j + 1], inv, inv_lo, w1, up));
                }
            }
            *reinterpret_cast<uint2*>(out.q + at) = make_uint2(c[0] | c[1] << 16, c[2] | c[3] << 16);
            if ((p & 3) == 0) out.scales[at / 32] = (uint8_t)code;
        }
    }
}

int launch_add_rms_norm(const void* x, const void* residual, int n, int H, const void* w, float eps, const NormOut& out, cudaStream_t stream) {
    const int pieces = H / 8;
    // As few threads a row as hold it in four pieces each (eight of the longest rows) while there are rows enough to fill the
    // GPU (8192 rows of 2048 with 64 threads a row); two or one piece a thread, the shorter way, for a few rows.  Threads in
    // warps, not powers of two: 777 rows of 5120 take 5.3 us with 160 a row, with 256, for which there is no room at once, 6.8.
    DeviceInfo di;
    IMX_TRY(current_device(&di));
    auto threads = [&](int nv) { return ceil_div(ceil_div(pieces, nv), 32) * 32; };
    int nv = threads(4) <= max_threads(4) ? 4 : 8;
    while (nv > 1 && threads(nv / 2) <= max_threads(nv / 2) && (threads(nv / 2) == threads(nv) || (long)n * threads(nv / 2) <= 1024L * di.sms)) nv /= 2;
    const int T = threads(nv), rows = T < 256 ? 256 / T : 1, block = T * rows;
    const unsigned grid = (unsigned)(((long)n + rows - 1) / rows);
    auto kernel = nv <= 1 ? add_rms_norm_kernel<1> : (nv <= 2 ? add_rms_norm_kernel<2> : (nv <= 4 ? add_rms_norm_kernel<4> : add_rms_norm_kernel<8>));
    kernel<<<grid, block, 0, stream>>>((const __nv_bfloat16*)x, (const __nv_bfloat16*)residual, n, H, (const __nv_bfloat16*)w, eps,
                                       out, T, 1. / H); IMX_LAUNCHED();
    IMX_CHECK_CUDA(cudaGetLastError());
    return IMX_OK;
}

}  // namespace

}  // namespace imx

using namespace imx;

extern "C" int imx_add_rms_norm(const void* x, const void* residual, int n_rows, int hidden, const void* weight, float eps,
                                void* h, void* y, void* y_q, void* y_scales, void* stream) {
    IMX_REQUIRE(n_rows >= 0, "add_rms_norm: negative row count");
    IMX_REQUIRE(hidden > 0 && hidden % 8 == 0 && hidden <= kMaxRow,
                "add_rms_norm: the row length (%d) must be a positive multiple of 8, at most %d", hidden, kMaxRow);
    if (n_rows == 0) return IMX_OK;
    IMX_REQUIRE((y_q == nullptr) == (y_scales == nullptr), "add_rms_norm: y_q and y_scales go together");
    IMX_REQUIRE(y_q == nullptr || hidden % 32 == 0, "add_rms_norm: 8-bit rows need a row length (%d) that is a multiple of 32", hidden);
    IMX_REQUIRE(x != nullptr && (h != nullptr || y != nullptr || y_q != nullptr), "add_rms_norm: x and an output are required");
    IMX_REQUIRE((((uintptr_t)x | (uintptr_t)residual | (uintptr_t)weight | (uintptr_t)h | (uintptr_t)y | (uintptr_t)y_q) % 16) == 0,
                "add_rms_norm: arrays must be 16-byte aligned");
    const size_t values = (size_t)n_rows * hidden;
    const void* outs[4] = {h, y, y_q, y_scales};
    const size_t sizes[4] = {values * 2, values * 2, values, values / 32};
    for (int i = 0; i < 4; ++i) {
        for (int j = i + 1; j < 4; ++j)
            IMX_REQUIRE(!overlap(outs[i], sizes[i], outs[j], sizes[j]), "add_rms_norm: two outputs overlap");
        IMX_REQUIRE(!overlap(outs[i], sizes[i], weight, (size_t)hidden * 2), "add_rms_norm: an output overlaps the weight");
        for (const void* in : {x, residual})
            IMX_REQUIRE(!overlap(outs[i], sizes[i], in, values * 2) || (i < 2 && outs[i] == in),
                        "add_rms_norm: an output overlaps an input without being it");
    }
    return launch_add_rms_norm(x, residual, n_rows, hidden, weight, eps,
                               NormOut{(__nv_bfloat16*)h, (__nv_bfloat16*)y, (uint8_t*)y_q, (uint8_t*)y_scales}, (cudaStream_t)stream);
}
