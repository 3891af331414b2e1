// Matrix product of 8-bit integers with a scale a row (token, pixel) and a scale a channel:
//   y[m][n] = act( (sum_k a[m][k] * w[n][k]) * (a_scale[m] * w_scale[n]) + bias[n] )
// The sum is exact: products of 8-bit integers in 32-bit accumulators, at most Y5_I8_MAX_K of them.  One rounding to the output type.
#include "y5_common.h"

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

struct GemmArgs {
    const signed char* a;
    const signed char* w;
    const float* a_scale;
    const float* w_scale;
    const float* bias;
    void* y;
    long long m, y_ld;
    int n, ld;  // ld: bytes of a row of a and of w
    int act;
    float slope;
};

__device__ __forceinline__ float act1(float v, int act, float slope) {
    if (act == Y5_ACT_LEAKY) return v > 0.f ? v : v * slope;
    if (act == Y5_ACT_SILU) return v * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(v * -1.44269504088896341f));
    return v;
}

// 64 x 64 outputs a workgroup, 32 x 32 a wave; fragments straight from memory.
template <typename T>
__global__ __launch_bounds__(256) void gemm_simple_kernel(const GemmArgs g) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int lr = lane & 15, lq = lane >> 4;
    const long long m0 = (long long)blockIdx.x * 64 + (wave & 1) * 32;
    const int n0 = blockIdx.y * 64 + (wave >> 1) * 32;
    i32x4 acc[2][2] = {};
    for (int k0 = 0; k0 < g.ld; k0 += 64) {  // every lane takes every turn: the matrix instruction reads all of them
        const int k = k0 + lq * 16;
        i32x4 pa[2], pw[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const long long m = m0 + i * 16 + lr;
            const int n = n0 + i * 16 + lr;
            pa[i] = pw[i] = i32x4{0, 0, 0, 0};
            if (m < g.m && k < g.ld) pa[i] = *reinterpret_cast<const i32x4*>(g.a + m * g.ld + k);
            if (n < g.n && k < g.ld) pw[i] = *reinterpret_cast<const i32x4*>(g.w + (long long)n * g.ld + k);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(pw[j], pa[i], acc[i][j], 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const long long m = m0 + i * 16 + lr;
        if (m >= g.m) continue;
        const float as = g.a_scale[m];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int n = n0 + j * 16 + lq * 4 + e;
                if (n >= g.n) continue;
                float v = (float)acc[i][j][e] * (as * g.w_scale[n]);
                if (g.bias) v += g.bias[n];
                static_cast<T*>(g.y)[m * g.y_ld + n] = (T)act1(v, g.act, g.slope);
            }
    }
}

}  // namespace

int y5_launch_gemm_i8(const y5_gemm_i8_desc& d, hipStream_t st) {
    Y5_REQUIRE(d.a && d.a_scale && d.w && d.w_scale && d.y, "gemm_i8: null tensor pointer");
    Y5_REQUIRE(d.dtype == Y5_F16 || d.dtype == Y5_BF16 || d.dtype == Y5_F32, "gemm_i8: dtype %d", d.dtype);
    Y5_REQUIRE(d.m > 0 && d.m <= 0x7fffffff && d.n > 0 && d.n <= 1 << 20, "gemm_i8: %lld rows, %d channels", (long long)d.m, d.n);
    Y5_REQUIRE(d.k > 0 && d.k <= Y5_I8_MAX_K, "gemm_i8: %d values a row (1 to %d)", d.k, Y5_I8_MAX_K);
    Y5_REQUIRE(d.ld == (d.k + 15) / 16 * 16, "gemm_i8: a row of a and w is %d bytes for %d values (got %d)", (d.k + 15) / 16 * 16, d.k, d.ld);
    Y5_REQUIRE(d.y_ld >= d.n, "gemm_i8: output pitch %lld for %d channels", (long long)d.y_ld, d.n);
    Y5_REQUIRE(d.act == Y5_ACT_NONE || d.act == Y5_ACT_LEAKY || d.act == Y5_ACT_SILU, "gemm_i8: activation %d", d.act);
    Y5_REQUIRE(y5_aligned16(d.a) && y5_aligned16(d.w), "gemm_i8: a and w must be 16-byte aligned");
    const int es = d.dtype == Y5_F32 ? 4 : 2;
    Y5_REQUIRE(reinterpret_cast<uintptr_t>(d.y) % es == 0 && reinterpret_cast<uintptr_t>(d.a_scale) % 4 == 0 && reinterpret_cast<uintptr_t>(d.w_scale) % 4 == 0 && reinterpret_cast<uintptr_t>(d.bias) % 4 == 0, "gemm_i8: misaligned pointer");
    GemmArgs g{};
    g.a = static_cast<const signed char*>(d.a);
    g.w = static_cast<const signed char*>(d.w);
    g.a_scale = d.a_scale;
    g.w_scale = d.w_scale;
    g.bias = d.bias;
    g.y = d.y;
    g.m = d.m;
    g.y_ld = d.y_ld;
    g.n = d.n;
    g.ld = d.ld;
    g.act = d.act;
    g.slope = d.slope;
    const dim3 grid((unsigned)((d.m + 63) / 64), (unsigned)((d.n + 63) / 64));
    if (d.dtype == Y5_F16) hipLaunchKernelGGL((gemm_simple_kernel<f16>), grid, dim3(256), 0, st, g);
    else if (d.dtype == Y5_BF16) hipLaunchKernelGGL((gemm_simple_kernel<bf16>), grid, dim3(256), 0, st, g);
    else hipLaunchKernelGGL((gemm_simple_kernel<float>), grid, dim3(256), 0, st, g);
    Y5_LAUNCH_CHECK("gemm_simple_kernel");
    return Y5_OK;
}
