// The 8-bit product where there is little of it: a few tokens through a layer, or a map of some hundred pixels.
//
// What counts is how soon every byte of the weights is on its way.  A workgroup makes (16 MI) x (16 NI) outputs and its eight waves
// split K: each reads its 64-byte steps of the rows and channels straight into the matrix instruction's layout (lane l: row l & 15, 16
// bytes at 16 * (l >> 4)), four steps ahead, and nothing waits for anything until the partial sums meet in LDS - exact in any order:
// integers.  For up to Y5_FEW_ROWS rows the quantisation is done here too, by every workgroup for itself (a few KiB from the cache
// against a launch of its own), while its first weights are in flight.  1 x 4096 x 4096 bf16: 6.3 us (16.8 MB of weights at 2.7
// TB/s: launch, quantisation and one round of loads are latencies, not rates); 333 x 1000 x 255: 4.0, 400 x 512 x 512: 4.6 (bound by
// the workgroups' starts).
#include "y5_common.h"

namespace {

#include "conv_common.h"
#include "gemm_i8.h"
#include "norm_rows.h"
#include "quant_rows.h"

constexpr int kWaves = 8, kAhead = 4;

struct FewArgs {
    GemmArgs g;
    const void* x;  // rows in their own type at pitch x_ld, k values each
    long long x_ld;
    int k;
    int tiles_n;  // workgroups side by side
};

// Rows to 8 bits in LDS: q[row][ld], scale[row].  tops: LDS, one word a row, zero.
template <typename TI>
__device__ __forceinline__ void quantise_to_lds(const FewArgs& a, unsigned char* q, float* scale, unsigned* tops) {
    constexpr int V = NormElem<TI>::V;
    const int t = threadIdx.x, T = kWaves * 64, rows = (int)a.g.m;
    for (int r = 0; r < rows; ++r) {
        const TI* x = static_cast<const TI*>(a.x) + r * a.x_ld;
        unsigned top = 0;
        for (int k = t * V; k < a.k; k += T * V) {
            TI v[V];
            if (a.k - k >= V) ld_vec(x + k, v);
            else ld_part(x + k, a.k - k, v);
#pragma unroll
            for (int e = 0; e < V; ++e) top = max_bits(top, (float)v[e]);
        }
        top = max_over(top, 64);
        if ((t & 63) == 0) atomicMax(&tops[r], top);  // the same whatever the order
    }
    __syncthreads();
    for (int r = 0; r < rows; ++r) {
        const TI* x = static_cast<const TI*>(a.x) + r * a.x_ld;
        const unsigned top = tops[r];
        const bool fine = top < 0x7f800000u;
        float m;
        const float s = row_scale(top, &m);
        if (t == 0) scale[r] = s;
        typename InvOf<TI, false>::type inv;
        inv.set(m, fine);
        for (int k = t * V; k < a.g.ld; k += T * V) {
            TI v[V];
            if (a.k - k >= V) ld_vec(x + k, v);
            else ld_part(x + k, a.k - k, v);
            unsigned w[V];
#pragma unroll
            for (int e = 0; e < V; ++e) w[e] = inv((float)v[e]);
#pragma unroll
            for (int e = 0; e < V; e += 4) *reinterpret_cast<int*>(q + r * a.g.ld + k + e) = pack_bytes(w[e], w[e + 1], w[e + 2], w[e + 3], fine);
        }
    }
    __syncthreads();
}

// TI: signed char for rows that are 8-bit already.  LDS: partial sums of waves 1 .. 7; with quantisation the rows behind them.
template <typename TI, typename T, int ACT, int MI, int NI>
__global__ __launch_bounds__(kWaves * 64) void gemm_few_kernel(const FewArgs a) {
    constexpr bool QUANT = sizeof(TI) != 1;
    static_assert(!QUANT || MI == 1, "few rows");
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    __shared__ float scale[Y5_FEW_ROWS];
    __shared__ unsigned tops[Y5_FEW_ROWS];
    const GemmArgs& g = a.g;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int lr = lane & 15, lq = lane >> 4;
    const int wm = blockIdx.x / a.tiles_n;
    const long long m0 = (long long)wm * (16 * MI);
    const int n0 = (blockIdx.x - wm * a.tiles_n) * (16 * NI);
    i32x4(*part)[MI * NI][64] = reinterpret_cast<i32x4(*)[MI * NI][64]>(smem);
    unsigned char* q = smem + (kWaves - 1) * MI * NI * 1024;
    const signed char *pa[MI], *pw[NI];
#pragma unroll
    for (int i = 0; i < MI; ++i) pa[i] = m0 + 16 * i + lr < g.m ? g.a + (m0 + 16 * i + lr) * g.ld : nullptr;
#pragma unroll
    for (int j = 0; j < NI; ++j) pw[j] = n0 + 16 * j + lr < g.n ? g.w + (long long)(n0 + 16 * j + lr) * g.ld : nullptr;
    const int steps = (g.ld + 63) / 64;  // of 64 bytes; wave w takes w, w + 8, ...
    i32x4 fw[kAhead][NI];
    auto load_w = [&](int s) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int k = (s + u * kWaves) * 64 + lq * 16;
#pragma unroll
            for (int j = 0; j < NI; ++j) {
                fw[u][j] = i32x4{0, 0, 0, 0};
                if (k < g.ld && pw[j]) fw[u][j] = *reinterpret_cast<const i32x4*>(pw[j] + k);
            }
        }
    };
    load_w(wave);
    if constexpr (QUANT) {
        if (t < Y5_FEW_ROWS) tops[t] = 0;
        __syncthreads();
        quantise_to_lds<TI>(a, q, scale, tops);
    }
    i32x4 acc[MI][NI];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
    for (int s = wave; s < steps; s += kAhead * kWaves) {  // every lane takes every turn: the matrix instruction reads all of them
        if (s != wave) load_w(s);
        i32x4 fa[kAhead][MI];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int k = (s + u * kWaves) * 64 + lq * 16;
#pragma unroll
            for (int i = 0; i < MI; ++i) {
                fa[u][i] = i32x4{0, 0, 0, 0};
                if constexpr (QUANT) {
                    if (k < g.ld && lr < g.m) fa[u][i] = *reinterpret_cast<const i32x4*>(q + lr * g.ld + k);
                } else {
                    if (k < g.ld && pa[i]) fa[u][i] = *reinterpret_cast<const i32x4*>(pa[i] + k);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j = 0; j < NI; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[u][j], fa[u][i], acc[i][j], 0, 0, 0);
    }
    if (wave) {
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j) part[wave - 1][i * NI + j][lane] = acc[i][j];
    }
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int i = 0; i < MI; ++i) {
        const long long m = m0 + 16 * i + lr;
        const float as = m >= g.m ? 0.f : QUANT ? scale[lr & (Y5_FEW_ROWS - 1)] : g.a_scale[m];
#pragma unroll
        for (int j = 0; j < NI; ++j) {
            i32x4 s = acc[i][j];
#pragma unroll
            for (int w = 0; w < kWaves - 1; ++w) s += part[w][i * NI + j][lane];
            const int n = n0 + 16 * j + 4 * lq;
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bool in = n + e < g.n;
                v[e] = (float)s[e] * (as * (in ? g.w_scale[n + e] : 0.f)) + (in && g.bias ? g.bias[n + e] : 0.f);
            }
            act_n<ACT>(v, g.slope);
            if (m < g.m && n < g.n) {
                T* p = static_cast<T*>(g.y) + m * g.y_ld + n;
                if (n + 4 <= g.n) {
                    const T o[4] = {(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
                    st_out<T, 4>(p, o);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (n + e < g.n) p[e] = (T)v[e];
                }
            }
        }
    }
}

template <typename TI, typename T, int ACT, int MI, int NI>
int launch(FewArgs a, hipStream_t st) {
    a.tiles_n = (a.g.n + 16 * NI - 1) / (16 * NI);
    const long long total = (a.g.m + 16 * MI - 1) / (16 * MI) * a.tiles_n;
    Y5_REQUIRE(total <= 0x7fffffffLL, "gemm_i8: %lld tiles", total);
    const dim3 grid((unsigned)total);
    const size_t lds = (size_t)(kWaves - 1) * MI * NI * 1024 + (a.x ? (size_t)a.g.m * a.g.ld : 0);
    if (lds + 64 > 64 << 10) Y5_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(gemm_few_kernel<TI, T, ACT, MI, NI>), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    hipLaunchKernelGGL((gemm_few_kernel<TI, T, ACT, MI, NI>), grid, dim3(kWaves * 64), lds, st, a);
    Y5_LAUNCH_CHECK("gemm_few_kernel");
    return Y5_OK;
}

template <typename T, int ACT>
int by_rows(const FewArgs& a, int rows, hipStream_t st) {
    if (a.x) return launch<T, T, ACT, 1, 1>(a, st);
    if (rows == 16) return launch<signed char, T, ACT, 1, 1>(a, st);
    return launch<signed char, T, ACT, 2, 1>(a, st);
}

template <typename T>
int by_act(const FewArgs& a, int rows, hipStream_t st) {
    if (a.g.act == Y5_ACT_LEAKY) return by_rows<T, Y5_ACT_LEAKY>(a, rows, st);
    if (a.g.act == Y5_ACT_SILU) return by_rows<T, Y5_ACT_SILU>(a, rows, st);
    return by_rows<T, Y5_ACT_NONE>(a, rows, st);
}

}  // namespace

int y5_launch_gemm_few(const y5_gemm_i8_desc& d, const void* x, int64_t x_ld, int rows, hipStream_t st) {
    FewArgs a{};
    a.g = make_gemm_args(d);
    a.x = x;
    a.x_ld = x_ld;
    a.k = d.k;
    if (d.dtype == Y5_F16) return by_act<f16>(a, rows, st);
    if (d.dtype == Y5_BF16) return by_act<bf16>(a, rows, st);
    return by_act<float>(a, rows, st);
}
