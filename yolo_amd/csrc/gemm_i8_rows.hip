// The 8-bit product for many rows of few values: weights resident in LDS, rows quantised in the registers that read them.
//
// Such layers (1x1 convolutions on the finer maps) move far more bytes than they multiply, so a row is read once, in its own type,
// and its results are written once: y = act((sum q w) (scale_row scale_channel) + bias) with q and scale_row computed on the way
// (or read, where the rows are 8-bit already).  A wave owns blocks of 16 MI rows and shares nothing with the others: lane (lr, lq)
// reads the 16 values 64 f + 16 lq .. of row lr for every fragment f - which is v_mfma_i32_16x16x64_i8's operand layout, so that the
// quantised values never move between lanes; the row's maximum needs two moves between lanes.  The next block's values are loaded as soon as the
// fragments are made and fly under the products and the stores.  Accumulators cover 64 channels at a time, with the weight rows
// ordered so that a lane ends up with 16 consecutive channels.  Bound by HBM: 819200 x 64 x 64 fp16 in 41 us for 210 MB (5.1 TB/s, a
// cold copy's rate); 204800 x 256 x 256 from 8-bit rows 35 us for 157 MB, from fp16 46 for 210 MB (4.6 TB/s).  One block of 16 rows
// a wave (two of 64 values): with two the registers halve the waves (61 instead of 46 us).
#include "y5_common.h"

namespace {

#include "conv_common.h"
#include "gemm_i8.h"
#include "norm_rows.h"
#include "quant_rows.h"

struct RowsGemm {
    GemmArgs g;
    const void* x;     // rows in their own type, k values at pitch x_ld (k a multiple of 16); unused for 8-bit rows
    long long x_ld;
    int k;
    int chunks;        // of 64 channels
    long long blocks;  // of 16 MI rows
};

template <typename TI>
struct Frag {  // 16 values of a row as they are in memory
    static constexpr int NV = (int)sizeof(TI);
    norm_u32x4 v[NV];
    // the empty statement keeps the compiler from holding the values unpacked
    __device__ __forceinline__ NormArr<TI> unpack(int u) {
        asm volatile("" : "+v"(v[u]));
        return __builtin_bit_cast(NormArr<TI>, v[u]);
    }
};

template <typename TI, typename T, int ACT, int MI, int KF>
__global__ __launch_bounds__(512, sizeof(TI) == 4 && KF == 4 ? 2 : 4) void gemm_rows_kernel(const RowsGemm a) {
    constexpr bool QUANT = sizeof(TI) != 1;
    constexpr bool AHEAD = KF <= 4;  // the next block's values fly under this one's products; of 512 values a row there is no room for two
    constexpr int SV = 16 / (int)sizeof(T);
    extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
    const GemmArgs& g = a.g;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, lr = lane & 15, lq = lane >> 4;
    const int frags = a.chunks * 4;
    float* ws = reinterpret_cast<float*>(smem + frags * KF * 1024);
    float* bs = ws + a.chunks * 64;
    // fragment (chunk c, j, k-fragment f): lane (lr, lq) holds 16 bytes of channel 64 c + 16 (lr >> 2) + 4 j + (lr & 3), so that element e of
    // accumulator j of lane (., lq) is channel 64 c + 16 lq + 4 j + e
    for (int p = t; p < frags * KF * 64; p += 512) {
        const int l = p & 63, fk = p >> 6, f = fk % KF, cj = fk / KF;
        const int n = (cj >> 2) * 64 + ((l & 15) >> 2) * 16 + 4 * (cj & 3) + (l & 3), k = f * 64 + (l >> 4) * 16;
        i32x4 v = {0, 0, 0, 0};
        if (n < g.n && k < g.ld) v = *reinterpret_cast<const i32x4*>(g.w + (long long)n * g.ld + k);
        *reinterpret_cast<i32x4*>(smem + p * 16) = v;
    }
    for (int p = t; p < a.chunks * 64; p += 512) {
        ws[p] = p < g.n ? g.w_scale[p] : 0.f;
        bs[p] = p < g.n && g.bias ? g.bias[p] : 0.f;
    }
    __syncthreads();

    typedef typename std::conditional<QUANT, TI, f16>::type TX;
    Frag<TX> raw[QUANT ? MI : 1][QUANT ? KF : 1];
    i32x4 qn[QUANT ? 1 : MI][QUANT ? 1 : KF];
    float sn[MI];
    auto load = [&](long long blk) {
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            const long long row = blk * (16 * MI) + i * 16 + lr;
            if constexpr (!QUANT) sn[i] = row < g.m ? g.a_scale[row] : 0.f;
#pragma unroll
            for (int f = 0; f < KF; ++f) {
                const int k = f * 64 + lq * 16;
                if constexpr (QUANT) {
                    const TX* p = static_cast<const TX*>(a.x) + row * a.x_ld + k;
                    const bool in = row < g.m && k < a.k;
#pragma unroll
                    for (int u = 0; u < Frag<TX>::NV; ++u) {
                        raw[i][f].v[u] = norm_u32x4{0, 0, 0, 0};
                        if (in) raw[i][f].v[u] = reinterpret_cast<const NormVec<TX>*>(p + u * NormElem<TX>::V)->v;
                    }
                } else {
                    qn[i][f] = i32x4{0, 0, 0, 0};
                    if (row < g.m && k < g.ld) qn[i][f] = *reinterpret_cast<const i32x4*>(g.a + row * g.ld + k);
                }
            }
        }
    };
    const long long stride = (long long)gridDim.x * 8;
    long long blk = (long long)blockIdx.x * 8 + wave;
    if (AHEAD && blk < a.blocks) load(blk);
    for (; blk < a.blocks; blk += stride) {
        if constexpr (!AHEAD) load(blk);
        i32x4 q[MI][KF];
        float s[MI];
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            if constexpr (QUANT) {
                unsigned top = 0;
#pragma unroll
                for (int f = 0; f < KF; ++f)
#pragma unroll
                    for (int u = 0; u < Frag<TX>::NV; ++u) {
                        const NormArr<TX> x = raw[i][f].unpack(u);
#pragma unroll
                        for (int e = 0; e < NormElem<TX>::V; ++e) top = max_bits(top, (float)x.v[e]);
                    }
                top = max_over<16>(top, 64);  // of the four lanes that share a row
                const bool fine = top < 0x7f800000u;
                float m;
                s[i] = row_scale(top, &m);
                typename InvOf<TX, false>::type inv;
                inv.set(m, fine);
#pragma unroll
                for (int f = 0; f < KF; ++f) {
                    unsigned w[16];
#pragma unroll
                    for (int u = 0; u < Frag<TX>::NV; ++u) {
                        const NormArr<TX> x = raw[i][f].unpack(u);
#pragma unroll
                        for (int e = 0; e < NormElem<TX>::V; ++e) w[u * NormElem<TX>::V + e] = inv((float)x.v[e]);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) q[i][f][e] = pack_bytes(w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3], fine);
                }
            } else {
                s[i] = sn[i];
#pragma unroll
                for (int f = 0; f < KF; ++f) q[i][f] = qn[i][f];
            }
        }
        if (AHEAD && blk + stride < a.blocks) load(blk + stride);
        for (int c = 0; c < a.chunks; ++c) {
            i32x4 acc[MI][4];
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
#pragma unroll
            for (int f = 0; f < KF; ++f)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const i32x4 wf = *reinterpret_cast<const i32x4*>(smem + (((c * 4 + j) * KF + f) * 64 + lane) * 16);
#pragma unroll
                    for (int i = 0; i < MI; ++i) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf, q[i][f], acc[i][j], 0, 0, 0);
                }
            const int n = c * 64 + lq * 16;
            if (n < g.n) {
#pragma unroll
                for (int i = 0; i < MI; ++i) {
                    const long long row = blk * (16 * MI) + i * 16 + lr;
                    T out[16];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const f32x4 w4 = *reinterpret_cast<const f32x4*>(ws + n + 4 * j), b4 = *reinterpret_cast<const f32x4*>(bs + n + 4 * j);
                        float v[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] = (float)acc[i][j][e] * (s[i] * w4[e]) + b4[e];
                        act_n<ACT>(v, g.slope);
#pragma unroll
                        for (int e = 0; e < 4; ++e) out[4 * j + e] = (T)v[e];
                    }
                    if (row < g.m) {
                        T* p = static_cast<T*>(g.y) + row * g.y_ld + n;
#pragma unroll
                        for (int k = 0; k < 16 / SV; ++k) {
                            if (n + (k + 1) * SV <= g.n) {
                                st_out<T, SV>(p + k * SV, out + k * SV);
                            } else {
#pragma unroll
                                for (int e = 0; e < SV; ++e)
                                    if (n + k * SV + e < g.n) p[k * SV + e] = out[k * SV + e];
                            }
                        }
                    }
                }
            }
        }
    }
}

template <typename TI, typename T, int ACT, int MI, int KF>
int launch(RowsGemm a, hipStream_t st) {
    a.chunks = (a.g.n + 63) / 64;
    a.blocks = (a.g.m + 16 * MI - 1) / (16 * MI);
    const int lds = a.chunks * 64 * (KF * 64 + 8);
    static std::atomic<unsigned long long> attr_set{0};  // one bit per device: the attribute is per function and device
    const unsigned long long bit = 1ull << y5_current_device();
    if (!(attr_set.load() & bit)) {
        Y5_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(gemm_rows_kernel<TI, T, ACT, MI, KF>), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
        attr_set.fetch_or(bit);
    }
    const long long most = (long long)cu_count() * (lds <= 80 * 1024 ? 2 : 1), want = (a.blocks + 7) / 8;
    hipLaunchKernelGGL((gemm_rows_kernel<TI, T, ACT, MI, KF>), dim3((unsigned)(want < most ? want : most)), dim3(512), lds, st, a);
    Y5_LAUNCH_CHECK("gemm_rows_kernel");
    return Y5_OK;
}

template <typename TI, typename T, int ACT>
int by_width(const RowsGemm& a, hipStream_t st) {
    const int kf = (a.k + 63) / 64;
    constexpr bool wide = sizeof(TI) == 4;  // fp32 values take twice the registers
    if (kf == 1) return launch<TI, T, ACT, 2, 1>(a, st);
    if (kf == 2) return launch<TI, T, ACT, 1, 2>(a, st);
    if (kf <= 4) return launch<TI, T, ACT, 1, 4>(a, st);
    if constexpr (!wide) return launch<TI, T, ACT, 1, 8>(a, st);
    return y5_fail(Y5_EINVAL, "gemm_i8: internal: %d values a row", a.k);
}

template <typename TI, typename T>
int by_act(const RowsGemm& a, hipStream_t st) {
    if (a.g.act == Y5_ACT_LEAKY) return by_width<TI, T, Y5_ACT_LEAKY>(a, st);
    if (a.g.act == Y5_ACT_SILU) return by_width<TI, T, Y5_ACT_SILU>(a, st);
    return by_width<TI, T, Y5_ACT_NONE>(a, st);
}

}  // namespace

// quantise: the rows come in their own type
bool y5_gemm_rows_fits(int n, int k, bool quantise, int dtype) {
    const int kf = (k + 63) / 64, kp = kf == 1 ? 1 : kf == 2 ? 2 : kf <= 4 ? 4 : 8;
    if (quantise && k % 16 != 0) return false;
    return kf <= (quantise && dtype == Y5_F32 ? 4 : 8) && (n + 63) / 64 * 64 * (kp * 64 + 8) <= 144 * 1024;
}

int y5_launch_gemm_rows(const y5_gemm_i8_desc& d, const void* x, int64_t x_ld, hipStream_t st) {
    RowsGemm a{};
    a.g = make_gemm_args(d);
    a.x = x;
    a.x_ld = x_ld;
    a.k = x ? d.k : d.ld;
    if (x) {
        if (d.dtype == Y5_F16) return by_act<f16, f16>(a, st);
        if (d.dtype == Y5_BF16) return by_act<bf16, bf16>(a, st);
        return by_act<float, float>(a, st);
    }
    if (d.dtype == Y5_F16) return by_act<signed char, f16>(a, st);
    if (d.dtype == Y5_BF16) return by_act<signed char, bf16>(a, st);
    return by_act<signed char, float>(a, st);
}
