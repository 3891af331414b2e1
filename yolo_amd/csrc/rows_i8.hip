// Rows of 8-bit integers with a scale a row, from 16- or 32-bit values (y5_quantize_rows_i8) or straight from a group norm
// with its activation (y5_group_norm_rows_i8): a = max |v| of the row, scale = a / 127, q = the whole number nearest to
// 127 v / a.  Rows with a below 2^-120 (127 / a would overflow) count as zero: scale 0.  A row with an infinity or a NaN gets
// the scale NaN and zeros, so that everything computed from it is NaN.
//
// Memory bound: a value is read once, and written as one byte.  A row lives in the registers of the lanes that read it, so the
// maximum is a few moves between lanes; with the group norm the normalised value is rounded once, to 8 bits, and no 16-bit tensor in between
// is written or read.  12800 x 1024 fp16: 9 us, 16384 x 4096 bf16: 37 us (5.4 TB/s); after a group norm 204800 x 256 with silu: 37
// us for 157 MB (4.2 TB/s), bound by memory and the vector units together (a launch that keeps those busier for fewer loads - two vectors
// a lane - takes 38), behind the 30 us of gn_stats_kernel.
#include "y5_common.h"

namespace {

#include "conv_common.h"
#include "norm_rows.h"
#include "quant_rows.h"

enum { kPlain, kNormLeaky, kNormSilu };  // what happens to a value before it is quantised

struct RowsArgs {
    const void* x;
    signed char* q;
    float* scale;
    long long rows, x_ld;
    int k, q_ld;   // values of a row; bytes of a row of q (a multiple of 16; zeros behind the k-th)
    int lanes;     // lanes of a row (a power of two up to 64)
    int run;       // rows of a workgroup
    // with the group norm only
    NormShape s;
    const float2* part;
    const void *weight, *bias;
};

// V bytes of a row, from the low bytes of v
template <int V>
__device__ __forceinline__ void st_bytes(signed char* p, const unsigned (&v)[V], bool fine) {
    if constexpr (V == 8) *reinterpret_cast<uint2*>(p) = make_uint2(pack_bytes(v[0], v[1], v[2], v[3], fine), pack_bytes(v[4], v[5], v[6], v[7], fine));
    else *reinterpret_cast<int*>(p) = pack_bytes(v[0], v[1], v[2], v[3], fine);
}

// Lanes share a row: vector v of lane l covers elements ((v * lanes) + l) * V.  NV vectors a lane.
// grid: runs of `run` rows (x batch with NORM, where a workgroup's rows are pixels of one image)
// LDS with NORM: red[2 * blockDim.x], gmean, grstd[groups], A[q_ld], B[q_ld] (z = x * A + B)
template <typename T, int NORM, int NV>
__global__ __launch_bounds__(256) void rows_kernel(const RowsArgs a) {
    constexpr int V = NormElem<T>::V;
    extern __shared__ float lds[];
    const int t = threadIdx.x, TB = blockDim.x;
    const int l = t & (a.lanes - 1), sub = t / a.lanes, step = TB / a.lanes;
    long long row0 = (long long)blockIdx.x * a.run, rows = a.rows, base = 0;
    int b = 0;
    if constexpr (NORM != kPlain) {
        b = a.s.batch - 1 - blockIdx.y;  // from the end: the statistics pass read that last
        row0 = (long long)(gridDim.x - 1 - blockIdx.x) * a.run;
        rows = a.s.pixels;
        base = (long long)b * a.s.pixels;
    }
    const long long row1 = row0 + a.run < rows ? row0 + a.run : rows;
    int off[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) off[v] = (v * a.lanes + l) * V;
    norm_u32x4 raw[NV];  // the values as they are in memory
    // the row to load next and the row to store next, moved along by additions: 64-bit products of row and pitch would cost a tenth of
    // all that a row of 256 values takes
    const T* xr = static_cast<const T*>(a.x) + (base + row0 + sub) * a.x_ld;
    signed char* qr = a.q + (size_t)(base + row0 + sub) * a.q_ld;
    float* sr = a.scale + base + row0 + sub;
    const long long x_step = step * a.x_ld, q_step = (long long)step * a.q_ld;
    auto load = [&](long long row) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int n = row < row1 ? a.k - off[v] : 0;
            if (n >= V) raw[v] = reinterpret_cast<const NormVec<T>*>(xr + off[v])->v;
            else {
                NormArr<T> u;
                ld_part(xr + off[v], n, u.v);
                raw[v] = __builtin_bit_cast(norm_u32x4, u);
                asm volatile("" : "+v"(raw[v]));  // packed here: the elements would take their registers through the whole loop
            }
        }
        xr += x_step;
    };
    auto unpack = [&](int v) {  // the empty statement keeps the compiler from holding the values unpacked
        asm volatile("" : "+v"(raw[v]));
        return __builtin_bit_cast(NormArr<T>, raw[v]);
    };
    if constexpr (NORM != kPlain) load(row0 + sub);  // on its way while the statistics are merged
    // up to two vectors a lane the coefficients live in registers (from LDS they would cost eight times the bytes of the values)
    constexpr bool HELD = NORM != kPlain && NV <= 2;
    float* coef = nullptr;
    float A[HELD ? NV : 1][V], B[HELD ? NV : 1][V];
    if constexpr (NORM != kPlain) {
        const NormShape& s = a.s;
        float *red = lds, *gmean = red + 2 * TB, *grstd = gmean + s.groups;
        coef = grstd + s.groups;
        float w0[2], b0[2];  // the first parameters too
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int c = t + i * TB;
            w0[i] = c < s.c ? ld_param(a.weight, c, s.param_dtype, 1.f) : 0.f;
            b0[i] = c < s.c ? ld_param(a.bias, c, s.param_dtype, 0.f) : 0.f;
        }
        norm_merge_chunks(s, a.part, b, red, gmean, grstd);
        // mean and beta in one number: that rounds as coarsely as holding the mean in 32 bits does (its magnitude over a
        // deviation, times 2^-24), and is far below the 2^-8 of the rounding that follows wherever that mean is
        for (int c = t; c < a.q_ld; c += TB) {
            float ca = 0.f, cb = 0.f;
            if (c < s.c) {
                const int g = (int)fdiv((unsigned)c, s.by_cpg);
                const bool first = c < 2 * TB;
                ca = (first ? w0[c >= TB] : ld_param(a.weight, c, s.param_dtype, 1.f)) * grstd[g];
                cb = __builtin_fmaf(-gmean[g], ca, first ? b0[c >= TB] : ld_param(a.bias, c, s.param_dtype, 0.f));
            }
            coef[c] = ca;
            coef[a.q_ld + c] = cb;
        }
        __syncthreads();
        if constexpr (HELD) {
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    A[v][e] = off[v] < a.q_ld ? coef[off[v] + e] : 0.f;
                    B[v][e] = off[v] < a.q_ld ? coef[a.q_ld + off[v] + e] : 0.f;
                }
        }
    }
    // every lane of a wave takes every turn: a row of lanes past the end reads and writes nothing
    for (long long first = row0; first < row1; first += step) {
        const long long row = first + sub;
        if constexpr (NORM == kPlain) load(row);
        unsigned top = 0;
        float z[NORM != kPlain ? NV : 1][V];
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            float f[V];
            const NormArr<T> x = unpack(v);
#pragma unroll
            for (int e = 0; e < V; ++e) f[e] = (float)x.v[e];
            if constexpr (NORM != kPlain) {
                if (HELD || off[v] < a.q_ld) {
#pragma unroll
                    for (int e = 0; e < V; ++e) f[e] = HELD ? __builtin_fmaf(f[e], A[HELD ? v : 0][e], B[HELD ? v : 0][e]) : __builtin_fmaf(f[e], coef[off[v] + e], coef[a.q_ld + off[v] + e]);
                    norm_act<NORM == kNormSilu>(f, a.s.slope);
                }
#pragma unroll
                for (int e = 0; e < V; ++e) z[v][e] = f[e];
            }
#pragma unroll
            for (int e = 0; e < V; ++e) top = max_bits(top, f[e]);
        }
        if constexpr (NORM != kPlain) load(row + step);  // the values are in z: the next row flies under the rest
        top = max_over(top, a.lanes);
        float m;
        const float scale = row_scale(top, &m);
        typename InvOf<T, NORM != kPlain>::type inv;
        inv.set(m, top < 0x7f800000u);
        if (row < row1) {
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                if (off[v] >= a.q_ld) continue;
                unsigned w[V];
                if constexpr (NORM != kPlain) {  // raw holds the next row: not touched here, or its loads would be waited for
#pragma unroll
                    for (int e = 0; e < V; ++e) w[e] = inv(z[v][e]);
                } else {
                    const NormArr<T> x = unpack(v);
#pragma unroll
                    for (int e = 0; e < V; ++e) w[e] = inv((float)x.v[e]);
                }
                st_bytes<V>(qr + off[v], w, top < 0x7f800000u);
            }
            if (l == 0) *sr = scale;
        }
        qr += q_step;
        sr += step;
    }
}

// One workgroup a row: long rows, or few of them.  The row is read twice, the second time from the cache.
template <typename T>
__global__ __launch_bounds__(256) void long_rows_kernel(const RowsArgs a) {
    constexpr int V = NormElem<T>::V;
    __shared__ unsigned tops[4];
    const int t = threadIdx.x;
    const long long row = blockIdx.x;
    const T* xr = static_cast<const T*>(a.x) + row * a.x_ld;
    unsigned top = 0;
    for (int off = t * V; off < a.k; off += 256 * V) {
        T x[V];
        if (a.k - off >= V) ld_vec(xr + off, x);
        else ld_part(xr + off, a.k - off, x);
#pragma unroll
        for (int e = 0; e < V; ++e) top = max_bits(top, (float)x[e]);
    }
    top = max_over(top, 64);
    if ((t & 63) == 0) tops[t >> 6] = top;
    __syncthreads();
    top = tops[0];
#pragma unroll
    for (int i = 1; i < 4; ++i) top = tops[i] > top ? tops[i] : top;
    float m;
    const float scale = row_scale(top, &m);
    typename InvOf<T, false>::type inv;
    inv.set(m, top < 0x7f800000u);
    for (int off = t * V; off < a.q_ld; off += 256 * V) {
        T x[V];
        if (a.k - off >= V) ld_vec(xr + off, x);
        else ld_part(xr + off, a.k - off, x);
        unsigned w[V];
#pragma unroll
        for (int e = 0; e < V; ++e) w[e] = inv((float)x[e]);
        st_bytes<V>(a.q + (size_t)row * a.q_ld + off, w, top < 0x7f800000u);
    }
    if (t == 0) a.scale[row] = scale;
}

template <typename T>
int quantize(RowsArgs a, hipStream_t st) {
    constexpr int V = NormElem<T>::V;
    const int vecs = a.q_ld / V;
    if (vecs > 64 * 8) {  // more than a wave's registers hold
        hipLaunchKernelGGL((long_rows_kernel<T>), dim3((unsigned)a.rows), dim3(256), 0, st, a);
        Y5_LAUNCH_CHECK("long_rows_kernel");
        return Y5_OK;
    }
    a.lanes = 1;
    while (a.lanes < 64 && a.lanes < vecs) a.lanes *= 2;
    const int nv = (vecs + a.lanes - 1) / a.lanes;
    const int step = 256 / a.lanes;  // rows of a workgroup in one turn
    // four turns a workgroup, fewer where that would leave the chip empty; rows of many vectors have enough in flight in one
    int turns = nv > 2 ? 1 : 4;
    while (turns > 1 && a.rows / ((long long)step * turns) < 1024) turns /= 2;
    a.run = step * turns;
    const dim3 grid((unsigned)((a.rows + a.run - 1) / a.run));
    if (nv == 1) hipLaunchKernelGGL((rows_kernel<T, kPlain, 1>), grid, dim3(256), 0, st, a);
    else if (nv == 2) hipLaunchKernelGGL((rows_kernel<T, kPlain, 2>), grid, dim3(256), 0, st, a);
    else if (nv <= 4) hipLaunchKernelGGL((rows_kernel<T, kPlain, 4>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((rows_kernel<T, kPlain, 8>), grid, dim3(256), 0, st, a);
    Y5_LAUNCH_CHECK("rows_kernel");
    return Y5_OK;
}

template <typename T, int NORM>
int norm_rows(RowsArgs a, hipStream_t st) {
    constexpr int V = NormElem<T>::V;
    const int vecs = a.q_ld / V;
    a.lanes = 1;
    while (a.lanes < 64 && a.lanes < vecs) a.lanes *= 2;
    const int nv = (vecs + a.lanes - 1) / a.lanes;
    const int step = 256 / a.lanes;
    long long run = norm_run_bytes(a.s, (int)sizeof(T)) / ((long long)a.k * (int)sizeof(T));
    run = run < step ? step : run / step * step;
    a.run = (int)run;
    const dim3 grid((unsigned)((a.s.pixels + run - 1) / run), (unsigned)a.s.batch);
    const size_t lds = (2 * 256 + 2 * (size_t)a.s.groups + 2 * (size_t)a.q_ld) * 4;  // at most 2 + 32 + 32 KiB + 128
    auto launch = [&](auto kernel) -> int {
        if (lds > 64 << 10) Y5_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
        hipLaunchKernelGGL(kernel, grid, dim3(256), lds, st, a);
        Y5_LAUNCH_CHECK("rows_kernel");
        return Y5_OK;
    };
    if (nv == 1) return launch(rows_kernel<T, NORM, 1>);
    if (nv == 2) return launch(rows_kernel<T, NORM, 2>);
    if (nv <= 4) return launch(rows_kernel<T, NORM, 4>);
    if constexpr (V == 4) {
        if (nv > 8) return launch(rows_kernel<T, NORM, 16>);
    }
    return launch(rows_kernel<T, NORM, 8>);
}

int check_rows(const char* name, const void* q, const void* scale, int k, int q_ld) {
    Y5_REQUIRE(q && scale, "%s: null output", name);
    Y5_REQUIRE(k > 0 && k <= Y5_I8_MAX_K, "%s: %d values a row (1 to %d)", name, k, Y5_I8_MAX_K);
    Y5_REQUIRE(q_ld == (k + 15) / 16 * 16, "%s: a row of q is %d bytes for %d values (got %d)", name, (k + 15) / 16 * 16, k, q_ld);
    Y5_REQUIRE(y5_aligned16(q) && reinterpret_cast<uintptr_t>(scale) % 4 == 0, "%s: misaligned output", name);
    return Y5_OK;
}

}  // namespace

int y5_launch_quantize_rows(const void* x, int64_t x_ld, int dtype, int64_t rows, int k, void* q, int q_ld, float* scale, hipStream_t st) {
    Y5_REQUIRE(x, "quantize_rows: null x");
    Y5_REQUIRE(dtype == Y5_F16 || dtype == Y5_BF16 || dtype == Y5_F32, "quantize_rows: dtype %d", dtype);
    if (int rc = check_rows("quantize_rows", q, scale, k, q_ld)) return rc;
    Y5_REQUIRE(rows > 0 && rows <= 0x7fffffff, "quantize_rows: %lld rows", (long long)rows);
    Y5_REQUIRE(x_ld >= k, "quantize_rows: pitch %lld for %d values", (long long)x_ld, k);
    Y5_REQUIRE(reinterpret_cast<uintptr_t>(x) % norm_elem_size(dtype) == 0, "quantize_rows: misaligned x");
    RowsArgs a{};
    a.x = x;
    a.q = static_cast<signed char*>(q);
    a.scale = scale;
    a.rows = rows;
    a.x_ld = x_ld;
    a.k = k;
    a.q_ld = q_ld;
    if (dtype == Y5_F16) return quantize<f16>(a, st);
    if (dtype == Y5_BF16) return quantize<bf16>(a, st);
    return quantize<float>(a, st);
}

int y5_launch_group_norm_rows(const y5_group_norm_desc& d, void* q, int q_ld, float* scale, hipStream_t st) {
    RowsArgs a{};
    if (int rc = norm_make_shape(d, &a.s)) return rc;
    if (int rc = norm_check_pitch(d, a.s, "x", d.x, d.x_ld)) return rc;
    if (int rc = check_rows("group_norm_rows", q, scale, d.c, q_ld)) return rc;
    const size_t need = (size_t)a.s.batch * a.s.chunks * a.s.groups * sizeof(float2);
    if (!d.workspace || d.workspace_bytes < need) return y5_fail(Y5_EWORKSPACE, "group_norm_rows: workspace of %zu bytes, %zu needed", d.workspace ? d.workspace_bytes : (size_t)0, need);
    Y5_REQUIRE(y5_aligned16(d.workspace), "group_norm_rows: misaligned workspace");
    if (int rc = y5_launch_group_norm_stats(d, st)) return rc;
    a.x = d.x;
    a.q = static_cast<signed char*>(q);
    a.scale = scale;
    a.x_ld = d.x_ld;
    a.k = d.c;
    a.q_ld = q_ld;
    a.part = static_cast<const float2*>(d.workspace);
    a.weight = d.weight;
    a.bias = d.bias;
    const bool silu = d.act == Y5_ACT_SILU;
    if (d.dtype == Y5_F16) return silu ? norm_rows<f16, kNormSilu>(a, st) : norm_rows<f16, kNormLeaky>(a, st);
    if (d.dtype == Y5_BF16) return silu ? norm_rows<bf16, kNormSilu>(a, st) : norm_rows<bf16, kNormLeaky>(a, st);
    return silu ? norm_rows<float, kNormSilu>(a, st) : norm_rows<float, kNormLeaky>(a, st);
}
