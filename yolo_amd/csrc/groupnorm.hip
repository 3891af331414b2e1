// Group norm with an activation over channels-last tensors, and its gradient.
//
//   mean, var over the pixels and the cpg = C / G channels of a group of one image;  xh = (x - mean) / sqrt(var + eps)
//   z = gamma_c xh + beta_c,  y = act(z)
//   dz = dy act'(z);  dbeta_c = sum dz, dgamma_c = sum dz xh (over batch and pixels)
//   dx = (gamma_c dz - S1 / n - xh S2 / n) / sqrt(var + eps),  S1 = sum gamma dz, S2 = sum gamma dz xh over the group's n values
//
// ~10 operations a value against 4 bytes moved: memory bound at every size, so all that counts is how often a value crosses
// HBM.  Every output needs sums over the whole image, which leaves two forms:
//   resident  one workgroup owns a slice of whole groups of one image and keeps its values in registers between the sums and
//             the normalisation: every value is read once and written once, one launch.  For slices of up to 16 vectors a
//             thread.  20 x 20 x 512 fp16 in 32 groups: 7 us, latency of one chain (load, sums, squares, store);
//             4 x 40 x 40 x 256 fp32: 10 us (1.3 TB/s; 128 workgroups), its gradient 12.8.
//   split     a statistics pass over chunks of every image, then a pass that merges the chunks' statistics and normalises.
//             The second pass walks the images in the opposite order, so that what the first one read last is still in the
//             256 MB cache in front of HBM.  32 x 160 x 160 x 64 fp16 with silu: 30 us (105 MB from HBM, while the last call's result
//             is written back; 23 behind nothing of the kind) and 40 us (5.3 TB/s, read from that cache and written);
//             32 x 80 x 80 x 256 bf16 for training: 21 (5.1 TB/s) and 37, the gradient 40 (5.3 TB/s) and 51 (6.2 TB/s).  A copy
//             reaches 5.2 TB/s from HBM, 7.1 from the cache.
// One kernel for large maps would save the second read, but its workgroups would have to wait for each other, which two such
// kernels on two streams can turn into a wait for ever.
// The sums are taken in a fixed order (no atomics): the same call gives the same bits.
#include "y5_common.h"

namespace {

#include "conv_common.h"
#include "norm_rows.h"

struct GnArgs {
    NormShape s;
    const void *x, *dy, *weight, *bias;
    void *y, *dx, *dweight, *dbias;
    float *mean, *rstd;  // [batch][groups]
    float2* part;        // [batch][chunks][groups]: a chunk's statistics (forward) or its S1, S2 (backward)
    float* cpart;        // backward: [batch * chunks][2][c], a chunk's sums of dz and of dz * xh
    long long x_row, y_row, dy_row, dx_row;  // pitch of a virtual row, in elements
    long long x_img, y_img, dy_img, dx_img;  // of an image
    int past;  // y or dx is stored past the cache in front of HBM
};

// tot[j * N + i] = sum of v[i] over the threads of column j, in a fixed order.  part: blockDim.x * N floats of LDS.
template <int N>
__device__ __forceinline__ void col_sum(float (&v)[N], int j, int r, int RT, int cols, float* part, float* tot) {
    const int t = threadIdx.x, T = blockDim.x, E = cols * N;
    int rows;
    if (cols < 64 && (cols & (cols - 1)) == 0) {  // a wave holds 64 / cols rows of every column: they meet in registers
        for (int off = 32; off >= cols; off >>= 1) {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] += __shfl_xor(v[i], off);
        }
        const int lane = t & 63;
        if (lane < cols) {
#pragma unroll
            for (int i = 0; i < N; ++i) part[(t >> 6) * E + lane * N + i] = v[i];
        }
        rows = T >> 6;
    } else {
        if (r < RT) {
#pragma unroll
            for (int i = 0; i < N; ++i) part[r * E + j * N + i] = v[i];
        }
        rows = RT;
    }
    __syncthreads();
    for (int i = t; i < E; i += T) {
        float a = 0.f;
#pragma unroll 8
        for (int k = 0; k < rows; ++k) a += part[k * E + i];
        tot[i] = a;
    }
    __syncthreads();
}

// f(g, sums) for G groups, sums = the sums over the group's entries of at(entry), two at a time: entries rep * rep_pitch + g * n + i for
// rep < reps, i < n.  A thread a group, or a wave where a group has many entries:
// for the resident kernels, whose values leave few registers (the other form makes 300 x 20 x 20 x 75 fp16 41 us instead of 36).
template <typename At, typename F>
__device__ __forceinline__ void group_sum2(int G, int n, int reps, int rep_pitch, At at, F f) {
    const int t = threadIdx.x, T = blockDim.x;
    if (n * reps <= 32) {
        for (int g = t; g < G; g += T) {
            float2 a = make_float2(0.f, 0.f);
            for (int k = 0; k < reps; ++k)
                for (int i = 0; i < n; ++i) {
                    const float2 v = at(k * rep_pitch + g * n + i);
                    a.x += v.x;
                    a.y += v.y;
                }
            f(g, a);
        }
    } else {
        const int lane = t & 63;
        for (int g = t >> 6; g < G; g += T >> 6) {
            float2 a = make_float2(0.f, 0.f);
            for (int k = 0; k < reps; ++k)
                for (int i = lane; i < n; i += 64) {
                    const float2 v = at(k * rep_pitch + g * n + i);
                    a.x += v.x;
                    a.y += v.y;
                }
            for (int off = 32; off; off >>= 1) {
                a.x += __shfl_xor(a.x, off);
                a.y += __shfl_xor(a.y, off);
            }
            if (lane == 0) f(g, a);
        }
    }
    __syncthreads();
}

// The same with as many lanes a group as keep every thread at work, with four entries each or more (statistics of 64 x 20 x 20 x 255 in 51
// groups 27 -> 14 us, in 15 groups 17 -> 15)
template <typename At, typename F>
__device__ __forceinline__ void group_sum2_split(int G, int n, int reps, int rep_pitch, At at, F f) {
    const int t = threadIdx.x, T = blockDim.x, entries = n * reps;
    int lanes = 1;
    while (lanes < 64 && 2 * lanes * G <= T && 8 * lanes <= entries) lanes *= 2;
    const int l = t & (lanes - 1), step = T / lanes;
    for (int g0 = 0; g0 < G; g0 += step) {  // every lane takes every turn: they add up across lanes
        const int g = g0 + t / lanes;
        float2 a = make_float2(0.f, 0.f);
        if (g < G) {
#pragma unroll 4
            for (int e = l; e < entries; e += lanes) {
                const int k = reps == 1 ? 0 : e / n;
                const float2 v = at(k * rep_pitch + g * n + e - k * n);
                a.x += v.x;
                a.y += v.y;
            }
        }
        for (int off = lanes >> 1; off; off >>= 1) {
            a.x += __shfl_xor(a.x, off);
            a.y += __shfl_xor(a.y, off);
        }
        if (l == 0 && g < G) f(g, a);
    }
    __syncthreads();
}

// How the elements of a vector lie to groups and rows: all of one group; each of a group of its own (a group is no multiple of a
// vector); each of a group of its own in virtual rows of several pixels, the last of which may be cut short
enum { kUniform, kMixed, kCut };

// The vector column a thread owns: element offset in the virtual row, channels, groups and parameters of its elements.
template <typename T, int M>
struct Column {
    static constexpr int V = NormElem<T>::V, NG = M ? V : 1;
    int off;      // element offset of the vector in the virtual row
    int ch0;      // channel of its first element
    int grp[NG];  // group of each element
    __device__ __forceinline__ void init(const NormShape& s, int col) {
        off = col * V;
        ch0 = M == kCut ? mod_c(s, off) : off;
        if (M) {
#pragma unroll
            for (int e = 0; e < V; ++e) grp[e] = (int)fdiv((unsigned)channel(s, e), s.by_cpg);
        } else {
            grp[0] = (int)fdiv((unsigned)off, s.by_cpg);
        }
    }
    __device__ __forceinline__ int channel(const NormShape& s, int e) const {
        const int c = ch0 + e;  // below s.c + V: a virtual row of narrow pixels may hold several of them in one vector
        return M == kCut ? mod_c(s, c) : c;
    }
    static __device__ __forceinline__ int mod_c(const NormShape& s, int i) { return i - (int)fdiv((unsigned)i, s.by_c) * s.c; }
    // a parameter vector's values for the elements
    __device__ __forceinline__ void params(const NormShape& s, const void* p, float def, float (&v)[V]) const {
        if constexpr (M == kCut) {
            if (!p || s.param_dtype == Y5_F32) {
#pragma unroll
                for (int e = 0; e < V; ++e) v[e] = p ? static_cast<const float*>(p)[channel(s, e)] : def;
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const unsigned short b = static_cast<const unsigned short*>(p)[channel(s, e)];
                    v[e] = s.param_dtype == Y5_F16 ? (float)__builtin_bit_cast(f16, b) : __uint_as_float((unsigned)b << 16);
                }
            }
        } else {
            ld_params(p, ch0, s.param_dtype, def, v);
        }
    }
    // elements of the vector that virtual row `row` has
    __device__ __forceinline__ int valid(const NormShape& s, int row) const {
        if (M != kCut) return V;
        const long long left = (long long)s.pixels * s.c - ((long long)row * s.W + off);
        return left >= V ? V : left > 0 ? (int)left : 0;
    }
};

// The rows of a resident slice that a thread holds: r, r + RT, ... below `limit` as whole vectors, and `tail` elements of the last row
// where that is cut short within the thread's vector.  One piece of code for the one vector that may be cut: in every turn of the
// unrolled loops it would be most of the kernel, and a small map's time is that of fetching it.
template <typename T, int M>
struct Held {
    bool active;
    int limit, tail;
    __device__ __forceinline__ void init(const NormShape& s, const Column<T, M>& col, int r, int RT) {
        active = r < RT;
        limit = s.vrows;
        tail = 0;
        if constexpr (M == kCut) {
            const int last = s.vrows - 1, nv = col.valid(s, last);
            if (nv < NormElem<T>::V) {
                limit = last;
                if (active && last % RT == r) tail = nv;
            }
        }
    }
    __device__ __forceinline__ bool has(int row) const { return active && row < limit; }
};

// A vector of T as the 16 bytes it is in memory: what is kept across a barrier stays packed.
typedef norm_u32x4 Raw;
template <typename T, int M>
__device__ __forceinline__ Raw ld_col(const T* p, int nv) {
    if (M != kCut || nv >= NormElem<T>::V) return reinterpret_cast<const NormVec<T>*>(p)->v;
    NormArr<T> u;
    ld_part(p, nv, u.v);
    return __builtin_bit_cast(Raw, u);
}
// its elements; the empty statement keeps the compiler from unpacking it where it was loaded, or once for every use
template <typename T>
__device__ __forceinline__ NormArr<T> unpack(Raw& r) {
    asm volatile("" : "+v"(r));
    return __builtin_bit_cast(NormArr<T>, r);
}
template <typename T, int M>
__device__ __forceinline__ void st_col(T* p, int nv, const Raw& r, int past) {
    if (M != kCut || nv >= NormElem<T>::V) {
        if (past) {
            asm volatile("" ::: "memory");  // keeps the compiler from making one store of the two
            __builtin_nontemporal_store(r, &reinterpret_cast<NormVec<T>*>(p)->v);
            asm volatile("" ::: "memory");
        } else {
            reinterpret_cast<NormVec<T>*>(p)->v = r;
        }
    } else st_part(p, nv, __builtin_bit_cast(NormArr<T>, r).v);
}

// z = act(gamma (x - mean) rstd + beta) of one vector, rounded once
template <typename T, bool SILU, int NG>
__device__ __forceinline__ Raw normalise(Raw& raw, const float (&mean)[NG], const float (&A)[NormElem<T>::V], const float (&B)[NormElem<T>::V],
                                         float slope) {
    constexpr int V = NormElem<T>::V;
    const NormArr<T> in = unpack<T>(raw);
    NormArr<T> out;
    float z[V];
#pragma unroll
    for (int e = 0; e < V; ++e) z[e] = __builtin_fmaf((float)in.v[e] - mean[NG == 1 ? 0 : e], A[e], B[e]);
    norm_act<SILU>(z, slope);
#pragma unroll
    for (int e = 0; e < V; ++e) out.v[e] = (T)z[e];
    return __builtin_bit_cast(Raw, out);
}

// ------------------------------------------------------------------------------------------ forward, resident

// grid: slices * batch.  LDS: part[blockDim.x * NG], tot[cols * NG], gs[2 * groups of the slice]
template <typename T, int M, bool SILU, int R>
__global__ __launch_bounds__(R > 8 ? 1024 : R > 4 ? 512 : 256, 4) void gn_resident_kernel(const GnArgs a, const FastDiv by_cols, int slices) {
    constexpr int V = NormElem<T>::V, NG = M ? V : 1;
    extern __shared__ float lds[];
    const NormShape& s = a.s;
    // slices of an image share cache lines: neighbours run on one XCD, behind one L2
    const int at = xcd_remap(blockIdx.x, gridDim.x), b = at / slices, slice = at - b * slices;
    const int t = threadIdx.x, TB = blockDim.x, cols = (int)by_cols.d;
    const int RT = (int)fdiv((unsigned)TB, by_cols), r = (int)fdiv((unsigned)t, by_cols), j = t - r * cols;
    const bool active = r < RT;
    float *part = lds, *tot = part + TB * NG, *gs = tot + cols * NG;
    Column<T, M> col;
    col.init(s, slice * cols + j);
    const int g0 = (int)fdiv(slice * cols * V, s.by_cpg);  // first group of the slice (a slice holds whole groups)
    const int G = M == kCut ? s.groups : (int)fdiv(cols * V, s.by_cpg);  // its groups
    const int gn = M ? s.cpg : s.cpg / V;                        // entries of a group in tot
    const T* xb = static_cast<const T*>(a.x) + (size_t)b * a.x_img + col.off;
    Raw raw[R];
    Held<T, M> held;
    held.init(s, col, r, RT);
#pragma unroll
    for (int i = 0; i < R; ++i)
        if (held.has(r + i * RT)) raw[i] = ld_col<T, M>(xb + (size_t)(r + i * RT) * a.x_row, V);
    Raw cut = {0, 0, 0, 0};
    if (held.tail) cut = ld_col<T, M>(xb + (size_t)held.limit * a.x_row, held.tail);
    float A[V], B[V];  // gamma (times 1 / deviation, later) and beta: on their way with the values
    col.params(s, a.weight, 1.f, A);
    col.params(s, a.bias, 0.f, B);
    float acc[NG];
#pragma unroll
    for (int e = 0; e < NG; ++e) acc[e] = 0.f;
#pragma unroll
    for (int i = 0; i < R; ++i)
        if (held.has(r + i * RT)) {
            const NormArr<T> x = unpack<T>(raw[i]);
#pragma unroll
            for (int e = 0; e < V; ++e) acc[M ? e : 0] += (float)x.v[e];
        }
    if constexpr (M == kCut) {
        const NormArr<T> x = unpack<T>(cut);
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] += (float)x.v[e];
    }
    const float inv_n = 1.f / ((float)s.pixels * (float)s.cpg);
    col_sum<NG>(acc, j, r, RT, cols, part, tot);
    group_sum2(G, gn, s.k, s.c, [&](int i) { return make_float2(tot[i], 0.f); }, [&](int g, float2 v) { gs[2 * g] = v.x * inv_n; });
    float mean[NG];
#pragma unroll
    for (int e = 0; e < NG; ++e) {
        mean[e] = active ? gs[2 * (col.grp[e] - g0)] : 0.f;
        acc[e] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < R; ++i)
        if (held.has(r + i * RT)) {
            const NormArr<T> x = unpack<T>(raw[i]);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float d = (float)x.v[e] - mean[M ? e : 0];
                acc[M ? e : 0] = __builtin_fmaf(d, d, acc[M ? e : 0]);
            }
        }
    if constexpr (M == kCut) {
        const NormArr<T> x = unpack<T>(cut);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float d = (float)x.v[e] - mean[e];
            if (e < held.tail) acc[e] = __builtin_fmaf(d, d, acc[e]);
        }
    }
    col_sum<NG>(acc, j, r, RT, cols, part, tot);
    group_sum2(G, gn, s.k, s.c, [&](int i) { return make_float2(tot[i], 0.f); }, [&](int g, float2 v) { gs[2 * g + 1] = 1.f / sqrtf(v.x * inv_n + s.eps); });
    if (a.mean) {
        for (int g = t; g < G; g += TB) {
            a.mean[(size_t)b * s.groups + g0 + g] = gs[2 * g];
            a.rstd[(size_t)b * s.groups + g0 + g] = gs[2 * g + 1];
        }
    }
    if (!active) return;
#pragma unroll
    for (int e = 0; e < V; ++e) A[e] *= gs[2 * (col.grp[M ? e : 0] - g0) + 1];
    T* yb = static_cast<T*>(a.y) + (size_t)b * a.y_img + col.off;
#pragma unroll
    for (int i = 0; i < R; ++i)
        if (held.has(r + i * RT)) st_col<T, M>(yb + (size_t)(r + i * RT) * a.y_row, V, normalise<T, SILU, NG>(raw[i], mean, A, B, s.slope), a.past);
    if (held.tail) st_col<T, M>(yb + (size_t)held.limit * a.y_row, held.tail, normalise<T, SILU, NG>(cut, mean, A, B, s.slope), a.past);
}

// ------------------------------------------------------------------------------------------ forward, split

// grid (chunks, batch): (mean, M2) of every group over the chunk.  Bound by HBM; four loads of 16 bytes in flight a thread and 6 to 8
// waves a SIMD hide its latency.  A thread sums differences from the first value it reads (K):
// where a map's mean is many deviations from zero, sum and sum of squares of the raw values would cancel.  The threads' means and
// squares then meet as differences from one thread's mean of each group.
template <typename T, int M>
__global__ __launch_bounds__(1024, sizeof(T) == 4 || M == kUniform ? 8 : 6) void gn_stats_kernel(const GnArgs a) {
    constexpr int V = NormElem<T>::V, NG = M ? V : 1, NA = M ? V : 4;
    extern __shared__ float lds[];
    const NormShape& s = a.s;
    const int t = threadIdx.x, TB = blockDim.x, b = blockIdx.y, cols = s.cols;
    const int RT = (int)fdiv((unsigned)TB, s.by_cols), r = (int)fdiv((unsigned)t, s.by_cols), j = t - r * cols;
    const bool active = r < RT;
    float *part = lds, *tot = part + TB * 2 * NG, *gs = tot + cols * 2 * NG;
    Column<T, M> col;
    col.init(s, j);
    const int row0 = blockIdx.x * s.chunk_rows;
    const int row1 = row0 + s.chunk_rows < s.vrows ? row0 + s.chunk_rows : s.vrows;
    const T* xb = static_cast<const T*>(a.x) + (size_t)b * a.x_img + col.off;
    float K[NG], S[NA], Q[NA], n[NG];
#pragma unroll
    for (int e = 0; e < NA; ++e) S[e] = Q[e] = 0.f;
#pragma unroll
    for (int e = 0; e < NG; ++e) K[e] = n[e] = 0.f;
    if (active && row0 + r < row1) {
        int row = row0 + r;
        {
            Raw raw = ld_col<T, M>(xb + (size_t)row * a.x_row, col.valid(s, row));
            const NormArr<T> v = unpack<T>(raw);
#pragma unroll
            for (int e = 0; e < NG; ++e) K[e] = (float)v.v[e];
        }
        auto take = [&](Raw& raw, int nv) {
            const NormArr<T> v = unpack<T>(raw);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float d = (float)v.v[e] - K[M ? e : 0];
                if (M != kCut || e < nv) {
                    S[e % NA] += d;
                    Q[e % NA] = __builtin_fmaf(d, d, Q[e % NA]);
                    if (M == kCut) n[e] += 1.f;
                }
            }
        };
        const long long step = (long long)RT * a.x_row;
        const T* p = xb + (size_t)row * a.x_row;
        // four loads in flight; the last row of an image may be cut short and is left to the loop behind
        for (; row + 3 * RT < row1 - (M == kCut ? 1 : 0); row += 4 * RT, p += 4 * step) {
            Raw v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) v[u] = ld_col<T, M>(p + u * step, V);
#pragma unroll
            for (int u = 0; u < 4; ++u) take(v[u], V);
        }
        for (; row < row1; row += RT, p += step) {
            const int nv = col.valid(s, row);
            Raw v = ld_col<T, M>(p, nv);
            take(v, nv);
        }
        if (M != kCut) {
            const float rows = (float)((row1 - 1 - row0 - r) / RT + 1);
#pragma unroll
            for (int e = 0; e < NG; ++e) n[e] = M ? rows : rows * V;
        }
    }
    float m[NG], q[NG];
#pragma unroll
    for (int e = 0; e < NG; ++e) {
        const float sum = M ? S[e] : (S[0] + S[1]) + (S[2] + S[3]), sq = M ? Q[e] : (Q[0] + Q[1]) + (Q[2] + Q[3]);
        const float d = n[e] > 0.f ? sum / n[e] : 0.f;
        m[e] = K[e] + d;
        q[e] = sq - sum * d;
    }
    // the reference of a group: the mean that the first row's thread of its first element has (element g * cpg of a chunk's first
    // virtual row is always there)
    const int G = s.groups, gn = M ? s.cpg : s.cpg / V;
    if (r == 0) {
#pragma unroll
        for (int e = 0; e < NG; ++e)
            if (col.off + e < s.c && col.grp[e] * s.cpg == col.off + e) gs[col.grp[e]] = m[e];
    }
    __syncthreads();
    float acc[2 * NG];
#pragma unroll
    for (int e = 0; e < NG; ++e) {
        const float d = m[e] - gs[col.grp[e]];
        acc[2 * e] = n[e] > 0.f ? n[e] * d : 0.f;
        acc[2 * e + 1] = n[e] > 0.f ? __builtin_fmaf(n[e] * d, d, q[e]) : 0.f;
    }
    col_sum<2 * NG>(acc, j, r, RT, cols, part, tot);
    float2* out = a.part + ((size_t)b * s.chunks + blockIdx.x) * s.groups;
    const float N = (float)norm_chunk_pixels(s, blockIdx.x) * (float)s.cpg;
    group_sum2_split(G, gn, s.k, s.c, [&](int i) { return make_float2(tot[2 * i], tot[2 * i + 1]); }, [&](int g, float2 v) {
        const float d = v.x / N;
        out[g] = make_float2(gs[g] + d, v.y - v.x * d);
    });
}

// grid (runs of rows, batch), walked from the end.  Bound by the cache's reads and HBM's writes, with silu almost as much by the vector
// units (busy for 23 of the 40 us that 52 million values take; the gradient below: 35 of 51).  A thread's first rows are on their way while the chunks' statistics are merged.
template <typename T, int M, bool SILU>
__global__ __launch_bounds__(1024, 6) void gn_apply_kernel(const GnArgs a, int run_rows) {
    constexpr int V = NormElem<T>::V, NG = M ? V : 1, U = 4;
    extern __shared__ float lds[];
    const NormShape& s = a.s;
    const int t = threadIdx.x, TB = blockDim.x, cols = s.cols;
    const int b = s.batch - 1 - blockIdx.y, run = gridDim.x - 1 - blockIdx.x;
    const int RT = (int)fdiv((unsigned)TB, s.by_cols), r = (int)fdiv((unsigned)t, s.by_cols), j = t - r * cols;
    float *red = lds, *gmean = red + 2 * TB, *grstd = gmean + s.groups;
    Column<T, M> col;
    col.init(s, j);
    const int row0 = run * run_rows + r;
    const int row1 = r < RT ? (run * run_rows + run_rows < s.vrows ? run * run_rows + run_rows : s.vrows) : 0;
    const T* xb = static_cast<const T*>(a.x) + (size_t)b * a.x_img + col.off;
    T* yb = static_cast<T*>(a.y) + (size_t)b * a.y_img + col.off;
    Raw v[U];
    auto load = [&](int row) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (row + u * RT < row1) v[u] = ld_col<T, M>(xb + (size_t)(row + u * RT) * a.x_row, col.valid(s, row + u * RT));
    };
    load(row0);
    float mean[NG], A[V], B[V];
    col.params(s, a.weight, 1.f, A);
    col.params(s, a.bias, 0.f, B);
    norm_merge_chunks(s, a.part, b, red, gmean, grstd);
    if (a.mean && run == 0) {
        for (int g = t; g < s.groups; g += TB) {
            a.mean[(size_t)b * s.groups + g] = gmean[g];
            a.rstd[(size_t)b * s.groups + g] = grstd[g];
        }
    }
#pragma unroll
    for (int e = 0; e < NG; ++e) mean[e] = gmean[col.grp[e]];
#pragma unroll
    for (int e = 0; e < V; ++e) A[e] *= grstd[col.grp[M ? e : 0]];
    for (int row = row0; row < row1; row += U * RT) {
        Raw o[U];
#pragma unroll
        for (int u = 0; u < U; ++u) o[u] = normalise<T, SILU, NG>(v[u], mean, A, B, s.slope);
        load(row + U * RT);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (row + u * RT < row1) st_col<T, M>(yb + (size_t)(row + u * RT) * a.y_row, col.valid(s, row + u * RT), o[u], a.past);
    }
}

// ------------------------------------------------------------------------------------------ backward

// Parameters of a thread's column for the gradient: mean, rstd of its groups, gamma and beta of its channels
template <typename T, int M>
struct GradColumn : Column<T, M> {
    static constexpr int V = NormElem<T>::V, NG = M ? V : 1;
    float mean[NG], rstd[NG], gamma[V], beta[V];
    __device__ __forceinline__ void load(const GnArgs& a, int b, int col) {
        const NormShape& s = a.s;
        this->init(s, col);
#pragma unroll
        for (int e = 0; e < NG; ++e) {
            mean[e] = a.mean[(size_t)b * s.groups + this->grp[e]];
            rstd[e] = a.rstd[(size_t)b * s.groups + this->grp[e]];
        }
        this->params(s, a.weight, 1.f, gamma);
        this->params(s, a.bias, 0.f, beta);
    }
    // xh and dz of one vector
    template <bool SILU>
    __device__ __forceinline__ void local(Raw& rx, Raw& rd, float (&xh)[V], float (&dz)[V], float slope) const {
        const NormArr<T> x = unpack<T>(rx), dy = unpack<T>(rd);
        float z[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            xh[e] = ((float)x.v[e] - mean[M ? e : 0]) * rstd[M ? e : 0];
            z[e] = __builtin_fmaf(xh[e], gamma[e], beta[e]);
            dz[e] = (float)dy.v[e];
        }
        norm_act_grad<SILU>(dz, z, slope);
    }
    // dx of one vector from s1 = S1 / n and s2 = S2 / n of its groups
    __device__ __forceinline__ Raw grad(const float (&xh)[V], const float (&dz)[V], const float (&s1)[NG], const float (&s2)[NG]) const {
#pragma clang fp contract(off)  // a group of one value has gamma dz = S1 exactly and a gradient of exactly zero
        NormArr<T> dx;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float w = gamma[e] * dz[e];
            const float u = w - s1[M ? e : 0];
            const float v = xh[e] * s2[M ? e : 0];
            dx.v[e] = (T)(rstd[M ? e : 0] * (u - v));
        }
        return __builtin_bit_cast(Raw, dx);
    }
};

// The per-element column sums tot[col][2][V] (dz, dz * xh) of cols * V elements from channel c0 on: per channel to `out`
// ([2][c]), and gs[2 g], gs[2 g + 1] = S1, S2 of the G groups (times scale)
template <int V>
__device__ __forceinline__ void grad_sums(const GnArgs& a, const float* tot, int c0, int channels, int G, float scale, float* out, float* gs) {
    const NormShape& s = a.s;
    auto at = [&](int el, int which) { return tot[(el / V) * 2 * V + which * V + el % V]; };
    for (int i = threadIdx.x; i < 2 * channels; i += blockDim.x) {
        const int which = i >= channels, c = i - which * channels;
        float v = 0.f;
        for (int k = 0; k < s.k; ++k) v += at(k * s.c + c, which);
        out[(size_t)which * s.c + c0 + c] = v;
    }
    group_sum2_split(G, s.cpg, s.k, s.c,
               [&](int i) {
                   const float w = ld_param(a.weight, c0 + i - (int)fdiv((unsigned)i, s.by_c) * s.c, s.param_dtype, 1.f);
                   return make_float2(w * at(i, 0), w * at(i, 1));
               },
               [&](int g, float2 v) {
                   gs[2 * g] = v.x * scale;
                   gs[2 * g + 1] = v.y * scale;
               });
}

// Gradient of a resident slice: x and dy stay in registers, xh and dz are computed twice from them (cheaper than the registers they would
// take).  grid: slices * batch; LDS: part[blockDim.x * 2 V], tot[cols * 2 V], gs[2 * groups of the slice]
template <typename T, int M, bool SILU, int R>
__global__ __launch_bounds__(R > 2 ? 512 : 256, sizeof(T) == 2 && (R > 4 || M == kCut) ? 3 : 4) void gn_bwd_resident_kernel(const GnArgs a, const FastDiv by_cols, int slices) {
    constexpr int V = NormElem<T>::V, NG = M ? V : 1;
    extern __shared__ float lds[];
    const NormShape& s = a.s;
    // slices of an image share cache lines: neighbours run on one XCD, behind one L2
    const int at = xcd_remap(blockIdx.x, gridDim.x), b = at / slices, slice = at - b * slices;
    const int t = threadIdx.x, TB = blockDim.x, cols = (int)by_cols.d;
    const int RT = (int)fdiv((unsigned)TB, by_cols), r = (int)fdiv((unsigned)t, by_cols), j = t - r * cols;
    const bool active = r < RT;
    float *part = lds, *tot = part + TB * 2 * V, *gs = tot + cols * 2 * V;
    GradColumn<T, M> col;
    col.load(a, b, slice * cols + j);
    const T* xb = static_cast<const T*>(a.x) + (size_t)b * a.x_img + col.off;
    const T* db = static_cast<const T*>(a.dy) + (size_t)b * a.dy_img + col.off;
    Raw rx[R], rd[R];
    Held<T, M> held;
    held.init(s, col, r, RT);
#pragma unroll
    for (int i = 0; i < R; ++i) {
        if (held.has(r + i * RT)) {
            rx[i] = ld_col<T, M>(xb + (size_t)(r + i * RT) * a.x_row, V);
            rd[i] = ld_col<T, M>(db + (size_t)(r + i * RT) * a.dy_row, V);
        }
    }
    Raw cx = {0, 0, 0, 0}, cd = {0, 0, 0, 0};
    if (held.tail) {
        cx = ld_col<T, M>(xb + (size_t)held.limit * a.x_row, held.tail);
        cd = ld_col<T, M>(db + (size_t)held.limit * a.dy_row, held.tail);
    }
    float acc[2 * V];
#pragma unroll
    for (int e = 0; e < 2 * V; ++e) acc[e] = 0.f;
#pragma unroll
    for (int i = 0; i < R; ++i)
        if (held.has(r + i * RT)) {
            float xh[V], dz[V];
            col.template local<SILU>(rx[i], rd[i], xh, dz, s.slope);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                acc[e] += dz[e];
                acc[V + e] = __builtin_fmaf(dz[e], xh[e], acc[V + e]);
            }
        }
    if (held.tail) {
        float xh[V], dz[V];
        col.template local<SILU>(cx, cd, xh, dz, s.slope);
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (e < held.tail) {
                acc[e] += dz[e];
                acc[V + e] = __builtin_fmaf(dz[e], xh[e], acc[V + e]);
            }
    }
    col_sum<2 * V>(acc, j, r, RT, cols, part, tot);
    const int c0 = s.k > 1 ? 0 : slice * cols * V, channels = s.k > 1 ? s.c : cols * V;
    const int g0 = (int)fdiv(c0, s.by_cpg), G = (int)fdiv(channels, s.by_cpg);
    grad_sums<V>(a, tot, c0, channels, G, 1.f / ((float)s.pixels * (float)s.cpg), a.cpart + (size_t)b * 2 * s.c, gs);
    if (!active || !a.dx) return;
    float s1[NG], s2[NG];
#pragma unroll
    for (int e = 0; e < NG; ++e) {
        s1[e] = gs[2 * (col.grp[e] - g0)];
        s2[e] = gs[2 * (col.grp[e] - g0) + 1];
    }
    T* ob = static_cast<T*>(a.dx) + (size_t)b * a.dx_img + col.off;
#pragma unroll
    for (int i = 0; i < R; ++i)
        if (held.has(r + i * RT)) {
            float xh[V], dz[V];
            col.template local<SILU>(rx[i], rd[i], xh, dz, s.slope);
            st_col<T, M>(ob + (size_t)(r + i * RT) * a.dx_row, V, col.grad(xh, dz, s1, s2), a.past);
        }
    if (held.tail) {
        float xh[V], dz[V];
        col.template local<SILU>(cx, cd, xh, dz, s.slope);
        st_col<T, M>(ob + (size_t)held.limit * a.dx_row, held.tail, col.grad(xh, dz, s1, s2), a.past);
    }
}

// S1, S2 and the channels' sums of a chunk: x and dy read once, bound by HBM (210 MB: 40 us, 5.3 TB/s).
// grid (chunks, batch); LDS as above for all groups
template <typename T, int M, bool SILU>
__global__ __launch_bounds__(1024, M == kUniform || sizeof(T) == 4 ? 5 : 4) void gn_bwd_stats_kernel(const GnArgs a) {
    constexpr int V = NormElem<T>::V;
    extern __shared__ float lds[];
    const NormShape& s = a.s;
    const int t = threadIdx.x, TB = blockDim.x, b = blockIdx.y, cols = s.cols;
    const int RT = (int)fdiv((unsigned)TB, s.by_cols), r = (int)fdiv((unsigned)t, s.by_cols), j = t - r * cols;
    float *part = lds, *tot = part + TB * 2 * V, *gs = tot + cols * 2 * V;
    GradColumn<T, M> col;
    col.load(a, b, j);
    float acc[2 * V];
#pragma unroll
    for (int e = 0; e < 2 * V; ++e) acc[e] = 0.f;
    const int row0 = blockIdx.x * s.chunk_rows;
    const int row1 = row0 + s.chunk_rows < s.vrows ? row0 + s.chunk_rows : s.vrows;
    if (r < RT) {
        const T* xb = static_cast<const T*>(a.x) + (size_t)b * a.x_img + col.off;
        const T* db = static_cast<const T*>(a.dy) + (size_t)b * a.dy_img + col.off;
        auto take = [&](Raw& x, Raw& d, int nv) {
            float xh[V], dz[V];
            col.template local<SILU>(x, d, xh, dz, s.slope);
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (M != kCut || e < nv) {
                    acc[e] += dz[e];
                    acc[V + e] = __builtin_fmaf(dz[e], xh[e], acc[V + e]);
                }
        };
        int row = row0 + r;
        for (; row + RT < row1 - (M == kCut ? 1 : 0); row += 2 * RT) {
            Raw x[2], d[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                x[u] = ld_col<T, M>(xb + (size_t)(row + u * RT) * a.x_row, V);
                d[u] = ld_col<T, M>(db + (size_t)(row + u * RT) * a.dy_row, V);
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) take(x[u], d[u], V);
        }
        for (; row < row1; row += RT) {
            const int nv = col.valid(s, row);
            Raw x = ld_col<T, M>(xb + (size_t)row * a.x_row, nv), d = ld_col<T, M>(db + (size_t)row * a.dy_row, nv);
            take(x, d, nv);
        }
    }
    col_sum<2 * V>(acc, j, r, RT, cols, part, tot);
    const size_t at = (size_t)b * s.chunks + blockIdx.x;
    grad_sums<V>(a, tot, 0, s.c, s.groups, 1.f / ((float)s.pixels * (float)s.cpg), a.cpart + at * 2 * s.c, gs);
    for (int g = t; g < s.groups; g += TB) a.part[at * s.groups + g] = make_float2(gs[2 * g], gs[2 * g + 1]);
}

// dbeta_c and dgamma_c, in a fixed order (4 us as a launch of its own, of which 2 are the launch): the rows of cpart ([rows][2][c]) added up, 16 of the 2 c columns by T threads.  red: T floats of LDS.
__device__ __forceinline__ void sum_params(const float* __restrict__ cpart, int rows, int c, int dt, void* dweight, void* dbias, int block, float* red) {
    const int T = blockDim.x / 16 * 16, t = threadIdx.x;
    const int lc = t & 15, q = t >> 4, Q = T >> 4;
    const int i = block * 16 + lc;
    float v = 0.f;
    if (t < T && i < 2 * c) {
#pragma unroll 8
        for (int k = q; k < rows; k += Q) v += cpart[(size_t)k * 2 * c + i];
    }
    if (t < T) red[q * 16 + lc] = v;
    __syncthreads();
    if (q || i >= 2 * c) return;
    for (int k = 1; k < Q; ++k) v += red[k * 16 + lc];
    if (i < c) {
        if (dbias) st_param(dbias, i, dt, v);
    } else if (dweight) {
        st_param(dweight, i - c, dt, v);
    }
}
__global__ __launch_bounds__(256) void gn_dparam_kernel(const float* __restrict__ cpart, int rows, int c, int dt, void* dweight, void* dbias) {
    __shared__ float red[256];
    sum_params(cpart, rows, c, dt, dweight, dbias, blockIdx.x, red);
}

// grid (param_blocks + runs of rows * batch): the first workgroups add up the parameters' gradients, beside the others' work on dx, which
// walk the images from the end.  LDS: red[2 * blockDim.x], gs[2 * groups]
template <typename T, int M, bool SILU>
__global__ __launch_bounds__(1024, M == kUniform || sizeof(T) == 4 ? 5 : 4) void gn_bwd_apply_kernel(const GnArgs a, int run_rows, int runs, int param_blocks) {
    constexpr int V = NormElem<T>::V, NG = M ? V : 1, U = 2;
    extern __shared__ float lds[];
    const NormShape& s = a.s;
    const int t = threadIdx.x, TB = blockDim.x, cols = s.cols;
    float *red = lds, *gs = lds + 2 * TB;
    if ((int)blockIdx.x < param_blocks) {
        sum_params(a.cpart, s.batch * s.chunks, s.c, s.param_dtype, a.dweight, a.dbias, blockIdx.x, red);
        return;
    }
    const int at = gridDim.x - 1 - blockIdx.x;
    const int b = at / runs, run = at - b * runs;
    const int RT = (int)fdiv((unsigned)TB, s.by_cols), r = (int)fdiv((unsigned)t, s.by_cols), j = t - r * cols;
    GradColumn<T, M> col;
    col.load(a, b, j);
    const T* xb = static_cast<const T*>(a.x) + (size_t)b * a.x_img + col.off;
    const T* db = static_cast<const T*>(a.dy) + (size_t)b * a.dy_img + col.off;
    T* ob = static_cast<T*>(a.dx) + (size_t)b * a.dx_img + col.off;
    const int row0 = run * run_rows + r;
    const int row1 = r < RT ? (run * run_rows + run_rows < s.vrows ? run * run_rows + run_rows : s.vrows) : 0;
    Raw x[U], d[U];
    auto load = [&](int row) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (row + u * RT < row1) {
                const int nv = col.valid(s, row + u * RT);
                x[u] = ld_col<T, M>(xb + (size_t)(row + u * RT) * a.x_row, nv);
                d[u] = ld_col<T, M>(db + (size_t)(row + u * RT) * a.dy_row, nv);
            }
    };
    load(row0);
    const float2* pb = a.part + (size_t)b * s.chunks * s.groups;
    for (int g0 = 0; g0 < s.groups; g0 += TB) {  // S1 / n and S2 / n of every group: the chunks' sums added up
        const int G = s.groups - g0 < TB ? s.groups - g0 : TB;
        const int S = norm_merge_threads(s, TB, G), g = t % G, q = t / G;
        float s1 = 0.f, s2 = 0.f;
        if (q < S) {
            norm_each_chunk(s, pb + g0 + g, q, S, [&](int, float2 m) {
                s1 += m.x;
                s2 += m.y;
            });
            red[2 * t] = s1;
            red[2 * t + 1] = s2;
        }
        __syncthreads();
        if (t < G) {
            for (int i = 1; i < S; ++i) {
                s1 += red[2 * (t + i * G)];
                s2 += red[2 * (t + i * G) + 1];
            }
            gs[2 * (g0 + t)] = s1;
            gs[2 * (g0 + t) + 1] = s2;
        }
        __syncthreads();
    }
    float s1[NG], s2[NG];
#pragma unroll
    for (int e = 0; e < NG; ++e) {
        s1[e] = gs[2 * col.grp[e]];
        s2[e] = gs[2 * col.grp[e] + 1];
    }
    for (int row = row0; row < row1; row += U * RT) {
        Raw o[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float xh[V], dz[V];
            col.template local<SILU>(x[u], d[u], xh, dz, s.slope);
            o[u] = col.grad(xh, dz, s1, s2);
        }
        load(row + U * RT);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (row + u * RT < row1) st_col<T, M>(ob + (size_t)(row + u * RT) * a.dx_row, col.valid(s, row + u * RT), o[u], a.past);
    }
}

// ------------------------------------------------------------------------------------------ host

// threads of a workgroup of the split kernels: 256 or a little less in whole columns, more for wide rows
int split_threads(int cols) {
    const int rows = cols >= 256 ? 1 : 256 / cols;
    return (rows * cols + 63) / 64 * 64;
}

// Virtual rows of a workgroup of the second pass
int run_rows(const NormShape& s, int esize) {
    const long long rows = norm_run_bytes(s, esize) / ((long long)s.W * esize);
    return rows < 1 ? 1 : (int)rows;
}

// Bytes of a slice that few workgroups (below 64; below 128 four times of it) may hold all the same: a larger one is read by a few compute
// units while the others idle.  With 64 to 127 workgroups 2 x 40 x 40 x 512, 51 KB, resident 9.5 us (fp32 11), split 13 (17);
// 2 x 20 x 20 x 1024 fp32 7.2, split 12; 64 x 40 x 40 x 64 in one group, 205 KB, 21, split 18.  Below 64 it depends: 20 x 20 x 1024 fp32
// 7.1, split 11, but the gradient of 60 x 60 x 256 fp16 30 with the forward, split 24, and 3 x 45 x 27 x 75 fp16, 182 KB, 28, split 14.
// Images of odd channel counts, whose split form has more to set up, have no second bound (64 x 20 x 20 x 255, 204 KB: 30, split 45).
constexpr int kResidentAlone = 32 << 10;
constexpr long long kCache = 256 << 20;  // bytes of the cache in front of HBM

long long tensor_bytes(const NormShape& s, int esize) { return (long long)s.batch * s.pixels * s.c * esize; }

// A resident slice: whole groups, and 128 bytes of a pixel - a cache line - or as much as leaves a workgroup for every compute unit (from
// 64 bytes to 128, forward and gradient: 64 x 40 x 40 x 256 fp16 90 -> 83 us, 512 x 10 x 10 x 512 fp16 104 -> 86, fp32 171 -> 131).  False where
// no slice fits the registers, or where a few workgroups would work long while the chip idles.
// The gradient of 16-bit values has registers for four vectors of x and dy a thread; eight leave half the waves, which a narrower slice is
// better than (32 x 20 x 20 x 512: 30 us against 32) and only in small calls the split form is not (32 x 40 x 40 x 128, 13 MB a tensor: 33 us
// against 42 split; 128 x 20 x 20 x 256, 26 MB: 52 against 50).  Parts of lines are read and written twice, which costs little as long as the
// cache holds the call (64 bytes of 26 MB: 47 us against 56 split; of 105 MB: 162 against 142).
struct Resident {
    int cols, threads, r;
};
constexpr int kFwdCap[][2] = {{256, 4}, {512, 8}, {1024, 16}};  // threads, vectors a thread
constexpr int kBwdCap[][2] = {{256, 2}, {256, 4}, {512, 4}, {512, 8}};

template <int N>
bool resident_fit(const NormShape& s, int cols, const int (&cap)[N][2], Resident* out) {
    for (const auto& c : cap) {
        if (cols <= c[0] && (long long)(c[0] / cols) * c[1] >= s.vrows) {
            *out = {cols, c[0], c[1]};
            return true;
        }
    }
    return false;
}

bool resident_of(const NormShape& s, int esize, bool bwd, Resident* out) {
    const int V = 16 / esize;
    const long long tensors = 3 * tensor_bytes(s, esize);
    for (int width = 128; width >= 64; width /= 2) {
        int cols = s.cols;
        if (s.k == 1) {
            cols = s.cpg / norm_gcd(s.cpg, V);  // lcm(cpg, V) / V columns hold whole groups and whole vectors
            while (cols * 16 < width && s.cols % (cols * 2) == 0 && (long long)s.batch * (s.cols / (cols * 2)) >= 256) cols *= 2;
        }
        const long long wgs = (long long)s.batch * (s.cols / cols), bytes = (long long)s.vrows * cols * 16;
        if ((bytes > kResidentAlone && wgs < 64) || (s.k == 1 && bytes > 4 * kResidentAlone && wgs < 128)) return false;
        if (!bwd) {
            if (resident_fit(s, cols, kFwdCap, out)) return true;
        } else if (resident_fit(s, cols, kBwdCap, out)) {
            if (esize == 2 && out->r > 4 ? width == 64 && tensors <= 64 << 20 : cols * 16 >= 128 || tensors <= kCache) return true;
        }
    }
    return false;
}

// What the caller has on hand beside the result is worth more in the cache than the result: a map that fills it with dirty lines makes the
// next kernels wait for those to be written (the statistics of 105 MB take 23 us where the cache holds clean lines, 30 after such a map, 42
// after twice of it).  The result goes past the cache where x and y - for training x, y or dx, and dy - do not fit it together: 210 MB norm
// and 1 x 1 convolution in turn 372 -> 351 us, forward and gradient 323 -> 276 (105 MB: 155 -> 146).  Where they fit, what reads the result
// next pays more than is gained (norm and convolution of 105 MB: 104 -> 107 us, 79 MB: 81 -> 82).
// Not for resident slices of an image, whose parts of lines meet in the cache (64 bytes of 157 MB: 110 -> 120 us with a pass over the result
// behind it; 128 bytes of 157 MB: 101 -> 111); for whole images (219 MB of 75 channels) 257 -> 245.
int past_cache(const NormShape& s, int esize, int tensors, const Resident* res) {
    return (!res || res->cols == s.cols) && tensors * tensor_bytes(s, esize) > kCache;
}

GnArgs make_args(const y5_group_norm_desc& d, const NormShape& s) {
    GnArgs a{};
    a.s = s;
    a.x = d.x;
    a.dy = d.dy;
    a.weight = d.weight;
    a.bias = d.bias;
    a.y = d.y;
    a.dx = d.dx;
    a.dweight = d.dweight;
    a.dbias = d.dbias;
    a.mean = d.mean;
    a.rstd = d.rstd;
    const int ld[4] = {d.x_ld, d.y_ld, d.dy_ld, d.dx_ld};
    long long* row[4] = {&a.x_row, &a.y_row, &a.dy_row, &a.dx_row};
    long long* img[4] = {&a.x_img, &a.y_img, &a.dy_img, &a.dx_img};
    for (int i = 0; i < 4; ++i) {
        *row[i] = s.k == 1 ? ld[i] : s.W;
        *img[i] = (long long)d.pixels * ld[i];
    }
    return a;
}

template <typename F>
int with_lds(F kernel, size_t bytes) {  // more than 64 KiB of LDS have to be asked for
    if (bytes > 64 << 10) Y5_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    return Y5_OK;
}

// Launches kernel(args...) with `lds` bytes of LDS, or returns from the caller with the error
#define GN_LAUNCH(NAME, KERNEL, GRID, THREADS, LDS, ...)                                    \
    do {                                                                                    \
        if (int rc_ = with_lds(KERNEL, LDS)) return rc_;                                    \
        hipLaunchKernelGGL(KERNEL, GRID, dim3(THREADS), LDS, st, __VA_ARGS__);              \
        Y5_LAUNCH_CHECK(NAME);                                                              \
    } while (0)

template <typename T, int M>
int stats(const GnArgs& a, hipStream_t st) {
    const int threads = split_threads(a.s.cols);
    const size_t lds = ((size_t)(threads + a.s.cols) * 2 * (M ? NormElem<T>::V : 1) + a.s.groups) * 4;
    GN_LAUNCH("gn_stats_kernel", (gn_stats_kernel<T, M>), dim3(a.s.chunks, a.s.batch), threads, lds, a);
    return Y5_OK;
}

template <typename T, int M, bool SILU>
int forward(const GnArgs& a, const Resident* res, hipStream_t st) {
    const NormShape& s = a.s;
    constexpr int V = NormElem<T>::V, NG = M ? V : 1;
    if (res) {
        const int slices = s.k == 1 ? s.cols / res->cols : 1;
        const dim3 grid((unsigned)slices * s.batch);
        const size_t lds = ((size_t)(res->threads + res->cols) * NG + 2 * (s.k == 1 ? res->cols * V / s.cpg : s.groups)) * 4;
        if (res->r == 4) GN_LAUNCH("gn_resident_kernel", (gn_resident_kernel<T, M, SILU, 4>), grid, res->threads, lds, a, make_fastdiv((unsigned)res->cols), slices);
        else if (res->r == 8) GN_LAUNCH("gn_resident_kernel", (gn_resident_kernel<T, M, SILU, 8>), grid, res->threads, lds, a, make_fastdiv((unsigned)res->cols), slices);
        else GN_LAUNCH("gn_resident_kernel", (gn_resident_kernel<T, M, SILU, 16>), grid, res->threads, lds, a, make_fastdiv((unsigned)res->cols), slices);
        return Y5_OK;
    }
    if (int rc = stats<T, M>(a, st)) return rc;
    const int threads = split_threads(s.cols), rr = run_rows(s, sizeof(T));
    const size_t lds = (2 * (size_t)threads + 2 * s.groups) * 4;
    GN_LAUNCH("gn_apply_kernel", (gn_apply_kernel<T, M, SILU>), dim3((s.vrows + rr - 1) / rr, s.batch), threads, lds, a, rr);
    return Y5_OK;
}

template <typename T, int M, bool SILU>
int backward(const GnArgs& a, const Resident* res, hipStream_t st) {
    const NormShape& s = a.s;
    constexpr int V = NormElem<T>::V;
    if (res) {
        const int slices = s.k == 1 ? s.cols / res->cols : 1;
        const dim3 grid((unsigned)slices * s.batch);
        const size_t lds = ((size_t)(res->threads + res->cols) * 2 * V + 2 * (s.k == 1 ? res->cols * V / s.cpg : s.groups)) * 4;
        if (res->r == 2) GN_LAUNCH("gn_bwd_resident_kernel", (gn_bwd_resident_kernel<T, M, SILU, 2>), grid, res->threads, lds, a, make_fastdiv((unsigned)res->cols), slices);
        else if (res->r == 4) GN_LAUNCH("gn_bwd_resident_kernel", (gn_bwd_resident_kernel<T, M, SILU, 4>), grid, res->threads, lds, a, make_fastdiv((unsigned)res->cols), slices);
        else GN_LAUNCH("gn_bwd_resident_kernel", (gn_bwd_resident_kernel<T, M, SILU, 8>), grid, res->threads, lds, a, make_fastdiv((unsigned)res->cols), slices);
    } else {
        const int threads = split_threads(s.cols), rr = run_rows(s, sizeof(T)), runs = (s.vrows + rr - 1) / rr;
        size_t lds = ((size_t)(threads + s.cols) * 2 * V + 2 * s.groups) * 4;
        GN_LAUNCH("gn_bwd_stats_kernel", (gn_bwd_stats_kernel<T, M, SILU>), dim3(s.chunks, s.batch), threads, lds, a);
        if (a.dx) {
            const int param_blocks = a.dweight || a.dbias ? (2 * s.c + 15) / 16 : 0;
            Y5_REQUIRE((long long)runs * s.batch + param_blocks <= 0x7fffffffLL, "group_norm_backward: %d images of %d pixels", s.batch, s.pixels);
            lds = (2 * (size_t)threads + 2 * s.groups) * 4;
            GN_LAUNCH("gn_bwd_apply_kernel", (gn_bwd_apply_kernel<T, M, SILU>), dim3(runs * s.batch + param_blocks), threads, lds, a, rr, runs, param_blocks);
            return Y5_OK;
        }
    }
    if (a.dweight || a.dbias) {
        const int rows = res ? s.batch : s.batch * s.chunks;
        GN_LAUNCH("gn_dparam_kernel", gn_dparam_kernel, dim3((2 * s.c + 15) / 16), 256, 0, a.cpart, rows, s.c, s.param_dtype, a.dweight, a.dbias);
    }
    return Y5_OK;
}

template <typename T, int M>
int forward_act(const GnArgs& a, const Resident* res, hipStream_t st) {
    return a.s.act == Y5_ACT_SILU ? forward<T, M, true>(a, res, st) : forward<T, M, false>(a, res, st);
}
template <typename T, int M>
int backward_act(const GnArgs& a, const Resident* res, hipStream_t st) {
    return a.s.act == Y5_ACT_SILU ? backward<T, M, true>(a, res, st) : backward<T, M, false>(a, res, st);
}

struct GnWork {
    size_t part, total;  // offset of cpart behind part; bytes
};
GnWork work_of(const NormShape& s, bool resident, bool bwd) {
    GnWork w{0, 0};
    if (!resident) w.part = norm_align16((size_t)s.batch * s.chunks * s.groups * sizeof(float2));
    w.total = w.part + (bwd ? (size_t)s.batch * (resident ? 1 : s.chunks) * 2 * s.c * 4 : 0);
    return w;
}

int mode_of(const NormShape& s, int esize) { return s.k > 1 ? kCut : s.cpg % (16 / esize) != 0 ? kMixed : kUniform; }

// f<type, mode>(args...) of a call's dtype and mode
#define GN_DISPATCH(F, DTYPE, MODE, ...)                                                                                              \
    ((DTYPE) == Y5_F16    ? ((MODE) == kCut ? F<f16, kCut>(__VA_ARGS__) : (MODE) == kMixed ? F<f16, kMixed>(__VA_ARGS__) : F<f16, kUniform>(__VA_ARGS__)) \
     : (DTYPE) == Y5_BF16 ? ((MODE) == kCut ? F<bf16, kCut>(__VA_ARGS__) : (MODE) == kMixed ? F<bf16, kMixed>(__VA_ARGS__) : F<bf16, kUniform>(__VA_ARGS__)) \
                          : ((MODE) == kCut ? F<float, kCut>(__VA_ARGS__) : (MODE) == kMixed ? F<float, kMixed>(__VA_ARGS__) : F<float, kUniform>(__VA_ARGS__)))

}  // namespace

int y5_launch_group_norm_stats(const y5_group_norm_desc& d, hipStream_t st) {
    NormShape s;
    if (int rc = norm_make_shape(d, &s)) return rc;
    GnArgs a = make_args(d, s);
    a.part = static_cast<float2*>(d.workspace);
    return GN_DISPATCH(stats, d.dtype, mode_of(s, norm_elem_size(d.dtype)), a, st);
}

int y5_group_norm_work(const y5_group_norm_desc& d, int what, size_t* bytes) {
    Y5_REQUIRE(what == Y5_GN_FORWARD || what == Y5_GN_BACKWARD || what == Y5_GN_ROWS, "group_norm_workspace: call %d", what);
    NormShape s;
    int rc = norm_make_shape(d, &s);
    if (rc) return rc;
    Resident r;
    const int es = norm_elem_size(d.dtype);
    const bool res = what != Y5_GN_ROWS && resident_of(s, es, what == Y5_GN_BACKWARD, &r);
    *bytes = work_of(s, res, what == Y5_GN_BACKWARD).total;
    return Y5_OK;
}

int y5_launch_group_norm(const y5_group_norm_desc& d, hipStream_t st) {
    NormShape s;
    int rc = norm_make_shape(d, &s);
    if (rc) return rc;
    if ((rc = norm_check_pitch(d, s, "x", d.x, d.x_ld)) || (rc = norm_check_pitch(d, s, "y", d.y, d.y_ld))) return rc;
    Y5_REQUIRE(!d.mean == !d.rstd, "group_norm: mean and rstd go together");
    const int es = norm_elem_size(d.dtype);
    Resident r;
    const bool res = resident_of(s, es, false, &r);
    const GnWork w = work_of(s, res, false);
    if (w.total && (!d.workspace || d.workspace_bytes < w.total)) return y5_fail(Y5_EWORKSPACE, "group_norm: workspace of %zu bytes, %zu needed", d.workspace ? d.workspace_bytes : (size_t)0, w.total);
    Y5_REQUIRE(!w.total || y5_aligned16(d.workspace), "group_norm: misaligned workspace");
    GnArgs a = make_args(d, s);
    a.past = past_cache(s, es, d.mean ? 3 : 2, res ? &r : nullptr);
    a.part = static_cast<float2*>(d.workspace);
    return GN_DISPATCH(forward_act, d.dtype, mode_of(s, es), a, res ? &r : nullptr, st);
}

int y5_launch_group_norm_bwd(const y5_group_norm_desc& d, hipStream_t st) {
    NormShape s;
    int rc = norm_make_shape(d, &s);
    if (rc) return rc;
    if ((rc = norm_check_pitch(d, s, "x", d.x, d.x_ld)) || (rc = norm_check_pitch(d, s, "dy", d.dy, d.dy_ld)) || (d.dx && (rc = norm_check_pitch(d, s, "dx", d.dx, d.dx_ld)))) return rc;
    Y5_REQUIRE(d.mean && d.rstd, "group_norm_backward: null mean or rstd");
    const int es = norm_elem_size(d.dtype);
    Resident r;
    const bool res = resident_of(s, es, true, &r);
    const GnWork w = work_of(s, res, true);
    if (!d.workspace || d.workspace_bytes < w.total) return y5_fail(Y5_EWORKSPACE, "group_norm_backward: workspace of %zu bytes, %zu needed", d.workspace ? d.workspace_bytes : (size_t)0, w.total);
    Y5_REQUIRE(y5_aligned16(d.workspace), "group_norm_backward: misaligned workspace");
    GnArgs a = make_args(d, s);
    a.past = past_cache(s, es, 3, res ? &r : nullptr);
    a.part = static_cast<float2*>(d.workspace);
    a.cpart = reinterpret_cast<float*>(static_cast<char*>(d.workspace) + w.part);
    return GN_DISPATCH(backward_act, d.dtype, mode_of(s, es), a, res ? &r : nullptr, st);
}
