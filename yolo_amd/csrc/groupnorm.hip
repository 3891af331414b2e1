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
//             thread.
//   split     a statistics pass over chunks of every image, then a pass that merges the chunks' statistics and normalises.
//             The second pass walks the images in the opposite order, so that what the first one read last is still in the
//             256 MB cache in front of HBM.
// The sums are taken in a fixed order (no atomics): the same call gives the same bits.
#include "y5_common.h"

namespace {

#include "norm_rows.h"

struct GnArgs {
    NormShape s;
    const void *x, *dy, *weight, *bias;
    void *y, *dx;
    float *mean, *rstd;  // [batch][groups]
    float2* part;        // [batch][chunks][groups]: a chunk's statistics (forward) or its S1, S2 (backward)
    float* cpart;        // backward: [batch * chunks][2][c], a chunk's sums of dz and of dz * xh
    long long x_row, y_row, dy_row, dx_row;  // pitch of a virtual row, in elements
    long long x_img, y_img, dy_img, dx_img;  // of an image
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

// f(g, sum) for the G groups from g0 on, sum = sum over the group's entries of at(entry): entries rep * rep_pitch + g * n + i
// for rep < reps, i < n.  A thread a group, or a wave where a group has many entries.
template <typename At, typename F>
__device__ __forceinline__ void group_sum(int G, int n, int reps, int rep_pitch, At at, F f) {
    const int t = threadIdx.x, T = blockDim.x;
    if (n * reps <= 32) {
        for (int g = t; g < G; g += T) {
            float a = 0.f;
            for (int k = 0; k < reps; ++k)
                for (int i = 0; i < n; ++i) a += at(k * rep_pitch + g * n + i);
            f(g, a);
        }
    } else {
        const int lane = t & 63;
        for (int g = t >> 6; g < G; g += T >> 6) {
            float a = 0.f;
            for (int k = 0; k < reps; ++k)
                for (int i = lane; i < n; i += 64) a += at(k * rep_pitch + g * n + i);
            for (int off = 32; off; off >>= 1) a += __shfl_xor(a, off);
            if (lane == 0) f(g, a);
        }
    }
    __syncthreads();
}

// The vector column a thread owns: element offset in the virtual row, channels, groups and parameters of its elements.
// PER: every element may belong to another group (a group is no multiple of a vector, or a virtual row is several pixels).
template <typename T, bool PER>
struct Column {
    static constexpr int V = NormElem<T>::V, NG = PER ? V : 1;
    int off;      // element offset of the vector in the virtual row
    int ch0;      // channel of its first element
    int grp[NG];  // group of each element
    __device__ __forceinline__ void init(const NormShape& s, int col) {
        off = col * V;
        ch0 = s.k == 1 ? off : off % s.c;
        if (PER) {
#pragma unroll
            for (int e = 0; e < V; ++e) grp[e] = channel(s, e) / s.cpg;
        } else {
            grp[0] = off / s.cpg;
        }
    }
    __device__ __forceinline__ int channel(const NormShape& s, int e) const {
        const int c = ch0 + e;  // below s.c + V: a virtual row of narrow pixels may hold several of them in one vector
        return PER && c >= s.c ? c % s.c : c;
    }
    // elements of the vector that virtual row `row` has
    __device__ __forceinline__ int valid(const NormShape& s, int row) const {
        if (!PER || s.k == 1) return V;
        const long long left = (long long)s.pixels * s.c - ((long long)row * s.W + off);
        return left >= V ? V : left > 0 ? (int)left : 0;
    }
};

template <typename T, bool PER>
__device__ __forceinline__ void ld_col(const T* p, int nv, T (&v)[NormElem<T>::V]) {
    if (!PER || nv >= NormElem<T>::V) ld_vec(p, v);
    else ld_part(p, nv, v);
}
template <typename T, bool PER>
__device__ __forceinline__ void st_col(T* p, int nv, const T (&v)[NormElem<T>::V]) {
    if (!PER || nv >= NormElem<T>::V) st_vec(p, v);
    else st_part(p, nv, v);
}

// z = act(gamma (x - mean) rstd + beta) of one vector, rounded once
template <typename T, int NG>
__device__ __forceinline__ void normalise(const T (&in)[NormElem<T>::V], T (&out)[NormElem<T>::V], const float (&mean)[NG],
                                          const float (&A)[NormElem<T>::V], const float (&B)[NormElem<T>::V], int act, float slope) {
    constexpr int V = NormElem<T>::V;
    float z[V];
#pragma unroll
    for (int e = 0; e < V; ++e) z[e] = __builtin_fmaf((float)in[e] - mean[NG == 1 ? 0 : e], A[e], B[e]);
    norm_act(z, act, slope);
#pragma unroll
    for (int e = 0; e < V; ++e) out[e] = (T)z[e];
}

// ------------------------------------------------------------------------------------------ forward, resident

// grid (slices, batch).  LDS: part[blockDim.x * NG], tot[cols * NG], gs[2 * groups of the slice]
template <typename T, bool PER, int R>
__global__ __launch_bounds__(R > 8 ? 1024 : R > 4 ? 512 : 256) void gn_resident_kernel(const GnArgs a, int cols) {
    constexpr int V = NormElem<T>::V, NG = PER ? V : 1;
    extern __shared__ float lds[];
    const NormShape& s = a.s;
    const int t = threadIdx.x, TB = blockDim.x, b = blockIdx.y;
    const int RT = TB / cols, r = t / cols, j = t - r * cols;
    const bool active = r < RT;
    float *part = lds, *tot = part + TB * NG, *gs = tot + cols * NG;
    Column<T, PER> col;
    col.init(s, blockIdx.x * cols + j);
    const int g0 = blockIdx.x * cols * V / s.cpg;                  // first group of the slice (a slice holds whole groups)
    const int G = PER && s.k > 1 ? s.groups : cols * V / s.cpg;    // its groups
    const int gn = PER ? s.cpg : s.cpg / V;                        // entries of a group in tot
    const T* xb = static_cast<const T*>(a.x) + (size_t)b * a.x_img + col.off;
    T raw[R][V];
    int nv[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int row = r + i * RT;
        nv[i] = active && row < s.vrows ? col.valid(s, row) : 0;
        if (nv[i]) ld_col<T, PER>(xb + (size_t)row * a.x_row, nv[i], raw[i]);
    }
    float acc[NG];
#pragma unroll
    for (int e = 0; e < NG; ++e) acc[e] = 0.f;
#pragma unroll
    for (int i = 0; i < R; ++i)
        if (nv[i]) {
#pragma unroll
            for (int e = 0; e < V; ++e) acc[PER ? e : 0] += (float)raw[i][e];
        }
    const float inv_n = 1.f / ((float)s.pixels * (float)s.cpg);
    col_sum<NG>(acc, j, r, RT, cols, part, tot);
    group_sum(G, gn, s.k, s.c, [&](int i) { return tot[i]; }, [&](int g, float v) { gs[2 * g] = v * inv_n; });
    float mean[NG];
#pragma unroll
    for (int e = 0; e < NG; ++e) {
        mean[e] = active ? gs[2 * (col.grp[e] - g0)] : 0.f;
        acc[e] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < R; ++i)
        if (nv[i]) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float d = (float)raw[i][e] - mean[PER ? e : 0];
                if (!PER || e < nv[i]) acc[PER ? e : 0] = __builtin_fmaf(d, d, acc[PER ? e : 0]);
            }
        }
    col_sum<NG>(acc, j, r, RT, cols, part, tot);
    group_sum(G, gn, s.k, s.c, [&](int i) { return tot[i]; }, [&](int g, float v) { gs[2 * g + 1] = 1.f / sqrtf(v * inv_n + s.eps); });
    if (a.mean) {
        for (int g = t; g < G; g += TB) {
            a.mean[(size_t)b * s.groups + g0 + g] = gs[2 * g];
            a.rstd[(size_t)b * s.groups + g0 + g] = gs[2 * g + 1];
        }
    }
    if (!active) return;
    float A[V], B[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const int c = col.channel(s, e);
        A[e] = ld_param(a.weight, c, s.param_dtype, 1.f) * gs[2 * (col.grp[PER ? e : 0] - g0) + 1];
        B[e] = ld_param(a.bias, c, s.param_dtype, 0.f);
    }
    T* yb = static_cast<T*>(a.y) + (size_t)b * a.y_img + col.off;
#pragma unroll
    for (int i = 0; i < R; ++i)
        if (nv[i]) {
            T out[V];
            normalise<T, NG>(raw[i], out, mean, A, B, s.act, s.slope);
            st_col<T, PER>(yb + (size_t)(r + i * RT) * a.y_row, nv[i], out);
        }
}

// ------------------------------------------------------------------------------------------ forward, split

// grid (chunks, batch): (mean, M2) of every group over the chunk.  A thread sums differences from the first value it reads
// (K): where a map's mean is many deviations from zero, sum and sum of squares of the raw values would cancel.
template <typename T, bool PER>
__global__ __launch_bounds__(1024) void gn_stats_kernel(const GnArgs a) {
    constexpr int V = NormElem<T>::V, NG = PER ? V : 1, NA = PER ? V : 4;
    extern __shared__ float lds[];
    const NormShape& s = a.s;
    const int t = threadIdx.x, TB = blockDim.x, b = blockIdx.y, cols = s.cols;
    const int RT = TB / cols, r = t / cols, j = t - r * cols;
    const bool active = r < RT;
    float *part = lds, *tot = part + TB * NG, *gs = tot + cols * NG;
    Column<T, PER> col;
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
            T v[V];
            const int nv = col.valid(s, row);
            ld_col<T, PER>(xb + (size_t)row * a.x_row, nv, v);
#pragma unroll
            for (int e = 0; e < NG; ++e) K[e] = (float)v[e];
        }
        auto take = [&](const T (&v)[V], int nv) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float d = (float)v[e] - K[PER ? e : 0];
                if (!PER || e < nv) {
                    S[e % NA] += d;
                    Q[e % NA] = __builtin_fmaf(d, d, Q[e % NA]);
                    if (PER) n[e] += 1.f;
                }
            }
            if (!PER) n[0] += (float)V;
        };
        const long long step = (long long)RT * a.x_row;
        const T* p = xb + (size_t)row * a.x_row;
        // four loads in flight; the last row of an image may be cut short and is left to the loop behind
        for (; row + 3 * RT < row1 - (PER ? 1 : 0); row += 4 * RT, p += 4 * step) {
            T v[4][V];
#pragma unroll
            for (int u = 0; u < 4; ++u) ld_vec(p + u * step, v[u]);
#pragma unroll
            for (int u = 0; u < 4; ++u) take(v[u], V);
        }
        for (; row < row1; row += RT, p += step) {
            T v[V];
            const int nv = col.valid(s, row);
            ld_col<T, PER>(p, nv, v);
            take(v, nv);
        }
    }
    float m[NG], q[NG];
    if (PER) {
#pragma unroll
        for (int e = 0; e < NG; ++e) {
            const float d = n[e] > 0.f ? S[e] / n[e] : 0.f;
            m[e] = K[e] + d;
            q[e] = Q[e] - S[e] * d;
        }
    } else {
        const float sum = (S[0] + S[1]) + (S[2] + S[3]), sq = (Q[0] + Q[1]) + (Q[2] + Q[3]);
        const float d = n[0] > 0.f ? sum / n[0] : 0.f;
        m[0] = K[0] + d;
        q[0] = sq - sum * d;
    }
    const int G = s.groups, gn = PER ? s.cpg : s.cpg / V;
    const float inv_n = 1.f / ((float)norm_chunk_pixels(s, blockIdx.x) * (float)s.cpg);
    float acc[NG];
#pragma unroll
    for (int e = 0; e < NG; ++e) acc[e] = n[e] > 0.f ? n[e] * m[e] : 0.f;
    col_sum<NG>(acc, j, r, RT, cols, part, tot);
    group_sum(G, gn, s.k, s.c, [&](int i) { return tot[i]; }, [&](int g, float v) { gs[g] = v * inv_n; });
#pragma unroll
    for (int e = 0; e < NG; ++e) {
        const float d = active ? m[e] - gs[col.grp[e]] : 0.f;
        acc[e] = n[e] > 0.f ? __builtin_fmaf(n[e] * d, d, q[e]) : 0.f;
    }
    col_sum<NG>(acc, j, r, RT, cols, part, tot);
    float2* out = a.part + ((size_t)b * s.chunks + blockIdx.x) * s.groups;
    group_sum(G, gn, s.k, s.c, [&](int i) { return tot[i]; }, [&](int g, float v) { out[g] = make_float2(gs[g], v); });
}

// grid (runs of rows, batch), walked from the end
template <typename T, bool PER>
__global__ __launch_bounds__(1024) void gn_apply_kernel(const GnArgs a, int run_rows) {
    constexpr int V = NormElem<T>::V, NG = PER ? V : 1;
    extern __shared__ float lds[];
    const NormShape& s = a.s;
    const int t = threadIdx.x, TB = blockDim.x, cols = s.cols;
    const int b = s.batch - 1 - blockIdx.y, run = gridDim.x - 1 - blockIdx.x;
    const int RT = TB / cols, r = t / cols, j = t - r * cols;
    float *red = lds, *gmean = red + 2 * TB, *grstd = gmean + s.groups;
    norm_merge_chunks(s, a.part, b, red, gmean, grstd);
    if (a.mean && run == 0) {
        for (int g = t; g < s.groups; g += TB) {
            a.mean[(size_t)b * s.groups + g] = gmean[g];
            a.rstd[(size_t)b * s.groups + g] = grstd[g];
        }
    }
    if (r >= RT) return;
    Column<T, PER> col;
    col.init(s, j);
    float mean[NG], A[V], B[V];
#pragma unroll
    for (int e = 0; e < NG; ++e) mean[e] = gmean[col.grp[e]];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const int c = col.channel(s, e);
        A[e] = ld_param(a.weight, c, s.param_dtype, 1.f) * grstd[col.grp[PER ? e : 0]];
        B[e] = ld_param(a.bias, c, s.param_dtype, 0.f);
    }
    const int row0 = run * run_rows;
    const int row1 = row0 + run_rows < s.vrows ? row0 + run_rows : s.vrows;
    const T* xb = static_cast<const T*>(a.x) + (size_t)b * a.x_img + col.off;
    T* yb = static_cast<T*>(a.y) + (size_t)b * a.y_img + col.off;
    int row = row0 + r;
    for (; row + 3 * RT < row1 - (PER ? 1 : 0); row += 4 * RT) {
        T v[4][V], o[V];
#pragma unroll
        for (int u = 0; u < 4; ++u) ld_vec(xb + (size_t)(row + u * RT) * a.x_row, v[u]);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            normalise<T, NG>(v[u], o, mean, A, B, s.act, s.slope);
            st_vec(yb + (size_t)(row + u * RT) * a.y_row, o);
        }
    }
    for (; row < row1; row += RT) {
        const int nv = col.valid(s, row);
        if (!nv) continue;
        T v[V], o[V];
        ld_col<T, PER>(xb + (size_t)row * a.x_row, nv, v);
        normalise<T, NG>(v, o, mean, A, B, s.act, s.slope);
        st_col<T, PER>(yb + (size_t)row * a.y_row, nv, o);
    }
}

// ------------------------------------------------------------------------------------------ backward

// Parameters of a thread's column for the gradient: mean, rstd of its groups, gamma and beta of its channels
template <typename T, bool PER>
struct GradColumn : Column<T, PER> {
    static constexpr int V = NormElem<T>::V, NG = PER ? V : 1;
    float mean[NG], rstd[NG], gamma[V], beta[V];
    __device__ __forceinline__ void load(const GnArgs& a, int b, int col) {
        const NormShape& s = a.s;
        this->init(s, col);
#pragma unroll
        for (int e = 0; e < NG; ++e) {
            mean[e] = a.mean[(size_t)b * s.groups + this->grp[e]];
            rstd[e] = a.rstd[(size_t)b * s.groups + this->grp[e]];
        }
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const int c = this->channel(s, e);
            gamma[e] = ld_param(a.weight, c, s.param_dtype, 1.f);
            beta[e] = ld_param(a.bias, c, s.param_dtype, 0.f);
        }
    }
    // xh and dz of one vector
    __device__ __forceinline__ void local(const T (&x)[V], const T (&dy)[V], float (&xh)[V], float (&dz)[V], int act, float slope) const {
        float z[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            xh[e] = ((float)x[e] - mean[PER ? e : 0]) * rstd[PER ? e : 0];
            z[e] = __builtin_fmaf(xh[e], gamma[e], beta[e]);
            dz[e] = (float)dy[e];
        }
        norm_act_grad(dz, z, act, slope);
    }
    // dx of one vector from s1 = S1 / n and s2 = S2 / n of its groups
    __device__ __forceinline__ void grad(const float (&xh)[V], const float (&dz)[V], const float (&s1)[NG], const float (&s2)[NG], T (&dx)[V]) const {
#pragma clang fp contract(off)  // a group of one value has gamma dz = S1 exactly and a gradient of exactly zero
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float w = gamma[e] * dz[e];
            const float u = w - s1[PER ? e : 0];
            const float v = xh[e] * s2[PER ? e : 0];
            dx[e] = (T)(rstd[PER ? e : 0] * (u - v));
        }
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
    for (int which = 0; which < 2; ++which)
        group_sum(G, s.cpg, s.k, s.c, [&](int i) { return ld_param(a.weight, c0 + i % s.c, s.param_dtype, 1.f) * at(i, which); },
                  [&](int g, float v) { gs[2 * g + which] = v * scale; });
}

// grid (slices, batch); LDS: part[blockDim.x * 2 V], tot[cols * 2 V], gs[2 * groups of the slice]
template <typename T, bool PER, int R>
__global__ __launch_bounds__(R > 4 ? 512 : 256) void gn_bwd_resident_kernel(const GnArgs a, int cols) {
    constexpr int V = NormElem<T>::V, NG = PER ? V : 1;
    extern __shared__ float lds[];
    const NormShape& s = a.s;
    const int t = threadIdx.x, TB = blockDim.x, b = blockIdx.y;
    const int RT = TB / cols, r = t / cols, j = t - r * cols;
    const bool active = r < RT;
    float *part = lds, *tot = part + TB * 2 * V, *gs = tot + cols * 2 * V;
    GradColumn<T, PER> col;
    col.load(a, b, blockIdx.x * cols + j);
    const T* xb = static_cast<const T*>(a.x) + (size_t)b * a.x_img + col.off;
    const T* db = static_cast<const T*>(a.dy) + (size_t)b * a.dy_img + col.off;
    T rx[R][V], rd[R][V];
    int nv[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int row = r + i * RT;
        nv[i] = active && row < s.vrows ? col.valid(s, row) : 0;
        if (nv[i]) {
            ld_col<T, PER>(xb + (size_t)row * a.x_row, nv[i], rx[i]);
            ld_col<T, PER>(db + (size_t)row * a.dy_row, nv[i], rd[i]);
        }
    }
    float acc[2 * V];
#pragma unroll
    for (int e = 0; e < 2 * V; ++e) acc[e] = 0.f;
#pragma unroll
    for (int i = 0; i < R; ++i)
        if (nv[i]) {
            float xh[V], dz[V];
            col.local(rx[i], rd[i], xh, dz, s.act, s.slope);
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (!PER || e < nv[i]) {
                    acc[e] += dz[e];
                    acc[V + e] = __builtin_fmaf(dz[e], xh[e], acc[V + e]);
                }
        }
    col_sum<2 * V>(acc, j, r, RT, cols, part, tot);
    const int c0 = s.k > 1 ? 0 : blockIdx.x * cols * V, channels = s.k > 1 ? s.c : cols * V;
    const int g0 = c0 / s.cpg, G = channels / s.cpg;
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
        if (nv[i]) {
            float xh[V], dz[V];
            T dx[V];
            col.local(rx[i], rd[i], xh, dz, s.act, s.slope);
            col.grad(xh, dz, s1, s2, dx);
            st_col<T, PER>(ob + (size_t)(r + i * RT) * a.dx_row, nv[i], dx);
        }
}

// grid (chunks, batch); LDS as above for all groups
template <typename T, bool PER>
__global__ __launch_bounds__(1024) void gn_bwd_stats_kernel(const GnArgs a) {
    constexpr int V = NormElem<T>::V;
    extern __shared__ float lds[];
    const NormShape& s = a.s;
    const int t = threadIdx.x, TB = blockDim.x, b = blockIdx.y, cols = s.cols;
    const int RT = TB / cols, r = t / cols, j = t - r * cols;
    float *part = lds, *tot = part + TB * 2 * V, *gs = tot + cols * 2 * V;
    GradColumn<T, PER> col;
    col.load(a, b, j);
    float acc[2 * V];
#pragma unroll
    for (int e = 0; e < 2 * V; ++e) acc[e] = 0.f;
    const int row0 = blockIdx.x * s.chunk_rows;
    const int row1 = row0 + s.chunk_rows < s.vrows ? row0 + s.chunk_rows : s.vrows;
    if (r < RT) {
        const T* xb = static_cast<const T*>(a.x) + (size_t)b * a.x_img + col.off;
        const T* db = static_cast<const T*>(a.dy) + (size_t)b * a.dy_img + col.off;
        auto take = [&](const T (&x)[V], const T (&d)[V], int nv) {
            float xh[V], dz[V];
            col.local(x, d, xh, dz, s.act, s.slope);
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (!PER || e < nv) {
                    acc[e] += dz[e];
                    acc[V + e] = __builtin_fmaf(dz[e], xh[e], acc[V + e]);
                }
        };
        int row = row0 + r;
        for (; row + RT < row1 - (PER ? 1 : 0); row += 2 * RT) {
            T x[2][V], d[2][V];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                ld_vec(xb + (size_t)(row + u * RT) * a.x_row, x[u]);
                ld_vec(db + (size_t)(row + u * RT) * a.dy_row, d[u]);
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) take(x[u], d[u], V);
        }
        for (; row < row1; row += RT) {
            const int nv = col.valid(s, row);
            T x[V], d[V];
            ld_col<T, PER>(xb + (size_t)row * a.x_row, nv, x);
            ld_col<T, PER>(db + (size_t)row * a.dy_row, nv, d);
            take(x, d, nv);
        }
    }
    col_sum<2 * V>(acc, j, r, RT, cols, part, tot);
    const size_t at = (size_t)b * s.chunks + blockIdx.x;
    grad_sums<V>(a, tot, 0, s.c, s.groups, 1.f / ((float)s.pixels * (float)s.cpg), a.cpart + at * 2 * s.c, gs);
    for (int g = t; g < s.groups; g += TB) a.part[at * s.groups + g] = make_float2(gs[2 * g], gs[2 * g + 1]);
}

// grid (runs of rows, batch), walked from the end; LDS: red[2 * blockDim.x], gs[2 * groups]
template <typename T, bool PER>
__global__ __launch_bounds__(1024) void gn_bwd_apply_kernel(const GnArgs a, int run_rows) {
    constexpr int V = NormElem<T>::V, NG = PER ? V : 1;
    extern __shared__ float lds[];
    const NormShape& s = a.s;
    const int t = threadIdx.x, TB = blockDim.x, cols = s.cols;
    const int b = s.batch - 1 - blockIdx.y, run = gridDim.x - 1 - blockIdx.x;
    const int RT = TB / cols, r = t / cols, j = t - r * cols;
    float *red = lds, *gs = lds + 2 * TB;
    const float2* pb = a.part + (size_t)b * s.chunks * s.groups;
    for (int g0 = 0; g0 < s.groups; g0 += TB) {  // S1 / n and S2 / n of every group: the chunks' sums added up
        const int G = s.groups - g0 < TB ? s.groups - g0 : TB;
        const int S = TB / G, g = t % G, q = t / G;
        float s1 = 0.f, s2 = 0.f;
        if (q < S) {
#pragma unroll 8
            for (int i = q; i < s.chunks; i += S) {
                const float2 m = pb[(size_t)i * s.groups + g0 + g];
                s1 += m.x;
                s2 += m.y;
            }
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
    if (r >= RT) return;
    GradColumn<T, PER> col;
    col.load(a, b, j);
    float s1[NG], s2[NG];
#pragma unroll
    for (int e = 0; e < NG; ++e) {
        s1[e] = gs[2 * col.grp[e]];
        s2[e] = gs[2 * col.grp[e] + 1];
    }
    const int row0 = run * run_rows;
    const int row1 = row0 + run_rows < s.vrows ? row0 + run_rows : s.vrows;
    const T* xb = static_cast<const T*>(a.x) + (size_t)b * a.x_img + col.off;
    const T* db = static_cast<const T*>(a.dy) + (size_t)b * a.dy_img + col.off;
    T* ob = static_cast<T*>(a.dx) + (size_t)b * a.dx_img + col.off;
    int row = row0 + r;
    for (; row + RT < row1 - (PER ? 1 : 0); row += 2 * RT) {
        T x[2][V], d[2][V], o[V];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            ld_vec(xb + (size_t)(row + u * RT) * a.x_row, x[u]);
            ld_vec(db + (size_t)(row + u * RT) * a.dy_row, d[u]);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            float xh[V], dz[V];
            col.local(x[u], d[u], xh, dz, s.act, s.slope);
            col.grad(xh, dz, s1, s2, o);
            st_vec(ob + (size_t)(row + u * RT) * a.dx_row, o);
        }
    }
    for (; row < row1; row += RT) {
        const int nv = col.valid(s, row);
        if (!nv) continue;
        T x[V], d[V], o[V];
        ld_col<T, PER>(xb + (size_t)row * a.x_row, nv, x);
        ld_col<T, PER>(db + (size_t)row * a.dy_row, nv, d);
        float xh[V], dz[V];
        col.local(x, d, xh, dz, s.act, s.slope);
        col.grad(xh, dz, s1, s2, o);
        st_col<T, PER>(ob + (size_t)row * a.dx_row, nv, o);
    }
}

// dbeta_c and dgamma_c: the rows of cpart ([rows][2][c]) added up.  A workgroup takes 16 of the 2 c columns, 16 threads each.
__global__ __launch_bounds__(256) void gn_dparam_kernel(const float* __restrict__ cpart, int rows, int c, int dt, void* dweight, void* dbias) {
    __shared__ float red[16][17];
    const int lc = threadIdx.x & 15, q = threadIdx.x >> 4;
    const int i = blockIdx.x * 16 + lc;
    float v = 0.f;
    if (i < 2 * c) {
#pragma unroll 8
        for (int k = q; k < rows; k += 16) v += cpart[(size_t)k * 2 * c + i];
    }
    red[q][lc] = v;
    __syncthreads();
    if (q || i >= 2 * c) return;
#pragma unroll
    for (int k = 1; k < 16; ++k) v += red[k][lc];
    if (i < c) {
        if (dbias) st_param(dbias, i, dt, v);
    } else if (dweight) {
        st_param(dweight, i - c, dt, v);
    }
}

// ------------------------------------------------------------------------------------------ host

// threads of a workgroup of the split kernels: 256 or a little less in whole columns, more for wide rows
int split_threads(int cols) {
    const int rows = cols >= 256 ? 1 : 256 / cols;
    return (rows * cols + 63) / 64 * 64;
}

// Rows of a workgroup of the second pass: 32 KiB
int run_rows(const NormShape& s, int esize) {
    const long long rows = (32 << 10) / ((long long)s.W * esize);
    return rows < 1 ? 1 : (int)rows;
}

// A resident slice: the fewest columns that hold whole groups and 64 bytes of a pixel (half a cache line; narrower slices
// read lines that other workgroups read again).  False where no slice fits R vectors a thread.
struct Resident {
    int cols, threads, r;
};
bool resident_of(const NormShape& s, int esize, const int (&cap)[3][2], Resident* out) {
    const int V = 16 / esize;
    int cols = s.cols;
    if (s.k == 1) {
        const int unit = s.cpg / norm_gcd(s.cpg, V);  // lcm(cpg, V) / V columns hold whole groups and whole vectors
        cols = unit;
        while (cols * 16 < 64 && cols * 2 <= s.cols && s.cols % (cols * 2) == 0) cols *= 2;
    }
    for (const auto& c : cap) {
        const int threads = c[0], r = c[1];
        if (cols > threads) continue;
        if ((long long)(threads / cols) * r >= s.vrows) {
            *out = {cols, threads, r};
            return true;
        }
    }
    return false;
}
constexpr int kFwdCap[3][2] = {{256, 4}, {512, 8}, {1024, 16}};
constexpr int kBwdCap[3][2] = {{256, 2}, {256, 4}, {512, 8}};

GnArgs make_args(const y5_group_norm_desc& d, const NormShape& s) {
    GnArgs a{};
    a.s = s;
    a.x = d.x;
    a.dy = d.dy;
    a.weight = d.weight;
    a.bias = d.bias;
    a.y = d.y;
    a.dx = d.dx;
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

template <typename T, bool PER>
int stats(const GnArgs& a, hipStream_t st) {
    const int threads = split_threads(a.s.cols);
    const size_t lds = ((size_t)(threads + a.s.cols) * (PER ? NormElem<T>::V : 1) + a.s.groups) * 4;
    GN_LAUNCH("gn_stats_kernel", (gn_stats_kernel<T, PER>), dim3(a.s.chunks, a.s.batch), threads, lds, a);
    return Y5_OK;
}

template <typename T, bool PER>
int forward(const GnArgs& a, const Resident* res, hipStream_t st) {
    const NormShape& s = a.s;
    constexpr int V = NormElem<T>::V, NG = PER ? V : 1;
    if (res) {
        const dim3 grid(s.k == 1 ? s.cols / res->cols : 1, s.batch);
        const size_t lds = ((size_t)(res->threads + res->cols) * NG + 2 * (s.k == 1 ? res->cols * V / s.cpg : s.groups)) * 4;
        if (res->r == 4) GN_LAUNCH("gn_resident_kernel", (gn_resident_kernel<T, PER, 4>), grid, res->threads, lds, a, res->cols);
        else if (res->r == 8) GN_LAUNCH("gn_resident_kernel", (gn_resident_kernel<T, PER, 8>), grid, res->threads, lds, a, res->cols);
        else GN_LAUNCH("gn_resident_kernel", (gn_resident_kernel<T, PER, 16>), grid, res->threads, lds, a, res->cols);
        return Y5_OK;
    }
    if (int rc = stats<T, PER>(a, st)) return rc;
    const int threads = split_threads(s.cols), rr = run_rows(s, sizeof(T));
    const size_t lds = (2 * (size_t)threads + 2 * s.groups) * 4;
    GN_LAUNCH("gn_apply_kernel", (gn_apply_kernel<T, PER>), dim3((s.vrows + rr - 1) / rr, s.batch), threads, lds, a, rr);
    return Y5_OK;
}

template <typename T, bool PER>
int backward(const GnArgs& a, const Resident* res, void* dweight, void* dbias, hipStream_t st) {
    const NormShape& s = a.s;
    constexpr int V = NormElem<T>::V;
    if (res) {
        const dim3 grid(s.k == 1 ? s.cols / res->cols : 1, s.batch);
        const size_t lds = ((size_t)(res->threads + res->cols) * 2 * V + 2 * (s.k == 1 ? res->cols * V / s.cpg : s.groups)) * 4;
        if (res->r == 2) GN_LAUNCH("gn_bwd_resident_kernel", (gn_bwd_resident_kernel<T, PER, 2>), grid, res->threads, lds, a, res->cols);
        else if (res->r == 4) GN_LAUNCH("gn_bwd_resident_kernel", (gn_bwd_resident_kernel<T, PER, 4>), grid, res->threads, lds, a, res->cols);
        else GN_LAUNCH("gn_bwd_resident_kernel", (gn_bwd_resident_kernel<T, PER, 8>), grid, res->threads, lds, a, res->cols);
    } else {
        const int threads = split_threads(s.cols), rr = run_rows(s, sizeof(T));
        size_t lds = ((size_t)(threads + s.cols) * 2 * V + 2 * s.groups) * 4;
        GN_LAUNCH("gn_bwd_stats_kernel", (gn_bwd_stats_kernel<T, PER>), dim3(s.chunks, s.batch), threads, lds, a);
        lds = (2 * (size_t)threads + 2 * s.groups) * 4;
        if (a.dx) GN_LAUNCH("gn_bwd_apply_kernel", (gn_bwd_apply_kernel<T, PER>), dim3((s.vrows + rr - 1) / rr, s.batch), threads, lds, a, rr);
    }
    if (dweight || dbias) {
        const int rows = res ? s.batch : s.batch * s.chunks;
        GN_LAUNCH("gn_dparam_kernel", gn_dparam_kernel, dim3((2 * s.c + 15) / 16), 256, 0, a.cpart, rows, s.c, s.param_dtype, dweight, dbias);
    }
    return Y5_OK;
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

bool per_element(const NormShape& s, int esize) { return s.k > 1 || s.cpg % (16 / esize) != 0; }

}  // namespace

int y5_launch_group_norm_stats(const y5_group_norm_desc& d, hipStream_t st) {
    NormShape s;
    if (int rc = norm_make_shape(d, &s)) return rc;
    GnArgs a = make_args(d, s);
    a.part = static_cast<float2*>(d.workspace);
    const bool per = per_element(s, norm_elem_size(d.dtype));
    if (d.dtype == Y5_F16) return per ? stats<f16, true>(a, st) : stats<f16, false>(a, st);
    if (d.dtype == Y5_BF16) return per ? stats<bf16, true>(a, st) : stats<bf16, false>(a, st);
    return per ? stats<float, true>(a, st) : stats<float, false>(a, st);
}

int y5_group_norm_work(const y5_group_norm_desc& d, int what, size_t* bytes) {
    Y5_REQUIRE(what == Y5_GN_FORWARD || what == Y5_GN_BACKWARD || what == Y5_GN_ROWS, "group_norm_workspace: call %d", what);
    NormShape s;
    int rc = norm_make_shape(d, &s);
    if (rc) return rc;
    Resident r;
    const int es = norm_elem_size(d.dtype);
    const bool res = what == Y5_GN_BACKWARD ? resident_of(s, es, kBwdCap, &r) : what == Y5_GN_FORWARD && resident_of(s, es, kFwdCap, &r);
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
    const bool res = resident_of(s, es, kFwdCap, &r);
    const GnWork w = work_of(s, res, false);
    if (w.total && (!d.workspace || d.workspace_bytes < w.total)) return y5_fail(Y5_EWORKSPACE, "group_norm: workspace of %zu bytes, %zu needed", d.workspace ? d.workspace_bytes : (size_t)0, w.total);
    Y5_REQUIRE(!w.total || y5_aligned16(d.workspace), "group_norm: misaligned workspace");
    GnArgs a = make_args(d, s);
    a.part = static_cast<float2*>(d.workspace);
    const bool per = per_element(s, es);
    const Resident* rp = res ? &r : nullptr;
    if (d.dtype == Y5_F16) return per ? forward<f16, true>(a, rp, st) : forward<f16, false>(a, rp, st);
    if (d.dtype == Y5_BF16) return per ? forward<bf16, true>(a, rp, st) : forward<bf16, false>(a, rp, st);
    return per ? forward<float, true>(a, rp, st) : forward<float, false>(a, rp, st);
}

int y5_launch_group_norm_bwd(const y5_group_norm_desc& d, hipStream_t st) {
    NormShape s;
    int rc = norm_make_shape(d, &s);
    if (rc) return rc;
    if ((rc = norm_check_pitch(d, s, "x", d.x, d.x_ld)) || (rc = norm_check_pitch(d, s, "dy", d.dy, d.dy_ld)) || (d.dx && (rc = norm_check_pitch(d, s, "dx", d.dx, d.dx_ld)))) return rc;
    Y5_REQUIRE(d.mean && d.rstd, "group_norm_backward: null mean or rstd");
    const int es = norm_elem_size(d.dtype);
    Resident r;
    const bool res = resident_of(s, es, kBwdCap, &r);
    const GnWork w = work_of(s, res, true);
    if (!d.workspace || d.workspace_bytes < w.total) return y5_fail(Y5_EWORKSPACE, "group_norm_backward: workspace of %zu bytes, %zu needed", d.workspace ? d.workspace_bytes : (size_t)0, w.total);
    Y5_REQUIRE(y5_aligned16(d.workspace), "group_norm_backward: misaligned workspace");
    GnArgs a = make_args(d, s);
    a.part = static_cast<float2*>(d.workspace);
    a.cpart = reinterpret_cast<float*>(static_cast<char*>(d.workspace) + w.part);
    const bool per = per_element(s, es);
    const Resident* rp = res ? &r : nullptr;
    if (d.dtype == Y5_F16) return per ? backward<f16, true>(a, rp, d.dweight, d.dbias, st) : backward<f16, false>(a, rp, d.dweight, d.dbias, st);
    if (d.dtype == Y5_BF16) return per ? backward<bf16, true>(a, rp, d.dweight, d.dbias, st) : backward<bf16, false>(a, rp, d.dweight, d.dbias, st);
    return per ? backward<float, true>(a, rp, d.dweight, d.dbias, st) : backward<float, false>(a, rp, d.dweight, d.dbias, st);
}
