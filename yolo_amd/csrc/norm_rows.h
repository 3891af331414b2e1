// Pieces shared by the channels-last group norm (groupnorm.hip) and the 8-bit row quantisation (rows_i8.hip): element types,
// 16-byte accesses at any element alignment, activations, and the group statistics that several chunks of an image left in
// the workspace.  Included inside an anonymous namespace, after conv_common.h.
#pragma once

template <typename T>
struct NormElem {
    static constexpr int V = 16 / (int)sizeof(T);  // elements of a 16-byte vector
};

// A pixel of a tensor whose channel count or pitch is not a multiple of 8 starts anywhere: the accesses below are 16 bytes at
// element alignment, which the memory pipeline serves like aligned ones, in one or two more cache lines.  One 16-byte value, not
// V elements: as elements the compiler splits such an access up where a branch beside it touches some of them.
typedef unsigned norm_u32x4 __attribute__((ext_vector_type(4)));
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) NormVec {
    norm_u32x4 v;
};
template <typename T>
struct NormArr {
    T v[NormElem<T>::V];
};

template <typename T>
__device__ __forceinline__ void ld_vec(const T* p, T (&v)[NormElem<T>::V]) {
    const NormArr<T> u = __builtin_bit_cast(NormArr<T>, reinterpret_cast<const NormVec<T>*>(p)->v);
#pragma unroll
    for (int e = 0; e < NormElem<T>::V; ++e) v[e] = u.v[e];
}
// the first n elements, zeros behind them; nothing behind the n-th is touched: the first is read in its place, so that all are on their way
// at once (a branch an element waits for each)
template <typename T>
__device__ __forceinline__ void ld_part(const T* p, int n, T (&v)[NormElem<T>::V]) {
#pragma unroll
    for (int e = 0; e < NormElem<T>::V; ++e) v[e] = (T)0.f;
    if (n > 0) {
#pragma unroll
        for (int e = 0; e < NormElem<T>::V; ++e) {
            const T x = p[e < n ? e : 0];
            v[e] = e < n ? x : (T)0.f;
        }
    }
}
template <typename T>
__device__ __forceinline__ void st_vec(T* p, const T (&v)[NormElem<T>::V]) {
    NormArr<T> u;
#pragma unroll
    for (int e = 0; e < NormElem<T>::V; ++e) u.v[e] = v[e];
    reinterpret_cast<NormVec<T>*>(p)->v = __builtin_bit_cast(norm_u32x4, u);
}
template <typename T>
__device__ __forceinline__ void st_part(T* p, int n, const T (&v)[NormElem<T>::V]) {
#pragma unroll
    for (int e = 0; e < NormElem<T>::V; ++e)
        if (e < n) p[e] = v[e];
}

// element i of a parameter vector of type dt (Y5_F16 / Y5_BF16 / Y5_F32); def where there is none
__device__ __forceinline__ float ld_param(const void* p, int i, int dt, float def) {
    if (!p) return def;
    if (dt == Y5_F32) return static_cast<const float*>(p)[i];
    if (dt == Y5_F16) return (float)static_cast<const f16*>(p)[i];
    return (float)static_cast<const bf16*>(p)[i];
}
// N consecutive ones from element i on
template <int N>
__device__ __forceinline__ void ld_params(const void* p, int i, int dt, float def, float (&v)[N]) {
    if (!p) {
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = def;
    } else if (dt == Y5_F32) {
#pragma unroll
        for (int u = 0; u < N / 4; ++u) {
            float w[4];
            ld_vec(static_cast<const float*>(p) + i + 4 * u, w);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[4 * u + e] = w[e];
        }
    } else {
        struct __attribute__((packed, aligned(2))) Half {
            unsigned w[N / 2];
        };
        const Half h = *reinterpret_cast<const Half*>(static_cast<const unsigned short*>(p) + i);
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const unsigned short b = (unsigned short)(h.w[e / 2] >> (16 * (e & 1)));
            v[e] = dt == Y5_F16 ? (float)__builtin_bit_cast(f16, b) : __uint_as_float((unsigned)b << 16);
        }
    }
}
__device__ __forceinline__ void st_param(void* p, int i, int dt, float v) {
    if (dt == Y5_F32) static_cast<float*>(p)[i] = v;
    else if (dt == Y5_F16) static_cast<f16*>(p)[i] = (f16)v;
    else static_cast<bf16*>(p)[i] = (bf16)v;
}

// 1 / (1 + exp(-z)): exp2 and the hardware reciprocal, each within an ulp; exp2 overflows to infinity for z below -127, whose
// reciprocal is the 0 that belongs there
__device__ __forceinline__ float norm_sigmoid(float z) {
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * -1.44269504088896341f));
}
// The activation is a template parameter (no activation is LeakyReLU of slope 1): a test at run time makes the compiler keep
// several versions of everything around it.
template <bool SILU, int N>
__device__ __forceinline__ void norm_act(float (&z)[N], float slope) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
        if constexpr (SILU) z[e] = z[e] * norm_sigmoid(z[e]);
        else z[e] = z[e] > 0.f ? z[e] : z[e] * slope;
    }
}
// d[e] *= act'(z[e])
template <bool SILU, int N>
__device__ __forceinline__ void norm_act_grad(float (&d)[N], const float (&z)[N], float slope) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
        if constexpr (SILU) {
            const float p = norm_sigmoid(z[e]);
            d[e] *= p * __builtin_fmaf(z[e], 1.f - p, 1.f);
        } else {
            d[e] = z[e] > 0.f ? d[e] : d[e] * slope;
        }
    }
}

// The shape of one call as the kernels walk it: an image is `vrows` virtual rows of W elements at pitch `pitch`.  A virtual
// row is one pixel where the channel count fills whole 16-byte vectors, and otherwise the `k` consecutive pixels of a dense
// tensor whose k * c elements do (then the last row of an image may be cut short, at `total` elements).  A thread keeps one
// vector column for the whole kernel, so the channels of its elements - and their parameters - never change.
struct NormShape {
    int c, groups, cpg;  // channels, groups, channels of a group
    int k, W, cols;      // pixels of a virtual row, its elements, its vectors
    int vrows;           // virtual rows of an image
    int pixels;          // pixels of an image
    int chunks, chunk_rows;  // an image's virtual rows are cut into `chunks` runs of chunk_rows (the last one shorter)
    int batch;
    int act, param_dtype;
    float slope, eps;
    FastDiv by_c, by_cpg, by_cols;
};

// Merging the chunks of a group: norm_merge_threads() of T threads for G groups share it, each adds up four chunks or more, four of them on
// their way at a time, and one of the threads the others' sums, one after the other (with every thread of few groups that alone
// took 9 us)
__device__ __forceinline__ int norm_merge_threads(const NormShape& s, int T, int G) {
    const int all = T / G, most = (s.chunks + 3) / 4;
    return all < most ? all : most;
}
// f(chunk, what it left) for thread r of S; p: what the group's first chunk left
template <typename F>
__device__ __forceinline__ void norm_each_chunk(const NormShape& s, const float2* __restrict__ p, int r, int S, F f) {
    for (int i = r; i < s.chunks; i += 4 * S) {
        float2 m[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int k = i + u * S < s.chunks ? i + u * S : i;
            m[u] = p[(size_t)k * s.groups];
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (i + u * S < s.chunks) f(i + u * S, m[u]);
    }
}

// pixels of chunk i of an image
__device__ __forceinline__ int norm_chunk_pixels(const NormShape& s, int i) {
    const long long p0 = (long long)i * s.chunk_rows * s.k, p1 = p0 + (long long)s.chunk_rows * s.k;
    return (int)((p1 < s.pixels ? p1 : (long long)s.pixels) - p0);
}

// Mean and 1 / standard deviation of every group of image b from the chunks' (mean, sum of squared differences from it):
//   mean = K + sum n_i (m_i - K) / N,   M2 = sum (M2_i + n_i (m_i - K)^2) - N (mean - K)^2,   K = the first chunk's mean,
// which keeps the digits that sum and sum of squares of the raw values would lose where a mean is far from zero.
// red: 2 * blockDim.x floats of LDS.  Results in gmean / grstd[groups] (LDS), after a barrier.
__device__ __forceinline__ void norm_merge_chunks(const NormShape& s, const float2* __restrict__ part, int b, float* red, float* gmean,
                                                  float* grstd) {
    const int t = threadIdx.x, T = blockDim.x;
    const float2* pb = part + (size_t)b * s.chunks * s.groups;
    const float npix = (float)s.cpg;
    for (int g0 = 0; g0 < s.groups; g0 += T) {
        const int G = s.groups - g0 < T ? s.groups - g0 : T;
        const int S = norm_merge_threads(s, T, G);
        const int g = t % G, r = t / G;
        float s1 = 0.f, s2 = 0.f, K = 0.f;
        if (r < S) {
            K = pb[g0 + g].x;
            norm_each_chunk(s, pb + g0 + g, r, S, [&](int i, float2 m) {
                const float n = (float)norm_chunk_pixels(s, i) * npix;
                const float d = m.x - K;
                s1 = __builtin_fmaf(n, d, s1);
                s2 += __builtin_fmaf(n * d, d, m.y);
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
            const float N = (float)s.pixels * npix;
            const float d = s1 / N;
            float var = (s2 - s1 * d) / N;
            // not max(): that would turn the NaN of a group with an infinity or a NaN in it into a variance of zero
            var = var < 0.f ? 0.f : var;
            gmean[g0 + t] = K + d;
            grstd[g0 + t] = 1.f / sqrtf(var + s.eps);
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------------------------------------ host

constexpr int kNormMaxW = 4096;     // elements of a virtual row
constexpr int kNormMaxChunks = 128;  // chunks of an image in the split form

inline int norm_gcd(int a, int b) {
    while (b) {
        const int t = a % b;
        a = b;
        b = t;
    }
    return a;
}

inline int norm_elem_size(int dtype) { return dtype == Y5_F32 ? 4 : 2; }

// Checks what does not depend on the direction and fills the shape.
inline int norm_make_shape(const y5_group_norm_desc& d, NormShape* out) {
    Y5_REQUIRE(d.dtype == Y5_F16 || d.dtype == Y5_BF16 || d.dtype == Y5_F32, "group_norm: dtype %d", d.dtype);
    Y5_REQUIRE(d.param_dtype == Y5_F16 || d.param_dtype == Y5_BF16 || d.param_dtype == Y5_F32, "group_norm: param_dtype %d", d.param_dtype);
    Y5_REQUIRE(d.batch > 0 && d.batch <= 65535 && d.pixels > 0 && d.pixels <= 1 << 30 && d.c > 0, "group_norm: batch %d (at most 65535), pixels %d (at most 2^30), channels %d", d.batch, d.pixels, d.c);
    Y5_REQUIRE(d.groups > 0 && d.c % d.groups == 0, "group_norm: %d channels do not divide into %d groups", d.c, d.groups);
    Y5_REQUIRE(d.act == Y5_ACT_NONE || d.act == Y5_ACT_LEAKY || d.act == Y5_ACT_SILU, "group_norm: activation %d", d.act);
    Y5_REQUIRE(d.eps >= 0.f, "group_norm: eps %g", d.eps);
    NormShape s{};
    const int V = 16 / norm_elem_size(d.dtype);
    s.c = d.c;
    s.groups = d.groups;
    s.cpg = d.c / d.groups;
    s.k = V / norm_gcd(d.c, V);
    Y5_REQUIRE((long long)d.c * s.k <= kNormMaxW, "group_norm: %d channels (at most %d at this divisibility)", d.c, kNormMaxW / s.k);
    s.W = d.c * s.k;
    s.cols = s.W / V;
    s.pixels = d.pixels;
    s.vrows = (d.pixels + s.k - 1) / s.k;
    s.batch = d.batch;
    s.act = d.act;
    s.param_dtype = d.param_dtype;
    s.slope = d.act == Y5_ACT_LEAKY ? d.slope : 1.f;
    s.eps = d.eps;
    // Chunks of the split form: as many workgroups as the chip holds at a time (1024 of 256 threads: 105 MB of 32 images in 27 us; twice
    // as many leave a second, emptier round and more to merge: 32 us), at least 8 KiB each, at most kNormMaxChunks of an image (every
    // workgroup of the second pass reads all of them)
    const long long bytes = (long long)d.pixels * d.c * norm_elem_size(d.dtype);
    long long chunks = 1024 / d.batch < kNormMaxChunks ? 1024 / d.batch : kNormMaxChunks;
    chunks = chunks < bytes / 8192 ? chunks : bytes / 8192;
    chunks = chunks < 1 ? 1 : chunks;
    s.chunk_rows = (int)((s.vrows + chunks - 1) / chunks);
    s.chunks = (s.vrows + s.chunk_rows - 1) / s.chunk_rows;
    s.by_c = make_fastdiv((unsigned)s.c);
    s.by_cpg = make_fastdiv((unsigned)s.cpg);
    s.by_cols = make_fastdiv((unsigned)s.cols);
    *out = s;
    return Y5_OK;
}

inline int norm_check_pitch(const y5_group_norm_desc& d, const NormShape& s, const char* what, const void* p, int ld) {
    Y5_REQUIRE(p, "group_norm: null %s", what);
    Y5_REQUIRE(ld >= d.c && (s.k == 1 || ld == d.c), "group_norm: %s pitch %d for %d channels (a pitch above the channels needs channels in whole 16-byte vectors)", what, ld, d.c);
    Y5_REQUIRE(reinterpret_cast<uintptr_t>(p) % norm_elem_size(d.dtype) == 0, "group_norm: misaligned %s", what);
    return Y5_OK;
}

// What a workgroup of the split form's second pass reads: 32 KiB (merging the chunks' statistics is then little beside it; 64 KiB: 56
// instead of 52 us for the gradient of 105 MB, 128 KiB: 60), less where that would leave compute units without one
inline long long norm_run_bytes(const NormShape& s, int esize) {
    const long long each = (long long)s.batch * s.pixels * s.c * esize / 2048;
    return each < 4096 ? 4096 : each > 32768 ? 32768 : each;
}

inline size_t norm_align16(size_t n) { return (n + 15) / 16 * 16; }
