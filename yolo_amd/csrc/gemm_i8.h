// Pieces shared by the 8-bit product's kernels (included inside an anonymous namespace after conv_common.h).
#pragma once

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
    int nk, tiles_n, tiles_total;  // phased kernel: 128-byte K-tiles, output tiles
    int whole;                     // its output: rows start on 16 bytes, channels are whole 16-byte vectors
};

// The activation is a template parameter: an epilogue holds up to 128 values a lane in named registers, and testing for it at
// run time there is code that every tile pays for.
template <int ACT, int N>
__device__ __forceinline__ void act_n(float (&v)[N], float slope) {
    if constexpr (ACT == Y5_ACT_LEAKY) {
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = v[e] > 0.f ? v[e] : v[e] * slope;
    } else if constexpr (ACT == Y5_ACT_SILU) {
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = v[e] * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(v[e] * -1.44269504088896341f));
    }
}

// N consecutive values (16 or 8 bytes) stored as one value at element alignment (as elements the compiler would split the store up
// beside the branch of a cut-off one)
template <typename T, int N>
__device__ __forceinline__ void st_out(T* p, const T* v) {
    typedef T Vec __attribute__((ext_vector_type(N)));
    typedef unsigned Raw __attribute__((ext_vector_type(N * sizeof(T) / 4)));
    struct __attribute__((packed, aligned(sizeof(T)))) At {
        Raw v;
    };
    Vec o;
#pragma unroll
    for (int e = 0; e < N; ++e) o[e] = v[e];
    reinterpret_cast<At*>(p)->v = __builtin_bit_cast(Raw, o);
}

// 16 bytes at descriptor base + voff; lanes that fail the range check store nothing
#if defined(__HIP_DEVICE_COMPILE__)
__device__ __forceinline__ void st16_buf(i32x4 v, BufRsrc r, unsigned voff) {
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), r, voff, 0, 0);
}
#else
__device__ inline void st16_buf(i32x4, BufRsrc, unsigned) {}
#endif

inline int cu_count() {
    static std::atomic<int> cached[64];
    const int dev = y5_current_device();
    int n = cached[dev].load();
    if (n == 0) {
        int real = 0;
        if (hipGetDevice(&real) != hipSuccess || hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, real) != hipSuccess || n <= 0) n = 256;
        cached[dev].store(n);
    }
    return n;
}

inline GemmArgs make_gemm_args(const y5_gemm_i8_desc& d) {
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
    return g;
}
