// The arithmetic of 8-bit rows, shared by the kernels that quantise (rows_i8.hip, gemm_i8_rows.hip, gemm_i8_few.hip).  Included
// inside an anonymous namespace.
#pragma once

constexpr float kZeroRow = 7.52316384526264e-37f;  // 2^-120

// The multiplier of a row with the largest magnitude `bits` (as the bits of a float); 0 for a row of zeros.
__device__ __forceinline__ float row_scale(unsigned bits, float* a) {
    const float m = __uint_as_float(bits);
    *a = m >= kZeroRow ? m : 0.f;
    if (bits >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
    return *a / 127.f;
}

// The whole number nearest to v * 127 / a.  fp32 values are scaled in 64 bits: their 24 digits leave no room for an error of
// the multiplication, which would put values next to a half on its other side.  16-bit values have 13 digits of room.
struct Inv32 {
    float f;
    __device__ __forceinline__ void set(float a, bool ok) { f = ok && a > 0.f ? 127.f / a : 0.f; }
    __device__ __forceinline__ int operator()(float v) const { return (int)__builtin_rintf(v * f); }
};
struct Inv64 {
    double f;
    __device__ __forceinline__ void set(float a, bool ok) { f = ok && a > 0.f ? 127.0 / (double)a : 0.0; }
    __device__ __forceinline__ int operator()(float v) const { return (int)__builtin_rint((double)v * f); }
};
template <typename T, bool NORM>
struct InvOf {
    typedef Inv32 type;
};
template <>
struct InvOf<float, false> {
    typedef Inv64 type;
};

// the larger of two magnitudes as the bits of floats: NaN > infinity > every number
__device__ __forceinline__ unsigned max_bits(unsigned top, float v) {
    const unsigned u = __float_as_uint(v) & 0x7fffffffu;
    return u > top ? u : top;
}

__device__ __forceinline__ int pack_bytes(int a, int b, int c, int d) {  // each in [-128, 127]
    const unsigned lo = __builtin_amdgcn_perm((unsigned)b, (unsigned)a, 0x0c0c0400u), hi = __builtin_amdgcn_perm((unsigned)d, (unsigned)c, 0x0c0c0400u);
    return (int)__builtin_amdgcn_perm(hi, lo, 0x05040100u);
}
