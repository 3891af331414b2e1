// The arithmetic of 8-bit rows, shared by the kernels that quantise (rows_i8.hip, gemm_i8_rows.hip, gemm_i8_few.hip).  Included
// inside an anonymous namespace.
#pragma once

constexpr float kZeroRow = 7.52316384526264e-37f;  // 2^-120

// The multiplier of a row with the largest magnitude `bits` (as the bits of a float); 0 for a row of zeros.
__device__ __forceinline__ float row_scale(unsigned bits, float* a) {
    const float m = __uint_as_float(bits);
    *a = m >= kZeroRow ? m : 0.f;
    if (bits >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
    // a / 127 to nearest: quotient by the rounded reciprocal, its exact remainder, one step (that is what a division does, without the
    // cases it also has to cover; equal to it for every value from 2^-120 up)
    const float y = 1.f / 127.f, q = *a * y;
    return __builtin_fmaf(__builtin_fmaf(-q, 127.f, *a), y, q);
}

// The whole number nearest to v * 127 / a, as the low byte of a word (the rest of the word is not zero).  Adding 1.5 * 2^23 (2^52)
// leaves the number, to nearest with ties to even, in the low bits of the mantissa: one instruction for rounding and
// converting.  The product is rounded before that, not in one step with it: its rounding takes the error of 127 / a back where the
// quotient is exactly a half, which 16-bit values make of a few in ten thousand, and those then go to even.  fp32 values are
// scaled in 64 bits: their 24 digits leave no room for the error of 127 / a, which would put values next to a half on its other side.
struct Inv32 {
    float f;
    __device__ __forceinline__ void set(float a, bool ok) { f = ok && a > 0.f ? 127.f / a : 0.f; }
    __device__ __forceinline__ unsigned operator()(float v) const {
#pragma clang fp contract(off)
        const float t = v * f;
        return __float_as_uint(t + 12582912.f);
    }
};
struct Inv64 {
    double f;
    __device__ __forceinline__ void set(float a, bool ok) { f = ok && a > 0.f ? 127.0 / (double)a : 0.0; }
    __device__ __forceinline__ unsigned operator()(float v) const {
#pragma clang fp contract(off)
        const double t = (double)v * f;
        return (unsigned)__builtin_bit_cast(unsigned long long, t + 6755399441055744.0);
    }
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

// The low bytes of four words; zeros for a row that is not fine
__device__ __forceinline__ int pack_bytes(unsigned a, unsigned b, unsigned c, unsigned d, bool fine) {
    const unsigned lo = __builtin_amdgcn_perm(b, a, 0x0c0c0400u), hi = __builtin_amdgcn_perm(d, c, 0x0c0c0400u);
    return fine ? (int)__builtin_amdgcn_perm(hi, lo, 0x05040100u) : 0;
}

// The largest of `top` over aligned groups of `lanes` lanes (a power of two), FROM of them known to hold the same already.  Moves between
// lanes of 16 and swaps of rows, which cost an instruction each; a shuffle through LDS costs its latency.
template <int CTRL>
__device__ __forceinline__ unsigned max_moved(unsigned top) {
    const unsigned o = (unsigned)__builtin_amdgcn_update_dpp(0, (int)top, CTRL, 0xf, 0xf, true);
    return o > top ? o : top;
}
template <int FROM = 1>
__device__ __forceinline__ unsigned max_over(unsigned top, int lanes) {
    if (FROM < 2 && lanes > 1) top = max_moved<0xb1>(top);    // lane ^ 1
    if (FROM < 4 && lanes > 2) top = max_moved<0x4e>(top);    // lane ^ 2
    if (FROM < 8 && lanes > 4) top = max_moved<0x141>(top);   // mirrored in 8
    if (FROM < 16 && lanes > 8) top = max_moved<0x140>(top);  // mirrored in 16
#if defined(__HIP_DEVICE_COMPILE__)
    if (lanes > 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(top, top, false, false);
        top = r[0] > r[1] ? r[0] : r[1];
    }
    if (lanes > 32) {
        const auto r = __builtin_amdgcn_permlane32_swap(top, top, false, false);
        top = r[0] > r[1] ? r[0] : r[1];
    }
#endif
    return top;
}
