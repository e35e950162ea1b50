// Device helpers of the position rotation and the q8_0 / q4_0 quantisers,
// shared by every kernel that rotates or requantises rows, so that they all
// give the same bits. Files that include this are compiled with -fmad=false.
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cstdint>

namespace kvmret {
namespace {

__device__ __forceinline__ float h2f(uint16_t h) {
    return __half2float(__ushort_as_half(h));
}
__device__ __forceinline__ uint16_t f2h(float f) {
    return __half_as_ushort(__float2half_rn(f));
}

// RoPE table: cos / sin of the float angle pos * theta[i] (rope.cpp:27-33).
// The angle is the reference's float product; cos and sin are evaluated in
// double and rounded once to float, i.e. correctly rounded, so the table does
// not add the few-ulp error of a float sincos. Window positions come from a
// per-context table built once at creation; the stateless entry points build a
// temporary table for their positions.
__device__ __forceinline__ float2 rope_cs(int32_t pos, float theta) {
    const float ang = __fmul_rn(static_cast<float>(pos), theta);
    double s, c;
    sincos(static_cast<double>(ang), &s, &c);
    return make_float2(__double2float_rn(c), __double2float_rn(s));
}

// round-half-away-from-zero (C roundf) for |y| < 2^23: truncate y + s, s =
// copysign(0.5 - 2^-25, y) (the float just below one half). Exactness: for
// |y| >= 1 the sum is exact or rounds only across the binade edge, where
// truncation already gives the rounded value; for |y| < 1 the only
// candidates for a wrong carry are the ties y = +-0.5 (sum 1 - 2^-25 rounds
// to 1, as wanted) and y = +-(0.5 - 2^-25) (sum 1 - 2^-24, exact, truncates
// to 0). Checked against the host roundf on every float of magnitude < 256.
// The truncation is the conversion to an integer (toward zero), whose low
// byte is then the int8.
__device__ __forceinline__ int round_away_int(float y) {
    return __float2int_rz(__fadd_rn(y, copysignf(0.49999997f, y)));
}

__device__ __forceinline__ uint32_t pack_low_bytes(uint32_t b0, uint32_t b1, uint32_t b2,
                                                   uint32_t b3) {
    return __byte_perm(__byte_perm(b0, b1, 0x0040u), __byte_perm(b2, b3, 0x0040u), 0x5410u);
}

// x / 127 correctly rounded, by division by a constant known in advance
// (Brisebarre, Muller and Raina, IEEE Trans. Computers 53(8), 2004): with
// zh = RN(1/127) and zl = RN(1/127 - zh), RN(x zh + RN(x zl)) is the
// correctly rounded quotient. Checked against IEEE division on every
// non-negative float: it holds for all x >= 2^-100 (below that x zl loses
// bits to underflow), so smaller x take the division.
__device__ __forceinline__ float div127_rn(float x) {
    if (!(x >= 0x1p-100f)) return __fdiv_rn(x, 127.0f);
    return __fmaf_rn(x, 0x1.020408p-7f, __fmul_rn(x, 0x1.020408p-35f));
}

}  // namespace
}  // namespace kvmret
