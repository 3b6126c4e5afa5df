// Microscaling formats: 32 neighbours along a row share a power of two.
//
// A group of 32 values is 32 small floating-point numbers times 2^(s - 127), s a byte (255: the group is no number). Rows of
// activations hold e4m3 numbers (8 bits, up to 448), matrices e2m1 numbers (4 bits: 0, 0.5, 1, 1.5, 2, 3, 4, 6). gfx950's conversions
// (v_cvt_scalef32_pk_bf16_fp4, _bf16_fp8, _f32_fp4) give two of them with their scale an instruction, exactly: a few bits times a power of two are a
// bfloat16.
//
// The group's power of two follows from its largest magnitude alone, amax = m 2^x with 1 <= m < 2: s - 127 = x - emax, one more
// where m > 1.75; emax = 8 for e4m3, 2 for e2m1. In e4m3 the largest number is 1.75 * 2^8, so nothing is cut off; in e2m1 what lies in
// (6, 7] becomes 6, off by at most 1, which is half the step above 4 and so no more than a rounding. (The other rule in use, x - emax
// throughout, cuts e4m3's upper eighth off.)
//
// A matrix [N, K] is laid out once as the matrix instructions read it: blocks of 16 rows (a strip) and 128 k (a chunk), strip after
// strip, 1,088 bytes each. Lane 16 g + r of a wave finds the 32 numbers of row r and group g of the block in bytes [16 lane, 16 lane +
// 16), k ascending from the low half of the first byte, and their scale in byte 1,024 + lane. A wave's read of a block is one
// stretch of memory and its registers are operands as they are. What lies outside the matrix holds zeros with scale 0.
#pragma once

#include "common.h"

namespace liyab {

constexpr int kMxGroup = 32;
constexpr int kMxChunk = 128;        // k of a block
constexpr int kMxStrip = 16;         // rows of a block
constexpr int kMxBlockBytes = 1088;  // 64 lanes x 16 bytes, then 64 scales
constexpr int kE4m3Max = 8, kE2m1Max = 2;  // exponents of the largest numbers

typedef __attribute__((ext_vector_type(2))) float mx_f32x2;
typedef __attribute__((ext_vector_type(2))) __bf16 mx_bf16x2;

inline __host__ __device__ int mx_chunks(int k) { return (k + kMxChunk - 1) / kMxChunk; }
inline __host__ __device__ int mx_strips(int n) { return (n + kMxStrip - 1) / kMxStrip; }

// |v| as bits: magnitudes compare as these do, infinities and NaN above every number.
__device__ __forceinline__ uint32_t mx_magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// A group's scale from the bits of its largest magnitude (the carry out of the mantissa is m > 1.75).
__device__ __forceinline__ uint32_t mx_scale(uint32_t amax, int emax) {
    const int s = static_cast<int>((amax + 0x1fffffu) >> 23) - emax;
    return amax >= 0x7f800000u ? 255u : static_cast<uint32_t>(s > 0 ? s : 0);
}
// What the group's values are multiplied by ahead of rounding, 2^(127 - s): s <= 253 where it is a number's. (Exact: a product by a power
// of two, and what underflows is far below half the least number.)
__device__ __forceinline__ float mx_factor(uint32_t s) { return __uint_as_float((254u - s) << 23); }
// 2^(s - 127) as the conversions read it: they look at the exponent's bits alone, so that 0 is 2^-127 and 255 makes every value NaN.
__device__ __forceinline__ float mx_power(uint32_t s) { return __uint_as_float(s << 23); }

// Eight values of a group in e4m3, rounded to nearest, ties to even; zeros where the group is no number.
__device__ __forceinline__ uint2 mx_e4m3(const float (&v)[8], uint32_t s) {
    const float f = mx_factor(s);
    int lo = 0, hi = 0;
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * f, v[1] * f, lo, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * f, v[3] * f, lo, true);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4] * f, v[5] * f, hi, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[6] * f, v[7] * f, hi, true);
    return s == 255u ? make_uint2(0u, 0u) : make_uint2(static_cast<uint32_t>(lo), static_cast<uint32_t>(hi));
}

}  // namespace liyab
