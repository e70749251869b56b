// 4-bit floating point rows (E2M1 values with a scale per block): the record a
// quantized row is kept in and the arithmetic of the quantizers.
//
//   NVFP4: a row's factor is the smallest 2^e with 6 * 448 * 2^e >= max |x| (at
//     least 2^-100), each block of 16 has scale = e4m3(max |x| / (6 factor)),
//     and x becomes e2m1(x / (scale factor));
//   MXFP4: each block of 32 has scale 2^e, the smallest with 6 * 2^e >= max |x|
//     (e8m0: e + 127), and x becomes e2m1(x / 2^e).
// All roundings are to nearest, ties to even, and the largest E2M1 value is 6.  A
// power of two as the row's factor adds no rounding, so a value halfway between
// two codes is seen as one (a factor of amax / 2688 moved such ties, 0.05 % of
// the scales of normally distributed bf16 rows, by its own rounding).  A NaN or an infinity makes the
// factor (NVFP4: the whole row) or the block's scale (MXFP4) a NaN.
//
// A record is one run of bytes per row: K / 2 of codes (the even column in the
// low bits), K / 16 or K / 32 scales, and for NVFP4, on the next multiple of
// four, the f32 factor; padded with zeros to a multiple of 16.  One record moves
// whole where rows are sorted by expert, and rows of records suit TMA's strides.
#pragma once

#include "common.cuh"
#include "fp8_device.cuh"
#include "layout.cuh"
#include "swiglu.cuh"
#include "vec.cuh"

namespace b200moe {

constexpr int kNv = 0, kMx = 1;  // as B200MOE_NVFP4 and B200MOE_MXFP4

__host__ __device__ constexpr int fp4_block(int fmt) { return fmt == kMx ? 32 : 16; }
__host__ __device__ constexpr int fp4_factor_at(int64_t K) { return int(K / 2 + (K / 16 + 3) / 4 * 4); }
__host__ __device__ constexpr int fp4_used(int fmt, int64_t K) {
  return fmt == kMx ? int(K / 2 + K / 32) : fp4_factor_at(K) + 4;
}
__host__ __device__ constexpr int fp4_stride(int fmt, int64_t K) { return (fp4_used(fmt, K) + 15) / 16 * 16; }

constexpr float kFp4Floor = 0x1p-100f;

__device__ __forceinline__ float fp4_nan() { return __uint_as_float(0x7fffffffu); }

// The row's factor from its largest magnitude's bits (a NaN above infinity, as abs_bits orders them).
__device__ __forceinline__ float nvfp4_factor(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return fp4_nan();
  const uint32_t b = max(amax_bits, __float_as_uint(kFp4Floor));
  // amax = m 2^x, 1 <= m < 2: 2688 = 1.3125 * 2^11 reaches m up to 1.3125 with 2^(x - 11)
  const int x = int(b >> 23) - 127;
  const int e = (b & 0x7fffffu) <= 0x280000u ? x - 11 : x - 10;
  return __uint_as_float(uint32_t(e + 127) << 23);
}

// A block's E4M3 scale byte and its scale times the factor.
__device__ __forceinline__ uint32_t nvfp4_scale(float bmax, float factor, float& unit) {
  uint16_t pair;
  const float s = __fdiv_rn(bmax, 6.f * factor);  // 6 * 2^e is exact
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %1;" : "=h"(pair) : "f"(s));
  const uint32_t byte = factor == factor ? pair & 0x7fu : 0u;
  const uint32_t ex = byte >> 3, mn = byte & 7u;
  const float v = ex ? __uint_as_float(((ex + 120u) << 23) | (mn << 20)) : float(mn) * 0x1p-9f;
  unit = byte ? v * factor : 0.f;
  return byte;
}

// A block's E8M0 byte and 2^-e; bmax a magnitude (or a NaN).
__device__ __forceinline__ uint32_t mxfp4_scale(float bmax, float& inv) {
  const uint32_t b = __float_as_uint(bmax);
  if (b >= 0x7f800000u) {
    inv = 0.f;
    return 255u;
  }
  if (b == 0u) {
    inv = 1.f;
    return 127u;
  }
  const int e = max(mx_exponent(bmax), -127);  // at most 126
  inv = __uint_as_float(uint32_t(127 - e) << 23);
  return uint32_t(e + 127);
}

// Eight values to E2M1, v[0] in the lowest four bits.
__device__ __forceinline__ uint32_t e2m1x8(const float* v) {
  uint32_t o;
  asm("{ .reg .b8 b0, b1, b2, b3;\n"
      " cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n"
      " cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n"
      " mov.b32 %0, {b0, b1, b2, b3}; }"
      : "=r"(o)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return o;
}

// 16 values of one NVFP4 block to codes. The quotient is rounded correctly by one step from the product with the
// reciprocal (Markstein: the remainder x - q unit is exact in a fused operation), so ties are the definition's.
__device__ __forceinline__ uint2 nvfp4_codes(const float (&v)[16], float unit) {
  const float inv = unit > 0.f ? __frcp_rn(unit) : 0.f;
  float t[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float q = __fmul_rn(v[i], inv);
    t[i] = __fmaf_rn(__fmaf_rn(-q, unit, v[i]), inv, q);
  }
  uint2 o = make_uint2(e2m1x8(t), e2m1x8(t + 8));
  if (!(unit > 0.f)) o = make_uint2(0u, 0u);
  return o;
}

// 16 of the 32 values of an MXFP4 block (inv 0: a block whose scale is a NaN, whatever its codes).
__device__ __forceinline__ uint2 mxfp4_codes(const float (&v)[16], float inv) {
  float t[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) t[i] = v[i] * inv;
  return make_uint2(e2m1x8(t), e2m1x8(t + 8));
}

__device__ __forceinline__ float magnitude16(const float (&v)[16]) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) m = max_nan(m, fabsf(v[i]));
  return m;
}

// The bytes of a record behind its scales: zeros, and the factor.
__device__ __forceinline__ void finish_record(uint8_t* rec, int fmt, int K, float factor) {
  const int begin = K / 2 + K / fp4_block(fmt), end = fp4_stride(fmt, K);
  if (fmt == kNv && begin % 16 == 0) {  // K a multiple of 256
    *reinterpret_cast<uint4*>(rec + begin) = make_uint4(__float_as_uint(factor), 0u, 0u, 0u);
    return;
  }
  for (int i = begin; i < end; ++i) rec[i] = 0;
  if (fmt == kNv) *reinterpret_cast<float*>(rec + fp4_factor_at(K)) = factor;
}

// A product's factors, its row's and its matrix's: sum * first * second. Their product and 1 where that is a normal number (a
// power of two as the row's makes it exact: one rounding). Else both, the one first that leaves the sum (at most 2^40) inside
// f32 if the result is: rows near f32's largest times a small matrix factor came out infinite as (sum * row's) * matrix's.
struct Fp4Factors {
  float first, second;
};
__device__ __forceinline__ Fp4Factors fp4_factors(float row, float matrix) {
  const float both = row * matrix, m = fabsf(both);
  if ((m >= 0x1p-126f && m < INFINITY) || !(fabsf(row) > 0.f && fabsf(matrix) > 0.f)) return {both, 1.f};  // 0, NaN too
  const bool less = fabsf(row) < fabsf(matrix);
  const float small = less ? row : matrix, large = less ? matrix : row;
  return m < 1.f ? Fp4Factors{large, small} : Fp4Factors{small, large};
}

__device__ __forceinline__ float e4m3_f32(uint32_t byte) {  // 0x7f / 0xff are NaN
  if ((byte & 0x7fu) == 0x7fu) return fp4_nan();
  const uint32_t ex = (byte >> 3) & 15u, mn = byte & 7u;
  const float v = ex ? __uint_as_float(((ex + 120u) << 23) | (mn << 20)) : float(mn) * 0x1p-9f;
  return byte & 0x80u ? -v : v;
}
__device__ __forceinline__ float e8m0_f32(uint32_t byte) {  // 255 is NaN
  return byte == 255u ? fp4_nan() : byte ? __uint_as_float(byte << 23) : 0x1p-127f;
}

}  // namespace b200moe
