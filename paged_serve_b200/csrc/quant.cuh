// The 8-bit KV cache format: codes and their conversion.
//
// A row x (one token's K or V of one KV head, D values) is held as D codes and
// one fp32 scale, x[d] ~ code[d] * scale:
//   scale   = max(max_d |x[d]| / qmax, 2^-126)     qmax = 448 (e4m3) or 127 (int8)
//   code[d] = round_to_code(x[d] * (1 / scale))     ties to even
// with every operation rounded to fp32, so the codes are reproducible to the
// bit. 2^-126 keeps 1 / scale finite for rows of zeros (their codes are 0).
// A NaN or an infinity in a row makes its scale NaN, and with it every value read
// back from the row.
#pragma once

#include "common.cuh"

namespace ps {

// kInvHi + kInvLo = 1 / kMax to twice float's precision: the constant's reciprocal rounded
// to float, and what that leaves, rounded again.
struct CodeE4M3 {
  static constexpr float kMax = 448.f;
  static constexpr float kInvHi = static_cast<float>(1.0 / 448.0);
  static constexpr float kInvLo = static_cast<float>(1.0 / 448.0 - static_cast<double>(kInvHi));
};
struct CodeInt8 {
  static constexpr float kMax = 127.f;
  static constexpr float kInvHi = static_cast<float>(1.0 / 127.0);
  static constexpr float kInvLo = static_cast<float>(1.0 / 127.0 - static_cast<double>(kInvHi));
};

constexpr float kMinScale = 1.17549435e-38f;  // 2^-126

// max(a, b), NaN when either is NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Largest of |a|, |b|, |c|, NaN when one of them is.
__device__ __forceinline__ float max3_abs_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// amax / kMax, correctly rounded, as fma(amax, kInvHi, amax * kInvLo): division by a
// constant known in advance (Brisebarre, Muller and Raina 2004); for both constants every
// significand gives the division's result (tested). Below 2^-60 the small product could
// underflow, so the division itself is used there.
template <typename C>
__device__ __forceinline__ float row_scale(float amax) {
  float q = __fmaf_rn(amax, C::kInvHi, __fmul_rn(amax, C::kInvLo));
  if (amax < 0x1p-60f) q = __fdiv_rn(amax, C::kMax);
  // amax * 0 is NaN for an infinite maximum and 0 otherwise.
  return max_nan(__fadd_rn(q, __fmul_rn(amax, 0.f)), kMinScale);
}

// Four values (already divided by the scale) to four codes, the first in the low byte.
template <typename C>
__device__ __forceinline__ uint32_t encode4(float2 ab, float2 cd);
template <>
__device__ __forceinline__ uint32_t encode4<CodeE4M3>(float2 ab, float2 cd) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\t"
      "mov.b32 %0, {lo, hi};\n\t}"
      : "=r"(r)
      : "f"(ab.x), "f"(ab.y), "f"(cd.x), "f"(cd.y));
  return r;
}
template <>
__device__ __forceinline__ uint32_t encode4<CodeInt8>(float2 ab, float2 cd) {
  // |x * (1/scale)| <= 127 * (1 + 2^-22), so rounding to an integer never leaves
  // [-127, 127]. Adding 1.5 * 2^23 rounds to nearest even and leaves the integer
  // in the low byte of the sum's bits. Scalar additions: a packed one is fused with the
  // packed multiplication before it, which then is not rounded (some codes came out
  // one off).
  constexpr float kRound = 12582912.f;
  const uint32_t x = __float_as_uint(__fadd_rn(ab.x, kRound));
  const uint32_t y = __float_as_uint(__fadd_rn(ab.y, kRound));
  const uint32_t z = __float_as_uint(__fadd_rn(cd.x, kRound));
  const uint32_t w = __float_as_uint(__fadd_rn(cd.y, kRound));
  return __byte_perm(__byte_perm(x, y, 0x0040), __byte_perm(z, w, 0x0040), 0x5410);
}

// Four codes to two pairs of fp16 values, exactly: every e4m3 code and every
// int8 code is an fp16 value. lo = codes 0 and 1, hi = codes 2 and 3.
template <typename C>
__device__ __forceinline__ void decode4(uint32_t codes, uint32_t& lo, uint32_t& hi);
template <>
__device__ __forceinline__ void decode4<CodeE4M3>(uint32_t codes, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\t"
      "mov.b32 {a, b}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, a;\n\t"
      "cvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(codes));
}
template <>
__device__ __forceinline__ void decode4<CodeInt8>(uint32_t codes, uint32_t& lo, uint32_t& hi) {
  // code + 128 as the low mantissa byte of an fp16 in [1024, 2048) is
  // 1024 + code + 128; the subtraction is exact.
  const uint32_t u = codes ^ 0x80808080u;
  const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140);
  const uint32_t b = __byte_perm(u, 0x64646464u, 0x4342);
  const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));  // 1152
  const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), bias);
  const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&b), bias);
  lo = *reinterpret_cast<const uint32_t*>(&x);
  hi = *reinterpret_cast<const uint32_t*>(&y);
}

}  // namespace ps
