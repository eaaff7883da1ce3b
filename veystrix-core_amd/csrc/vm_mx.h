// MX rows: e4m3 values with one e8m0 scale per group of 32 along the row.
//
// The scale of a group is the least 2^e, e >= -127, with max|v| <= 448 * 2^e (448 is e4m3's largest value), stored as
// e + 127; a value is v * 2^-e rounded to the nearest e4m3, ties to even.  No value saturates, and the product with
// 2^-e is exact in fp32 but for results below its normal range, so the one rounding is e4m3's.  A group that holds an
// infinity or a NaN has the scale 0xff (NaN) and NaN values.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace vm {

constexpr uint32_t kMxGroup = 32;

// Magnitude bits whose unsigned maximum over a group is the group's largest |v|; NaN is above infinity.
__device__ __forceinline__ uint32_t mx_magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// The e8m0 byte from the largest magnitude's bits: 448 = 1.75 * 2^8, so the exponent goes one up where the mantissa
// is over .75 (0x600000): adding 0x1fffff carries exactly then.
__device__ __forceinline__ uint32_t mx_scale(uint32_t magnitude) {
  if (magnitude >= 0x7f800000u) return 0xffu;
  const uint32_t e = (magnitude + 0x1fffffu) >> 23;
  return e > 8u ? e - 8u : 0u;
}

// 2^-e of a finite scale byte (at most 247: a normal float).
__device__ __forceinline__ float mx_inverse(uint32_t scale) { return __uint_as_float((254u - scale) << 23); }

// Four values of one group, packed; `scale` is the group's byte.
__device__ __forceinline__ uint32_t mx_pack4(float a, float b, float c, float d, uint32_t scale) {
  if (scale == 0xffu) return 0x7f7f7f7fu;
  const float m = mx_inverse(scale);
  int v = __builtin_amdgcn_cvt_pk_fp8_f32(a * m, b * m, 0, false);
  v = __builtin_amdgcn_cvt_pk_fp8_f32(c * m, d * m, v, true);
  return static_cast<uint32_t>(v);
}

}  // namespace vm
