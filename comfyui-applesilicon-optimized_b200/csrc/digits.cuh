// Exact-integer products of 16-bit activations: a value scaled by a power of two is
// split into three int8 digits, v = p0 + p1 / 128 + p2 / 128^2, that the integer
// tensor path multiplies with codes as they are stored.
#pragma once

#include "numerics.cuh"

namespace b200q {

// Three int8 digits of v, |v| < 64, in the low bytes: adding 1.5 * 2^23 leaves the
// nearest integer in the mantissa's low bits.
__device__ __forceinline__ void digits3(float v, uint32_t& p0, uint32_t& p1, uint32_t& p2) {
  const float m = 12582912.0f;
  const float a = v + m;
  const float r = (v - (a - m)) * 128.0f;
  const float c = r + m;
  const float e = (r - (c - m)) * 128.0f + m;
  p0 = __float_as_uint(a);
  p1 = __float_as_uint(c);
  p2 = __float_as_uint(e);
}
// 2^E above the largest |value| of 16-bit bits `top`, as (2^-E * 64, 2^E / 64);
// NaN for a row holding inf or NaN.
__device__ __forceinline__ void digit_scale(uint32_t top, int f16, float* down, float* up) {
  const uint16_t tb = static_cast<uint16_t>(top);
  const float m = f16 ? __half2float(*reinterpret_cast<const __half*>(&tb))
                      : __uint_as_float(top << 16);
  int ex = static_cast<int>(__float_as_uint(m) >> 23);  // biased: m < 2^(ex - 126)
  const bool bad = ex == 255;
  ex = min(max(ex, 8), 254);
  *down = __uint_as_float(static_cast<uint32_t>(259 - ex) << 23);
  *up = bad ? __uint_as_float(0x7FC00000u) : __uint_as_float(static_cast<uint32_t>(ex - 5) << 23);
}
// The low bytes of four words as one.
__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

}  // namespace b200q
