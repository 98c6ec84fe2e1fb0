// The 8-bit form of an activation.  A pixel's (row's) channels are cut into blocks of 32; a block shares the power of two
// 2^e, the smallest with max|x| <= 127 * 2^e (e in [-126, 121]), and holds q = round-to-even(x / 2^e), |q| <= 127, per
// element.  So |x - q 2^e| <= 2^(e-1) (up to 2^e in the one block exponent 121, where the next power would leave
// float32), and q 2^e is exact in bfloat16 as well as in float32: seven bits of significand.  The code -128 stands for
// an element that is not finite and reads back as NaN; such an element does not enter its block's maximum.
//   codes  int8  [rows][channels]
//   exps   uint8 [rows][ceil(channels / 32)], e + 127
#pragma once
#include <hip/hip_runtime.h>

namespace sg2im {

constexpr int C8_BLOCK = 32;

__device__ __forceinline__ float c8_magnitude(float v) {        // |v|, 0 for what is not finite
  const unsigned b = __float_as_uint(v) & 0x7fffffffu;
  return b < 0x7f800000u ? __uint_as_float(b) : 0.f;
}
// e + 127 of a block: with amax = 1.f * 2^(E-127), amax <= 127 * 2^(E-133)  <=>  1.f <= 127/64  <=>  f <= 0x7E0000
__device__ __forceinline__ int c8_exponent(float amax) {
  const unsigned b = __float_as_uint(amax);
  const int e = (int)(b >> 23) - ((b & 0x7fffffu) <= 0x7E0000u ? 133 : 132);
  return (e < -126 ? -126 : e > 121 ? 121 : e) + 127;
}
__device__ __forceinline__ float c8_scale(int biased) { return __uint_as_float((unsigned)biased << 23); }            // 2^e
__device__ __forceinline__ float c8_inverse(int biased) { return __uint_as_float((unsigned)(254 - biased) << 23); }  // 2^-e
__device__ __forceinline__ signed char c8_encode(float v, float inverse) {
  if ((__float_as_uint(v) & 0x7fffffffu) >= 0x7f800000u) return (signed char)-128;
  const float q = rintf(v * inverse);
  return (signed char)(int)fminf(fmaxf(q, -127.f), 127.f);
}
__device__ __forceinline__ float c8_decode(signed char q, float scale) {
  return q == -128 ? __uint_as_float(0x7fc00000u) : (float)q * scale;
}

}  // namespace sg2im
