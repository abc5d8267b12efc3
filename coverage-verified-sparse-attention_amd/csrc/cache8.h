// Values of 8 bits (e4m3 payloads) with powers of two as scales, held as their
// exponents' bytes (2^(byte - 127), 255: NaN): what the kernels that write such
// caches share.
#pragma once
#include "cvsa_common.h"

namespace cvsa {

constexpr int kLowExponent = -110, kHighExponent = 119;  // of scales that are written

// The byte of the smallest scale 2^e with top <= 448 * 2^e = 1.75 * 2^(8 + e), top
// given by its bits.
__device__ __forceinline__ int scale_byte(uint32_t top) {
  const int e = (int)(top >> 23) - 127 - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, kLowExponent), kHighExponent) + 127;
}
// 2^e, subnormal ones too (the inverse of a caller's own scale of 2^127).
__device__ __forceinline__ float power_of_two(int e) { return ldexpf(1.f, e); }
__device__ __forceinline__ bool finite_bits(uint32_t u) {
  return (u & 0x7f800000u) != 0x7f800000u;
}

// 8 values times `inv`, rounded to nearest even; NaN and infinities become NaN.
// clamp: finite ones past 448 become it (those of the largest scale; others cannot
// pass it).
__device__ __forceinline__ uint2 to_8_bits(const float (&f)[8], float inv, bool clamp) {
  float y[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = f[e] * inv;
  if (clamp) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (finite_bits(__float_as_uint(f[e]))) y[e] = fminf(fmaxf(y[e], -448.f), 448.f);
  }
  uint2 w;
  w.x = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
  w.x = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w.x, true);
  w.y = __builtin_amdgcn_cvt_pk_fp8_f32(y[4], y[5], 0, false);
  w.y = __builtin_amdgcn_cvt_pk_fp8_f32(y[6], y[7], w.y, true);
  return w;
}
__device__ __forceinline__ void from_8_bits(const uint2 &w, float (&f)[8]) {
  f[0] = __builtin_amdgcn_cvt_f32_fp8(w.x, 0);
  f[1] = __builtin_amdgcn_cvt_f32_fp8(w.x, 1);
  f[2] = __builtin_amdgcn_cvt_f32_fp8(w.x, 2);
  f[3] = __builtin_amdgcn_cvt_f32_fp8(w.x, 3);
  f[4] = __builtin_amdgcn_cvt_f32_fp8(w.y, 0);
  f[5] = __builtin_amdgcn_cvt_f32_fp8(w.y, 1);
  f[6] = __builtin_amdgcn_cvt_f32_fp8(w.y, 2);
  f[7] = __builtin_amdgcn_cvt_f32_fp8(w.y, 3);
}
// Payloads times 2^shift, shift not positive.
__device__ __forceinline__ uint2 shifted_8_bits(const uint2 &w, int shift) {
  float f[8];
  from_8_bits(w, f);
  return to_8_bits(f, power_of_two(shift), false);
}
__device__ __forceinline__ uint4 shifted_8_bits(const uint4 &w, int shift) {
  const uint2 x = shifted_8_bits(make_uint2(w.x, w.y), shift);
  const uint2 y = shifted_8_bits(make_uint2(w.z, w.w), shift);
  return make_uint4(x.x, x.y, y.x, y.y);
}

}  // namespace cvsa
