// What makes 8-bit rows, shared by the kernels that write them (fp8_rows.hip) and the
// products that take a few bfloat16 rows themselves (fp8_linear.hip).
#pragma once

#include "common.h"

namespace sa {

constexpr int kQBlock = 128;

// y + lo (|lo| at most half an ulp of y) rounded to odd: y where lo is 0 or y is
// odd, else its neighbour towards lo, which is odd.  A y of 0, infinity or NaN stays
__device__ __forceinline__ float to_odd(float y, float lo) {
  const uint32_t b = __float_as_uint(y);
  const int step = (static_cast<int>(b ^ __float_as_uint(lo)) >> 31) | 1;
  return __uint_as_float(lo != 0.0f && fabsf(lo) < fabsf(y) && (b & 1u) == 0u ? b + step : b);
}

// e8m0 byte of the scale of a block with the largest finite magnitude top
__device__ __forceinline__ uint32_t scale_byte(float top) {
  const uint32_t b = __float_as_uint(top);
  // 448 = 1.75 2^8: the mantissa decides between 2^(E - 8) and the next one
  const int e = static_cast<int>(b >> 23) - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return b == 0u ? 127u : static_cast<uint32_t>(max(e, 1));
}
__device__ __forceinline__ float scale_inverse(uint32_t byte) {   // 2^(127 - byte); byte is 1..247
  return __uint_as_float((254u - byte) << 23);
}

// |v|, 0 where v is not finite
__device__ __forceinline__ float finite_abs(float v) {
  const float m = fabsf(v);
  return m < __builtin_inff() ? m : 0.0f;
}

// four codes of v inv (v / scale); an infinity or NaN gives NaN
__device__ __forceinline__ uint32_t encode4(const float* v, float inv) {
  float q[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) q[i] = fmaf(0.0f, v[i], v[i] * inv);
  int p = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
  p = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], p, true);
  return static_cast<uint32_t>(p);
}

}  // namespace sa
