// What makes 8-bit rows, shared by the kernels that write them (fp8_rows.hip) and the
// products that take a few bfloat16 rows themselves (fp8_linear.hip).
#pragma once

#include "common.h"

#include <type_traits>

namespace sa {

constexpr int kQBlock = 128;

// y + lo (|lo| at most half an ulp of y) rounded to odd: y where lo is 0 or y is
// odd, else its neighbour towards lo, which is odd.  A y of 0, infinity or NaN stays
__device__ __forceinline__ float to_odd(float y, float lo) {
  const uint32_t b = __float_as_uint(y);
  const int step = (static_cast<int>(b ^ __float_as_uint(lo)) >> 31) | 1;
  return __uint_as_float(lo != 0.0f && fabsf(lo) < fabsf(y) && (b & 1u) == 0u ? b + step : b);
}

// v rounded to fp32 to odd; beyond its range infinite, below it 0
__device__ __forceinline__ float to_odd(double v) {
  const float y = static_cast<float>(v);
  const uint32_t b = __float_as_uint(y);
  const bool moves = static_cast<double>(y) != v && (b & 1u) == 0u && y != 0.0f && fabsf(y) < __builtin_inff();
  return __uint_as_float(!moves ? b : fabs(v) > fabs(static_cast<double>(y)) ? b + 1 : b - 1);
}

// e8m0 byte of the scale of a block with the largest finite magnitude top
__device__ __forceinline__ uint32_t scale_byte(float top) {
  const uint32_t b = __float_as_uint(top);
  // 448 = 1.75 2^8: the mantissa decides between 2^(E - 8) and the next one
  const int e = static_cast<int>(b >> 23) - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return b == 0u ? 127u : static_cast<uint32_t>(max(e, 1));
}
__device__ __forceinline__ float scale_value(uint32_t byte) {   // 2^(byte - 127); byte is 1..247
  return __uint_as_float(byte << 23);
}

// the largest of 16 lanes, in each: rotations within them, which cost a VALU
// instruction where a shuffle through LDS costs its latency
template <int N>
__device__ __forceinline__ float ror16(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x120 + N, 0xf, 0xf, false));
}
__device__ __forceinline__ float max16(float v) {
  v = fmaxf(v, ror16<8>(v));
  v = fmaxf(v, ror16<4>(v));
  v = fmaxf(v, ror16<2>(v));
  return fmaxf(v, ror16<1>(v));
}
// a wave's sum in fp64, in each lane, likewise; then halves of 32 and of 64 lanes swapped
__device__ __forceinline__ double join64(uint32_t lo, uint32_t hi) {
  return __hiloint2double(static_cast<int>(hi), static_cast<int>(lo));
}
__device__ __forceinline__ double wave_sum64(double v) {
  auto rotated = [&](auto n) {
    return join64(__float_as_uint(ror16<decltype(n)::value>(__int_as_float(__double2loint(v)))),
                  __float_as_uint(ror16<decltype(n)::value>(__int_as_float(__double2hiint(v)))));
  };
  v += rotated(std::integral_constant<int, 8>{});
  v += rotated(std::integral_constant<int, 4>{});
  v += rotated(std::integral_constant<int, 2>{});
  v += rotated(std::integral_constant<int, 1>{});
  {
    const uint32_t lo = __double2loint(v), hi = __double2hiint(v);
    const auto l = __builtin_amdgcn_permlane16_swap(lo, lo, false, false), h = __builtin_amdgcn_permlane16_swap(hi, hi, false, false);
    v = join64(l[0], h[0]) + join64(l[1], h[1]);
  }
  const uint32_t lo = __double2loint(v), hi = __double2hiint(v);
  const auto l = __builtin_amdgcn_permlane32_swap(lo, lo, false, false), h = __builtin_amdgcn_permlane32_swap(hi, hi, false, false);
  return join64(l[0], h[0]) + join64(l[1], h[1]);
}

typedef short v2s __attribute__((ext_vector_type(2)));
// four codes of v / scale, a NaN a NaN; without infinities
__device__ __forceinline__ uint32_t encode4(const float* v, float scale) {
  v2s p = {0, 0};
  p = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(p, v[0], v[1], scale, false);
  p = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(p, v[2], v[3], scale, true);
  return __builtin_bit_cast(uint32_t, p);
}
// of two words of bfloat16
__device__ __forceinline__ uint32_t encode4(uint32_t a, uint32_t b, float scale) {
  v2s p = {0, 0};
  p = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(p, __builtin_bit_cast(v2bf, a), scale, false);
  p = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(p, __builtin_bit_cast(v2bf, b), scale, true);
  return __builtin_bit_cast(uint32_t, p);
}
// what the rows keep of an infinity: a NaN, which no scale takes note of
__device__ __forceinline__ float no_infinity(float v) { return fmaf(0.0f, v, v); }

}  // namespace sa
