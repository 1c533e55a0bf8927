// e4m3.hpp -- rows of a cache in 8 bits: e4m3 codes (4 bits of exponent, 3 of
// mantissa, no infinity) and a power-of-two scale for each row, kept as the byte
// e + 127 of 2^e.
//
//   e = the least integer >= -126 with max |x| <= 448 2^e;  code = e4m3(x 2^-e)
//
// A power of two costs a code no accuracy that another scale would keep (the
// steps of a code are relative to its value; only codes 2^14 below the row's
// largest lose steps), x 2^-e is exact, so a value is rounded once, and what a
// code stands for is exact in bf16.  Values that are not finite do not count for
// the largest and become NaN codes: nothing that overflowed is hidden.
#pragma once

#include <hip/hip_runtime.h>

#include "half_types.hpp"

namespace cfa {
namespace e4m3 {

// A value's magnitude as bits that compare as it does; 0 if it is not finite.
__device__ __forceinline__ uint32_t magnitude(float x) {
  const uint32_t u = __float_as_uint(x) & 0x7fffffffu;
  return u < 0x7f800000u ? u : 0u;
}

// The scale's byte for a row's largest magnitude (448 is 1.75 2^8).
__device__ __forceinline__ uint32_t scale_byte(uint32_t largest) {
  const int byte = (int)(largest >> 23) - 8 + ((largest & 0x7fffffu) > 0x600000u ? 1 : 0);
  return (uint32_t)max(byte, 1);
}

// 2^(127 - byte) and 2^(byte - 127), bytes from 1 to 253.
__device__ __forceinline__ float inverse_scale(uint32_t byte) {
  return __uint_as_float((254u - byte) << 23);
}
__device__ __forceinline__ float scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// x as it is coded in a cache of T: in fp16 the largest values, which would round
// to 65536, stop at 61440.
template <class T>
__device__ __forceinline__ float codable(float x) {
  if constexpr (__is_same(T, FP16)) {
    if (fabsf(x) <= 65504.0f) x = fminf(fmaxf(x, -61440.0f), 61440.0f);
  }
  return fabsf(x) < INFINITY ? x : __uint_as_float(0x7fc00000u);
}

// Four codes of a word.
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
  const int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

// Two codes of a word (the upper ones if HI), times `scale`, as a pair of T; exact
// in bf16, in fp16 within its range.
template <class T, bool HI>
__device__ __forceinline__ uint32_t unpack_pair(uint32_t w, float scale) {
  if constexpr (__is_same(T, BF16))
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HI));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, HI));
}

}  // namespace e4m3
}  // namespace cfa
