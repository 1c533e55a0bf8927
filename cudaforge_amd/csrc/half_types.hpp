// half_types.hpp -- the two 16-bit element types of the operators that take
// either: conversions of packed pairs with one rounding (to nearest even).
#pragma once

#include <hip/hip_runtime.h>

namespace cfa {

struct BF16 {
  typedef __bf16 elem;
};
struct FP16 {
  typedef _Float16 elem;
};

// The two elements of a 32-bit word, and back.
template <class T>
__device__ __forceinline__ void unpack2(uint32_t w, float &lo, float &hi);
template <>
__device__ __forceinline__ void unpack2<BF16>(uint32_t w, float &lo, float &hi) {
  lo = __uint_as_float(w << 16);
  hi = __uint_as_float(w & 0xffff0000u);
}
template <>
__device__ __forceinline__ void unpack2<FP16>(uint32_t w, float &lo, float &hi) {
  lo = (float)__builtin_bit_cast(_Float16, (uint16_t)w);
  hi = (float)__builtin_bit_cast(_Float16, (uint16_t)(w >> 16));
}
template <class T>
__device__ __forceinline__ uint16_t pack1(float f) {
  return __builtin_bit_cast(uint16_t, (typename T::elem)f);
}
template <class T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  typedef typename T::elem pair __attribute__((ext_vector_type(2)));
  typedef float floats __attribute__((ext_vector_type(2)));
  // one instruction for bf16
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((floats{lo, hi}), pair));
}

}  // namespace cfa
