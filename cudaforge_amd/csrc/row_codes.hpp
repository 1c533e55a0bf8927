// row_codes.hpp -- logits as whole numbers in their order, ranges of these as fp32
// comparisons, and the logarithm behind min-p's border (sample_rows.hip).
#pragma once

#include <float.h>
#include <math.h>

#include "common.hpp"

namespace cfa {
namespace rows {

enum Type { kF32 = 0, kBF16 = 1, kFP16 = 2 };

// The values of a type as codes, whole numbers in their order: the bits of the
// fp32 value, turned over where it is negative, less the low ones that the type
// does not have (16 in bf16, 13 in fp16), so that equal values are neighbours'
// distance of one apart from the next.
template <int TYPE>
struct Code {
  static constexpr int kDrop = TYPE == kF32 ? 0 : (TYPE == kBF16 ? 16 : 13);
  static constexpr float kMost =
      TYPE == kF32 ? FLT_MAX : (TYPE == kBF16 ? 3.38953138925153547590e38f : 65504.0f);
  static CFA_HD uint32_t of(float x) {
    const uint32_t b = f2u(x);
    return ((b & 0x80000000u) ? ~b : b | 0x80000000u) >> kDrop;
  }
  static CFA_HD float value(uint32_t c) {
    c <<= kDrop;
    return u2f((c & 0x80000000u) ? c & 0x7fffffffu : ~(c | ((1u << kDrop) - 1)));
  }
  static CFA_HD uint32_t lowest() { return of(-kMost); }
  static CFA_HD uint32_t most() { return of(kMost); }
  // A logit as the rules take it: NaN as -inf, +inf as the largest finite, -0 as 0.
  static CFA_HD float clean(float x) { return x != x ? -INFINITY : fminf(x, kMost) + 0.0f; }
};

// The tokens whose codes, once clean, are lo .. hi (both finite values'), by
// comparisons of the values as they are read: NaN nowhere, +inf with the largest.
template <int TYPE>
struct Span {
  using C = Code<TYPE>;
  float least, most;
  bool none;
  CFA_HD Span(uint32_t lo, uint32_t hi) {
    // -0 has a code, which no clean token has: as the upper border it would
    // compare as 0, whose code lies behind the range
    if (hi == C::of(-0.0f)) --hi;
    none = lo > hi;
    least = C::value(lo);
    most = hi >= C::most() ? INFINITY : C::value(hi);
  }
  CFA_HD bool holds(float x) const { return x >= least && x <= most; }
};

constexpr int kSub = 16;  // bins per octave of weight

// log2(f) for f in [1, 2), from an approximation l of it (off by 2^-19 at most): l
// and what it misses, from f 2^-l - 1 by two terms of its series (the third is below
// 2^-57).  2^-l is table[j] = 2^((j + 1/2) / 16) times a power series of which eight
// terms leave 2^-69.  Off by 2^-50 at most, all roundings counted.
CFA_HD double log2_from(double f, float l, const double *table) {
  const double z = -(double)l * kSub, q = floor(z);
  const double x = (z - q - 0.5) * (0.69314718055994530942 / kSub);
  double p = 1.0;
  for (int k = 8; k >= 1; --k) p = fma(p, x * (1.0 / k), 1.0);
  const double d = fma(f, ldexp(table[(int)q & (kSub - 1)] * p, (int)q >> 4), -1.0);
  return l + (d - 0.5 * d * d) * 1.4426950408889634074;
}

}  // namespace rows
}  // namespace cfa
