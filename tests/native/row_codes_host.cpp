// row_codes_host.cpp -- csrc/row_codes.hpp for the CPU tests.  TEST
// INFRASTRUCTURE.
#include "../../cudaforge_amd/csrc/row_codes.hpp"

using namespace cfa::rows;

namespace {
// How many of the values are held by a range of codes but lie outside of it, or
// the other way round.
template <int TYPE>
int wrong(uint32_t lo, uint32_t hi, const float *x, int n) {
  using C = Code<TYPE>;
  const Span<TYPE> in(lo, hi);
  int bad = 0;
  for (int i = 0; i < n; ++i) {
    const uint32_t c = C::of(C::clean(x[i]));
    const bool want = x[i] == x[i] && lo <= c && c <= hi;
    bad += want != (!in.none && in.holds(x[i]));
  }
  return bad;
}
template <class F>
auto of_type(int type, F f) {
  return type == kF32 ? f(Code<kF32>()) : type == kBF16 ? f(Code<kBF16>()) : f(Code<kFP16>());
}
}  // namespace

extern "C" int codes_wrong(int type, uint32_t lo, uint32_t hi, const float *x, int n) {
  return type == kF32 ? wrong<kF32>(lo, hi, x, n)
                      : type == kBF16 ? wrong<kBF16>(lo, hi, x, n) : wrong<kFP16>(lo, hi, x, n);
}
extern "C" uint32_t codes_of(int type, float x) {
  return of_type(type, [&](auto c) { return decltype(c)::of(x); });
}
extern "C" float codes_value(int type, uint32_t c) {
  return of_type(type, [&](auto t) { return decltype(t)::value(c); });
}

// log2_from with an approximation that is `off` from the fp32 logarithm.
extern "C" double codes_log2(double f, float off) {
  double table[kSub];
  for (int j = 0; j < kSub; ++j) table[j] = exp2((j + 0.5) / kSub);
  return log2_from(f, log2f((float)f) + off, table);
}
