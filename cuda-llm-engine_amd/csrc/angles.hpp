// Rotary angles, shared by the kernels that turn rows in 64 bits.
#pragma once

#include "common.hpp"

namespace llmk {

// Cosine and sine of an angle, in 64 bits: the quarter turns are taken off in two parts (the angles
// of far positions lose their fraction in 32 bits), and what is left, at most pi / 4, goes through
// the series of both, which end below 2^-48 there. Their number, of up to 2^51, is the low bits of
// a sum with 1.5 * 2^52, whose last one is 1: a conversion to 32 bits would end at 2^31.
__device__ __forceinline__ double2 cos_sin(double angle) {
  constexpr double kWhole = 6755399441055744.0;
  const double turns = __builtin_fma(angle, 0.63661977236758134308, kWhole), k = turns - kWhole;
  double r = __builtin_fma(-k, 1.57079632679489655800, angle);
  r = __builtin_fma(-k, 6.12323399573676603587e-17, r);
  const double z = r * r;
  double s = -7.6471637318198164759e-13;  // (-1)^i / (2 i + 1)!, from i = 7 on down
  s = __builtin_fma(s, z, 1.6059043836821614599e-10);
  s = __builtin_fma(s, z, -2.5052108385441718775e-08);
  s = __builtin_fma(s, z, 2.7557319223985890653e-06);
  s = __builtin_fma(s, z, -1.9841269841269841270e-04);
  s = __builtin_fma(s, z, 8.3333333333333333333e-03);
  s = __builtin_fma(s, z, -1.6666666666666666667e-01);
  s = __builtin_fma(r * z, s, r);
  double c = -1.1470745597729724714e-11;  // (-1)^i / (2 i)!
  c = __builtin_fma(c, z, 2.0876756987868098979e-09);
  c = __builtin_fma(c, z, -2.7557319223985890653e-07);
  c = __builtin_fma(c, z, 2.4801587301587301587e-05);
  c = __builtin_fma(c, z, -1.3888888888888888889e-03);
  c = __builtin_fma(c, z, 4.1666666666666666667e-02);
  c = __builtin_fma(c, z, -0.5);
  c = __builtin_fma(c, z, 1.0);
  const int q = (int)(uint32_t)__builtin_bit_cast(uint64_t, turns) & 3;
  const double cq = (q & 1) ? s : c, sq = (q & 1) ? c : s;
  return make_double2(q == 1 || q == 2 ? -cq : cq, q >= 2 ? -sq : sq);
}

}  // namespace llmk
