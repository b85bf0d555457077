// The exponential that the sampler's weights are taken with.
#pragma once

namespace fa {

constexpr int SA_EXP_TABLE = 64;      // table[i] = 2^(i / 64)

// e^z for z <= 0, within 2.2 x 2^-52 of itself; below e^-700: 0.  z = (n / 64) ln 2 + r with |r| <= ln 2 / 128, the reduction
// with ln 2 in two parts (W. J. Cody and W. Waite, Software Manual for the Elementary Functions, 1980) and n rounded by
// adding 1.5 * 2^52; 2^((n mod 64) / 64) from a table (P. T. P. Tang, Table-driven implementation of the exponential
// function in IEEE floating-point arithmetic, ACM TOMS 15, 1989), e^r by its Taylor polynomial of degree 5 (remainder
// r^6 / 720 = 4e-17), n / 64 added to the exponent.
__device__ __forceinline__ double sa_exp(double z, const double* table) {
  const double t = fma(z, 64.0 * 1.4426950408889634, 6755399441055744.0);
  const int n = __double2loint(t);
  const double nf = t - 6755399441055744.0;
  double r = fma(nf, -0.6931471805599453 / 64.0, z);  // ln 2 as a sum of two doubles
  r = fma(nf, -2.3190468138462996e-17 / 64.0, r);
  double p = 1.0 / 120.0;
  p = fma(p, r, 1.0 / 24.0);
  p = fma(p, r, 1.0 / 6.0);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0) * table[n & (SA_EXP_TABLE - 1)];
  const double e = __hiloint2double(__double2hiint(p) + ((n >> 6) << 20), __double2loint(p));
  return z < -700.0 ? 0.0 : e;
}

}  // namespace fa
