// The logarithm of a row's sum of exponentials, as the policy loss and the
// log-probabilities take it: both round their log-probabilities from 64 bits.
#pragma once

#include <math.h>

// log of a positive finite float to 1e-9: s = 2^k f with f in [1/sqrt 2,
// sqrt 2), log f = 2 atanh(q), q = (f - 1) / (f + 1), |q| < 0.172: the odd
// series to q^11 in 64 bits (next term 2e-11).  Zero, infinity and NaN go
// to log().
__device__ __forceinline__ double log_row_sum(float s) {
  if (!(s >= 1.17549435e-38f && s <= 3.4e38f)) return log((double)s);
  const int bits = __float_as_int(s);
  int k = (bits >> 23) - 127;
  float f = __int_as_float((bits & 0x007fffff) | 0x3f800000);
  if (f > 1.41421356f) {
    f *= 0.5f;
    k += 1;
  }
  const double den = (double)f + 1.0;
  double r = (double)__frcp_rn((float)den);
  r = r * (2.0 - den * r);
  const double q = ((double)f - 1.0) * r, q2 = q * q;
  double c = 1.0 / 11.0;
  c = fma(c, q2, 1.0 / 9.0);
  c = fma(c, q2, 1.0 / 7.0);
  c = fma(c, q2, 1.0 / 5.0);
  c = fma(c, q2, 1.0 / 3.0);
  c = fma(c, q2, 1.0);
  return fma(2.0 * q, c, (double)k * 0.693147180559945309417);
}
