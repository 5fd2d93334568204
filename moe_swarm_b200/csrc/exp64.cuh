// The exponential that routing scores are defined by, evaluated in double.
#pragma once

namespace moe {

// exp(y) in double for -708 < y <= 100: y = k*ln2 + r with k = rint(y / ln2) and a two-part ln2
// (fdlibm's split, k*ln2_hi exact), exp(r) for |r| <= ln2/2 by its Taylor series to degree 13
// (truncation below 5e-18, under double rounding), then scaled by 2^k through the exponent field.
// About 20 double operations, several times fewer than the library's general double exp, which
// dominated the routing time.  (2^k is a normal double in that range.)
__device__ __forceinline__ double exp_series(double y) {
  const double k = rint(y * 1.4426950408889634074);
  double r = fma(-k, 6.93147180369123816490e-01, y);
  r = fma(-k, 1.90821492927058770002e-10, r);
  double p = 1.0 / 6227020800.0;
  p = fma(p, r, 1.0 / 479001600.0);
  p = fma(p, r, 1.0 / 39916800.0);
  p = fma(p, r, 1.0 / 3628800.0);
  p = fma(p, r, 1.0 / 362880.0);
  p = fma(p, r, 1.0 / 40320.0);
  p = fma(p, r, 1.0 / 5040.0);
  p = fma(p, r, 1.0 / 720.0);
  p = fma(p, r, 1.0 / 120.0);
  p = fma(p, r, 1.0 / 24.0);
  p = fma(p, r, 1.0 / 6.0);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  const double scale = __hiloint2double((static_cast<int>(k) + 1023) << 20, 0);
  return p * scale;
}

// exp(y) rounded once to fp32.  For every fp32 argument the result equals the library's double
// exp rounded to fp32 (checked exhaustively on a B200: all 2,246,049,794 floats with |x| <= 120
// give the same bits; beyond that both saturate to +inf or 0).
__device__ __forceinline__ float exp_to_f32(double y) {
  if (y != y) return static_cast<float>(y);
  if (y > 100.0) return __int_as_float(0x7f800000);   // above FLT_MAX: +inf
  if (y < -110.0) return 0.f;                         // below half the smallest denormal
  return static_cast<float>(exp_series(y));
}

}  // namespace moe
