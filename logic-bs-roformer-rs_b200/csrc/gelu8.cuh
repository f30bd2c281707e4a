// GELU of the 8-bit product's epilogue.
//
// gelu(x) = x Phi(x) = max(x, 0) - a T(a), a = |x|, T(a) = 1 - Phi(a) = 2^P(a)
// with the degree-5 fit of gelu8_fit.py (|2^P - T| <= 2.9e-7).  Per value this
// is six FMAs and one MUFU operation against thirteen and two of the
// erf formula the fp16 epilogue follows; with the roundings of P (at most
// 3 x 2^-24 of |P| ln 2 T, under 1.5e-7) and of ex2.approx (2^-22) its error
// stays below 2^-20 |x|, a 2^-16 of an e4m3 rounding step.  An infinite or NaN
// x gives NaN.
#pragma once
#include "gelu.cuh"

namespace lbrr {

__device__ __forceinline__ float neg_abs(float x) { return __uint_as_float(__float_as_uint(x) | 0x80000000u); }

__device__ __forceinline__ float2 gelu8(float2 x) {
  const float2 n = f2(neg_abs(x.x), neg_abs(x.y));  // -a; the odd coefficients change sign
  float2 p = __ffma2_rn(n, f2(5.188582732e-04f, 5.188582732e-04f), f2(7.387199601e-03f, 7.387199601e-03f));
  p = __ffma2_rn(p, n, f2(5.253801530e-02f, 5.253801530e-02f));
  p = __ffma2_rn(p, n, f2(-4.592766851e-01f, -4.592766851e-01f));
  p = __ffma2_rn(p, n, f2(1.151083144e+00f, 1.151083144e+00f));
  p = __ffma2_rn(p, n, f2(-1.000000836e+00f, -1.000000836e+00f));
  const float2 t = f2(ex2_approx(p.x), ex2_approx(p.y));
  return __ffma2_rn(n, t, f2(fmaxf(x.x, 0.0f), fmaxf(x.y, 0.0f)));
}

}  // namespace lbrr
