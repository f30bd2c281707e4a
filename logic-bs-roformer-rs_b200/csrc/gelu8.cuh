// GELU of the 8-bit product's epilogue.
//
// gelu(x) = x Phi(x) = max(x, 0) - a T(a), a = |x|, T(a) = 1 - Phi(a) = 2^P(a)
// with the fits of gelu8_fit.py: degree 8 on [0, 5.5], and degree 5 on [5.5, 14]
// for the x below -5.5 of blocks that hold nothing large.  What counts is the error
// relative to gelu(x), not to x: a block whose x are all negative holds nothing but
// a T(a), and its scale is the largest of them.  Each fit keeps 2^P within
// 2^-20 (1 + a^2) of T, relative; with the roundings of P (a few 2^-24 of |P|,
// which is near a^2 / 1.4) and of ex2.approx (2^-22) the error stays below
// 2^-19 (1 + a^2) of a T(a): that of an x off by 2^-19.  A positive x has T's absolute
// error beside it, below 2^-20 x.
//
// Per value this is nine FMAs and one MUFU operation against thirteen and two of
// the erf formula that the fp16 epilogue follows.  The FMA pipe sets the pace
// (71362 x 1024 x 256: 1-3 us a degree), so one polynomial for the whole range, of
// degree 12, is dearer: 74 us against 61 with the second fit apart, which is rarely
// evaluated (100 us where every block needs it).  Degree 5 took 55 us; its scales of
// blocks of negative values were off by percents.  An infinite or NaN x gives NaN.
#pragma once
#include "gelu.cuh"

namespace lbrr {

constexpr float kGelu8Tail = -5.5f;
// A block (1 x 128) with an x of this or more has a value of 0.185 or more.  Below -5.5 the first fit falls faster than
// T does and is off by less than 1e-10: a 2^-11 of half a step of the smallest codes beside such a value.
constexpr float kGelu8Large = 0.3f;

__device__ __forceinline__ float neg_abs(float x) { return __uint_as_float(__float_as_uint(x) | 0x80000000u); }
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float min3(float a, float b, float c) {
  float r;
  asm("min.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// x for gelu8, with those below `from` (kGelu8Tail, or -infinity for none) replaced by 2 gelu(x): gelu of that is
// gelu(x), its argument being so near 0 (2.1e-7 at most: gelu(z) = z / 2 + 0.4 z^2).  The power is formed as
// 2^(P + 32): a T(a) may be below the normal range.
__device__ __forceinline__ float2 before_gelu8(float2 x, float from) {
  float2 p = __ffma2_rn(x, f2(3.565373180e-06f, 3.565373180e-06f), f2(2.118331685e-04f, 2.118331685e-04f));
  p = __ffma2_rn(p, x, f2(5.314929489e-03f, 5.314929489e-03f));
  p = __ffma2_rn(p, x, f2(-6.465477077e-01f, -6.465477077e-01f));
  p = __ffma2_rn(p, x, f2(7.121801961e-01f, 7.121801961e-01f));
  p = __ffma2_rn(p, x, f2(32.0f - 1.466802610e+00f, 32.0f - 1.466802610e+00f));
  const float2 t = f2(ex2_approx(p.x), ex2_approx(p.y));
  const float2 y = __fmul2_rn(__fmul2_rn(x, f2(0x1p-31f, 0x1p-31f)), t);
  return f2(x.x < from ? y.x : x.x, x.y < from ? y.y : x.y);
}

// Right to 2^-19 (1 + x^2) of itself for x from kGelu8Tail on; the absolute error stays below 2^-20 |x| everywhere.
__device__ __forceinline__ float2 gelu8(float2 x) {
  const float2 n = f2(neg_abs(x.x), neg_abs(x.y));  // -a; the odd coefficients change sign
  float2 p = __ffma2_rn(n, f2(-3.988912771e-07f, -3.988912771e-07f), f2(-6.430051192e-06f, -6.430051192e-06f));
  p = __ffma2_rn(p, n, f2(-7.279479608e-06f, -7.279479608e-06f));
  p = __ffma2_rn(p, n, f2(6.352800485e-04f, 6.352800485e-04f));
  p = __ffma2_rn(p, n, f2(7.817403010e-03f, 7.817403010e-03f));
  p = __ffma2_rn(p, n, f2(5.309967058e-02f, 5.309967058e-02f));
  p = __ffma2_rn(p, n, f2(-4.589785478e-01f, -4.589785478e-01f));
  p = __ffma2_rn(p, n, f2(1.151137392e+00f, 1.151137392e+00f));
  p = __ffma2_rn(p, n, f2(-9.999992686e-01f, -9.999992686e-01f));
  const float2 t = f2(ex2_approx(p.x), ex2_approx(p.y));
  return __ffma2_rn(n, t, f2(fmaxf(x.x, 0.0f), fmaxf(x.y, 0.0f)));
}

}  // namespace lbrr
