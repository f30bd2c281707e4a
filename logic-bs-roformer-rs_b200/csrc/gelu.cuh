// GELU of the feed-forward epilogues, and the approximate reciprocal and
// power of two it and the other epilogues use.
#pragma once
#include "common.cuh"

namespace lbrr {

__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float ex2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float2 f2(float a, float b) { return make_float2(a, b); }

// GELU of two values with the Abramowitz-Stegun 7.1.26 erf approximation (the
// published formula the reference's FF1 epilogue uses, src/main.rs:2928-2935),
// written with packed fp32x2 FMA/MUL/ADD (same IEEE result per element as the
// scalar ops, half the instructions).
__device__ __forceinline__ float2 gelu_as2(float2 v) {
  const float2 a = __fmul2_rn(f2(fabsf(v.x), fabsf(v.y)), f2(0.70710678f, 0.70710678f));
  const float2 den = __ffma2_rn(a, f2(0.3275911f, 0.3275911f), f2(1.0f, 1.0f));
  const float2 t = f2(rcp_approx(den.x), rcp_approx(den.y));
  float2 p = __ffma2_rn(f2(1.061405429f, 1.061405429f), t, f2(-1.453152027f, -1.453152027f));
  p = __ffma2_rn(p, t, f2(1.421413741f, 1.421413741f));
  p = __ffma2_rn(p, t, f2(-0.284496736f, -0.284496736f));
  p = __ffma2_rn(p, t, f2(0.254829592f, 0.254829592f));
  p = __fmul2_rn(p, t);
  // exp(-a^2) = 2^(-a^2 * log2 e)
  const float2 arg = __fmul2_rn(__fmul2_rn(a, a), f2(-1.4426950408889634f, -1.4426950408889634f));
  const float2 e = f2(ex2_approx(arg.x), ex2_approx(arg.y));
  const float2 erfc = __fmul2_rn(p, e);
  const float2 erfa = f2(copysignf(1.0f - erfc.x, v.x), copysignf(1.0f - erfc.y, v.y));
  const float2 h = __fmul2_rn(v, f2(0.5f, 0.5f));
  return __ffma2_rn(h, erfa, h);  // 0.5 v (1 + erf)
}

}  // namespace lbrr
