// 8-bit floating point (e4m3) with a 32-bit scale for every block of 128
// columns: device helpers shared by the quantising kernels and the epilogue
// of the 8-bit matrix product.
//
// A block with largest magnitude t is held as q = e4m3(v / s), s = t / 448
// (448: the largest finite e4m3 value).  Two roundings are choices: v / s is
// computed as v * (1 / s) (within 2 ulp of 32 bits, far below e4m3's half
// step of 2^-4), and q is rounded to nearest even with saturation, so the
// block's largest value, which may land an ulp above 448, stays 448.  s is at
// least 2^-126, so 1 / s is finite and a block of zeros is held as zeros.  A
// block that holds an infinity or a NaN gets scale NaN and NaN codes (0x7f):
// nothing in it could be told apart.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "common.cuh"
#include "kernels.h"

namespace lbrr {

constexpr int kBlock8 = 128;
constexpr float kE4m3Max = 448.0f;
constexpr float kMinScale8 = 1.17549435e-38f;  // 2^-126

// Magnitude as an integer: ordered like the value, with infinity above every
// number and NaN above infinity, so an integer maximum keeps a NaN.
__device__ __forceinline__ uint32_t mag_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// max(a, |b|, |c|) for a >= 0; NaN if one of them is.
__device__ __forceinline__ float max_mag3(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

struct Scale8 {
  float s, inv;
};
// Scale of a block from the largest magnitude's bits.
__device__ __forceinline__ Scale8 scale8(uint32_t top) {
  Scale8 r;
  if (top >= 0x7f800000u) {
    r.s = r.inv = __uint_as_float(0x7fffffffu);
  } else {
    // t / 448, correctly rounded: the product with 1 / 448, corrected once by its remainder (exact in an FMA)
    const float t = __uint_as_float(top), c = 1.0f / kE4m3Max;
    const float q = t * c;
    r.s = fmaxf(fmaf(fmaf(-q, kE4m3Max, t), c, q), kMinScale8);
    asm("rcp.approx.f32 %0, %1;" : "=f"(r.inv) : "f"(r.s));  // within 1 ulp
  }
  return r;
}

// Two values -> two e4m3 bytes, the first in the low byte.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  return e4m3x2(a, b) | (e4m3x2(c, d) << 16);
}

// ---------------------------------------------------------------------------
// Loads and stores of 32- and 16-bit values as 32-bit floats
// ---------------------------------------------------------------------------
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) {
  return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi, __half) {
  __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __nv_bfloat16) {
  __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack2(uint32_t w, __half) {
  return __half22float2(*reinterpret_cast<__half2*>(&w));
}
__device__ __forceinline__ float2 unpack2(uint32_t w, __nv_bfloat16) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// Eight consecutive values, 16-byte aligned.
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
  v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
template <class T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  const uint4 a = *reinterpret_cast<const uint4*>(p);
  const float2 f0 = unpack2(a.x, T()), f1 = unpack2(a.y, T()), f2 = unpack2(a.z, T()), f3 = unpack2(a.w, T());
  v[0] = f0.x, v[1] = f0.y, v[2] = f1.x, v[3] = f1.y;
  v[4] = f2.x, v[5] = f2.y, v[6] = f3.x, v[7] = f3.y;
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
template <class T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack2(v[0], v[1], T()), pack2(v[2], v[3], T()), pack2(v[4], v[5], T()),
                                            pack2(v[6], v[7], T()));
}

// How the 32 lanes share 256 columns: 16 lanes per block of 128, 8 values
// each.  VEC: lane l holds the 8 consecutive columns from 8 * l; otherwise
// (rows that do not start on 16-byte boundaries) value j is column
// 128 * (l / 16) + l % 16 + 16 * j, so 16 lanes read 16 neighbours.
template <bool VEC>
__device__ __forceinline__ int lane_col(int lane, int j) {
  return VEC ? lane * 8 + j : (lane >> 4) * kBlock8 + (lane & 15) + 16 * j;
}
template <bool VEC, class T>
__device__ __forceinline__ void load_cols(const T* row, int c0, int cols, int lane, float (&v)[8]) {
  if (VEC && c0 + lane * 8 + 8 <= cols) {
    load8(row + c0 + lane * 8, v);
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int c = c0 + lane_col<VEC>(lane, j);
    v[j] = c < cols ? to_f32(row[c]) : 0.0f;
  }
}
template <bool VEC, class T>
__device__ __forceinline__ void store_cols(T* row, int c0, int cols, int lane, const float (&v)[8]) {
  if (VEC && c0 + lane * 8 + 8 <= cols) {
    store8(row + c0 + lane * 8, v);
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int c = c0 + lane_col<VEC>(lane, j);
    if (c < cols) row[c] = from_f32<T>(v[j]);
  }
}
template <bool VEC>
__device__ __forceinline__ void store_codes(uint8_t* row, int c0, int cols, int lane, const float (&v)[8],
                                            float inv) {
  const uint32_t lo = e4m3x4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
  const uint32_t hi = e4m3x4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv);
  if (VEC && c0 + lane * 8 + 8 <= cols) {
    *reinterpret_cast<uint2*>(row + c0 + lane * 8) = make_uint2(lo, hi);
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int c = c0 + lane_col<VEC>(lane, j);
    if (c < cols) row[c] = static_cast<uint8_t>((j < 4 ? lo >> (8 * j) : hi >> (8 * (j - 4))) & 0xffu);
  }
}
__device__ __forceinline__ uint32_t top_of(const float (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = max(m, mag_bits(v[j]));
  return m;
}
// Maximum over the 16 lanes that share a block.
__device__ __forceinline__ uint32_t half_warp_max(uint32_t m) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}

}  // namespace lbrr
