// 8-bit floating point (e4m3) with a 32-bit scale for every block of 128
// columns: device helpers shared by the quantising kernels and the epilogue
// of the 8-bit matrix product.
//
// A block with largest magnitude t is held as q = e4m3(v / s), s = t / 448
// (448: the largest finite e4m3 value).  Where the values are a caller's, v / s
// is the fp32 quotient (`Quotient8`): 11-bit inputs land on e4m3's rounding
// borders often, and a quotient an ulp off falls on the wrong side of them (six
// codes in 10^5 of fp16 rows).  Where the values are a kernel's own, with
// several roundings in them, it is v * (1 / s), within 2 ulp of 32 bits.  q is
// rounded to nearest even with saturation, so the block's largest value, which
// may land an ulp above 448, stays 448.  s is at
// least 2^-126, so 1 / s is finite and a block of zeros is held as zeros.  A
// block that holds an infinity or a NaN gets scale NaN and NaN codes (0x7f):
// nothing in it could be told apart.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <type_traits>

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
    // t / 448, rounded once: the product with the reciprocal, corrected by its remainder, which one FMA forms
    // exactly (Markstein's division, IBM J. Res. Dev. 34, 1990)
    const float t = __uint_as_float(top), c = 1.0f / kE4m3Max;
    const float q = t * c;
    r.s = fmaxf(fmaf(fmaf(-q, kE4m3Max, t), c, q), kMinScale8);
    asm("rcp.approx.f32 %0, %1;" : "=f"(r.inv) : "f"(r.s));  // within 1 ulp
  }
  return r;
}

// Division of a block's values by its scale: v hi + v lo in one FMA after a
// product, hi + lo = 1 / s to 2^-44 (a sum of two fp32 numbers, Dekker, Numer.
// Math. 18, 1971; lo is hi's correction of second order), so the result is v / s rounded
// once, the fp32 quotient but for quotients that close to the middle between two
// fp32 numbers.  hi is taken a little low: lo is then positive, and a zero keeps
// its sign.  lo would leave the normal range beside a huge s, so those blocks are
// divided as (2^-64 v) / (2^-64 s).
constexpr float kHugeScale8 = 0x1p80f, kHugeDown8 = 0x1p-64f;
struct Quotient8 {
  float hi, lo;
  __device__ __forceinline__ float2 of(float2 v) const {
    return __ffma2_rn(v, make_float2(hi, hi), __fmul2_rn(v, make_float2(lo, lo)));
  }
};
__device__ __forceinline__ Quotient8 quotient8(Scale8 by) {
  const bool huge = by.s > kHugeScale8;
  const float s = huge ? by.s * kHugeDown8 : by.s;
  Quotient8 r;
  r.hi = (huge ? by.inv * (1.0f / kHugeDown8) : by.inv) * (1.0f - 0x1p-22f);
  const float e = fmaf(-s, r.hi, 1.0f);  // up to 2^-21: 1 / s = hi (1 + e + e^2 + ..)
  r.lo = fmaf(e, e, e) * r.hi;
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
// Eight values as they are in memory, for loads that are issued well before their use.
template <class T>
struct Raw8 {
  union {
    uint4 w[sizeof(T) / 2];
    T t[8];
  };
  __device__ __forceinline__ Raw8() {}
  __device__ __forceinline__ void get(float (&v)[8]) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        v[4 * j] = __uint_as_float(w[j].x), v[4 * j + 1] = __uint_as_float(w[j].y);
        v[4 * j + 2] = __uint_as_float(w[j].z), v[4 * j + 3] = __uint_as_float(w[j].w);
      }
    } else {
      const float2 f0 = unpack2(w[0].x, T()), f1 = unpack2(w[0].y, T()), f2 = unpack2(w[0].z, T()),
                   f3 = unpack2(w[0].w, T());
      v[0] = f0.x, v[1] = f0.y, v[2] = f1.x, v[3] = f1.y;
      v[4] = f2.x, v[5] = f2.y, v[6] = f3.x, v[7] = f3.y;
    }
  }
};
// UNITS: an aligned row's last 16-byte unit is loaded whole and `drop_past` zeroes
// what is past the last column; otherwise it is loaded value by value.  Which of
// the two costs fewer registers depends on the kernel.
template <bool VEC, bool UNITS = false, class T>
__device__ __forceinline__ void load_raw(const T* row, int c0, int cols, int lane, Raw8<T>& r) {
  if constexpr (VEC && UNITS) {
    constexpr int kPer = 16 / sizeof(T);
#pragma unroll
    for (int j = 0; j < static_cast<int>(sizeof(T) / 2); ++j) {
      const int c = c0 + lane * 8 + j * kPer;
      r.w[j] = make_uint4(0u, 0u, 0u, 0u);
      if (c < cols) r.w[j] = *reinterpret_cast<const uint4*>(row + c);
    }
    return;
  }
  if (VEC && c0 + lane * 8 + 8 <= cols) {
#pragma unroll
    for (int j = 0; j < static_cast<int>(sizeof(T) / 2); ++j)
      r.w[j] = reinterpret_cast<const uint4*>(row + c0 + lane * 8)[j];
    return;
  }
#pragma unroll
  for (int j = 0; j < static_cast<int>(sizeof(T) / 2); ++j) r.w[j] = make_uint4(0u, 0u, 0u, 0u);
  if (VEC && c0 + lane * 8 >= cols) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int c = c0 + lane_col<VEC>(lane, j);
    if (c < cols) r.t[j] = row[c];
  }
}
__device__ __forceinline__ void drop_past(int c0, int cols, int lane, float (&v)[8]) {
  if (c0 + lane * 8 + 8 <= cols) return;
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (c0 + lane * 8 + j >= cols) v[j] = 0.0f;
}
// Eight consecutive columns of a row that does not start on a 16-byte boundary,
// as VEC's lanes hold them.  LANES lanes load the 16-byte units that their
// columns lie in, the first lane from the unit that column c0 is in, and shift
// the values into place with the following lane's: as many loads as for an
// aligned row, where value by value it would be eight (37889 x 588 bf16: 42 -> 32
// us).  A unit is loaded if it
// holds a value of the row, so no page without one is touched.
template <int LANES, class T>
struct Shifted8 {
  static constexpr int kUnits = sizeof(T) / 2;  // 16-byte units per lane
  uint4 unit[kUnits], extra;                    // extra: the unit after the last lane's

  // `lane`: this lane's place among the LANES.
  __device__ __forceinline__ void load(const T* row, int c0, int cols, int lane) {
    const int bytes = min(cols - c0, 2 * kBlock8 + 8) * static_cast<int>(sizeof(T));  // of the row, as far as it matters
    const uintptr_t at = reinterpret_cast<uintptr_t>(row + c0);
    const int d = static_cast<int>(at & 15);
    const uint4* from = reinterpret_cast<const uint4*>(at - d);
#pragma unroll
    for (int j = 0; j < kUnits; ++j) {
      const int u = lane * kUnits + j;
      unit[j] = make_uint4(0u, 0u, 0u, 0u);
      if (u * 16 - d < bytes) unit[j] = from[u];
    }
    extra = make_uint4(0u, 0u, 0u, 0u);
    if (lane == LANES - 1 && d != 0 && LANES * kUnits * 16 - d < bytes) extra = from[LANES * kUnits];
  }
  // The values, zero past the last column; every lane of the warp calls it.
  __device__ __forceinline__ void get(const T* row, int c0, int cols, int lane, float (&v)[8]) const {
    uint32_t w[4 * kUnits + 4];
#pragma unroll
    for (int j = 0; j < kUnits; ++j)
      w[4 * j] = unit[j].x, w[4 * j + 1] = unit[j].y, w[4 * j + 2] = unit[j].z, w[4 * j + 3] = unit[j].w;
    const uint32_t d = reinterpret_cast<uintptr_t>(row + c0) & 15;
    const bool last = lane == LANES - 1;
    const uint4 e = extra;
    const uint32_t after[4] = {e.x, e.y, e.z, e.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t n = __shfl_down_sync(0xffffffffu, w[j], 1, LANES);
      w[4 * kUnits + j] = last ? after[j] : n;
    }
#pragma unroll
    for (int i = 0; i < 4 * kUnits + 2; ++i) w[i] = (d & 8) ? w[i + 2] : w[i];
#pragma unroll
    for (int i = 0; i < 4 * kUnits + 1; ++i) w[i] = (d & 4) ? w[i + 1] : w[i];
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = unpack2(__funnelshift_r(w[i], w[i + 1], (d & 2) * 8), T());
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
      }
    }
    drop_past(c0, cols, lane, v);
  }
};
// What a lane of the quantising kernels loads ahead.
template <bool VEC, int LANES, class T>
struct Ahead8 {
  std::conditional_t<VEC, Raw8<T>, Shifted8<LANES, T>> raw;
  __device__ __forceinline__ void load(const T* row, int c0, int cols, int lane) {
    if constexpr (VEC)
      load_raw<true>(row, c0, cols, lane, raw);
    else
      raw.load(row, c0, cols, lane);
  }
  __device__ __forceinline__ void get(const T* row, int c0, int cols, int lane, float (&v)[8]) const {
    if constexpr (VEC)
      raw.get(v);
    else
      raw.get(row, c0, cols, lane, v);
  }
};
template <bool VEC>
__device__ __forceinline__ void load_cols(const float* row, int c0, int cols, int lane, float (&v)[8]) {
  if (VEC && c0 + lane * 8 + 8 <= cols) {
    load8(row + c0 + lane * 8, v);
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = 0.0f;
  if (VEC && c0 + lane * 8 >= cols) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int c = c0 + lane_col<VEC>(lane, j);
    if (c < cols) v[j] = row[c];
  }
}
template <bool VEC, class T>
__device__ __forceinline__ void store_cols(T* row, int c0, int cols, int lane, const float (&v)[8]) {
  if (VEC && c0 + lane * 8 + 8 <= cols) {
    store8(row + c0 + lane * 8, v);
    return;
  }
  if (VEC && c0 + lane * 8 >= cols) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int c = c0 + lane_col<VEC>(lane, j);
    if (c < cols) row[c] = from_f32<T>(v[j]);
  }
}
// Eight codes, four to a word.
__device__ __forceinline__ uint2 codes8(const float (&v)[8], float inv) {
  const float2 f = make_float2(inv, inv);
  const float2 a = __fmul2_rn(make_float2(v[0], v[1]), f), b = __fmul2_rn(make_float2(v[2], v[3]), f);
  const float2 c = __fmul2_rn(make_float2(v[4], v[5]), f), d = __fmul2_rn(make_float2(v[6], v[7]), f);
  return make_uint2(e4m3x4(a.x, a.y, b.x, b.y), e4m3x4(c.x, c.y, d.x, d.y));
}
__device__ __forceinline__ uint2 codes8(const float (&v)[8], const Quotient8& by) {
  const float2 a = by.of(make_float2(v[0], v[1])), b = by.of(make_float2(v[2], v[3]));
  const float2 c = by.of(make_float2(v[4], v[5])), d = by.of(make_float2(v[6], v[7]));
  return make_uint2(e4m3x4(a.x, a.y, b.x, b.y), e4m3x4(c.x, c.y, d.x, d.y));
}
template <bool VEC, class By>
__device__ __forceinline__ void store_codes(uint8_t* row, int c0, int cols, int lane, const float (&v)[8],
                                            const By& by, bool aligned = true) {
  const uint2 q = codes8(v, by);
  if (VEC && aligned && c0 + lane * 8 + 8 <= cols) {
    *reinterpret_cast<uint2*>(row + c0 + lane * 8) = q;
    return;
  }
  if (VEC && c0 + lane * 8 >= cols) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int at = c0 + lane_col<VEC>(lane, j);
    if (at < cols) row[at] = static_cast<uint8_t>((j < 4 ? q.x >> (8 * j) : q.y >> (8 * (j - 4))) & 0xffu);
  }
}
// Largest magnitude of eight values, as bits (NaN above all).
__device__ __forceinline__ uint32_t top_of(const float (&v)[8]) {
  const float a = max_mag3(0.0f, v[0], v[1]), b = max_mag3(0.0f, v[4], v[5]);
  return __float_as_uint(max_mag3(max_mag3(a, v[2], v[3]), max_mag3(b, v[6], v[7]), 0.0f));
}

// The scales of R blocks (1, 2 or 4) that 16 lanes hold together, from every
// lane's own maxima.  The exchange halves the number of blocks a lane follows
// until it has one, so R blocks take R + 3 shuffles (and one to hand a number on),
// not 4 R, and one scale per lane is computed, not R.  Every lane of the warp
// calls these.
template <int R>
struct Scales8 {
  Scale8 own;      // of block own_block
  int own_block;
  bool writer;     // one lane per block

  __device__ __forceinline__ float of(float own_number, int block, int lane) const {
    return R == 1 ? own_number : __shfl_sync(0xffffffffu, own_number, (lane & 16) | (block * (16 / R)));
  }
};
template <int R>
__device__ __forceinline__ Scales8<R> half_warp_scales(const uint32_t (&top)[R], int lane) {
  static_assert(R == 1 || R == 2 || R == 4, "blocks");
  constexpr unsigned all = 0xffffffffu;
  uint32_t k;
  const bool b3 = lane & 8, b2 = lane & 4;
  Scales8<R> r;
  if constexpr (R == 4) {
    const uint32_t x = max(b3 ? top[2] : top[0], __shfl_xor_sync(all, b3 ? top[0] : top[2], 8));
    const uint32_t y = max(b3 ? top[3] : top[1], __shfl_xor_sync(all, b3 ? top[1] : top[3], 8));
    k = max(b2 ? y : x, __shfl_xor_sync(all, b2 ? x : y, 4));
    r.own_block = (lane >> 2) & 3;
    r.writer = (lane & 3) == 0;
  } else if constexpr (R == 2) {
    k = max(b3 ? top[1] : top[0], __shfl_xor_sync(all, b3 ? top[0] : top[1], 8));
    k = max(k, __shfl_xor_sync(all, k, 4));
    r.own_block = (lane >> 3) & 1;
    r.writer = (lane & 7) == 0;
  } else {
    k = max(top[0], __shfl_xor_sync(all, top[0], 8));
    k = max(k, __shfl_xor_sync(all, k, 4));
    r.own_block = 0;
    r.writer = (lane & 15) == 0;
  }
  k = max(k, __shfl_xor_sync(all, k, 2));
  k = max(k, __shfl_xor_sync(all, k, 1));
  r.own = scale8(k);
  return r;
}
// Every block's inverse scale in every lane.
template <int R>
__device__ __forceinline__ void inverses(const Scales8<R>& sc, int lane, float (&inv)[R]) {
#pragma unroll
  for (int i = 0; i < R; ++i) inv[i] = sc.of(sc.own.inv, i, lane);
}

}  // namespace lbrr
