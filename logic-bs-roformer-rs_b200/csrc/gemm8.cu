// 8-bit matrix product with block scales.
//
//   acc[m][n] = sum over 128-column blocks b of
//               a_scale[b][m] * w_scale[b][n / 128] * sum over k in b of A[m][k] W[n][k]
//   out = acc + bias[n] + resid[m][n], or gelu(acc + bias) -> (q, scales) by 1 x 128.
//
// Products of two e4m3 values are exact in 32 bits; each block's sum is formed
// first, then multiplied once by its two scales and added to the 32-bit total.
#include "quant8.cuh"

namespace lbrr {

__device__ __forceinline__ float e4m3_f32(uint8_t c) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(c)));
  return __half2float(__ushort_as_half(static_cast<unsigned short>(h & 0xffffu)));
}
__device__ __forceinline__ float gelu8(float h) { return 0.5f * h * (1.0f + erff(h * 0.70710678f)); }

// A block of 256 threads computes 32 rows x 128 columns; warp w owns rows
// 4w..4w+3, lane l columns l + 32j.
constexpr int kTm = 32, kTn = 128, kTk = 32;
template <class TO, bool QUANT>
__global__ void __launch_bounds__(256) gemm8_simple_kernel(const Gemm8 g) {
  __shared__ float sa[kTm][kTk + 1], sw[kTn][kTk + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int m0 = blockIdx.x * kTm, n0 = blockIdx.y * kTn;
  float acc[4][4] = {}, part[4][4] = {};
  for (int k0 = 0; k0 < g.k; k0 += kTk) {
    for (int i = threadIdx.x; i < kTm * kTk; i += 256) {
      const int r = i / kTk, k = i % kTk;
      sa[r][k] = m0 + r < g.m && k0 + k < g.k ? e4m3_f32(g.a[(m0 + r) * g.lda + k0 + k]) : 0.0f;
    }
    for (int i = threadIdx.x; i < kTn * kTk; i += 256) {
      const int r = i / kTk, k = i % kTk;
      sw[r][k] = n0 + r < g.n && k0 + k < g.k ? e4m3_f32(g.w[(n0 + r) * g.ldw + k0 + k]) : 0.0f;
    }
    __syncthreads();
    for (int k = 0; k < kTk; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) part[i][j] = fmaf(sa[warp * 4 + i][k], sw[lane + 32 * j][k], part[i][j]);
    __syncthreads();
    if ((k0 + kTk) % kBlock8 == 0 || k0 + kTk >= g.k) {
      const int kb = k0 / kBlock8;
      const float ws = g.w_scales[kb * g.ldws + blockIdx.y];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int m = m0 + warp * 4 + i;
        const float s = m < g.m ? g.a_scales[kb * g.ldas + m] * ws : 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          acc[i][j] = fmaf(part[i][j], s, acc[i][j]);
          part[i][j] = 0.0f;
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int m = m0 + warp * 4 + i;
    if (m >= g.m) break;
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + lane + 32 * j;
      if (n >= g.n) continue;
      float h = acc[i][j] + (g.bias ? g.bias[n] : 0.0f);
      if (QUANT) {
        h = acc[i][j] = gelu8(h);
        top = max(top, mag_bits(h));
      } else {
        if (g.resid) h += to_f32(static_cast<const TO*>(g.resid)[m * g.ldr + n]);
        static_cast<TO*>(g.out)[m * g.ldo + n] = from_f32<TO>(h);
      }
    }
    if (QUANT) {
      const Scale8 s = scale8(__reduce_max_sync(0xffffffffu, top));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int n = n0 + lane + 32 * j;
        if (n < g.n) g.q[m * g.ldq + n] = static_cast<uint8_t>(e4m3x2(acc[i][j] * s.inv, 0.0f) & 0xffu);
      }
      if (lane == 0) g.scales[blockIdx.y * g.lds + m] = s.s;
    }
  }
}

cudaError_t gemm8(const Gemm8& g, int* status, cudaStream_t st) {
  (void)status;
  const dim3 grid((g.m + kTm - 1) / kTm, (g.n + kTn - 1) / kTn);
  count_launch();
  if (!g.out)
    gemm8_simple_kernel<float, true><<<grid, 256, 0, st>>>(g);
  else if (g.out_type == Elem::F32)
    gemm8_simple_kernel<float, false><<<grid, 256, 0, st>>>(g);
  else if (g.out_type == Elem::F16)
    gemm8_simple_kernel<__half, false><<<grid, 256, 0, st>>>(g);
  else
    gemm8_simple_kernel<__nv_bfloat16, false><<<grid, 256, 0, st>>>(g);
  return cudaGetLastError();
}

}  // namespace lbrr
