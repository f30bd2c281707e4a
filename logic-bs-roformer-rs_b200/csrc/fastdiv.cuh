// Division by a launch constant in the GEMM kernels.
#pragma once
#include <stdint.h>

namespace lbrr {

// ---------------------------------------------------------------------------
// Division by a launch constant: q = umulhi(x, m), m = ceil(2^32 / d), which is
// exact for x * d < 2^32 (|error| of x*m/2^32 - x/d stays below 1/d); the host
// leaves m = 0, meaning a plain division, when that bound does not hold.
// ---------------------------------------------------------------------------
struct FastDiv {
  uint32_t d = 1, m = 0;
  __device__ __forceinline__ int div(int x) const {
    const uint32_t u = static_cast<uint32_t>(x);
    return static_cast<int>(m ? __umulhi(u, m) : (d == 1 ? u : u / d));
  }
};
static inline FastDiv make_fastdiv(uint32_t d, uint64_t x_max) {
  FastDiv f;
  f.d = d;
  if (d > 1 && x_max * d < (1ull << 32)) f.m = static_cast<uint32_t>(((1ull << 32) + d - 1) / d);
  return f;
}

}  // namespace lbrr
