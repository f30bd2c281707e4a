// Quantising kernels of the 8-bit path: blocks of 1 x 128 or 128 x 128 of a
// matrix to e4m3 with scales, and the trunk's RMSNorm with the residual's
// addition and an 8-bit output.  Both are one pass over their data (every
// value is read once, held in registers while its block's or row's statistics
// form, and written once), so HBM bounds them.
#include <cmath>

#include "quant8.cuh"

namespace lbrr {

// ---------------------------------------------------------------------------
// v -> (q, scales), blocks of 1 x 128.  A warp takes kRows8 rows of 256
// columns (16 lanes per block), all loads issued before the first use; eight
// warps cover 32 rows, so the scales of a block column leave as whole sectors.
// ---------------------------------------------------------------------------
constexpr int kRows8 = 4;
constexpr int kWarps8 = 8;

template <class T, bool VEC>
__global__ void __launch_bounds__(kWarps8 * 32)
    quant_rows_kernel(const T* __restrict__ x, int64_t ldx, int rows, int cols, uint8_t* __restrict__ q, int64_t ldq,
                      float* __restrict__ scales, int64_t lds) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r0 = (blockIdx.x * kWarps8 + warp) * kRows8;
  const int c0 = blockIdx.y * 2 * kBlock8;
  float v[kRows8][8];
#pragma unroll
  for (int i = 0; i < kRows8; ++i) {
    if (r0 + i < rows) {
      load_cols<VEC>(x + static_cast<int64_t>(r0 + i) * ldx, c0, cols, lane, v[i]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
    }
  }
  uint32_t top[kRows8];
#pragma unroll
  for (int i = 0; i < kRows8; ++i) top[i] = top_of(v[i]);
  const Scales8<kRows8> sc = half_warp_scales<kRows8>(top, lane);
#pragma unroll
  for (int i = 0; i < kRows8; ++i)
    if (r0 + i < rows) store_codes<VEC>(q + static_cast<int64_t>(r0 + i) * ldq, c0, cols, lane, v[i], sc.inv[i]);
  const int kb = blockIdx.y * 2 + (lane >> 4);
  if (sc.writer && r0 + sc.own_block < rows && kb * kBlock8 < cols) scales[kb * lds + r0 + sc.own_block] = sc.own;
}

// Blocks of 128 x 128: one CTA per block, 32 values per thread.
constexpr int kTileThreads8 = 512;
template <class T, bool VEC>
__global__ void __launch_bounds__(kTileThreads8)
    quant_tiles_kernel(const T* __restrict__ x, int64_t ldx, int rows, int cols, uint8_t* __restrict__ q, int64_t ldq,
                       float* __restrict__ scales, int64_t lds) {
  constexpr int kPer = kBlock8 * kBlock8 / kTileThreads8 / 8;  // row groups per thread
  constexpr int kStep = kTileThreads8 / 16;                    // rows per group
  __shared__ uint32_t part[kTileThreads8 / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int l16 = lane & 15;  // the 16 lanes of a row
  const int r0 = blockIdx.y * kBlock8 + (threadIdx.x >> 4);
  const int c0 = blockIdx.x * kBlock8;
  float v[kPer][8];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int r = r0 + i * kStep;
    if (r < rows) {
      load_cols<VEC>(x + static_cast<int64_t>(r) * ldx, c0, cols, l16, v[i]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
    }
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) top = max(top, top_of(v[i]));
  top = __reduce_max_sync(0xffffffffu, top);
  if (lane == 0) part[warp] = top;
  __syncthreads();
  top = __reduce_max_sync(0xffffffffu, part[lane & (kTileThreads8 / 32 - 1)]);
  const Scale8 s = scale8(top);
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int r = r0 + i * kStep;
    if (r < rows) store_codes<VEC>(q + static_cast<int64_t>(r) * ldq, c0, cols, l16, v[i], s.inv);
  }
  if (threadIdx.x == 0) scales[blockIdx.x * lds + blockIdx.y] = s.s;
}

static bool rows_aligned(const void* p, int64_t ld, size_t size, size_t to) {
  return (reinterpret_cast<uintptr_t>(p) % to) == 0 && (static_cast<uint64_t>(ld) * size) % to == 0;
}

template <class T>
static cudaError_t quant8_t(const void* xv, int64_t ldx, int rows, int cols, int block_rows, uint8_t* q, int64_t ldq,
                            float* scales, int64_t lds, cudaStream_t st) {
  const T* x = static_cast<const T*>(xv);
  const bool vec = rows_aligned(x, ldx, sizeof(T), 16) && rows_aligned(q, ldq, 1, 8);
  count_launch();
  if (block_rows == 1) {
    const dim3 grid((rows + kWarps8 * kRows8 - 1) / (kWarps8 * kRows8), (cols + 2 * kBlock8 - 1) / (2 * kBlock8));
    auto k = vec ? quant_rows_kernel<T, true> : quant_rows_kernel<T, false>;
    k<<<grid, kWarps8 * 32, 0, st>>>(x, ldx, rows, cols, q, ldq, scales, lds);
  } else {
    const dim3 grid((cols + kBlock8 - 1) / kBlock8, (rows + kBlock8 - 1) / kBlock8);
    auto k = vec ? quant_tiles_kernel<T, true> : quant_tiles_kernel<T, false>;
    k<<<grid, kTileThreads8, 0, st>>>(x, ldx, rows, cols, q, ldq, scales, lds);
  }
  return cudaGetLastError();
}

cudaError_t quant8(const void* x, Elem type, int64_t ldx, int rows, int cols, int block_rows, uint8_t* q, int64_t ldq,
                   float* scales, int64_t lds, cudaStream_t st) {
  switch (type) {
    case Elem::F32: return quant8_t<float>(x, ldx, rows, cols, block_rows, q, ldq, scales, lds, st);
    case Elem::F16: return quant8_t<__half>(x, ldx, rows, cols, block_rows, q, ldq, scales, lds, st);
    case Elem::BF16: return quant8_t<__nv_bfloat16>(x, ldx, rows, cols, block_rows, q, ldq, scales, lds, st);
  }
  return cudaErrorInvalidValue;
}

// ---------------------------------------------------------------------------
// y = x + resid; n = y * inv * gamma, inv = 1 / max(sqrt(mean(y^2) + eps),
// 1e-12 / sqrt(cols)); n -> (q, scales) by 1 x 128.
//
// With eps = 0 this is the trunk's norm, y * sqrt(cols) / max(|y|, 1e-12).  A
// row belongs to `warps` warps (one warp up to 1024 columns, so those rows need
// no block barrier), each holding C chunks of 256 columns in registers; the
// sum of squares is 32-bit.  Where it overflows (rows beyond 1e17) the row is
// scaled by the power of two that brings its largest value near 2^32 and
// summed again.
// ---------------------------------------------------------------------------
struct RowSum {
  float part[32];
  uint32_t top[32];
};

__device__ __forceinline__ float row_sum(float v, float* part, int warps, int wr, int lane) {
  v = warp_sum(v);
  if (warps == 1) return v;
  __syncthreads();  // the previous use of `part` has been read
  if (lane == 0) part[wr] = v;
  __syncthreads();
  float t = 0.0f;
  for (int i = 0; i < warps; ++i) t += part[i];  // the same order in every warp
  return t;
}
__device__ __forceinline__ uint32_t row_max(uint32_t v, uint32_t* part, int warps, int wr, int lane) {
  v = __reduce_max_sync(0xffffffffu, v);
  if (warps == 1) return v;
  __syncthreads();
  if (lane == 0) part[wr] = v;
  __syncthreads();
  uint32_t t = 0;
  for (int i = 0; i < warps; ++i) t = max(t, part[i]);
  return t;
}

template <class TX, class TR, int C, bool VEC>
__global__ void __launch_bounds__(C >= 4 ? 1024 : 512)
    add_norm_quant_kernel(const TX* x, int64_t ldx, const TR* resid, int64_t ldr, const float* __restrict__ gamma,
                          float eps, TR* y, int64_t ldy, uint8_t* __restrict__ q, int64_t ldq,
                          float* __restrict__ scales, int64_t lds, int rows, int cols, int warps, float inv_cols,
                          float most) {
  __shared__ RowSum sh;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per_cta = warps == 1 ? blockDim.x >> 5 : 1;
  const int wr = warps == 1 ? 0 : warp;  // this warp's place in its row
  const int row = blockIdx.x * per_cta + (warps == 1 ? warp : 0);
  if (row >= rows) return;  // whole warps, and whole blocks where a row spans a block
  float v[C][8];
#pragma unroll
  for (int i = 0; i < C; ++i) load_cols<VEC>(x + row * ldx, (wr + i * warps) * 256, cols, lane, v[i]);
  if (resid) {
#pragma unroll
    for (int i = 0; i < C; ++i) {
      float r[8];
      load_cols<VEC>(resid + row * ldr, (wr + i * warps) * 256, cols, lane, r);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] += r[j];
    }
    if (y) {
#pragma unroll
      for (int i = 0; i < C; ++i) store_cols<VEC>(y + row * ldy, (wr + i * warps) * 256, cols, lane, v[i]);
    }
  }
  float2 sq = make_float2(0.0f, 0.0f);
#pragma unroll
  for (int i = 0; i < C; ++i)
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const float2 u = make_float2(v[i][j], v[i][j + 1]);
      sq = __ffma2_rn(u, u, sq);
    }
  const float ss = row_sum(sq.x + sq.y, sh.part, warps, wr, lane);
  float inv;
  if (ss == __int_as_float(0x7f800000)) {  // the same for every thread of the row
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < C; ++i) top = max(top, top_of(v[i]));
    top = row_max(top, sh.top, warps, wr, lane);
    if (top >= 0x7f800000u) {
      inv = 0.0f;  // an infinity in the row: its finite values are 0 beside it, itself NaN
    } else {
      const float down = __uint_as_float((286u - (top >> 23)) << 23);  // brings the largest value to [2^32, 2^33)
      float t = 0.0f;
#pragma unroll
      for (int i = 0; i < C; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          v[i][j] *= down;
          t = fmaf(v[i][j], v[i][j], t);
        }
      t = row_sum(t, sh.part, warps, wr, lane);
      inv = rsqrtf(t * inv_cols);  // eps and the floor are below rounding here
    }
  } else {
    inv = fminf(rsqrtf(ss * inv_cols + eps), most);  // rsqrtf: within 2 ulp
    if (ss != ss) inv = ss;  // fminf drops a NaN
  }
  uint32_t tops[C];
#pragma unroll
  for (int i = 0; i < C; ++i) {
    float g[8];
    load_cols<VEC>(gamma, (wr + i * warps) * 256, cols, lane, g);
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const float2 u = __fmul2_rn(__fmul2_rn(make_float2(v[i][j], v[i][j + 1]), make_float2(inv, inv)),
                                  make_float2(g[j], g[j + 1]));
      v[i][j] = u.x;
      v[i][j + 1] = u.y;
    }
    tops[i] = top_of(v[i]);
  }
  const Scales8<C> sc = half_warp_scales<C>(tops, lane);
#pragma unroll
  for (int i = 0; i < C; ++i) store_codes<VEC>(q + row * ldq, (wr + i * warps) * 256, cols, lane, v[i], sc.inv[i]);
  const int kb = (wr + sc.own_block * warps) * 2 + (lane >> 4);
  if (sc.writer && kb * kBlock8 < cols) scales[kb * lds + row] = sc.own;
}

template <class TX, class TR>
static cudaError_t add_norm_quant8_t(const AddNorm8& a, cudaStream_t st) {
  const TX* x = static_cast<const TX*>(a.x);
  const TR* resid = static_cast<const TR*>(a.resid);
  TR* y = static_cast<TR*>(a.y);
  const bool vec = rows_aligned(x, a.ldx, sizeof(TX), 16) && (!resid || rows_aligned(resid, a.ldr, sizeof(TR), 16)) &&
                   (!y || rows_aligned(y, a.ldy, sizeof(TR), 16)) && rows_aligned(a.q, a.ldq, 1, 8) &&
                   rows_aligned(a.gamma, 0, 4, 16);
  const int chunks = (a.cols + 255) / 256;
  int c, warps, threads;
  if (chunks <= 4) {  // one warp per row
    c = chunks <= 1 ? 1 : chunks <= 2 ? 2 : 4;
    warps = 1;
    threads = 128;
  } else {  // one block per row
    c = chunks <= 32 ? 2 : 4;
    warps = (chunks + c - 1) / c;
    threads = warps * 32;
  }
  const float inv_cols = 1.0f / static_cast<float>(a.cols);
  const float most = static_cast<float>(std::sqrt(static_cast<double>(a.cols)) * 1e12);  // 1 / the norm's floor
  const int per_cta = warps == 1 ? threads / 32 : 1;
  const int grid = (a.rows + per_cta - 1) / per_cta;
  count_launch();
#define LBRR_LAUNCH(CC)                                                                                            \
  (vec ? add_norm_quant_kernel<TX, TR, CC, true> : add_norm_quant_kernel<TX, TR, CC, false>)<<<grid, threads, 0,   \
                                                                                               st>>>(             \
      x, a.ldx, resid, a.ldr, a.gamma, a.eps, y, a.ldy, a.q, a.ldq, a.scales, a.lds, a.rows, a.cols, warps, inv_cols, most)
  switch (c) {
    case 1: LBRR_LAUNCH(1); break;
    case 2: LBRR_LAUNCH(2); break;
    default: LBRR_LAUNCH(4); break;
  }
#undef LBRR_LAUNCH
  return cudaGetLastError();
}

cudaError_t add_norm_quant8(const AddNorm8& a, cudaStream_t st) {
  if (a.x_type == Elem::F32 && a.resid_type == Elem::F32) return add_norm_quant8_t<float, float>(a, st);
  if (a.x_type == Elem::F16 && a.resid_type == Elem::F32) return add_norm_quant8_t<__half, float>(a, st);
  if (a.x_type == Elem::F16 && a.resid_type == Elem::F16) return add_norm_quant8_t<__half, __half>(a, st);
  if (a.x_type == Elem::BF16 && a.resid_type == Elem::F32) return add_norm_quant8_t<__nv_bfloat16, float>(a, st);
  if (a.x_type == Elem::BF16 && a.resid_type == Elem::BF16)
    return add_norm_quant8_t<__nv_bfloat16, __nv_bfloat16>(a, st);
  return cudaErrorInvalidValue;
}

}  // namespace lbrr
