// Quantising kernels of the 8-bit path: blocks of 1 x 128 or 128 x 128 of a
// matrix to e4m3 with scales, and the trunk's RMSNorm with the residual's
// addition and an 8-bit output.  Both are one pass over their data (every
// value is read once, held in registers while its block's or row's statistics
// form, and written once), so HBM bounds them where there are rows enough to
// fill the GPU.  What made the difference was having the next rows' loads in
// flight while a block is worked on (71362 x 512 fp16 28 -> 20 us, 5.4 TB/s;
// norm 4099 x 5000 bf16 46 -> 29 us, 5.0 TB/s) and few instructions per value (a
// division per block, sixteen compares per eight values and a reduction per
// block cost 15-25 %).  Norm of 71362 x 256 (fp16 branch, fp32 stream): 33 us,
// 6.0 TB/s.
#include <algorithm>
#include <cmath>

#include "quant8.cuh"

namespace lbrr {

// ---------------------------------------------------------------------------
// v -> (q, scales), blocks of 1 x 128.  A warp takes kRows8 rows of 256
// columns (16 lanes per block) at a time and has the next ones' loads in flight
// meanwhile; eight warps cover 32 rows, so the scales of a block column leave
// as whole sectors.  Unaligned rows (Shifted8) leave no registers for the loads
// ahead (at four blocks per SM: 71362 x 257 fp32 45 us, 53 with them; 37889 x 588
// bf16 32 and 33).
// ---------------------------------------------------------------------------
constexpr int kRows8 = 4;
constexpr int kWarps8 = 8;
// Blocks per SM: four where 64 registers a thread are enough, three otherwise
// (four, with spills: 71362 x 512 fp32 40 us and 30, 300000 x 64 fp16 22.5 and
// 20.7, 37889 x 588 bf16 32.6 and 27.5, 71362 x 257 fp16 37 and 32).
template <class T, bool VEC, bool NARROW>
constexpr int kBlocksPerSm8 = VEC && !NARROW && sizeof(T) == 2 ? 4 : 3;

// NARROW (up to 128 columns): the two halves of a warp take rows of their own.
template <class T, bool VEC, bool NARROW>
__global__ void __launch_bounds__(kWarps8 * 32, kBlocksPerSm8<T, VEC, NARROW>)
    quant_rows_kernel(const T* __restrict__ x, int64_t ldx, int rows, int cols, uint8_t* __restrict__ q, int64_t ldq,
                      float* __restrict__ scales, int64_t lds, bool q_aligned) {
  constexpr int kPerWarp = NARROW ? 2 * kRows8 : kRows8;  // rows
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int half = lane >> 4, at = NARROW ? lane & 15 : lane;  // `at`: this lane's columns
  const int c0 = blockIdx.y * 2 * kBlock8;
  constexpr bool kAhead = VEC;
  auto row_of = [&](int r0, int i) { return NARROW ? r0 + 2 * i + half : r0 + i; };
  Ahead8<VEC, NARROW ? 16 : 32, T> next[kRows8];
  auto row_at = [&](int r0, int i) { return x + static_cast<int64_t>(row_of(r0, i)) * ldx; };
  auto fetch = [&](int r0) {
#pragma unroll
    for (int i = 0; i < kRows8; ++i)
      if (row_of(r0, i) < rows) next[i].load(row_at(r0, i), c0, cols, at);
  };
  const int step = gridDim.x * kWarps8 * kPerWarp;
  int r0 = (blockIdx.x * kWarps8 + warp) * kPerWarp;
  if (kAhead) fetch(r0);
  for (; r0 < rows; r0 += step) {
    if (!kAhead) fetch(r0);
    float v[kRows8][8];
    uint32_t top[kRows8];
#pragma unroll
    for (int i = 0; i < kRows8; ++i) {
      if (!VEC || row_of(r0, i) < rows) {  // rows past the last one: whole warps shift, nothing is stored
        next[i].get(row_at(r0, i), c0, cols, at, v[i]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
      }
      top[i] = top_of(v[i]);
    }
    if (kAhead) fetch(r0 + step);
    const Scales8<kRows8> sc = half_warp_scales<kRows8>(top, lane);
    const Quotient8 own_quotient = quotient8(sc.own);
    if (__any_sync(0xffffffffu, sc.own.s > kHugeScale8)) {
      const float own_down = sc.own.s > kHugeScale8 ? kHugeDown8 : 1.0f;
#pragma unroll
      for (int i = 0; i < kRows8; ++i) {
        const float down = sc.of(own_down, i, lane);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] *= down;
      }
    }
#pragma unroll
    for (int i = 0; i < kRows8; ++i) {
      const Quotient8 quotient{sc.of(own_quotient.hi, i, lane), sc.of(own_quotient.lo, i, lane)};
      if (row_of(r0, i) < rows)
        store_codes<true>(q + static_cast<int64_t>(row_of(r0, i)) * ldq, c0, cols, at, v[i], quotient, VEC || q_aligned);
    }
    const int own = row_of(r0, sc.own_block), kb = NARROW ? 0 : blockIdx.y * 2 + half;
    if (sc.writer && own < rows && kb * kBlock8 < cols) scales[kb * lds + own] = sc.own.s;
  }
}

// Blocks of 128 x 128: 32 values per thread.  16-bit inputs: two CTAs per SM
// walk the blocks with the next one's loads in flight (71362 x 512: 33 -> 21 us);
// 32-bit inputs and unaligned rows leave no registers for that, so each block has
// its own CTA (8192 x 8192 fp32: 51 us, 61 with the loop; 9402 x 1227 bf16: 11
// and 16.6).  `blocks_x`: blocks side by side.
constexpr int kTileThreads8 = 512;
template <class T, bool VEC>
__global__ void __launch_bounds__(kTileThreads8, 2)
    quant_tiles_kernel(const T* __restrict__ x, int64_t ldx, int rows, int cols, uint8_t* __restrict__ q, int64_t ldq,
                       float* __restrict__ scales, int64_t lds, bool q_aligned, int blocks_x, int blocks) {
  constexpr int kPer = kBlock8 * kBlock8 / kTileThreads8 / 8;  // row groups per thread
  constexpr int kStep = kTileThreads8 / 16;                    // rows per group
  __shared__ uint32_t part[2][kTileThreads8 / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int l16 = lane & 15;  // the 16 lanes of a row
  Ahead8<VEC, 16, T> next[kPer];
  auto fetch = [&](int block) {
    const int by = block / blocks_x, c0 = (block - by * blocks_x) * kBlock8;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int r = by * kBlock8 + (threadIdx.x >> 4) + i * kStep;
      if (r < rows) next[i].load(x + static_cast<int64_t>(r) * ldx, c0, cols, l16);
    }
  };
  constexpr bool kAhead = VEC && sizeof(T) == 2;
  int block = blockIdx.x;
  fetch(block);
  for (int it = 0; block < blocks; block += gridDim.x, it ^= 1) {
    const int by = block / blocks_x, bx = block - by * blocks_x;
    const int r0 = by * kBlock8 + (threadIdx.x >> 4);
    float v[kPer][8];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int r = r0 + i * kStep;
      if (!VEC || r < rows) next[i].get(x + static_cast<int64_t>(r) * ldx, bx * kBlock8, cols, l16, v[i]);
      if (r >= rows) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
      }
      top = max(top, top_of(v[i]));
    }
    if (kAhead && block + static_cast<int>(gridDim.x) < blocks) fetch(block + gridDim.x);
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) part[it][warp] = top;
    __syncthreads();  // one per block: the next block writes the other half of `part`
    top = __reduce_max_sync(0xffffffffu, part[it][lane & (kTileThreads8 / 32 - 1)]);
    const Scale8 s = scale8(top);
    const Quotient8 quotient = quotient8(s);
    if (s.s > kHugeScale8) {  // the same for every thread
#pragma unroll
      for (int i = 0; i < kPer; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] *= kHugeDown8;
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int r = r0 + i * kStep;
      if (r < rows) store_codes<true>(q + static_cast<int64_t>(r) * ldq, bx * kBlock8, cols, l16, v[i], quotient, VEC || q_aligned);
    }
    if (threadIdx.x == 0) scales[bx * lds + by] = s.s;
    if (!kAhead) break;
  }
}

static bool rows_aligned(const void* p, int64_t ld, size_t size, size_t to) {
  return (reinterpret_cast<uintptr_t>(p) % to) == 0 && (static_cast<uint64_t>(ld) * size) % to == 0;
}

template <class T>
static cudaError_t quant8_t(const void* xv, int64_t ldx, int rows, int cols, int block_rows, uint8_t* q, int64_t ldq,
                            float* scales, int64_t lds, cudaStream_t st) {
  const T* x = static_cast<const T*>(xv);
  const bool q_aligned = rows_aligned(q, ldq, 1, 8), vec = q_aligned && rows_aligned(x, ldx, sizeof(T), 16);
  count_launch();
  if (block_rows == 1) {
    const bool narrow = cols <= kBlock8;
    const int per_block = kWarps8 * kRows8 * (narrow ? 2 : 1);
    const int groups = (rows + per_block - 1) / per_block, chunks = (cols + 2 * kBlock8 - 1) / (2 * kBlock8);
    const int per_sm = vec ? (narrow ? kBlocksPerSm8<T, true, true> : kBlocksPerSm8<T, true, false>)
                           : (narrow ? kBlocksPerSm8<T, false, true> : kBlocksPerSm8<T, false, false>);
    const int resident = std::max(1, per_sm * kSms / chunks);  // blocks per column chunk that run at one time
    const dim3 grid(std::min(groups, resident), chunks);
    auto k = vec ? (narrow ? quant_rows_kernel<T, true, true> : quant_rows_kernel<T, true, false>)
                 : (narrow ? quant_rows_kernel<T, false, true> : quant_rows_kernel<T, false, false>);
    k<<<grid, kWarps8 * 32, 0, st>>>(x, ldx, rows, cols, q, ldq, scales, lds, q_aligned);
  } else {
    const int blocks_x = (cols + kBlock8 - 1) / kBlock8;
    const int blocks = blocks_x * ((rows + kBlock8 - 1) / kBlock8);
    auto k = vec ? quant_tiles_kernel<T, true> : quant_tiles_kernel<T, false>;
    k<<<vec && sizeof(T) == 2 ? std::min(blocks, 2 * kSms) : blocks, kTileThreads8, 0, st>>>(x, ldx, rows, cols, q, ldq, scales, lds,
                                                                                   q_aligned, blocks_x, blocks);
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
// row belongs to `warps` warps (one warp up to 512 columns, so those rows need
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

template <class TX, class TR, int C, bool VEC, bool LOOP, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == 512 ? 2 : 1)
    add_norm_quant_kernel(const TX* x, int64_t ldx, const TR* resid, int64_t ldr, const float* __restrict__ gamma,
                          float eps, TR* y, int64_t ldy, uint8_t* __restrict__ q, int64_t ldq,
                          float* __restrict__ scales, int64_t lds, int rows, int cols, int warps, float inv_cols,
                          float most) {
  __shared__ RowSum sh;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per_cta = warps == 1 ? blockDim.x >> 5 : 1;
  const int wr = warps == 1 ? 0 : warp;  // this warp's place in its row
  const int step = gridDim.x * per_cta;
  constexpr bool kUnits = VEC && C == 2;  // 4099 x 5000 fp16 + fp32: 46 -> 42 us; for C = 4, 500 x 24000: 33 -> 38
  Raw8<TX> nx[C];
  Raw8<TR> nr[C];
  auto fetch = [&](int64_t r) {
#pragma unroll
    for (int i = 0; i < C; ++i) {
      load_raw<VEC, kUnits>(x + r * ldx, (wr + i * warps) * 256, cols, lane, nx[i]);
      if (resid) load_raw<VEC, kUnits>(resid + r * ldr, (wr + i * warps) * 256, cols, lane, nr[i]);
    }
  };
  int64_t row = blockIdx.x * per_cta + (warps == 1 ? warp : 0);
  if (row >= rows) return;  // whole warps, and whole blocks where a row spans a block
  fetch(row);
  for (;; row += step) {
    float v[C][8];
#pragma unroll
    for (int i = 0; i < C; ++i) {
      nx[i].get(v[i]);
      if (kUnits) drop_past((wr + i * warps) * 256, cols, lane, v[i]);
    }
    if (resid) {
#pragma unroll
      for (int i = 0; i < C; ++i) {
        float r[8];
        nr[i].get(r);
        if (kUnits) drop_past((wr + i * warps) * 256, cols, lane, r);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] += r[j];
      }
      if (LOOP && row + step < rows) fetch(row + step);
      if (y) {
#pragma unroll
        for (int i = 0; i < C; ++i) store_cols<VEC>(y + row * ldy, (wr + i * warps) * 256, cols, lane, v[i]);
      }
    } else if (LOOP && row + step < rows) {
      fetch(row + step);
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
    float inverse[C];
    inverses(sc, lane, inverse);
#pragma unroll
    for (int i = 0; i < C; ++i) store_codes<VEC>(q + row * ldq, (wr + i * warps) * 256, cols, lane, v[i], inverse[i]);
    const int kb = (wr + sc.own_block * warps) * 2 + (lane >> 4);
    if (sc.writer && kb * kBlock8 < cols) scales[kb * lds + row] = sc.own.s;
    if (!LOOP || row + step >= rows) break;
  }
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
  const float inv_cols = 1.0f / static_cast<float>(a.cols);
  const float most = static_cast<float>(std::sqrt(static_cast<double>(a.cols)) * 1e12);  // 1 / the norm's floor
  count_launch();
  constexpr bool kAhead = sizeof(TX) + sizeof(TR) < 8;
#define LBRR_LAUNCH(CC, LOOP, MAX)                                                                          \
  (vec ? add_norm_quant_kernel<TX, TR, CC, true, LOOP && kAhead, MAX>                                        \
       : add_norm_quant_kernel<TX, TR, CC, false, false, MAX>)                                               \
      <<<grid, threads, 0, st>>>(x, a.ldx, resid, a.ldr, a.gamma, a.eps, y, a.ldy, a.q, a.ldq, a.scales, a.lds, \
                                 a.rows, a.cols, warps, inv_cols, most)
  if (chunks <= 2) {  // a warp per row
    constexpr int warps = 1, threads = 128;
    const int grid = (a.rows + 3) / 4;
    if (chunks == 1)
      LBRR_LAUNCH(1, false, threads);
    else
      LBRR_LAUNCH(2, false, threads);
  } else if (chunks <= 64) {  // a block per row
    // As many blocks as run at one time, the next row's loads in flight (4099 x
    // 5000 bf16: 46 -> 30 us).  Where that needs more registers than there are, as
    // many blocks as rows: both inputs fp32 (4099 x 5000: 44 us, 57 with loads
    // ahead), and unaligned rows, which load value by value (9402 x 1227 bf16: 26
    // and 37).
    const int warps = (chunks + 1) / 2, threads = warps * 32;
    const int grid = vec && kAhead ? std::min(a.rows, kSms * (1024 / threads)) : a.rows;
    if (threads <= 512)
      LBRR_LAUNCH(2, true, 512);
    else
      LBRR_LAUNCH(2, true, 1024);
  } else {  // rows whose registers leave no room for the next one's
    const int warps = (chunks + 3) / 4, threads = warps * 32, grid = a.rows;
    LBRR_LAUNCH(4, false, 1024);
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
