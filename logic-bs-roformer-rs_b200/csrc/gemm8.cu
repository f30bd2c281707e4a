// 8-bit matrix product with block scales.
//
//   acc[m][n] = sum over 128-column blocks b of
//               a_scale[b][m] * w_scale[b][n / 128] * sum over k in b of A[m][k] W[n][k]
//   out = acc + bias[n] + resid[m][n], or gelu(acc + bias) -> (q, scales) by 1 x 128.
//
// Products of two e4m3 values are exact in 32 bits; each block's sum is formed
// by the tensor core in TMEM, then multiplied once by its two scales and added
// to the 32-bit total in registers.
//
// A pair of CTAs (cluster of two, cta_group::2) walks 256 x 256 tiles, each CTA
// holding 128 rows of A, half of W's rows and the totals of its own 128 rows:
// against one CTA per 128 x 256 tile the operands' L2 traffic falls by a third
// (12 TB/s of L2 reads at 0.54 ms for 8192^3).  A K-block of 128
// is four tcgen05.mma (kind::f8f6f4, 256 x 256 x 32) into one of two 256-column
// accumulators, so the tensor cores work on block b + 1 while eight warps of
// each CTA (two per TMEM lane quadrant, one accumulator row per thread, 128 of
// the 256 columns each) read block b, scale it and add it to 128 totals per
// thread.  A 128-column part is one scale block of W, so the factor of a block
// is one number per thread.  After the last block the same warps write the tile
// through shared memory and TMA stores while the tensor cores run ahead into
// the next tile.  Warps: 0..7 totals and output, 8 TMA loads, 9 TMEM
// allocation and (CTA 0) MMA issue, 10 the tiles' places and bias and the
// blocks' scales (asynchronous copies into rings in shared memory, so the output
// warps never wait for a global load), 11 none (it completes the warpgroup that
// gives its registers away).
//
// Measured (B200, replayed back to back, SM clock under the 1000 W cap): 8192^3
// to bf16 0.52-0.55 ms (2.0-2.1 PFLOP/s) at 1.39 GHz, 740 cycles a K-block where
// its MMAs take 512 and the same kernel without the totals' work 630: power and
// the totals' latency bound it.  71362 x 1536 x 256 to fp16 57 us (4.2 TB/s, 3950
// cycles a tile: totals 1300, conversion and staging 950, stores 300-500, waits
// 500), 71362 x 256 x 1024 with fp32 residual 52 us (4.3 TB/s; a CTA's 384 KB a
// tile take 16.7 k of its 21 k cycles), 71362 x 1024 x 256 with GELU to 8 bits 61
// us (about 6600 cycles a tile, 3700 of them GELU, whose MUFU part alone is 2070).
// Tried and left out: one CTA per 128 x 256 tile (8192^3 662 us against 607 for
// the pair at that time), a second issuing warp (the two accumulators' MMAs
// interleave and end together: 675), 256 x 128 tiles with two sets of output
// warps on alternate tiles (8192^3 696, 71362 x 1024 x 256 55), an L2 prefetch of
// the residual (52 -> 60 us), the bias added with the conversions (57 -> 65 us).
#include <math_constants.h>

#include <atomic>

#include "cp_async.cuh"
#include "fastdiv.cuh"
#include "gelu8.cuh"
#include "gemm8_few.cuh"
#include "quant8.cuh"
#include "ring.h"

namespace lbrr {

constexpr int kM8 = 128, kN8 = 256, kK8 = 128;
constexpr int kStages8 = 4;
constexpr int kABytes8 = kM8 * kK8, kWBytes8 = kN8 / 2 * kK8;  // a CTA's rows of A, its half of the tile's W rows
constexpr int kStageBytes8 = kABytes8 + kWBytes8;
constexpr int kOutWarps8 = 8;
constexpr int kPart8 = 128, kParts8 = kN8 / kPart8;  // columns of an output warp; output warps per TMEM lane quadrant
constexpr int kBufBytes8 = 4096;                     // 32 rows x 128 bytes; two per output warp
constexpr int kBufOff8 = kStages8 * kStageBytes8;
constexpr int kRing8 = 8, kAhead8 = 4;               // K-blocks of scales (and tiles) held, and fetched ahead
constexpr int kBlockFloats8 = kM8 + 4;               // a K-block: 128 rows' scales, then W's of the two parts
constexpr int kRingOff8 = kBufOff8 + kOutWarps8 * 2 * kBufBytes8;
constexpr int kTileOff8 = kRingOff8 + kRing8 * kBlockFloats8 * 4;
constexpr int kTileFloats8 = kN8 + 4;                // a tile: its bias, its first row and column
constexpr int kTailOff8 = kTileOff8 + kRing8 * kTileFloats8 * 4;  // 33rd words of the residual's rows, per buffer
constexpr int kBarOff8 = kTailOff8 + kOutWarps8 * 2 * 32 * 4;
constexpr int kSmem8 = kBarOff8 + 256;
constexpr int kThreads8 = kOutWarps8 * 32 + 128;
constexpr int kLoadWarp8 = kOutWarps8, kMmaWarp8 = kOutWarps8 + 1, kScaleWarp8 = kOutWarps8 + 2;
constexpr int kRegsOut8 = 216, kRegsOther8 = 72;
constexpr int kLaunchRegs8 = 168;
static_assert(kSmem8 <= 232448, "exceeds the 227 KB per-CTA shared memory limit");
static_assert(kOutWarps8 * 32 * kRegsOut8 + 128 * kRegsOther8 <= kThreads8 * kLaunchRegs8, "register split");

enum class Out8 { F32, F16, BF16, Q8 };
template <Out8 O>
struct OutType {
  using T = float;
};
template <>
struct OutType<Out8::F16> {
  using T = __half;
};
template <>
struct OutType<Out8::BF16> {
  using T = __nv_bfloat16;
};
template <>
struct OutType<Out8::Q8> {
  using T = uint8_t;
};

struct Params8 {
  Gemm8 g;
  int mt, nt;          // row tiles (of the pair), column tiles
  FastDiv per;         // division by kGroup8 * nt, the tiles of a group
  int kb;             // K-blocks
  bool out_tma;       // the output's rows allow TMA stores
  bool out_tail;      // ... of a last, partial block too: a TMA store ends on a 16-byte boundary, not on the
                      // matrix's last column (measured: it wrote the rest of the 16 bytes)
  bool out_pairs;     // ... two blocks at a time (tmOut is [blocks][rows][128 bytes])
  bool resid_vec;     // the residual's rows allow 16-byte copies
};

// Tiles in groups of kGroup8 row tiles, rows fastest: the pairs running at one
// time share both their A rows and their W rows in L2.
constexpr int kGroup8 = 8;
__device__ __forceinline__ void tile8(const Params8& p, int idx, int& m0, int& n0) {
  const int gi = p.per.div(idx), rem = idx - gi * (kGroup8 * p.nt);
  const int rows = p.mt - gi * kGroup8;
  const int n = rows >= kGroup8 ? rem / kGroup8 : rem / rows;
  m0 = (gi * kGroup8 + rem - n * min(rows, kGroup8)) * (2 * kM8);
  n0 = n * kN8;
}

// Byte o of row r in a buffer of 32 rows of 128 bytes with the TMA 128-byte swizzle.
__device__ __forceinline__ uint32_t swz(int r, int o) {
  return static_cast<uint32_t>(r * 128 + ((((o >> 4) ^ (r & 7)) << 4) | (o & 15)));
}

// Rows R0, R0 + DR, ... of a whole block between a buffer and global memory in
// 4-byte words, `at` being this lane's word of row R0.  Two warps per scheduler
// hide little latency, so what counts is instructions per row: no predicates, one
// addition per address (3500 x 4618 x 71 fp32:
// 48 -> 29 us, 20 where rows are aligned).
template <int R0, int DR>
__device__ __forceinline__ void load_words(uint8_t* buf, uintptr_t at, int64_t step, int lane) {
#pragma unroll 8
  for (int r = R0; r < 32; r += DR, at += step)
    cp_async4(buf + swz(r, lane * 4), reinterpret_cast<const void*>(at), true);
}
// HALF: the rows are halves that start between words; word j of a row holds columns 2j - 1 and 2j.
template <int R0, int DR, bool HALF>
__device__ __forceinline__ void store_words(const uint8_t* buf, uintptr_t at, int64_t step, int lane) {
#pragma unroll 8
  for (int r = R0; r < 32; r += DR, at += step) {
    uint32_t w = *reinterpret_cast<const uint32_t*>(buf + swz(r, lane * 4));
    if (HALF) w = __funnelshift_l(__shfl_up_sync(0xffffffffu, w, 1), w, 16);
    if (!HALF || lane > 0) *reinterpret_cast<uint32_t*>(at) = w;
  }
}

// One 32-row block of up to 128 bytes per row from global memory to a buffer,
// asynchronously.  Rows on 16-byte boundaries and whole: 16 bytes a copy.
// Otherwise 4-byte words: rows of halves that start between words come with the
// half before them (word j holds halves 2j - 1 and 2j) and their 33rd word goes to
// `tail`; the reader shifts them.  A word is copied if it holds a value of the
// block, so no other word is touched.
template <class T>
__device__ __forceinline__ void load_block(uint8_t* buf, uint32_t* tail, const T* src, int64_t ld, int rows, int cols,
                                           bool vec, int lane) {
  constexpr int E = 128 / sizeof(T);
  if (vec && cols >= E) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = i * 4 + lane / 8, v = lane % 8;
      if (r < rows) cp_async16(buf + swz(r, v * 16), src + r * ld + v * (16 / static_cast<int>(sizeof(T))));
    }
    return;
  }
  if (rows >= 32 && cols >= E) {
    const uintptr_t word = ~uintptr_t(3), at = reinterpret_cast<uintptr_t>(src);
    const int64_t step = ld * static_cast<int64_t>(sizeof(T));
    if ((step & 3) == 0) {
      load_words<0, 1>(buf, (at & word) + lane * 4, step, lane);
    } else {  // every other row starts between words
      load_words<0, 2>(buf, (at & word) + lane * 4, 2 * step, lane);
      load_words<1, 2>(buf, ((at + step) & word) + lane * 4, 2 * step, lane);
    }
  } else {
#pragma unroll 4
    for (int r = 0; r < 32; ++r) {
      const uintptr_t at = reinterpret_cast<uintptr_t>(src + r * ld);
      const int half = (at & 2) != 0;  // never for 32-bit values
      const int first = lane * (4 / static_cast<int>(sizeof(T))) - half;
      if (r < rows && first < cols)
        cp_async4(buf + swz(r, lane * 4), reinterpret_cast<const void*>((at & ~uintptr_t(3)) + lane * 4), true);
    }
  }
  if (sizeof(T) == 2 && lane < rows && cols >= E) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(src + lane * ld);
    if (at & 2) cp_async4(tail + lane, reinterpret_cast<const void*>((at & ~uintptr_t(3)) + 128), true);
  }
}
// ... and back, where a TMA store cannot: in words, and single values where a row begins or ends inside one
// (bytes whose rows do not start on words go one by one).
template <class T>
__device__ __forceinline__ void store_block(const uint8_t* buf, T* dst, int64_t ld, int rows, int cols, int lane) {
  constexpr int E = 128 / sizeof(T), P = 4 / sizeof(T);  // values per row and per word
  cols = min(cols, E);
  auto value = [&](int r, int c) { return *reinterpret_cast<const T*>(buf + swz(r, c * static_cast<int>(sizeof(T)))); };
  const uintptr_t off = reinterpret_cast<uintptr_t>(dst) | (static_cast<uintptr_t>(ld) * sizeof(T));
  const bool whole = rows >= 32 && cols == E && sizeof(T) > 1;
  const int64_t step = ld * static_cast<int64_t>(sizeof(T));
  const uintptr_t at = reinterpret_cast<uintptr_t>(dst) + lane * 4;
  if (whole && (off & 3) == 0) {
    store_words<0, 1, false>(buf, at, step, lane);
  } else if ((off & 3) == 0) {
    const int words = cols / P;
#pragma unroll 8
    for (int r = 0; r < 32; ++r)
      if (r < rows && lane < words)
        *reinterpret_cast<uint32_t*>(dst + r * ld + lane * P) = *reinterpret_cast<const uint32_t*>(buf + swz(r, lane * 4));
    for (int c = words * P; c < cols; ++c)
      if (lane < rows) dst[lane * ld + c] = value(lane, c);
  } else if (sizeof(T) == 2) {
    // rows that start between words
    if (whole) {
      if ((step & 3) == 0) {
        store_words<0, 1, true>(buf, at - 2, step, lane);
      } else if ((at & 2) == 0) {
        store_words<0, 2, false>(buf, at, 2 * step, lane);
        store_words<1, 2, true>(buf, at + step - 2, 2 * step, lane);
      } else {
        store_words<0, 2, true>(buf, at - 2, 2 * step, lane);
        store_words<1, 2, false>(buf, at + step, 2 * step, lane);
      }
    } else {
#pragma unroll 8
      for (int r = 0; r < 32; ++r) {
        T* row = dst + r * ld;
        const int half = static_cast<int>(reinterpret_cast<uintptr_t>(row) >> 1) & 1, c = 2 * lane - half;
        const uint32_t own = *reinterpret_cast<const uint32_t*>(buf + swz(r, lane * 4));
        const uint32_t before = __shfl_up_sync(0xffffffffu, own, 1);
        if (r < rows && c >= 0 && c + 1 < cols)
          *reinterpret_cast<uint32_t*>(row + c) = __funnelshift_l(before, own, half * 16);
      }
    }
    if (lane < rows) {
      T* row = dst + lane * ld;
      const int half = static_cast<int>(reinterpret_cast<uintptr_t>(row) >> 1) & 1;
      if (half) row[0] = value(lane, 0);
      if ((cols + half) & 1) row[cols - 1] = value(lane, cols - 1);
    }
  } else {
#pragma unroll 8
    for (int r = 0; r < 32; ++r)
#pragma unroll
      for (int c = lane; c < E; c += 32)
        if (r < rows && c < cols) dst[r * ld + c] = value(r, c);
  }
}

// Columns of the pair's tile that the MMA computes: whole 32s, 16 per CTA's half of W.
__device__ __forceinline__ int tile_cols8(const Params8& p, int n0) { return min(kN8, (p.g.n - n0 + 31) & ~31); }

// 32 columns of a block's sums, times the block's factor, added to the totals.
template <int B>
__device__ __forceinline__ void add_scaled(float2 (&acc)[kPart8 / 2], const uint32_t (&v)[32], float s) {
  const float2 f = make_float2(s, s);
#pragma unroll
  for (int i = 0; i < 16; ++i)
    acc[16 * B + i] =
        __ffma2_rn(make_float2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), f, acc[16 * B + i]);
}

// Keeps the compiler from starting on these values before, or leaving them for after, this point.
template <int N>
__device__ __forceinline__ void hold(float2* x) {
#pragma unroll
  for (int i = 0; i < N; i += 4)
    asm volatile("" : "+f"(x[i].x), "+f"(x[i].y), "+f"(x[i + 1].x), "+f"(x[i + 1].y), "+f"(x[i + 2].x), "+f"(x[i + 2].y), "+f"(x[i + 3].x), "+f"(x[i + 3].y));
}
// ODD: a 16-bit residual with rows that may start between 4-byte words.
template <Out8 O, bool ODD>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads8, 1)
    gemm8_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmW,
                 const __grid_constant__ CUtensorMap tmOut, const __grid_constant__ Params8 p, int* status) {
  extern __shared__ __align__(1024) uint8_t smem[];
  using T = typename OutType<O>::T;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kBarOff8);  // CTA 0's: both CTAs' loads
  uint64_t* empty = full + kStages8;
  uint64_t* acc_full = empty + kStages8;  // [2], the block's sums and its scales
  uint64_t* acc_empty = acc_full + 2;     // [2], CTA 0's: both CTAs' output warps
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  if ((smem_u32(smem) & 1023u) != 0) {  // the same in both CTAs: nothing allocated yet
    if (threadIdx.x == 0) report_status(status, kDevSmemMisaligned);
    return;
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages8; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&acc_full[s], 2);
      mbar_init(&acc_empty[s], 2 * kOutWarps8);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == kLoadWarp8 && lane == 0) {
    tma_prefetch(&tmA);
    tma_prefetch(&tmW);
  }
  if (warp == kMmaWarp8) tmem_alloc_pair(tmem_slot, 512);
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int n_tiles = p.mt * p.nt, first = blockIdx.x / 2, step = gridDim.x / 2;
  // the launcher checks the compiled register count before the first launch
  if (warp >= kOutWarps8) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther8));

  if (warp == kLoadWarp8) {
    if (lane == 0) {
      uint32_t c = 0;
      bool ok = true;
      for (int tile = first; ok && tile < n_tiles; tile += step) {
        int m0, n0;
        tile8(p, tile, m0, n0);
        const int a_row = m0 + rank * kM8, w_row = n0 + rank * (tile_cols8(p, n0) / 2);
        for (int kb = 0; kb < p.kb; ++kb, ++c) {
          const int s = c % kStages8;
          if (!(ok = mbar_wait(&empty[s], ((c / kStages8) & 1) ^ 1u, abort_flag, status))) break;
          uint8_t* sa = smem + s * kStageBytes8;
          const uint32_t bar = map_to_rank(&full[s], 0);
          if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * kStageBytes8);
          tma_load_2d_pair(sa, &tmA, bar, kb * kK8, a_row);
          tma_load_2d_pair(sa + kABytes8, &tmW, bar, kb * kK8, w_row);
        }
      }
      // The commits that free the stages arrive on both CTAs' barriers by themselves, and the final cluster barrier does
      // not wait for them: the last ones have arrived before either CTA may go.
      ok = ok && drain_ring<kStages8>(c, [&](int s, uint32_t parity) {
             return mbar_wait(&empty[s], parity, abort_flag, status);
           });
      if (!ok && rank == 0) {  // the pair's copies in flight land before its shared memory goes
        for (uint32_t i = c > kStages8 ? c - kStages8 : 0; i < c; ++i) {
          int none = 0;
          mbar_wait(&full[i % kStages8], (i / kStages8) & 1, &none, nullptr);
        }
      }
    }
  } else if (warp == kMmaWarp8) {
    if (rank == 0) {  // the whole warp, so that descriptors and addresses stay uniform; one lane issues
      const uint32_t leader = elect_one();
      uint32_t c = 0;
      bool ok = true, loaded = false;  // loaded: block c's operands were seen to have landed
      for (int tile = first; ok && tile < n_tiles; tile += step) {
        int m0, n0;
        tile8(p, tile, m0, n0);
        const uint32_t idesc = idesc_e4m3_f32(2 * kM8, tile_cols8(p, n0));
        for (int kb = 0; kb < p.kb; ++kb, ++c) {
          const int s = c % kStages8, slot = c & 1;
          // the accumulator, waited for last, is what the MMAs usually wait for
          if (!__all_sync(0xffffffffu, loaded) &&
              !(ok = mbar_wait(&full[s], (c / kStages8) & 1, abort_flag, status)))
            break;
          if (!(ok = mbar_wait(&acc_empty[slot], ((c >> 1) & 1) ^ 1u, abort_flag, status))) break;
          __syncwarp();
          tc_fence_after();
          const uint64_t da = sdesc_sw128(smem_u32(smem) + s * kStageBytes8, 1024, 16);
#pragma unroll
          for (int k = 0; k < kK8 / 32; ++k)  // 32 bytes along a row, in the descriptors' units of 16
            mma_f8_ss_pair(leader, tmem + slot * kN8, da + k * 2, da + kABytes8 / 16 + k * 2, idesc,
                           k != 0 ? 1u : 0u);
          mma_commit_pair(leader, &acc_full[slot]);
          mma_commit_pair(leader, &empty[s]);
          loaded = mbar_test(&full[(c + 1) % kStages8], ((c + 1) / kStages8) & 1);
        }
      }
    }
  } else if (warp == kScaleWarp8) {
    // The blocks' scales and, with a tile's first block, the tile's place and bias.  The copies for block
    // c + kAhead8 are issued once block c - 2's sums are complete: the accumulator of block c - 2 was then free, so
    // every output warp is done with block c - 4 and has read what there is of its tile; theirs are the places that
    // are written.
    float* ring = reinterpret_cast<float*>(smem + kRingOff8);
    float* tiles = reinterpret_cast<float*>(smem + kTileOff8);
    uint32_t issued = 0, i_tiles = 0;
    int i_tile = first, i_kb = 0, m0 = 0, n0 = 0;
    const float *a = nullptr, *w = nullptr;
    auto issue = [&]() {
      if (i_tile < n_tiles) {
        if (i_kb == 0) {
          tile8(p, i_tile, m0, n0);
          m0 += rank * kM8;
          a = p.g.a_scales + m0;
          w = p.g.w_scales + n0 / kBlock8;
          const int left = p.g.bias ? p.g.n - n0 : 0;  // without a bias: zeros
          float* dst = tiles + i_tiles++ % kRing8 * kTileFloats8;
          if (lane == 0) *reinterpret_cast<int2*>(dst + kN8) = make_int2(m0, n0);
#pragma unroll
          for (int j = 0; j < kN8 / 32; ++j) {
            const int cc = lane + 32 * j;
            cp_async4(dst + cc, cc < left ? p.g.bias + n0 + cc : p.g.a_scales, cc < left);
          }
        }
        float* dst = ring + issued % kRing8 * kBlockFloats8;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = lane + 32 * j;
          const bool in = m0 + r < p.g.m;
          cp_async4(dst + r, in ? a + r : p.g.a_scales, in);
        }
        if (lane < kParts8) {
          const bool in = n0 + lane * kPart8 < p.g.n;
          cp_async4(dst + kM8 + lane, in ? w + lane : p.g.w_scales, in);
        }
        a += p.g.ldas;
        w += p.g.ldws;
        if (++i_kb == p.kb) {
          i_kb = 0;
          i_tile += step;
        }
        ++issued;
      }
      cp_async_commit();
    };
    for (int i = 0; i < kAhead8; ++i) issue();
    for (uint32_t c = 0; c < issued; ++c) {
      cp_async_wait<kAhead8 - 1>();
      __syncwarp();
      const int slot = c & 1;
      if (c >= 2 && !mbar_wait(&acc_full[slot], ((c - 2) >> 1) & 1, abort_flag, status)) break;
      if (lane == 0) mbar_arrive(&acc_full[slot]);
      issue();
    }
    cp_async_wait<0>();
  } else if (warp < kOutWarps8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsOut8));
    const int quad = warp & 3, part = warp >> 2;
    const uint32_t acc_free = map_to_rank(acc_empty, 0);
    const uint32_t tm = tmem + (static_cast<uint32_t>(quad * 32) << 16) + part * kPart8;
    uint8_t* bufs = smem + kBufOff8 + warp * 2 * kBufBytes8;
    uint32_t* tails = reinterpret_cast<uint32_t*>(smem + kTailOff8) + warp * 64;
    const float* ring = reinterpret_cast<const float*>(smem + kRingOff8);
    const float* tiles = reinterpret_cast<const float*>(smem + kTileOff8);
    constexpr int E = 128 / sizeof(T);    // output columns per buffer
    constexpr int kBlocks = kPart8 / E;   // buffers per tile
    uint32_t c = 0, i_tile = 0;
    const uint32_t leader = elect_one();
    bool ok = true;
    auto wait_sums = [&]() {
      ok = mbar_wait(&acc_full[c & 1], (c >> 1) & 1, abort_flag, status);
      __syncwarp();
      return ok;
    };
    for (int tile = first; tile < n_tiles; tile += step, ++i_tile) {
      if (!wait_sums()) break;
      const float* bias = tiles + i_tile % kRing8 * kTileFloats8;
      const int2 at = *reinterpret_cast<const int2*>(bias + kN8);
      bias += part * kPart8;
      const int m0 = at.x + quad * 32, n0 = at.y + part * kPart8;
      const int cols = p.g.n - n0;  // columns left from this warp's first
      const int rows = p.g.m - m0;  // rows left from this warp's first
      const bool live = cols > 0 && rows > 0;
      // The residual's first two blocks arrive in the output buffers while the sums form; f32 fetches
      // the other two once the first two have left.
      auto fetch_resid = [&](int b) {
        if (b * E < cols)
          load_block(bufs + (b & 1) * kBufBytes8, tails + (b & 1) * 32,
                     static_cast<const T*>(p.g.resid) + static_cast<int64_t>(m0) * p.g.ldr + n0 + b * E, p.g.ldr, rows,
                     cols - b * E, p.resid_vec, lane);
        cp_async_commit();
      };
      if constexpr (O != Out8::Q8) {
        if (live && p.g.resid) {
          if (lane == 0) tma_store_wait_read<0>();
          __syncwarp();
          fetch_resid(0);
          fetch_resid(1);
        }
      }
      float2 acc[kPart8 / 2];
      // The block's latency, not its arithmetic, sets the pace: two 32-column loads are in flight, two waits a
      // block, and the next block's first loads start before this block's last multiplications when its sums
      // are already there.
      uint32_t va[32], vb[32];
      float f = 0.0f;
      auto begin = [&](bool a, bool b) {  // first loads of block c, whose barrier has completed
        if (a) {
          tc_fence_after();
          const float* sp = ring + c % kRing8 * kBlockFloats8;
          f = sp[quad * 32 + lane] * sp[kM8 + part];
          tmem_ld32_converged(tm + (c & 1) * kN8, va);
        }
        if (b) tmem_ld32_converged(tm + (c & 1) * kN8 + 32, vb);
      };
      if (live) {
#pragma unroll  // the totals start from the bias
        for (int i = 0; i < kPart8 / 4; ++i) {
          const float4 v = *reinterpret_cast<const float4*>(bias + 4 * i);
          acc[2 * i] = make_float2(v.x, v.y);
          acc[2 * i + 1] = make_float2(v.z, v.w);
        }
        begin(true, true);
        for (int kb = 0;;) {
          const uint32_t t = tm + (c & 1) * kN8, freed = acc_free + (c & 1) * 8;
          const float f0 = f;
          tmem_ld_wait(va);
          tmem_ld_wait(vb);
          add_scaled<0>(acc, va, f0);
          tmem_ld32_converged(t + 64, va);
          add_scaled<1>(acc, vb, f0);
          tmem_ld32_converged(t + 96, vb);
          ++c;
          const bool more = ++kb < p.kb;
          const bool ready = more && mbar_test(&acc_full[c & 1], (c >> 1) & 1);
          tmem_ld_wait(va);
          tmem_ld_wait(vb);
          tc_fence_before();  // all read: the accumulator is free before the last multiplications
          mbar_arrive_cluster(leader, freed);
          if (__all_sync(0xffffffffu, ready)) {
            add_scaled<2>(acc, va, f0);
            begin(true, false);
            add_scaled<3>(acc, vb, f0);
            begin(false, true);
          } else {
            add_scaled<2>(acc, va, f0);
            add_scaled<3>(acc, vb, f0);
            if (!more || !wait_sums()) break;
            begin(true, true);
          }
        }
      } else {
        for (int kb = 0;;) {
          tc_fence_before();
          mbar_arrive_cluster(leader, acc_free + (c & 1) * 8);
          ++c;
          if (++kb == p.kb || !wait_sums()) break;
        }
      }
      if (!ok) break;
      // ---------------- output ----------------
      if (!live) continue;
      float inv = 0.0f;
      if constexpr (O == Out8::Q8) {
        float top = 0.0f;
        if (cols < kPart8) {
#pragma unroll
          for (int i = 0; i < kPart8 / 2; ++i) {
            if (2 * i >= cols) acc[i].x = 0.0f;
            if (2 * i + 1 >= cols) acc[i].y = 0.0f;
          }
        }
        // A row whose block holds nothing large needs the tail's own fit.  A large value is usually among the first
        // columns; where a row of the warp has none there, all columns are looked at.  No row's bits depend on another.
        float high = -CUDART_INF_F;
#pragma unroll
        for (int i = 0; i < kPart8 / 8; ++i) high = max3(high, acc[i].x, acc[i].y);
        if (__any_sync(0xffffffffu, high < kGelu8Large)) {
          float low = 0.0f;
#pragma unroll
          for (int i = 0; i < kPart8 / 2; ++i) {
            high = max3(high, acc[i].x, acc[i].y);
            low = min3(low, acc[i].x, acc[i].y);
          }
          const bool tail = high < kGelu8Large && low < kGelu8Tail;
          if (__any_sync(0xffffffffu, tail)) {
            const float from = tail ? kGelu8Tail : -CUDART_INF_F;
#pragma unroll
            for (int i = 0; i < kPart8 / 2; ++i) acc[i] = before_gelu8(acc[i], from);
          }
        }
#pragma unroll
        for (int i = 0; i < kPart8 / 2; i += 8) {
          hold<8>(acc + i);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            acc[i + j] = gelu8(acc[i + j]);
            top = max_mag3(top, acc[i + j].x, acc[i + j].y);
          }
          hold<8>(acc + i);
        }
        const Scale8 s = scale8(__float_as_uint(top));
        inv = s.inv;
        if (lane < rows) p.g.scales[static_cast<int64_t>(n0 / kBlock8) * p.g.lds + m0 + lane] = s.s;
      }
      // two buffers at a time: written, published to the TMA stores with one fence, stored
#pragma unroll
      for (int b0 = 0; b0 < kBlocks; b0 += 2) {
        if (b0 * E >= cols) break;
        if (O == Out8::Q8 || !p.g.resid || b0 > 0) {  // the buffers' last stores have read them
          if (lane == 0) tma_store_wait_read<0>();
          __syncwarp();
        }
        if constexpr (O != Out8::Q8) {
          if (p.g.resid) {
            if (b0 > 0) {
              fetch_resid(b0);
              fetch_resid(b0 + 1);
            }
            cp_async_wait<0>();
            __syncwarp();
          }
        }
#pragma unroll
        for (int b = b0; b < (b0 + 2 < kBlocks ? b0 + 2 : kBlocks); ++b) {
          uint8_t* buf = bufs + (b & 1) * kBufBytes8;
#pragma unroll
          for (int v = 0; v < 8; ++v) {
            uint4* at = reinterpret_cast<uint4*>(buf + swz(lane, v * 16));
            uint32_t w[4];
            if constexpr (O == Out8::Q8) {
              const float2 inv2 = make_float2(inv, inv);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float2 x = __fmul2_rn(acc[8 * v + 2 * i], inv2), y = __fmul2_rn(acc[8 * v + 2 * i + 1], inv2);
                w[i] = e4m3x4(x.x, x.y, y.x, y.y);
              }
            } else {
              uint4 r = make_uint4(0u, 0u, 0u, 0u);
              if (p.g.resid) r = *at;
              if constexpr (ODD) {  // the row's halves start in the middle of its first word
                const T* from = static_cast<const T*>(p.g.resid) + static_cast<int64_t>(m0 + lane) * p.g.ldr + n0;
                const uint32_t sh = (reinterpret_cast<uintptr_t>(from) & 2) * 8;
                const uint32_t next = v < 7 ? *reinterpret_cast<const uint32_t*>(buf + swz(lane, v * 16 + 16))
                                            : tails[(b & 1) * 32 + lane];
                r = make_uint4(__funnelshift_r(r.x, r.y, sh), __funnelshift_r(r.y, r.z, sh),
                               __funnelshift_r(r.z, r.w, sh), __funnelshift_r(r.w, next, sh));
              }
              const uint32_t rw[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                if constexpr (O == Out8::F32) {
                  const float2 a = acc[(b * E + v * 4 + i) / 2];
                  const float h = (i & 1) ? a.y : a.x;
                  w[i] = __float_as_uint(p.g.resid ? h + __uint_as_float(rw[i]) : h);
                } else {
                  float2 a = acc[b * E / 2 + v * 4 + i];
                  if (p.g.resid) a = __fadd2_rn(a, unpack2(rw[i], T()));
                  w[i] = pack2(a.x, a.y, T());
                }
              }
            }
            *at = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (p.out_pairs) {
          if (lane == 0) tma_store_3d(&tmOut, bufs, 0, m0, (n0 + b0 * E) / E);
        }
#pragma unroll
        for (int b = b0; b < (b0 + 2 < kBlocks ? b0 + 2 : kBlocks); ++b) {
          const int cb = b * E;
          if (p.out_pairs || cb >= cols) break;
          const uint8_t* buf = bufs + (b & 1) * kBufBytes8;
          if (p.out_tma && (cols - cb >= E || p.out_tail)) {
            if (lane == 0) tma_store_2d(&tmOut, buf, n0 + cb, m0);
          } else {
            T* dst = O == Out8::Q8 ? reinterpret_cast<T*>(p.g.q) : static_cast<T*>(p.g.out);
            const int64_t ld = O == Out8::Q8 ? p.g.ldq : p.g.ldo;
            store_block(buf, dst + static_cast<int64_t>(m0) * ld + n0 + cb, ld, rows, cols - cb, lane);
          }
        }
        if (lane == 0) tma_store_commit();
        __syncwarp();
      }
    }
    cp_async_wait<0>();
    if (lane == 0) tma_store_wait_all();
    __syncwarp();
  }
  tc_fence_before();
  __syncwarp();
  cluster_sync();  // neither CTA goes while the other may still reach its shared memory
  if (warp == kMmaWarp8) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

// Pairs of a kernel that run at one time on the current device.
template <Out8 O, bool ODD>
static int resident_pairs() {
  static std::atomic<int> known[64];
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 1;
  if ((n = known[dev].load(std::memory_order_relaxed)) > 0) return n;
  int sms = 0;
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(sms / 2 * 2);
  cfg.blockDim = dim3(kThreads8);
  cfg.dynamicSmemBytes = kSmem8;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = 2;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  if (cudaOccupancyMaxActiveClusters(&n, gemm8_kernel<O, ODD>, &cfg) != cudaSuccess || n < 1) {
    cudaGetLastError();
    n = sms / 2 > 0 ? sms / 2 : 1;
  }
  known[dev].store(n, std::memory_order_relaxed);
  return n;
}

template <Out8 O, bool ODD = false>
static cudaError_t launch8(const CUtensorMap& ta, const CUtensorMap& tw, const CUtensorMap& to, const Params8& p,
                           int* status, cudaStream_t st) {
  static unsigned long long configured = 0;
  cudaError_t e = once_per_device(configured, [] {
    cudaError_t r = cudaFuncSetAttribute(gemm8_kernel<O, ODD>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem8);
    if (r != cudaSuccess) return r;
    // setmaxnreg.inc waits until the block's launch registers cover the split
    cudaFuncAttributes fa;
    r = cudaFuncGetAttributes(&fa, gemm8_kernel<O, ODD>);
    if (r != cudaSuccess) return r;
    return fa.numRegs >= kLaunchRegs8 ? cudaSuccess : cudaErrorInvalidConfiguration;
  });
  if (e != cudaSuccess) return e;
  const int tiles = p.mt * p.nt;
  const int pairs = resident_pairs<O, ODD>();
  count_launch();
  gemm8_kernel<O, ODD><<<2 * (tiles < pairs ? tiles : pairs), kThreads8, kSmem8, st>>>(ta, tw, to, p, status);
  return cudaGetLastError();
}

static cudaError_t gemm8_tiled(const Gemm8& g, int* status, cudaStream_t st) {
  CUtensorMap ta, tw, to;
  Params8 p;
  p.g = g;
  p.mt = (g.m + 2 * kM8 - 1) / (2 * kM8);
  p.nt = (g.n + kN8 - 1) / kN8;
  p.per = make_fastdiv(static_cast<uint32_t>(kGroup8 * p.nt), static_cast<uint64_t>(p.mt) * p.nt);
  p.kb = (g.k + kK8 - 1) / kK8;
  cudaError_t e = make_map_2d(&ta, g.a, g.k, g.m, g.lda, kK8, kM8, MapElem::U8);
  if (e == cudaSuccess) e = make_map_2d(&tw, g.w, g.k, g.n, g.ldw, kK8, kN8 / 2, MapElem::U8);
  if (e != cudaSuccess) return e;
  const int size = !g.out ? 1 : g.out_type == Elem::F32 ? 4 : 2;
  const void* dst = g.out ? g.out : g.q;
  const int64_t ld = (g.out ? g.ldo : g.ldq) * size;
  p.out_tma = reinterpret_cast<uintptr_t>(dst) % 16 == 0 && ld % 16 == 0;
  p.out_tail = (static_cast<int64_t>(g.n) * size) % 16 == 0;
  p.resid_vec = reinterpret_cast<uintptr_t>(g.resid) % 16 == 0 && (g.ldr * size) % 16 == 0;
  const MapElem me = size == 1   ? MapElem::U8
                     : size == 4 ? MapElem::F32
                                 : g.out_type == Elem::F16 ? MapElem::F16 : MapElem::BF16;
  to = ta;
  const int per_block = 128 / size;
  p.out_pairs = p.out_tma && size > 1 && g.n % per_block == 0;
  if (p.out_pairs)
    e = make_map_3d(&to, dst, per_block, g.m, g.n / per_block, ld, 128, per_block, 32, 2, me);
  else if (p.out_tma)
    e = make_map_2d(&to, dst, g.n, g.m, ld, per_block, 32, me);
  if (e != cudaSuccess) return e;
  const bool odd = g.resid && size == 2 && (reinterpret_cast<uintptr_t>(g.resid) % 4 != 0 || g.ldr % 2 != 0);
  if (!g.out) return launch8<Out8::Q8>(ta, tw, to, p, status, st);
  switch (g.out_type) {
    case Elem::F32: return launch8<Out8::F32>(ta, tw, to, p, status, st);
    case Elem::F16:
      return odd ? launch8<Out8::F16, true>(ta, tw, to, p, status, st) : launch8<Out8::F16>(ta, tw, to, p, status, st);
    case Elem::BF16:
      return odd ? launch8<Out8::BF16, true>(ta, tw, to, p, status, st)
                 : launch8<Out8::BF16>(ta, tw, to, p, status, st);
  }
  return cudaErrorInvalidValue;
}

static cudaError_t gemm8_few(const Gemm8& g, int* status, cudaStream_t st) {
  FewParams p;
  p.g = g;
  p.kb = (g.k + 127) / 128;
  p.kind = g.out ? static_cast<int>(g.out_type) : 3;
  const size_t size = !g.out ? 1 : g.out_type == Elem::F32 ? 4 : 2;
  auto fours = [&](const void* ptr, int64_t ld, size_t sz) {  // 4 values at once from any multiple of 4 columns
    return reinterpret_cast<uintptr_t>(ptr) % (4 * sz) == 0 && ld % 4 == 0;
  };
  p.vec = fours(g.out ? g.out : g.q, g.out ? g.ldo : g.ldq, size) && (!g.resid || fours(g.resid, g.ldr, size)) &&
          (!g.bias || fours(g.bias, 0, 4));
  const int nt = g.m <= 16 ? 16 : g.m <= 32 ? 32 : 64;
  const int64_t tiles = static_cast<int64_t>((g.n + 127) / 128) * ((g.m + nt - 1) / nt);
  // as many CTAs per tile as two per SM allow, each with a K-block at least
  p.lg = 0;
  while ((1 << p.lg) < kFewMaxSplit && (tiles << (p.lg + 1)) <= 2 * kSms && (2 << p.lg) <= p.kb) ++p.lg;
  p.split = 1 << p.lg;
  return nt == 16 ? launch_few<16>(p, status, st)
                  : nt == 32 ? launch_few<32>(p, status, st) : launch_few<64>(p, status, st);
}

// Few rows of A, or so few 128 x 64 tiles that each SM has at most one, go to the kernel that splits K; measured
// (bf16 out): 62 x 1536 x 256 5.1 us (tiled 6.3), 256 x 4096 x 4096 15.7 (18.4), 512 x 2048 x 2048 10.7 (12.2),
// against 512 x 4096 x 4096 24.5 (18.9), 1024 x 2048 x 2048 15.4 (12.7), 2294 x 1536 x 256 10.2 (7.1).
cudaError_t gemm8(const Gemm8& g, int* status, cudaStream_t st) {
  const int64_t tiles = static_cast<int64_t>((g.m + 63) / 64) * ((g.n + 127) / 128);
  return g.m <= 64 || tiles <= kSms ? gemm8_few(g, status, st) : gemm8_tiled(g, status, st);
}

}  // namespace lbrr
