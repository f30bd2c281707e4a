// The 8-bit product for few rows (gemm8.cu): the operands change places.
//
// With few rows of A the weights' bytes are the cost, and 256 x 256 tiles leave
// most SMs without work.  Here W's rows are the MMA's 128 rows and NT rows of A
// its columns, so a tile holds 128 outputs n of NT rows m; K is split over a
// cluster of up to eight CTAs, so that a single row against a square weight
// still occupies the whole GPU.  Per CTA: one warp loads W and A tiles by TMA (a
// ring that holds the whole K range of a short split at once), another warp
// issues four tcgen05.mma per 128-column block into one of four accumulators,
// and four or eight warps (one output n per thread, NT or NT / 2 rows m) scale
// each block's sums and add them to totals in registers; each keeps its own copy
// of the scales, fetched asynchronously four to eight blocks ahead.  At the end
// every CTA leaves its totals in its shared memory as [m][128]; the cluster's
// CTAs share out the rows m, and one bulk copy per CTA pair brings each row's
// totals to its CTA, where a warp sums them in rank order (the same bits every
// time) and writes the row, 128 neighbouring outputs at once; the row's block
// maximum for an 8-bit output is then one warp reduction.  Everything here runs
// once or a few times, so latency is all there is: no step waits for another
// that it does not need, and the code is kept short, because its first execution
// waits for instruction fetches.
//
// Measured: 1 x 4096 x 4096 6.0 us (2.8 TB/s of weights; the tiled kernel 16.8),
// 1 x 32768 x 4096 23 us (5.8 TB/s), 62 x 1536 x 256 5.2 us and 62 x 1024 x 256
// with GELU to 8 bits 6.0 us, of which a launch is about 2.5.  Remote loads of
// the totals by the rows' warps took 1 us longer at 62 rows, remote stores 5 us.
#pragma once
#include "cp_async.cuh"
#include "gelu8.cuh"
#include "quant8.cuh"
#include "ring.h"

namespace lbrr {

constexpr int kFewSlots = 4;
constexpr int kFewWBytes = 128 * 128;
constexpr int kFewScaleBlocks = 8, kFewScaleAhead = 4;  // K-blocks whose scales a warp holds, and fetches at a time
constexpr int kFewMaxSplit = 8;

template <int NT>
struct FewLayout {
  static constexpr int kParts = NT < 32 ? 1 : 2;  // output warps per TMEM lane quadrant
  static constexpr int kCols = NT / kParts;       // rows m of an output warp
  static constexpr int kOutWarps = 4 * kParts, kLoadWarp = kOutWarps, kMmaWarp = kOutWarps + 1;
  static constexpr int kWarps = kOutWarps + 2, kThreads = kWarps * 32;
  static constexpr int kStages = NT < 64 ? 4 : 3;
  static constexpr int kStageBytes = kFewWBytes + NT * 128;
  static constexpr int kRecvOff = kStages * kStageBytes;  // [split][NT / split][128], from the cluster's CTAs
  static constexpr int kScaleFloats = kFewScaleBlocks * (kCols + 1);  // a warp's: [block][kCols], then W's
  static constexpr int kScaleOff = kRecvOff + NT * 128 * 4;
  static constexpr int kBarOff = kScaleOff + kOutWarps * kScaleFloats * 4;
  static constexpr int kSmem = kBarOff + 256;
  static constexpr uint32_t kTmemCols = kFewSlots * NT;
  static_assert(NT * 128 * 4 <= kStages * kStageBytes, "the totals reuse the ring");
  static_assert(kSmem <= 113 * 1024, "two CTAs per SM");
  // a block of the tiled kernel (200 KB, all 512 TMEM columns) must not fit beside one of these
  static_assert(kSmem >= 40 * 1024, "see above");
};

struct FewParams {
  Gemm8 g;
  int kb;         // K-blocks
  int split, lg;  // CTAs per cluster, a power of two, and its logarithm
  int kind;   // output: 0 f32, 1 f16, 2 bf16, 3 8-bit with GELU
  bool vec;   // output and residual rows, and bias, allow accesses of 4 values
};

// Shared memory of this CTA to that of another of the cluster (cluster addresses), completing on a barrier there.
__device__ __forceinline__ void bulk_to_cta(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
      "r"(smem_u32(src)), "r"(bytes), "r"(bar)
      : "memory");
}
// Not for data: that the other CTAs run, and later that they have what they need of this one.
__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }

template <class T>
__device__ __forceinline__ void few_add4(const T* p, bool vec, int left, float (&h)[4]) {
  if (vec && left >= 4) {
    if constexpr (sizeof(T) == 4) {
      const float4 v = *reinterpret_cast<const float4*>(p);
      h[0] += v.x, h[1] += v.y, h[2] += v.z, h[3] += v.w;
    } else {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      const float2 a = unpack2(v.x, T()), b = unpack2(v.y, T());
      h[0] += a.x, h[1] += a.y, h[2] += b.x, h[3] += b.y;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < left) h[i] += to_f32(p[i]);
}
template <class T>
__device__ __forceinline__ void few_store4(T* p, bool vec, int left, const float (&h)[4]) {
  if (vec && left >= 4) {
    if constexpr (sizeof(T) == 4)
      *reinterpret_cast<float4*>(p) = make_float4(h[0], h[1], h[2], h[3]);
    else
      *reinterpret_cast<uint2*>(p) = make_uint2(pack2(h[0], h[1], T()), pack2(h[2], h[3], T()));
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < left) p[i] = from_f32<T>(h[i]);
}
// The rows r = warp, warp + WARPS, .. of this CTA: sum over the CTAs, bias, and the residual and output's type
// (T), or GELU and 8-bit codes (T = uint8_t).  in: [split][share][128].
template <class T, int WARPS>
__device__ __forceinline__ void few_rows(const FewParams& p, const float* in, int share, int rows, int64_t m0, int n0,
                                         int warp, int lane, const float (&bias)[4]) {
  const int n = n0 + lane * 4, left = p.g.n - n;
  const bool vec = p.vec;
#pragma unroll 1
  for (int r = warp; r < rows; r += WARPS) {
    const float* t = in + r * 128 + lane * 4;
    float4 v[kFewMaxSplit];
#pragma unroll
    for (int s = 0; s < kFewMaxSplit; ++s)
      if (s < p.split) v[s] = *reinterpret_cast<const float4*>(t + s * share * 128);
    float h[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
#pragma unroll
    for (int s = 1; s < kFewMaxSplit; ++s)
      if (s < p.split) h[0] += v[s].x, h[1] += v[s].y, h[2] += v[s].z, h[3] += v[s].w;
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] += bias[i];
    const int64_t m = m0 + r;
    if constexpr (sizeof(T) == 1) {
      if (__any_sync(0xffffffffu, fminf(min3(h[0], h[1], h[2]), h[3]) < kGelu8Tail)) {
        const float2 a = before_gelu8(make_float2(h[0], h[1]), kGelu8Tail);
        const float2 b = before_gelu8(make_float2(h[2], h[3]), kGelu8Tail);
        h[0] = a.x, h[1] = a.y, h[2] = b.x, h[3] = b.y;
      }
      const float2 a = gelu8(make_float2(h[0], h[1])), b = gelu8(make_float2(h[2], h[3]));
      uint32_t top = 0;
      if (0 < left) top = max(top, mag_bits(a.x));
      if (1 < left) top = max(top, mag_bits(a.y));
      if (2 < left) top = max(top, mag_bits(b.x));
      if (3 < left) top = max(top, mag_bits(b.y));
      const Scale8 s = scale8(__reduce_max_sync(0xffffffffu, top));
      const uint32_t q = e4m3x4(a.x * s.inv, a.y * s.inv, b.x * s.inv, b.y * s.inv);
      uint8_t* dst = p.g.q + m * p.g.ldq + n;
      if (vec && left >= 4) {
        *reinterpret_cast<uint32_t*>(dst) = q;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i < left) dst[i] = static_cast<uint8_t>(q >> (8 * i));
      }
      if (lane == 0) p.g.scales[static_cast<int64_t>(n0 / kBlock8) * p.g.lds + m] = s.s;
    } else if (left > 0) {
      if (p.g.resid) few_add4(static_cast<const T*>(p.g.resid) + m * p.g.ldr + n, vec, left, h);
      few_store4(static_cast<T*>(p.g.out) + m * p.g.ldo + n, vec, left, h);
    }
  }
}

template <int NT>
__global__ void __launch_bounds__(FewLayout<NT>::kThreads, 2)
    gemm8_few_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmA,
                     const __grid_constant__ FewParams p, int* status) {
  using L = FewLayout<NT>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kBarOff);
  uint64_t* empty = full + L::kStages;
  uint64_t* acc_full = empty + L::kStages;
  uint64_t* acc_empty = acc_full + kFewSlots;
  uint64_t* recv_full = acc_empty + kFewSlots;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(recv_full + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  if ((smem_u32(smem) & 1023u) != 0) {  // the same in every CTA: nothing allocated yet
    if (threadIdx.x == 0) report_status(status, kDevSmemMisaligned);
    return;
  }
  const int nb = blockIdx.x >> p.lg, n0 = nb * 128, m0 = blockIdx.y * NT;
  const int kb0 = static_cast<int>((p.kb * rank) >> p.lg);
  const int blocks = static_cast<int>((p.kb * (rank + 1)) >> p.lg) - kb0;
  auto load = [&](int c) {
    const int s = c % L::kStages;
    uint8_t* sw = smem + s * L::kStageBytes;
    mbar_arrive_expect_tx(&full[s], L::kStageBytes);
    tma_load_2d(sw, &tmW, &full[s], (kb0 + c) * 128, n0);
    tma_load_2d(sw + kFewWBytes, &tmA, &full[s], (kb0 + c) * 128, m0);
  };
  const int ahead = min(blocks, L::kStages);
  if (warp == L::kLoadWarp) {
    if (lane == 0) {
      for (int s = 0; s < L::kStages; ++s) {
        mbar_init(&full[s], 1);
        mbar_init(&empty[s], 1);
      }
      for (int s = 0; s < kFewSlots; ++s) {
        mbar_init(&acc_full[s], 1);
        mbar_init(&acc_empty[s], L::kOutWarps);
      }
      mbar_init(recv_full, 1);
      *abort_flag = 0;
      fence_barrier_init();
      mbar_arrive_expect_tx(recv_full, NT * 128 * 4);
    }
    __syncwarp();
    asm volatile("bar.arrive 1, %0;" ::"n"(L::kThreads) : "memory");  // the barriers exist; no wait for the others
    if (lane == 0)
      for (int c = 0; c < ahead; ++c) load(c);
    __syncwarp();
  }
  if (warp == L::kMmaWarp) {
    tmem_alloc(tmem_slot, L::kTmemCols);
    tmem_relinquish();
  }
  float bias4[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // of the four outputs that this lane writes at the end
  if (p.g.bias && n0 + lane * 4 < p.g.n) few_add4(p.g.bias + n0 + lane * 4, p.vec, p.g.n - n0 - lane * 4, bias4);
  constexpr int C = L::kCols;
  const int quad = warp & 3, col0 = (warp >> 2) * C;  // of an output warp
  float2 acc[C / 2];
#pragma unroll
  for (int i = 0; i < C / 2; ++i) acc[i] = make_float2(0.0f, 0.0f);
  float* scales = reinterpret_cast<float*>(smem + L::kScaleOff) + warp * L::kScaleFloats;
  auto fetch_scales = [&](int c) {  // of blocks c .. c + kFewScaleAhead - 1
#pragma unroll 1
    for (int i = c; i < min(c + kFewScaleAhead, blocks); ++i) {
      const int at = i % kFewScaleBlocks;
      const bool in = m0 + col0 + lane < p.g.m;
      if (lane < C) cp_async4(scales + at * C + lane, p.g.a_scales + (in ? (kb0 + i) * p.g.ldas + m0 + col0 + lane : 0), in);
      if (lane == 0) cp_async4(scales + kFewScaleBlocks * C + at, p.g.w_scales + (kb0 + i) * p.g.ldws + nb, true);
    }
    cp_async_commit();
  };
  if (warp < L::kOutWarps) fetch_scales(0);
  tc_fence_before();
  if (warp != L::kLoadWarp) asm volatile("bar.sync 1, %0;" ::"n"(L::kThreads) : "memory");
  cluster_arrive();  // waited for before the first copy into another CTA
  tc_fence_after();

  if (warp == L::kLoadWarp) {
    if (lane == 0) {
      int c = ahead;
      bool ok = true;
      for (; c < blocks; ++c) {
        if (!(ok = mbar_wait(&empty[c % L::kStages], ((c / L::kStages) & 1) ^ 1u, abort_flag, status))) break;
        load(c);
      }
      // the commits that free the stages have arrived before the block may go
      ok = ok && drain_ring<L::kStages>(blocks, [&](int s, uint32_t parity) {
             return mbar_wait(&empty[s], parity, abort_flag, status);
           });
      if (!ok) {  // the copies in flight land before the block's shared memory goes
        for (int i = c > L::kStages ? c - L::kStages : 0; i < c; ++i) {
          int none = 0;
          mbar_wait(&full[i % L::kStages], (i / L::kStages) & 1, &none, nullptr);
        }
      }
    }
  } else if (warp == L::kMmaWarp) {
    const uint32_t leader = elect_one(), tmem = *tmem_slot;
    constexpr uint32_t idesc = idesc_e4m3_f32(128, NT);
    for (int c = 0; c < blocks; ++c) {
      const int s = c % L::kStages, slot = c % kFewSlots;
      if (!mbar_wait(&full[s], (c / L::kStages) & 1, abort_flag, status)) break;
      if (!mbar_wait(&acc_empty[slot], ((c / kFewSlots) & 1) ^ 1u, abort_flag, status)) break;
      __syncwarp();
      tc_fence_after();
      const uint64_t dw = sdesc_sw128(smem_u32(smem) + s * L::kStageBytes, 1024, 16);
#pragma unroll
      for (int k = 0; k < 4; ++k)  // 32 bytes along a row, in the descriptors' units of 16
        mma_f8_ss(leader, tmem + slot * NT, dw + k * 2, dw + kFewWBytes / 16 + k * 2, idesc, k != 0 ? 1u : 0u);
      mma_commit_leader(leader, &acc_full[slot]);
      mma_commit_leader(leader, &empty[s]);
    }
  } else {
    const uint32_t tm = *tmem_slot + (static_cast<uint32_t>(quad * 32) << 16) + col0;
#pragma unroll 1
    for (int c = 0; c < blocks; ++c) {
      if (c % kFewScaleAhead == 0) {
        __syncwarp();  // the places of the blocks fetched now have been read
        fetch_scales(c + kFewScaleAhead);
        cp_async_wait<1>();
        __syncwarp();
      }
      const int slot = c % kFewSlots;
      if (!mbar_wait(&acc_full[slot], (c / kFewSlots) & 1, abort_flag, status)) break;
      __syncwarp();
      tc_fence_after();
      const float* f = scales + c % kFewScaleBlocks * C;
      const float ws = scales[kFewScaleBlocks * C + c % kFewScaleBlocks];
      const float2 w = make_float2(ws, ws);
      uint32_t v[C];
      if constexpr (C == 16) {
        tmem_ld16_converged(tm + slot * NT, v);
        tmem_ld_wait16(v);
      } else {
        tmem_ld32_converged(tm + slot * NT, v);
        tmem_ld_wait(v);
      }
#pragma unroll
      for (int i = 0; i < C / 4; ++i) {
        const float4 s = *reinterpret_cast<const float4*>(f + 4 * i);
        acc[2 * i] = __ffma2_rn(make_float2(__uint_as_float(v[4 * i]), __uint_as_float(v[4 * i + 1])),
                                __fmul2_rn(make_float2(s.x, s.y), w), acc[2 * i]);
        acc[2 * i + 1] = __ffma2_rn(make_float2(__uint_as_float(v[4 * i + 2]), __uint_as_float(v[4 * i + 3])),
                                    __fmul2_rn(make_float2(s.z, s.w), w), acc[2 * i + 1]);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[slot]);
    }
  }
  // every MMA is complete (the last block's sums have been read) or the block gave up
  float* totals = reinterpret_cast<float*>(smem);  // [NT][128]
  const int share = NT >> p.lg;  // rows of a CTA
  if (warp < L::kOutWarps) {
#pragma unroll
    for (int i = 0; i < C / 2; ++i) {
      totals[(col0 + 2 * i) * 128 + quad * 32 + lane] = acc[i].x;
      totals[(col0 + 2 * i + 1) * 128 + quad * 32 + lane] = acc[i].y;
    }
    cp_async_wait<0>();
  }
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  int in_off = 0;
  __syncwarp();
  cluster_wait();  // every CTA of the cluster runs and has its barrier
  if (p.split > 1) {
    in_off = L::kRecvOff;
    if (warp == L::kLoadWarp && lane < p.split)
      bulk_to_cta(map_to_rank(smem + L::kRecvOff + rank * share * 512, lane), totals + lane * share * 128, share * 512,
                  map_to_rank(recv_full, lane));
    __syncwarp();
    if (warp == L::kMmaWarp) {
      tc_fence_after();
      tmem_dealloc(*tmem_slot, L::kTmemCols);
    }
    mbar_wait(recv_full, 0, abort_flag, status);
    __syncwarp();
  } else if (warp == L::kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(*tmem_slot, L::kTmemCols);
  }
  cluster_arrive();
  const float* in = reinterpret_cast<const float*>(smem + in_off);
  const int row0 = rank * share, rows = min(share, p.g.m - m0 - row0);
  const int64_t m = m0 + row0;
  if (p.kind == 0)
    few_rows<float, L::kWarps>(p, in, share, rows, m, n0, warp, lane, bias4);
  else if (p.kind == 1)
    few_rows<__half, L::kWarps>(p, in, share, rows, m, n0, warp, lane, bias4);
  else if (p.kind == 2)
    few_rows<__nv_bfloat16, L::kWarps>(p, in, share, rows, m, n0, warp, lane, bias4);
  else
    few_rows<uint8_t, L::kWarps>(p, in, share, rows, m, n0, warp, lane, bias4);
  __syncwarp();
  cluster_wait();  // every CTA has its rows: this one's totals may go
}

template <int NT>
inline cudaError_t launch_few(const FewParams& p, int* status, cudaStream_t st) {
  using L = FewLayout<NT>;
  static unsigned long long configured = 0;
  cudaError_t e = once_per_device(configured, [] {
    return cudaFuncSetAttribute(gemm8_few_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmem);
  });
  CUtensorMap tw, ta;
  if (e == cudaSuccess) e = make_map_2d(&tw, p.g.w, p.g.k, p.g.n, p.g.ldw, 128, 128, MapElem::U8);
  if (e == cudaSuccess) e = make_map_2d(&ta, p.g.a, p.g.k, p.g.m, p.g.lda, 128, NT, MapElem::U8);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((p.g.n + 127) / 128 * p.split, (p.g.m + NT - 1) / NT);
  cfg.blockDim = dim3(L::kThreads);
  cfg.dynamicSmemBytes = L::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = p.split;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  count_launch();
  e = cudaLaunchKernelEx(&cfg, gemm8_few_kernel<NT>, tw, ta, p, status);
  return e == cudaSuccess ? cudaGetLastError() : e;
}

}  // namespace lbrr
