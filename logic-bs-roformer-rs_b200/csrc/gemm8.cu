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
// One persistent CTA per SM walks 128 x 256 tiles.  A K-block of 128 is four
// tcgen05.mma (kind::f8f6f4, 128 x 256 x 32) into one of two 256-column
// accumulators, so the tensor core works on block b + 1 while eight warps
// (two per TMEM lane quadrant, one accumulator row per thread, 128 of the 256
// columns each) read block b, scale it and add it to 128 totals per thread.
// A 128-column part is one scale block of W, so the factor of a block is one
// number per thread.  After the last block the same warps write the tile
// through shared memory and TMA stores while the tensor core runs ahead into
// the next tile.  Warps: 0..7 totals and output, 8 TMA loads, 9 TMEM
// allocation and MMA issue, 10 and 11 idle (they complete the warpgroup that
// gives its registers away).
#include "gelu.cuh"
#include "quant8.cuh"

namespace lbrr {

constexpr int kM8 = 128, kN8 = 256, kK8 = 128;
constexpr int kStages8 = 3;
constexpr int kA8Bytes = kM8 * kK8, kB8Bytes = kN8 * kK8;  // 16 KB, 32 KB
constexpr int kStage8Bytes = kA8Bytes + kB8Bytes;
constexpr int kOutWarps8 = 8;
constexpr int kPart8 = kN8 / 2;                             // columns per output warp
constexpr int kBuf8Words = 1024;                            // 32 rows x 128 bytes; two per output warp
constexpr int kBuf8Off = kStages8 * kStage8Bytes;
constexpr int kBias8Off = kBuf8Off + kOutWarps8 * 2 * kBuf8Words * 4;
constexpr int kBar8Off = kBias8Off + kOutWarps8 * kPart8 * 4;
constexpr int kSmem8 = kBar8Off + 256;
constexpr int kThreads8 = kOutWarps8 * 32 + 128;
constexpr int kLoadWarp8 = kOutWarps8, kMmaWarp8 = kOutWarps8 + 1;
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
  int mt, nt, group;  // row tiles, column tiles, row tiles per group
  int kb;             // K-blocks
  bool out_tma;       // the output's rows allow TMA stores
  bool out_tail;      // ... of a last, partial block too: a TMA store ends on a 16-byte boundary, not on the
                      // matrix's last column (measured: it wrote the rest of the 16 bytes)
  bool resid_vec;     // the residual's rows allow 16-byte loads
};

// Tiles in groups of `group` row tiles, rows fastest: the CTAs running at one
// time share both their A rows and their W rows in L2.
__device__ __forceinline__ void tile8(const Params8& p, int idx, int& m0, int& n0) {
  const int per = p.group * p.nt, gi = idx / per, rem = idx - gi * per;
  const int rows = min(p.group, p.mt - gi * p.group);
  const int n = rem / rows;
  m0 = (gi * p.group + rem - n * rows) * kM8;
  n0 = n * kN8;
}

__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// Byte o of row r in a buffer of 32 rows of 128 bytes with the TMA 128-byte swizzle.
__device__ __forceinline__ uint32_t swz(int r, int o) {
  return static_cast<uint32_t>(r * 128 + ((((o >> 4) ^ (r & 7)) << 4) | (o & 15)));
}

// One 32-row block of 128 bytes per row between global memory and a buffer,
// coalesced; rows and columns outside the matrix are left alone.
template <class T>
__device__ __forceinline__ void load_block(uint8_t* buf, const T* src, int64_t ld, int rows, int cols, bool vec,
                                           int lane) {
  constexpr int E = 128 / sizeof(T);
  if (vec && cols >= E) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = i * 4 + lane / 8, v = lane % 8;
      if (r < rows) cp_async16(buf + swz(r, v * 16), src + r * ld + v * (16 / static_cast<int>(sizeof(T))));
    }
    return;
  }
  for (int r = 0; r < min(rows, 32); ++r)
    for (int c = lane; c < min(cols, E); c += 32)
      *reinterpret_cast<T*>(buf + swz(r, c * static_cast<int>(sizeof(T)))) = src[r * ld + c];
}
template <class T>
__device__ __forceinline__ void store_block(const uint8_t* buf, T* dst, int64_t ld, int rows, int cols, int lane) {
  constexpr int E = 128 / sizeof(T);
  for (int r = 0; r < min(rows, 32); ++r)
    for (int c = lane; c < min(cols, E); c += 32)
      dst[r * ld + c] = *reinterpret_cast<const T*>(buf + swz(r, c * static_cast<int>(sizeof(T))));
}

__device__ __forceinline__ float4 lds4f(const float* p) { return *reinterpret_cast<const float4*>(p); }

// The scales of the K-blocks to come, two ahead of their use and across tiles.
struct ScaleStream {
  int tile, kb, m, nb;
  bool more;
  __device__ __forceinline__ void at_tile(const Params8& p, int n_tiles, int row, int part) {
    more = tile < n_tiles;
    if (!more) return;
    int m0, n0;
    tile8(p, tile, m0, n0);
    m = m0 + row;
    nb = n0 / kBlock8 + part;
  }
  // The block's two scales, multiplied where they are used: the loads are not waited for here.
  __device__ __forceinline__ float2 next(const Params8& p, int n_tiles, int row, int part) {
    float2 s = make_float2(0.0f, 0.0f);
    if (!more) return s;
    if (m < p.g.m) s.x = __ldg(p.g.a_scales + kb * p.g.ldas + m);
    if (nb * kBlock8 < p.g.n) s.y = __ldg(p.g.w_scales + kb * p.g.ldws + nb);
    if (++kb == p.kb) {
      kb = 0;
      tile += gridDim.x;
      at_tile(p, n_tiles, row, part);
    }
    return s;
  }
};

template <Out8 O>
__global__ void __launch_bounds__(kThreads8, 1)
    gemm8_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmW,
                 const __grid_constant__ CUtensorMap tmOut, const __grid_constant__ Params8 p, int* status) {
  extern __shared__ __align__(1024) uint8_t smem[];
  using T = typename OutType<O>::T;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kBar8Off);
  uint64_t* empty = full + kStages8;
  uint64_t* acc_full = empty + kStages8;  // [2]
  uint64_t* acc_empty = acc_full + 2;     // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  if ((smem_u32(smem) & 1023u) != 0) {
    if (threadIdx.x == 0) report_status(status, kDevSmemMisaligned);
    return;
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages8; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&acc_full[s], 1);
      mbar_init(&acc_empty[s], kOutWarps8);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == kLoadWarp8 && lane == 0) {
    tma_prefetch(&tmA);
    tma_prefetch(&tmW);
  }
  if (warp == kMmaWarp8) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int n_tiles = p.mt * p.nt;
  // the launcher checks the compiled register count before the first launch
  if (warp >= kOutWarps8) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther8));

  if (warp == kLoadWarp8) {
    if (lane == 0) {
      uint32_t c = 0;
      bool ok = true;
      for (int tile = blockIdx.x; ok && tile < n_tiles; tile += gridDim.x) {
        int m0, n0;
        tile8(p, tile, m0, n0);
        for (int kb = 0; kb < p.kb; ++kb, ++c) {
          const int s = c % kStages8;
          if (!(ok = mbar_wait(&empty[s], ((c / kStages8) & 1) ^ 1u, abort_flag, status))) break;
          uint8_t* sa = smem + s * kStage8Bytes;
          mbar_arrive_expect_tx(&full[s], kStage8Bytes);
          tma_load_2d(sa, &tmA, &full[s], kb * kK8, m0);
          tma_load_2d(sa + kA8Bytes, &tmW, &full[s], kb * kK8, n0);
        }
      }
      if (!ok) {  // the copies in flight land before the block's shared memory goes
        const uint32_t first = c > kStages8 ? c - kStages8 : 0;
        for (uint32_t i = first; i < c; ++i) {
          int none = 0;
          mbar_wait(&full[i % kStages8], (i / kStages8) & 1, &none, nullptr);
        }
      }
    }
  } else if (warp == kMmaWarp8) {
    if (lane == 0) {
      uint32_t c = 0;
      bool ok = true;
      for (int tile = blockIdx.x; ok && tile < n_tiles; tile += gridDim.x) {
        int m0, n0;
        tile8(p, tile, m0, n0);
        const uint32_t idesc = idesc_e4m3_f32(kM8, min(kN8, (p.g.n - n0 + 15) & ~15));
        for (int kb = 0; kb < p.kb; ++kb, ++c) {
          const int s = c % kStages8, slot = c & 1;
          if (!(ok = mbar_wait(&acc_empty[slot], ((c >> 1) & 1) ^ 1u, abort_flag, status))) break;
          if (!(ok = mbar_wait(&full[s], (c / kStages8) & 1, abort_flag, status))) break;
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + s * kStage8Bytes), sb = sa + kA8Bytes;
#pragma unroll
          for (int k = 0; k < kK8 / 32; ++k)
            mma_f8_ss(tmem + slot * kN8, sdesc_sw128(sa + k * 32, 1024, 16), sdesc_sw128(sb + k * 32, 1024, 16),
                      idesc, k != 0 ? 1u : 0u);
          mma_commit(&empty[s]);
          mma_commit(&acc_full[slot]);
        }
      }
    }
  } else if (warp < kOutWarps8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsOut8));
    const int quad = warp & 3, part = warp >> 2;
    const int row = quad * 32 + lane;
    const uint32_t tm = tmem + (static_cast<uint32_t>(quad * 32) << 16) + part * kPart8;
    uint8_t* bufs = smem + kBuf8Off + warp * 2 * kBuf8Words * 4;
    float* bias = reinterpret_cast<float*>(smem + kBias8Off) + warp * kPart8;
    constexpr int E = 128 / sizeof(T);  // output columns per buffer
    int phase = 0;
    ScaleStream ss;
    ss.tile = blockIdx.x;
    ss.kb = 0;
    ss.at_tile(p, n_tiles, row, part);
    float2 s0 = ss.next(p, n_tiles, row, part), s1 = ss.next(p, n_tiles, row, part);
    uint32_t c = 0;
    bool ok = true;
    for (int tile = blockIdx.x; tile < n_tiles; tile += gridDim.x) {
      int m0, n0;
      tile8(p, tile, m0, n0);
      n0 += part * kPart8;
      const int cols = p.g.n - n0;              // columns left from this warp's first
      const int rows = p.g.m - (m0 + quad * 32);  // rows left from this warp's first
      const bool live = cols > 0;
      float2 acc[kPart8 / 2];
#pragma unroll
      for (int i = 0; i < kPart8 / 2; ++i) acc[i] = make_float2(0.0f, 0.0f);
      for (int kb = 0; kb < p.kb; ++kb, ++c) {
        const int slot = c & 1;
        const float2 cur = s0;
        s0 = s1;
        s1 = ss.next(p, n_tiles, row, part);
        if (!(ok = mbar_wait(&acc_full[slot], (c >> 1) & 1, abort_flag, status))) break;
        tc_fence_after();
        if (live) {
          const uint32_t t = tm + slot * kN8;
          const float2 f = make_float2(cur.x * cur.y, cur.x * cur.y);
          uint32_t va[32], vb[32];
          tmem_ld32(t, va);
          tmem_ld_wait(va);
#pragma unroll
          for (int b = 0; b < kPart8 / 32; b += 2) {
            tmem_ld32(t + 32 * (b + 1), vb);
#pragma unroll
            for (int i = 0; i < 16; ++i)
              acc[16 * b + i] = __ffma2_rn(make_float2(__uint_as_float(va[2 * i]), __uint_as_float(va[2 * i + 1])), f,
                                           acc[16 * b + i]);
            tmem_ld_wait(vb);
            if (b + 2 < kPart8 / 32) tmem_ld32(t + 32 * (b + 2), va);
#pragma unroll
            for (int i = 0; i < 16; ++i)
              acc[16 * (b + 1) + i] = __ffma2_rn(
                  make_float2(__uint_as_float(vb[2 * i]), __uint_as_float(vb[2 * i + 1])), f, acc[16 * (b + 1) + i]);
            if (b + 2 < kPart8 / 32) tmem_ld_wait(va);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&acc_empty[slot]);
      }
      if (!ok) break;
      if (!live || rows <= 0) continue;
      // ---------------- output ----------------
      if (p.g.bias) {
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int cc = lane + 32 * i;
          bias[cc] = cc < cols ? __ldg(p.g.bias + n0 + cc) : 0.0f;
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kPart8 / 4; ++i) {
          const float4 v = lds4f(bias + 4 * i);
          acc[2 * i] = __fadd2_rn(acc[2 * i], make_float2(v.x, v.y));
          acc[2 * i + 1] = __fadd2_rn(acc[2 * i + 1], make_float2(v.z, v.w));
        }
      }
      float inv = 0.0f;
      if constexpr (O == Out8::Q8) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < kPart8 / 2; ++i) {
          acc[i] = gelu_as2(acc[i]);
          if (2 * i < cols) top = max(top, mag_bits(acc[i].x));
          if (2 * i + 1 < cols) top = max(top, mag_bits(acc[i].y));
        }
        const Scale8 s = scale8(top);
        inv = s.inv;
        if (lane < rows) p.g.scales[static_cast<int64_t>(n0 / kBlock8) * p.g.lds + m0 + row] = s.s;
      }
#pragma unroll
      for (int b = 0; b < kPart8 / E; ++b) {
        const int cb = b * E;
        if (cb >= cols) break;
        uint8_t* buf = bufs + (phase++ & 1) * kBuf8Words * 4;
        if (lane == 0) tma_store_wait_read<1>();
        __syncwarp();
        uint32_t w[32];
        if constexpr (O == Out8::Q8) {
#pragma unroll
          for (int i = 0; i < 32; ++i)
            w[i] = e4m3x4(acc[2 * i].x * inv, acc[2 * i].y * inv, acc[2 * i + 1].x * inv, acc[2 * i + 1].y * inv);
        } else {
          if (p.g.resid) {
            load_block(buf, static_cast<const T*>(p.g.resid) + static_cast<int64_t>(m0 + quad * 32) * p.g.ldr + n0 + cb,
                       p.g.ldr, rows, cols - cb, p.resid_vec, lane);
            cp_async_wait_all();
            __syncwarp();
          }
#pragma unroll
          for (int v = 0; v < 8; ++v) {
            uint4 r = make_uint4(0u, 0u, 0u, 0u);
            if (p.g.resid) r = *reinterpret_cast<const uint4*>(buf + swz(lane, v * 16));
            const uint32_t rw[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if constexpr (O == Out8::F32) {
                const float2 a = acc[(cb + v * 4 + i) / 2];
                const float h = (i & 1) ? a.y : a.x;
                w[v * 4 + i] = __float_as_uint(p.g.resid ? h + __uint_as_float(rw[i]) : h);
              } else {
                float2 a = acc[cb / 2 + v * 4 + i];
                if (p.g.resid) a = __fadd2_rn(a, unpack2(rw[i], T()));
                w[v * 4 + i] = pack2(a.x, a.y, T());
              }
            }
          }
          __syncwarp();
        }
#pragma unroll
        for (int v = 0; v < 8; ++v)
          *reinterpret_cast<uint4*>(buf + swz(lane, v * 16)) =
              make_uint4(w[4 * v], w[4 * v + 1], w[4 * v + 2], w[4 * v + 3]);
        if (p.out_tma && (cols - cb >= E || p.out_tail)) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&tmOut, buf, n0 + cb, m0 + quad * 32);
            tma_store_commit();
          }
        } else {
          __syncwarp();
          T* dst = O == Out8::Q8 ? reinterpret_cast<T*>(p.g.q) : static_cast<T*>(p.g.out);
          const int64_t ld = O == Out8::Q8 ? p.g.ldq : p.g.ldo;
          store_block(buf, dst + static_cast<int64_t>(m0 + quad * 32) * ld + n0 + cb, ld, rows, cols - cb, lane);
        }
      }
    }
    if (lane == 0) tma_store_wait_all();
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp8) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

static int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return 148;
  return n;
}

template <Out8 O>
static cudaError_t launch8(const CUtensorMap& ta, const CUtensorMap& tw, const CUtensorMap& to, const Params8& p,
                           int* status, cudaStream_t st) {
  static unsigned long long configured = 0;
  cudaError_t e = once_per_device(configured, [] {
    cudaError_t r = cudaFuncSetAttribute(gemm8_kernel<O>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem8);
    if (r != cudaSuccess) return r;
    // setmaxnreg.inc waits until the block's launch registers cover the split
    cudaFuncAttributes fa;
    r = cudaFuncGetAttributes(&fa, gemm8_kernel<O>);
    if (r != cudaSuccess) return r;
    return fa.numRegs >= kLaunchRegs8 ? cudaSuccess : cudaErrorInvalidConfiguration;
  });
  if (e != cudaSuccess) return e;
  const int tiles = p.mt * p.nt, sms = sm_count();
  count_launch();
  gemm8_kernel<O><<<tiles < sms ? tiles : sms, kThreads8, kSmem8, st>>>(ta, tw, to, p, status);
  return cudaGetLastError();
}

cudaError_t gemm8(const Gemm8& g, int* status, cudaStream_t st) {
  CUtensorMap ta, tw, to;
  Params8 p;
  p.g = g;
  p.mt = (g.m + kM8 - 1) / kM8;
  p.nt = (g.n + kN8 - 1) / kN8;
  p.group = 8;
  p.kb = (g.k + kK8 - 1) / kK8;
  cudaError_t e = make_map_2d(&ta, g.a, g.k, g.m, g.lda, kK8, kM8, MapElem::U8);
  if (e == cudaSuccess) e = make_map_2d(&tw, g.w, g.k, g.n, g.ldw, kK8, kN8, MapElem::U8);
  if (e != cudaSuccess) return e;
  const int size = !g.out ? 1 : g.out_type == Elem::F32 ? 4 : 2;
  const void* dst = g.out ? g.out : g.q;
  const int64_t ld = (g.out ? g.ldo : g.ldq) * size;
  p.out_tma = reinterpret_cast<uintptr_t>(dst) % 16 == 0 && ld % 16 == 0;
  p.out_tail = (static_cast<int64_t>(g.n) * size) % 16 == 0;
  p.resid_vec = reinterpret_cast<uintptr_t>(g.resid) % 16 == 0 && (g.ldr * size) % 16 == 0;
  const MapElem me = size == 1 ? MapElem::U8 : size == 4 ? MapElem::F32 : g.out_type == Elem::F16 ? MapElem::F16 : MapElem::BF16;
  to = ta;
  if (p.out_tma) e = make_map_2d(&to, dst, g.n, g.m, ld, 128 / size, 32, me);
  if (e != cudaSuccess) return e;
  if (!g.out) return launch8<Out8::Q8>(ta, tw, to, p, status, st);
  switch (g.out_type) {
    case Elem::F32: return launch8<Out8::F32>(ta, tw, to, p, status, st);
    case Elem::F16: return launch8<Out8::F16>(ta, tw, to, p, status, st);
    case Elem::BF16: return launch8<Out8::BF16>(ta, tw, to, p, status, st);
  }
  return cudaErrorInvalidValue;
}

}  // namespace lbrr
