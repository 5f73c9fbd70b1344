// Block-scaled 8-bit product for sm_100a:
//
//   y[m, n] = sum_b a_scale[m, b] w_scale[n / 128, b] sum_{k in block b} a[m, k] w[n, k]
//
// a and w e4m3, one block = 128 columns = one 128-byte swizzled row of a
// shared-memory operand tile.  The tensor cores (tcgen05, kind::f8f6f4) form
// each block's inner sum into TMEM from zero; warps read it back, multiply by
// the block's scales and add into fp32 registers, so no partial sum of
// differently scaled blocks is ever mixed and the running sum is plain fp32.
// Every output has one fixed summation order: the same bits on every call.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>
#include <cstdint>
#include <type_traits>

#include "llvq_b200.h"
#include "llvq_internal.h"
#include "tcgen05.cuh"

namespace llvq {

PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder();  // gemm.cu

namespace {

constexpr uint32_t kWaitLimit = 1u << 22;

__device__ __forceinline__ void store_out(void* y, int64_t i, float v, int type) {
  if (type == LLVQ_DT_F32) static_cast<float*>(y)[i] = v;
  else if (type == LLVQ_DT_F16) static_cast<__half*>(y)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(y)[i] = __float2bfloat16_rn(v);
}

// ---------------------------------------------------------------- few rows
// Weights are the 128-row side of the MMA (TMEM lane = weight row), the
// activation rows its N side (kAct columns), so few rows waste little and the
// weights stream through once.  The K blocks of a tile are split over the
// CTAs of a cluster, which add their partial sums through distributed shared
// memory in rank order.
//
// Roles: warp 0 loads both operands with TMA, warp 1 issues the MMAs, warps
// 2..5 add up.  TMEM holds kBufs block sums so the MMAs run ahead of the
// additions.  The scales of a block (kAct row scales and the tile's weight
// scale) travel through a ring of kRing slots filled with cp.async.
constexpr int kFewThreads = 192;
constexpr int kTileRows = 128;
constexpr int kRing = 8;

template <int kAct>
struct Few {
  static constexpr int kStageBytes = kTileRows * 128 + kAct * 128;
  // two CTAs per SM: at least 76 KB each, so that a third, which could run out of TMEM, never fits
  static constexpr int kStages = (100 * 1024) / kStageBytes;
  static constexpr int kTmemCols = kAct <= 16 ? 128 : 256;
  static constexpr int kBufs = kTmemCols / kAct > 8 ? 8 : kTmemCols / kAct;
  static constexpr int kRingFloats = kAct + 4;  // row scales, then the weight scale
  static constexpr int kRingOff = kStages * kStageBytes;
  static constexpr int kBarOff = kRingOff + kRing * kRingFloats * 4;
  static constexpr int kBars = 2 * kStages + 2 * kBufs + 1;
  static constexpr size_t kSmem = (size_t)kBarOff + 8 * kBars + 16 + 1024;
  static_assert(kStages >= 3 && kAct * kTileRows * 4 <= kRingOff && kRingOff % 16 == 0 && kBarOff % 8 == 0);
  static_assert(kSmem > 76 * 1024 && kSmem <= 113 * 1024);
};

template <int kAct>
__global__ void __launch_bounds__(kFewThreads, 2)
    few_rows_kernel(const __grid_constant__ CUtensorMap tw, const __grid_constant__ CUtensorMap ta, int blocks,
                    const float* __restrict__ as, int64_t as_row, int64_t as_col, const float* __restrict__ ws,
                    int64_t ws_row, int64_t ws_col, int m_total, int n_total, void* __restrict__ y, int64_t ldy,
                    int y_type, int splits, int* error_flag) {
  using F = Few<kAct>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(base + F::kBarOff);
  uint32_t* holder = reinterpret_cast<uint32_t*>(bars + F::kBars);
  float* ring = reinterpret_cast<float*>(base + F::kRingOff);
  const uint32_t sbase = tc::smem_addr(base);
  auto full = [&](int st) { return tc::smem_addr(&bars[st]); };
  auto empty = [&](int st) { return tc::smem_addr(&bars[F::kStages + st]); };
  auto acc_full = [&](int b) { return tc::smem_addr(&bars[2 * F::kStages + b]); };
  auto acc_empty = [&](int b) { return tc::smem_addr(&bars[2 * F::kStages + F::kBufs + b]); };
  const uint32_t drain = tc::smem_addr(&bars[F::kBars - 1]);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = (int)(blockIdx.x % (unsigned)splits), tile = (int)(blockIdx.x / (unsigned)splits);
  const int n0 = tile * kTileRows, m0 = (int)blockIdx.y * kAct;
  const int b_begin = (int)((int64_t)blocks * rank / splits), b_end = (int)((int64_t)blocks * (rank + 1) / splits);
  const int count = b_end - b_begin;
  if (tid == 0) {
    for (int i = 0; i < F::kStages; ++i) {
      tc::mbar_init(full(i), 1);
      tc::mbar_init(empty(i), 1);
    }
    for (int i = 0; i < F::kBufs; ++i) {
      tc::mbar_init(acc_full(i), 1);
      tc::mbar_init(acc_empty(i), 4);  // one arrival per adding warp
    }
    tc::mbar_init(drain, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) tc::tmem_alloc(tc::smem_addr(holder), F::kTmemCols);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = *holder;
  bool failed = false;
  float acc[kAct];

  if (warp == 0) {
    if (lane == 0) {  // TMA producer
      int i = 0;
      for (; i < count; ++i) {
        const int st = i % F::kStages, use = i / F::kStages;
        if (use > 0 && !tc::mbar_wait(empty(st), (use - 1) & 1, kWaitLimit)) {
          failed = true;
          break;
        }
        const uint32_t dst = sbase + st * F::kStageBytes;
        tc::mbar_arrive_expect_tx(full(st), F::kStageBytes);
        tc::tma_load_2d(dst, &tw, (b_begin + i) * kFp8Block, n0, full(st));
        tc::tma_load_2d(dst + kTileRows * 128, &ta, (b_begin + i) * kFp8Block, m0, full(st));
      }
      // no copy may still be in flight when the block exits: wait for the last use of every stage
      for (int u = i > F::kStages ? i - F::kStages : 0; u < i; ++u)
        tc::mbar_wait(full(u % F::kStages), (u / F::kStages) & 1, kWaitLimit);
    }
  } else if (warp == 1) {
    if (lane == 0) {  // MMA issuer
      constexpr uint32_t idesc = tc::idesc_e4m3_f32(kTileRows, kAct);
      for (int i = 0; i < count; ++i) {
        const int st = i % F::kStages, buf = i % F::kBufs, use = i / F::kBufs;
        if ((use > 0 && !tc::mbar_wait(acc_empty(buf), (use - 1) & 1, kWaitLimit)) ||
            !tc::mbar_wait(full(st), (i / F::kStages) & 1, kWaitLimit)) {
          failed = true;
          break;
        }
        tc::fence_after_sync();
        const uint32_t sw = sbase + st * F::kStageBytes, sa = sw + kTileRows * 128;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
          tc::mma_f8(tmem + buf * kAct, tc::desc_sw128(sw + ks * 32), tc::desc_sw128(sa + ks * 32), idesc, ks > 0);
        tc::commit(empty(st));
        tc::commit(acc_full(buf));
      }
      // every MMA issued has finished before TMEM is freed
      tc::commit(drain);
      tc::mbar_wait(drain, 0, kWaitLimit);
    }
  } else {  // warps 2..5 read TMEM lane quarters 2, 3, 0, 1
    const int t = tid - 64;
    const uint32_t t0 = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    // scales of block i into slot i % kRing: thread t brings row scale t, thread 0 the weight scale too
    auto fetch = [&](int i) {
      if (i < count) {
        float* slot = ring + (i % kRing) * F::kRingFloats;
        const int64_t b = b_begin + i;
        if (t < kAct) {
          const bool live = m0 + t < m_total;
          tc::cp_async4(tc::smem_addr(slot + t), as + (live ? (m0 + t) * as_row + b * as_col : 0), live);
        }
        if (t == 0) tc::cp_async4(tc::smem_addr(slot + kAct), ws + tile * ws_row + b * ws_col, true);
      }
      tc::cp_async_commit();
    };
#pragma unroll
    for (int j = 0; j < kAct; ++j) acc[j] = 0.f;
    for (int i = 0; i < kRing - 1; ++i) fetch(i);
    for (int i = 0; i < count; ++i) {
      const int buf = i % F::kBufs;
      tc::cp_async_wait<kRing - 2>();
      asm volatile("bar.sync 1, 128;" ::: "memory");  // slot i is whole, and nobody reads slot i - 1 any more
      fetch(i + kRing - 1);
      if (!failed && !tc::mbar_wait(acc_full(buf), (i / F::kBufs) & 1, kWaitLimit)) failed = true;
      tc::fence_after_sync();
      const float* slot = ring + (i % kRing) * F::kRingFloats;
      const float wsc = slot[kAct];
#pragma unroll
      for (int c = 0; c < kAct; c += 16) {
        float v[16];
        tc::tmem_ld16(t0 + buf * kAct + c, v);
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[c + j] = fmaf(v[j] * wsc, slot[c + j], acc[c + j]);
      }
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(acc_empty(buf));
    }
    const int n = n0 + (warp & 3) * 32 + lane;
    if (splits == 1) {
#pragma unroll
      for (int j = 0; j < kAct; ++j)
        if (n < n_total && m0 + j < m_total) store_out(y, (int64_t)(m0 + j) * ldy + n, acc[j], y_type);
    } else {
      // the last block's sums have been read, so every stage has been consumed: reuse them
      float* red = reinterpret_cast<float*>(base);
#pragma unroll
      for (int j = 0; j < kAct; ++j) red[j * kTileRows + (warp & 3) * 32 + lane] = acc[j];
    }
  }
  __syncwarp();
  if (failed && error_flag) atomicExch(error_flag, 1);
  if (splits > 1) {
    tc::cluster_sync();
    if (warp >= 2) {  // CTA `rank` adds activation rows rank, rank + splits, ...
      const int t = tid - 64, n = n0 + t;
      for (int j = rank; j < kAct && m0 + j < m_total; j += splits) {
        const uint32_t at = sbase + (uint32_t)(j * kTileRows + t) * 4;
        float sum = 0.f;
        for (int r = 0; r < splits; ++r) sum += tc::ld_cluster(tc::map_rank(at, r));
        if (n < n_total) store_out(y, (int64_t)(m0 + j) * ldy + n, sum, y_type);
      }
    }
    __syncwarp();
    tc::cluster_sync();  // no CTA leaves while another still reads its sums
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  if (warp == 0) tc::tmem_dealloc(tmem, F::kTmemCols);
}

// ---------------------------------------------------------------- many rows
// Two CTAs of a cluster share a tile of 256 activation rows x kTileN weight
// rows (tcgen05 cta_group::2, M = 256): each loads 128 activation rows and
// half of the weight rows, so a CTA reads 16 + kTileN / 16 KB per block for
// 128 x kTileN outputs, two thirds of what a CTA alone would at 256.  TMEM lane = activation row,
// so a lane's scale for a block is one number, a_scale[row] w_scale, and the
// addition is one packed fused multiply-add per two outputs.
//
// Roles: warps 0..15 add up (lane quarter warp % 4, column quarter warp / 4),
// warp 16 loads with TMA, warp 17 of the leading CTA issues the MMAs of both,
// warps 18 and 19 bring the scales, kScaleGroup blocks at a time and two
// groups in flight.  Adding is a chain of waits (block sum ready, TMEM load, hand
// back), so it takes four warps per scheduler to keep up with the tensor
// cores: with two, of twice the columns, a block took 1300 cycles for the 512
// of its MMAs.  TMEM holds kBufs block sums of kTileN columns.  The leader's
// full[] takes the bytes of both CTAs' loads; empty[] and acc_full[] are
// committed in both CTAs; the leader's acc_empty[] takes the arrivals of all 32
// adding warps.
constexpr int kAddWarps = 16;
constexpr int kPairThreads = kAddWarps * 32 + 128;
// 640 threads launch with 96 registers each: 61,440 = 512 x 112 + 128 x 32
constexpr int kAddRegs = 112, kOtherRegs = 32;
constexpr int kPairRows = 256;
constexpr int kScaleGroup = 8;
constexpr int kScaleBlock = 2 * 128 * 8;  // bytes of a block's scales: 2 column halves x 128 rows x (pre, factor)

template <int kTileN>
struct Pair {
  static constexpr int kStageA = 128 * 128, kStageB = kTileN / 2 * 128;
  static constexpr int kStageBytes = kStageA + kStageB;
  static constexpr int kStages = 128 * 1024 / kStageBytes;
  static constexpr int kBufs = 512 / kTileN;
  static constexpr int kCols = kTileN / (kAddWarps / 4);  // columns of an adding warp
  static constexpr int kStoreOff = kStages * kStageBytes;      // 4 KB per adding warp
  static constexpr int kScaleOff = kStoreOff + kAddWarps * 4096;
  static constexpr int kBarOff = kScaleOff + 2 * kScaleGroup * kScaleBlock;
  static constexpr int kBars = 2 * kStages + 2 * kBufs + 5;
  static constexpr size_t kSmem = (size_t)kBarOff + 8 * kBars + 16 + 1024;
  static_assert(kSmem <= 227 * 1024);
};

__device__ __forceinline__ uint64_t pack2(uint32_t lo, uint32_t hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
  return r;
}

__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

__device__ __forceinline__ void unpack2(uint64_t v, float& lo, float& hi) {
  uint32_t a, b;
  asm("mov.b64 {%0, %1}, %2;" : "=r"(a), "=r"(b) : "l"(v));
  lo = __uint_as_float(a);
  hi = __uint_as_float(b);
}

// The scale of a block's sums as (pre, factor): (1, as * ws), or where that
// product comes near the ends of the range of fp32 (or is not finite) (ws, as),
// applied one after the other.
__device__ __forceinline__ float2 split_scale(float as, float ws) {
  const float f = as * ws;
  return fabsf(f) >= 0x1p-60f && fabsf(f) <= 0x1p60f ? make_float2(1.f, f) : make_float2(ws, as);
}

// acc + v * pre * factor; by the lane, so that no row depends on another.
template <int kCount>
__device__ __forceinline__ void add_scaled(uint64_t* acc, uint32_t* v, float pre, float factor) {
  if (pre != 1.f) {
#pragma unroll
    for (int j = 0; j < kCount; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) * pre);
  }
  const uint64_t ff = pack2(__float_as_uint(factor), __float_as_uint(factor));
#pragma unroll
  for (int j = 0; j < kCount / 2; ++j) acc[j] = fma2(pack2(v[2 * j], v[2 * j + 1]), ff, acc[j]);
}

// A warp's 32 rows x kCols columns to y, through its 4 KB of shared memory (32
// rows of 128 bytes, 16-byte chunks swizzled by the row) so that the global
// stores are whole 128-byte lines.
template <typename T, int kCols>
__device__ __forceinline__ void store_rows(const uint64_t* acc, uint8_t* buf, T* __restrict__ y, int64_t ldy, int row0,
                                           int col0, int m_total, int n_total, int lane) {
  constexpr int kPerLine = 128 / (int)sizeof(T), kPerChunk = 16 / (int)sizeof(T);
  const bool whole = ldy * (int64_t)sizeof(T) % 16 == 0 && reinterpret_cast<uintptr_t>(y) % 16 == 0;
#pragma unroll
  for (int c0 = 0; c0 < kCols; c0 += kPerLine) {
#pragma unroll
    for (int ch = 0; ch < 8; ++ch) {
      alignas(16) T e[kPerChunk];
#pragma unroll
      for (int j = 0; j < kPerChunk; j += 2) {
        float lo, hi;
        unpack2(acc[(c0 + ch * kPerChunk + j) / 2], lo, hi);
        if constexpr (sizeof(T) == 4) {
          e[j] = lo;
          e[j + 1] = hi;
        } else if constexpr (std::is_same_v<T, __half>) {
          e[j] = __float2half_rn(lo);
          e[j + 1] = __float2half_rn(hi);
        } else {
          e[j] = __float2bfloat16_rn(lo);
          e[j + 1] = __float2bfloat16_rn(hi);
        }
      }
      *reinterpret_cast<uint4*>(buf + lane * 128 + ((ch ^ (lane & 7)) * 16)) = *reinterpret_cast<const uint4*>(e);
    }
    __syncwarp();
#pragma unroll
    for (int it = 0; it < 8; ++it) {
      const int r = it * 4 + (lane >> 3), ch = lane & 7;
      const int row = row0 + r, col = col0 + c0 + ch * kPerChunk;
      const uint4 v = *reinterpret_cast<const uint4*>(buf + r * 128 + ((ch ^ (r & 7)) * 16));
      if (row < m_total && col < n_total) {
        T* dst = y + (int64_t)row * ldy + col;
        if (whole && col + kPerChunk <= n_total) {
          *reinterpret_cast<uint4*>(dst) = v;
        } else {
          const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
          for (int j = 0; j < kPerChunk; ++j)
            if (col + j < n_total) dst[j] = e[j];
        }
      }
    }
    __syncwarp();
  }
}

// Tile `t` of tm x tn: groups of 16 tile rows, column by column within a
// group, so that the tiles in flight share operands in L2.
__device__ __forceinline__ void tile_at(int t, int tm, int tn, int& mt, int& nt) {
  const int group = t / (16 * tn), in = t - group * 16 * tn;
  const int height = min(16, tm - group * 16);
  mt = group * 16 + in % height;
  nt = in / height;
}

template <int kTileN>
__global__ void __launch_bounds__(kPairThreads, 1)
    pair_kernel(const __grid_constant__ CUtensorMap ta, const __grid_constant__ CUtensorMap tw, int blocks,
                const float* __restrict__ as, int64_t as_row, int64_t as_col, const float* __restrict__ ws,
                int64_t ws_row, int64_t ws_col, int m_total, int n_total, void* __restrict__ y, int64_t ldy, int y_type,
                int tm, int tn, int* error_flag) {
  using P = Pair<kTileN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(base + P::kBarOff);
  uint32_t* holder = reinterpret_cast<uint32_t*>(bars + P::kBars);
  const uint32_t sbase = tc::smem_addr(base);
  auto full = [&](int st) { return tc::smem_addr(&bars[st]); };
  auto empty = [&](int st) { return tc::smem_addr(&bars[P::kStages + st]); };
  auto acc_full = [&](int b) { return tc::smem_addr(&bars[2 * P::kStages + b]); };
  auto acc_empty = [&](int b) { return tc::smem_addr(&bars[2 * P::kStages + P::kBufs + b]); };
  auto scale_full = [&](int i) { return tc::smem_addr(&bars[2 * P::kStages + 2 * P::kBufs + i]); };
  auto scale_empty = [&](int i) { return tc::smem_addr(&bars[2 * P::kStages + 2 * P::kBufs + 2 + i]); };
  const uint32_t drain = tc::smem_addr(&bars[P::kBars - 1]);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = (int)tc::cluster_rank(), pair = (int)blockIdx.x >> 1, pairs = (int)gridDim.x >> 1;
  const int tiles = tm * tn;
  if (tid == 0) {
    for (int i = 0; i < P::kStages; ++i) {
      tc::mbar_init(full(i), 1);
      tc::mbar_init(empty(i), 1);
    }
    for (int i = 0; i < P::kBufs; ++i) {
      tc::mbar_init(acc_full(i), 1);
      tc::mbar_init(acc_empty(i), 2 * kAddWarps);
    }
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(scale_full(i), 2);
      tc::mbar_init(scale_empty(i), kAddWarps);
    }
    tc::mbar_init(drain, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncwarp();
  if (warp == kAddWarps) tc::tmem_alloc_pair(tc::smem_addr(holder), 512);
  tc::fence_before_sync();
  tc::cluster_sync();
  tc::fence_after_sync();
  const uint32_t tmem = *holder;
  bool failed = false;

  if (warp >= kAddWarps) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == kAddWarps && lane == 0) {  // TMA producer of this CTA's halves
      uint32_t g = 0;
      for (int t = pair; t < tiles && !failed; t += pairs) {
        int mt, nt;
        tile_at(t, tm, tn, mt, nt);
        const int m0 = mt * kPairRows + rank * 128, n0 = nt * kTileN + rank * (kTileN / 2);
        for (int b = 0; b < blocks; ++b, ++g) {
          const int st = (int)(g % P::kStages);
          const uint32_t use = g / P::kStages;
          if (use > 0 && !tc::mbar_wait(empty(st), (use - 1) & 1u, kWaitLimit)) {
            failed = true;
            break;
          }
          const uint32_t dst = sbase + st * P::kStageBytes, bar = tc::map_rank(full(st), 0);
          if (rank == 0) tc::mbar_arrive_expect_tx(full(st), 2 * P::kStageBytes);
          tc::tma_load_2d_pair(dst, &ta, b * kFp8Block, m0, bar);
          tc::tma_load_2d_pair(dst + P::kStageA, &tw, b * kFp8Block, n0, bar);
        }
      }
      // every stage loaded has been consumed before the CTA may exit
      for (uint32_t u = g > (uint32_t)P::kStages ? g - P::kStages : 0u; u < g; ++u)
        if (!tc::mbar_wait(empty((int)(u % P::kStages)), (u / P::kStages) & 1u, kWaitLimit)) failed = true;
    }
    if (warp == kAddWarps + 1 && rank == 0) {  // MMA issuer of the pair: the warp waits, one thread issues
      constexpr uint32_t idesc = tc::idesc_e4m3_f32(kPairRows, kTileN);
      const bool issuer = tc::elect_one();
      const uint64_t desc0 = tc::desc_sw128(sbase);
      uint32_t st = 0, st_use = 0, buf = 0, buf_use = 0;
      for (int t = pair; t < tiles && !failed; t += pairs) {
        for (int b = 0; b < blocks; ++b) {
          // even lanes poll for the operands, odd ones for the TMEM columns: one latency instead of two
          const uint32_t bar = (lane & 1) ? acc_empty(buf) : full(st);
          const uint32_t parity = (lane & 1) ? (buf_use - 1) & 1u : st_use & 1u;
          const bool ready = ((lane & 1) && buf_use == 0) || tc::mbar_wait(bar, parity, kWaitLimit);
          if (!__all_sync(0xffffffffu, ready)) {
            failed = true;
            break;
          }
          tc::fence_after_sync();
          if (issuer) {
            const uint64_t da = desc0 + st * (P::kStageBytes >> 4), dw = da + (P::kStageA >> 4);
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) tc::mma_f8_pair(tmem + buf * kTileN, da + 2 * ks, dw + 2 * ks, idesc, ks > 0);
            tc::commit_pair(acc_full(buf));
            tc::commit_pair(empty(st));
          }
          __syncwarp();
          if (++st == P::kStages) st = 0, ++st_use;
          if (++buf == P::kBufs) buf = 0, ++buf_use;
        }
      }
      // every MMA issued has finished before TMEM is freed
      if (issuer) tc::commit_pair(drain);
      __syncwarp();
      tc::mbar_wait(drain, 0, kWaitLimit);
    }
    if (warp >= kAddWarps + 2) {  // scales: thread i brings those of rows i and i + 64 for both column halves
      const int i = tid - (kAddWarps + 2) * 32;
      uint32_t gg = 0;
      for (int t = pair; t < tiles && !failed; t += pairs) {
        int mt, nt;
        tile_at(t, tm, tn, mt, nt);
        const int row0 = mt * kPairRows + rank * 128 + i, block0 = nt * kTileN / kFp8Block;
        const int block1 = block0 + (kTileN > kFp8Block && nt * kTileN + kFp8Block < n_total ? 1 : 0);
        const bool live0 = row0 < m_total, live1 = row0 + 64 < m_total;
        const float *pa0 = as + (live0 ? row0 * as_row : 0), *pa1 = as + (live1 ? (row0 + 64) * as_row : 0);
        const float *pw0 = ws + block0 * ws_row, *pw1 = ws + block1 * ws_row;
        for (int b0 = 0; b0 < blocks; b0 += kScaleGroup, ++gg) {
          if (gg > 1 && !tc::mbar_wait(scale_empty(gg & 1), ((gg >> 1) - 1) & 1u, kWaitLimit)) {
            failed = true;
            break;
          }
          float2* dst = reinterpret_cast<float2*>(base + P::kScaleOff + (gg & 1) * kScaleGroup * kScaleBlock);
#pragma unroll 1
          for (int q = 0; q < kScaleGroup; q += 2) {  // two blocks at a time: this warpgroup has few registers
            float a0[2], a1[2], w0[2], w1[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const int b = min(b0 + q + u, blocks - 1);
              a0[u] = live0 ? pa0[b * as_col] : 0.f;
              a1[u] = live1 ? pa1[b * as_col] : 0.f;
              w0[u] = pw0[b * ws_col];
              w1[u] = pw1[b * ws_col];
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              float2* d = dst + (q + u) * 256 + i;
              d[0] = split_scale(a0[u], w0[u]);
              d[64] = split_scale(a1[u], w0[u]);
              d[128] = split_scale(a0[u], w1[u]);
              d[192] = split_scale(a1[u], w1[u]);
            }
          }
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(scale_full(gg & 1));
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kAddRegs));
    const int strip = warp >> 2, quarter = warp & 3;
    const uint32_t t0 = tmem + ((uint32_t)(quarter * 32) << 16) + strip * P::kCols;
    uint8_t* buf4k = base + P::kStoreOff + warp * 4096;
    const uint32_t scales = sbase + P::kScaleOff + (strip * P::kCols / kFp8Block) * 1024 + (quarter * 32 + lane) * 8;
    uint32_t release[P::kBufs];
#pragma unroll
    for (int i = 0; i < P::kBufs; ++i) release[i] = tc::map_rank(acc_empty(i), 0);
    uint32_t g = 0, gg = 0;
    for (int t = pair; t < tiles && !failed; t += pairs) {
      int mt, nt;
      tile_at(t, tm, tn, mt, nt);
      const int row0 = mt * kPairRows + rank * 128 + quarter * 32, col0 = nt * kTileN + strip * P::kCols;
      uint64_t acc[P::kCols / 2];
#pragma unroll
      for (int j = 0; j < P::kCols / 2; ++j) acc[j] = 0;
      for (int b0 = 0; b0 < blocks; b0 += kScaleGroup, ++gg) {
        if (!failed && !tc::mbar_wait(scale_full(gg & 1), (gg >> 1) & 1u, kWaitLimit)) failed = true;
        uint32_t slot = scales + (gg & 1) * kScaleGroup * kScaleBlock;
        const int last = min(blocks - b0, kScaleGroup);
#pragma unroll 1
        for (int u = 0; u < last; ++u, ++g, slot += kScaleBlock) {
          const uint32_t buf = g % P::kBufs;
          if (!failed && !tc::mbar_wait(acc_full(buf), (g / P::kBufs) & 1u, kWaitLimit)) failed = true;
          tc::fence_after_sync();
          float pre, f;
#pragma unroll
          for (int c = 0; c < P::kCols; c += 32) {
            uint32_t v[32];
            tc::tmem_ld32(t0 + buf * kTileN + c, v);
            if (c == 0) tc::ld_shared2(slot, pre, f);
            tc::tmem_wait_ld();
            if (c + 32 == P::kCols) {
              tc::fence_before_sync();
              __syncwarp();
              if (lane == 0) tc::mbar_arrive_cluster(P::kBufs == 2 ? release[buf & 1] : tc::map_rank(acc_empty(buf), 0));
            }
            add_scaled<32>(acc + c / 2, v, pre, f);
          }
        }
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(scale_empty(gg & 1));
      }
      if (y_type == LLVQ_DT_F32)
        store_rows<float, P::kCols>(acc, buf4k, static_cast<float*>(y), ldy, row0, col0, m_total, n_total, lane);
      else if (y_type == LLVQ_DT_F16)
        store_rows<__half, P::kCols>(acc, buf4k, static_cast<__half*>(y), ldy, row0, col0, m_total, n_total, lane);
      else
        store_rows<__nv_bfloat16, P::kCols>(acc, buf4k, static_cast<__nv_bfloat16*>(y), ldy, row0, col0, m_total,
                                            n_total, lane);
    }
  }
  __syncwarp();
  if (failed && error_flag) atomicExch(error_flag, 1);
  tc::fence_before_sync();
  tc::cluster_sync();  // no arrival or commit is under way to a CTA that has left
  tc::fence_after_sync();
  if (warp == kAddWarps) tc::tmem_dealloc_pair(tmem, 512);
}

// e4m3 row-major [rows, cols] (row stride `ld` bytes), box 128 columns x
// box_rows rows, 128-byte swizzle, zero fill outside the matrix.
cudaError_t encode_e4m3_map(CUtensorMap* map, const void* ptr, int64_t cols, int64_t rows, int64_t ld, int box_rows) {
  const auto enc = tensor_map_encoder();
  if (!enc) return cudaErrorNotSupported;
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)ld};
  const cuuint32_t box[2] = {kFp8Block, (cuuint32_t)box_rows};
  const cuuint32_t elem[2] = {1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, elem,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

// Sets a kernel's dynamic shared memory limit once per device (idempotent if raced).
cudaError_t configure_once(const void* kernel, size_t smem, std::atomic<bool>* done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
  if (done[dev].load(std::memory_order_acquire)) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e == cudaSuccess) done[dev].store(true, std::memory_order_release);
  return e;
}

template <int kAct>
cudaError_t few_rows_launch(const Fp8Operand& a, const Fp8Operand& w, int m, int n, int k, void* y, int64_t ldy,
                            int y_type, int* error_flag, int sms, cudaStream_t stream) {
  static std::atomic<bool> done[kMaxDevices];
  cudaError_t e = configure_once((const void*)few_rows_kernel<kAct>, Few<kAct>::kSmem, done);
  if (e != cudaSuccess) return e;
  CUtensorMap tw, ta;
  e = encode_e4m3_map(&tw, w.q, k, n, w.ld, kTileRows);
  if (e != cudaSuccess) return e;
  e = encode_e4m3_map(&ta, a.q, k, m, a.ld, kAct);
  if (e != cudaSuccess) return e;
  const int blocks = (k + kFp8Block - 1) / kFp8Block;
  const int64_t tn = (n + kTileRows - 1) / kTileRows, tm = (m + kAct - 1) / kAct;
  if (tm > 65535) return cudaErrorInvalidValue;
  // as many CTAs per tile as fit two per SM, at most a portable cluster of 8
  const int splits = (int)std::max<int64_t>(1, std::min<int64_t>({2 * sms / (tn * tm), 8, blocks}));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tn * splits), (unsigned)tm, 1);
  cfg.blockDim = dim3(kFewThreads, 1, 1);
  cfg.dynamicSmemBytes = Few<kAct>::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)splits;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, few_rows_kernel<kAct>, tw, ta, blocks, a.scale, a.scale_row, a.scale_col, w.scale,
                            w.scale_row, w.scale_col, m, n, y, ldy, y_type, splits, error_flag);
}

template <int kTileN>
cudaError_t pair_launch(const Fp8Operand& a, const Fp8Operand& w, int m, int n, int k, void* y, int64_t ldy,
                        int y_type, int* error_flag, int sms, cudaStream_t stream) {
  static std::atomic<bool> done[kMaxDevices];
  cudaError_t e = configure_once((const void*)pair_kernel<kTileN>, Pair<kTileN>::kSmem, done);
  if (e != cudaSuccess) return e;
  CUtensorMap ta, tw;
  e = encode_e4m3_map(&ta, a.q, k, m, a.ld, 128);
  if (e != cudaSuccess) return e;
  e = encode_e4m3_map(&tw, w.q, k, n, w.ld, kTileN / 2);
  if (e != cudaSuccess) return e;
  const int64_t tm = (m + (int64_t)kPairRows - 1) / kPairRows, tn = (n + (int64_t)kTileN - 1) / kTileN;
  if (tm * tn > (1 << 30)) return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * std::min<int64_t>(tm * tn, sms / 2)), 1, 1);
  cfg.blockDim = dim3(kPairThreads, 1, 1);
  cfg.dynamicSmemBytes = Pair<kTileN>::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, pair_kernel<kTileN>, ta, tw, (k + kFp8Block - 1) / kFp8Block, a.scale, a.scale_row,
                            a.scale_col, w.scale, w.scale_row, w.scale_col, m, n, y, ldy, y_type, (int)tm, (int)tn,
                            error_flag);
}

}  // namespace

cudaError_t fp8_gemm_launch(Fp8Operand a, Fp8Operand w, int64_t m, int64_t n, int64_t k, void* y, int64_t ldy,
                            int y_type, int* error_flag, cudaStream_t stream) {
  if (m <= 0 || n <= 0) return cudaSuccess;
  if (k <= 0) {
    const int size = y_type == LLVQ_DT_F32 ? 4 : 2;
    return cudaMemset2DAsync(y, (size_t)ldy * size, 0, (size_t)n * size, (size_t)m, stream);
  }
  int sms = 0;
  const cudaError_t e = device_sms(&sms);
  if (e != cudaSuccess) return e;
#define LLVQ_FEW(N) few_rows_launch<N>(a, w, (int)m, (int)n, (int)k, y, ldy, y_type, error_flag, sms, stream)
  if (m <= 16) return LLVQ_FEW(16);
  if (m <= 32) return LLVQ_FEW(32);
  if (m <= 64) return LLVQ_FEW(64);
  if (m <= 256) return LLVQ_FEW(128);
  return pair_launch<256>(a, w, (int)m, (int)n, (int)k, y, ldy, y_type, error_flag, sms, stream);
#undef LLVQ_FEW
}

}  // namespace llvq
