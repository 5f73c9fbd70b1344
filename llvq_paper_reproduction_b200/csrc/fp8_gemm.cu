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

#include "fp8_launch.cuh"
#include "llvq_b200.h"
#include "llvq_internal.h"
#include "tcgen05.cuh"

namespace llvq {

PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder();  // gemm.cu

namespace {

constexpr int kMaxSplits = 8;  // CTAs that share a tile's K blocks: a portable cluster

template <typename T>
__device__ __forceinline__ T to_out(float v) {
  if constexpr (sizeof(T) == 4) return v;
  else if constexpr (std::is_same_v<T, __half>) return __float2half_rn(v);
  else return __float2bfloat16_rn(v);
}

// Two fp32 values in a register pair.
__device__ __forceinline__ uint64_t pack2(uint32_t lo, uint32_t hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
  return r;
}

__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
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

// Four neighbouring outputs, `count` of them in the matrix; whole: 16-byte stores are possible.
__device__ __forceinline__ void store4(void* y, int64_t i, float4 v, int type, bool whole, int count) {
  if (type == LLVQ_DT_F32) {
    float* p = static_cast<float*>(y) + i;
    if (whole && count >= 4) {
      *reinterpret_cast<float4*>(p) = v;
    } else {
      p[0] = v.x;
      if (count > 1) p[1] = v.y;
      if (count > 2) p[2] = v.z;
      if (count > 3) p[3] = v.w;
    }
    return;
  }
  uint2 w;
  if (type == LLVQ_DT_F16) {
    const __half2 lo = __floats2half2_rn(v.x, v.y), hi = __floats2half2_rn(v.z, v.w);
    w = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
  } else {
    const __nv_bfloat162 lo = __floats2bfloat162_rn(v.x, v.y), hi = __floats2bfloat162_rn(v.z, v.w);
    w = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
  }
  uint16_t* p = static_cast<uint16_t*>(y) + i;
  if (whole && count >= 4) {
    *reinterpret_cast<uint2*>(p) = w;
  } else {
    p[0] = (uint16_t)w.x;
    if (count > 1) p[1] = (uint16_t)(w.x >> 16);
    if (count > 2) p[2] = (uint16_t)w.y;
    if (count > 3) p[3] = (uint16_t)(w.y >> 16);
  }
}

// Whether rows of y can be stored in 16-byte chunks.
__device__ __forceinline__ bool whole_chunks(const void* y, int64_t ldy, int type) {
  const int64_t size = type == LLVQ_DT_F32 ? 4 : 2;
  return ldy * size % 16 == 0 && reinterpret_cast<uintptr_t>(y) % 16 == 0;
}

// Partial sums of a tile in shared memory: rows of kWidth fp32 in 16-byte chunks, kSwizzle: exchanged by the row.
template <int kWidth, bool kSwizzle>
__device__ __forceinline__ uint32_t partial_at(uint32_t base, int row, int chunk) {
  return base + (uint32_t)row * (kWidth * 4) + (uint32_t)((kSwizzle ? chunk ^ (row & 7) : chunk) * 16);
}

// Adds the tile's parts over the cluster in rank order and stores them; this
// CTA takes a 1 / splits share.  Rolled loops, as the code runs once (an unrolled
// form took 9300 cycles of a 20,000-cycle kernel), that load kU elements of kS parts
// together: two of two where there are two parts (512 x 4096 x 4096: 16.7 us
// against 17.8), one of four where there are more (256 x 4096 x 4096, four parts:
// 12.8 us, two of two 13.5, two of four 13.5).
template <int kWidth, bool kSwizzle, int kU, int kS>
__device__ __forceinline__ void add_parts(uint32_t partial, int begin, int end, int splits, void* y, int64_t ldy,
                                          int y_type, int m0, int n0, int n_total, int t, int threads) {
  constexpr int kChunks = kWidth / 4;
  const bool whole = whole_chunks(y, ldy, y_type);
#pragma unroll 1
  for (int e = begin + t; e < end; e += kU * threads) {
    uint32_t at[kU];
    float4 sum[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int f = u == 0 ? e : min(e + u * threads, end - 1);
      at[u] = partial_at<kWidth, kSwizzle>(partial, f / kChunks, f % kChunks);
      sum[u] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll 1
    for (int s = 0; s < splits; s += kS) {
      float4 p[kU][kS];
#pragma unroll
      for (int i = 0; i < kS; ++i)
#pragma unroll
        for (int u = 0; u < kU; ++u)
          p[u][i] = s + i < splits ? tc::ld_cluster4(tc::map_rank(at[u], s + i)) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int i = 0; i < kS; ++i)
#pragma unroll
        for (int u = 0; u < kU; ++u)
          sum[u].x += p[u][i].x, sum[u].y += p[u][i].y, sum[u].z += p[u][i].z, sum[u].w += p[u][i].w;
    }
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int f = e + u * threads, col = n0 + f % kChunks * 4;
      if (f < end && col < n_total)
        store4(y, (int64_t)(m0 + f / kChunks) * ldy + col, sum[u], y_type, whole, n_total - col);
    }
  }
}

template <int kWidth, bool kSwizzle>
__device__ __forceinline__ void store_reduced(uint32_t partial, int rank, int splits, void* y, int64_t ldy, int y_type,
                                              int m0, int n0, int rows, int n_total, int t, int threads) {
  const int all = rows * (kWidth / 4), begin = all * rank / splits, end = all * (rank + 1) / splits;
  if (splits == 2)
    add_parts<kWidth, kSwizzle, 2, 2>(partial, begin, end, splits, y, ldy, y_type, m0, n0, n_total, t, threads);
  else
    add_parts<kWidth, kSwizzle, 1, 4>(partial, begin, end, splits, y, ldy, y_type, m0, n0, n_total, t, threads);
}

// ---------------------------------------------------------------- few rows
// Weights are the 128-row side of the MMA (TMEM lane = weight row), the
// activation rows its N side (kAct columns), so few rows waste little and the
// weights stream through once.  The K blocks of a tile are split over the
// CTAs of a cluster, which add their partial sums through distributed shared
// memory in rank order.
//
// Roles: warp 0 loads both operands with TMA, warp 1 issues the MMAs, warps
// 2..5 add up.  The adders take kGroup blocks at a time (64 columns of TMEM, one
// load): a pass is a chain of latencies, about 1000 cycles however narrow the
// sums are.  TMEM holds kBufs such groups so the MMAs run ahead.  Scales come
// with cp.async, kChunk blocks at a time and one chunk ahead.
constexpr int kFewThreads = 192;
constexpr int kTileRows = 128;

template <int kAct>
struct Few {
  static constexpr int kStageBytes = kTileRows * 128 + kAct * 128;
  // two CTAs per SM: at least 76 KB each, so that a third, which could run out of TMEM, never fits
  static constexpr int kStages = (98 * 1024) / kStageBytes;
  static constexpr int kGroup = kAct < 64 ? 64 / kAct : 1;
  static constexpr int kTmemCols = 256;
  static constexpr int kBufs = kTmemCols / (kAct * kGroup);
  static constexpr int kChunk = 1024 / kAct < 64 ? 1024 / kAct : 64;  // blocks
  static constexpr int kScaleFloats = kChunk * (kAct + 4);  // row scales of every block, then its weight scale
  static constexpr int kScaleOff = kStages * kStageBytes;
  static constexpr int kBarOff = kScaleOff + 2 * kScaleFloats * 4;
  static constexpr int kBars = 2 * kStages + 2 * kBufs + 1;
  static constexpr size_t kSmem = (size_t)kBarOff + 8 * kBars + 16 + 1024;
  static_assert(kAct * kGroup == 64 && kStages >= 2 && kAct * kTileRows * 4 <= kScaleOff && kScaleOff % 16 == 0 && kBarOff % 8 == 0);
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
  auto load_stage = [&](int i) {
    const int st = i % F::kStages;
    const uint32_t dst = sbase + st * F::kStageBytes;
    tc::mbar_arrive_expect_tx(full(st), F::kStageBytes);
    tc::tma_load_2d(dst, &tw, (b_begin + i) * kFp8Block, n0, full(st));
    tc::tma_load_2d(dst + kTileRows * 128, &ta, (b_begin + i) * kFp8Block, m0, full(st));
  };
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
    tc::fence_proxy_async();
    // the first loads are under way while the CTA sets up, the weights' on their way to L2 even before the
    // kernel ahead of this one has ended
    for (int i = 0; i < F::kStages && i < count; ++i) tc::tma_prefetch_2d(&tw, (b_begin + i) * kFp8Block, n0);
    wait_for_inputs();
    for (int i = 0; i < F::kStages && i < count; ++i) load_stage(i);
  }
  if (warp == 1) tc::tmem_alloc(tc::smem_addr(holder), F::kTmemCols);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = *holder;
  bool failed = false;
  uint64_t acc[kAct / 2];
  wait_for_inputs();

  if (warp == 0) {
    if (lane == 0) {  // TMA producer
      int i = F::kStages;
      for (; i < count; ++i) {
        if (!tc::mbar_wait_for<0>(empty(i % F::kStages), (i / F::kStages - 1) & 1)) {
          failed = true;
          break;
        }
        load_stage(i);
      }
      // no copy may still be in flight when the block exits: wait for the last use of every stage
      i = min(i, count);
      for (int u = i > F::kStages ? i - F::kStages : 0; u < i; ++u)
        tc::mbar_wait_for<0>(full(u % F::kStages), (u / F::kStages) & 1);
    }
  } else if (warp == 1) {  // MMA issuer: the warp waits, one thread issues
    constexpr uint32_t idesc = tc::idesc_e4m3_f32(kTileRows, kAct);
    const bool issuer = tc::elect_one();
    const uint64_t desc0 = tc::desc_sw128(sbase);
    uint32_t st = 0, st_use = 0;
    for (int i = 0; i < count; ++i) {
      const uint32_t in_group = i % F::kGroup, buf = i / F::kGroup % F::kBufs, use = i / F::kGroup / F::kBufs;
      if ((in_group == 0 && use > 0 && !tc::mbar_wait_for<0>(acc_empty(buf), (use - 1) & 1u)) ||
          !tc::mbar_wait_for<0>(full(st), st_use & 1u)) {
        failed = true;
        break;
      }
      tc::fence_after_sync();
      if (issuer) {
        const uint64_t dw = desc0 + st * (F::kStageBytes >> 4), da = dw + (kTileRows * 128 >> 4);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
          tc::mma_f8(tmem + (buf * F::kGroup + in_group) * kAct, dw + 2 * ks, da + 2 * ks, idesc, ks > 0);
        tc::commit(empty(st));
        if (in_group == F::kGroup - 1 || i == count - 1) tc::commit(acc_full(buf));
      }
      __syncwarp();
      if (++st == F::kStages) st = 0, ++st_use;
    }
    // every MMA issued has finished before TMEM is freed
    if (issuer) tc::commit(drain);
    __syncwarp();
    tc::mbar_wait_for<64>(drain, 0);
  } else {  // warps 2..5 read TMEM lane quarters 2, 3, 0, 1
    const int t = tid - 64;
    const uint32_t t0 = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    float* scales = reinterpret_cast<float*>(base + F::kScaleOff);
    // chunk c of kChunk blocks into half c & 1 of the scales
    auto fetch = [&](int c) {
      const int first = c * F::kChunk, last = min(count, first + F::kChunk);
      const uint32_t half = tc::smem_addr(scales + (c & 1) * F::kScaleFloats);
      for (int e = t; e < (last - first) * kAct; e += 128) {
        const int i = e / kAct, j = e % kAct;
        const bool live = m0 + j < m_total;
        tc::cp_async4(half + (i * (kAct + 4) + j) * 4,
                      as + (live ? (m0 + j) * as_row + (b_begin + first + i) * as_col : 0), live);
      }
      for (int i = t; i < last - first; i += 128)
        tc::cp_async4(half + (i * (kAct + 4) + kAct) * 4, ws + tile * ws_row + (b_begin + first + i) * ws_col, true);
      tc::cp_async_commit();
    };
#pragma unroll
    for (int j = 0; j < kAct / 2; ++j) acc[j] = 0;
    uint32_t seen = 0;  // the next group's sums are known to be there
    fetch(0);
    for (int i0 = 0; i0 < count; i0 += F::kGroup) {
      if (i0 % F::kChunk == 0) {
        tc::cp_async_wait<0>();
        __syncwarp();
        asm volatile("bar.sync 1, 128;" ::: "memory");  // this chunk is whole, and nobody reads the last one any more
        if (i0 + F::kChunk < count) fetch(i0 / F::kChunk + 1);
      }
      const int g = i0 / F::kGroup, buf = g % F::kBufs;
      if (!seen && !failed && !tc::mbar_wait_for<0>(acc_full(buf), (g / F::kBufs) & 1)) failed = true;
      __syncwarp();  // lanes leave a wait one by one, and a TMEM load is the whole warp's
      tc::fence_after_sync();
      uint32_t v[64];
      tc::tmem_ld64(t0 + buf * 64, v);
      const uint32_t slot =
          tc::smem_addr(scales) + ((i0 / F::kChunk & 1) * F::kScaleFloats + i0 % F::kChunk * (kAct + 4)) * 4;
      tc::tmem_wait_ld();
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(acc_empty(buf));
      seen = tc::mbar_peek(acc_full((g + 1) % F::kBufs), ((g + 1) / F::kBufs) & 1);
#pragma unroll
      for (int u = 0; u < F::kGroup; ++u) {
        if (i0 + u < count) {
          const uint32_t row = slot + u * (kAct + 4) * 4;
          const uint32_t w = tc::ld_shared_bits(row + kAct * 4);
          const uint64_t ww = pack2(w, w);
#pragma unroll
          for (int j = 0; j < kAct; j += 4) {  // the weight's scale, then the row's: their product may leave fp32's range
            uint64_t s0, s1;
            tc::ld_shared_pairs(row + j * 4, s0, s1);
            const uint32_t* x = v + u * kAct + j;
            acc[j / 2] = fma2(mul2(pack2(x[0], x[1]), ww), s0, acc[j / 2]);
            acc[j / 2 + 1] = fma2(mul2(pack2(x[2], x[3]), ww), s1, acc[j / 2 + 1]);
          }
        }
      }
    }
    // the last block's sums have been read, so every stage has been consumed: reuse them
    float* part = reinterpret_cast<float*>(base) + (warp & 3) * 32 + lane;
#pragma unroll
    for (int j = 0; j < kAct; j += 2) unpack2(acc[j / 2], part[j * kTileRows], part[(j + 1) * kTileRows]);
  }
  // at the end: the next product's CTAs find no room before (at the start, 64 x 4096 x 14336: 15.0 us both)
  dependents_may_start();
  __syncwarp();
  if (failed && error_flag) atomicExch(error_flag, 1);
  __syncwarp();
  tc::cluster_sync();
  if (warp >= 2)
    store_reduced<kTileRows, false>(sbase, rank, splits, y, ldy, y_type, m0, n0, min(kAct, m_total - m0), n_total,
                                    tid - 64, 128);
  __syncwarp();
  tc::cluster_sync();  // no CTA leaves while another still reads its sums
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  if (warp == 1) tc::tmem_dealloc(tmem, F::kTmemCols);
}

// ---------------------------------------------------------------- many rows
// Activations are the M side: TMEM lane = activation row, so a lane's scale
// for a block is one number, a_scale[row] w_scale, and the addition is one
// packed fused multiply-add per two outputs.  Tiles are 256 weight rows wide.
//
// Wide<2>: two CTAs of a cluster share a tile of 256 activation rows (tcgen05
// cta_group::2, M = 256); each loads 128 activation rows and half of the weight
// rows, so a block costs a CTA 32 KB for 128 x 256 outputs instead of 48.
// Persistent: one pair per two SMs.
// Wide<1>: a CTA per tile of 128 activation rows, where that fits one wave; the
// K blocks are split over a cluster, which adds its partial sums through
// distributed shared memory in rank order.
//
// Roles: warps 0..7 add up (lane quarter warp % 4, column half warp / 4), warp 8
// loads with TMA, warp 9 (of the leading CTA) issues the MMAs, warps 10 and 11
// bring the scales, kScaleGroup blocks at a time and two groups in flight.  TMEM
// holds two block sums of 256 columns.  In a pair the leader's full[] takes the
// bytes of both CTAs' loads; empty[] and acc_full[] are committed in both CTAs;
// the leader's acc_empty[] takes the arrivals of all 16 adding warps.
//
// What bounds it: a block costs about 860 cycles where its MMAs take 512
// (4096 x 14336 x 4096 in a captured graph at 1.69 GHz: 219 us, 2.2 PFLOP/s; without
// the additions 191, without the TMEM loads too 176; call after call, at the
// 1.48 GHz of the power limit, 257 us, 1.87 PFLOP/s).  Beside that pairs idle where the
// tiles leave their last round partly empty: 896 tiles there, 13 rounds for the work of 12.1;
// 1280 x 4096, 80 tiles, two rounds for 1.08.  An adding warp's pass is a chain of latencies: the
// block's sums ready, a TMEM load, 32 FFMA2, a second load, the buffer handed
// back, 32 FFMA2 (2.4 cycles each on a scheduler); hence loads of 64 columns, and
// the look for the next block before the last additions.  Measured beside it:
// 16 warps of 64 columns at 112 registers 225 us; halves of the buffer handed
// back apart 237; tiles of 192 columns read in one piece 262.
constexpr int kAddWarps = 8;
constexpr int kWideThreads = kAddWarps * 32 + 128;
// 384 threads launch with 168 registers each: 64,512 = 256 x 224 + 128 x 56
constexpr int kAddRegs = 224, kOtherRegs = 56;
constexpr int kTileN = 256;
constexpr int kCols = kTileN / (kAddWarps / 4);  // columns of an adding warp
constexpr int kAccBufs = 512 / kTileN;
constexpr int kScaleGroup = 8, kScaleGroups = 2;
constexpr int kScaleBlock = (128 + 4) * 4;  // bytes of a block's scales: 128 rows, two column halves

template <int kCtas>
struct Wide {
  static constexpr int kStageA = 128 * 128, kStageB = kTileN / kCtas * 128;
  static constexpr int kStageBytes = kStageA + kStageB;
  static constexpr int kStages = kCtas == 2 ? 5 : 4;
  // 4 KB per adding warp to store through; a CTA with a single tile stores when its stages are free, 16 KB
  static constexpr int kStoreBufs = kCtas == 2 ? 1 : 4;
  static constexpr int kStoreOff = kCtas == 2 ? kStages * kStageBytes : 0;
  static constexpr int kScaleOff = kCtas == 2 ? kStoreOff + kAddWarps * 4096 : kStages * kStageBytes;
  static constexpr int kBarOff = kScaleOff + kScaleGroups * kScaleGroup * kScaleBlock;
  static constexpr int kBars = 2 * kStages + 2 * kAccBufs + 2 * kScaleGroups + 1;
  static constexpr size_t kSmem = (size_t)kBarOff + 8 * kBars + 16 + 1024;
  static_assert(kSmem <= 227 * 1024 && kScaleOff >= 128 * kTileN * 4 && kStoreOff + kAddWarps * kStoreBufs * 4096 <= kScaleOff);
};

// acc + v * (as ws).  Where that product is below fp32's normal numbers or not
// finite (plain false), the two are applied one after the other; by the lane, so
// that no row depends on another.  A normal product is rounded once, wherever it
// lies: rows of zeros, whose scale is the floor's 2^-108.8, stay on the plain side
// (400 x 14336 x 4096 with a quarter of the rows zero: 35.4 us; 42.7 when 2^-60 was the end).
struct Scale {
  float factor, pre;
  bool plain;
  __device__ __forceinline__ Scale(float as, float ws) : factor(as * ws), pre(ws) {
    plain = ((__float_as_uint(factor) >> 23) & 255u) - 1u < 254u;  // normal
    if (!plain) factor = as;
  }
};

template <int kCount>
__device__ __forceinline__ void add_scaled(uint64_t* acc, uint32_t* v, const Scale& s) {
  if (!s.plain) {
#pragma unroll
    for (int j = 0; j < kCount; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) * s.pre);
  }
  const uint64_t ff = pack2(__float_as_uint(s.factor), __float_as_uint(s.factor));
#pragma unroll
  for (int j = 0; j < kCount / 2; ++j) acc[j] = fma2(pack2(v[2 * j], v[2 * j + 1]), ff, acc[j]);
}

// The buffer of store_rows where y's rows start on 8-byte boundaries: 16 lanes a row.
template <typename T>
__device__ __forceinline__ void store_halves(const uint8_t* buf, T* __restrict__ y, int64_t ldy, int row0, int col0,
                                             int m_total, int n_total, int lane) {
  constexpr int kPer = 8 / (int)sizeof(T);
  const int byte = (lane & 15) * 8, col = col0 + (lane & 15) * kPer;
  if (col >= n_total) return;
#pragma unroll 4
  for (int r = lane >> 4; r < 32; r += 2) {
    if (row0 + r >= m_total) continue;
    const uint2 v = *reinterpret_cast<const uint2*>(buf + r * 128 + (((byte >> 4) ^ (r & 7)) * 16) + (byte & 15));
    T* dst = y + (int64_t)(row0 + r) * ldy + col;
    if (col + kPer <= n_total) {
      *reinterpret_cast<uint2*>(dst) = v;
    } else {
      const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
      for (int j = 0; j < kPer; ++j)
        if (col + j < n_total) dst[j] = e[j];
    }
  }
}

// ... and where they start anywhere: eight lanes a row, whose 128 bytes they store
// as the 16-byte chunks of memory that lie within them, each put together from five
// words of the buffer, and the elements before the first and behind the last chunk
// one a lane (together one chunk's, or none).  1317 x 13418 x 152, bf16: 29.1 us,
// by stores of four bytes 32.5; of two, at 13417, 35.5.  By store_halves 13420
// columns take 22.7 us, so 29.1; 13416, by TMA, 14.7.
template <typename T>
__device__ __forceinline__ void store_shifted(const uint8_t* buf, T* __restrict__ y, int64_t ldy, int row0, int col0,
                                              int m_total, int n_total, int lane) {
  constexpr int kLine = 128 / (int)sizeof(T), kChunk = 16 / (int)sizeof(T);
  const int c = lane & 7, left = min(kLine, n_total - col0), rows = min(32, m_total - row0);
  if (left <= 0) return;
  auto at = [&](int r, int byte) { return buf + r * 128 + (((byte >> 4) ^ (r & 7)) * 16) + (byte & 15); };
  T* const y0 = y + (int64_t)row0 * ldy + col0;
  // elements of row r before a boundary
  auto head_of = [&](int r) {
    return (int)((16 - (reinterpret_cast<uintptr_t>(y0 + r * ldy) & 15)) & 15) / (int)sizeof(T);
  };
#pragma unroll 4
  for (int r = lane >> 3; r < 32; r += 4) {
    const int first = head_of(r) + c * kChunk, byte = first * (int)sizeof(T);
    uint32_t w[5];
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = *reinterpret_cast<const uint32_t*>(at(r, ((byte & ~3) + 4 * i) & 127));
    const uint32_t shift = (byte & 3) * 8;
    if (r < rows && first + kChunk <= left)
      *reinterpret_cast<uint4*>(y0 + r * ldy + first) =
          make_uint4(__funnelshift_r(w[0], w[1], shift), __funnelshift_r(w[1], w[2], shift),
                     __funnelshift_r(w[2], w[3], shift), __funnelshift_r(w[3], w[4], shift));
  }
  for (int e = c; e < (left < kLine ? 16 : 8); e += 8) {  // twice where the matrix cuts the line off
#pragma unroll 4
    for (int r = lane >> 3; r < 32; r += 4) {
      const int heads = min(head_of(r), left), end = heads + (left - heads) / kChunk * kChunk;
      const int i = e < heads ? e : end + e - heads;
      const T v = *reinterpret_cast<const T*>(at(r, i * (int)sizeof(T) & 127));
      if (r < rows && i < left) y0[r * ldy + i] = v;
    }
  }
}

// A warp's 32 rows x kWidth columns to y, through kBufs times 4 KB of shared memory
// (32 rows of 128 bytes in the 128-byte swizzle).  Where y's rows start and end on
// 16-byte boundaries (tma) the buffer leaves by an asynchronous TMA store, clipped at
// the matrix's ends; else by store_halves or store_shifted.
template <typename T, int kWidth, int kBufs>
__device__ __forceinline__ void store_rows(const uint64_t* acc, uint8_t* bufs, const CUtensorMap* ty, bool tma,
                                           T* __restrict__ y, int64_t ldy, int row0, int col0, int m_total, int n_total,
                                           int lane) {
  constexpr int kPerLine = 128 / (int)sizeof(T), kPerChunk = 16 / (int)sizeof(T);
#pragma unroll
  for (int c0 = 0; c0 < kWidth; c0 += kPerLine) {
    uint8_t* buf = bufs + c0 / kPerLine % kBufs * 4096;
    if (tma && kBufs * kPerLine < kWidth) {
      if (lane == 0) tc::bulk_wait_read();  // the store before has read the buffer
      __syncwarp();
    }
#pragma unroll
    for (int ch = 0; ch < 8; ++ch) {
      alignas(16) T e[kPerChunk];
#pragma unroll
      for (int j = 0; j < kPerChunk; j += 2) {
        float lo, hi;
        unpack2(acc[(c0 + ch * kPerChunk + j) / 2], lo, hi);
        e[j] = to_out<T>(lo);
        e[j + 1] = to_out<T>(hi);
      }
      *reinterpret_cast<uint4*>(buf + lane * 128 + ((ch ^ (lane & 7)) * 16)) = *reinterpret_cast<const uint4*>(e);
    }
    if (tma) {
      tc::fence_proxy_async();
      __syncwarp();
      if (lane == 0 && row0 < m_total && col0 + c0 < n_total) tc::tma_store_2d(ty, col0 + c0, row0, tc::smem_addr(buf));
    } else {
      __syncwarp();
      if ((reinterpret_cast<uintptr_t>(y) | (uintptr_t)(ldy * (int64_t)sizeof(T))) % 8 == 0)
        store_halves(buf, y, ldy, row0, col0 + c0, m_total, n_total, lane);
      else
        store_shifted(buf, y, ldy, row0, col0 + c0, m_total, n_total, lane);
      __syncwarp();
    }
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

// Wide<2>: `split` is 1 and a pair takes tiles pair, + pairs, ...  Wide<1>: one
// tile per cluster of `split` CTAs.
template <int kCtas>
__global__ void __launch_bounds__(kWideThreads, 1)
    wide_kernel(const __grid_constant__ CUtensorMap ta, const __grid_constant__ CUtensorMap tw,
                const __grid_constant__ CUtensorMap ty, bool tma_store, int blocks_total,
                const float* __restrict__ as, int64_t as_row, int64_t as_col, const float* __restrict__ ws,
                int64_t ws_row, int64_t ws_col, int m_total, int n_total, void* __restrict__ y, int64_t ldy, int y_type,
                int tm, int tn, int splits, int* error_flag) {
  using P = Wide<kCtas>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(base + P::kBarOff);
  uint32_t* holder = reinterpret_cast<uint32_t*>(bars + P::kBars);
  const uint32_t sbase = tc::smem_addr(base);
  auto full = [&](int st) { return tc::smem_addr(&bars[st]); };
  auto empty = [&](int st) { return tc::smem_addr(&bars[P::kStages + st]); };
  auto acc_full = [&](int b) { return tc::smem_addr(&bars[2 * P::kStages + b]); };
  auto acc_empty = [&](int b) { return tc::smem_addr(&bars[2 * P::kStages + kAccBufs + b]); };
  auto scale_full = [&](int i) { return tc::smem_addr(&bars[2 * P::kStages + 2 * kAccBufs + i]); };
  auto scale_empty = [&](int i) { return tc::smem_addr(&bars[2 * P::kStages + 2 * kAccBufs + kScaleGroups + i]); };
  const uint32_t drain = tc::smem_addr(&bars[P::kBars - 1]);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // rank: of the CTA in its pair; part: its share of the K blocks
  const int rank = kCtas == 2 ? (int)tc::cluster_rank() : 0, part = kCtas == 1 ? (int)tc::cluster_rank() : 0;
  const int tiles = tm * tn, first = kCtas == 2 ? (int)blockIdx.x >> 1 : (int)blockIdx.x / splits;
  const int step = kCtas == 2 ? (int)gridDim.x >> 1 : tiles;
  const int b_begin = (int)((int64_t)blocks_total * part / splits);
  const int blocks = (int)((int64_t)blocks_total * (part + 1) / splits) - b_begin;
  auto load_stage = [&](uint32_t st, int b, int m0, int n0) {
    const uint32_t dst = sbase + st * P::kStageBytes, bar = kCtas == 2 ? tc::map_rank(full(st), 0) : full(st);
    if (rank == 0) tc::mbar_arrive_expect_tx(full(st), kCtas * P::kStageBytes);
    tc::Ctas<kCtas>::tma_load(dst, &ta, (b_begin + b) * kFp8Block, m0, bar);
    tc::Ctas<kCtas>::tma_load(dst + P::kStageA, &tw, (b_begin + b) * kFp8Block, n0, bar);
  };
  if (tid == kAddWarps * 32) {  // the producer
    for (int i = 0; i < P::kStages; ++i) {
      tc::mbar_init(full(i), 1);
      tc::mbar_init(empty(i), 1);
    }
    for (int i = 0; i < kAccBufs; ++i) {
      tc::mbar_init(acc_full(i), 1);
      tc::mbar_init(acc_empty(i), kCtas * kAddWarps);
    }
    for (int i = 0; i < kScaleGroups; ++i) {
      tc::mbar_init(scale_full(i), 64);  // the threads of two warps, when their copies are there
      tc::mbar_init(scale_empty(i), kAddWarps);
    }
    tc::mbar_init(drain, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    tc::fence_proxy_async();
    wait_for_inputs();
    if (kCtas == 1) {  // nothing to wait for: the first loads are under way while the CTA sets up
      int mt, nt;
      tile_at(first, tm, tn, mt, nt);
      for (int b = 0; b < P::kStages && b < blocks; ++b) load_stage(b, b, mt * 128, nt * kTileN);
    }
  }
  __syncwarp();
  if (warp == kAddWarps + 1) tc::Ctas<kCtas>::alloc(tc::smem_addr(holder), 512);
  tc::fence_before_sync();
  if (kCtas == 1) __syncthreads();
  else tc::cluster_sync();
  tc::fence_after_sync();
  const uint32_t tmem = *holder;
  bool failed = false;
  wait_for_inputs();

  if (warp >= kAddWarps) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == kAddWarps && lane == 0) {  // TMA producer of this CTA's operands
      uint32_t g = 0;
      for (int t = first; t < tiles && !failed; t += step) {
        int mt, nt;
        tile_at(t, tm, tn, mt, nt);
        const int m0 = (mt * kCtas + rank) * 128, n0 = nt * kTileN + rank * (kTileN / kCtas);
        for (int b = 0; b < blocks; ++b, ++g) {
          const int st = (int)(g % P::kStages);
          const uint32_t use = g / P::kStages;
          if (use > 0 && !tc::mbar_wait_for<64>(empty(st), (use - 1) & 1u)) {
            failed = true;
            break;
          }
          if (kCtas == 2 || use > 0) load_stage(st, b, m0, n0);
        }
      }
      // every stage loaded has been consumed before the CTA may exit
      for (uint32_t u = g > (uint32_t)P::kStages ? g - P::kStages : 0u; u < g; ++u)
        if (!tc::mbar_wait_for<0>(empty((int)(u % P::kStages)), (u / P::kStages) & 1u)) failed = true;
    }
    if (warp == kAddWarps + 1 && rank == 0) {  // MMA issuer: the warp waits, one thread issues
      constexpr uint32_t idesc = tc::idesc_e4m3_f32(128 * kCtas, kTileN);
      const bool issuer = tc::elect_one();
      const uint64_t desc0 = tc::desc_sw128(sbase);
      uint32_t st = 0, st_use = 0, buf = 0, buf_use = 0;
      for (int t = first; t < tiles && !failed; t += step) {
        for (int b = 0; b < blocks; ++b) {
          // even lanes poll for the operands, odd ones for the TMEM columns: one latency instead of two
          const uint32_t bar = (lane & 1) ? acc_empty(buf) : full(st);
          const uint32_t parity = (lane & 1) ? (buf_use - 1) & 1u : st_use & 1u;
          const bool ready = ((lane & 1) && buf_use == 0) || tc::mbar_wait_for<0>(bar, parity);
          if (!__all_sync(0xffffffffu, ready)) {
            failed = true;
            break;
          }
          tc::fence_after_sync();
          if (issuer) {
            const uint64_t da = desc0 + st * (P::kStageBytes >> 4), dw = da + (P::kStageA >> 4);
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
              tc::Ctas<kCtas>::mma(tmem + buf * kTileN, da + 2 * ks, dw + 2 * ks, idesc, ks > 0);
            tc::Ctas<kCtas>::commit(acc_full(buf));
            tc::Ctas<kCtas>::commit(empty(st));
          }
          __syncwarp();
          if (++st == P::kStages) st = 0, ++st_use;
          if (++buf == kAccBufs) buf = 0, ++buf_use;
        }
      }
      // every MMA issued has finished before TMEM is freed
      if (issuer) tc::Ctas<kCtas>::commit(drain);
      __syncwarp();
      tc::mbar_wait_for<64>(drain, 0);
    }
    if (warp >= kAddWarps + 2) {  // scales: thread i copies those of rows i and i + 64, threads 0 and 1 the weights'
      const int i = tid - (kAddWarps + 2) * 32;
      uint32_t slot = 0, use = 0;
      for (int t = first; t < tiles && !failed; t += step) {
        int mt, nt;
        tile_at(t, tm, tn, mt, nt);
        // rows past the last take the last one's scale, not zero: zero is outside the plain range, and a tile
        // that is not full would run the additions' other branch (400 x 14336 x 4096: 42 us against 35)
        const int row0 = (mt * kCtas + rank) * 128 + i, last_row = m_total - 1;
        const int half = min(nt * (kTileN / kFp8Block) + i, (n_total - 1) / kFp8Block);
        const float *pa0 = as + min(row0, last_row) * as_row, *pa1 = as + min(row0 + 64, last_row) * as_row;
        const float* pw = ws + half * ws_row;
        for (int b0 = 0; b0 < blocks; b0 += kScaleGroup) {
          if (use > 0 && !tc::mbar_wait_for<256>(scale_empty(slot), (use - 1) & 1u)) {
            failed = true;
            break;
          }
          uint32_t dst = sbase + P::kScaleOff + slot * (kScaleGroup * kScaleBlock) + i * 4;
          const int last = min(b0 + kScaleGroup, blocks);
          for (int b = b_begin + b0; b < b_begin + last; ++b, dst += kScaleBlock) {
            tc::cp_async4(dst, pa0 + b * as_col, true);
            tc::cp_async4(dst + 256, pa1 + b * as_col, true);
            if (i < 2) tc::cp_async4(dst + 512, pw + b * ws_col, true);
          }
          tc::cp_async_arrive(scale_full(slot));
          if (++slot == kScaleGroups) slot = 0, ++use;
        }
      }
      tc::cp_async_commit();
      tc::cp_async_wait<0>();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kAddRegs));
    const int strip = warp >> 2, quarter = warp & 3;
    const uint32_t t0 = tmem + ((uint32_t)(quarter * 32) << 16) + strip * kCols;
    uint8_t* buf = base + P::kStoreOff + warp * (P::kStoreBufs * 4096);
    const float* scales = reinterpret_cast<const float*>(base + P::kScaleOff);
    const int my_row = quarter * 32 + lane, my_half = 128 + strip * kCols / kFp8Block;
    // Of the block's TMEM buffer, exchanged from block to block: its columns, its
    // acc_full and the issuer's acc_empty.
    static_assert(kAccBufs == 2 && kTileN == 256);
    uint32_t columns = t0, ready = acc_full(0), release = tc::map_rank(acc_empty(0), kCtas == 2 ? 0 : part);
    const uint32_t other_ready = ready ^ acc_full(1);
    const uint32_t other_release = release ^ tc::map_rank(acc_empty(1), kCtas == 2 ? 0 : part);
    uint32_t g = 0, gg = 0, seen = 0;  // seen: block g's sums are known to be there
    for (int t = first; t < tiles && !failed; t += step) {
      int mt, nt;
      tile_at(t, tm, tn, mt, nt);
      const int row0 = (mt * kCtas + rank) * 128 + quarter * 32, col0 = nt * kTileN + strip * kCols;
      uint64_t acc[kCols / 2];
#pragma unroll
      for (int j = 0; j < kCols / 2; ++j) acc[j] = 0;
      for (int b0 = 0; b0 < blocks; b0 += kScaleGroup, ++gg) {
        if (!failed && !tc::mbar_wait_for<0>(scale_full(gg % kScaleGroups), (gg / kScaleGroups) & 1u)) failed = true;
        const float* slot = scales + gg % kScaleGroups * (kScaleGroup * kScaleBlock / 4);
        const int last = min(blocks - b0, kScaleGroup);
#pragma unroll 1
        for (int u = 0; u < last; ++u, ++g, slot += kScaleBlock / 4) {
          if (!seen && !failed && !tc::mbar_wait_for<0>(ready, (g >> 1) & 1u)) failed = true;
          __syncwarp();  // lanes leave a wait one by one, and a TMEM load is the whole warp's
          tc::fence_after_sync();
          uint32_t v[64];
          tc::tmem_ld64(columns, v);
          const Scale scale(slot[my_row], slot[my_half]);
          tc::tmem_wait_ld();
          add_scaled<64>(acc, v, scale);
          __syncwarp();  // after the branch by the lane
          tc::tmem_ld64(columns + 64, v);
          tc::tmem_wait_ld();
          tc::fence_before_sync();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive_cluster(release);
          columns ^= kTileN;  // TMEM is this CTA's alone: the first buffer starts at column 0
          ready ^= other_ready;
          release ^= other_release;
          seen = tc::mbar_peek(ready, ((g + 1) >> 1) & 1u);
          add_scaled<64>(acc + 32, v, scale);
        }
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(scale_empty(gg % kScaleGroups));
      }
      if (kCtas == 1 && splits > 1) {
        // the last block's sums have been read by this warp, so every stage has been consumed: reuse them
#pragma unroll
        for (int j = 0; j < kCols / 4; ++j) {
          float x, y_, z, w;
          unpack2(acc[2 * j], x, y_);
          unpack2(acc[2 * j + 1], z, w);
          tc::st_shared4(partial_at<kTileN, true>(sbase, my_row, strip * (kCols / 4) + j), x, y_, z, w);
        }
      } else if (y_type == LLVQ_DT_F32) {
        store_rows<float, kCols, P::kStoreBufs>(acc, buf, &ty, tma_store, static_cast<float*>(y), ldy, row0, col0, m_total, n_total,
                                 lane);
      } else if (y_type == LLVQ_DT_F16) {
        store_rows<__half, kCols, P::kStoreBufs>(acc, buf, &ty, tma_store, static_cast<__half*>(y), ldy, row0, col0, m_total, n_total,
                                  lane);
      } else {
        store_rows<__nv_bfloat16, kCols, P::kStoreBufs>(acc, buf, &ty, tma_store, static_cast<__nv_bfloat16*>(y), ldy, row0, col0,
                                         m_total, n_total, lane);
      }
    }
  }
  if (warp < kAddWarps && lane == 0) tc::bulk_wait();  // y is written before the kernel ends
  // at the end: the next product's CTAs find no room before (at the start, 64 x 4096 x 14336: 15.0 us both)
  dependents_may_start();
  __syncwarp();
  if (failed && error_flag) atomicExch(error_flag, 1);
  __syncwarp();
  tc::fence_before_sync();
  tc::cluster_sync();  // partial sums are there; no arrival or commit is under way to a CTA that has left
  tc::fence_after_sync();
  if (kCtas == 1 && splits > 1) {
    if (warp < kAddWarps) {
      int mt, nt;
      tile_at(first, tm, tn, mt, nt);
      store_reduced<kTileN, true>(sbase, part, splits, y, ldy, y_type, mt * 128, nt * kTileN,
                                  min(128, m_total - mt * 128), n_total, tid, kAddWarps * 32);
    }
    __syncwarp();
    tc::cluster_sync();  // no CTA leaves while another still reads its sums
  }
  if (warp == kAddWarps + 1) tc::Ctas<kCtas>::dealloc(tmem, 512);
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

// y [rows, cols] of LLVQ_DT_* type (row stride ld elements), box 32 rows x 128 bytes, 128-byte swizzle.
cudaError_t encode_out_map(CUtensorMap* map, void* ptr, int64_t cols, int64_t rows, int64_t ld, int type) {
  const auto enc = tensor_map_encoder();
  if (!enc) return cudaErrorNotSupported;
  const int size = type == LLVQ_DT_F32 ? 4 : 2;
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)(ld * size)};
  const cuuint32_t box[2] = {(cuuint32_t)(128 / size), 32};
  const cuuint32_t elem[2] = {1, 1};
  const CUresult r = enc(map, size == 4 ? CU_TENSOR_MAP_DATA_TYPE_UINT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, ptr, dims,
                         strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
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

// CTAs per tile, in one wave, by the cycles measured for a CTA: 650 a block
// while an SM holds one, 1000 and 2500 more where it holds two; 7500 to start, add
// the parts and store.  At m = 1, 4096 x 4096: 4 CTAs a tile 5.7 us, 8 6.2; 4096 x
// 14336: 4 13.0, 8 11.7; 11008 x 4096: 3 CTAs 9.6, 1 11.9.
int few_splits(int64_t tiles, int64_t blocks, int sms, int64_t* cycles) {
  int best = 1;
  *cycles = INT64_MAX;
  for (int s = 1; s <= kMaxSplits && s <= blocks && (s == 1 || s * tiles <= 2 * sms); ++s) {
    const bool alone = s * tiles <= sms;
    const int64_t cost = (alone ? 7500 : 10000) + (alone ? 650 : 1000) * ((blocks + s - 1) / s);
    if (cost < *cycles) {
      *cycles = cost;
      best = s;
    }
  }
  return best;
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
  int64_t cycles = 0;
  const int splits = few_splits(tn * tm, blocks, sms, &cycles);
  return launch_overlapped(few_rows_kernel<kAct>, dim3((unsigned)(tn * splits), (unsigned)tm), kFewThreads,
                           Few<kAct>::kSmem, splits, stream, tw, ta, blocks, a.scale, a.scale_row, a.scale_col,
                           w.scale, w.scale_row, w.scale_col, m, n, y, ldy, y_type, splits, error_flag);
}

template <int kCtas>
cudaError_t configure_wide() {
  static std::atomic<bool> done[kMaxDevices];
  return configure_once((const void*)wide_kernel<kCtas>, Wide<kCtas>::kSmem, done);
}

// Clusters of 1..kMaxSplits CTAs of Wide<1> that the current device holds at once (they have to fit its GPCs).
cudaError_t resident_clusters(int dev, int (&held)[kMaxSplits + 1]) {
  static std::atomic<int> cache[kMaxDevices][kMaxSplits + 1];
  if (cache[dev][1].load(std::memory_order_acquire) == 0) {
    for (int s = kMaxSplits; s >= 1; --s) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3((unsigned)s, 1, 1);
      cfg.blockDim = dim3(kWideThreads, 1, 1);
      cfg.dynamicSmemBytes = Wide<1>::kSmem;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = (unsigned)s;
      attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      int n = 0;
      const cudaError_t e = cudaOccupancyMaxActiveClusters(&n, wide_kernel<1>, &cfg);
      if (e != cudaSuccess) return e;
      cache[dev][s].store(std::max(n, 1), std::memory_order_release);  // [1] last: the table is whole when it is set
    }
  }
  for (int s = 1; s <= kMaxSplits; ++s) held[s] = cache[dev][s].load(std::memory_order_relaxed);
  return cudaSuccess;
}

// CTAs per tile for Wide<1>: the shortest time over the waves of clusters, in
// cycles as measured: 850 a block, a wave starts and stores in about 9 blocks'
// time, and adding the parts takes 10 more, most of it the reads of distributed
// shared memory.  (7 for two parts would gain 512 x 4096 x 2560, 14.1 to 13.3 us,
// and lose 128 x 14336 x 2048, 12.6 to 13.1.)
cudaError_t choose_splits(int64_t tiles, int64_t blocks, int* splits, int64_t* cycles) {
  int dev = 0, held[kMaxSplits + 1];
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
  e = configure_wide<1>();
  if (e != cudaSuccess) return e;
  e = resident_clusters(dev, held);
  if (e != cudaSuccess) return e;
  *cycles = INT64_MAX;
  for (int s = 1; s <= kMaxSplits && s <= blocks; ++s) {
    const int64_t waves = (tiles + held[s] - 1) / held[s];
    const int64_t cost = 850 * waves * ((blocks + s - 1) / s + (s > 1 ? 19 : 9));
    if (cost < *cycles) {
      *cycles = cost;
      *splits = s;
    }
  }
  return cudaSuccess;
}

// splits: CTAs per tile (Wide<1>).
template <int kCtas>
cudaError_t wide_launch(const Fp8Operand& a, const Fp8Operand& w, int m, int n, int k, void* y, int64_t ldy,
                        int y_type, int* error_flag, int sms, int splits, cudaStream_t stream) {
  cudaError_t e = configure_wide<kCtas>();
  if (e != cudaSuccess) return e;
  CUtensorMap ta, tw, ty = {};
  e = encode_e4m3_map(&ta, a.q, k, m, a.ld, 128);
  if (e != cudaSuccess) return e;
  e = encode_e4m3_map(&tw, w.q, k, n, w.ld, kTileN / kCtas);
  if (e != cudaSuccess) return e;
  const int64_t tm = (m + 128LL * kCtas - 1) / (128 * kCtas), tn = (n + (int64_t)kTileN - 1) / kTileN;
  if (tm * tn > (1 << 27)) return cudaErrorInvalidValue;
  const int size = y_type == LLVQ_DT_F32 ? 4 : 2;
  // A TMA store is clipped along a row by 16-byte chunks: where padded rows end inside one it would write
  // the chunk's other bytes.  (By the line in the kernel instead, for the sake of such rows' other lines, every
  // call was slower: 4096 x 14336 x 4096 227 us against 216.)
  const bool tma_store = ldy * size % 16 == 0 && (int64_t)n * size % 16 == 0 && reinterpret_cast<uintptr_t>(y) % 16 == 0;
  if (tma_store) {
    e = encode_out_map(&ty, y, n, m, ldy, y_type);
    if (e != cudaSuccess) return e;
  }
  const int64_t grid = kCtas == 2 ? 2 * std::min<int64_t>(tm * tn, sms / 2) : tm * tn * splits;
  return launch_overlapped(wide_kernel<kCtas>, dim3((unsigned)grid), kWideThreads, Wide<kCtas>::kSmem,
                           kCtas == 2 ? 2 : splits, stream, ta, tw, ty, tma_store, (k + kFp8Block - 1) / kFp8Block, a.scale,
                           a.scale_row, a.scale_col, w.scale, w.scale_row, w.scale_col, m, n, y, ldy, y_type, (int)tm,
                           (int)tn, splits, error_flag);
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
  cudaError_t e = device_sms(&sms);
  if (e != cudaSuccess) return e;
#define LLVQ_CALL a, w, (int)m, (int)n, (int)k, y, ldy, y_type, error_flag, sms
  if (m <= 16) return few_rows_launch<16>(LLVQ_CALL, stream);
  if (m <= 32) return few_rows_launch<32>(LLVQ_CALL, stream);
  if (m <= 64) return few_rows_launch<64>(LLVQ_CALL, stream);
  const int64_t blocks = (k + kFp8Block - 1) / kFp8Block, tiles = (m + 127) / 128 * ((n + kTileN - 1) / kTileN);
  if (tiles > sms) return wide_launch<2>(LLVQ_CALL, 1, stream);
  int splits = 1;
  int64_t cycles = 0;
  e = choose_splits(tiles, blocks, &splits, &cycles);
  if (e != cudaSuccess) return e;
  // Tiles of 64 activation rows are shorter where the wide ones would be few and
  // their parts many.  128 x 4096 x 4096: 9.9 us against 13.3; 512 x 1024 x 4096:
  // 9.2 against 12.4; 128 x 4096 x 14336 (wide): 19.7 against 20.0.
  const int64_t few = (m + 63) / 64 * ((n + kTileRows - 1) / kTileRows);
  if (2 * few <= sms) {
    int64_t few_cycles = 0;
    few_splits(few, blocks, sms, &few_cycles);
    if (few_cycles < cycles) return few_rows_launch<64>(LLVQ_CALL, stream);
  }
  return wide_launch<1>(LLVQ_CALL, splits, stream);
#undef LLVQ_CALL
}

}  // namespace llvq
