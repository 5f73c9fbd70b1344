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
  return LLVQ_FEW(128);
#undef LLVQ_FEW
}

}  // namespace llvq
