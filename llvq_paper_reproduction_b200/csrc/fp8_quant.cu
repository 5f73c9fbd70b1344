// 8-bit operands for the block-scaled product (sm_100a): quantizers of
// activation rows and of weights, the gated activation and the RMS norm with
// the residual's addition, each writing e4m3 values and fp32 scales.
//
// For a block B of values y (1 x 128 columns, or 128 x 128 for weights):
//   amax = max(2^-100, max |y|)      scale = amax / 448      q = e4m3(448 y / amax)
// 448 is the largest e4m3 value, so nothing saturates; the quotient is formed
// correctly rounded in fp32 and rounded to e4m3 once (ties to even).  NaN in
// a block makes amax, hence the whole block, NaN; an infinity makes scale
// infinite, its own value NaN and the others 0.  The floor 2^-100 keeps the
// reciprocal finite: blocks below it (zeros above all) give q = 0 or values
// that small a scale can hold.
//
// All of them read each input once and write each output once, so the bound
// is HBM; sums and statistics are fp32.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "llvq_b200.h"
#include "llvq_internal.h"

namespace llvq {

namespace {

constexpr int kVec = 8;                          // elements a thread handles at a time
constexpr int kGroup = kFp8Block / kVec;         // 16 threads share one block of 128 columns
constexpr float kE4m3Max = 448.f;
constexpr float kAmaxFloor = 0x1p-100f;

template <typename T>
__device__ __forceinline__ float to_float(T v) {
  if constexpr (sizeof(T) == 4) return v;
  else return static_cast<float>(v);
}

template <typename T>
__device__ __forceinline__ T from_float(float v) {
  if constexpr (sizeof(T) == 4) return v;
  else if constexpr (std::is_same_v<T, __half>) return __float2half_rn(v);
  else return __float2bfloat16_rn(v);
}

// Eight elements as they lie in memory.
template <typename T>
struct alignas(16) Raw {
  T v[kVec];
};

// kAligned: every full group of eight starts on a 16-byte boundary.
template <typename T, bool kAligned>
__device__ __forceinline__ Raw<T> load8(const T* p, int valid) {
  Raw<T> r;
  if (kAligned && valid >= kVec) {
    const uint4* s = reinterpret_cast<const uint4*>(p);
    uint4* d = reinterpret_cast<uint4*>(&r);
#pragma unroll
    for (int i = 0; i < (int)(sizeof(r) / 16); ++i) d[i] = __ldg(s + i);
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i) r.v[i] = i < valid ? p[i] : from_float<T>(0.f);
  }
  return r;
}

template <typename T, bool kAligned>
__device__ __forceinline__ void store8(T* p, const Raw<T>& r, int valid) {
  if (kAligned && valid >= kVec) {
    uint4* d = reinterpret_cast<uint4*>(p);
    const uint4* s = reinterpret_cast<const uint4*>(&r);
#pragma unroll
    for (int i = 0; i < (int)(sizeof(r) / 16); ++i) d[i] = s[i];
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      if (i < valid) p[i] = r.v[i];
  }
}

// max |.| that keeps NaN (fmaxf would drop it).
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ float amax8(const float (&v)[kVec]) {
  float m = fabsf(v[0]);
#pragma unroll
  for (int i = 1; i < kVec; ++i) m = max_nan(m, fabsf(v[i]));
  return m;
}

// Largest of the 16 threads that share a block (a half warp).
__device__ __forceinline__ float group_max(float m) {
#pragma unroll
  for (int o = kGroup / 2; o; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}

// 448 v / amax correctly rounded, from the reciprocal r = RN(1 / amax) and one
// residual step (Markstein 1990: q0 = z r, q = q0 + (z - q0 amax) r).  The
// multiplier 448 and amax are both taken times 2^-64 where 448 amax could
// overflow; an infinite amax gives 0 for finite values and NaN for infinite ones.
struct Quotient {
  float mul, d, r, scale;
  __device__ __forceinline__ explicit Quotient(float amax) {
    amax = max_nan(amax, kAmaxFloor);
    scale = __fdiv_rn(amax, kE4m3Max);
    const bool big = amax > 0x1p100f;
    mul = big ? kE4m3Max * 0x1p-64f : kE4m3Max;
    d = big ? amax * 0x1p-64f : amax;
    r = __frcp_rn(d);
    if (isinf(amax)) d = 0.f;
  }
  __device__ __forceinline__ float operator()(float v) const {
    const float z = v * mul, q = z * r;
    return fmaf(fmaf(-q, d, z), r, q);
  }
};

// Two e4m3 bytes, lo in the low one.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ void store_q8(uint8_t* p, const float (&v)[kVec], const Quotient& quo, int valid) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    w[i] = e4m3x2(quo(v[4 * i]), quo(v[4 * i + 1])) | e4m3x2(quo(v[4 * i + 2]), quo(v[4 * i + 3])) << 16;
  if (valid >= kVec) {
    *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      if (i < valid) p[i] = (uint8_t)(w[i >> 2] >> (8 * (i & 3)));
  }
}

__device__ __forceinline__ int valid_of(int64_t cols, int64_t c) {
  const int64_t left = cols - c;
  return left >= kVec ? kVec : left > 0 ? (int)left : 0;
}

// ---------------------------------------------------------------- rows
// One half warp per (row, block of 128 columns): a thread's eight elements
// are 16 bytes of a 16-bit input, and consecutive half warps read consecutive
// blocks, so every access is whole lines.  kGated: y = gate / (1 + exp(-gate)) * up.
constexpr int kRowThreads = 256;

template <typename T, bool kGated, bool kAligned>
__global__ void __launch_bounds__(kRowThreads) rows_kernel(const T* __restrict__ x, int64_t ldx,
                                                           const T* __restrict__ up, int64_t ldu, uint32_t units,
                                                           uint32_t blocks, int64_t cols, Fp8Out out) {
  const uint32_t u = blockIdx.x * (kRowThreads / kGroup) + threadIdx.x / kGroup;
  const bool live = u < units;  // no early return: the whole warp meets in the shuffles
  const uint32_t row = live ? u / blocks : 0, b = live ? u % blocks : 0;
  const int64_t c = (int64_t)b * kFp8Block + (threadIdx.x % kGroup) * kVec;
  const int valid = live ? valid_of(cols, c) : 0;
  const Raw<T> rx = load8<T, kAligned>(x + row * ldx + c, valid);
  float v[kVec];
  if constexpr (kGated) {
    const Raw<T> ru = load8<T, kAligned>(up + row * ldu + c, valid);
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const float g = to_float(rx.v[i]);
      v[i] = __fdiv_rn(g, 1.f + expf(-g)) * to_float(ru.v[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i) v[i] = to_float(rx.v[i]);
  }
  const Quotient quo(group_max(amax8(v)));
  if (!live) return;
  store_q8(out.q + row * out.ld + c, v, quo, valid);
  if (threadIdx.x % kGroup == 0) out.scale[row * out.scale_row + b * out.scale_col] = quo.scale;
}

// ---------------------------------------------------------------- 128 x 128 blocks
// One CTA per block: 256 threads hold its 16,384 values in registers (64 per
// thread, as they lie in memory) between the maximum and the store.
constexpr int kBlockThreads = 256;
constexpr int kBlockRowsPass = kBlockThreads / kGroup;       // 16 rows a pass
constexpr int kBlockPasses = kFp8Block / kBlockRowsPass;     // 8

template <typename T, bool kAligned>
__global__ void __launch_bounds__(kBlockThreads) blocks_kernel(const T* __restrict__ x, int64_t ldx, int64_t rows,
                                                               int64_t cols, uint32_t col_blocks, Fp8Out out) {
  __shared__ float red[kBlockThreads / 32];
  const uint32_t rb = blockIdx.x / col_blocks, cb = blockIdx.x % col_blocks;
  const int64_t c = (int64_t)cb * kFp8Block + (threadIdx.x % kGroup) * kVec;
  const int64_t r0 = (int64_t)rb * kFp8Block + threadIdx.x / kGroup;
  const int valid = valid_of(cols, c);
  Raw<T> raw[kBlockPasses];
#pragma unroll
  for (int p = 0; p < kBlockPasses; ++p) {
    const int64_t r = r0 + p * kBlockRowsPass;
    raw[p] = load8<T, kAligned>(x + (r < rows ? r * ldx + c : 0), r < rows ? valid : 0);
  }
  float m = 0.f;
#pragma unroll
  for (int p = 0; p < kBlockPasses; ++p) {
    float v[kVec];
#pragma unroll
    for (int i = 0; i < kVec; ++i) v[i] = to_float(raw[p].v[i]);
    m = max_nan(m, amax8(v));
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kBlockThreads / 32; ++w) m = max_nan(m, red[w]);
  const Quotient quo(m);
#pragma unroll
  for (int p = 0; p < kBlockPasses; ++p) {
    const int64_t r = r0 + p * kBlockRowsPass;
    if (r < rows) {
      float v[kVec];
#pragma unroll
      for (int i = 0; i < kVec; ++i) v[i] = to_float(raw[p].v[i]);
      store_q8(out.q + r * out.ld + c, v, quo, valid);
    }
  }
  if (threadIdx.x == 0) out.scale[rb * out.scale_row + cb * out.scale_col] = quo.scale;
}

// ---------------------------------------------------------------- RMS norm
// One CTA per row; the row stays in registers (kChunks groups of eight per
// thread) between the sum of squares and the 8-bit store:
//   h = x + residual (fp32; hidden = h rounded once)    y = h rsqrt(mean h^2 + eps) weight
// The norm uses the unrounded sum h.  Threads past the row hold zeros.
// One chunk up to 512 threads, more chunks up to 1024 (64 registers each).
template <int kChunks>
constexpr int kNormThreads = kChunks == 1 ? 512 : 1024;

template <typename T, typename W, int kChunks, bool kResidual, bool kAligned>
__global__ void __launch_bounds__(kNormThreads<kChunks>) rms_norm_kernel(const T* __restrict__ x, int64_t ldx, const T* __restrict__ residual, int64_t ldr,
                                const W* __restrict__ weight, float eps, int64_t cols, T* __restrict__ hidden,
                                int64_t ldh, Fp8Out out) {
  __shared__ float red[32];
  const int64_t row = blockIdx.x;
  float h[kChunks][kVec];
  Raw<T> rx[kChunks], rr[kChunks];
  Raw<W> rw[kChunks];
#pragma unroll
  for (int j = 0; j < kChunks; ++j) {
    const int64_t c = ((int64_t)j * blockDim.x + threadIdx.x) * kVec;
    const int valid = valid_of(cols, c);
    rx[j] = load8<T, kAligned>(x + row * ldx + c, valid);
    if constexpr (kResidual) rr[j] = load8<T, kAligned>(residual + row * ldr + c, valid);
    rw[j] = load8<W, kAligned>(weight + c, valid);
  }
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < kChunks; ++j) {
    const int64_t c = ((int64_t)j * blockDim.x + threadIdx.x) * kVec;
    Raw<T> rh;
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      h[j][i] = to_float(rx[j].v[i]);
      if constexpr (kResidual) {
        h[j][i] += to_float(rr[j].v[i]);
        rh.v[i] = from_float<T>(h[j][i]);
      }
      ss = fmaf(h[j][i], h[j][i], ss);
    }
    if constexpr (kResidual) store8<T, kAligned>(hidden + row * ldh + c, rh, valid_of(cols, c));
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = ss;
  __syncthreads();
  float total = 0.f;
  for (unsigned w = 0; w < blockDim.x / 32; ++w) total += red[w];
  const float rstd = __fdiv_rn(1.f, __fsqrt_rn(__fdiv_rn(total, (float)cols) + eps));
#pragma unroll
  for (int j = 0; j < kChunks; ++j) {
    const int64_t c = ((int64_t)j * blockDim.x + threadIdx.x) * kVec;
    const int valid = valid_of(cols, c);
    float y[kVec];
#pragma unroll
    for (int i = 0; i < kVec; ++i) y[i] = valid > i ? h[j][i] * rstd * to_float(rw[j].v[i]) : 0.f;
    const Quotient quo(group_max(amax8(y)));
    store_q8(out.q + row * out.ld + c, y, quo, valid);
    if (threadIdx.x % kGroup == 0 && valid > 0)
      out.scale[row * out.scale_row + c / kFp8Block * out.scale_col] = quo.scale;
  }
}

template <typename T>
bool aligned16(const void* p, int64_t ld) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * (int64_t)sizeof(T) % 16 == 0;
}

template <typename T, bool kGated>
cudaError_t rows_typed(Fp8In x, Fp8In up, int64_t rows, int64_t cols, Fp8Out out, cudaStream_t stream) {
  const int64_t blocks = (cols + kFp8Block - 1) / kFp8Block, units = rows * blocks;
  if (units > 0xFFFFFFF0LL) return cudaErrorInvalidValue;
  const int64_t grid = (units + kRowThreads / kGroup - 1) / (kRowThreads / kGroup);
  const T *px = static_cast<const T*>(x.ptr), *pu = static_cast<const T*>(up.ptr);
  const bool ok = aligned16<T>(px, x.ld) && (!kGated || aligned16<T>(pu, up.ld));
  if (ok)
    rows_kernel<T, kGated, true><<<(unsigned)grid, kRowThreads, 0, stream>>>(px, x.ld, pu, up.ld, (uint32_t)units,
                                                                             (uint32_t)blocks, cols, out);
  else
    rows_kernel<T, kGated, false><<<(unsigned)grid, kRowThreads, 0, stream>>>(px, x.ld, pu, up.ld, (uint32_t)units,
                                                                              (uint32_t)blocks, cols, out);
  return cudaGetLastError();
}

template <typename T>
cudaError_t blocks_typed(Fp8In x, int64_t rows, int64_t cols, Fp8Out out, cudaStream_t stream) {
  const int64_t rb = (rows + kFp8Block - 1) / kFp8Block, cb = (cols + kFp8Block - 1) / kFp8Block;
  if (rb * cb > 0x7FFFFFFFLL) return cudaErrorInvalidValue;
  const T* px = static_cast<const T*>(x.ptr);
  if (aligned16<T>(px, x.ld))
    blocks_kernel<T, true><<<(unsigned)(rb * cb), kBlockThreads, 0, stream>>>(px, x.ld, rows, cols, (uint32_t)cb, out);
  else
    blocks_kernel<T, false><<<(unsigned)(rb * cb), kBlockThreads, 0, stream>>>(px, x.ld, rows, cols, (uint32_t)cb,
                                                                               out);
  return cudaGetLastError();
}

template <typename T, typename W, int kChunks>
cudaError_t norm_chunks(const T* x, int64_t ldx, const T* r, int64_t ldr, const W* w, float eps, int64_t rows,
                        int64_t cols, T* hidden, int64_t ldh, Fp8Out out, cudaStream_t stream) {
  const int64_t groups = (cols + kVec - 1) / kVec;
  const unsigned threads = (unsigned)(((groups + kChunks - 1) / kChunks + 31) / 32 * 32);
  const bool ok = aligned16<T>(x, ldx) && aligned16<W>(w, 0) &&
                  (!r || (aligned16<T>(r, ldr) && aligned16<T>(hidden, ldh)));
#define LLVQ_NORM(R, A) \
  rms_norm_kernel<T, W, kChunks, R, A><<<(unsigned)rows, threads, 0, stream>>>(x, ldx, r, ldr, w, eps, cols, hidden, \
                                                                              ldh, out)
  if (r) {
    if (ok) LLVQ_NORM(true, true);
    else LLVQ_NORM(true, false);
  } else {
    if (ok) LLVQ_NORM(false, true);
    else LLVQ_NORM(false, false);
  }
#undef LLVQ_NORM
  return cudaGetLastError();
}

template <typename T, typename W>
cudaError_t norm_typed(Fp8In x, Fp8In r, const void* w, float eps, int64_t rows, int64_t cols, void* hidden,
                       int64_t ldh, Fp8Out out, cudaStream_t stream) {
  const T *px = static_cast<const T*>(x.ptr), *pr = static_cast<const T*>(r.ptr);
  T* ph = static_cast<T*>(hidden);
  const W* pw = static_cast<const W*>(w);
  if (cols <= 512 * kVec)
    return norm_chunks<T, W, 1>(px, x.ld, pr, r.ld, pw, eps, rows, cols, ph, ldh, out, stream);
  if (cols <= 1024 * kVec * 2)
    return norm_chunks<T, W, 2>(px, x.ld, pr, r.ld, pw, eps, rows, cols, ph, ldh, out, stream);
  return norm_chunks<T, W, 4>(px, x.ld, pr, r.ld, pw, eps, rows, cols, ph, ldh, out, stream);
}

}  // namespace

cudaError_t fp8_quantize_launch(Fp8In x, int type, int64_t rows, int64_t cols, int block_rows, Fp8Out out,
                                cudaStream_t stream) {
  if (rows <= 0 || cols <= 0) return cudaSuccess;
  if (block_rows == 1) {
    if (type == LLVQ_DT_F32) return rows_typed<float, false>(x, Fp8In{}, rows, cols, out, stream);
    if (type == LLVQ_DT_F16) return rows_typed<__half, false>(x, Fp8In{}, rows, cols, out, stream);
    return rows_typed<__nv_bfloat16, false>(x, Fp8In{}, rows, cols, out, stream);
  }
  if (type == LLVQ_DT_F32) return blocks_typed<float>(x, rows, cols, out, stream);
  if (type == LLVQ_DT_F16) return blocks_typed<__half>(x, rows, cols, out, stream);
  return blocks_typed<__nv_bfloat16>(x, rows, cols, out, stream);
}

cudaError_t fp8_swiglu_launch(Fp8In gate, Fp8In up, int type, int64_t rows, int64_t cols, Fp8Out out,
                              cudaStream_t stream) {
  if (rows <= 0 || cols <= 0) return cudaSuccess;
  if (type == LLVQ_DT_F32) return rows_typed<float, true>(gate, up, rows, cols, out, stream);
  if (type == LLVQ_DT_F16) return rows_typed<__half, true>(gate, up, rows, cols, out, stream);
  return rows_typed<__nv_bfloat16, true>(gate, up, rows, cols, out, stream);
}

cudaError_t fp8_rms_norm_launch(Fp8In x, Fp8In residual, int type, const void* weight, int weight_type, float eps,
                                int64_t rows, int64_t cols, void* hidden, int64_t ld_hidden, Fp8Out out,
                                cudaStream_t stream) {
  if (rows <= 0 || cols <= 0) return cudaSuccess;
  if (cols > kFp8NormMaxCols || rows > 0x7FFFFFFFLL) return cudaErrorInvalidValue;
#define LLVQ_NORM(T, W) norm_typed<T, W>(x, residual, weight, eps, rows, cols, hidden, ld_hidden, out, stream)
  if (type == LLVQ_DT_F32) return LLVQ_NORM(float, float);
  if (type == LLVQ_DT_F16) return weight_type == LLVQ_DT_F32 ? LLVQ_NORM(__half, float) : LLVQ_NORM(__half, __half);
  return weight_type == LLVQ_DT_F32 ? LLVQ_NORM(__nv_bfloat16, float) : LLVQ_NORM(__nv_bfloat16, __nv_bfloat16);
#undef LLVQ_NORM
}

}  // namespace llvq
