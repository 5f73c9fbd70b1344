// C entry points of the 8-bit operators (include/llvq_b200.h): argument
// checks, then the launchers of fp8_quant.cu and fp8_gemm.cu.
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "llvq_b200.h"
#include "llvq_internal.h"

using llvq::abi_cuda_error;
using llvq::abi_error;

namespace {

bool known_type(int32_t t) { return t == LLVQ_DT_F32 || t == LLVQ_DT_F16 || t == LLVQ_DT_BF16; }
bool on_boundary(const void* p, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
// Elements of a type lie on their own boundary (an access off it would fault).
bool elements_at(const void* p, int32_t type) { return on_boundary(p, type == LLVQ_DT_F32 ? 4 : 2); }
constexpr const char* kOffBoundary = "an address is off its elements' boundary";

// Outputs of a quantizer over [rows, cols].
const char* bad_out(const uint8_t* q, int64_t ldq, const float* scale, int64_t rows, int64_t cols) {
  if (rows == 0 || cols == 0) return nullptr;
  if (!q || !scale) return "null output";
  if (rows > llvq::kFp8MaxUnits / ((cols - 1) / llvq::kFp8Block + 1)) return "more than 2^32 - 2^16 blocks";
  if (!on_boundary(scale, 4)) return kOffBoundary;
  if (ldq < cols || ldq % 16 || !on_boundary(q, 16)) return "e4m3 rows must be 16-byte aligned (base and stride)";
  return nullptr;
}

}  // namespace

extern "C" {

int llvq_fp8_quantize(const void* x, int32_t x_type, int64_t ldx, int64_t rows, int64_t cols, int32_t block_rows,
                      uint8_t* q, int64_t ldq, float* scale, int64_t scale_row, int64_t scale_col, void* stream) {
  if (rows < 0 || cols < 0 || !known_type(x_type) || (block_rows != 1 && block_rows != 128) || (rows > 1 && ldx < 0))
    return abi_error(LLVQ_ERR_INVALID_ARGUMENT, "fp8_quantize: bad size, type or block (1 or 128 rows)");
  if (const char* why = bad_out(q, ldq, scale, rows, cols)) return abi_error(LLVQ_ERR_INVALID_ARGUMENT, why);
  if (rows > 0 && cols > 0 && !x) return abi_error(LLVQ_ERR_INVALID_ARGUMENT, "fp8_quantize: null input");
  if (!elements_at(x, x_type)) return abi_error(LLVQ_ERR_INVALID_ARGUMENT, kOffBoundary);
  const cudaError_t e = llvq::fp8_quantize_launch({x, ldx}, x_type, rows, cols, block_rows,
                                                  {q, ldq, scale, scale_row, scale_col}, (cudaStream_t)stream);
  return e == cudaSuccess ? LLVQ_OK : abi_cuda_error(e, "fp8_quantize launch");
}

int llvq_fp8_swiglu(const void* gate, int64_t ld_gate, const void* up, int64_t ld_up, int32_t type, int64_t rows,
                    int64_t cols, uint8_t* q, int64_t ldq, float* scale, int64_t scale_row, int64_t scale_col,
                    void* stream) {
  if (rows < 0 || cols < 0 || !known_type(type) || (rows > 1 && (ld_gate < 0 || ld_up < 0)))
    return abi_error(LLVQ_ERR_INVALID_ARGUMENT, "fp8_swiglu: bad size or type");
  if (const char* why = bad_out(q, ldq, scale, rows, cols)) return abi_error(LLVQ_ERR_INVALID_ARGUMENT, why);
  if (rows > 0 && cols > 0 && (!gate || !up)) return abi_error(LLVQ_ERR_INVALID_ARGUMENT, "fp8_swiglu: null input");
  if (!elements_at(gate, type) || !elements_at(up, type)) return abi_error(LLVQ_ERR_INVALID_ARGUMENT, kOffBoundary);
  const cudaError_t e = llvq::fp8_swiglu_launch({gate, ld_gate}, {up, ld_up}, type, rows, cols,
                                                {q, ldq, scale, scale_row, scale_col}, (cudaStream_t)stream);
  return e == cudaSuccess ? LLVQ_OK : abi_cuda_error(e, "fp8_swiglu launch");
}

int llvq_fp8_rms_norm(const void* x, int64_t ldx, const void* residual, int64_t ld_residual, int32_t type,
                      const void* weight, int32_t weight_type, float eps, int64_t rows, int64_t cols, void* hidden,
                      int64_t ld_hidden, uint8_t* q, int64_t ldq, float* scale, int64_t scale_row, int64_t scale_col,
                      void* stream) {
  if (rows < 0 || cols < 0 || !known_type(type) || (weight_type != type && weight_type != LLVQ_DT_F32) ||
      (rows > 1 && (ldx < 0 || (residual && (ld_residual < 0 || ld_hidden < cols)))))
    return abi_error(LLVQ_ERR_INVALID_ARGUMENT,
                     "fp8_rms_norm: bad size or type (the weight has the input's type or fp32)");
  if (!std::isfinite(eps) || eps < 0.f)
    return abi_error(LLVQ_ERR_INVALID_ARGUMENT, "fp8_rms_norm: eps must be finite and not negative");
  if (cols > LLVQ_FP8_NORM_MAX_COLS)
    return abi_error(LLVQ_ERR_INVALID_ARGUMENT, "fp8_rms_norm: more than 32768 columns");
  if (const char* why = bad_out(q, ldq, scale, rows, cols)) return abi_error(LLVQ_ERR_INVALID_ARGUMENT, why);
  if (rows > 0 && cols > 0 && (!x || !weight || (!residual != !hidden)))
    return abi_error(LLVQ_ERR_INVALID_ARGUMENT, "fp8_rms_norm: null pointer (residual and hidden come together)");
  if (!elements_at(x, type) || !elements_at(residual, type) || !elements_at(hidden, type) ||
      !elements_at(weight, weight_type))
    return abi_error(LLVQ_ERR_INVALID_ARGUMENT, kOffBoundary);
  const cudaError_t e =
      llvq::fp8_rms_norm_launch({x, ldx}, {residual, ld_residual}, type, weight, weight_type, eps, rows, cols, hidden,
                                ld_hidden, {q, ldq, scale, scale_row, scale_col}, (cudaStream_t)stream);
  return e == cudaSuccess ? LLVQ_OK : abi_cuda_error(e, "fp8_rms_norm launch");
}

int llvq_fp8_gemm(const uint8_t* a, int64_t lda, const float* a_scale, int64_t a_scale_row, int64_t a_scale_col,
                  const uint8_t* w, int64_t ldw, const float* w_scale, int64_t w_scale_row, int64_t w_scale_col,
                  int64_t m, int64_t n, int64_t k, void* y, int64_t ldy, int32_t y_type, int32_t* error_flag,
                  void* stream) {
  // coordinates are 32-bit and run up to one tile past the matrix
  constexpr int64_t kMost = (1LL << 31) - 512;
  if (m < 0 || n < 0 || k < 0 || m > kMost || n > kMost || k > kMost || !known_type(y_type) || ldy < n)
    return abi_error(LLVQ_ERR_INVALID_ARGUMENT, "fp8_gemm: bad size, output type or output stride");
  if (m == 0 || n == 0) return LLVQ_OK;
  if (!y || (k > 0 && (!a || !w || !a_scale || !w_scale)))
    return abi_error(LLVQ_ERR_INVALID_ARGUMENT, "fp8_gemm: null pointer");
  if (k > 0 && (lda < k || ldw < k || lda % 16 || ldw % 16 || !on_boundary(a, 16) || !on_boundary(w, 16)))
    return abi_error(LLVQ_ERR_INVALID_ARGUMENT, "fp8_gemm: e4m3 rows must be 16-byte aligned (base and stride)");
  if (!elements_at(y, y_type) || !on_boundary(error_flag, 4) ||
      (k > 0 && (!on_boundary(a_scale, 4) || !on_boundary(w_scale, 4))))
    return abi_error(LLVQ_ERR_INVALID_ARGUMENT, kOffBoundary);
  const cudaError_t e =
      llvq::fp8_gemm_launch({a, lda, a_scale, a_scale_row, a_scale_col}, {w, ldw, w_scale, w_scale_row, w_scale_col},
                            m, n, k, y, ldy, y_type, error_flag, (cudaStream_t)stream);
  return e == cudaSuccess ? LLVQ_OK : abi_cuda_error(e, "fp8_gemm launch");
}

}  // extern "C"
