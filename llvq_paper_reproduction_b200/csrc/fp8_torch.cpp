// Tensor front end of the 8-bit operators: checks, outputs and the call of the
// C entry point in one step, for fp8.py.  A call on a few tokens is shorter
// than what Python spends on its checks, its output tensors and ctypes (15 us
// against 6 for the norm of one token), so this file does that part; the
// operators themselves are the C entry points of include/llvq_b200.h, whose
// addresses bind() receives from the library that _native.py loaded.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <string>

#include "llvq_b200.h"

namespace {

constexpr int64_t kBlock = 128;

// A Python exception to raise: type (borrowed) and message.
struct Raise {
  PyObject* type;
  std::string text;
};

[[noreturn]] void value_error(const std::string& text) { throw Raise{PyExc_ValueError, text}; }

struct Entries {
  decltype(&llvq_fp8_quantize) quantize = nullptr;
  decltype(&llvq_fp8_swiglu) swiglu = nullptr;
  decltype(&llvq_fp8_rms_norm) rms_norm = nullptr;
  decltype(&llvq_fp8_gemm) gemm = nullptr;
  decltype(&llvq_status_string) status_string = nullptr;
  decltype(&llvq_last_error) last_error = nullptr;
} g;

// The exception types of _native.check().
void check(int status, const char* what) {
  if (status == LLVQ_OK) return;
  const std::string text = std::string(what) + ": " + g.status_string(status) + ": " + g.last_error();
  if (status == LLVQ_ERR_INVALID_ARGUMENT || status == LLVQ_ERR_UNSUPPORTED) value_error(text);
  throw Raise{status == LLVQ_ERR_OUT_OF_MEMORY ? PyExc_MemoryError : PyExc_RuntimeError, text};
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) throw Raise{PyExc_TypeError, std::string(name) + " must be a tensor"};
  return THPVariable_Unpack(o);
}

int code_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return LLVQ_DT_F32;
    case at::kHalf: return LLVQ_DT_F16;
    case at::kBFloat16: return LLVQ_DT_BF16;
    default: return -1;
  }
}

void no_grad(const at::Tensor& x, const char* name) {
  if (x.requires_grad() && at::GradMode::is_enabled())
    value_error(std::string(name) + " requires grad: the 8-bit operators are forward only (use torch.no_grad)");
  if (c10::AutogradState::get_tls_state().get_fw_grad_mode() && x._fw_grad(/*level=*/0).defined())
    value_error(std::string(name) + " carries a tangent: the 8-bit operators have no derivatives (use unpack_dual)");
}

// A 2-D CUDA matrix of a supported type whose rows are dense and whose memory holds its values.
at::Tensor input(PyObject* o, const char* name) {
  const at::Tensor& x = tensor(o, name);
  if (!x.is_cuda()) value_error(std::string(name) + " must be a CUDA tensor");
  if (code_of(x.scalar_type()) < 0)
    value_error(std::string(name) + " must be bfloat16, float16 or float32, got " + c10::toString(x.scalar_type()));
  if (x.dim() != 2) value_error(std::string(name) + " must have two dimensions, got " + std::to_string(x.dim()));
  no_grad(x, name);
  const bool dense = x.stride(1) == 1 || x.size(1) <= 1;
  if (dense && !x.is_neg()) return x;
  const c10::cuda::CUDAGuard guard(x.device());
  return dense ? x.resolve_neg() : x.contiguous();
}

std::string describe(const at::Tensor& x) {
  std::string s = "[";
  for (int64_t i = 0; i < x.dim(); ++i) s += (i ? ", " : "") + std::to_string(x.size(i));
  return s + "] " + c10::toString(x.scalar_type()) + " on " + x.device().str();
}

void same(const at::Tensor& x, const at::Tensor& like, const char* name) {
  if (x.sizes() != like.sizes() || x.scalar_type() != like.scalar_type() || x.device() != like.device())
    value_error(std::string(name) + " must match the input: " + describe(like) + ", got " + describe(x));
}

int64_t blocks(int64_t n) { return (n + kBlock - 1) / kBlock; }
// Bytes from row to row of e4m3: whole lines where that adds an eighth at most, else
// the 16 bytes that the product needs.  (64 x 14336 x 4100: 15.4 us with rows of 4224
// bytes, 18.3 with 4112, whose 128-byte pieces touch five sectors instead of four.)
int64_t row_bytes(int64_t cols) { return cols >= 1024 ? (cols + 127) / 128 * 128 : (cols + 15) / 16 * 16; }

at::Tensor empty(at::IntArrayRef size, at::IntArrayRef stride, at::ScalarType type, at::Device device) {
  return at::Tensor(at::detail::empty_strided_cuda(size, stride, type, device));
}

// e4m3 rows as the product reads them.
at::Tensor empty_e4m3(int64_t rows, int64_t cols, at::Device device) {
  return empty({rows, cols}, {row_bytes(cols), 1}, at::kFloat8_e4m3fn, device);
}

// Scales of activations lie block by block (row fastest), as the product's warps read them.
at::Tensor empty_row_scales(int64_t rows, int64_t cols, at::Device device) {
  return empty({rows, blocks(cols)}, {1, rows}, at::kFloat, device);
}

uint8_t* bytes(const at::Tensor& q) { return static_cast<uint8_t*>(q.data_ptr()); }
float* floats(const at::Tensor& s) { return static_cast<float*>(s.data_ptr()); }
void* stream(at::Device device) { return c10::cuda::getCurrentCUDAStream(device.index()).stream(); }

PyObject* tuple(std::initializer_list<at::Tensor> out) {
  PyObject* t = PyTuple_New((Py_ssize_t)out.size());
  if (!t) return nullptr;
  Py_ssize_t i = 0;
  for (const at::Tensor& x : out) {
    PyObject* o = THPVariable_Wrap(x);
    if (!o) {
      Py_DECREF(t);
      return nullptr;
    }
    PyTuple_SET_ITEM(t, i++, o);
  }
  return t;
}

// Runs f, turning C++ exceptions into Python's: none may leave a C entry.
template <typename F>
PyObject* guarded(F f) {
  try {
    return f();
  } catch (const Raise& r) {
    PyErr_SetString(r.type, r.text.c_str());
  } catch (const c10::OutOfMemoryError& e) {
    PyObject* torch = PyImport_ImportModule("torch");
    PyObject* type = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
    if (!type) PyErr_Clear();
    PyErr_SetString(type ? type : PyExc_MemoryError, e.what());
    Py_XDECREF(type);
    Py_XDECREF(torch);
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

bool count_is(Py_ssize_t n, Py_ssize_t want) {
  if (n == want) return true;
  PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, n);
  return false;
}

// bind(quantize, swiglu, rms_norm, gemm, status_string, last_error): addresses.
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (!count_is(n, 6)) return nullptr;
  void* p[6];
  for (int i = 0; i < 6; ++i) {
    p[i] = PyLong_AsVoidPtr(args[i]);
    if (PyErr_Occurred()) return nullptr;
  }
  g.quantize = reinterpret_cast<decltype(g.quantize)>(p[0]);
  g.swiglu = reinterpret_cast<decltype(g.swiglu)>(p[1]);
  g.rms_norm = reinterpret_cast<decltype(g.rms_norm)>(p[2]);
  g.gemm = reinterpret_cast<decltype(g.gemm)>(p[3]);
  g.status_string = reinterpret_cast<decltype(g.status_string)>(p[4]);
  g.last_error = reinterpret_cast<decltype(g.last_error)>(p[5]);
  Py_RETURN_NONE;
}

// quantize_rows(x), quantize_blocks(w)
template <bool kRows>
PyObject* quantize(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (!count_is(n, 1)) return nullptr;
  return guarded([&] {
    const at::Tensor x = input(args[0], kRows ? "x" : "w");
    const int64_t m = x.size(0), k = x.size(1), kb = blocks(k);
    const c10::cuda::CUDAGuard guard(x.device());
    const at::Tensor q = empty_e4m3(m, k, x.device());
    const at::Tensor scale = kRows ? empty_row_scales(m, k, x.device())
                                   : empty({blocks(m), kb}, {kb, 1}, at::kFloat, x.device());
    check(g.quantize(x.data_ptr(), code_of(x.scalar_type()), x.stride(0), m, k, kRows ? 1 : kBlock, bytes(q),
                     row_bytes(k), floats(scale), kRows ? 1 : kb, kRows ? m : 1, stream(x.device())),
          "llvq_fp8_quantize");
    return tuple({q, scale});
  });
}

// swiglu(gate, up)
PyObject* swiglu(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (!count_is(n, 2)) return nullptr;
  return guarded([&] {
    const at::Tensor gate = input(args[0], "gate"), up = input(args[1], "up");
    same(up, gate, "up");
    const int64_t m = gate.size(0), k = gate.size(1);
    const c10::cuda::CUDAGuard guard(gate.device());
    const at::Tensor q = empty_e4m3(m, k, gate.device()), scale = empty_row_scales(m, k, gate.device());
    check(g.swiglu(gate.data_ptr(), gate.stride(0), up.data_ptr(), up.stride(0), code_of(gate.scalar_type()), m, k,
                   bytes(q), row_bytes(k), floats(scale), 1, m, stream(gate.device())),
          "llvq_fp8_swiglu");
    return tuple({q, scale});
  });
}

// rms_norm(x, weight, eps, residual or None)
PyObject* rms_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (!count_is(n, 4)) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor x = input(args[0], "x");
    at::Tensor weight = tensor(args[1], "weight"), residual, hidden;
    const double eps = PyFloat_AsDouble(args[2]);
    if (PyErr_Occurred()) return nullptr;
    const int64_t m = x.size(0), k = x.size(1);
    const at::Device device = x.device();
    if (weight.dim() != 1 || weight.size(0) != k || weight.device() != device ||
        (weight.scalar_type() != x.scalar_type() && weight.scalar_type() != at::kFloat))
      value_error("weight must be [" + std::to_string(k) + "] of " + c10::toString(x.scalar_type()) +
                  " or Float on " + device.str() + ", got " + describe(weight));
    no_grad(weight, "weight");
    if (k > LLVQ_FP8_NORM_MAX_COLS)
      value_error("rms_norm takes at most " + std::to_string(LLVQ_FP8_NORM_MAX_COLS) + " columns, got " +
                  std::to_string(k));
    const bool with = args[3] != Py_None;
    if (with) {
      residual = input(args[3], "residual");
      same(residual, x, "residual");
    }
    const c10::cuda::CUDAGuard guard(device);
    if (!weight.is_contiguous()) weight = weight.contiguous();
    if (weight.is_neg()) weight = weight.resolve_neg();
    const at::Tensor q = empty_e4m3(m, k, device), scale = empty_row_scales(m, k, device);
    if (with) hidden = empty({m, k}, {k, 1}, x.scalar_type(), device);
    check(g.rms_norm(x.data_ptr(), x.stride(0), with ? residual.data_ptr() : nullptr, with ? residual.stride(0) : 0,
                     code_of(x.scalar_type()), weight.data_ptr(), code_of(weight.scalar_type()), (float)eps, m, k,
                     with ? hidden.data_ptr() : nullptr, k, bytes(q), row_bytes(k), floats(scale), 1, m,
                     stream(device)),
          "llvq_fp8_rms_norm");
    return with ? tuple({q, scale, hidden}) : tuple({q, scale});
  });
}

// An e4m3 operand whose rows start on 16-byte boundaries, and its row stride;
// others (none that the functions above made) are copied.
at::Tensor operand(PyObject* o, const char* name, int64_t* ld) {
  const at::Tensor& q = tensor(o, name);
  if (!q.is_cuda() || q.scalar_type() != at::kFloat8_e4m3fn || q.dim() != 2)
    value_error(std::string(name) + " must be a float8_e4m3fn CUDA matrix");
  if (q.is_neg()) value_error(std::string(name) + " is a view with the negative bit, which e4m3 memory has no form for");
  no_grad(q, name);
  const int64_t rows = q.size(0), cols = q.size(1);
  *ld = row_bytes(cols);
  if (reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0 && (q.stride(1) == 1 || cols <= 1)) {
    if (rows <= 1) return q;
    if (q.stride(0) % 16 == 0 && q.stride(0) >= cols) {
      *ld = q.stride(0);
      return q;
    }
  }
  const c10::cuda::CUDAGuard guard(q.device());
  at::Tensor copy = empty_e4m3(rows, cols, q.device());
  copy.view(at::kByte).copy_(q.view(at::kByte));
  return copy;
}

at::Tensor scales(PyObject* o, const char* name, int64_t rows, int64_t cols, at::Device device) {
  const at::Tensor& s = tensor(o, name);
  if (s.scalar_type() != at::kFloat || s.dim() != 2 || s.size(0) != rows || s.size(1) != cols || s.device() != device)
    value_error(std::string(name) + " must be [" + std::to_string(rows) + ", " + std::to_string(cols) +
                "] Float on " + device.str() + ", got " + describe(s));
  no_grad(s, name);
  if (!s.is_neg()) return s;
  const c10::cuda::CUDAGuard guard(device);
  return s.resolve_neg();
}

// gemm(a, a_scale, w, w_scale, type code of the output, address of the error flag)
PyObject* gemm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (!count_is(n, 6)) return nullptr;
  const long type = PyLong_AsLong(args[4]);
  void* flag = PyLong_AsVoidPtr(args[5]);
  if (PyErr_Occurred()) return nullptr;
  return guarded([&] {
    int64_t lda, ldw;
    const at::Tensor a = operand(args[0], "a", &lda), w = operand(args[2], "w", &ldw);
    const int64_t m = a.size(0), k = a.size(1), rows = w.size(0);
    const at::Device device = a.device();
    if (w.size(1) != k) value_error("a has " + std::to_string(k) + " columns, w has " + std::to_string(w.size(1)));
    if (w.device() != device) value_error("a is on " + device.str() + ", w on " + w.device().str());
    const at::Tensor sa = scales(args[1], "a_scale", m, blocks(k), device);
    const at::Tensor sw = scales(args[3], "w_scale", blocks(rows), blocks(k), device);
    const c10::cuda::CUDAGuard guard(device);
    const at::ScalarType out = type == LLVQ_DT_F32 ? at::kFloat : type == LLVQ_DT_F16 ? at::kHalf : at::kBFloat16;
    const at::Tensor y = empty({m, rows}, {rows, 1}, out, device);
    check(g.gemm(bytes(a), lda, floats(sa), sa.stride(0), sa.stride(1), bytes(w), ldw, floats(sw), sw.stride(0),
                 sw.stride(1), m, rows, k, y.data_ptr(), rows, (int32_t)type, static_cast<int32_t*>(flag),
                 stream(device)),
          "llvq_fp8_gemm");
    return THPVariable_Wrap(y);
  });
}

#define LLVQ_METHOD(name, f) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {LLVQ_METHOD("bind", bind),
                         LLVQ_METHOD("quantize_rows", quantize<true>),
                         LLVQ_METHOD("quantize_blocks", quantize<false>),
                         LLVQ_METHOD("swiglu", swiglu),
                         LLVQ_METHOD("rms_norm", rms_norm),
                         LLVQ_METHOD("gemm", gemm),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fp8_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fp8_torch(void) { return PyModule_Create(&module); }
