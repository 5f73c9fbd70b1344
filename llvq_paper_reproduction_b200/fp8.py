"""8-bit products for large batches and the kernels that make their operands.

An 8-bit matrix is a pair (q, scale): q float8_e4m3fn [rows, cols], scale
fp32 per block of 128 columns, value = q * scale of its block.  Activations
have a scale per row ([rows, ceil(cols / 128)]), weights one per 128 x 128
block ([ceil(rows / 128), ceil(cols / 128)]); last blocks may be partial.
The operators' q have rows on 16-byte boundaries, from 1024 columns on whole
128-byte lines, so q is a view with gaps unless its columns are such a multiple.

    x, hidden     -> rms_norm       -> 8-bit x      (residual addition, norm)
    8-bit x, W    -> gemm           -> gate and up
    gate, up      -> swiglu         -> 8-bit activations
    any x         -> quantize_rows  -> 8-bit x
    weight        -> quantize_blocks (or LeechLatticeVectorQuantizerGpu.dequantize_fp8) -> 8-bit W

Every call is one kernel on torch's current stream of the inputs' device (one
more for each operand that has to be copied first), never synchronises, keeps
nothing between calls and may be captured in a CUDA graph; but the first
product on a device makes its error flag, which is kept: that call synchronises
once and is refused while a graph is captured.  Forward only: an input that
requires grad is refused while grad mode is on, one that carries a forward-mode
tangent while that mode is.  Checks, outputs and the call of the library are
one step of compiled code (``csrc/fp8_torch.cpp``), which a call on a few
tokens would otherwise spend most of its time on.  The reference has no 8-bit
path; there is no fallback to anything but the in-tree library.
"""
from __future__ import annotations

import ctypes
import importlib.machinery
import importlib.util
from pathlib import Path

import torch

from . import _native

BLOCK = 128
E4M3 = torch.float8_e4m3fn
NORM_MAX_COLS = 32768
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}  # LLVQ_DT_*
_EXT_PATH = Path(__file__).resolve().parent / "_lib" / "_fp8_torch.so"


def _load():
    if not _EXT_PATH.exists():
        raise ImportError(f"{_EXT_PATH} is missing: build it with `python -m llvq_paper_reproduction_b200.build`")
    lib = _native.load()
    loader = importlib.machinery.ExtensionFileLoader("_fp8_torch", str(_EXT_PATH))
    ext = importlib.util.module_from_spec(importlib.util.spec_from_loader("_fp8_torch", loader))
    loader.exec_module(ext)
    ext.bind(*(ctypes.cast(getattr(lib, name), ctypes.c_void_p).value
               for name in ("llvq_fp8_quantize", "llvq_fp8_swiglu", "llvq_fp8_rms_norm", "llvq_fp8_gemm",
                            "llvq_status_string", "llvq_last_error")))
    return ext


_ext = _load()


def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x [rows, cols] -> (q, scale [rows, ceil(cols / 128)]): per block of 128
    columns amax = max(2^-100, max |x|), scale = amax / 448 and
    q = e4m3(448 x / amax), rounded to nearest even: the right byte for every 16-bit
    x; of fp32 the quotient is rounded to fp32 first (within 2^-23).  NaN makes its block NaN;
    an infinity makes the block's scale infinite."""
    return _ext.quantize_rows(x)


def quantize_blocks(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """w [rows, cols] -> (q, scale [ceil(rows / 128), ceil(cols / 128)]): as
    ``quantize_rows``, with one scale per 128 x 128 block (weights, laid out once)."""
    return _ext.quantize_blocks(w)


def swiglu(gate: torch.Tensor, up: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """gate / (1 + exp(-gate)) * up in fp32, quantized as ``quantize_rows``;
    also for gates whose exponential fp32 cannot hold, down to -174 (0 below).
    gate and up [rows, cols] may be the halves of one product's rows
    (``y.chunk(2, dim=1)``): nothing is copied."""
    return _ext.swiglu(gate, up)


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5, residual: torch.Tensor | None = None):
    """h = x + residual, y = h * weight / sqrt(mean(h^2) + eps) per row in
    fp32, quantized as ``quantize_rows``.  Returns (q, scale), or with a
    residual (q, scale, hidden) where hidden = h rounded once to x's type (the
    next residual); the norm itself uses the unrounded h.  weight [cols] has
    x's type or fp32; at most 32,768 columns."""
    return _ext.rms_norm(x, weight, eps, residual)


def gemm(a: torch.Tensor, a_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
         out_dtype: torch.dtype = torch.bfloat16, check: bool = False) -> torch.Tensor:
    """``A @ W.T`` [m, n] for 8-bit activations (a [m, k], a_scale
    [m, ceil(k / 128)]) and an 8-bit weight (w [n, k], w_scale
    [ceil(n / 128), ceil(k / 128)]): the tensor cores sum each block of 128
    columns, the sums are scaled and added in fp32 and rounded once to
    out_dtype (bfloat16, float16 or float32).  One summation order per output,
    shape and GPU: the same bits on every call.  Scales may have any strides; 8-bit
    rows that do not start on 16-byte boundaries are copied.  Asynchronous: a
    tensor-core wait that timed out is counted in ``pending_errors``;
    ``check=True`` synchronises and raises RuntimeError at once (not while a
    graph is captured)."""
    dtype = _TYPES.get(out_dtype)
    if dtype is None:
        raise ValueError(f"out_dtype must be bfloat16, float16 or float32, got {out_dtype}")
    if check and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("check=True synchronises, which a capture cannot: capture without it, "
                           "call raise_pending_errors after a replay")
    index = a.get_device()
    flag = _flags.get(index) or _flag(index)
    y = _ext.gemm(a, a_scale, w, w_scale, dtype, flag[1])
    if check:
        raise_pending_errors(a.device)
    return y


# Sticky per-device flag of gemm, set when a tensor-core wait timed out: (tensor, address).
_flags: dict[int, tuple[torch.Tensor | None, int]] = {}


def _flag(index: int) -> tuple[torch.Tensor | None, int]:
    if index < 0:  # not a CUDA tensor: refused by the call
        return None, 0
    if torch.cuda.is_current_stream_capturing():
        # memory taken during a capture belongs to that graph
        raise RuntimeError("call fp8.gemm once on this device before capturing it in a CUDA graph")
    with torch.inference_mode(False):  # made by a first call inside, it is cleared outside
        f = torch.zeros((1,), dtype=torch.int32, device=torch.device("cuda", index))
    torch.cuda.synchronize(index)  # once: whichever stream sets it first
    return _flags.setdefault(index, (f, f.data_ptr()))


def pending_errors(device: str | torch.device = "cuda") -> dict:
    """Errors of the products the current stream has waited for, since the
    last reset (synchronises the host with the device)."""
    f = _flags.get(_index(device))
    return {"gemm_timeout": 0 if f is None else int(f[0].item())}


def raise_pending_errors(device: str | torch.device = "cuda") -> None:
    """Read and clear the flag of ``gemm``; raise RuntimeError if it was set."""
    if pending_errors(device)["gemm_timeout"]:
        _flags[_index(device)][0].zero_()
        raise RuntimeError("tensor-core wait timed out in the 8-bit product")


def _index(device: str | torch.device) -> int:
    device = torch.device(device)
    return torch.cuda.current_device() if device.index is None else device.index


__all__ = ["BLOCK", "E4M3", "NORM_MAX_COLS", "gemm", "pending_errors", "quantize_blocks", "quantize_rows",
           "raise_pending_errors", "rms_norm", "swiglu"]
