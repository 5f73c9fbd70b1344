"""8-bit products for large batches and the kernels that make their operands.

An 8-bit matrix is a pair (q, scale): q float8_e4m3fn [rows, cols], scale
fp32 per block of 128 columns, value = q * scale of its block.  Activations
have a scale per row ([rows, ceil(cols / 128)]), weights one per 128 x 128
block ([ceil(rows / 128), ceil(cols / 128)]); last blocks may be partial.

    x, hidden     -> rms_norm       -> 8-bit x      (residual addition, norm)
    8-bit x, W    -> gemm           -> gate and up
    gate, up      -> swiglu         -> 8-bit activations
    any x         -> quantize_rows  -> 8-bit x
    weight        -> quantize_blocks (or LeechLatticeVectorQuantizerGpu.dequantize_fp8) -> 8-bit W

Every call is one kernel on torch's current stream of the inputs' device,
never synchronises, keeps nothing between calls and may be captured in a CUDA
graph.  Forward only: an input that requires grad is refused while grad mode
is on.  The reference has no 8-bit path; there is no fallback to anything but
the in-tree library.
"""
from __future__ import annotations

import torch

from . import _native

BLOCK = 128
E4M3 = torch.float8_e4m3fn
NORM_MAX_COLS = 32768
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}  # LLVQ_DT_*


_raw_stream = torch._C._cuda_getCurrentRawStream  # current_stream().cuda_stream without building a Stream (3 us)
_empty = torch.empty_strided  # the shortest way to a tensor of given strides


def _launch(fn, device: torch.device, *args) -> None:
    """fn(*args, stream) on the current stream of `device`."""
    index = device.index
    if index == torch.cuda.current_device():
        fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(device):
            fn(*args, _raw_stream(index))


def _input(x: torch.Tensor, name: str) -> torch.Tensor:
    """A 2-D CUDA matrix of a supported type whose rows are dense."""
    if not x.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if x.dtype not in _TYPES:
        raise ValueError(f"{name} must be bfloat16, float16 or float32, got {x.dtype}")
    if x.dim() != 2:
        raise ValueError(f"{name} must have two dimensions, got {x.dim()}")
    if x.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires grad: the 8-bit operators are forward only (use torch.no_grad)")
    return x if x.stride(1) == 1 or x.shape[1] <= 1 else x.contiguous()


def _same(x: torch.Tensor, like: torch.Tensor, name: str) -> None:
    if x.shape != like.shape or x.dtype != like.dtype or x.device != like.device:
        raise ValueError(f"{name} must match the input: {tuple(like.shape)} {like.dtype} on {like.device}, "
                         f"got {tuple(x.shape)} {x.dtype} on {x.device}")


def _blocks(n: int) -> int:
    return (n + BLOCK - 1) // BLOCK


def _empty_e4m3(rows: int, cols: int, device: torch.device) -> tuple[torch.Tensor, int]:
    """Rows that start on 16-byte boundaries, as the product reads them, and their stride."""
    ld = (cols + 15) // 16 * 16
    return _empty((rows, cols), (ld, 1), dtype=E4M3, device=device), ld


def _empty_rows(rows: int, cols: int, device: torch.device) -> tuple[torch.Tensor, int, torch.Tensor]:
    """8-bit activations; their scales lie block by block (row fastest), as the product's warps read them."""
    q, ld = _empty_e4m3(rows, cols, device)
    return q, ld, _empty((rows, _blocks(cols)), (1, rows), dtype=torch.float32, device=device)


def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x [rows, cols] -> (q, scale [rows, ceil(cols / 128)]): per block of 128
    columns amax = max(2^-100, max |x|), scale = amax / 448 and
    q = e4m3(448 x / amax), rounded to nearest even.  NaN makes its block NaN;
    an infinity makes the block's scale infinite."""
    x = _input(x, "x")
    m, k = x.shape
    device = x.device
    q, ldq, scale = _empty_rows(m, k, device)
    _launch(_native.fp8_quantize, device, x.data_ptr(), _TYPES[x.dtype], x.stride(0), m, k, 1, q.data_ptr(), ldq,
            scale.data_ptr(), 1, m)
    return q, scale


def quantize_blocks(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """w [rows, cols] -> (q, scale [ceil(rows / 128), ceil(cols / 128)]): as
    ``quantize_rows``, with one scale per 128 x 128 block (weights, laid out once)."""
    w = _input(w, "w")
    n, k = w.shape
    device, kb = w.device, _blocks(k)
    q, ldq = _empty_e4m3(n, k, device)
    scale = _empty((_blocks(n), kb), (kb, 1), dtype=torch.float32, device=device)
    _launch(_native.fp8_quantize, device, w.data_ptr(), _TYPES[w.dtype], w.stride(0), n, k, BLOCK, q.data_ptr(), ldq,
            scale.data_ptr(), kb, 1)
    return q, scale


def swiglu(gate: torch.Tensor, up: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """gate / (1 + exp(-gate)) * up in fp32, quantized as ``quantize_rows``.
    gate and up [rows, cols] may be the halves of one product's rows
    (``y.chunk(2, dim=1)``): nothing is copied."""
    gate, up = _input(gate, "gate"), _input(up, "up")
    _same(up, gate, "up")
    m, k = gate.shape
    device = gate.device
    q, ldq, scale = _empty_rows(m, k, device)
    _launch(_native.fp8_swiglu, device, gate.data_ptr(), gate.stride(0), up.data_ptr(), up.stride(0),
            _TYPES[gate.dtype], m, k, q.data_ptr(), ldq, scale.data_ptr(), 1, m)
    return q, scale


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5, residual: torch.Tensor | None = None):
    """h = x + residual, y = h * weight / sqrt(mean(h^2) + eps) per row in
    fp32, quantized as ``quantize_rows``.  Returns (q, scale), or with a
    residual (q, scale, hidden) where hidden = h rounded once to x's type (the
    next residual); the norm itself uses the unrounded h.  weight [cols] has
    x's type or fp32; at most 32,768 columns."""
    x = _input(x, "x")
    m, k = x.shape
    device, dtype = x.device, x.dtype
    if weight.shape != (k,) or weight.device != device or weight.dtype not in (dtype, torch.float32):
        raise ValueError(f"weight must be [{k}] of {dtype} or float32 on {device}")
    if weight.requires_grad and torch.is_grad_enabled():
        raise ValueError("weight requires grad: the 8-bit operators are forward only (use torch.no_grad)")
    if k > NORM_MAX_COLS:
        raise ValueError(f"rms_norm takes at most {NORM_MAX_COLS} columns, got {k}")
    if not weight.is_contiguous():
        weight = weight.contiguous()
    q, ldq, scale = _empty_rows(m, k, device)
    args = (_TYPES[dtype], weight.data_ptr(), _TYPES[weight.dtype], eps, m, k)
    if residual is None:
        _launch(_native.fp8_rms_norm, device, x.data_ptr(), x.stride(0), 0, 0, *args, 0, k, q.data_ptr(), ldq,
                scale.data_ptr(), 1, m)
        return q, scale
    residual = _input(residual, "residual")
    _same(residual, x, "residual")
    hidden = _empty((m, k), (k, 1), dtype=dtype, device=device)
    _launch(_native.fp8_rms_norm, device, x.data_ptr(), x.stride(0), residual.data_ptr(), residual.stride(0), *args,
            hidden.data_ptr(), k, q.data_ptr(), ldq, scale.data_ptr(), 1, m)
    return q, scale, hidden


def _operand(q: torch.Tensor, name: str) -> tuple[torch.Tensor, int]:
    """An e4m3 operand whose rows start on 16-byte boundaries, and its row
    stride; others (none that this module made) are copied."""
    if not q.is_cuda or q.dtype != E4M3 or q.dim() != 2:
        raise ValueError(f"{name} must be a float8_e4m3fn CUDA matrix")
    rows, cols = q.shape
    if q.data_ptr() % 16 == 0 and (q.stride(1) == 1 or cols <= 1):
        if rows <= 1:
            return q, (cols + 15) // 16 * 16
        if q.stride(0) % 16 == 0 and q.stride(0) >= cols:
            return q, q.stride(0)
    copy, ld = _empty_e4m3(rows, cols, q.device)
    copy.view(torch.uint8).copy_(q.view(torch.uint8))
    return copy, ld


def _scales(s: torch.Tensor, rows: int, blocks: int, device: torch.device, name: str) -> tuple[int, int, int]:
    if s.dtype != torch.float32 or s.shape != (rows, blocks) or s.device != device:
        raise ValueError(f"{name} must be float32 [{rows}, {blocks}] on {device}, got {s.dtype} {tuple(s.shape)} on "
                         f"{s.device}")
    if s.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires grad: the 8-bit operators are forward only (use torch.no_grad)")
    return s.data_ptr(), *s.stride()


def gemm(a: torch.Tensor, a_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
         out_dtype: torch.dtype = torch.bfloat16, check: bool = False) -> torch.Tensor:
    """``A @ W.T`` [m, n] for 8-bit activations (a [m, k], a_scale
    [m, ceil(k / 128)]) and an 8-bit weight (w [n, k], w_scale
    [ceil(n / 128), ceil(k / 128)]): the tensor cores sum each block of 128
    columns, the sums are scaled and added in fp32 and rounded once to
    out_dtype (bfloat16, float16 or float32).  One summation order per output:
    the same bits on every call.  Scales may have any strides.  Asynchronous:
    a tensor-core wait that timed out is counted in ``pending_errors``;
    ``check=True`` synchronises and raises RuntimeError at once."""
    if out_dtype not in _TYPES:
        raise ValueError(f"out_dtype must be bfloat16, float16 or float32, got {out_dtype}")
    a, lda = _operand(a, "a")
    w, ldw = _operand(w, "w")
    (m, k), (n, kw) = a.shape, w.shape
    if k != kw:
        raise ValueError(f"a has {k} columns, w has {kw}")
    device, kb = a.device, _blocks(k)
    if w.device != device:
        raise ValueError(f"a is on {device}, w on {w.device}")
    a_s, w_s = _scales(a_scale, m, kb, device, "a_scale"), _scales(w_scale, _blocks(n), kb, device, "w_scale")
    y = _empty((m, n), (n, 1), dtype=out_dtype, device=device)
    flag = _flags.get(device.index)
    _launch(_native.fp8_gemm, device, a.data_ptr(), lda, *a_s, w.data_ptr(), ldw, *w_s, m, n, k, y.data_ptr(), n,
            _TYPES[out_dtype], (_flag(device) if flag is None else flag).data_ptr())
    if check:
        raise_pending_errors(device)
    return y


# Sticky per-device flag of gemm: set when a tensor-core wait timed out.
_flags: dict[int, torch.Tensor] = {}


def _flag(device: torch.device) -> torch.Tensor:
    if torch.cuda.is_current_stream_capturing():
        # memory taken during a capture belongs to that graph
        raise RuntimeError("call fp8.gemm once on this device before capturing it in a CUDA graph")
    return _flags.setdefault(device.index, torch.zeros((1,), dtype=torch.int32, device=device))


def pending_errors(device: str | torch.device = "cuda") -> dict:
    """Errors of the products the current stream has waited for, since the
    last reset (synchronises the host with the device)."""
    device = torch.device(device)
    index = torch.cuda.current_device() if device.index is None else device.index
    f = _flags.get(index)
    return {"gemm_timeout": 0 if f is None else int(f.item())}


def raise_pending_errors(device: str | torch.device = "cuda") -> None:
    """Read and clear the flag of ``gemm``; raise RuntimeError if it was set."""
    device = torch.device(device)
    index = torch.cuda.current_device() if device.index is None else device.index
    if pending_errors(device)["gemm_timeout"]:
        _flags[index].zero_()
        raise RuntimeError("tensor-core wait timed out in the 8-bit product")


__all__ = ["BLOCK", "E4M3", "NORM_MAX_COLS", "gemm", "pending_errors", "quantize_blocks", "quantize_rows",
           "raise_pending_errors", "rms_norm", "swiglu"]
