"""The 8-bit operators without a GPU: refusals of the Python and C entry
points (all before any launch), and the 64-bit reference the GPU tests use."""
from __future__ import annotations

import pytest
import torch

from fp8_reference import check_quantized, e4m3
from llvq_paper_reproduction_b200 import _native, fp8


def test_reference_rounding_matches_torch():
    v = torch.cat([torch.linspace(-448, 448, 20001), torch.linspace(-0.1, 0.1, 20001), torch.zeros(1)])
    assert torch.equal(e4m3(v.double()).float(), v.to(torch.float8_e4m3fn).float())


def test_reference_check_sees_a_wrong_value():
    x = torch.randn((5, 300), generator=torch.Generator().manual_seed(0), dtype=torch.float64)
    a = x.abs().max().item()
    x[:, 0] = x[:, 128] = x[:, 256] = a  # one scale for all blocks
    scale = torch.full((5, 3), a / 448.0, dtype=torch.float32)
    q = (x * 448.0 / a).to(torch.float8_e4m3fn)
    check_quantized(q, scale, x, 1, 0.0)
    byte = q.view(torch.uint8)
    byte[2, 200] ^= 1  # the neighbouring value
    with pytest.raises(AssertionError):
        check_quantized(q, scale, x, 1, 0.0)


@pytest.mark.parametrize("call", [
    lambda: fp8.quantize_rows(torch.zeros(2, 128)),
    lambda: fp8.quantize_blocks(torch.zeros(2, 128)),
    lambda: fp8.swiglu(torch.zeros(2, 128), torch.zeros(2, 128)),
    lambda: fp8.rms_norm(torch.zeros(2, 128), torch.zeros(128)),
    lambda: fp8.gemm(torch.zeros(2, 128).to(fp8.E4M3), torch.ones(2, 1), torch.zeros(4, 128).to(fp8.E4M3),
                     torch.ones(1, 1)),
    lambda: fp8.gemm(torch.zeros(2, 128).to(fp8.E4M3), torch.ones(2, 1), torch.zeros(4, 128).to(fp8.E4M3),
                     torch.ones(1, 1), out_dtype=torch.float64),
])
def test_python_refuses_host_tensors_and_types(call):
    with pytest.raises(ValueError):
        call()


P = 1 << 20  # an address that is never read: every call below is refused first


@pytest.mark.parametrize("call", [
    lambda: _native.fp8_quantize(P, 3, 128, 1, 128, 1, P, 128, P, 1, 1, 0),        # unknown type
    lambda: _native.fp8_quantize(P, 0, 128, -1, 128, 1, P, 128, P, 1, 1, 0),       # negative rows
    lambda: _native.fp8_quantize(P, 0, 128, 1, 128, 64, P, 128, P, 1, 1, 0),       # block of 64 rows
    lambda: _native.fp8_quantize(P, 0, 128, 1, 128, 1, P + 4, 128, P, 1, 1, 0),    # e4m3 base off its boundary
    lambda: _native.fp8_quantize(P, 0, 128, 2, 128, 1, P, 132, P, 1, 1, 0),        # e4m3 stride off its boundary
    lambda: _native.fp8_quantize(P, 0, 128, 2, 128, 1, P, 120, P, 1, 1, 0),        # e4m3 stride below the columns
    lambda: _native.fp8_quantize(0, 0, 128, 1, 128, 1, P, 128, P, 1, 1, 0),        # null input
    lambda: _native.fp8_quantize(P, 0, 128, 1, 128, 1, P, 128, 0, 1, 1, 0),        # null scale
    lambda: _native.fp8_quantize(P, 0, 1, 1 << 32, 1, 1, P, 16, P, 1, 1, 0),       # too many blocks
    lambda: _native.fp8_swiglu(P, 128, 0, 128, 0, 1, 128, P, 128, P, 1, 1, 0),     # null up
    lambda: _native.fp8_swiglu(P, 128, P, 128, 7, 1, 128, P, 128, P, 1, 1, 0),     # unknown type
    lambda: _native.fp8_rms_norm(P, 128, 0, 0, 1, P, 2, 1e-5, 1, 128, 0, 0, P, 128, P, 1, 1, 0),  # weight's type
    lambda: _native.fp8_rms_norm(P, 128, 0, 0, 1, P, 1, -1.0, 1, 128, 0, 0, P, 128, P, 1, 1, 0),  # negative eps
    lambda: _native.fp8_rms_norm(P, 128, 0, 0, 1, P, 1, float("nan"), 1, 128, 0, 0, P, 128, P, 1, 1, 0),
    lambda: _native.fp8_rms_norm(P, 128, P, 128, 1, P, 1, 1e-5, 1, 128, 0, 0, P, 128, P, 1, 1, 0),  # no hidden
    lambda: _native.fp8_rms_norm(P, 40000, 0, 0, 1, P, 1, 1e-5, 1, 40000, 0, 0, P, 40000, P, 1, 1, 0),  # too wide
    lambda: _native.fp8_gemm(P, 128, P, 1, 1, P, 128, P, 1, 1, 4, 4, 128, P, 4, 5, 0, 0),      # output type
    lambda: _native.fp8_gemm(P, 128, P, 1, 1, P, 128, P, 1, 1, -1, 4, 128, P, 4, 0, 0, 0),     # negative size
    lambda: _native.fp8_gemm(P, 128, P, 1, 1, P, 128, P, 1, 1, 1 << 31, 4, 128, P, 4, 0, 0, 0),  # past 32 bits
    lambda: _native.fp8_gemm(P, 128, P, 1, 1, P, 128, P, 1, 1, 4, 4, 128, P, 3, 0, 0, 0),      # output stride
    lambda: _native.fp8_gemm(P, 120, P, 1, 1, P, 128, P, 1, 1, 4, 4, 120, P, 4, 0, 0, 0),      # a's stride
    lambda: _native.fp8_gemm(P, 128, P, 1, 1, P + 8, 128, P, 1, 1, 4, 4, 128, P, 4, 0, 0, 0),  # w's base
    lambda: _native.fp8_gemm(P, 112, P, 1, 1, P, 128, P, 1, 1, 4, 4, 128, P, 4, 0, 0, 0),      # stride below columns
    lambda: _native.fp8_gemm(P, 128, 0, 1, 1, P, 128, P, 1, 1, 4, 4, 128, P, 4, 0, 0, 0),      # null scale
])
def test_c_entries_refuse(call):
    with pytest.raises(ValueError):
        call()


def test_c_entries_take_empty_calls():
    """No rows or no columns: nothing is launched, null pointers are fine."""
    _native.fp8_quantize(0, 2, 0, 0, 128, 1, 0, 128, 0, 1, 1, 0)
    _native.fp8_quantize(0, 2, 0, 4, 0, 128, 0, 1, 0, 1, 1, 0)
    _native.fp8_swiglu(0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 1, 1, 0)
    _native.fp8_rms_norm(0, 0, 0, 0, 2, 0, 2, 1e-5, 0, 64, 0, 0, 0, 64, 0, 1, 1, 0)
    _native.fp8_gemm(0, 0, 0, 1, 1, 0, 0, 0, 1, 1, 0, 4, 128, 0, 4, 0, 0, 0)
    _native.fp8_gemm(0, 0, 0, 1, 1, 0, 0, 0, 1, 1, 4, 0, 128, 0, 0, 0, 0, 0)



@pytest.mark.parametrize("call", [
    lambda: _native.fp8_quantize(P + 2, 0, 128, 1, 128, 1, P, 128, P, 1, 1, 0),
    lambda: _native.fp8_quantize(P + 1, 2, 128, 1, 128, 1, P, 128, P, 1, 1, 0),
    lambda: _native.fp8_quantize(P, 2, 128, 1, 128, 1, P, 128, P + 2, 1, 1, 0),                       # scale
    lambda: _native.fp8_swiglu(P, 128, P + 1, 128, 1, 1, 128, P, 128, P, 1, 1, 0),                    # up
    lambda: _native.fp8_swiglu(P + 2, 128, P, 128, 0, 1, 128, P, 128, P, 1, 1, 0),                    # gate
    lambda: _native.fp8_rms_norm(P, 128, 0, 0, 1, P + 2, 0, 1e-5, 1, 128, 0, 0, P, 128, P, 1, 1, 0),  # fp32 weight
    lambda: _native.fp8_rms_norm(P, 128, P + 1, 128, 1, P, 1, 1e-5, 1, 128, P, 128, P, 128, P, 1, 1, 0),  # residual
    lambda: _native.fp8_rms_norm(P, 128, P, 128, 1, P, 1, 1e-5, 1, 128, P + 1, 128, P, 128, P, 1, 1, 0),  # hidden
    lambda: _native.fp8_gemm(P, 128, P + 1, 1, 1, P, 128, P, 1, 1, 4, 4, 128, P, 4, 0, 0, 0),         # a's scales
    lambda: _native.fp8_gemm(P, 128, P, 1, 1, P, 128, P + 2, 1, 1, 4, 4, 128, P, 4, 0, 0, 0),         # w's scales
    lambda: _native.fp8_gemm(P, 128, P, 1, 1, P, 128, P, 1, 1, 4, 4, 128, P + 2, 4, 0, 0, 0),         # fp32 output
    lambda: _native.fp8_gemm(P, 128, P, 1, 1, P, 128, P, 1, 1, 4, 4, 128, P + 1, 4, 2, 0, 0),         # bf16 output
    lambda: _native.fp8_gemm(P, 128, P, 1, 1, P, 128, P, 1, 1, 4, 4, 128, P, 4, 2, P + 2, 0),         # error flag
])
def test_c_entries_refuse_addresses_off_their_elements_boundary(call):
    with pytest.raises(ValueError, match="boundary"):
        call()
