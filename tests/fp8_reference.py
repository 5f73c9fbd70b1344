"""The 8-bit operators' definitions in 64 bits (CPU or GPU tensors), for tests."""
from __future__ import annotations

import torch

BLOCK = 128
FLOOR = 2.0 ** -100


def step(v: torch.Tensor) -> torch.Tensor:
    """Spacing of e4m3 values around v (3 fraction bits, exponents from -6)."""
    _, e = torch.frexp(v.abs())
    return torch.exp2((e.double() - 1).clamp(min=-6) - 3)


def e4m3(v: torch.Tensor) -> torch.Tensor:
    """Nearest e4m3 value of each fp64 one, ties to even, for |v| <= 448."""
    s = step(v)
    return torch.round(v / s) * s


def spread(scale: torch.Tensor, rows: int, cols: int, block_rows: int) -> torch.Tensor:
    """A scale for every element."""
    s = scale.double().repeat_interleave(BLOCK, dim=1)[:, :cols]
    return s.repeat_interleave(block_rows, dim=0)[:rows]


def amax(y: torch.Tensor, block_rows: int) -> torch.Tensor:
    """max(2^-100, max |y|) of every block of an fp64 matrix."""
    m, k = y.shape
    p = torch.nn.functional.pad(y.abs(), (0, -k % BLOCK, 0, -m % block_rows))
    p = p.view(p.shape[0] // block_rows, block_rows, p.shape[1] // BLOCK, BLOCK)
    return p.amax(dim=(1, 3)).clamp(min=FLOOR)


def values(q: torch.Tensor, scale: torch.Tensor, block_rows: int = 1) -> torch.Tensor:
    """What an 8-bit matrix stands for."""
    return q.double() * spread(scale, *q.shape, block_rows)


def check_quantized(q: torch.Tensor, scale: torch.Tensor, y: torch.Tensor, block_rows: int, rel: float) -> None:
    """(q, scale) against the fp64 matrix y whose fp32 form is within `rel`
    of y, relatively.  The scale is then within rel plus the division's
    2^-24.  448 y / amax moves by at most 2 rel (numerator and amax) plus the
    quotient's 2^-24, and e4m3 rounds it by half a step."""
    a = amax(y, block_rows)
    assert scale.dtype == torch.float32 and scale.shape == a.shape
    assert ((scale.double() * 448.0 / a - 1.0).abs() <= rel + 2.0 ** -23).all()
    want = 448.0 * y / spread(a, *y.shape, block_rows)
    slack = (2 * rel + 2.0 ** -23) * want.abs()
    assert ((q.double() - want).abs() <= step(want.abs() + slack) / 2 + slack).all()


def product(a, a_scale, w, w_scale):
    """A W^T in fp64, and the sum of the absolute values of its terms."""
    x, z = values(a, a_scale), values(w, w_scale, BLOCK)
    return x @ z.t(), x.abs() @ z.abs().t()


def check_product(y: torch.Tensor, a, a_scale, w, w_scale) -> None:
    """Products of e4m3 values are exact in fp32.  Summing the 128 of a block
    takes 127 additions, the scales two products and the blocks one addition
    each, so an output is off by at most (127 + 3 + blocks) roundings of the
    sum of absolute values; a tensor core may truncate instead of rounding
    (2^-23).  Then one rounding to the output's type."""
    want, terms = product(a, a_scale, w, w_scale)
    blocks = a_scale.shape[1]
    fi = torch.finfo(y.dtype)
    bound = (130 * 2.0 ** -23 + blocks * 2.0 ** -24) * terms
    bound = bound + fi.eps / 2 * (want.abs() + bound) + fi.smallest_normal * fi.eps
    bad = (y.double() - want).abs() > bound
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist())
