"""The 8-bit operators on the shapes whose kernels, loops and branches smaller
calls do not reach.  Each test names the kernel it is about and asserts that
its calls take it, so that a changed rule of choice cannot empty the test.
Tolerances: as derived in fp8_reference.py and test_gpu_fp8.py."""
from __future__ import annotations

import pytest
import torch

from cuda_launches import launches
from fp8_reference import check_product

pytestmark = pytest.mark.gpu

WIDE, PAIRS = "wide_kernelILi1E", "wide_kernelILi2E"


def rand(shape, seed, dtype=torch.float32, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def operands(m, n, k, seed=0):
    from llvq_paper_reproduction_b200 import fp8

    return *fp8.quantize_rows(rand((m, k), seed)), *fp8.quantize_blocks(rand((n, k), seed + 1, scale=0.02))


def product(a, sa, w, sw, dtype, kernel, parts=1):
    """fp8.gemm, which has to take `kernel` with every tile's K in `parts`."""
    from llvq_paper_reproduction_b200 import fp8

    y = fp8.gemm(a, sa, w, sw, out_dtype=dtype, check=True)
    (launch,) = launches(lambda: fp8.gemm(a, sa, w, sw, out_dtype=dtype))
    assert kernel in launch.name and launch.cluster == (2 if kernel == PAIRS else parts), launch
    return y


# ------------------------------------------------------------------ the product's edges
@pytest.mark.parametrize("m,n,k,kernel", [(600, 4100, 300, WIDE), (500, 4099, 2000, WIDE), (2500, 4100, 300, PAIRS)])
def test_wide_products_write_only_their_output(m, n, k, kernel):
    """Through the C ABI: an output inside a wider buffer, with what lies around it left as it was."""
    from llvq_paper_reproduction_b200 import _native

    a, sa, w, sw = operands(m, n, k)
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    for dtype, code in ((torch.float32, 0), (torch.float16, 1), (torch.bfloat16, 2)):
        for ld in (n + 3, (n + 15) // 16 * 16 + 16, (n + 3) // 4 * 4 + 4, (n + 1) // 2 * 2 + 2, n | 1):
            y = torch.full((m + 2, ld), -7.0, dtype=dtype, device="cuda")

            def call():
                _native.fp8_gemm(a.data_ptr(), a.stride(0), sa.data_ptr(), sa.stride(0), sa.stride(1), w.data_ptr(),
                                 w.stride(0), sw.data_ptr(), sw.stride(0), sw.stride(1), m, n, k, y[1:].data_ptr(),
                                 ld, code, flag.data_ptr(), torch.cuda.current_stream().cuda_stream)

            assert kernel in launches(call)[0].name
            call()
            check_product(y[1:m + 1, :n], a, sa, w, sw)
            assert (y[0] == -7).all() and (y[m + 1] == -7).all() and (y[1:m + 1, n:] == -7).all()
    assert not flag.any()


# ------------------------------------------------------------------ scales and rows apart
@pytest.mark.parametrize("m,n,k,kernel", [(600, 4096, 400, WIDE), (2500, 4200, 400, PAIRS)])
def test_wide_rows_whose_scales_leave_the_range_beside_others(m, n, k, kernel):
    """Every other row's scale times the weight's is below the normal fp32
    numbers while the row's products are not: the two are applied one after the
    other, by the lane, with the warp's other lanes on the single product."""
    a, sa, w, sw = operands(m, n, k)
    sw = sw * 2.0 ** -30
    sa = sa.clone()
    sa[1::2] *= 2.0 ** -90
    factors = sa.double()[:, None, :] * sw.double()[None]
    assert (factors[1::2] < 2.0 ** -126).all() and (factors[::2] > 2.0 ** -60).all()
    y = product(a, sa, w, sw, torch.float32, kernel)
    assert (y[1::2].abs().amax(dim=1) > 2.0 ** -126).all()
    check_product(y, a, sa, w, sw)


# ------------------------------------------------------------------ the gate's lower end
# gate / (1 + exp(-gate)) * up below gate = -87 is (gate E) (E up), E = exp(gate / 2): each E
# within 2 units (2^-22), three products of 2^-24
LOW_REL = 2.0 ** -20


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("cols", [512, 515])
def test_swiglu_of_gates_whose_exponential_leaves_the_range(cols, dtype):
    """From -87.3 on the reciprocal of 1 + exp(-gate) is below the normal fp32
    numbers, from -88.8 on the exponential above the largest; with a large up the
    product is neither (with fp16's largest, 1/14 of the floor 2^-100: a byte of 32)."""
    from fp8_reference import check_quantized
    from llvq_paper_reproduction_b200 import fp8

    from llvq_paper_reproduction_b200.fp8 import E4M3

    gate = torch.linspace(-87.0, -100.0, 6 * cols, device="cuda").view(6, cols).to(dtype)
    gate[:, ::7] = rand((6, cols), 65, dtype)[:, ::7]  # ordinary ones among them
    up = (rand((6, cols), 66).sign() * torch.finfo(dtype).max * 0.9).to(dtype)
    up[:, ::7] = 1e-30 if dtype != torch.float16 else 0.0
    g = gate.double()
    y = g * torch.sigmoid(g) * up.double()
    q, scale = fp8.swiglu(gate, up)
    assert q.dtype == E4M3 and (q.float() != 0).float().mean() > (0.8 if dtype != torch.float16 else 0.05)
    check_quantized(q, scale, y, 1, LOW_REL)


def test_swiglu_far_below_and_not_finite():
    from llvq_paper_reproduction_b200 import fp8

    up = torch.full((1, 128), 3e38, device="cuda")
    for low in (-200.0, -1000.0, -3e38):
        gate = torch.full((1, 128), low, device="cuda")
        q, scale = fp8.swiglu(gate, up)
        assert not q.float().any() and scale.isfinite().all()
    gate[0, 5] = float("nan")
    assert fp8.swiglu(gate, up)[0].float().isnan().all()


@pytest.mark.parametrize("m,n,k,kernel", [(600, 4096, 400, WIDE), (2500, 4200, 400, PAIRS)])
def test_wide_rows_of_zeros_and_of_small_numbers(m, n, k, kernel):
    """Padding rows, whose scale is the floor's, and rows whose scale times the
    weight's lies anywhere down to the smallest normal fp32 number or up to 2^100."""
    from llvq_paper_reproduction_b200 import fp8

    x = rand((m, k), 2)
    x[m // 4::3] = 0.0
    a, sa = fp8.quantize_rows(x)
    w, sw = fp8.quantize_blocks(rand((n, k), 3, scale=0.02))
    sa = sa.clone()
    exponents = torch.arange(m, device="cuda") % 230 - 118
    live = x.any(dim=1)
    sa[live] *= torch.exp2(exponents[live].float())[:, None] / sa[live].amax(dim=1, keepdim=True)
    y = product(a, sa, w, sw * (2.0 ** -6 / sw.amax()), torch.float32, kernel)
    assert not y[~live].any() and y[live].isfinite().all()
    check_product(y, a, sa, w, sw * (2.0 ** -6 / sw.amax()))


# ------------------------------------------------------------------ what a call may be given
def calls(m=4, k=256, n=6):
    """Every input of every operator: a name, the tensor, and the call with it."""
    from llvq_paper_reproduction_b200 import fp8

    x, r, w = rand((m, k), 60), rand((m, k), 61), 1 + 0.1 * rand((k,), 62)
    a, sa, b, sb = operands(m, n, k)
    return [("quantize_rows x", x, fp8.quantize_rows), ("quantize_blocks w", x, fp8.quantize_blocks),
            ("swiglu gate", x, lambda t: fp8.swiglu(t, r)), ("swiglu up", r, lambda t: fp8.swiglu(x, t)),
            ("rms_norm x", x, lambda t: fp8.rms_norm(t, w)), ("rms_norm weight", w, lambda t: fp8.rms_norm(x, t)),
            ("rms_norm residual", r, lambda t: fp8.rms_norm(x, w, residual=t)),
            ("gemm a_scale", sa, lambda t: fp8.gemm(a, t, b, sb)), ("gemm w_scale", sb, lambda t: fp8.gemm(a, sa, b, t))]


def test_inputs_with_a_tangent_are_refused():
    """Forward only: a dual tensor's tangent would be dropped without a word."""
    import torch.autograd.forward_ad as fwd

    for name, x, call in calls():
        with fwd.dual_level():
            dual = fwd.make_dual(x, torch.ones_like(x))
            with pytest.raises(ValueError, match="tangent"):
                call(dual)
                pytest.fail(name)
            call(fwd.unpack_dual(dual).primal)  # the values alone


def test_lazy_negation_is_not_lost():
    """A view with the negative bit reads as its values; e4m3, whose bytes have no such form, is refused."""
    from llvq_paper_reproduction_b200 import fp8

    def same(got, want):
        for g, w in zip(got if isinstance(got, tuple) else (got,), want if isinstance(want, tuple) else (want,)):
            assert torch.equal(g.float(), w.float()), name

    for name, x, call in calls():
        same(call(torch._neg_view(x)), call(-x))
    z = torch.complex(rand((5, 1), 63), rand((5, 1), 64))
    same(fp8.quantize_rows(z.conj().imag), fp8.quantize_rows(-z.imag.contiguous()))
    a, sa, b, sb = operands(4, 6, 256)
    for bad in (lambda: fp8.gemm(torch._neg_view(a), sa, b, sb), lambda: fp8.gemm(a, sa, torch._neg_view(b), sb)):
        with pytest.raises(ValueError):
            bad()


def test_first_product_in_inference_mode(monkeypatch):
    """The error flag made there can be read and cleared outside."""
    from llvq_paper_reproduction_b200 import fp8

    monkeypatch.setattr(fp8, "_flags", {})  # as in a fresh process
    ops = operands(4, 6, 256)
    with torch.inference_mode():
        fp8.gemm(*ops)
        ((flag, _),) = fp8._flags.values()
        flag.fill_(1)  # as after a timeout
    with pytest.raises(RuntimeError, match="timed out"):
        fp8.raise_pending_errors()
    assert fp8.pending_errors() == {"gemm_timeout": 0}
    fp8.raise_pending_errors()
    fp8.gemm(*ops, check=True)
