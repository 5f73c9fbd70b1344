"""The 8-bit operators on the shapes whose kernels, loops and branches smaller
calls do not reach.  Each test names the kernel it is about and asserts that
its calls take it, so that a changed rule of choice cannot empty the test.
Tolerances: as derived in fp8_reference.py and test_gpu_fp8.py."""
from __future__ import annotations

import pytest
import torch

from cuda_launches import launches
from fp8_reference import BLOCK, check_product, check_quantized, e4m3

pytestmark = pytest.mark.gpu

FEW = {16: "few_rows_kernelILi16E", 32: "few_rows_kernelILi32E", 64: "few_rows_kernelILi64E"}
WIDE, PAIRS = "wide_kernelILi1E", "wide_kernelILi2E"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
NORM_REL = 2.0 ** -18  # test_gpu_fp8.py


def rand(shape, seed, dtype=torch.float32, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def operands(m, n, k, seed=0):
    from llvq_paper_reproduction_b200 import fp8

    return *fp8.quantize_rows(rand((m, k), seed)), *fp8.quantize_blocks(rand((n, k), seed + 1, scale=0.02))


def product(a, sa, w, sw, dtype, kernel, parts=1):
    """fp8.gemm, which has to take `kernel` with every tile's K in `parts` (3: or more)."""
    from llvq_paper_reproduction_b200 import fp8

    y = fp8.gemm(a, sa, w, sw, out_dtype=dtype, check=True)
    *_, launch = launches(lambda: fp8.gemm(a, sa, w, sw, out_dtype=dtype))  # behind copies of operands
    assert kernel in launch.name, launch
    assert launch.cluster == (2 if kernel == PAIRS else parts) or launch.cluster > parts > 2, launch
    return y


# ------------------------------------------------------------------ the product's loops
# CTA pairs: several tiles a pair, ragged in all three directions, K beyond the stage ring (5 blocks), the
# first scale group (8) and the first use of both scale slots (16); rows of the output stored by TMA (4200),
# in 8-byte words (bf16 4204, fp32 4202) and shifted (4201; bf16 4202)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", [(2500, 4200, 1000), (2500, 4201, 2200), (2500, 4202, 2200), (2500, 4204, 520),
                                   (5003, 2500, 2304)])
def test_pairs(m, n, k, dtype):
    ops = operands(m, n, k)
    check_product(product(*ops, dtype, PAIRS), *ops)


# a tile per CTA, the same limits (its ring has 4 stages)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", [(250, 14336, 4096), (250, 14337, 4200), (600, 4100, 400), (1000, 4098, 2300)])
def test_a_tile_per_cta(m, n, k, dtype):
    ops = operands(m, n, k)
    check_product(product(*ops, dtype, WIDE), *ops)


# K of a tile in parts, which are added in both forms (two parts, and three or more) over whole and cut tiles
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k,parts", [(512, 4096, 4096, 2), (500, 4099, 4000, 2), (256, 4096, 4096, 3),
                                         (250, 4090, 4000, 3), (130, 4096, 14336, 3), (128, 3000, 14300, 3),
                                         (128, 4097, 14300, 3)])
def test_wide_tiles_with_k_in_parts(m, n, k, parts, dtype):
    ops = operands(m, n, k)
    check_product(product(*ops, dtype, WIDE, parts), *ops)


# many rows of next to nothing, and a vocabulary's worth of columns
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k,kernel", [(20000, 8, 300, PAIRS), (20000, 1, 130, PAIRS), (20001, 300, 1, PAIRS),
                                          (10000, 5, 130, WIDE), (10001, 16, 16, WIDE), (3, 128300, 600, FEW[16])])
def test_narrow_and_shallow_products(m, n, k, kernel, dtype):
    ops = operands(m, n, k)
    check_product(product(*ops, dtype, kernel), *ops)


# more blocks in a CTA than one chunk of scales holds (64, 32 and 16 of them)
@pytest.mark.parametrize("m,rows,n,k", [(16, 16, 20000, 9000), (5, 16, 20001, 9000), (32, 32, 20000, 5000),
                                        (64, 64, 28672, 4096), (50, 64, 20001, 6000)])
def test_few_rows_with_several_chunks_of_scales(m, rows, n, k):
    ops = operands(m, n, k)
    check_product(product(*ops, torch.float32, FEW[rows]), *ops)


def test_products_of_every_kind_at_once():
    """On five streams, so that CTAs of different kernels share SMs and their
    tensor memory: the same bits as one after the other."""
    from llvq_paper_reproduction_b200 import fp8

    sizes = [(2500, 4200, 1000, PAIRS), (256, 4096, 4096, WIDE), (600, 4100, 400, WIDE), (5, 20001, 2000, FEW[16]),
             (64, 4096, 8000, FEW[64])]
    ops = [operands(m, n, k, i) for i, (m, n, k, _) in enumerate(sizes)]
    want = [fp8.gemm(*o) for o in ops]
    for o, (*_, kernel) in zip(ops, sizes):
        assert kernel in launches(lambda: fp8.gemm(*o))[0].name
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sizes]
    got = [[] for _ in sizes]
    for _ in range(12):
        for i, (o, s) in enumerate(zip(ops, streams)):
            with torch.cuda.stream(s):
                got[i] += [fp8.gemm(*o) for _ in range(1 + i)]
    torch.cuda.synchronize()
    fp8.raise_pending_errors()
    for w, ys in zip(want, got):
        assert all(torch.equal(w, y) for y in ys)


@pytest.mark.parametrize("m,n,k,kernel", [(600, 4096, 400, WIDE), (2500, 4200, 400, PAIRS)])
def test_wide_products_are_the_same_on_every_call_and_for_any_strides(m, n, k, kernel):
    from llvq_paper_reproduction_b200 import fp8

    a, sa, w, sw = operands(m, n, k)
    want = product(a, sa, w, sw, torch.float32, kernel)
    dense_a, dense_w = (t.view(torch.uint8).contiguous().view(fp8.E4M3) for t in (a, w))
    wide = torch.full((m, 1040), 0x7F, dtype=torch.uint8, device="cuda")  # NaN beside the operand
    wide[:, 16:16 + k] = dense_a.view(torch.uint8)
    turned = dense_w.view(torch.uint8).t().contiguous().view(fp8.E4M3).t()
    for b, sb, v, sv in ((a, sa, w, sw), (dense_a, sa.contiguous(), dense_w, sw.t().contiguous().t()),
                         (wide.view(fp8.E4M3)[:, 16:16 + k], sa, turned, sw)):
        assert torch.equal(want, product(b, sb, v, sv, torch.float32, kernel))
    one = (dense_a[:1].expand(m, -1), sa[:1].expand(m, -1), w, sw)
    check_product(fp8.gemm(*one, out_dtype=torch.float32, check=True), *one)


@pytest.mark.parametrize("m,n,k,kernel", [(600, 4096, 400, WIDE), (512, 4096, 2000, WIDE), (2500, 4200, 400, PAIRS)])
def test_wide_rows_that_are_not_finite_stay_in_their_rows(m, n, k, kernel):
    from llvq_paper_reproduction_b200 import fp8

    x, weight = rand((m, k), 20), fp8.quantize_blocks(rand((n, k), 21, scale=0.02))
    want = fp8.gemm(*fp8.quantize_rows(x), *weight, out_dtype=torch.float32, check=True)
    x[1, 300] = float("nan")
    x[m - 2, k - 1] = float("inf")
    bad = torch.zeros(m, dtype=torch.bool, device="cuda")
    bad[[1, m - 2]] = True
    q, s = fp8.quantize_rows(x)
    got = fp8.gemm(q, s, *weight, out_dtype=torch.float32, check=True)
    assert kernel in launches(lambda: fp8.gemm(q, s, *weight, out_dtype=torch.float32))[0].name
    assert got[bad].isnan().all() and torch.equal(got[~bad], want[~bad])


# ------------------------------------------------------------------ the product's edges
@pytest.mark.parametrize("m,n,k,kernel", [(3, 300, 500, FEW[16]), (30, 300, 1025, FEW[32]), (60, 300, 2200, FEW[64]),
                                          (600, 4096, 500, WIDE), (256, 4096, 4003, WIDE), (2500, 4200, 1001, PAIRS)])
def test_nothing_beside_the_columns_is_read_into_a_product(m, n, k, kernel):
    """Rows of k columns with NaN behind them, in the same 16 bytes and further on."""
    from llvq_paper_reproduction_b200 import fp8

    a, sa, w, sw = operands(m, n, k)

    def between_nans(q):
        held = torch.full((q.shape[0] + 1, q.stride(0) + 16), 0x7F, dtype=torch.uint8, device="cuda")
        held[:-1, :k] = q.view(torch.uint8)
        return held.view(fp8.E4M3)[:-1, :k]

    want = fp8.gemm(a, sa, w, sw, out_dtype=torch.float32, check=True)
    *_, launch = launches(lambda: fp8.gemm(between_nans(a), sa, between_nans(w), sw))
    assert kernel in launch.name
    assert torch.equal(want, fp8.gemm(between_nans(a), sa, between_nans(w), sw, out_dtype=torch.float32))


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


# ------------------------------------------------------------------ the norm's loop over rows
# every CTA takes several rows: the next row ahead of or behind the barrier (up to 8192 columns), two
# chunks (up to 16,384), two of 1024 threads, and rows on odd boundaries
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("m,k", [(5000, 4096), (3000, 4100), (1500, 11008), (700, 20000), (2500, 4097), (1000, 11009),
                                 (500, 20001)])
def test_norm_of_several_rows_a_cta(m, k, residual, dtype):
    from llvq_paper_reproduction_b200 import fp8

    x, r = rand((m, k), 70, dtype, 2.0), rand((m, k), 71, dtype) if residual else None
    w = (1 + 0.1 * rand((k,), 72)).to(dtype)
    (launch,) = launches(lambda: fp8.rms_norm(x, w, residual=r))
    assert "rms_norm_kernel" in launch.name and 2 * launch.grid < m, launch
    for _ in range(2):
        out = fp8.rms_norm(x, w, residual=r)
        h = x.double() + (r.double() if residual else 0)
        y = h * w.double() / torch.sqrt(h.square().mean(dim=1, keepdim=True) + 1e-5)
        check_quantized(out[0], out[1], y, 1, NORM_REL)
        assert not residual or torch.equal(out[2], (x.float() + r.float()).to(dtype))
        x.copy_(x.flip(0))  # other rows for every CTA


# ------------------------------------------------------------------ ties
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(900, 4096), (301, 1030), (140, 4099)])
def test_bytes_of_16_bit_inputs_are_the_rounded_quotient(shape, dtype):
    """448 x / amax of 16-bit numbers is a tie of e4m3 or at least 2^-16 of
    itself away from one, so the nearest byte is one and no other.  In 64 bits 448 x is exact
    and the quotient of a tie is the tie, so the reference's rounding is right."""
    from llvq_paper_reproduction_b200 import fp8

    x = rand(shape, 73, dtype)
    x[:, 5::BLOCK] = 7.0  # amax a multiple of 7: ties by the dozen
    m, k = shape
    for f, rows in ((fp8.quantize_rows, 1), (fp8.quantize_blocks, BLOCK)):
        q, _ = f(x)
        p = torch.nn.functional.pad(x.double(), (0, -k % BLOCK, 0, -m % rows))
        p = p.view(-1, rows, p.shape[1] // BLOCK, BLOCK)
        want = 448.0 * p / p.abs().amax(dim=(1, 3), keepdim=True)
        ties = (want / torch.exp2(torch.frexp(want)[1].clamp(min=-5).double() - 5)).remainder(2.0) == 1.0
        assert ties.sum() > 100
        assert torch.equal(q.double(), e4m3(want).view(-1, p.shape[2] * BLOCK)[:m, :k])


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
