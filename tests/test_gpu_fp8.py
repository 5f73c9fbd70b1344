"""The 8-bit operators on the GPU against their definitions in 64 bits.

Tolerances (fp8_reference.py derives the shared parts):
  quantizers  the fp32 form of y is exact (rel = 0)
  rms_norm    h: 2^-24; the mean of squares: at most 32 additions in a thread,
              5 in a warp, 32 over warps, each 2^-24, and a division; half of
              that after the root; root, division, two products: below 2^-18
  swiglu      exp 2 ulp (2^-22) weighted by e / (1 + e) < 1, one addition, one
              division, one product: below 2^-21
"""
from __future__ import annotations

import pytest
import torch

from fp8_reference import BLOCK, check_product, check_quantized, values

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
NORM_REL, SWIGLU_REL = 2.0 ** -18, 2.0 ** -21


def rand(shape, seed, dtype=torch.float32, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def operands(m, n, k, seed=0):
    from llvq_paper_reproduction_b200 import fp8

    return *fp8.quantize_rows(rand((m, k), seed)), *fp8.quantize_blocks(rand((n, k), seed + 1, scale=0.02))


# ------------------------------------------------------------------ quantizers
SHAPES = [(1, 1), (1, 128), (3, 127), (5, 129), (37, 4100), (130, 384), (129, 1000), (2, 14336), (300, 8)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_quantizers(shape, dtype):
    from llvq_paper_reproduction_b200 import fp8

    x = rand(shape, 1, dtype)
    q, scale = fp8.quantize_rows(x)
    check_quantized(q, scale, x.double(), 1, 0.0)
    q, scale = fp8.quantize_blocks(x)
    check_quantized(q, scale, x.double(), BLOCK, 0.0)


@pytest.mark.parametrize("rows", [1, BLOCK])
def test_quantizer_ties_and_range(rows):
    """Quotients on ties go to even, on subnormal values to their grid; the
    largest magnitude becomes 448; blocks far outside the usual range scale."""
    from llvq_paper_reproduction_b200 import fp8

    ticks = torch.arange(0, 897, device="cuda").float() / 2  # every value and tie up to 448
    x = torch.cat([ticks, torch.arange(0, 127, device="cuda").float() * 2.0 ** -11])
    x = x.view(-1, 128) if rows == 1 else x[:1024].view(8, 128)
    x[:, 0] = 448.0  # scale 1
    for factor in (1.0, -1.0, 2.0 ** 100, 2.0 ** -60, 2.0 ** 118):
        y = x * factor
        q, scale = (fp8.quantize_rows if rows == 1 else fp8.quantize_blocks)(y)
        check_quantized(q, scale, y.double(), rows, 0.0)
        assert torch.equal(q.float(), (x * (1 if factor > 0 else -1)).to(torch.float8_e4m3fn).float())


def test_quantizer_zeros_and_non_finite_values():
    from llvq_paper_reproduction_b200 import fp8

    x = rand((4, 512), 3, torch.bfloat16)
    x[0, 130] = float("nan")
    x[1, 260] = float("inf")
    x[2, 384:] = 0.0
    x[3, :128] = 1e-38
    q, scale = fp8.quantize_rows(x)
    qf = q.float()
    assert qf[0, 128:256].isnan().all() and scale[0, 1].isnan()
    assert qf[1, 260].isnan() and scale[1, 2].isinf() and (qf[1, 256:260] == 0).all() and (qf[1, 261:384] == 0).all()
    assert (qf[2, 384:] == 0).all() and 0 < scale[2, 3] < 1e-30
    assert scale[3, 0] == scale[2, 3] and qf[3, :128].isfinite().all()
    rest = torch.ones((4, 4), dtype=torch.bool, device="cuda")
    rest[0, 1] = rest[1, 2] = False  # the other blocks are as without their neighbours
    clean = x.clone()
    clean[0, 130] = clean[1, 260] = 0.0
    q2, s2 = fp8.quantize_rows(clean)
    keep = rest.repeat_interleave(128, dim=1)
    assert torch.equal(scale[rest], s2[rest]) and torch.equal(qf[keep], q2.float()[keep])
    qb, sb = fp8.quantize_blocks(x)
    assert qb.float()[:, 128:256].isnan().all() and sb[0, 1].isnan() and sb[0, 2].isinf() and sb[0, 0].isfinite()


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantizer_strides_and_empty(dtype):
    """Views with odd offsets and strides, a transposed and an expanded matrix, and sizes of zero."""
    from llvq_paper_reproduction_b200 import fp8

    base = rand((70, 1003), 4, dtype)
    for x in (base[:, 3:], base[5:, :640], base[::3, 1:258], base.t(), base[:1].expand(9, -1), base[:, 8:9]):
        for f, rows in ((fp8.quantize_rows, 1), (fp8.quantize_blocks, BLOCK)):
            q, scale = f(x)
            assert q.shape == x.shape and q.stride(0) % 16 == 0
            check_quantized(q, scale, x.double(), rows, 0.0)
    for shape in ((0, 128), (4, 0), (0, 0)):
        q, scale = fp8.quantize_rows(base.new_empty(shape))
        assert q.shape == shape and scale.shape == (shape[0], (shape[1] + 127) // 128)
        q, scale = fp8.quantize_blocks(base.new_empty(shape))
        assert q.shape == shape and scale.shape == ((shape[0] + 127) // 128, (shape[1] + 127) // 128)


def test_more_than_2_to_the_31_rows():
    """Rows are counted past 31 bits too: 2.2e9 rows of one column."""
    from llvq_paper_reproduction_b200 import fp8

    m = (1 << 31) + 70_000
    x = torch.zeros((m, 1), dtype=torch.bfloat16, device="cuda")
    x[-2:] = torch.tensor([[3.0], [-5.0]], device="cuda")
    q, scale = fp8.quantize_rows(x)
    assert q[-2:].float().flatten().tolist() == [448.0, -448.0] and not q[:1000].float().any()
    assert (scale[-2:].flatten() * 448 - torch.tensor([3.0, 5.0], device="cuda")).abs().max() < 1e-5
    del q, scale
    q, scale = fp8.rms_norm(x, torch.ones(1, dtype=torch.bfloat16, device="cuda"))
    assert q[-2:].float().flatten().tolist() == [448.0, -448.0]


def test_quantizer_past_32_bit_offsets():
    from llvq_paper_reproduction_b200 import fp8

    m, k = (1 << 18) + 5, 8320  # 2.18e9 elements
    x = torch.zeros((m, k), dtype=torch.bfloat16, device="cuda")
    x[-3:] = rand((3, k), 5, torch.bfloat16)
    for f, rows in ((fp8.quantize_rows, 1), (fp8.quantize_blocks, BLOCK)):
        q, scale = f(x)
        tail = m // BLOCK * BLOCK if rows == BLOCK else m - 3
        check_quantized(q[tail:], scale[tail // rows:], x[tail:].double(), rows, 0.0)
        assert not q[:BLOCK].float().any()
        del q, scale


# ------------------------------------------------------------------ norm and gate
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (1, 4096), (5, 4100), (2, 8200), (3, 16392), (2, 32768), (150, 256)])
@pytest.mark.parametrize("residual,wide_weight", [(False, True), (True, False)])
def test_rms_norm(shape, dtype, residual, wide_weight):
    from llvq_paper_reproduction_b200 import fp8

    m, k = shape
    x, r = rand(shape, 6, dtype, 2.0), rand(shape, 7, dtype) if residual else None
    w = (1 + 0.1 * rand((k,), 8)).to(torch.float32 if wide_weight else dtype)
    out = fp8.rms_norm(x, w, eps=1e-5, residual=r)
    h = x.double() + (r.double() if residual else 0)
    y = h * w.double() / torch.sqrt(h.square().mean(dim=1, keepdim=True) + 1e-5)
    check_quantized(out[0], out[1], y, 1, NORM_REL)
    assert len(out) == (3 if residual else 2)
    if residual:
        assert out[2].dtype == dtype and torch.equal(out[2], (x.float() + r.float()).to(dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(2000, 1001), (3, 2047), (131, 4097), (3, 9001), (2, 16383), (2, 16385), (2, 32767)])
def test_rows_on_odd_boundaries(shape, dtype):
    """Rows that start anywhere, NaN on both sides of each: nothing beside a
    row is read into it, nothing beside the hidden row is written."""
    from llvq_paper_reproduction_b200 import fp8

    m, k = shape

    def odd(seed):
        base = torch.full((m, k + 5 + k % 2), float("nan"), device="cuda", dtype=dtype)
        base[:, 3:3 + k] = rand(shape, seed, dtype)
        return base[:, 3:3 + k]

    x, r, w = odd(50), odd(51), (1 + 0.1 * rand((k + 1,), 52)).to(dtype)[1:]
    for residual in (None, r):
        out = fp8.rms_norm(x, w, residual=residual)
        h = x.double() + (0.0 if residual is None else r.double())
        y = h * w.double() / torch.sqrt(h.square().mean(dim=1, keepdim=True) + 1e-5)
        check_quantized(out[0], out[1], y, 1, NORM_REL)
    assert torch.equal(out[2], (x.float() + r.float()).to(dtype))
    q, scale = fp8.quantize_rows(x)
    check_quantized(q, scale, x.double(), 1, 0.0)
    q, scale = fp8.quantize_blocks(x)
    check_quantized(q, scale, x.double(), BLOCK, 0.0)
    q, scale = fp8.swiglu(x, r)
    g = x.double()
    check_quantized(q, scale, g * torch.sigmoid(g) * r.double(), 1, SWIGLU_REL)


def test_rms_norm_strides_zero_rows_and_nan():
    from llvq_paper_reproduction_b200 import fp8

    base, rbase = rand((9, 3 * 520), 9, torch.bfloat16), rand((9, 2 * 521), 10, torch.bfloat16)
    x, r, w = base[:, 520:1040], rbase[:, 521:1041], torch.ones(1040, device="cuda", dtype=torch.bfloat16)[::2]
    x[4] = 0.0
    r[4] = 0.0
    x[6, 11] = float("nan")
    q, scale, hidden = fp8.rms_norm(x, w, eps=1e-6, residual=r)
    h = x.double() + r.double()
    y = h / torch.sqrt(h.square().mean(dim=1, keepdim=True) + 1e-6)
    rows = [i for i in range(9) if i != 6]
    check_quantized(q.float()[rows], scale[rows], y[rows], 1, NORM_REL)
    assert not q[4].float().any() and q[6].float().isnan().all() and scale[6].isnan().all()
    assert hidden.isnan().sum() == 1
    q, scale = fp8.rms_norm(x[:0], w)
    assert q.shape == (0, 520) and scale.shape == (0, 5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (3, 127), (64, 1376), (5, 4100), (2, 14336)])
def test_swiglu(shape, dtype):
    from llvq_paper_reproduction_b200 import fp8

    m, k = shape
    gu = rand((m, 2 * k), 11, dtype, 3.0)
    for gate, up in (gu.chunk(2, dim=1), (rand(shape, 12, dtype), rand(shape, 13, dtype))):
        q, scale = fp8.swiglu(gate, up)
        g = gate.double()
        check_quantized(q, scale, g / (1 + torch.exp(-g)) * up.double(), 1, SWIGLU_REL)


def test_swiglu_extremes():
    from llvq_paper_reproduction_b200 import fp8

    gate = torch.tensor([[-1000.0, 1000.0, 0.0, -0.0, 80.0]], device="cuda")
    q, scale = fp8.swiglu(gate, torch.ones_like(gate))
    got = values(q, scale)[0]
    assert got[0] == 0 and got[2] == 0 and got[3] == 0
    assert abs(got[1] / 1000 - 1) < 1e-6 and abs(got[4] / 80 - 1) <= 2.0 ** -4
    gate[0, 1] = float("nan")
    q, scale = fp8.swiglu(gate, torch.ones_like(gate))
    assert q.float().isnan().all()


# ------------------------------------------------------------------ product
PRODUCTS = [(1, 1, 1), (1, 128, 128), (1, 100, 16), (2, 129, 127), (15, 256, 129), (16, 384, 384), (17, 128, 640),
            (33, 300, 257), (64, 4100, 2200), (65, 130, 130), (128, 128, 4096), (129, 257, 1000), (200, 513, 300),
            (256, 256, 256), (300, 260, 14336), (517, 1030, 520), (777, 128, 100), (1, 14336, 4096), (1, 4096, 14336),
            (600, 4096, 392), (2049, 1029, 264)]


@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_gemm(m, n, k):
    from llvq_paper_reproduction_b200 import fp8

    a, sa, w, sw = operands(m, n, k)
    for dtype in DTYPES:
        y = fp8.gemm(a, sa, w, sw, out_dtype=dtype, check=True)
        assert y.shape == (m, n) and y.dtype == dtype
        check_product(y, a, sa, w, sw)
    assert torch.equal(y, fp8.gemm(a, sa, w, sw, out_dtype=torch.float32))  # one summation order


@pytest.mark.parametrize("m", [1, 7, 64, 300, 1100])
def test_gemm_strides(m):
    """Operands and scales that lie otherwise than the quantizers leave them."""
    from llvq_paper_reproduction_b200 import fp8

    n, k = 333, 500
    a, sa, w, sw = operands(m, n, k)
    want = fp8.gemm(a, sa, w, sw, out_dtype=torch.float32)
    dense_a, dense_w = (t.view(torch.uint8).contiguous().view(fp8.E4M3) for t in (a, w))  # rows of 500 bytes: copied
    assert torch.equal(want, fp8.gemm(dense_a, sa.contiguous(), dense_w, sw.t().contiguous().t(),
                                      out_dtype=torch.float32))
    wide = torch.zeros((m, 1040), dtype=torch.uint8, device="cuda")
    wide[:, 16:16 + k] = dense_a.view(torch.uint8)
    wide = wide.view(fp8.E4M3)
    assert torch.equal(want, fp8.gemm(wide[:, 16:16 + k], sa, w, sw, out_dtype=torch.float32))
    turned = dense_w.view(torch.uint8).t().contiguous().view(fp8.E4M3).t()  # column major: copied
    assert torch.equal(want, fp8.gemm(a, sa, turned, sw, out_dtype=torch.float32))
    if m > 1:  # one row for all
        y = fp8.gemm(dense_a[:1].expand(m, -1), sa[:1].expand(m, -1), w, sw, out_dtype=torch.float32)
        check_product(y, dense_a[:1].expand(m, -1), sa[:1].expand(m, -1), w, sw)


@pytest.mark.parametrize("m", [3, 100, 700])
def test_gemm_non_finite_rows_stay_in_their_rows(m):
    from llvq_paper_reproduction_b200 import fp8

    x = rand((m, 400), 20)
    a, sa, w, sw = *fp8.quantize_rows(x), *fp8.quantize_blocks(rand((200, 400), 21))
    want = fp8.gemm(a, sa, w, sw, out_dtype=torch.float32)
    x[1, 300] = float("nan")
    x[2, 399] = float("inf")
    got = fp8.gemm(*fp8.quantize_rows(x), w, sw, out_dtype=torch.float32)
    assert got[1:3].isnan().all()
    keep = [i for i in range(m) if i not in (1, 2)]
    assert torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("m", [2, 90, 640])
def test_gemm_scales_far_apart(m):
    """Blocks whose scales differ by many orders: each is scaled by itself;
    scales whose product leaves the range of fp32 although the result does not."""
    from llvq_paper_reproduction_b200 import fp8

    a, sa, w, sw = operands(m, 260, 384)
    sa2, sw2 = sa.clone(), sw.clone()
    sa2[:, 1] *= 2.0 ** 90
    sw2[:, 1] *= 2.0 ** -90
    check_product(fp8.gemm(a, sa2, w, sw2, out_dtype=torch.float32), a, sa2, w, sw2)
    sa2[:, 2] *= 2.0 ** -20
    check_product(fp8.gemm(a, sa2, w, sw2, out_dtype=torch.float32), a, sa2, w, sw2)
    # the floor's scale times a small one: below the normal numbers, of zero values
    zero = torch.zeros((m, 384), device="cuda")
    y = fp8.gemm(*fp8.quantize_rows(zero), w, sw * 2.0 ** -60, out_dtype=torch.float32)
    assert not y.any()
    # 2^100 * 2^60 overflows, times zero values it is still zero
    y = fp8.gemm(fp8.quantize_rows(zero)[0], torch.full_like(sa, 2.0 ** 100), w, sw * 2.0 ** 60,
                 out_dtype=torch.float32)
    assert not y.any()


def test_gemm_empty():
    from llvq_paper_reproduction_b200 import fp8

    a, sa, w, sw = operands(4, 6, 256)
    assert fp8.gemm(a[:0], sa[:0], w, sw).shape == (0, 6)
    assert fp8.gemm(a, sa, w[:0], sw[:0]).shape == (4, 0)
    y = fp8.gemm(a[:, :0], sa[:, :0], w[:, :0], sw[:, :0])
    assert y.shape == (4, 6) and not y.any()


@pytest.mark.parametrize("m,n,k", [(1, 100, 200), (40, 131, 300), (300, 200, 256), (1030, 300, 384)])
def test_gemm_writes_only_its_output(m, n, k):
    """Through the C ABI: an output inside a wider buffer, with what lies around it left as it was."""
    from llvq_paper_reproduction_b200 import _native

    a, sa, w, sw = operands(m, n, k)
    for dtype, code in ((torch.float32, 0), (torch.bfloat16, 2)):
        for ld in (n + 3, (n + 15) // 16 * 16 + 16, (n + 3) // 4 * 4 + 4, (n + 1) // 2 * 2 + 2, n | 1):
            y = torch.full((m + 2, ld), -7.0, dtype=dtype, device="cuda")
            flag = torch.zeros(1, dtype=torch.int32, device="cuda")
            _native.fp8_gemm(a.data_ptr(), a.stride(0), sa.data_ptr(), sa.stride(0), sa.stride(1), w.data_ptr(),
                             w.stride(0), sw.data_ptr(), sw.stride(0), sw.stride(1), m, n, k, y[1:].data_ptr(), ld,
                             code, flag.data_ptr(), torch.cuda.current_stream().cuda_stream)
            check_product(y[1:m + 1, :n], a, sa, w, sw)
            assert (y[0] == -7).all() and (y[m + 1] == -7).all() and (y[1:m + 1, n:] == -7).all()
            assert not flag.any()


def test_gemm_past_32_bit_offsets():
    from llvq_paper_reproduction_b200 import fp8

    m, n, k = 70003, 32000, 16  # 2.24e9 outputs
    a, sa, w, sw = operands(m, n, k)
    y = fp8.gemm(a, sa, w, sw, check=True)
    for rows in (slice(0, 3), slice(m - 3, m)):
        check_product(y[rows], a[rows], sa[rows], w, sw)


def test_refusals():
    from llvq_paper_reproduction_b200 import fp8

    x = rand((4, 256), 0, torch.bfloat16)
    w = torch.ones(256, device="cuda", dtype=torch.bfloat16)
    a, sa, b, sb = operands(4, 6, 256)
    bad = [lambda: fp8.quantize_rows(x.double()), lambda: fp8.quantize_rows(x[0]), lambda: fp8.quantize_blocks(x.int()),
           lambda: fp8.quantize_rows(x.float().requires_grad_()),
           lambda: fp8.swiglu(x, x[:, :128]), lambda: fp8.swiglu(x, x.float()), lambda: fp8.swiglu(x, x.cpu()),
           lambda: fp8.rms_norm(x, w[:128]), lambda: fp8.rms_norm(x, w.half()), lambda: fp8.rms_norm(x, w.cpu()),
           lambda: fp8.rms_norm(x, w, residual=x[:2]), lambda: fp8.rms_norm(x, w, eps=-1.0),
           lambda: fp8.rms_norm(x, w, eps=float("nan")), lambda: fp8.rms_norm(x, w.float().requires_grad_()),
           lambda: fp8.rms_norm(rand((1, 32769), 0), torch.ones(32769, device="cuda")),
           lambda: fp8.gemm(a, sa, b[:, :128], sb[:, :1]), lambda: fp8.gemm(a, sa[:2], b, sb),
           lambda: fp8.gemm(a, sa[:, :1], b, sb), lambda: fp8.gemm(a, sa, b, sb.double()),
           lambda: fp8.gemm(a.float(), sa, b, sb), lambda: fp8.gemm(a, sa.cpu(), b, sb),
           lambda: fp8.gemm(a, sa, b, sb, out_dtype=fp8.E4M3), lambda: fp8.gemm(a, sa.requires_grad_(), b, sb)]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    with torch.no_grad():
        fp8.quantize_rows(x.float().requires_grad_())


def test_eight_bit_operands_that_require_grad_are_refused():
    from llvq_paper_reproduction_b200 import fp8

    a, sa, b, sb = operands(4, 6, 256)
    wants = a.detach().clone().requires_grad_()
    with pytest.raises(ValueError, match="requires grad"):
        fp8.gemm(wants, sa, b, sb)
    with pytest.raises(ValueError, match="requires grad"):
        fp8.gemm(a, sa, b.detach().clone().requires_grad_(), sb)
    with torch.no_grad():
        assert torch.equal(fp8.gemm(wants, sa, b, sb), fp8.gemm(a, sa, b, sb))


# ------------------------------------------------------------------ as they are used
def mlp(x, residual, norm_weight, gate_up, down):
    from llvq_paper_reproduction_b200 import fp8

    q, s, hidden = fp8.rms_norm(x, norm_weight, residual=residual)
    gate, up = fp8.gemm(q, s, *gate_up).chunk(2, dim=1)
    return fp8.gemm(*fp8.swiglu(gate, up), *down), hidden


def mlp_weights(k=520, inner=1376):
    from llvq_paper_reproduction_b200 import fp8

    return (torch.ones(k, device="cuda", dtype=torch.bfloat16), fp8.quantize_blocks(rand((2 * inner, k), 31, scale=0.05)),
            fp8.quantize_blocks(rand((k, inner), 32, scale=0.05)))


@pytest.mark.parametrize("m", [1, 5, 64, 400])
def test_mlp(m):
    """One layer's MLP, every operator fed by the one before it, against 64
    bits.  An e4m3 rounding is uniform within half a step of 1/8 of the
    binade: rms 0.036 of a value whose rms in the binade is 1.53, so 0.024
    relatively.  The first one reaches gate and up (each 0.024, their product
    below 0.036 with silu'^2 about as large as (silu / g)^2 on average), the
    second adds 0.024: sqrt(0.036^2 + 0.024^2) = 0.043 of the output's norm,
    bf16 (2^-8) next to nothing.  0.06 leaves room for the averages; a
    misplaced scale or block is off by far more."""
    x, r = rand((m, 520), 30, torch.bfloat16), rand((m, 520), 29, torch.bfloat16)
    norm_weight, gate_up, down = mlp_weights()
    y, hidden = mlp(x, r, norm_weight, gate_up, down)
    h = x.double() + r.double()
    z = h / torch.sqrt(h.square().mean(dim=1, keepdim=True) + 1e-5)
    g, u = (z @ values(*gate_up, BLOCK).t()).chunk(2, dim=1)
    want = (g / (1 + torch.exp(-g)) * u) @ values(*down, BLOCK).t()
    assert torch.linalg.norm(y.double() - want) < 0.06 * torch.linalg.norm(want)
    assert torch.equal(hidden, (x.float() + r.float()).to(torch.bfloat16))


@pytest.mark.parametrize("m", [1, 400])
def test_mlp_captured_and_on_another_stream(m):
    x, r = rand((m, 520), 33, torch.bfloat16), rand((m, 520), 34, torch.bfloat16)
    weights = mlp_weights()
    want, _ = mlp(x, r, *weights)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other, _ = mlp(x, r, *weights)
    graphs = []
    for _ in range(2):  # two graphs of the same calls share nothing
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = mlp(x, r, *weights)
        graphs.append((g, out))
    torch.cuda.current_stream().wait_stream(side)
    x2 = rand((m, 520), 35, torch.bfloat16)
    want2, hidden2 = mlp(x2, r, *weights)
    x.copy_(x2)
    for g, out in graphs:
        out[0].zero_()
        side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graphs[0][0].replay()  # while the other replays on this stream
    graphs[1][0].replay()
    torch.cuda.synchronize()
    assert torch.equal(want, other)
    for _, out in graphs:
        assert torch.equal(out[0], want2) and torch.equal(out[1], hidden2)


FIRST_CALLS = """
import torch
from llvq_paper_reproduction_b200 import fp8
x = torch.randn(600, 520, device="cuda").to(torch.bfloat16)
w = torch.ones(520, device="cuda", dtype=torch.bfloat16)
a, b = fp8.quantize_rows(x[:1]), fp8.quantize_blocks(x)
try:
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        fp8.gemm(*a, *b)
except RuntimeError as e:
    assert "before capturing" in str(e), e
else:
    raise AssertionError("the error flag would have been taken from the graph's memory")
torch.cuda.synchronize()
fp8.gemm(*a, *b)  # one size only: the other kernels are first called in the capture
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    q, s, h = fp8.rms_norm(x, w, residual=x)
    y = fp8.gemm(q, s, *b)
    z = fp8.swiglu(y, y)
g.replay()
torch.cuda.synchronize()
q2, s2, h2 = fp8.rms_norm(x, w, residual=x)
y2 = fp8.gemm(q2, s2, *b)
assert torch.equal(y, y2) and torch.equal(h, h2) and y.isfinite().all()
assert torch.equal(z[0].float(), fp8.swiglu(y2, y2)[0].float())
print("fine")
"""


def test_first_calls_inside_a_capture():
    """In a fresh process: kernels whose first call is captured, and the
    product's demand for one call before."""
    import subprocess
    import sys

    from conftest import ROOT

    done = subprocess.run([sys.executable, "-c", FIRST_CALLS], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and done.stdout.strip() == "fine", done.stderr[-2000:]


@pytest.mark.parametrize("m", [1, 40, 300, 2500])
def test_calls_read_what_the_call_before_wrote(m):
    """A call starts while the one ahead of it ends; the allocator hands the
    same memory out again and again, so anything read early would be old."""
    x0 = rand((m, 512), 5, torch.bfloat16)
    norm_weight = rand((512,), 6, torch.bfloat16)
    from llvq_paper_reproduction_b200 import fp8

    gate_up = fp8.quantize_blocks(rand((1024, 512), 7, torch.bfloat16))
    down = fp8.quantize_blocks(rand((512, 512), 8, torch.bfloat16))

    def chain(pause):
        x, hidden = x0, torch.zeros_like(x0)
        for _ in range(30):
            q, s, hidden = fp8.rms_norm(x, norm_weight, residual=hidden)
            pause()
            y = fp8.gemm(q, s, *gate_up)
            pause()
            q, s = fp8.swiglu(*y.chunk(2, dim=1))
            pause()
            x = fp8.gemm(q, s, *down)
            pause()
            q, s = fp8.quantize_rows(x)
            pause()
            x = x + fp8.gemm(q, s, *down)
            pause()
        return x, hidden

    want = chain(torch.cuda.synchronize)
    for _ in range(3):
        got = chain(lambda: None)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert bool(want[0].isfinite().all())


@pytest.mark.parametrize("m", [1, 40, 300])
def test_two_streams_that_join(m):
    """Activations on one stream, the weight on another, the product behind
    both: eagerly and as a graph with two branches, with inputs that change."""
    from llvq_paper_reproduction_b200 import fp8

    x, w = rand((m, 768), 0, torch.bfloat16), rand((1500, 768), 1, torch.bfloat16)
    norm_weight = torch.ones(768, device="cuda")
    side = torch.cuda.Stream()

    def forked():
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        q, s = fp8.rms_norm(x, norm_weight)
        with torch.cuda.stream(side):
            wq, ws = fp8.quantize_blocks(w)
        main.wait_stream(side)
        for t in (wq, ws):
            t.record_stream(main)
        return fp8.gemm(q, s, wq, ws)

    def plain():
        return fp8.gemm(*fp8.rms_norm(x, norm_weight), *fp8.quantize_blocks(w), check=True)

    assert torch.equal(forked(), plain())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = forked()
    for seed in range(2, 7):
        x.copy_(rand((m, 768), seed))
        w.copy_(rand((1500, 768), seed + 10))
        graph.replay()
        assert torch.equal(y, plain())


def test_check_is_refused_inside_a_capture():
    from llvq_paper_reproduction_b200 import fp8

    ops = operands(5, 256, 384)
    want = fp8.gemm(*ops, check=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="capture"):
            fp8.gemm(*ops, check=True)
        y = fp8.gemm(*ops)  # the capture is still whole
    graph.replay()
    fp8.raise_pending_errors()
    assert torch.equal(y, want)


def test_calls_do_not_synchronise_the_host():
    from llvq_paper_reproduction_b200 import fp8

    x, r = rand((64, 520), 36, torch.bfloat16), rand((64, 520), 37, torch.bfloat16)
    weights = mlp_weights()
    want, _ = mlp(x, r, *weights)
    torch.cuda.synchronize()
    torch.cuda._sleep(2_000_000_000)
    y, _ = mlp(x, r, *weights)
    assert not torch.cuda.current_stream().query()
    torch.cuda.synchronize()
    assert torch.equal(y, want)
    fp8.raise_pending_errors()
    assert fp8.pending_errors("cuda:0") == {"gemm_timeout": 0}


def test_dequantize_fp8():
    """Indices -> 8-bit weight -> product, against the framework's own decoder and dequant-GEMM."""
    from llvq_paper_reproduction_b200 import LeechLatticeVectorQuantizerGpu, fp8

    q = LeechLatticeVectorQuantizerGpu(max_shell=13, use_cache=False, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(40)
    idx = torch.randint(0, q.total_count, (300, 22), generator=g, device="cuda")
    scale = (torch.rand(300, generator=g, device="cuda") * 0.04 + 0.005).to(torch.float16)
    bf16 = q.dequantize_bf16(idx, scale)
    for cols in (None, 520, 0):
        w, sw = q.dequantize_fp8(idx, scale, cols=cols, check=True)
        ref = bf16 if cols is None else bf16[:, :cols]
        assert w.shape == ref.shape
        if cols != 0:
            check_quantized(w, sw, ref.double(), BLOCK, 0.0)
    w, sw = q.dequantize_fp8(q.pack_indices(idx), scale, cols=520)
    a, sa = fp8.quantize_rows(rand((70, 520), 41, torch.bfloat16))
    y = fp8.gemm(a, sa, w, sw, out_dtype=torch.float32)
    check_product(y, a, sa, w, sw)
    exact = q.gemm(values(a, sa).to(torch.bfloat16), idx, scale)
    # the weight's rounding (at most 2^-4 of a value, the bf16 activations 2^-8): well within 0.06 of the norm
    assert torch.linalg.norm(y - exact) < 0.06 * torch.linalg.norm(exact)
    for cols in (-1, 529):
        with pytest.raises(ValueError):
            q.dequantize_fp8(idx, scale, cols=cols)
