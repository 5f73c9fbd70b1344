"""The 8-bit operators as a serving program calls them: what is timed, on
which sizes, and their plain forms.

Operators (e4m3 values, one fp32 scale per block of 128 columns):
  gemm    a[m, k] x w[n, k]^T with scales per 1 x 128 (a) and 128 x 128 (w)
  norm    residual addition, RMS norm and 8-bit output with scales
  swiglu  silu(gate) * up with 8-bit output and scales
  rows    8-bit activations, a scale per 1 x 128 block
  blocks  8-bit weights, a scale per 128 x 128 block

The sizes are those of the Llama-2-7B and Llama-3-8B linears that the
framework's benchmark and whole-model path use (4096, 11008, 14336), and odd
ones around them.
"""
import math

import torch

own = False

BLOCK = 128
E4M3_MAX = 448.0
FLOOR = 2.0 ** -100  # smallest largest-magnitude a scale is made from
EPS = 1e-5
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one token through the gate projection: bound by the weight's bytes
        {"name": "gemm_token", "op": "gemm", "m": 1, "n": 14336, "k": 4096, "out": "bf16"},
        # a batch of 64 sequences, one token each, through the down projection
        {"name": "gemm_batch64", "op": "gemm", "m": 64, "n": 4096, "k": 14336, "out": "bf16"},
        # a short prompt on odd sizes: ragged tiles in all three directions, 32-bit output
        {"name": "gemm_ragged", "op": "gemm", "m": 517, "n": 4100, "k": 2200, "out": "fp32"},
        # a long prompt through the gate projection: bound by the tensor cores
        {"name": "gemm_prompt", "op": "gemm", "m": 4096, "n": 14336, "k": 4096, "out": "bf16"},
        # one token before a projection: latency
        {"name": "norm_token", "op": "norm", "m": 1, "k": 4096, "dtype": "bf16", "residual": True},
        # a long prompt before a projection
        {"name": "norm_prompt", "op": "norm", "m": 8192, "k": 4096, "dtype": "bf16", "residual": True},
        # a batch of 64 single tokens between the two products of an MLP
        {"name": "swiglu_batch64", "op": "swiglu", "m": 64, "k": 14336, "dtype": "bf16"},
        # a long prompt between the two products, the other model's width
        {"name": "swiglu_prompt", "op": "swiglu", "m": 4096, "k": 11008, "dtype": "bf16"},
        # attention outputs of a small odd batch before the output projection
        {"name": "rows_odd", "op": "rows", "m": 37, "k": 4100, "dtype": "fp16"},
        # attention outputs of a long prompt before the output projection
        {"name": "rows_prompt", "op": "rows", "m": 8192, "k": 4096, "dtype": "bf16"},
        # laying a small odd weight out in 8 bits
        {"name": "blocks_odd", "op": "blocks", "m": 1000, "k": 1100, "dtype": "fp16"},
        # laying a down projection out in 8 bits
        {"name": "blocks_down", "op": "blocks", "m": 4096, "k": 14336, "dtype": "bf16"},
    ]


def _log_uniform(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["gemm", "gemm", "gemm", "norm", "swiglu", "rows", "blocks"])
    if op == "gemm":
        # the product of a fused gate-and-up projection (28672) down to a small odd layer
        m, n, k = _log_uniform(rng, 1, 8192), _log_uniform(rng, 128, 28672), _log_uniform(rng, 128, 14336)
        if rng.random() < 0.5:  # half of them on whole blocks, as most models have it
            n, k = (n + 127) // 128 * 128, (k + 127) // 128 * 128
        m = max(1, min(m, 4096 * 14336 * 4096 // (n * k)))
        return {"op": op, "m": m, "n": n, "k": k, "out": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    m, k = _log_uniform(rng, 1, 8192), _log_uniform(rng, 128, 16384)
    if rng.random() < 0.5:
        k = (k + 127) // 128 * 128
    m = max(1, min(m, 8192 * 4096 // k))
    case = {"op": op, "m": m, "k": k, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    if op == "norm":
        case["residual"] = rng.random() < 0.75
    return case


# ------------------------------------------------------------------ inputs
def _activations(m, k, g):
    """Normal values with a few columns about twenty times as large, as a model's residual stream has them."""
    x = torch.randn((m, k), generator=g, device="cuda")
    return x * torch.where(torch.rand(k, generator=g, device="cuda") < 0.005, 20.0, 1.0)


def _weights(n, k, g):
    """Normal rows, their standard deviation log-normal around 0.02."""
    sigma = torch.exp(math.log(0.02) + 0.5 * torch.randn((n, 1), generator=g, device="cuda"))
    return torch.randn((n, k), generator=g, device="cuda") * sigma


def _rows_of_16_bytes(q):
    """8-bit rows that start on 16-byte boundaries, whatever their length."""
    m, k = q.shape
    held = torch.zeros((m, (k + 15) // 16 * 16), dtype=torch.uint8, device=q.device)
    held[:, :k] = q.view(torch.uint8)
    return held.view(torch.float8_e4m3fn)[:, :k]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, m, k = case["op"], case["m"], case["k"]
    if op == "gemm":
        a, a_scale = _plain_rows(_activations(m, k, g))
        w, w_scale = _plain_blocks(_weights(case["n"], k, g))
        # row scales lie block by block, as the quantizers leave them
        return {"op": op, "a": _rows_of_16_bytes(a), "a_scale": a_scale.t().contiguous().t(),
                "w": _rows_of_16_bytes(w), "w_scale": w_scale, "out": DTYPES[case["out"]]}
    dtype = DTYPES[case["dtype"]]
    if op == "norm":
        state = {"op": op, "x": _activations(m, k, g).to(dtype), "residual": None,
                 "weight": (1.0 + 0.1 * torch.randn(k, generator=g, device="cuda")).to(dtype)}
        if case["residual"]:
            state["residual"] = _activations(m, k, g).to(dtype)
        return state
    if op == "swiglu":  # gate and up are the halves of one product's rows
        return {"op": op, "gate_up": torch.randn((m, 2 * k), generator=g, device="cuda").to(dtype)}
    return {"op": op, "x": (_activations(m, k, g) if op == "rows" else _weights(m, k, g)).to(dtype)}


# ------------------------------------------------------------------ plain forms
def _pad_columns(x, value=0.0):
    return torch.nn.functional.pad(x, (0, -x.shape[1] % BLOCK), value=value)


def _plain_rows(y):
    """fp32 [m, k] -> e4m3 [m, k] and fp32 scales [m, ceil(k / 128)]."""
    m, k = y.shape
    tiles = _pad_columns(y).view(m, -1, BLOCK)
    amax = tiles.abs().amax(dim=2).clamp(min=FLOOR)
    q = (tiles * (E4M3_MAX / amax)[:, :, None]).clamp(-E4M3_MAX, E4M3_MAX)
    return q.view(m, -1)[:, :k].to(torch.float8_e4m3fn), amax / E4M3_MAX


def _plain_blocks(w):
    """fp32 [n, k] -> e4m3 [n, k] and fp32 scales [ceil(n / 128), ceil(k / 128)]."""
    n, k = w.shape
    tiles = torch.nn.functional.pad(w, (0, -k % BLOCK, 0, -n % BLOCK))
    nb, kb = tiles.shape[0] // BLOCK, tiles.shape[1] // BLOCK
    tiles = tiles.view(nb, BLOCK, kb, BLOCK)
    amax = tiles.abs().amax(dim=(1, 3)).clamp(min=FLOOR)
    q = (tiles * (E4M3_MAX / amax)[:, None, :, None]).clamp(-E4M3_MAX, E4M3_MAX)
    return q.view(nb * BLOCK, kb * BLOCK)[:n, :k].to(torch.float8_e4m3fn), amax / E4M3_MAX


def _plain_gemm(s):
    k, n = s["a"].shape[1], s["w"].shape[0]
    a = s["a"].float() * s["a_scale"].repeat_interleave(BLOCK, dim=1)[:, :k]
    spread = s["w_scale"].repeat_interleave(BLOCK, dim=0)[:n].repeat_interleave(BLOCK, dim=1)[:, :k]
    return (a @ (s["w"].float() * spread).t()).to(s["out"])


def _plain_norm(s):
    h = s["x"].float()
    if s["residual"] is not None:
        h = h + s["residual"].float()
    y = h * torch.rsqrt(h.square().mean(dim=1, keepdim=True) + EPS) * s["weight"].float()
    q, scale = _plain_rows(y)
    return (q, scale) if s["residual"] is None else (q, scale, h.to(s["x"].dtype))


def run(s):
    op = s["op"]
    if own:
        from llvq_paper_reproduction_b200 import fp8
        if op == "gemm":
            return fp8.gemm(s["a"], s["a_scale"], s["w"], s["w_scale"], out_dtype=s["out"])
        if op == "norm":
            return fp8.rms_norm(s["x"], s["weight"], eps=EPS, residual=s["residual"])
        if op == "swiglu":
            gate, up = s["gate_up"].chunk(2, dim=1)
            return fp8.swiglu(gate, up)
        return fp8.quantize_rows(s["x"]) if op == "rows" else fp8.quantize_blocks(s["x"])
    if op == "gemm":
        return _plain_gemm(s)
    if op == "norm":
        return _plain_norm(s)
    if op == "swiglu":
        gate, up = s["gate_up"].float().chunk(2, dim=1)
        return _plain_rows(gate / (1.0 + torch.exp(-gate)) * up)
    return _plain_rows(s["x"].float()) if op == "rows" else _plain_blocks(s["x"].float())


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    op, m, k = case["op"], case["m"], case["k"]
    kb = (k + BLOCK - 1) // BLOCK
    if op == "gemm":
        n = case["n"]
        nb = (n + BLOCK - 1) // BLOCK
        return {"bytes": m * k + n * k + 4 * (m * kb + nb * kb) + m * n * SIZE[case["out"]], "flops": 2 * m * n * k}
    size = SIZE[case["dtype"]]
    if op == "norm":
        extra = 2 * m * k * size if case["residual"] else 0
        return {"bytes": m * k * size + extra + k * size + m * k + 4 * m * kb, "flops": 8 * m * k}
    if op == "swiglu":
        return {"bytes": 2 * m * k * size + m * k + 4 * m * kb, "flops": 8 * m * k}
    scales = m * kb if op == "rows" else (m + BLOCK - 1) // BLOCK * kb
    return {"bytes": m * k * size + m * k + 4 * scales, "flops": 3 * m * k}


# ------------------------------------------------------------------ the definitions in 64 bits
def _e4m3(v):
    """The nearest e4m3 value of each 64-bit one: 3 fraction bits, exponents from -6, ties to even, at most 448."""
    _, e = torch.frexp(v)
    step = torch.exp2((e - 1).clamp(min=-6).double() - 3)
    return (torch.round(v / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def _exact_rows(y):
    m, k = y.shape
    kb = (k + BLOCK - 1) // BLOCK
    scale = torch.empty((m, kb), dtype=torch.float64, device=y.device)
    q = torch.empty_like(y)
    for b in range(kb):
        part = y[:, b * BLOCK:(b + 1) * BLOCK]
        scale[:, b] = part.abs().amax(dim=1).clamp(min=FLOOR) / E4M3_MAX
        q[:, b * BLOCK:(b + 1) * BLOCK] = _e4m3(part / scale[:, b:b + 1])
    return q, scale


def exact(case, seed):
    s = prepare(case, seed)
    op = s["op"]
    if op == "gemm":
        a, w = s["a"].double(), s["w"].double()
        y = torch.zeros((a.shape[0], w.shape[0]), dtype=torch.float64, device="cuda")
        for b in range(s["a_scale"].shape[1]):
            cols = slice(b * BLOCK, (b + 1) * BLOCK)
            by_row = s["w_scale"][:, b].double()[torch.arange(w.shape[0], device="cuda") // BLOCK]
            y += (a[:, cols] * s["a_scale"][:, b:b + 1].double()) @ (w[:, cols] * by_row[:, None]).t()
        return y
    if op == "norm":
        h = s["x"].double() + (0 if s["residual"] is None else s["residual"].double())
        y = s["weight"].double() * h / torch.sqrt((h * h).sum(dim=1, keepdim=True) / h.shape[1] + EPS)
        q, scale = _exact_rows(y)
        return (q, scale) if s["residual"] is None else (q, scale, h)
    if op == "swiglu":
        k = case["k"]
        gate, up = s["gate_up"][:, :k].double(), s["gate_up"][:, k:].double()
        return _exact_rows(gate * torch.sigmoid(gate) * up)
    x = s["x"].double()
    if op == "rows":
        return _exact_rows(x)
    q, scales = torch.empty_like(x), []
    for i in range(0, x.shape[0], BLOCK):
        # the block of rows laid out as one row per column block
        part = x[i:i + BLOCK]
        wide = torch.nn.functional.pad(part, (0, -part.shape[1] % BLOCK))
        largest = wide.abs().amax(dim=0).view(-1, BLOCK).amax(dim=1).clamp(min=FLOOR)
        scales.append(largest / E4M3_MAX)
        by_column = scales[-1][torch.arange(x.shape[1], device="cuda") // BLOCK]
        q[i:i + BLOCK] = _e4m3(part / by_column)
    return q, torch.stack(scales)
