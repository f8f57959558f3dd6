"""The 8-bit operators of the compute pods, as a pod's program calls them, and their plain forms.

Numbers are held in 8-bit floating point (e4m3: 4 significant bits, up to 448; e5m2: 3 significant
bits, up to 57344) with one power of two for each block of 128 values.  The operators:

  checkpoint   an activation kept in 8 bits between the forward and the backward pass, and given back:
               by rows as it was stored, or with its columns in front and blocks along the tokens, the
               form in which the gradient of a weight reads it
  gemm         C[M,N] = A[M,K] B[N,K]^T of two operands in 8 bits with their block scales
  serve        a linear layer with weights in 8 bits, for few tokens or a prompt
  train        a linear layer's forward and backward pass, its input kept as an 8-bit checkpoint

A block's scale is 2^e with the smallest e for which its largest finite magnitude is at most the
largest value of the 8-bit type (e = 0 for a block of zeros); its values are rounded once, to the
nearest, ties to even, after the exact division by 2^e.

`own` false: elementary torch operations in 32 bits; true: the package's kernels.
"""
import math

import torch

own = False

BLOCK = 128
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32,
          "e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
LARGEST = {torch.float8_e4m3fn: 448.0, torch.float8_e5m2: 57344.0}


def listed():
    return [
        # one decoded token's activations kept and given back: launches and nothing else
        {"name": "checkpoint_token", "kind": "checkpoint", "rows": 1, "cols": 4096, "dtype": "bf16", "columns": False},
        # a ragged batch, partial blocks at both ends, float16 activations
        {"name": "checkpoint_ragged", "kind": "checkpoint", "rows": 1000, "cols": 5001, "dtype": "f16", "columns": False},
        # a full batch's activations: memory bandwidth
        {"name": "checkpoint_batch", "kind": "checkpoint", "rows": 8192, "cols": 8192, "dtype": "bf16", "columns": False},
        # the same kept for the gradient of a weight, which reads it by columns
        {"name": "checkpoint_columns", "kind": "checkpoint", "rows": 8192, "cols": 4096, "dtype": "bf16", "columns": True},
        # one token's product: the weights are read once, memory bandwidth
        {"name": "gemm_token", "kind": "gemm", "rows": 1, "cols": 8192, "inner": 8192, "a": "e4m3", "b": "e4m3",
         "b_block": 128, "out": "bf16"},
        # odd and ragged sizes, mixed types, a scale for each row of both operands
        {"name": "gemm_ragged", "kind": "gemm", "rows": 333, "cols": 1001, "inner": 2050, "a": "e5m2", "b": "e4m3",
         "b_block": 1, "out": "f16"},
        # the two sizes of the compute pods
        {"name": "gemm_4096", "kind": "gemm", "rows": 4096, "cols": 4096, "inner": 4096, "a": "e4m3", "b": "e4m3",
         "b_block": 128, "out": "bf16"},
        {"name": "gemm_8192", "kind": "gemm", "rows": 8192, "cols": 8192, "inner": 8192, "a": "e4m3", "b": "e4m3",
         "b_block": 128, "out": "bf16"},
        # a decoding batch of 16 sequences
        {"name": "serve_batch", "kind": "serve", "rows": 16, "cols": 4096, "inner": 8192, "dtype": "bf16"},
        # a prompt of 512 tokens
        {"name": "serve_prompt", "kind": "serve", "rows": 512, "cols": 8192, "inner": 4096, "dtype": "bf16"},
        # a small ragged training step in float16
        {"name": "train_ragged", "kind": "train", "rows": 1000, "cols": 1500, "inner": 2000, "dtype": "f16"},
        # a large training step
        {"name": "train_batch", "kind": "train", "rows": 4096, "cols": 8192, "inner": 8192, "dtype": "bf16"},
    ]


def _spread(rng, low, high):
    """A size of [low, high], spread over its logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(["checkpoint", "gemm", "serve", "train"])
    if kind == "checkpoint":
        return {"kind": kind, "rows": _spread(rng, 1, 8192), "cols": _spread(rng, 16, 8192),
                "dtype": rng.choice(["bf16", "f16", "f32"]), "columns": rng.random() < 0.5}
    if kind == "gemm":
        return {"kind": kind, "rows": _spread(rng, 1, 8192), "cols": _spread(rng, 16, 8192),
                "inner": _spread(rng, 16, 8192), "a": rng.choice(["e4m3", "e5m2"]), "b": rng.choice(["e4m3", "e5m2"]),
                "b_block": rng.choice([1, 128]), "out": rng.choice(["bf16", "f16"])}
    rows = _spread(rng, 1, 2048) if kind == "serve" else _spread(rng, 1, 4096)
    return {"kind": kind, "rows": rows, "cols": _spread(rng, 64, 8192), "inner": _spread(rng, 64, 8192),
            "dtype": rng.choice(["bf16", "f16"])}


# ---- the plain form: 32 bits, elementary operations ----

def _pow2(e):
    """2^e in 32 bits for whole e in [-126, 127], from its bits."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _blocks(x, block_rows):
    """[rows / block_rows, columns / 128] blocks of x: [R, block_rows, C, 128], zeros behind the ends."""
    m, k = x.shape
    r, c = -(-m // block_rows), -(-k // BLOCK)
    full = torch.zeros(r * block_rows, c * BLOCK, dtype=x.dtype, device=x.device)
    full[:m, :k] = x
    return full.reshape(r, block_rows, c, BLOCK)


def _exponents(blocks, dtype):
    """The scale's exponent of each block: LARGEST is 1.75 * 2^p for both types."""
    size = blocks.abs()
    size = torch.where(torch.isfinite(size), size, torch.zeros_like(size))
    mantissa, exponent = torch.frexp(size.amax(dim=(1, 3)))  # mantissa in [1/2, 1)
    p = 8 if dtype == torch.float8_e4m3fn else 15
    e = exponent - 1 - p + (mantissa > 0.875).to(exponent.dtype)
    return torch.where(mantissa == 0, torch.zeros_like(e), e).clamp(-127, 127)


def _quantized(x, dtype, block_rows):
    """(8-bit values [m, k], exponents [blocks of rows, blocks of columns])."""
    m, k = x.shape
    blocks = _blocks(x.float(), block_rows)
    e = _exponents(blocks, dtype)
    q = (blocks * _pow2(-e)[:, None, :, None]).to(dtype)
    r, b, c, _ = q.shape
    return q.reshape(r * b, c * BLOCK)[:m, :k], e


def _values(q, e, block_rows):
    """The numbers that q stands for, in 32 bits."""
    m, k = q.shape
    scale = _pow2(e).repeat_interleave(block_rows, 0)[:m].repeat_interleave(BLOCK, 1)[:, :k]
    return q.float() * scale


def _rounded(x, dtype, block_rows=1):
    return _values(*_quantized(x, dtype, block_rows), block_rows)


# ---- inputs ----

def _activations(m, k, g, dtype):
    """Normal values whose spread differs by feature, a few features far larger, a few tokens of padding (zeros)."""
    x = torch.randn(m, k, device="cuda", generator=g)
    x = x * torch.exp(0.5 * torch.randn(k, device="cuda", generator=g))
    x = x * torch.where(torch.rand(k, device="cuda", generator=g) < 0.002, 30.0, 1.0)
    if m > 8:
        x = x * (torch.rand(m, 1, device="cuda", generator=g) > 0.02)
    return x.to(dtype)


def _stored(q, e):
    """An operand as a program holds it: rows that start at multiples of 16 bytes, scales in 8 bits at multiples of 4."""
    m, k = q.shape
    rows = torch.zeros(m, -(-k // 16) * 16, dtype=torch.uint8, device=q.device).view(q.dtype)
    rows[:, :k] = q
    scales = torch.zeros(e.shape[0], -(-e.shape[1] // 4) * 4, dtype=torch.uint8, device=q.device)
    scales[:, :e.shape[1]] = (e + 127).to(torch.uint8)
    return rows[:, :k], scales.view(torch.float8_e8m0fnu)[:, :e.shape[1]]


def _held(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, m = case["kind"], case["rows"]
    if kind == "checkpoint":
        return {"x": _activations(m, case["cols"], g, DTYPES[case["dtype"]])}
    n, k = case["cols"], case["inner"]
    weight = torch.randn(n, k, device="cuda", generator=g) * 0.02
    if kind == "gemm":
        a = _stored(*_quantized(_activations(m, k, g, torch.float32), DTYPES[case["a"]], 1))
        b = _stored(*_quantized(weight, DTYPES[case["b"]], case["b_block"]))
        return {"a": a[0], "a_scale": a[1], "b": b[0], "b_scale": b[1]}
    dtype = DTYPES[case["dtype"]]
    x = _activations(m, k, g, dtype)
    if kind == "serve":
        w = _stored(*_quantized(weight, torch.float8_e4m3fn, BLOCK))
        return {"x": x, "weight": w[0], "weight_scale": w[1]}
    grad = (torch.randn(m, n, device="cuda", generator=g) * 0.01).to(dtype)
    return {"x": x.requires_grad_(), "weight": weight.to(dtype).requires_grad_(), "grad": grad}


def prepare(case, seed):
    return {"case": case, **_held(case, seed)}


# ---- one pass ----

def _run_own(case, s):
    from kubernetes_gpu_exporter_amd.ops.fp8 import (dequantize_fp8, gemm_fp8, linear_fp8, quantize_fp8,
                                                     transpose_fp8)
    if case["kind"] == "checkpoint":
        q, scale = quantize_fp8(s["x"])
        if case["columns"]:
            q, scale = transpose_fp8(q, scale)
        return dequantize_fp8(q, scale, s["x"].dtype)
    if case["kind"] == "gemm":
        return gemm_fp8(s["a"], s["a_scale"], s["b"], s["b_scale"], out_dtype=DTYPES[case["out"]])
    if case["kind"] == "serve":
        return linear_fp8(s["x"], s["weight"], s["weight_scale"])
    y = linear_fp8(s["x"], s["weight"])
    return (y.detach(), *torch.autograd.grad(y, (s["x"], s["weight"]), s["grad"]))


def run(state):
    case, s = state["case"], state
    if own:
        return _run_own(case, s)
    with torch.no_grad():
        e4m3 = torch.float8_e4m3fn
        if case["kind"] == "checkpoint":
            kept = _rounded(s["x"], e4m3)
            if case["columns"]:
                kept = _rounded(kept.T.contiguous(), e4m3)
            return kept.to(s["x"].dtype)
        if case["kind"] == "gemm":
            a = _values(s["a"], s["a_scale"].view(torch.uint8).int() - 127, 1)
            b = _values(s["b"], s["b_scale"].view(torch.uint8).int() - 127, case["b_block"])
            return (a @ b.T).to(DTYPES[case["out"]])
        if case["kind"] == "serve":
            w = _values(s["weight"], s["weight_scale"].view(torch.uint8).int() - 127, BLOCK)
            return (_rounded(s["x"], e4m3) @ w.T).to(s["x"].dtype)
        x, w, grad, dtype = _rounded(s["x"], e4m3), _rounded(s["weight"], e4m3, BLOCK), s["grad"], s["x"].dtype
        y = x @ w.T
        dx = _rounded(grad, e4m3) @ w
        dw = _rounded(grad.T.contiguous(), e4m3) @ _rounded(x.T.contiguous(), e4m3).T
        return y.to(dtype), dx.to(dtype), dw.to(dtype)


# ---- 64 bits, from the definition ----

def _exact_rounded(x, largest, significant, lowest, block_rows):
    """x (64 bits) with every block rounded: `significant` bits, the exponents of the 8-bit type not below `lowest`."""
    m, k = x.shape
    r, c = -(-m // block_rows), -(-k // BLOCK)
    at = (torch.arange(m, device=x.device)[:, None] // block_rows) * c + torch.arange(k, device=x.device) // BLOCK
    top = torch.zeros(r * c, dtype=torch.float64, device=x.device)
    top.scatter_reduce_(0, at.reshape(-1), x.abs().reshape(-1), "amax")
    e = torch.ceil(torch.log2(top / largest))
    e = torch.where(top > 0, e, torch.zeros_like(e))
    power = lambda v: ((v.to(torch.int64) + 1023) << 52).view(torch.float64)  # noqa: E731
    e = torch.where((top > 0) & (top <= largest * power(e - 1)), e - 1, e)
    e = torch.where(top > largest * power(e), e + 1, e).clamp(-127, 127)
    scale = power(e)[at]
    v = x / scale
    step = torch.floor(torch.log2(torch.where(v == 0, torch.ones_like(v), v.abs())))
    step = torch.where(power(step) > v.abs(), step - 1, step)
    step = torch.where(power(step + 1) <= v.abs(), step + 1, step)
    unit = power(step.clamp(min=lowest) - (significant - 1))
    return torch.round(v / unit) * unit * scale


def exact(case, seed):
    e4m3 = (448.0, 4, -6)
    with torch.no_grad():
        s = {k: v.double() if k in ("x", "grad", "a", "b") or (k == "weight" and case["kind"] == "train") else v
             for k, v in _held(case, seed).items()}
        if case["kind"] == "checkpoint":
            kept = _exact_rounded(s["x"], *e4m3, 1)
            return _exact_rounded(kept.T.contiguous(), *e4m3, 1) if case["columns"] else kept

        def whole(q, scale, block_rows):
            m, k = q.shape
            e = scale.view(torch.uint8).to(torch.int64) - 127
            row = torch.arange(m, device=q.device) // block_rows
            col = torch.arange(k, device=q.device) // BLOCK
            return q.double() * ((e[row[:, None], col] + 1023) << 52).view(torch.float64)

        if case["kind"] == "gemm":
            return whole(s["a"], s["a_scale"], 1) @ whole(s["b"], s["b_scale"], case["b_block"]).T
        if case["kind"] == "serve":
            return _exact_rounded(s["x"], *e4m3, 1) @ whole(s["weight"], s["weight_scale"], BLOCK).T
        x, w = _exact_rounded(s["x"], *e4m3, 1), _exact_rounded(s["weight"], *e4m3, BLOCK)
        dx = _exact_rounded(s["grad"], *e4m3, 1) @ w
        dw = _exact_rounded(s["grad"].T.contiguous(), *e4m3, 1) @ _exact_rounded(x.T.contiguous(), *e4m3, 1).T
        return x @ w.T, dx, dw


def work(case):
    m, n, size = case["rows"], case["cols"], 2
    if case["kind"] == "checkpoint":  # the values in, the checkpoint out and in again, the values out
        size = torch.empty(0, dtype=DTYPES[case["dtype"]]).element_size()
        return {"bytes": m * n * (2 * size + 2), "flops": 0}
    k = case["inner"]
    if case["kind"] == "gemm":
        return {"bytes": m * k + n * k + m * n * size, "flops": 2 * m * n * k}
    if case["kind"] == "serve":
        return {"bytes": m * k * size + n * k + m * n * size, "flops": 2 * m * n * k}
    # activations, weights and the gradient in; the result and two gradients out
    return {"bytes": 2 * size * (m * k + n * k + m * n), "flops": 6 * m * n * k}
