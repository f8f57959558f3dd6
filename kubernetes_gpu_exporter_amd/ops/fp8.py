"""8-bit floating point with block scales (hand-written HIP for gfx950, csrc/kernels/fp8_quant.hip
and gemm_fp8.hip): the fp8 counterpart of ops.gemm for compute pods that train or serve in 8 bits.

A tensor in 8 bits is a pair (q, scale).  `q` [rows, cols] is torch.float8_e4m3fn or
float8_e5m2; `scale` is torch.float8_e8m0fnu, one power of two for each block of 128 along the
columns and 1 row (activations, gradients: scale [rows, ceil(cols/128)]) or 128 rows (weights:
scale [ceil(rows/128), ceil(cols/128)]).  q[i, j] stands for q * scale of its block.  A block's
scale is the smallest 2^e, e >= -127, that brings its largest finite magnitude to at most the
type's largest value (448 or 57344); each value is rounded once, to nearest even.  Rows of q start
at multiples of 16 bytes and rows of scale at multiples of 4: the functions here make them so.

  quantize_fp8 / dequantize_fp8   an activation checkpoint in 8 bits, kept and given back
  transpose_fp8                   the same checkpoint by columns: the gradient of a weight reads it so
  gemm_fp8                        C = A B^T of two such operands on the matrix cores
  linear_fp8                      a linear layer on these, for training and for serving

Everything runs on torch's current stream of the tensors' device, or on `stream` (a raw handle as
in ops.gemm): then results are allocated on that stream, the inputs are kept from reuse until it
is done with them, and ordering against other streams is the caller's.  All calls can be captured
into a graph; linear_fp8's backward pass too, as any torch backward pass, only while no eager
graph of the same leaves is alive.
"""
from __future__ import annotations

import math

import torch

from .gemm import kernels

BLOCK = 128
_TYPES = {torch.float8_e4m3fn: 0, torch.float8_e5m2: 1}
_WIDE = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_E8M0 = torch.float8_e8m0fnu


def _elsewhere(stream, *tensors):
    """The context in which a call on a raw stream handle runs: torch's current stream is that
    stream, and the inputs' memory is not reused before it has passed this call."""
    device = tensors[0].device
    s = torch.cuda.ExternalStream(stream, device=device) if stream else torch.cuda.default_stream(device)
    for t in tensors:
        t.record_stream(s)
    return torch.cuda.stream(s)


def _launch(device, native, *args):
    """A native call on torch's current stream of `device`, which it makes the current device."""
    stream = torch._C._cuda_getCurrentRawStream(device.index)  # (torch.cuda.current_stream makes an object: 2 us)
    if torch.cuda.current_device() == device.index:
        native(*args, stream)
    else:
        with torch.cuda.device(device):
            native(*args, stream)


def _gpu(name, *tensors):
    device = tensors[0].device
    if device.type == "cuda":
        for t in tensors:
            if t.device != device:
                break
        else:
            return device
    raise ValueError(f"{name}: tensors must be on the same GPU, got {[str(t.device) for t in tensors]}")


def _empty(rows, cols, dtype, pad, device):
    """[rows, cols] of 1-byte values whose rows start at multiples of `pad` bytes."""
    ld = -(-cols // pad) * pad
    t = torch.empty((rows, ld), dtype=dtype, device=device)
    return t if ld == cols else t[:, :cols]


def _held(rows, cols, dtype, block_rows, device):
    return (_empty(rows, cols, dtype, 16, device),
            _empty(-(-rows // block_rows), -(-cols // BLOCK), _E8M0, 4, device))


def _row_stride(name, t, rows, cols, pad):
    """Bytes between rows of a 1-byte tensor [rows, cols] whose rows start at multiples of `pad`."""
    if not (rows and cols):
        return -(-cols // pad) * pad
    ld, step = t.stride()
    if cols > 1 and step != 1:
        raise ValueError(f"{name} must have its columns next to each other, got strides {(ld, step)}")
    if rows == 1:
        ld = -(-cols // pad) * pad
    if ld % pad or ld < cols or t.data_ptr() % pad:
        raise ValueError(f"{name}'s rows must start at multiples of {pad} bytes and not overlap (row stride "
                         f"{ld}, address % {pad} = {t.data_ptr() % pad}); quantize_fp8 makes such tensors")
    return ld


def _operand(name, q, scale):
    """(q, scale, ld, lds, block_rows, type) of a checked pair, for the native calls."""
    if q.dtype not in _TYPES:
        raise TypeError(f"{name} must be float8_e4m3fn or float8_e5m2, got {q.dtype}")
    if scale.dtype != _E8M0:
        raise TypeError(f"the scales of {name} must be float8_e8m0fnu, got {scale.dtype}")
    if q.dim() != 2 or scale.dim() != 2:
        raise ValueError(f"{name} and its scales must be 2-dimensional, got {tuple(q.shape)} and {tuple(scale.shape)}")
    rows, cols = q.shape
    nb, scale_shape = -(-cols // BLOCK), scale.shape
    if scale_shape == (rows, nb):
        block_rows = 1
    elif scale_shape == (-(-rows // BLOCK), nb):
        block_rows = BLOCK
    else:
        raise ValueError(f"the scales of {name} {tuple(q.shape)} must be {(rows, nb)} (blocks of 1 x 128) or "
                         f"{(-(-rows // BLOCK), nb)} (128 x 128), got {tuple(scale.shape)}")
    ld = _row_stride(name, q, rows, cols, 16)
    lds = _row_stride(name + "'s scale", scale, scale_shape[0], nb, 4)
    if not (rows and cols):  # (no address where there is nothing: an empty view may have any)
        return 0, 0, ld, lds, block_rows, _TYPES[q.dtype]
    return q.data_ptr(), scale.data_ptr(), ld, lds, block_rows, _TYPES[q.dtype]


def _wide(name, x):
    if x.dtype not in _WIDE:
        raise TypeError(f"{name} must be bfloat16, float16 or float32, got {x.dtype}")
    if x.dim() != 2:
        raise ValueError(f"{name} must be 2-dimensional, got {tuple(x.shape)}")
    rows, cols = x.shape
    if not _row_major(x):
        raise ValueError(f"{name} must be row-major with its columns next to each other, got strides {tuple(x.stride())}")
    return x.stride(0) if rows > 1 else cols


def _row_major(x):
    """Columns next to each other, rows that do not overlap."""
    rows, cols = x.shape
    return not x.numel() or ((cols == 1 or x.stride(1) == 1) and (rows == 1 or x.stride(0) >= cols))


def _quantize(x, dtype, block_rows, rows=True, columns=False):
    """((q, scale) or None, (q^T, scale) or None), both in one pass over x."""
    if dtype not in _TYPES:
        raise TypeError(f"quantize_fp8 makes float8_e4m3fn or float8_e5m2, not {dtype}")
    if block_rows not in (1, BLOCK):
        raise ValueError(f"block_rows is 1 or {BLOCK}, got {block_rows}")
    ld = _wide("x", x)
    device = _gpu("quantize_fp8", x)
    m, k = x.shape
    out = _held(m, k, dtype, block_rows, device) if rows else None
    out_t = _held(k, m, dtype, block_rows, device) if columns else None
    if m and k:
        args = []
        for o in (out, out_t):
            args += [0, 0, 0, 0] if o is None else [o[0].data_ptr(), o[1].data_ptr(), o[0].stride(0), o[1].stride(0)]
        _launch(device, kernels().quantize_fp8, x.data_ptr(), _WIDE[x.dtype], ld, m, k, _TYPES[dtype], block_rows,
                *args)
    return out, out_t


def quantize_fp8(x, dtype=torch.float8_e4m3fn, block_rows: int = 1, stream=None):
    """x [rows, cols] (bf16, f16 or f32, columns next to each other, any row stride) in 8 bits:
    (q, scale).  block_rows 1: a scale for each 128 values of a row (activations, gradients);
    128: for each 128 x 128 block (weights).  Infinities and NaN do not count for a scale; they
    become the type's NaN (e4m3) or stay as they are (e5m2)."""
    if stream is not None:
        _gpu("quantize_fp8", x)
        with _elsewhere(stream, x):
            return quantize_fp8(x, dtype, block_rows)
    return _quantize(x, dtype, block_rows)[0]


def dequantize_fp8(q, scale, dtype=torch.bfloat16, stream=None):
    """The values that (q, scale) stands for, [rows, cols] contiguous, in bf16, f16 or f32.  Exact
    wherever `dtype` has the exponent's range."""
    op = _operand("q", q, scale)
    if dtype not in _WIDE:
        raise TypeError(f"dequantize_fp8 gives bfloat16, float16 or float32, not {dtype}")
    device = _gpu("dequantize_fp8", q, scale)
    if stream is not None:
        with _elsewhere(stream, q, scale):
            return dequantize_fp8(q, scale, dtype)
    rows, cols = q.shape
    x = torch.empty((rows, cols), dtype=dtype, device=device)
    if rows and cols:
        _launch(device, kernels().dequantize_fp8, *op, rows, cols, x.data_ptr(), _WIDE[dtype], cols)
    return x


def transpose_fp8(q, scale, stream=None):
    """The transpose [cols, rows] of a tensor in 8 bits, itself in 8 bits: (q_t, scale_t).  Blocks
    of 128 x 128 stay what they are.  Blocks of 1 x 128 become blocks of 1 x 128 along the
    transpose's own rows: the values are quantised anew from what they stand for, which, both
    scales being powers of two, changes only values below the type's normal range in their new
    block (2^-14 of its largest for e4m3, 2^-29 for e5m2, and less)."""
    op = _operand("q", q, scale)
    device = _gpu("transpose_fp8", q, scale)
    if stream is not None:
        with _elsewhere(stream, q, scale):
            return transpose_fp8(q, scale)
    rows, cols = q.shape
    qt, st = _held(cols, rows, q.dtype, op[4], device)
    if rows and cols:
        _launch(device, kernels().transpose_fp8, *op, rows, cols, qt.data_ptr(), st.data_ptr(), qt.stride(0),
                st.stride(0))
    return qt, st


def gemm_fp8(a, a_scale, b, b_scale, out=None, out_dtype=torch.bfloat16, stream=None, variant: int = 0):
    """out[M, N] = a[M, K] @ b[N, K]^T for operands in 8 bits with their block scales; each may be
    e4m3 or e5m2 and have blocks of 1 x 128 or 128 x 128.  Any M, N, K >= 0 (K = 0 gives zeros).
    Sums are held in 32 bits and rounded once into bf16 or f16 (`out_dtype`, or `out`'s type; `out`
    needs its columns next to each other, its rows may be further apart).  The matrix instruction
    drops a product 2^-14 and more below the largest of the 32 it adds at once.  variant 0 picks the
    kernel by the sizes; 1 / 2 force the 128x128 / 256x256 tile (the
    latter for K >= 144), 3 / 6 the kernel for few rows (M <= 16) with 16 / 32
    rows of b per wave, 4 the 64x64 tile, 5 the 128x128 tile with two blocks per CU."""
    oa, ob = _operand("a", a, a_scale), _operand("b", b, b_scale)
    (M, K), N = a.shape, b.shape[0]
    if b.shape[1] != K:
        raise ValueError(f"shape mismatch {tuple(a.shape)} x {tuple(b.shape)}^T")
    dtype = out_dtype if out is None else out.dtype
    if dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"gemm_fp8 writes bfloat16 or float16, not {dtype}")
    if out is not None and (tuple(out.shape) != (M, N) or not _row_major(out)):
        raise ValueError(f"out must be {(M, N)} with its columns next to each other, got {tuple(out.shape)}, strides "
                         f"{tuple(out.stride())}")
    device = _gpu("gemm_fp8", a, a_scale, b, b_scale, *([] if out is None else [out]))
    if stream is not None:
        with _elsewhere(stream, a, a_scale, b, b_scale, *([] if out is None else [out])):
            return gemm_fp8(a, a_scale, b, b_scale, out, out_dtype, variant=variant)
    if out is None:
        out = torch.empty((M, N), dtype=dtype, device=device)
    if M and N:
        _launch(device, kernels().gemm_fp8, *oa, *ob, out.data_ptr(), out.stride(0) if M > 1 else N, M, N, K,
                _WIDE[dtype], variant)
    return out


def _forward(x, weight, want_dx, want_dw):
    """(y, what the backward pass needs) of x [M, K] and weight [N, K], one native call."""
    (M, K), N = x.shape, weight.shape[0]
    kept_bytes, temp_bytes, _ = kernels().linear_fp8_bytes(M, N, K, want_dx, want_dw)
    y = x.new_empty((M, N))
    kept = torch.empty(kept_bytes, dtype=torch.uint8, device=x.device)
    temp = torch.empty(temp_bytes, dtype=torch.uint8, device=x.device)
    _launch(x.device, kernels().linear_fp8_forward, M, N, K, want_dx, want_dw, x.data_ptr(), _wide("x", x),
            _WIDE[x.dtype], weight.data_ptr(), _wide("weight", weight), _WIDE[weight.dtype], kept.data_ptr(),
            temp.data_ptr(), y.data_ptr())
    return y, kept


class _LinearFp8(torch.autograd.Function):
    """y = x W^T with both operands in 8 bits; what it keeps for the backward pass is in 8 bits."""

    @staticmethod
    def forward(ctx, x, weight):
        ctx.want = ctx.needs_input_grad
        ctx.sizes = x.shape[0], weight.shape[0], x.shape[1]
        ctx.weight_dtype = weight.dtype
        y, kept = _forward(x, weight, *ctx.want)
        ctx.save_for_backward(kept)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        (kept,), (M, N, K), (want_dx, want_dw) = ctx.saved_tensors, ctx.sizes, ctx.want
        grad = _rows(grad)
        dx = grad.new_empty((M, K)) if want_dx else None
        dw = torch.empty((N, K), dtype=ctx.weight_dtype, device=grad.device) if want_dw else None
        temp = torch.empty(kernels().linear_fp8_bytes(M, N, K, want_dx, want_dw)[2], dtype=torch.uint8,
                           device=grad.device)
        _launch(grad.device, kernels().linear_fp8_backward, M, N, K, want_dx, want_dw, grad.data_ptr(),
                _wide("grad", grad), _WIDE[grad.dtype], _WIDE[ctx.weight_dtype], kept.data_ptr(), temp.data_ptr(),
                dx.data_ptr() if want_dx else 0, dw.data_ptr() if want_dw else 0)
        return dx, dw


def _serve(x, N, op):
    """y of x [M, K] and a weight [N, K] in 8 bits (`op`: its checked operand), one native call."""
    M, K = x.shape
    y = x.new_empty((M, N))
    temp = torch.empty(kernels().serve_fp8_bytes(M, N, K), dtype=torch.uint8, device=x.device)
    _launch(x.device, kernels().serve_fp8, x.data_ptr(), _WIDE[x.dtype], _wide("x", x), *op, M, N, K, y.data_ptr(),
            temp.data_ptr())
    return y


class _ServeFp8(torch.autograd.Function):
    """The same with a weight that is in 8 bits already and takes no gradient."""

    @staticmethod
    def forward(ctx, x, weight, weight_scale, op):
        ctx.save_for_backward(weight, weight_scale)
        return _serve(x, weight.shape[0], op)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        gq = quantize_fp8(_rows(grad))
        return gemm_fp8(*gq, *transpose_fp8(*ctx.saved_tensors), out_dtype=grad.dtype), None, None, None


def _rows(x):
    """x [rows, cols] with its columns next to each other and rows that do not overlap (a copy if need be)."""
    return x if _row_major(x) else x.contiguous()


def linear_fp8(x, weight, weight_scale=None):
    """y[..., N] = x[..., K] @ weight[N, K]^T in 8 bits, in x's type (bf16 or f16).

    Training: `weight` in bf16 or f16.  Both operands are quantised to e4m3 (x in blocks of 1 x 128,
    the weight 128 x 128).  For the backward pass x is kept as its 8-bit checkpoint, half the memory
    of the activation; dx = Q(dy) W with the kept 8-bit weight, dW = Q(dy^T) x with the checkpoint
    transposed (as transpose_fp8 does).  A double backward is refused.

    Serving: `weight` in 8 bits with its `weight_scale`, as quantize_fp8(w, block_rows=128) gives
    them; x may take a gradient, the weight takes none."""
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"shape mismatch {tuple(x.shape)} x {tuple(weight.shape)}^T")
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"linear_fp8 takes bfloat16 or float16 activations, got {x.dtype}")
    x2 = x if x.dim() == 2 else x.reshape(math.prod(x.shape[:-1]), x.shape[-1])
    grad = torch.is_grad_enabled()
    if weight_scale is None:
        if weight.dtype not in (torch.bfloat16, torch.float16):
            raise TypeError("linear_fp8 takes bfloat16 or float16 weights, or 8-bit ones with weight_scale, got "
                            f"{weight.dtype}")
        _gpu("linear_fp8", x, weight)
        x2, weight = _rows(x2), _rows(weight)
        y = _LinearFp8.apply(x2, weight) if grad and (x2.requires_grad or weight.requires_grad) else \
            _forward(x2, weight, False, False)[0]
    else:
        if weight.requires_grad:
            raise ValueError("weights in 8 bits take no gradient")
        op = _operand("weight", weight, weight_scale)
        _gpu("linear_fp8", x, weight, weight_scale)
        x2 = _rows(x2)
        y = _ServeFp8.apply(x2, weight, weight_scale, op) if grad and x2.requires_grad else _serve(x2, weight.shape[0], op)
    return y if x.dim() == 2 else y.reshape(*x.shape[:-1], y.shape[1])
