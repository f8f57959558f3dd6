"""8-bit floating point with block scales (hand-written HIP for gfx950, csrc/kernels/fp8_quant.hip
and gemm_fp8.hip): the fp8 counterpart of ops.gemm for compute pods that train or serve in 8 bits.

A tensor in 8 bits is a pair (q, scale).  `q` [rows, cols] is torch.float8_e4m3fn or
float8_e5m2; `scale` is torch.float8_e8m0fnu, one power of two for each block of 128 along the
columns and 1 row (activations, gradients: scale [rows, ceil(cols/128)]) or 128 rows (weights:
scale [ceil(rows/128), ceil(cols/128)]).  q[i, j] stands for q * scale of its block.  A block's
scale is the smallest 2^e, e >= -127, that brings its largest finite magnitude to at most the
type's largest value (448 or 57344); each value is rounded once, to nearest even.  Rows of q start
at multiples of 16 bytes and rows of scale at multiples of 4: the functions here make them so, q's
at multiples of 128 where that takes at most an eighth more memory (q is then a view of wider rows).
clone(), contiguous(), a copy on another device or load_state_dict() into a new buffer may lay rows out
otherwise: align_fp8 puts such a copy right, once.

  quantize_fp8 / dequantize_fp8   an activation checkpoint in 8 bits, kept and given back
  align_fp8                       rows of a copy put where the others want them
  transpose_fp8                   the same checkpoint by columns: the gradient of a weight reads it so
  quantize_fp8_both               a tensor by rows and by columns in one pass
  gemm_fp8                        C = A B^T of two such operands on the matrix cores
  linear_fp8                      a linear layer on these, for training and for serving

Only linear_fp8 takes part in autograd; what the others return carries no gradient.

Everything runs on torch's current stream of the tensors' device, or on `stream` (a raw handle as
in ops.gemm): then results are allocated on that stream, the inputs are kept from reuse until it
is done with them, and ordering against other streams is the caller's.  All calls can be captured
into a graph; linear_fp8's backward pass too, as any torch backward pass, only while no eager
graph of the same leaves is alive.  To torch they are operators (torch.ops.gpuexp), so torch.jit.trace
and make_fx record them as such; a traced linear_fp8 has its gradients.  torch.compile runs them between
its graphs.
"""
from __future__ import annotations

import torch  # (first: the native module shares torch's HIP runtime)

try:
    from .. import _gpuexp_fp8 as _native
except ImportError as e:
    raise ImportError(f"native module _gpuexp_fp8 is not built; run `python build_native.py` where a ROCm "
                      f"build of torch is installed: {e}") from e


def _elsewhere(stream, *tensors):
    """The context in which a call on a raw stream handle runs: torch's current stream is that
    stream, and the inputs' memory is not reused before it has passed this call."""
    device = tensors[0].device
    if any(t.device.type != "cuda" for t in tensors):
        raise ValueError(f"a stream needs tensors on the same GPU, got {[str(t.device) for t in tensors]}")
    s = torch.cuda.ExternalStream(stream, device=device) if stream else torch.cuda.default_stream(device)
    for t in tensors:
        t.record_stream(s)
    return torch.cuda.stream(s)


def quantize_fp8(x, dtype=torch.float8_e4m3fn, block_rows: int = 1, stream=None):
    """x [rows, cols] (bf16, f16 or f32, columns next to each other, any row stride) in 8 bits:
    (q, scale).  block_rows 1: a scale for each 128 values of a row (activations, gradients);
    128: for each 128 x 128 block (weights).  Infinities and NaN do not count for a scale; they
    become the type's NaN (e4m3) or stay as they are (e5m2).  A value within half an 8-bit step of 2^16 (f16:
    from 63488 on in e4m3, 61440 in e5m2) or 2^128 (bf16, f32) is rounded up to that power, which its wide type
    does not hold: dequantize_fp8 into that type gives infinity."""
    if stream is not None:
        with _elsewhere(stream, x):
            return _native.quantize_fp8(x, dtype, block_rows)
    return _native.quantize_fp8(x, dtype, block_rows)


def quantize_fp8_both(x, dtype=torch.float8_e4m3fn, block_rows: int = 1, stream=None):
    """((q, scale), (q_t, scale_t)): quantize_fp8 of x and of its transpose in one pass over x, for a
    tensor that two products read along different axes (the gradient of a layer's result, a weight).
    With block_rows 1 each has its own blocks along its own rows; with 128 they are the same blocks."""
    if stream is not None:
        with _elsewhere(stream, x):
            return _native.quantize_fp8_both(x, dtype, block_rows)
    return _native.quantize_fp8_both(x, dtype, block_rows)


def dequantize_fp8(q, scale, dtype=torch.bfloat16, stream=None):
    """The values that (q, scale) stands for, [rows, cols] contiguous, in bf16, f16 or f32.  Exact
    wherever `dtype` has the exponent's range; a value past its largest number is infinite."""
    if stream is not None:
        with _elsewhere(stream, q, scale):
            return _native.dequantize_fp8(q, scale, dtype)
    return _native.dequantize_fp8(q, scale, dtype)


def align_fp8(q, scale, stream=None):
    """(q, scale) with rows where the functions here want them, for a pair that was cloned, made contiguous, moved
    between devices or loaded from a file (serving weights: once, after loading).  Strides may be any; a tensor that
    fits already is returned itself, not a copy.  On the CPU too."""
    if stream is not None:
        with _elsewhere(stream, q, scale):
            return _native.align_fp8(q, scale)
    return _native.align_fp8(q, scale)


def transpose_fp8(q, scale, stream=None):
    """The transpose [cols, rows] of a tensor in 8 bits, itself in 8 bits: (q_t, scale_t).  Blocks
    of 128 x 128 stay what they are (a single row's are 1 x 128: its scales have the same shape).  Blocks of 1 x 128 become blocks of 1 x 128 along the
    transpose's own rows: the values are quantised anew from what they stand for, which, both
    scales being powers of two, changes only values below the type's normal range in their new
    block (2^-14 of its largest for e4m3, 2^-29 for e5m2, and less)."""
    if stream is not None:
        with _elsewhere(stream, q, scale):
            return _native.transpose_fp8(q, scale)
    return _native.transpose_fp8(q, scale)


def gemm_fp8(a, a_scale, b, b_scale, out=None, out_dtype=torch.bfloat16, stream=None, variant: int = 0,
             parts: int = 0):
    """out[M, N] = a[M, K] @ b[N, K]^T for operands in 8 bits with their block scales; each may be
    e4m3 or e5m2 and have blocks of 1 x 128 or 128 x 128.  Any M, N and K <= 2^22 (K = 0 gives zeros).
    Sums are held in 32 bits and rounded once into bf16 or f16 (`out_dtype`, or `out`'s type; `out`
    needs its columns next to each other, its rows may be further apart; it must not overlap an
    input).  The matrix instruction drops a product 2^-14 and more below the largest of the 32 it
    adds at once.  variant 0 picks the kernel by the sizes; 1 / 2 force the 128x128 / 256x256 tile
    (the latter for K >= 144), 3 / 6 the kernel for few rows (M <= 16) with 16 / 32 rows of b per
    wave, 4 the 64x64 tile, 5 the 128x128 tile with two blocks per CU.  Where tiles are few and K is long, K is
    cut into parts, multiplied by blocks of their own into 32 bits and added in order by a second kernel;
    parts forces their number (variants 1 and 4, at most 16 and at most one for each 512 of K; 1: none)."""
    if stream is not None:
        with _elsewhere(stream, a, a_scale, b, b_scale, *([] if out is None else [out])):
            return _native.gemm_fp8(a, a_scale, b, b_scale, out, out_dtype, variant, parts)
    return _native.gemm_fp8(a, a_scale, b, b_scale, out, out_dtype, variant, parts)


def gemm_fp8_variant(M: int, N: int, K: int, variant: int = 0) -> int:
    """The kernel variant that gemm_fp8 runs for these sizes (0 resolved), -1 if they do not fit it."""
    return _native.gemm_fp8_plan(M, N, K, variant)[0]


def gemm_fp8_parts(M: int, N: int, K: int, variant: int = 0) -> int:
    """The number of parts into which gemm_fp8 cuts K for these sizes."""
    return _native.gemm_fp8_plan(M, N, K, variant)[1]


def linear_fp8(x, weight, weight_scale=None):
    """y[..., N] = x[..., K] @ weight[N, K]^T in 8 bits, in x's type (bf16 or f16).

    Training: `weight` in bf16 or f16.  Both operands are quantised to e4m3 (x in blocks of 1 x 128,
    the weight 128 x 128).  What the backward pass reads is kept in 8 bits: x's checkpoint where the
    weight takes a gradient (half the memory of the activation) and the transposed weight where x takes
    one (in every call: with fewer tokens than outputs the two are more than x in 16 bits);
    dx = Q(dy) W with the kept 8-bit weight, dW = Q(dy^T) x with the checkpoint
    transposed (as transpose_fp8 does).  A backward pass computes the gradients asked for.  A double backward and forward-mode derivatives are refused.  K is at most 2^22, and so is N
    where x takes a gradient and the number of x's rows where the weight takes one; each tensor that is quantised, the
    result's gradient among them, has fewer than 2^28 blocks of 128 along its rows.  Sizes that only the backward pass
    would not take are refused before the forward pass.

    Serving: `weight` in 8 bits with its `weight_scale`, as quantize_fp8(w, block_rows=128) gives
    them; x may take a gradient, the weight takes none (its backward pass transposes the weight each time).

    All three products are gemm_fp8's: sums in 32 bits, the matrix instruction drops products 2^-14 and more below
    the largest of the 32 it adds at once.  Sums may be added in another order than in separate calls."""
    return _native.linear_fp8(x, weight, weight_scale)
