"""The 8-bit operators on an MI355X against 64 bits (tests/fp8_oracle.py).

Tolerances.  Quantising, giving back and transposing are exact: powers of two and one rounding that
the definition fixes.  The product's operands here are small whole numbers times powers of two
(fp8_oracle.pair): every product of a group is a whole multiple of its unit and at most 16 units, far
from the 2^-14 that the matrix instruction cuts off, every sum stays below 2^24 units, so the sum is
exact and the result is the one rounding of the exact value.  On random operands a result may be off by
half a step of its type, eps / 2 relative, and by what the instruction cuts: 32 products at a time, each
by less than 2^-13 of the largest, at most 2^-8 of the sum of magnitudes; over many results these errors
have both signs, in norm they stay under 2^-13 (measured alone: 1.5e-5 < 2^-16)."""
import pytest
import torch
import torch.utils.checkpoint

from kubernetes_gpu_exporter_amd.ops.fp8 import (dequantize_fp8, gemm_fp8, gemm_fp8_parts, gemm_fp8_variant,
                                                 linear_fp8, quantize_fp8, quantize_fp8_both, transpose_fp8)
from tests.fp8_oracle import E4M3, E5M2, E8M0, pair, quantized, small_whole, values

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _gpu(on_gpu):
    pass


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def activations(m, k, g, dtype):
    x = torch.randn(m, k, device="cuda", generator=g) * torch.exp(2 * torch.randn(k, device="cuda", generator=g))
    return x.clamp(-60000, 60000).to(dtype)


def same(got, want):
    """Equal, NaN where NaN, the sign of a zero aside."""
    got, want = got.double(), want.double()
    assert got.shape == want.shape
    assert torch.equal(got.isnan(), want.isnan())
    bad = (got != want) & ~want.isnan()
    assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[:4].tolist(), got[bad][:4].tolist(), want[bad][:4].tolist())


SIZES = [(1, 1), (1, 128), (3, 5), (7, 129), (16, 2048), (130, 127), (128, 128), (257, 1000), (33, 4096), (1000, 8)]


@pytest.mark.parametrize("m,k", SIZES)
@pytest.mark.parametrize("xdtype", [BF16, F16, F32])
@pytest.mark.parametrize("dtype", [E4M3, E5M2])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_is_the_definition(m, k, xdtype, dtype, block_rows):
    x = activations(m, k, gen(m * 7 + k), xdtype)
    q, s = quantize_fp8(x, dtype, block_rows)
    want, e = quantized(x, dtype, block_rows)
    assert q.shape == x.shape and q.dtype == dtype and s.dtype == E8M0
    assert torch.equal(s.view(torch.uint8).int(), (e + 127).int())
    same(values(q, s), want)
    for back in (BF16, F16, F32):
        got = dequantize_fp8(q, s, back)
        assert got.dtype == back and got.is_contiguous()
        same(got, want.float().to(back))


@pytest.mark.parametrize("m,k", SIZES + [(129, 300)])
@pytest.mark.parametrize("dtype", [E4M3, E5M2])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_transpose_requantises_along_the_other_axis(m, k, dtype, block_rows):
    x = activations(m, k, gen(m + k), BF16)
    q, s = quantize_fp8(x, dtype, block_rows)
    qt, st = transpose_fp8(q, s)
    assert tuple(qt.shape) == (k, m) and qt.dtype == dtype
    kept = values(q, s)
    if block_rows == 128 and m > 1:
        same(values(qt, st), kept.T)
        assert torch.equal(st.view(torch.uint8), s.view(torch.uint8).T)
    else:
        want, e = quantized(kept.T.contiguous(), dtype)
        assert torch.equal(st.view(torch.uint8).int(), (e + 127).int())
        same(values(qt, st), want)


@pytest.mark.parametrize("m,k", [(1, 1), (5, 200), (128, 128), (300, 129), (257, 640)])
@pytest.mark.parametrize("xdtype", [BF16, F32])
def test_both_orientations_in_one_pass(m, k, xdtype):
    x = activations(m, k, gen(m * k), xdtype)
    for block_rows in (1, 128):
        (q, s), (qt, st) = quantize_fp8_both(x, E4M3, block_rows)
        want, e = quantized(x, E4M3, block_rows)
        same(values(q, s), want)
        want_t = quantized(x.T.contiguous(), E4M3)[0] if block_rows == 1 else want.T
        same(values(qt, st), want_t)



@pytest.mark.parametrize("dtype,xdtype", [(E4M3, F32), (E5M2, F32), (E4M3, BF16), (E4M3, F16)])
def test_quantize_borders(dtype, xdtype):
    """Values next to a scale's border, ties, the smallest and largest magnitudes, zeros, NaN and infinities."""
    largest = 448.0 if dtype == E4M3 else 57344.0
    g = gen(3)
    x = torch.zeros(40, 256, device="cuda", dtype=torch.float64)
    top = torch.finfo(xdtype).max
    for i in range(16):  # the block's largest just at, below and above largest * 2^n
        x[i] = torch.randn(256, device="cuda", generator=g, dtype=torch.float64)
        x[i, 0] = largest * 2.0 ** (i - 8) * (1 + (i % 3 - 1) * (2.0 ** -7 if xdtype == BF16 else 2.0 ** -10))
    x[16] = torch.linspace(-1, 1, 256, dtype=torch.float64)  # many ties
    x[17] = (torch.arange(256, device="cuda") - 128).double() / 16
    x[18] = 0.0
    x[19] = torch.finfo(xdtype).smallest_normal
    x[20] = torch.finfo(xdtype).smallest_normal * 2.0 ** (-7 if xdtype == BF16 else -9)  # subnormal
    x[21] = top
    x[22, ::3] = top
    x[23, 5] = float("inf")
    x[24, 5] = float("nan")
    x[25] = torch.randn(256, device="cuda", generator=g, dtype=torch.float64)
    x[25, 7], x[25, 8], x[25, 130] = float("inf"), float("-inf"), float("nan")
    x[26] = float("inf")
    x[27] = -0.0
    x[28] = torch.logspace(-30, 4, 256, dtype=torch.float64) if xdtype != F16 else torch.logspace(-7, 4, 256)
    x = x.to(xdtype)
    for block_rows in (1, 128):
        q, s = quantize_fp8(x, dtype, block_rows)
        want, e = quantized(x, dtype, block_rows)
        assert torch.equal(s.view(torch.uint8).int(), (e + 127).int())
        same(values(q, s), want)
    q, s = quantize_fp8(x, dtype)
    finite = x.clone()
    finite[21:23] = 1.0  # (their rounded values reach 2^128: not a 32-bit number)
    q, s = quantize_fp8(finite, dtype)
    qt, st = transpose_fp8(q, s)
    want, e = quantized(values(q, s).T.contiguous(), dtype)
    assert torch.equal(st.view(torch.uint8).int(), (e + 127).int())
    same(values(qt, st), want)


def test_every_value_of_the_types_survives():
    """Each finite code, quantised from its own value next to the type's largest, is itself again."""
    for dtype, largest in ((E4M3, 448.0), (E5M2, 57344.0)):
        codes = torch.arange(256, device="cuda", dtype=torch.int32).to(torch.uint8).view(dtype)
        x = codes.float()
        x = torch.where(x.isfinite(), x, 0.0).reshape(4, 64)
        x = torch.cat([torch.full((4, 1), largest, device="cuda"), x], 1)
        for wide in (F32, BF16, F16):
            q, s = quantize_fp8(x.to(wide), dtype)
            assert torch.equal(q.float(), x)
            assert torch.equal(dequantize_fp8(q, s, wide).float(), x)


@pytest.mark.parametrize("scales", [(0, 254, 255, 127), (0, 254, 100, 127), (0, 10, 40, 64), (190, 254, 200, 210),
                                    (60, 127, 90, 100), (63, 127, 64, 127), (255, 255, 255, 255), (0, 0, 0, 0)])
@pytest.mark.parametrize("dtype", [E4M3, E5M2])
def test_extreme_scales_given_from_outside(scales, dtype):
    """Scales next to 2^-127 and 2^127, NaN, near and far from each other, which quantize_fp8 itself does not make."""
    rows = torch.tensor([[1.0, -0.5, 448.0, 2.0 ** -9, 0.0] * 25, [1.75, 3.0, 1.0, 0.0, 0.0] * 25,
                         [0.0, 0.0, 2.0 ** -9, 0.0, 0.0] * 25, [0.0, 1.0, 0.0, -2.0 ** -9, 0.0] * 25], device="cuda")
    q = torch.zeros(4, 128, device="cuda").to(dtype)
    q[:, :125] = rows.to(dtype)
    s = torch.tensor(scales, dtype=torch.uint8, device="cuda").reshape(4, 1)
    s = torch.nn.functional.pad(s, (0, 3)).view(E8M0)[:, :1]
    same(dequantize_fp8(q, s, F32), values(q, s).float())
    qt, st = transpose_fp8(q, s)
    want, e = quantized(values(q, s).T.contiguous(), dtype)
    assert torch.equal(st.view(torch.uint8).int(), (e + 127).int())
    same(values(qt, st), want)


@pytest.mark.parametrize("offset,ld", [(0, 136), (1, 133), (8, 256), (3, 129)])
@pytest.mark.parametrize("xdtype", [BF16, F32])
def test_quantize_strided_and_unaligned_rows(offset, ld, xdtype):
    base = activations(1, 40 * 256 + 64, gen(ld), xdtype)[0]
    x = base[offset:offset + 40 * ld].view(40, ld)[:, :129]
    want, e = quantized(x, E4M3)
    q, s = quantize_fp8(x)
    same(values(q, s), want)
    want, e = quantized(x, E4M3, 128)
    q, s = quantize_fp8(x, block_rows=128)
    same(values(q, s), want)


@pytest.mark.parametrize("cols,ld", [(1, 16), (16, 16), (100, 112), (120, 128), (128, 128), (900, 912), (1001, 1024),
                                     (1024, 1024), (5000, 5120)])
def test_rows_start_at_lines_where_that_is_cheap(cols, ld):
    x = torch.randn(3, cols, device="cuda")
    for q in (quantize_fp8(x)[0], quantize_fp8(x, block_rows=128)[0], quantize_fp8_both(x)[0][0],
              quantize_fp8_both(x.T.contiguous())[1][0], transpose_fp8(*quantize_fp8(x.T.contiguous()))[0]):
        assert tuple(q.shape) == (3, cols) and q.stride() == (ld, 1)


def exact_product(a, sa, b, sb):
    return values(a, sa) @ values(b, sb).T


GEMMS = [(1, 1, 1), (1, 16, 128), (1, 1000, 640), (2, 129, 127), (5, 64, 16), (16, 256, 512), (17, 33, 300),
         (33, 4096, 1024), (64, 130, 2050), (100, 1, 129), (127, 255, 383), (128, 128, 128), (129, 129, 129),
         (256, 256, 256), (300, 500, 1000), (512, 512, 640), (257, 769, 2048), (1024, 256, 4096), (1000, 1111, 1234),
         (8, 8192, 8192), (1, 4096, 16384), (2048, 2048, 256), (2049, 2047, 129), (1900, 2300, 1010), (4096, 1024, 384),
         (2050, 2048, 2064)]


@pytest.mark.parametrize("m,n,k", GEMMS)
@pytest.mark.parametrize("variant", [0, 1, 2, 3, 4, 5, 6])
def test_gemm_is_exact_on_whole_numbers(m, n, k, variant):
    if gemm_fp8_variant(m, n, k, variant) < 0:
        pytest.skip("the kernel does not take these sizes")
    g = gen(m + n + k)
    for ta, tb, block_a, block_b, out in ((E4M3, E4M3, 1, 128, BF16), (E5M2, E4M3, 1, 1, F16), (E4M3, E5M2, 128, 128, F16),
                                          (E5M2, E5M2, 128, 1, BF16)):
        a, sa = pair(m, k, g, ta, block_a, spread=2, pad=16)
        b, sb = pair(n, k, g, tb, block_b, spread=1)
        got = gemm_fp8(a, sa, b, sb, out_dtype=out, variant=variant)
        want = exact_product(a, sa, b, sb)
        assert float(want.abs().max()) < 2.0 ** 20  # units of 2^-3: exact in 32 bits
        assert got.dtype == out and got.is_contiguous()
        same(got, want.float().to(out))


@pytest.mark.parametrize("m,n,k", [(1, 512, 4096), (48, 512, 4096), (512, 512, 4096), (2048, 1024, 8192)])
@pytest.mark.parametrize("out", [BF16, F16])
def test_gemm_on_random_operands(m, n, k, out):
    g = gen(k)
    a, sa = quantize_fp8(torch.randn(m, k, device="cuda", generator=g))
    b, sb = quantize_fp8(torch.randn(n, k, device="cuda", generator=g) * 0.02, block_rows=128)
    got = gemm_fp8(a, sa, b, sb, out_dtype=out).double()
    x, w = values(a, sa), values(b, sb)
    want, size = x @ w.T, x.abs() @ w.abs().T
    half = torch.finfo(out).eps / 2
    tiny = torch.finfo(out).smallest_normal * half
    assert bool(((got - want).abs() <= half * want.abs() + 2.0 ** -8 * size + tiny).all())
    assert float((got - want).norm()) <= (half + 2.0 ** -13) * float(want.norm())


@pytest.mark.parametrize("m", [1, 16, 40, 200, 700])
@pytest.mark.parametrize("variant", [0, 1, 2, 3, 4, 5, 6])
def test_gemm_repeats_bit_for_bit(m, variant):
    """Sums are joined in a fixed order: the same call gives the same bits (a tile read
    before it landed, or loaded over while read, would show here)."""
    if gemm_fp8_variant(m, 768, 4096, variant) < 0:
        pytest.skip("the kernel does not take these sizes")
    g = gen(m)
    a, sa = quantize_fp8(torch.randn(m, 4096, device="cuda", generator=g))
    b, sb = quantize_fp8(torch.randn(768, 4096, device="cuda", generator=g), block_rows=128)
    first = gemm_fp8(a, sa, b, sb, variant=variant)
    for _ in range(5):
        assert torch.equal(gemm_fp8(a, sa, b, sb, variant=variant), first)


@pytest.mark.parametrize("m,n", [(3, 5), (16, 257), (130, 70), (300, 300), (512, 256)])
@pytest.mark.parametrize("variant", [0, 1, 2, 3, 4, 5, 6])
def test_gemm_into_a_view_leaves_the_rest(m, n, variant):
    if gemm_fp8_variant(m, n, 384, variant) < 0:
        pytest.skip("the kernel does not take these sizes")
    g = gen(n)
    a, sa = pair(m, 384, g, pad=32)
    b, sb = pair(n, 384, g, block_rows=128)
    whole = torch.full((m + 2, n + 7), 77.0, device="cuda", dtype=BF16)
    got = gemm_fp8(a, sa, b, sb, out=whole[1:m + 1, 3:n + 3], variant=variant)
    want = exact_product(a, sa, b, sb).float().to(BF16)
    same(got, want)
    whole[1:m + 1, 3:n + 3] = 77.0
    assert bool((whole == 77.0).all())


@pytest.mark.parametrize("m,n,k", [(1, 1, 513), (17, 33, 1025), (40, 100, 1039), (64, 64, 1536), (65, 129, 4096), (128, 200, 2050),
                                   (100, 1, 5000), (300, 260, 8192), (129, 383, 8200)])
@pytest.mark.parametrize("variant", [1, 4])
@pytest.mark.parametrize("parts", [2, 3, 7, 16])
def test_gemm_with_k_in_parts(m, n, k, variant, parts):
    parts = min(parts, (k + 511) // 512)
    g = gen(m + n + k)
    for ta, tb, block_a, block_b, out in ((E4M3, E4M3, 1, 128, BF16), (E5M2, E5M2, 128, 1, F16)):
        a, sa = pair(m, k, g, ta, block_a, spread=2, pad=16)
        b, sb = pair(n, k, g, tb, block_b, spread=1)
        want = exact_product(a, sa, b, sb)
        assert float(want.abs().max()) < 2.0 ** 20
        whole = torch.full((m + 2, n + 7), 77.0, device="cuda", dtype=out)
        del_me = torch.full((16 * (m + 128) * (n + 128),), float("nan"), device="cuda")  # what the next workspace holds
        del del_me
        same(gemm_fp8(a, sa, b, sb, out=whole[1:m + 1, 3:n + 3], variant=variant, parts=parts), want.float().to(out))
        whole[1:m + 1, 3:n + 3] = 77.0
        assert bool((whole == 77.0).all())
        for _ in range(3):
            same(gemm_fp8(a, sa, b, sb, out_dtype=out, variant=variant, parts=parts), want.float().to(out))


@pytest.mark.parametrize("m,n,k", [(4, 6, 0), (0, 6, 128), (4, 0, 128), (0, 0, 0), (700, 300, 0)])
def test_gemm_of_empty_sizes(m, n, k):
    a, sa = quantize_fp8(torch.zeros(m, k, device="cuda"))
    b, sb = quantize_fp8(torch.zeros(n, k, device="cuda"), block_rows=128)
    got = gemm_fp8(a, sa, b, sb)
    assert tuple(got.shape) == (m, n) and not bool(got.any())
    assert tuple(dequantize_fp8(a, sa).shape) == (m, k) and tuple(transpose_fp8(a, sa)[0].shape) == (k, m)


@pytest.mark.parametrize("m,n,k", [(1, 40, 300), (20, 40, 300), (200, 300, 300), (512, 512, 500)])
@pytest.mark.parametrize("variant", [0, 1, 2, 3, 4, 5, 6])
def test_gemm_nan_and_inf_stay_in_their_row(m, n, k, variant):
    if gemm_fp8_variant(m, n, k, variant) < 0:
        pytest.skip("the kernel does not take these sizes")
    g = gen(9)
    a, sa = pair(m, k, g, E5M2)
    b, sb = pair(n, k, g, E4M3, 1)
    want = exact_product(a, sa, b, sb).float().to(BF16)
    a[m // 2, k - 1], b[n // 2, 7] = float("inf"), float("nan")
    b[:, k - 1] = torch.where(b[:, k - 1].float() == 0, torch.ones(n, device="cuda").to(E4M3).float(), b[:, k - 1].float()).to(E4M3)
    want = exact_product(a, sa, b, sb).float().to(BF16)
    got = gemm_fp8(a, sa, b, sb, variant=variant)
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
    ok = want.isfinite()
    assert torch.equal(got[ok], want[ok])


def test_offsets_past_32_bits():
    """An operand, its scales' rows and a result beyond 2^32 bytes: the last rows are right."""
    g = gen(4)
    m, k = (1 << 20) + 700, 4224
    x = torch.zeros(m, k, device="cuda", dtype=BF16)  # 8.9 GB
    tail = small_whole(300, k, g).to(BF16)
    x[-300:] = tail
    q, s = quantize_fp8(x)
    assert q.numel() > 1 << 32
    del x
    want, _ = quantized(tail, E4M3)
    same(values(q[-300:], s[-300:]), want)
    b, sb = pair(2050, k, g, block_rows=128, spread=1)
    got = gemm_fp8(q, s, b[:32], sb[:1])
    same(got[-300:], (want @ values(b[:32], sb[:1]).T).float().to(BF16))
    back = dequantize_fp8(q, s)
    assert torch.equal(back[-300:], tail)
    del back
    qt, st = transpose_fp8(q, s)
    same(values(qt[:, -188:], st[:, -2:])[:, -188:], want.T[:, -188:])
    del qt, st
    wide = gemm_fp8(q, s, b, sb)  # 4.3 GB of results
    same(wide[-300:], (want @ values(b, sb).T).float().to(BF16))


def reference_linear(x, w, grad, frozen=None):
    """(y, dx, dw) in 64 bits, from the definition."""
    xq, gq = quantized(x)[0], quantized(grad)[0]
    wq = quantized(w, block_rows=128)[0] if frozen is None else frozen
    gt, xt = quantized(grad.T.contiguous())[0], quantized(xq.T.contiguous())[0]
    return xq @ wq.T, gq @ wq, gt @ xt.T, (xq.abs() @ wq.abs().T, gq.abs() @ wq.abs(), gt.abs() @ xt.abs().T)


LINEARS = [(1, 64, 64), (3, 130, 70), (50, 1, 200), (128, 256, 512), (129, 200, 1000), (513, 384, 256), (17, 1000, 2048)]


@pytest.mark.parametrize("m,n,k", LINEARS)
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_linear_and_its_gradients(m, n, k, dtype):
    g = gen(m + n)
    x = torch.randn(m, k, device="cuda", generator=g).to(dtype)
    if m > 2:
        x[m // 2] = 0  # a padded token
    w = (torch.randn(n, k, device="cuda", generator=g) * 0.05).to(dtype)
    grad = (torch.randn(m, n, device="cuda", generator=g) * 0.1).to(dtype)
    x.requires_grad_()
    w.requires_grad_()
    y = linear_fp8(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), grad)
    *want, sizes = reference_linear(x.detach(), w.detach(), grad)
    half, tiny = torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    for got, ref, size in zip((y, dx, dw), want, sizes):
        assert got.dtype == dtype
        err = (got.detach().double() - ref).abs()
        assert bool((err <= half * ref.abs() + 2.0 ** -8 * size + tiny).all())
        assert float(err.norm()) <= (half + 2.0 ** -13) * float(ref.norm()) + tiny * ref.numel() ** 0.5


@pytest.mark.parametrize("m,n,k", [(1, 64, 96), (130, 70, 300), (260, 256, 384)])
def test_linear_gradients_against_differences(m, n, k):
    """On values that 8 bits hold exactly (each block's largest is 4, so 1/8 is a step), y is linear in x and in the
    weight to the last bit: differences are the gradients, exactly, as long as every sum is a 16-bit number."""
    g = gen(5)

    def whole(r, c):
        t = torch.randint(-1, 2, (r, c), device="cuda", generator=g).float()
        t[:, ::128] = 4.0
        return t
    x, w, grad = whole(m, k), whole(n, k), torch.zeros(m, n, device="cuda")
    grad[m // 2, n // 3] = 1.0
    grad[0, n - 1] = 2.0
    dx_dir, dw_dir = torch.zeros(m, k, device="cuda"), torch.zeros(n, k, device="cuda")
    dx_dir[m // 2, 1:100:7] = 1.0
    dx_dir[0, 5] = -1.0
    dw_dir[n // 3, 2:90:5] = 1.0
    dw_dir[n - 1, 11] = -1.0

    def loss(xx, ww):
        return float((linear_fp8(xx.to(F16), ww.to(F16)).double() * grad.double()).sum())
    xl, wl = x.to(F16).requires_grad_(), w.to(F16).requires_grad_()
    gx, gw = torch.autograd.grad(linear_fp8(xl, wl), (xl, wl), grad.to(F16))
    assert (loss(x + dx_dir, w) - loss(x - dx_dir, w)) / 2 == float((gx.double() * dx_dir.double()).sum())
    assert (loss(x, w + dw_dir) - loss(x, w - dw_dir)) / 2 == float((gw.double() * dw_dir.double()).sum())


def test_linear_of_one_gradient_only_and_broadcast_gradients():
    g = gen(6)
    x = torch.randn(2, 70, 256, device="cuda", generator=g).to(BF16)
    w = torch.randn(128, 256, device="cuda", generator=g).to(BF16)
    grad = torch.ones(1, 1, 1, device="cuda", dtype=BF16).expand(2, 70, 128)  # as sum().backward() hands it down
    want = reference_linear(x.reshape(140, 256), w, grad.reshape(140, 128))
    xl = x.clone().requires_grad_()
    y = linear_fp8(xl, w)
    assert tuple(y.shape) == (2, 70, 128)
    y.sum().backward()
    assert float((xl.grad.reshape(140, 256).double() - want[1]).norm()) <= 2.0 ** -7 * float(want[1].norm())
    wl = w.clone().requires_grad_()
    linear_fp8(x, wl).sum().backward()
    assert float((wl.grad.double() - want[2]).norm()) <= 2.0 ** -7 * float(want[2].norm())
    with torch.no_grad():
        assert not linear_fp8(x, wl).requires_grad
    strided = torch.randn(256, 90, device="cuda", generator=g).to(BF16).T  # columns not next to each other
    assert torch.equal(linear_fp8(strided, w), linear_fp8(strided.contiguous(), w))
    assert torch.equal(linear_fp8(x[0, 0], w), linear_fp8(x[0, :1], w)[0])
    for shape in ((0, 256), (2, 0, 256)):
        xe = torch.zeros(shape, device="cuda", dtype=BF16, requires_grad=True)
        ye = linear_fp8(xe, wl)
        ge, gw = torch.autograd.grad(ye.sum(), (xe, wl))
        assert tuple(ye.shape) == (*shape[:-1], 128) and ge.shape == xe.shape and not bool(gw.any())


@pytest.mark.parametrize("m,n,k", [(1, 64, 64), (17, 300, 130), (257, 384, 1000), (1030, 640, 512), (33, 520, 8200),
                                   (8200, 260, 500), (40, 8192, 300)])  # the last: K in parts for y, dw, dx
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_linear_is_the_operators_in_turn(m, n, k, dtype):
    """A layer's passes, the operators one after the other as a program would call them, and the two orientations in
    one pass: the same bits."""
    g = gen(m + k)
    x = torch.randn(m, k, device="cuda", generator=g).to(dtype).requires_grad_()
    w = (torch.randn(n, k, device="cuda", generator=g) * 0.05).to(dtype).requires_grad_()
    grad = torch.randn(m, n, device="cuda", generator=g).to(dtype)
    y = linear_fp8(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), grad)
    kept, weight, dy, dy_t = (quantize_fp8(x.detach()), quantize_fp8(w.detach(), block_rows=128), quantize_fp8(grad),
                              quantize_fp8(grad.T.contiguous()))
    assert torch.equal(y, gemm_fp8(*kept, *weight, out_dtype=dtype))
    assert torch.equal(dx, gemm_fp8(*dy, *transpose_fp8(*weight), out_dtype=dtype))
    assert torch.equal(dw, gemm_fp8(*dy_t, *transpose_fp8(*kept), out_dtype=dtype))
    both, both_w = quantize_fp8_both(grad), quantize_fp8_both(w.detach(), block_rows=128)
    assert torch.equal(dx, gemm_fp8(*both[0], *both_w[1], out_dtype=dtype))
    assert torch.equal(dw, gemm_fp8(*both[1], *transpose_fp8(*kept), out_dtype=dtype))


def test_activations_kept_in_8_bits_between_the_passes():
    """quantize_fp8 / dequantize_fp8 as torch's hooks on saved tensors: what an activation function keeps goes to 8
    bits, its gradient is taken where the checkpoint says the input was; around layers in 8 bits."""
    g = gen(21)
    x = torch.randn(200, 384, device="cuda", generator=g).to(BF16).requires_grad_()
    w1, w2 = ((torch.randn(r, c, device="cuda", generator=g) * 0.05).to(BF16).requires_grad_() for r, c in ((512, 384), (256, 512)))
    grad = torch.randn(200, 256, device="cuda", generator=g).to(BF16)
    h = linear_fp8(x, w1)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: quantize_fp8(t.detach()), lambda p: dequantize_fp8(*p)):
        act = torch.nn.functional.silu(h)
    y = linear_fp8(act, w2)
    got = torch.autograd.grad(y, (x, w1, w2), grad)
    # the same by hand
    ha = h.detach()
    a = torch.nn.functional.silu(ha).requires_grad_()
    da, dw2 = torch.autograd.grad(linear_fp8(a, w2), (a, w2), grad)
    back = dequantize_fp8(*quantize_fp8(ha)).requires_grad_()
    (dh,) = torch.autograd.grad(torch.nn.functional.silu(back), back, da)
    dx, dw1 = torch.autograd.grad(linear_fp8(x, w1), (x, w1), dh)
    for a_, b_ in zip(got, (dx, dw1, dw2)):
        assert torch.equal(a_, b_)


def test_out_counts_as_changed():
    """A tensor that autograd saved and gemm_fp8 then wrote into is reported, as after any in-place change."""
    a, sa = quantize_fp8(torch.randn(8, 128, device="cuda"))
    out = torch.ones(8, 8, device="cuda", dtype=BF16)
    p = torch.ones(8, 8, device="cuda", dtype=BF16, requires_grad=True)
    z = (p * out).sum()
    gemm_fp8(a, sa, a, sa, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()


def test_in_inference_mode_and_recomputed():
    """Without autograd's records, and with a layer's forward pass run again for its backward pass."""
    g = gen(5)
    x, w = (torch.randn(s, device="cuda", generator=g).to(BF16).requires_grad_() for s in ((3, 40, 384), (200, 384)))
    grad = torch.randn(3, 40, 200, device="cuda", generator=g).to(BF16)
    y = linear_fp8(x, w)
    want = torch.autograd.grad(y, (x, w), grad)
    again = torch.utils.checkpoint.checkpoint(lambda a: torch.sin(linear_fp8(a, w)), x, use_reentrant=False)
    got = torch.autograd.grad(again, (x, w), grad)
    plain = torch.autograd.grad(torch.sin(linear_fp8(x, w)), (x, w), grad)
    assert torch.equal(again, torch.sin(y)) and all(torch.equal(a, b) for a, b in zip(got, plain))
    with torch.inference_mode():
        pair_ = quantize_fp8(w, block_rows=128)
        kept = quantize_fp8(x.reshape(120, 384))
        out = torch.empty(120, 200, device="cuda", dtype=BF16)
        assert gemm_fp8(*kept, *pair_, out=out) is not None and torch.equal(out.view(3, 40, 200), y)
        assert torch.equal(linear_fp8(x, w), y) and torch.equal(linear_fp8(x, *pair_), y)
    assert want[0].shape == x.shape and all(bool(t.isfinite().all()) for t in want)
    with torch.enable_grad(), torch.autocast("cuda", dtype=BF16):
        assert torch.equal(linear_fp8(x, w), y)


def test_out_is_refused_where_it_cannot_be_written():
    a, sa = quantize_fp8(torch.randn(8, 128, device="cuda"))
    with pytest.raises(ValueError, match="gradient"):
        gemm_fp8(a, sa, a, sa, out=torch.ones(8, 8, device="cuda", dtype=BF16, requires_grad=True))
    store = torch.zeros(4096, device="cuda", dtype=torch.uint8)
    q = store[:1024].view(8, 128).view(E4M3)
    for first in (0, 896, 1008):
        with pytest.raises(ValueError, match="overlap"):
            gemm_fp8(q, sa, a, sa, out=store[first:first + 128].view(BF16).view(8, 8))
    gemm_fp8(q, sa, a, sa, out=store[1024:1152].view(BF16).view(8, 8))
    assert not bool(store.any())


def test_rows_longer_than_a_buffer_are_refused():
    k = 2**22
    x = torch.zeros(2, k + 1, device="cuda", dtype=BF16)
    q, s = quantize_fp8(x)  # (a checkpoint may be as long as memory is)
    assert torch.equal(dequantize_fp8(q, s), x)
    with pytest.raises(ValueError, match="4194304"):
        gemm_fp8(q, s, q, s)
    with pytest.raises(ValueError, match="4194304"):
        linear_fp8(x, x)
    long = torch.zeros(k + 1, 8, device="cuda", dtype=BF16, requires_grad=True)
    short = torch.zeros(4, 8, device="cuda", dtype=BF16, requires_grad=True)
    assert linear_fp8(long, short.detach()).shape == (k + 1, 4) and linear_fp8(short.detach(), long).shape == (4, k + 1)
    with pytest.raises(ValueError, match="4194304"):
        linear_fp8(long, short)
    with pytest.raises(ValueError, match="4194304"):
        linear_fp8(short, long)


def test_linear_keeps_8_bits_for_the_backward_pass():
    """Between the passes the layer holds its input in 8 bits (and the 8-bit weight), no 16-bit copy."""
    x = torch.randn(4096, 2048, device="cuda", dtype=BF16).requires_grad_()
    w = torch.randn(1024, 2048, device="cuda", dtype=BF16).requires_grad_()
    held = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: held.append(t) or t, lambda t: t):
        y = linear_fp8(x, w)
    assert sum(t.numel() * t.element_size() for t in held) <= (x.numel() + w.numel()) * 1.01
    with torch.no_grad():  # changes to the leaves between the passes do not reach what was kept
        gx, gw = torch.autograd.grad(y, (x, w), torch.ones_like(y), retain_graph=True)
        x.zero_()
        w.zero_()
    gx2, gw2 = torch.autograd.grad(y, (x, w), torch.ones_like(y))
    assert torch.equal(gx, gx2) and torch.equal(gw, gw2)


def test_linear_double_backward_is_refused():
    x = torch.randn(8, 64, device="cuda", dtype=BF16).requires_grad_()
    w = torch.randn(8, 64, device="cuda", dtype=BF16).requires_grad_()
    (gx,) = torch.autograd.grad(linear_fp8(x, w).sum(), x, create_graph=True)  # a constant dy: dx depends on w alone
    with pytest.raises(RuntimeError, match="differentiated twice"):
        gx.sum().backward()
    s = torch.ones((), device="cuda", dtype=BF16, requires_grad=True)
    for leaves in ((x, w), (x,), (w,)):
        y = linear_fp8(*(t if any(t is u for u in leaves) else t.detach() for t in (x, w)))
        grads = torch.autograd.grad((y * s).sum(), leaves, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiated twice"):
            sum(t.sum() for t in grads).backward()
    wq, ws = quantize_fp8(w.detach(), block_rows=128)
    (gx,) = torch.autograd.grad((linear_fp8(x, wq, ws) * s).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated twice"):
        gx.sum().backward()


@pytest.mark.parametrize("m,n,k", [(1, 4096, 2048), (16, 300, 1000), (5, 64, 64), (40, 512, 4096), (300, 512, 640)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_linear_with_weights_in_8_bits(m, n, k, dtype):
    g = gen(m)
    x = torch.randn(m, k, device="cuda", generator=g).to(dtype)
    wq, ws = quantize_fp8(torch.randn(n, k, device="cuda", generator=g) * 0.1, block_rows=128)
    y = linear_fp8(x, wq, ws)
    xq, xs = quantize_fp8(x)
    ref = quantized(x)[0] @ values(wq, ws).T
    half, tiny = torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    size = quantized(x)[0].abs() @ values(wq, ws).abs().T
    err = (y.double() - ref).abs()
    assert bool((err <= half * ref.abs() + 2.0 ** -8 * size + tiny).all())
    assert float(err.norm()) <= (half + 2.0 ** -13) * float(ref.norm()) + tiny * ref.numel() ** 0.5
    xl = x.clone().requires_grad_()
    grad = torch.randn(m, n, device="cuda", generator=g).to(dtype)
    (gx,) = torch.autograd.grad(linear_fp8(xl, wq, ws), xl, grad)
    want = quantized(grad)[0] @ values(wq, ws)
    assert float((gx.double() - want).norm()) <= (half + 2.0 ** -13) * float(want.norm()) + tiny * want.numel() ** 0.5


@pytest.mark.parametrize("m", [1, 2, 7, 16, 17])
@pytest.mark.parametrize("n,k", [(64, 64), (300, 1024), (1000, 4096), (33, 8192), (5000, 48), (256, 1000), (4096, 4608)])
def test_serving_quantises_as_quantize_fp8_does(m, n, k):
    """A few tokens' activations may be quantised inside the product: the same bits as in two calls, for rows at any
    address and distance."""
    g = gen(m * n)
    wq, ws = quantize_fp8(torch.randn(n, k, device="cuda", generator=g) * 0.1, block_rows=128)
    base = torch.randn(m * (k + 24) + 8, device="cuda", generator=g)
    base = base * torch.exp(3 * torch.randn(base.shape, device="cuda", generator=g))
    for dtype in (BF16, F16):
        for offset, ld in ((0, k), (8, k + 8), (0, k + 24), (1, k), (0, k + 3)):
            x = base.clamp(-60000, 60000).to(dtype)[offset:offset + m * ld].view(m, ld)[:, :k]
            got = linear_fp8(x, wq, ws)
            assert torch.equal(got, gemm_fp8(*quantize_fp8(x), wq, ws, out_dtype=dtype)), (dtype, offset, ld)


def test_linear_nan_tokens_stay_in_their_rows():
    g = gen(8)
    for m in (3, 40, 300):
        x = torch.randn(m, 512, device="cuda", generator=g).to(BF16)
        wq, ws = quantize_fp8(torch.randn(256, 512, device="cuda", generator=g), block_rows=128)
        clean = linear_fp8(x, wq, ws)
        x[1, 100], x[2, 5] = float("nan"), float("inf")
        y = linear_fp8(x, wq, ws)
        assert bool(y[1].isnan().all()) and bool(y[2].isnan().all())
        keep = [i for i in range(m) if i not in (1, 2)]
        assert torch.equal(y[keep], clean[keep])


def step(x, w, grad):
    y = linear_fp8(x, w)
    return (y.detach(), *torch.autograd.grad(y, (x, w), grad))


def test_captured_and_replayed():
    """A training step and a serving step in one graph, replayed with new inputs between eager work."""
    g = gen(11)
    x, w = (torch.randn(300, 640, device="cuda", generator=g).to(BF16).requires_grad_(),
            torch.randn(256, 640, device="cuda", generator=g).to(BF16).requires_grad_())
    grad = torch.randn(300, 256, device="cuda", generator=g).to(BF16)
    wq, ws = quantize_fp8(w.detach(), block_rows=128)
    token = torch.randn(2, 640, device="cuda", generator=g).to(BF16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, w, grad)
        linear_fp8(token, wq, ws)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = (*step(x, w, grad), linear_fp8(token, wq, ws))
    for seed in range(4):
        g2 = gen(100 + seed)
        with torch.no_grad():
            x.copy_(torch.randn(300, 640, device="cuda", generator=g2))
            token.copy_(torch.randn(2, 640, device="cuda", generator=g2))
            grad.copy_(torch.randn(300, 256, device="cuda", generator=g2))
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        want = (*step(x.detach().requires_grad_(), w.detach().requires_grad_(), grad), linear_fp8(token, wq, ws))
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_products_in_parts_captured_and_replayed():
    """All three products of a step with K in parts, and a serving step's, each with a workspace of its own."""
    g = gen(13)
    big = [torch.randn(s, device="cuda", generator=g).to(BF16) for s in ((40, 8192), (256, 8192), (4096, 200), (300, 200))]
    x, w, x2, w2 = (t.requires_grad_() for t in big)
    wq, ws = quantize_fp8(w.detach(), block_rows=128)
    assert gemm_fp8_parts(40, 256, 8192) > 1 and gemm_fp8_parts(300, 200, 4096) > 1
    grad, grad2 = (torch.randn(s, device="cuda", generator=g).to(BF16) for s in ((40, 256), (4096, 300)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, w, grad), step(x2, w2, grad2), linear_fp8(x.detach(), wq, ws)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = (*step(x, w, grad), *step(x2, w2, grad2), linear_fp8(x.detach(), wq, ws))
    for seed in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(x.shape, device="cuda", generator=gen(seed)))
            x2.copy_(torch.randn(x2.shape, device="cuda", generator=gen(seed)))
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        one, two = ([t.detach().requires_grad_() for t in pair_] for pair_ in ((x, w), (x2, w2)))
        want = (*step(*one, grad), *step(*two, grad2), linear_fp8(x.detach(), wq, ws))
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_two_graphs_and_streams_at_once():
    """Calls on two streams, and two captured graphs replayed at the same time, do not share anything."""
    g = gen(12)
    sets = []
    for i in range(2):
        a, sa = quantize_fp8(torch.randn(3 + 13 * i, 8192, device="cuda", generator=g))
        b, sb = quantize_fp8(torch.randn(512, 8192, device="cuda", generator=g), block_rows=128)
        sets.append((a, sa, b, sb))
    want = [gemm_fp8(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(gemm_fp8(*sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])
    graphs, outs = [], []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(gemm_fp8(*sets[i]))
        graphs.append(graph)
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                graphs[i].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


def test_on_a_raw_stream():
    g = gen(13)
    x = torch.randn(64, 1024, device="cuda", generator=g).to(BF16)
    q, s = quantize_fp8(x)
    want = gemm_fp8(q, s, q, s), dequantize_fp8(q, s), transpose_fp8(q, s)[0].float()
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    raw = st.cuda_stream
    q2, s2 = quantize_fp8(x, stream=raw)
    got = (gemm_fp8(q2, s2, q2, s2, stream=raw), dequantize_fp8(q2, s2, stream=raw), transpose_fp8(q2, s2, stream=raw)[0])
    st.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(got[2].float(), want[2])
    q3, _ = quantize_fp8(x, stream=0)
    torch.cuda.synchronize()
    assert torch.equal(q3.float(), q.float())


def test_fp8_gemm_pod_on_gpu():
    """models.GemmPod in fp8 runs the block-scaled kernel, faster than bf16 can go, and gives its product."""
    from kubernetes_gpu_exporter_amd.models import GemmPod, run
    p = GemmPod(size=512, iters=1, dtype="fp8")
    p.step()
    want = quantized(p.a)[0] @ quantized(p.b, block_rows=128)[0].T
    half = torch.finfo(BF16).eps / 2
    assert float((p.c.double() - want).norm()) <= (half + 2.0 ** -13) * float(want.norm())
    fast, slow = (run(GemmPod(size=4096, iters=8, dtype=d), steps=3, warmup=1) for d in ("fp8", "bf16"))
    assert fast["dtype"] == "fp8" and fast["tflops"] > slow["tflops"], (fast, slow)


def test_fp8_trainer_pod_on_gpu(tmp_path):
    """models.TrainerPod in fp8: a layer's forward and backward pass, then the strategy's collective (one rank)."""
    import torch.distributed as dist
    from kubernetes_gpu_exporter_amd.models import TrainerPod, run
    dist.init_process_group("nccl", init_method=f"file://{tmp_path}/rendezvous", rank=0, world_size=1)
    try:
        p = TrainerPod("dp", size=640, iters=2, comm_bytes=1 << 16, dtype="fp8")
        res = run(p, steps=2, warmup=1)
    finally:
        dist.destroy_process_group()
    assert res["comm_calls"] == {"allreduce": 2} and res["tflops"] > 0
    _, dx, dw, _ = reference_linear(p.a.detach(), p.b.detach(), p.grad)
    half = torch.finfo(BF16).eps / 2
    for got, want in zip(p.grads, (dx, dw)):
        assert float((got.double() - want).norm()) <= (half + 2.0 ** -13) * float(want.norm())


PROGRAMS = {
    "checkpoint": lambda x, w, wq, ws: dequantize_fp8(*transpose_fp8(*quantize_fp8(x))),
    "both": lambda x, w, wq, ws: dequantize_fp8(*quantize_fp8_both(x)[1]),
    "gemm": lambda x, w, wq, ws: gemm_fp8(*quantize_fp8(x), wq, ws),
    "gemm_out": lambda x, w, wq, ws: gemm_fp8(*quantize_fp8(x), wq, ws, out=torch.empty(x.shape[0], wq.shape[0], dtype=BF16,
                                                                                        device=x.device)),
    "serve": lambda x, w, wq, ws: linear_fp8(x, wq, ws),
    "layer": lambda x, w, wq, ws: linear_fp8(x, w),
}


@pytest.mark.parametrize("name", PROGRAMS)
@pytest.mark.parametrize("tracer", ["jit", "fx"])
def test_traced_programs_compute(name, tracer):
    """A recorded program holds the operators themselves, not the memory that one recorded call wrote."""
    from torch.fx.experimental.proxy_tensor import make_fx
    g = gen(31)
    w = torch.randn(96, 320, device="cuda", generator=g).to(BF16)
    x, other = (torch.randn(40, 320, device="cuda", generator=g).to(BF16) for _ in range(2))
    held = (w, *quantize_fp8(w, block_rows=128))
    want = [PROGRAMS[name](t, *held) for t in (x, other)]
    program = lambda t: PROGRAMS[name](t, *held)  # noqa: E731
    traced = torch.jit.trace(program, (x,), check_trace=False) if tracer == "jit" else make_fx(program)(x)
    for t, ref in ((x, want[0]), (other, want[1]), (x, want[0])):
        assert torch.equal(traced(t), ref)


def test_traced_training_steps_compute():
    """The gradients of a traced layer, and a traced step with its backward pass."""
    from torch.fx.experimental.proxy_tensor import make_fx
    g = gen(32)
    w = torch.randn(96, 320, device="cuda", generator=g).to(BF16)
    x, other = (torch.randn(40, 320, device="cuda", generator=g).to(BF16) for _ in range(2))
    grad = torch.randn(40, 96, device="cuda", generator=g).to(BF16)
    wq, ws = quantize_fp8(w, block_rows=128)

    def train(a, b, c):
        return step(a.detach().requires_grad_(), b.detach().requires_grad_(), c)

    def serve(a, c):
        a = a.detach().requires_grad_()
        y = linear_fp8(a, wq, ws)
        return y.detach(), torch.autograd.grad(y, a, c)[0]
    layer = torch.jit.trace(lambda a, b: linear_fp8(a, b), (x, w), check_trace=False)
    train_fx, serve_fx = make_fx(train)(x, w, grad), make_fx(serve)(x, grad)
    for t in (x, other):
        want = train(t, w, grad)
        a, b = t.detach().requires_grad_(), w.detach().requires_grad_()
        y = layer(a, b)
        for got in ((y.detach(), *torch.autograd.grad(y, (a, b), grad)), train_fx(t, w, grad)):
            assert all(torch.equal(p, r) for p, r in zip(got, want))
        assert all(torch.equal(p, r) for p, r in zip(serve_fx(t, grad), serve(t, grad)))


def test_forward_mode_is_refused_on_gpu():
    import torch.autograd.forward_ad as forward_ad
    x, w = (torch.randn(8, 128, device="cuda").to(BF16) for _ in range(2))
    wq, ws = quantize_fp8(w, block_rows=128)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: linear_fp8(dual, w), lambda: linear_fp8(dual, wq, ws), lambda: linear_fp8(x, forward_ad.make_dual(w, x))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        assert torch.equal(linear_fp8(x, w), linear_fp8(x, w.clone()))


def test_copies_laid_out_again():
    """A checkpoint and serving weights that went to the host, into a file's state or through clone(): align_fp8 lays them
    out as the operators want them, and results are those of the originals."""
    from kubernetes_gpu_exporter_amd.ops.fp8 import align_fp8
    g = gen(33)
    x = torch.randn(30, 1101, device="cuda", generator=g).to(BF16)
    w = torch.randn(200, 1101, device="cuda", generator=g).to(BF16)
    kept, weight = quantize_fp8(x), quantize_fp8(w, block_rows=128)
    module = torch.nn.Module()
    module.register_buffer("q", torch.empty(200, 1101, device="cuda", dtype=E4M3))
    module.register_buffer("scale", torch.empty(2, 9, device="cuda", dtype=E8M0))
    module.load_state_dict({"q": weight[0], "scale": weight[1]})
    assert torch.equal(dequantize_fp8(*align_fp8(kept[0].cpu().cuda(), kept[1].cpu().cuda())), dequantize_fp8(*kept))
    for copy in ((module.q, module.scale), tuple(t.contiguous() for t in weight), tuple(t.clone() for t in weight),
                 (weight[0].T.contiguous().T, weight[1].cpu().cuda())):
        again = align_fp8(*copy)
        assert torch.equal(linear_fp8(x, *again), linear_fp8(x, *weight))
        assert torch.equal(gemm_fp8(*kept, *again), gemm_fp8(*kept, *weight))
        assert torch.equal(transpose_fp8(*again)[0].float(), transpose_fp8(*weight)[0].float())


@pytest.mark.parametrize("m,n,k", [(40, 520, 4096), (300, 256, 640), (8200, 260, 500)])
def test_only_the_gradient_asked_for_is_computed(m, n, k):
    g = gen(34)
    x = torch.randn(m, k, device="cuda", generator=g).to(BF16).requires_grad_()
    w = torch.randn(n, k, device="cuda", generator=g).to(BF16).requires_grad_()
    grad = torch.randn(m, n, device="cuda", generator=g).to(BF16)
    y = linear_fp8(x, w)

    def asked(*leaves):
        before = torch.cuda.memory_stats()["requested_bytes.all.allocated"]
        got = torch.autograd.grad(y, leaves, grad, retain_graph=True)
        return got, torch.cuda.memory_stats()["requested_bytes.all.allocated"] - before
    (dx, dw), both = asked(x, w)
    (only_x,), of_x = asked(x)
    (only_w,), of_w = asked(w)
    assert torch.equal(only_x, dx) and torch.equal(only_w, dw)
    assert of_x <= both - 2 * dw.numel() and of_w <= both - 2 * dx.numel()
    y.backward(grad, inputs=[w])
    assert x.grad is None and torch.equal(w.grad, dw)


def test_traced_step_of_one_gradient_computes():
    from torch.fx.experimental.proxy_tensor import make_fx
    g = gen(36)
    w = torch.randn(96, 320, device="cuda", generator=g).to(BF16)
    x, other = (torch.randn(40, 320, device="cuda", generator=g).to(BF16) for _ in range(2))

    def of_weight(a, b):
        b = b.detach().requires_grad_()
        return torch.autograd.grad(linear_fp8(a.detach().requires_grad_(), b).float().square().sum(), b)[0]
    traced = make_fx(of_weight)(x, w)
    for t in (x, other):
        assert torch.equal(traced(t, w), of_weight(t, w))


def test_many_outputs_for_few_rows():
    """2^26 columns of C: more blocks of 1024 threads than a launch takes, fewer of those that this K needs."""
    n = 1 << 26
    b = torch.zeros(n, 16, device="cuda", dtype=E4M3)
    digits = torch.arange(n, device="cuda", dtype=torch.int32).remainder_(9).sub_(4).to(BF16)
    b[:, 0] = digits.to(E4M3)
    sb = torch.full((n // 128, 4), 127, device="cuda", dtype=torch.uint8).view(E8M0)[:, :1]
    a, sa = quantize_fp8(torch.full((1, 16), 2.0, device="cuda"))
    for variant in (0, 3, 4, 6):
        assert torch.equal(gemm_fp8(a, sa, b, sb, variant=variant)[0], 2 * digits)
    assert torch.equal(linear_fp8(torch.full((1, 16), 2.0, device="cuda", dtype=BF16), b, sb)[0], 2 * digits)


@pytest.mark.parametrize("dtype,xdtype,far", [(E4M3, F16, 63488.0), (E5M2, F16, 61440.0), (E4M3, BF16, 1.9375 * 2.0 ** 127),
                                              (E4M3, F32, 1.9375 * 2.0 ** 127), (E5M2, F32, 1.875 * 2.0 ** 127)])
def test_values_next_to_the_types_largest_come_back_infinite(dtype, xdtype, far):
    """From `far` on, the middle between the largest 8-bit number below 2^16 (f16) or 2^128 and that power itself, a value
    is rounded up to the power, which the wide type does not hold; below `far` it comes back finite."""
    top = torch.finfo(xdtype).max
    x = torch.zeros(3, 128, device="cuda", dtype=xdtype)
    x[0, 0], x[1, 0], x[2, 0] = top, -top, far * (1 - 2.0 ** -7)
    q, s = quantize_fp8(x, dtype)
    back = dequantize_fp8(q, s, xdtype)
    assert back[:2, 0].tolist() == [float("inf"), float("-inf")]
    assert torch.isfinite(back[2, 0]) and not bool(back[:, 1:].any())
    same(back, quantized(x, dtype)[0].float().to(xdtype))


@pytest.mark.parametrize("variant", [0, 1, 2, 3, 4, 5, 6])
def test_gemm_with_extreme_scales(variant):
    """Products of scales next to 2^-127 and 2^127: what leaves bf16's range is infinite or zero, a NaN scale gives NaN."""
    g = gen(35)
    m = 16 if variant in (3, 6) else 40
    a, sa = pair(m, 256, g, block_rows=1)
    b, sb = pair(48, 256, g, block_rows=1)
    ta = torch.tensor([0, 254, 255, 127, 100, 7, 200, 64], dtype=torch.uint8, device="cuda").repeat(5)[:m]
    tb = torch.tensor([254, 0, 127, 255, 150, 247], dtype=torch.uint8, device="cuda").repeat(8)
    sa.view(torch.uint8)[:], sb.view(torch.uint8)[:] = ta[:, None], tb[:, None]
    want = exact_product(a, sa, b, sb)
    got = gemm_fp8(a, sa, b, sb, variant=variant)
    e = (ta.int()[:, None] + tb.int()[None, :] - 254).double()
    for keep in ((ta == 255)[:, None] | (tb == 255)[None, :], e.abs() <= 110):
        same(got[keep], want.float().to(BF16)[keep])
    assert not bool(got[(e < -160) & ~want.isnan()].any())
    assert not bool(got[(e >= 128) & (want != 0)].isfinite().any())  # (a sum of infinities of both signs: NaN)


@pytest.mark.parametrize("m,n,k", [(8, 16, 8192), (8, 64, 8192), (8, 256, 8192), (16, 64, 4096), (5, 33, 8192)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_serving_few_weights_on_long_inputs(m, n, k, dtype):
    """Quantised inside the product where the two-call way would cut K into parts and add in another order: against 64
    bits, and on whole numbers, whose sums are exact in any order, the same bits as in two calls."""
    g = gen(m + n)
    wq, ws = quantize_fp8(torch.randn(n, k, device="cuda", generator=g) * 0.1, block_rows=128)
    x = torch.randn(m, k, device="cuda", generator=g).to(dtype)
    xq, w = quantized(x)[0], values(wq, ws)
    want, size = xq @ w.T, xq.abs() @ w.abs().T
    half, tiny = torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    assert bool(((linear_fp8(x, wq, ws).double() - want).abs() <= half * want.abs() + 2.0 ** -8 * size + tiny).all())
    whole, wide = pair(n, k, g, block_rows=128), small_whole(m, k, g).to(dtype)
    wide[:, ::128] = 4.0  # (each block's largest: the scale is the same everywhere, and every value exact)
    assert torch.equal(linear_fp8(wide, *whole), gemm_fp8(*quantize_fp8(wide), *whole, out_dtype=dtype))
