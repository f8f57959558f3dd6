"""The 8-bit operators' refusals (CPU: every check comes before anything is launched)."""
import pytest
import torch

from kubernetes_gpu_exporter_amd.ops.fp8 import (dequantize_fp8, gemm_fp8, gemm_fp8_parts, gemm_fp8_variant,
                                                 linear_fp8, quantize_fp8, quantize_fp8_both, transpose_fp8)
from tests.fp8_oracle import E4M3, E5M2, E8M0, pair, quantized, values


def q(m, k, block_rows=1, dtype=E4M3):
    return pair(m, k, torch.Generator().manual_seed(m * k), dtype, block_rows)


def test_types_are_refused():
    x = torch.zeros(4, 128)
    with pytest.raises(TypeError, match="bfloat16, float16 or float32"):
        quantize_fp8(x.double())
    with pytest.raises(TypeError, match="e4m3fn or float8_e5m2"):
        quantize_fp8(x, torch.float16)
    a, s = q(4, 128)
    with pytest.raises(TypeError, match="must be float8"):
        gemm_fp8(x, s, a, s)
    with pytest.raises(TypeError, match="e8m0"):
        gemm_fp8(a, s.view(torch.uint8), a, s)
    with pytest.raises(TypeError, match="writes bfloat16 or float16"):
        gemm_fp8(a, s, a, s, out_dtype=torch.float32)
    with pytest.raises(TypeError, match="gives bfloat16"):
        dequantize_fp8(a, s, torch.float64)
    with pytest.raises(TypeError, match="activations"):
        linear_fp8(x, x)
    with pytest.raises(TypeError, match="weights"):
        linear_fp8(x.bfloat16(), x)


@pytest.mark.parametrize("block_rows", [0, 2, 64, 256])
def test_block_rows_are_refused(block_rows):
    for call in (quantize_fp8, quantize_fp8_both):
        with pytest.raises(ValueError, match="block_rows"):
            call(torch.zeros(4, 128), block_rows=block_rows)


def test_shapes_are_refused():
    a, s = q(4, 256)
    b, t = q(8, 128)
    with pytest.raises(ValueError, match="shape mismatch"):
        gemm_fp8(a, s, b, t)
    with pytest.raises(ValueError, match="the scales of a"):
        gemm_fp8(a, s[:, :1], a, s)
    with pytest.raises(ValueError, match="the scales of b"):
        gemm_fp8(a, s, a, s[:3])
    with pytest.raises(ValueError, match="2-dimensional"):
        transpose_fp8(a[0], s)
    with pytest.raises(ValueError, match="2-dimensional"):
        quantize_fp8(torch.zeros(128))
    with pytest.raises(ValueError, match="out must be"):
        gemm_fp8(a, s, a, s, out=torch.zeros(4, 5, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="shape mismatch"):
        linear_fp8(torch.zeros(2, 3, dtype=torch.bfloat16), torch.zeros(4, 5, dtype=torch.bfloat16))


def test_layouts_are_refused():
    a, s = q(4, 256)
    with pytest.raises(ValueError, match="columns next to each other"):
        quantize_fp8(torch.zeros(128, 4).T)
    with pytest.raises(ValueError, match="columns next to each other"):
        quantize_fp8(torch.zeros(1, 128).expand(4, 128))  # rows that overlap
    with pytest.raises(ValueError, match="columns next to each other"):
        transpose_fp8(a.T, q(256, 4)[1])
    packed = torch.zeros(4 * 250, dtype=torch.uint8).view(E4M3).view(4, 250)
    with pytest.raises(ValueError, match="multiples of 16"):
        gemm_fp8(packed, s, packed, s)
    shifted = torch.zeros(4 * 256 + 16, dtype=torch.uint8)[8:8 + 4 * 256].view(E4M3).view(4, 256)
    with pytest.raises(ValueError, match="multiples of 16"):
        gemm_fp8(shifted, s, shifted, s)
    tight = torch.zeros(4, 2, dtype=torch.uint8).view(E8M0)
    with pytest.raises(ValueError, match="multiples of 4"):
        gemm_fp8(a, tight, a, tight)
    with pytest.raises(ValueError, match="multiples of 16"):
        gemm_fp8(a[:1].expand(4, 256), s, a, s)


def test_weights_in_8_bits_take_no_gradient():
    w, s = q(256, 128, 128)
    with pytest.raises(ValueError, match="no gradient"):
        linear_fp8(torch.zeros(2, 128, dtype=torch.bfloat16), w.clone().requires_grad_(), s)


def test_cpu_tensors_are_refused():
    a, s = q(4, 256)
    for call in (lambda: quantize_fp8(torch.zeros(4, 256)), lambda: quantize_fp8_both(torch.zeros(4, 256)),
                 lambda: quantize_fp8(torch.zeros(4, 256), stream=0), lambda: dequantize_fp8(a, s),
                 lambda: transpose_fp8(a, s), lambda: gemm_fp8(a, s, a, s),
                 lambda: linear_fp8(torch.zeros(4, 256).bfloat16(), torch.zeros(8, 256).bfloat16())):
        with pytest.raises(ValueError, match="same GPU"):
            call()


def test_variants_are_refused():
    a, s = q(4, 128)
    for variant in (-1, 2, 99):  # 2, the 256x256 tile, takes K >= 144
        with pytest.raises(ValueError, match="variant"):
            gemm_fp8(a, s, a, s, variant=variant)
    b, t = q(17, 256)
    for variant in (3, 6):  # few rows: up to 16
        with pytest.raises(ValueError, match="variant"):
            gemm_fp8(b, t, b, t, variant=variant)


def test_parts_are_refused():
    a, s = q(4, 1024)
    for variant, parts in ((1, -1), (1, 3), (4, 17), (0, 2), (2, 2), (3, 2), (5, 2), (6, 2)):  # 2 units of 512 in K
        with pytest.raises(ValueError, match="parts"):
            gemm_fp8(a, s, a, s, variant=variant, parts=parts)


@pytest.mark.parametrize("dtype", [E4M3, E5M2])
def test_oracle_matches_torch_rounding(dtype):
    """The oracle's rounding is torch's own cast where no scale applies (largest value = the type's)."""
    x = torch.randn(64, 128, generator=torch.Generator().manual_seed(1)) * torch.logspace(-4, 2, 128)
    x[:, 0] = 448.0 if dtype == E4M3 else 57344.0
    got, e = quantized(x.clamp(-57344 if dtype == E5M2 else -448, 57344 if dtype == E5M2 else 448), dtype)
    assert bool((e == 0).all())
    assert torch.equal(got.float(), x.clamp(-57344 if dtype == E5M2 else -448, 57344 if dtype == E5M2 else 448)
                       .to(dtype).float())


def test_oracle_values_of_a_hand_made_pair():
    a = torch.tensor([[1.0, -2.0, 448.0]]).to(E4M3)
    s = torch.tensor([[128]], dtype=torch.uint8).view(E8M0)
    assert values(a, s).tolist() == [[2.0, -4.0, 896.0]]


@pytest.mark.parametrize("M,N,K,variant,want", [
    (8192, 8192, 8192, 0, 2), (4096, 4096, 4096, 0, 2),  # many tiles: 256 x 256
    (2048, 4096, 4096, 0, 5), (1024, 4096, 4096, 0, 1), (333, 1001, 2050, 0, 4),
    (1, 4096, 4096, 0, 3), (16, 8192, 8192, 0, 6), (16, 32768, 4096, 0, 4),
    (8192, 8192, 128, 0, 5), (8192, 8192, 128, 2, -1),  # one K tile: not the 256 x 256 tile's
    (17, 64, 64, 3, -1), (17, 64, 64, 6, -1), (16, 64, 64, 6, 6), (1, 1, 0, 0, 3), (100, 100, 0, 0, 4),
    (64, 64, 64, 7, -1), (64, 64, 64, -1, -1),
])
def test_gemm_variant_resolution(M, N, K, variant, want):
    assert gemm_fp8_variant(M, N, K, variant) == want


@pytest.mark.parametrize("M,N,K,parts", [
    (64, 4096, 8192, 4), (64, 1024, 8192, 8), (1, 1024, 8192, 1), (16, 1024, 8192, 16), (256, 4096, 8192, 1),
    (64, 1024, 2048, 1), (64, 64, 0, 1), (0, 64, 8192, 1), (8192, 8192, 8192, 1)])
def test_gemm_parts_of_k(M, N, K, parts):
    assert gemm_fp8_parts(M, N, K) == parts


@pytest.mark.parametrize("reverse", [False, True])
def test_forward_mode_is_refused(reverse):
    """Also where no reverse-mode gradient is recorded, and under no_grad, which does not stop forward mode."""
    import torch.autograd.forward_ad as forward_ad
    x, w = torch.zeros(4, 128).bfloat16(), torch.zeros(8, 128).bfloat16().requires_grad_(reverse)
    wq, ws = q(256, 128, 128)
    with forward_ad.dual_level():
        for call in (lambda: linear_fp8(forward_ad.make_dual(x, x), w), lambda: linear_fp8(forward_ad.make_dual(x, x), wq, ws),
                     lambda: linear_fp8(x, forward_ad.make_dual(w, torch.zeros_like(w)))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                call()


@pytest.mark.parametrize("m,k,block_rows", [(1, 1, 1), (5, 300, 1), (130, 1101, 128), (4, 256, 1), (129, 0, 128), (0, 40, 1)])
def test_copies_are_aligned_on_the_cpu(m, k, block_rows):
    """Any strides in; rows at multiples of 16 and 4 bytes, the same codes and scales out; what fits stays itself."""
    from kubernetes_gpu_exporter_amd.ops.fp8 import align_fp8
    a, s = q(m, k, block_rows) if m and k else (torch.zeros(m, k).to(E4M3), torch.zeros(-(-m // block_rows), -(-k // 128)).to(E8M0))
    again = align_fp8(a, s)
    assert again[0] is a and again[1] is s
    for copy in (lambda t: t.clone(), lambda t: t.contiguous(), lambda t: t.T.contiguous().T,
                 lambda t: torch.cat([torch.zeros(1, dtype=torch.uint8), t.contiguous().view(torch.uint8).flatten()])[1:]
                 .view(t.dtype).view(t.shape)):
        b, t = align_fp8(copy(a), copy(s))
        assert torch.equal(b.float(), a.float()) and torch.equal(t.view(torch.uint8), s.view(torch.uint8))
        for got, pad in ((b, 16), (t, 4)):
            if got.numel():
                assert got.data_ptr() % pad == 0 and (got.shape[1] == 1 or got.stride(1) == 1)
                assert got.shape[0] == 1 or (got.stride(0) % pad == 0 and got.stride(0) >= got.shape[1])


def test_pairs_that_are_none_are_not_aligned():
    from kubernetes_gpu_exporter_amd.ops.fp8 import align_fp8
    a, s = q(4, 256)
    with pytest.raises(TypeError, match="float8"):
        align_fp8(a.float(), s)
    with pytest.raises(TypeError, match="e8m0"):
        align_fp8(a, s.view(torch.uint8))
    with pytest.raises(ValueError, match="the scales of q"):
        align_fp8(a, s[:, :1])
    with pytest.raises(ValueError, match="2-dimensional"):
        align_fp8(a[0], s)
    with pytest.raises(ValueError, match="align_fp8"):  # the refusal of a copy says what to do
        b, t = q(4, 250)
        gemm_fp8(b.contiguous(), t, b, t)


@pytest.mark.parametrize("M,N,K,variant,want", [
    (1, 1 << 26, 16, 3, 3), (1, 1 << 26, 16, 6, 6), (1, 1 << 26, 8192, 3, -1), (1, 1 << 26, 8192, 6, 6),
    (1, 1 << 27, 8192, 6, -1), (16, 1 << 30, 16, 6, 6), (16, 1 << 30, 16, 3, -1),
    (1 << 21, 1 << 16, 64, 4, -1), (1 << 21, 1 << 16, 64, 1, 1), (1 << 24, 1 << 24, 256, 2, -1), (1 << 24, 1 << 24, 256, 0, -1)])
def test_kernels_whose_launch_is_too_large_are_not_chosen(M, N, K, variant, want):
    """A launch has less than 2^32 threads: 64 for each 512 of K (at most 1024) and 16 or 32 columns of C, 256 or 512 a tile."""
    assert gemm_fp8_variant(M, N, K, variant) == want


@pytest.mark.parametrize("M,N,K", [(1, 1 << 26, 16), (16, 1 << 28, 64), (1, 1 << 26, 8192), (1 << 21, 1 << 16, 64),
                                   (1 << 23, 1 << 14, 16)])
def test_the_choice_passes_over_them(M, N, K):
    chosen = gemm_fp8_variant(M, N, K)
    assert chosen > 0 and gemm_fp8_variant(M, N, K, chosen) == chosen


@pytest.mark.parametrize("M,N,K,dx,dw,taken", [
    (1 << 22, 8192, 16, True, False, False), ((1 << 22) - 1, 8192, 16, True, False, True),  # 2^28 blocks of dy, just fewer
    (1 << 22, 8192, 16, False, False, True), (1 << 22, 8192, 16, False, True, False),
    (1 << 27, 129, 8, True, False, False), (1 << 27, 128, 8, True, False, True),
    (1 << 28, 8, 4, False, False, False)])  # x itself
def test_sizes_that_the_backward_pass_would_refuse(M, N, K, dx, dw, taken):
    """Refused before anything runs, the forward pass too; what is taken goes on to the next check."""
    x = torch.empty(M, K, dtype=torch.bfloat16).requires_grad_(dx)  # (never touched: no memory)
    w = torch.empty(N, K, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="same GPU" if taken else "larger than the kernels index"):
        linear_fp8(x, w.clone().requires_grad_(dw))
    if not dw:
        wq, ws = torch.zeros(N, 16, dtype=torch.uint8)[:, :K].view(E4M3), torch.zeros(-(-N // 128), 4, dtype=torch.uint8)
        with pytest.raises(ValueError, match="same GPU" if taken else "larger than the kernels index"):
            linear_fp8(x, wq, ws.view(E8M0)[:, :1])


@pytest.mark.parametrize("far", [1 << 32, (1 << 32) + 1, -(1 << 32)])
def test_variants_and_parts_past_32_bits_are_refused(far):
    a, s = q(4, 1024)
    with pytest.raises(ValueError, match="variant"):
        gemm_fp8(a, s, a, s, variant=far)
    with pytest.raises(ValueError, match="parts"):
        gemm_fp8(a, s, a, s, variant=1, parts=far)
    assert gemm_fp8_variant(4, 4, 1024, far) == -1
