"""The 8-bit operators in 64 bits, from their definition: blocks of 128 share 2^e, values are
rounded once to nearest even (tests/test_fp8.py, tests/test_fp8_gpu.py)."""
import torch

E4M3, E5M2, E8M0 = torch.float8_e4m3fn, torch.float8_e5m2, torch.float8_e8m0fnu
LARGEST = {E4M3: 448.0, E5M2: 57344.0}
STEPS = {E4M3: (3, -6), E5M2: (2, -14)}  # bits behind the point, the smallest normal exponent


def two(e):
    """2^e in 64 bits for whole e."""
    return torch.ldexp(torch.ones_like(e, dtype=torch.float64, device="cpu"), e.cpu().double()).to(e.device)


def floor_log2(v):
    """floor(log2 v) of v > 0."""
    return torch.frexp(v.cpu())[1].to(v.device) - 1


def blocked(x, block_rows):
    m, k = x.shape
    r, c = -(-m // block_rows), -(-k // 128)
    full = torch.zeros(r * block_rows, c * 128, dtype=torch.float64, device=x.device)
    full[:m, :k] = x.double()
    return full.reshape(r, block_rows, c, 128)


def quantized(x, dtype=E4M3, block_rows=1):
    """(the values that x becomes, in 64 bits; the exponents of its blocks)."""
    m, k = x.shape
    b = blocked(x, block_rows)
    top = torch.where(b.isfinite(), b.abs(), 0.0).amax(dim=(1, 3))
    largest = LARGEST[dtype]
    e = floor_log2(torch.where(top > 0, top / largest, 1.0))
    e = torch.where(top > largest * two(e), e + 1, e)  # the smallest e with top <= largest 2^e
    e = torch.where(top > 0, e.clamp(min=-127), torch.zeros_like(e))
    scale = two(e)[:, None, :, None]
    v = b / scale
    bits, lowest = STEPS[dtype]
    finite = torch.where(v.isfinite(), v, 0.0)
    unit = two(floor_log2(torch.where(finite == 0, 1.0, finite.abs())).clamp(min=lowest) - bits)
    q = torch.round(finite / unit) * unit
    q = torch.where(v.isfinite(), q, v if dtype == E5M2 else torch.full_like(v, float("nan")))
    r, s, c, _ = q.shape
    return (q * scale).reshape(r * s, c * 128)[:m, :k], e


def values(q, scale):
    """What (q, scale) stands for, in 64 bits."""
    m, k = q.shape
    block_rows = 1 if scale.shape[0] == m else 128
    e = scale.view(torch.uint8).to(torch.int64)
    s = torch.where(e == 255, float("nan"), two(e - 127))
    return q.double() * s.repeat_interleave(block_rows, 0)[:m].repeat_interleave(128, 1)[:, :k]


def small_whole(m, k, g, top=4):
    """Whole numbers of [-top, top]: exact in both 8-bit types, their sums exact in 32 bits."""
    return torch.randint(-top, top + 1, (m, k), generator=g, device=g.device).float()


def pair(m, k, g, dtype=E4M3, block_rows=1, spread=3, pad=0):
    """An operand made by hand, not by quantize_fp8: small whole numbers times powers of two of
    [2^-spread, 2^spread] per block; rows 16-byte aligned, `pad` more bytes of NaN behind each."""
    ld = -(-k // 16) * 16 + pad
    q = torch.full((m, ld), 0x7F, dtype=torch.uint8, device=g.device).view(dtype)
    q[:, :k] = small_whole(m, k, g).to(dtype)
    r, c = -(-m // block_rows), -(-k // 128)
    s = torch.full((r, -(-c // 4) * 4), 255, dtype=torch.uint8, device=g.device)
    s[:, :c] = torch.randint(127 - spread, 128 + spread, (r, c), generator=g, device=g.device).to(torch.uint8)
    return q[:, :k], s.view(E8M0)[:, :c]
