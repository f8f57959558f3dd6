"""Times of the 8-bit operators on one MI355X, and programs to profile (profiles/fp8/README.md says what was kept).

  python3 profiles/provenance/tools/fp8_times.py times > times.txt
  python3 profiles/provenance/tools/fp8_times.py choice 120 > choice.txt
  rocprofv3 --kernel-trace --stats ... -- python3 profiles/provenance/tools/fp8_times.py profile train 4096 8192 8192

A time is a call's share of a captured graph of many calls, best of 7 replays: no host time.  "memory": the calls
go round operands of 1 GiB and more in all, so each comes from memory; "caches": the same operands again.
"""
import math
import os
import random
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(__file__))))))
from kubernetes_gpu_exporter_amd.ops.fp8 import (dequantize_fp8, gemm_fp8, gemm_fp8_parts, gemm_fp8_variant,  # noqa: E402
                                                 linear_fp8, quantize_fp8, quantize_fp8_both, transpose_fp8)

BF16 = torch.bfloat16


def graph_us(calls, reps=7):
    """us a call of a graph of `calls` (functions), which run once before it is captured."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for f in calls:
            f()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for f in calls:
            f()
    best = math.inf
    for _ in range(reps):
        begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        begin.record()
        graph.replay()
        end.record()
        end.synchronize()
        best = min(best, begin.elapsed_time(end) * 1e3 / len(calls))
    return best


def random_codes(rows, cols):
    """8-bit values of random bits below e4m3's NaN, in rows as quantize_fp8 lays them out, without a wide tensor of the size."""
    ld = quantize_fp8(torch.zeros(2, cols, device="cuda", dtype=BF16))[0].stride(0)
    whole = torch.randint(0, 0x77, (rows, ld), device="cuda", dtype=torch.uint8)
    return whole.view(torch.float8_e4m3fn)[:, :cols]


def weight(n, k):
    scales = torch.full((-(-n // 128), -(-(-(-k // 128)) // 4) * 4), 120, device="cuda", dtype=torch.uint8)
    return random_codes(n, k), scales.view(torch.float8_e8m0fnu)[:, :-(-k // 128)]


def weights(n, k, memory):
    copies = max(2, min(256, -(-(1 << 30) // (n * k)))) if memory else 1
    return [weight(n, k) for _ in range(copies)]


def both(make, n, k):
    """(us from memory, us from the caches) of make(weight)."""
    out = []
    for memory in (True, False):
        ws = weights(n, k, memory)
        calls = [make(*w) for w in ws]
        out.append(graph_us(calls * max(1, -(-20 // len(calls)))))
    return out


def line(*parts):
    print(*parts, flush=True)


def times():
    line("# gemm_fp8: random values and zeros, us (operands from the caches where they fit)")
    for size in (4096, 8192):
        x = torch.randn(size, size, device="cuda", dtype=BF16)
        for name, t in (("random", x), ("zeros", torch.zeros_like(x))):
            a, b = quantize_fp8(t), quantize_fp8(t, block_rows=128)
            us = graph_us([lambda: gemm_fp8(*a, *b)] * 10)
            line(f"gemm {size}^3 {name}: {us:.1f} us, {2e-9 * size ** 3 / us:.3f} PFLOP/s")

    line("# linear_fp8 with 8-bit weights, us from memory / from the caches: as called, and as quantize_fp8 and gemm_fp8")
    for n, k in ((512, 512), (4096, 2048), (4096, 4096), (8192, 4096), (16384, 2048), (4096, 8192), (1024, 8192), (8192, 8192)):
        for m in (1, 4, 8, 16):
            x = torch.randn(m, k, device="cuda", dtype=BF16)
            one = both(lambda w, s: lambda: linear_fp8(x, w, s), n, k)
            two = both(lambda w, s: lambda: gemm_fp8(*quantize_fp8(x), w, s), n, k)
            line(f"serve {m} x {n} x {k}: {one[0]:.1f} / {one[1]:.1f}; two calls {two[0]:.1f} / {two[1]:.1f}")
    for m, n, k in ((64, 4096, 14336), (128, 4096, 8192), (256, 4096, 4096), (512, 8192, 4096), (512, 4096, 14336)):
        x = torch.randn(m, k, device="cuda", dtype=BF16)
        q = quantize_fp8(x)
        one = both(lambda w, s: lambda: linear_fp8(x, w, s), n, k)
        alone = both(lambda w, s: lambda: gemm_fp8(*q, w, s), n, k)
        line(f"serve {m} x {n} x {k}: {one[0]:.1f} / {one[1]:.1f}; its product {alone[0]:.1f} / {alone[1]:.1f} "
             f"(kernel {gemm_fp8_variant(m, n, k)}, {gemm_fp8_parts(m, n, k)} parts)")

    line("# serving's backward pass (quantise dy, transpose the weight, product), us from the caches")
    for m, n, k in ((16, 4096, 8192), (512, 8192, 4096)):
        w, s = weight(n, k)
        dy = torch.randn(m, n, device="cuda", dtype=BF16)
        line(f"serve backward {m} x {n} x {k}: {graph_us([lambda: gemm_fp8(*quantize_fp8(dy), *transpose_fp8(w, s))] * 10):.1f}, "
             f"of which the transposition {graph_us([lambda: transpose_fp8(w, s)] * 10):.1f}")

    line("# quantise, give back, transpose of 4096 x 8192, us, tensors in turn (eight of 64 MiB), TB/s of what they must move")
    m, k = 4096, 8192
    xs = [torch.randn(m, k, device="cuda", dtype=BF16) for _ in range(8)]
    n = m * k
    for block_rows in (1, 128):
        qs = [quantize_fp8(x, block_rows=block_rows) for x in xs]
        for name, make, moved in (("quantize_fp8", lambda x, q: lambda: quantize_fp8(x, block_rows=block_rows), 3 * n),
                                  ("quantize_fp8_both", lambda x, q: lambda: quantize_fp8_both(x, block_rows=block_rows), 4 * n),
                                  ("dequantize_fp8", lambda x, q: lambda: dequantize_fp8(*q), 3 * n),
                                  ("transpose_fp8", lambda x, q: lambda: transpose_fp8(*q), 2 * n)):
            us = graph_us([make(x, q) for x, q in zip(xs, qs)] * 2)
            line(f"{name} blocks of {block_rows} x 128: {us:.1f} us, {moved / us * 1e-6:.2f} TB/s")

    line("# what a CU loads: us a K tile from K = 4224 to 8320, and GB/s of both operands; b from memory / from the caches")
    for edge, variant, rows, cols in ((64, 4, 64, 64), (64, 4, 64, 4096), (64, 4, 64, 16384), (128, 1, 128, 128),
                                      (128, 1, 128, 8192), (128, 1, 256, 16384)):
        got = []
        for k in (4224, 8320):
            a = weight(rows, k)
            got.append(both(lambda *b: lambda: gemm_fp8(*a, *b, variant=variant, parts=1), cols, k))
        a, b = ((got[1][i] - got[0][i]) / 32 for i in range(2))
        line(f"{edge} x {edge} tile, {rows // edge * cols // edge} blocks: {a:.3f} / {b:.3f} us, "
             f"{2 * edge * 128 / a * 1e-3:.0f} / {2 * edge * 128 / b * 1e-3:.0f} GB/s a CU")

    line("# a training step of 4096 x 8192 x 8192, us, steps one after the other; one gradient alone")
    x, w = (torch.randn(s, 8192, device="cuda").to(BF16).requires_grad_() for s in (4096, 8192))
    dy = torch.randn(4096, 8192, device="cuda").to(BF16)
    for name, leaves in (("both gradients", (x, w)), ("dx alone", (x,)), ("dw alone", (w,))):
        best = math.inf
        for _ in range(4):
            begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            begin.record()
            for _ in range(8):
                torch.autograd.grad(linear_fp8(x, w), leaves, dy)
            end.record()
            end.synchronize()
            best = min(best, begin.elapsed_time(end) * 1e3 / 8)
        line(f"train, {name}: {best:.0f}")

    line("# a small training step, 64 x 512 x 512, both gradients: us on the host, steps one after the other")
    x, w = (torch.randn(s, 512, device="cuda").to(BF16).requires_grad_() for s in (64, 512))
    dy = torch.randn(64, 512, device="cuda").to(BF16)
    for name, layer in (("linear_fp8", linear_fp8), ("torch's linear in bf16", torch.nn.functional.linear)):
        best = math.inf
        for _ in range(10):
            torch.cuda.synchronize()
            begin = time.perf_counter()
            for _ in range(200):
                torch.autograd.grad(layer(x, w), (x, w), dy)
            torch.cuda.synchronize()
            best = min(best, (time.perf_counter() - begin) * 1e6 / 200)
        line(f"{name}: {best:.1f}")


def choice(count):
    """How far the chosen kernel is from the fastest, over random sizes."""
    rng = random.Random(20)

    def size(low, high):
        return round(math.exp(rng.uniform(math.log(low), math.log(high))))
    loss = []
    for i in range(count):
        memory = i % 2 == 0
        m, n, k = size(1, 16 if i % 3 == 0 else 8192), size(64, 16384), size(128, 16384)
        a = weight(m, k)[0], torch.full((m, -(-(-(-k // 128)) // 4) * 4), 120, device="cuda", dtype=torch.uint8).view(
            torch.float8_e8m0fnu)[:, :-(-k // 128)]
        ws = weights(n, k, memory)
        tried = {}
        for variant in (1, 2, 3, 4, 5, 6):
            for parts in (1, 2, 3, 4, 6, 8, 12, 16) if variant in (1, 4) else (1,):
                if parts > 1 and (parts > -(-k // 512) or -(-m // 128) * -(-n // 128) * parts > 512):
                    continue
                if gemm_fp8_variant(m, n, k, variant) < 0:
                    continue
                calls = [(lambda w, s: lambda: gemm_fp8(*a, w, s, variant=variant, parts=parts))(*w) for w in ws]
                tried[variant, parts] = graph_us((calls * max(1, -(-8 // len(calls))))[:max(8, min(len(calls), 64))], 4)
        calls = [(lambda w, s: lambda: gemm_fp8(*a, w, s))(*w) for w in ws]
        chosen = graph_us((calls * max(1, -(-8 // len(calls))))[:max(8, min(len(calls), 64))], 4)
        best = min(tried, key=tried.get)
        loss.append((m, max(0.0, chosen / tried[best] - 1)))
        line(f"{m} x {n} x {k} {'memory' if memory else 'caches'}: chosen {gemm_fp8_variant(m, n, k)}, "
             f"{gemm_fp8_parts(m, n, k)} parts {chosen:.1f} us; fastest {best} {tried[best]:.1f}")
    few = [v for m, v in loss if m <= 16]
    line(f"# {count} sizes: {100 * sum(v for _, v in loss) / count:.1f} % behind the fastest in the mean; up to 16 rows "
         f"{100 * sum(few) / max(1, len(few)):.1f} %")


def profile(kind, m, n, k):
    x = torch.randn(m, k, device="cuda").to(BF16)
    if kind == "train":
        x.requires_grad_()
        w = (torch.randn(n, k, device="cuda") * 0.02).to(BF16).requires_grad_()
        dy = torch.randn(m, n, device="cuda").to(BF16)
        for _ in range(10):
            torch.autograd.grad(linear_fp8(x, w), (x, w), dy)
    else:
        ws = weights(n, k, True)
        for i in range(100):
            linear_fp8(x, *ws[i % len(ws)])
    torch.cuda.synchronize()


if __name__ == "__main__":
    if sys.argv[1] == "times":
        times()
    elif sys.argv[1] == "choice":
        choice(int(sys.argv[2]))
    else:
        profile(sys.argv[2], *map(int, sys.argv[3:6]))
