"""The kernels of the 8-bit floating-point operators that large layers, few rows and long inner dimensions take,
against plain 64-bit computations, by the bounds of test_fp8_gpu.py. Each test states the kernel that its sizes are
meant for and asks the library whether they still take it.
"""

from __future__ import annotations

import pytest
import torch

from test_fp8_gpu import DTYPES, LEAST, any_scales, check_product, rand, values64

pytestmark = pytest.mark.gpu

# rows, columns, inner: the kernel, its tile, parts of the inner dimension
PRODUCTS = {
    **{(m, 1003, 14333): ("few rows", 16, 1) for m in (1, 2, 15, 16)},
    **{(m, 1003, 14333): ("few rows", 32, 1) for m in (17, 31, 32)},
    **{(m, 1003, 14333): ("few rows", 64, 1) for m in (33, 48, 49, 63, 64)},
    (3, 40000, 2000): ("few rows", 16, 1),      # a CTA's run holds whole tiles
    (20, 40000, 2000): ("few rows", 32, 1),
    (50, 28672, 4096): ("few rows", 64, 1),
    (32, 20000, 8000): ("few rows", 32, 1),     # long runs: each ring wraps around many times
    (300, 130, 20001): ("pairs", 128, 8),
    (100, 777, 20000): ("pairs", 128, 8),
    (300, 1500, 20000): ("pairs", 128, 3),
    (65, 3298, 19997): ("pairs", 256, 5),
    (257, 2000, 28672): ("pairs", 256, 4),
    (1100, 9001, 300): ("pairs", 256, 1),
    (520, 20000, 300): ("pairs", 256, 1),
    (777, 3001, 500): ("pairs", 256, 1),
    (600, 9001, 1000): ("pairs", 128, 1),
}
# rows, out, in: columns of a tile, parts of the rows (whatever dy's type), for bf16, fp16 and fp32
GRADIENTS = {
    (200, 4096, 4096): (256, 1),
    (777, 4096, 4096): (256, 1),
    (70, 5000, 4111): (256, 1),
    (130, 4353, 4352): (256, 1),
    (1, 9000, 9000): (256, 1),
}


def same_plan(wq, size) -> None:  # type: ignore[no-untyped-def]
    assert wq._kernels.fp8_gemm_plan(*size) == PRODUCTS[size], size


# ---- the product ---------------------------------------------------------------------


@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("size", PRODUCTS, ids=str)
def test_product_kernels(wq, cuda, size, transpose: bool) -> None:
    """Each kernel, from 8-bit operands with any scales and from a tensor (quantized on the way), into every type, with
    a bias, twice with the same bits."""
    same_plan(wq, size)
    M, N, K = size
    x = rand((M, K), 1, torch.bfloat16)
    w = any_scales(rand((K, N) if transpose else (N, K), 2, scale=0.02), wq)
    a = any_scales(x, wq, 1)
    bias = rand((N,), 3)
    w64 = values64(w) if transpose else values64(w).t()
    x64 = values64(wq.quantize_fp8(x))
    for dtype in DTYPES:
        y = wq.fp8_gemm(a, w, transpose=transpose, bias=bias, out_dtype=dtype)
        check_product(y, values64(a), w64, bias, f"{size} {dtype}")
        assert torch.equal(wq.fp8_gemm(a, w, transpose=transpose, bias=bias, out_dtype=dtype), y)
        y = wq.fp8_gemm(x, w, transpose=transpose, out_dtype=dtype)
        check_product(y, x64, w64, None, f"{size} {dtype} from a tensor")
        assert torch.equal(wq.fp8_gemm(x, w, transpose=transpose, out_dtype=dtype), y)


@pytest.mark.parametrize("size", PRODUCTS, ids=str)
def test_product_kernels_write_their_part_alone(wq, cuda, size) -> None:
    """Into a view inside a larger matrix, from columns that are not 16-byte aligned; values that are not finite stay
    in their rows."""
    same_plan(wq, size)
    M, N, K = size
    x = rand((M, K), 1, torch.bfloat16)
    w = wq.quantize_fp8(rand((N, K), 2, torch.bfloat16, 0.02), block_rows=128)
    y = wq.fp8_gemm(x, w)
    big = torch.full((M + 2, N + 11), 7.0, dtype=torch.bfloat16, device=cuda)
    got = wq.fp8_gemm(x, w, out=big[1:-1, 3:3 + N])
    assert torch.equal(got, y)
    big[1:-1, 3:3 + N] = 7.0
    assert bool((big == 7.0).all())
    x[M // 2, K - 1] = float("nan")
    y2 = wq.fp8_gemm(x, w)
    rest = torch.arange(M, device=cuda) != M // 2
    assert bool(y2[M // 2].isnan().all()) and torch.equal(y2[rest], y[rest])


@pytest.mark.parametrize("size", [(3, 40000, 2000), (32, 20000, 8000), (64, 1003, 14333),
                                  (16, 1003, 14333), (300, 130, 20001), (65, 3298, 19997), (1100, 9001, 300)], ids=str)
def test_product_kernels_back_to_back(wq, cuda, size) -> None:
    """Calls that follow one another without a wait, each on operands that were written just before it: the weights
    that are loaded ahead of the quantizer are the new ones."""
    same_plan(wq, size)
    M, N, K = size
    xs = [rand((M, K), s, torch.bfloat16) for s in (1, 2)]
    ws = [wq.quantize_fp8(rand((N, K), s, torch.bfloat16, 0.02), block_rows=128) for s in (3, 4)]
    want = [wq.fp8_gemm(x, w) for x, w in zip(xs, ws)]
    check_product(want[1], values64(wq.quantize_fp8(xs[1])), values64(ws[1]).t())
    x, w = xs[0].clone(), wq.Fp8Blocks(ws[0].codes.clone(), ws[0].scales.clone(), 128)
    outs = []
    for i in range(12):
        x.copy_(xs[i % 2])
        w.scales.copy_(ws[i % 2].scales)
        w.codes.copy_(ws[i % 2].codes)
        outs.append(wq.fp8_gemm(x, w))
        outs.append(wq.fp8_gemm(x, w))
    for i, y in enumerate(outs):
        assert torch.equal(y, want[i // 2 % 2]), i


@pytest.mark.parametrize("size", [(1, 1003, 14333), (32, 1003, 14333), (64, 1003, 14333), (300, 130, 20001),
                                  (65, 3298, 19997)], ids=str)
def test_product_kernels_streams_and_graphs(wq, cuda, size) -> None:
    """The kernels that add partial sums of several CTAs: on two streams at once, and in two captured graphs that
    are replayed in turn and at once on new values."""
    same_plan(wq, size)
    M, N, K = size
    jobs = []
    for s in (1, 2):
        x = rand((M, K), s, torch.bfloat16)
        w = wq.quantize_fp8(rand((N, K), s + 5, torch.bfloat16, 0.02), block_rows=128)
        jobs.append((x, w, wq.quantize_fp8(x)))

    def run(job):  # type: ignore[no-untyped-def]
        return wq.fp8_gemm(job[0], job[1]), wq.fp8_gemm(job[2], job[1])

    want = [run(j) for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    outs: list[list] = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(run(jobs[i]))
    torch.cuda.synchronize()
    for got, y in zip(outs, want):
        for a, b in got:
            assert torch.equal(a, y[0]) and torch.equal(b, y[1])
    graphs, held = [], []
    for j in jobs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held.append(run(j))
        graphs.append(g)
    for seed in (11, 12):
        for k, j in enumerate(jobs):
            j[0].copy_(rand((M, K), seed + 7 * k, torch.bfloat16))
        want = [run(j) for j in jobs]
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for got, y in zip(held, want):
            assert torch.equal(got[0], y[0]) and torch.equal(got[1], y[1])
    assert wq._kernels.fault_status() == 0


# ---- the weight gradient -----------------------------------------------------------


def same_tile(wq, size, dtype) -> None:  # type: ignore[no-untyped-def]
    assert wq._kernels.fp8_weight_grad_plan(*size, dtype) == GRADIENTS[size], (size, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", GRADIENTS, ids=str)
def test_weight_grad_wide_tile(wq, cuda, size, dtype) -> None:
    """The wide tile, several tiles to a pair of SMs: rows of dw that are written 32 bytes at a time and rows that are
    not, added to dw or not, in every type."""
    same_tile(wq, size, dtype)
    M, N, K = size
    dy = rand((M, N), 1, dtype, 1e-2)
    x = wq.quantize_fp8(rand((M, K), 2, torch.bfloat16))
    x64, dy64 = values64(x), dy.double().t()
    ref, size64 = dy64 @ x64, dy64.abs() @ x64.abs()
    for out in DTYPES:
        check_product(wq.fp8_weight_grad(dy, x, out_dtype=out), dy64, x64, what=f"{size} {dtype} {out}")
        g = rand((N, K), 5, out)
        want, mag = g.double() + ref, g.double().abs() + size64
        got = wq.fp8_weight_grad(dy, x, out=g, accumulate=True)
        assert got.data_ptr() == g.data_ptr()
        # LEAST: values below the type's least normal number lie a whole least subnormal apart (fp16 below 2^-14:
        # 2^-24), so the nearest is off by up to half of one, 2^-25, however small the value
        bound = torch.finfo(out).eps / 2 * want.abs() + 2.0 ** -23 * (M / 16 + M / 128 + 5) * mag + LEAST[out]
        assert bool(((g.double() - want).abs() <= bound).all()), (size, dtype, out)
    big = torch.full((N + 2, K + 9), 0.5, device=cuda)
    wq.fp8_weight_grad(dy, x, out=big[1:-1, 4:4 + K])
    check_product(big[1:-1, 4:4 + K], dy64, x64)
    big[1:-1, 4:4 + K] = 0.5
    assert bool((big == 0.5).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_weight_grad_operand_of_the_other_cta(wq, cuda, dtype) -> None:
    """Half of each tile's columns come from an operand that the pair's other CTA made in its own shared memory: many
    tiles and steps, many times over while the card is busy, every result with the same bits and right."""
    assert wq._kernels.fp8_weight_grad_plan(1000, 4096, 4096, dtype) == (256, 1)
    x = wq.quantize_fp8(rand((1000, 4096), 1, torch.bfloat16))
    dy = rand((1000, 4096), 2, dtype, 1e-2)
    dw = wq.fp8_weight_grad(dy, x)
    check_product(dw, dy.double().t(), values64(x))
    out = torch.empty_like(dw)
    for _ in range(40):
        out.fill_(float("nan"))
        wq.fp8_weight_grad(dy, x, out=out)
        assert torch.equal(out, dw)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("M,N,K", [(64, 2304, 768), (40, 4096, 4096)])
def test_weight_grad_terms_add_up_from_the_least(wq, cuda, M: int, N: int, K: int, dtype) -> None:
    """One step of rows, all products positive. dy's terms are 2^-8 and 2^-16 of it, and the sums of the lesser ones are
    in place before the first term's four additions (16 rows each), so those four are the only ones of the result's
    size: each off by at most a step, 2^-23 of it, the others by 2^-8 of that, then the fp32 registers' rounding by
    half a step. Were the first term added first, all twelve additions would cut at the result's size."""
    dy = rand((M, N), 1, dtype).abs()
    x = wq.quantize_fp8(rand((M, K), 2, torch.bfloat16).abs())
    dw = wq.fp8_weight_grad(dy, x)
    ref = dy.double().t() @ values64(x)
    steps = 4 * (1 + 2.0 ** -7 + 2.0 ** -15) + 0.5
    assert bool(((dw.double() - ref).abs() <= steps * 2.0 ** -23 * ref).all())


@pytest.mark.parametrize("M,N,K", [(200, 4096, 4096), (777, 300, 520), (5000, 256, 384)])
def test_weight_grad_any_scales(wq, cuda, M: int, N: int, K: int) -> None:
    """Scales that are no powers of two: each code * scale is rounded to bfloat16 (by half a step, 2^-8, after a
    rounding to fp32) before the product."""
    x = any_scales(rand((M, K), 2), wq, 1)
    for dtype in DTYPES:
        dy = rand((M, N), 1, dtype, 1e-2)
        dw = wq.fp8_weight_grad(dy, x)
        x64, dy64 = values64(x), dy.double().t()
        ref, size = dy64 @ x64, dy64.abs() @ x64.abs()
        bound = 2.0 ** -24 * ref.abs() + (2.0 ** -8 + 2.0 ** -23 * (M / 16 + M / 128 + 6)) * size
        assert bool(((dw.double() - ref).abs() <= bound).all()), dtype
