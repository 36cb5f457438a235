"""Blocks of 8-bit floating point on the GPU against plain 64-bit computations.

Tolerances. u = 2^-24 is half a step of fp32 and h half a step of the output's
type (2^-24, 2^-11, 2^-8). A product of K terms is held in fp32: at most
K / 16 + K / 128 + 4 sequential additions, each off by at most a whole step 2u
(a matrix unit may cut off what it adds), of partial sums no larger than
S = sum |a||w|; then one rounding to the output: |y - y64| <= h |y64| +
2u (K / 16 + K / 128 + 4) S (+ half the output type's least subnormal).
Quantization and reconstruction are exact statements and compared for equality.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
DTYPES = (torch.float32, torch.float16, torch.bfloat16)
LEAST = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def rand(shape, seed: int, dtype=torch.float32, scale: float = 1.0) -> torch.Tensor:  # type: ignore[no-untyped-def]
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


# every finite e4m3 value that is not negative, by its code
TABLE = torch.arange(127, dtype=torch.uint8).view(E4M3).to(torch.float64)


def codes64(x: torch.Tensor, block_rows: int) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes as uint8, scales as fp64) by the definition: block by block, the code of the nearest table entry."""
    x = x.double().cpu()
    rows, cols = x.shape
    codes = torch.empty(rows, cols, dtype=torch.uint8)
    scales = torch.empty(-(-rows // block_rows), -(-cols // 128), dtype=torch.float64)
    mid = (TABLE[1:] + TABLE[:-1]) / 2
    for i in range(scales.shape[0]):
        for j in range(scales.shape[1]):
            b = x[i * block_rows:(i + 1) * block_rows, j * 128:(j + 1) * 128]
            top = float(torch.where(b.isfinite(), b.abs(), torch.zeros_like(b)).max())
            s = 1.0
            if top > 0:
                s = 2.0 ** -117
                while top > 448.0 * s:
                    s *= 2.0
            v = b / s
            near = torch.searchsorted(mid, v.abs().contiguous(), right=False)
            tie = (near < 126) & (mid[near.clamp_max(125)] == v.abs())
            near = torch.where(tie & (near % 2 == 1), near + 1, near)     # to the even code
            c = near.to(torch.uint8) + torch.where(torch.signbit(v), 128, 0).to(torch.uint8)
            c = torch.where(b.isfinite(), c, torch.full_like(c, 0x7F))
            codes[i * block_rows:(i + 1) * block_rows, j * 128:(j + 1) * 128] = c
            scales[i, j] = s
    return codes, scales


def values64(q) -> torch.Tensor:  # type: ignore[no-untyped-def]
    s = q.scales.double().repeat_interleave(q.block_rows, 0)[: q.shape[0]]
    return q.codes.double() * s.repeat_interleave(128, 1)[:, : q.shape[1]]


def same_codes(got: torch.Tensor, want: torch.Tensor) -> None:
    got = got.view(torch.uint8).cpu() if got.dtype == E4M3 else got.cpu()
    nan = (want & 0x7F) == 0x7F
    assert torch.equal((got & 0x7F) == 0x7F, nan)
    assert torch.equal(got[~nan], want[~nan])


def check_product(y: torch.Tensor, a64: torch.Tensor, w64: torch.Tensor, bias=None, what: str = "") -> None:  # type: ignore[no-untyped-def]
    """y against a64 @ w64 (+ bias), both fp64, by the bound above."""
    K = a64.shape[1]
    ref, size = a64 @ w64, a64.abs() @ w64.abs()
    if bias is not None:
        ref, size = ref + bias.double(), size + bias.double().abs()
    h = torch.finfo(y.dtype).eps / 2
    bound = h * ref.abs() + 2.0 ** -23 * (K / 16 + K / 128 + 4) * size + LEAST[y.dtype]
    worst = float(((y.double() - ref).abs() / bound).max()) if y.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3g} of the bound"


def any_scales(w: torch.Tensor, wq, block_rows: int = 128):  # type: ignore[no-untyped-def]
    """An operand whose scales are no powers of two, laid out row by row."""
    q = wq.quantize_fp8(w, block_rows=block_rows)
    g = torch.Generator(device="cuda").manual_seed(7)
    return wq.Fp8Blocks(q.codes, (q.scales * (0.5 + torch.rand(q.scales.shape, generator=g, device="cuda"))).contiguous(),
                        block_rows)


# ---- quantization ----------------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_matches_the_definition(wq, cuda, dtype, block_rows: int) -> None:
    for seed, (rows, cols) in enumerate([(1, 1), (1, 128), (3, 127), (17, 129), (128, 128), (130, 255), (257, 640),
                                         (2, 8192), (300, 1000)]):
        x = rand((rows, cols), seed, dtype)
        x[:, :: 5] *= 1e-3
        x[rows // 2] = 0
        q = wq.quantize_fp8(x, block_rows=block_rows)
        codes, scales = codes64(x, block_rows)
        same_codes(q.codes, codes)
        assert torch.equal(q.scales.double().cpu(), scales), (rows, cols)
        back = values64(q)
        for out in DTYPES:
            assert torch.equal(wq.dequantize_fp8(q, dtype=out), back.to(out)), (rows, cols, out)


@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_borders(wq, cuda, block_rows: int) -> None:
    """Scale borders, ties, the floor of the scale, zeros, and values that are not finite."""
    inf, nan = float("inf"), float("nan")
    rows = [
        [448.0, 1.0], [448.0001, 1.0], [449.0, 232.0], [896.0, 17.0], [2.0 ** -9, 2.0 ** -10], [0.0, -0.0],
        [448.0, 26.0, 25.0, 27.0, 2.0 ** -10, 3 * 2.0 ** -10, -(2.0 ** -10), 2.0 ** -9, 2.0 ** -6, 15 * 2.0 ** -10],
        [3.3e38, -1.0], [1e-38, 5e-39], [2.0 ** -149, 0.0], [2.0 ** -117 * 448, 2.0 ** -126, 2.0 ** -127],
        [inf, 448.0, 3.0], [nan, 1.0], [-inf, nan], [1.0, nan, -inf, 0.25], [2.0 ** -130, nan],
    ]
    x = torch.zeros(len(rows), 256)
    for i, r in enumerate(rows):
        x[i, : len(r)] = torch.tensor(r)
        x[i, 130] = 1.0 / (i + 1)
    if block_rows == 128:   # one row to a tile
        tall = torch.zeros(128 * len(rows), 256)
        tall[64::128] = x
        x = tall
    q = wq.quantize_fp8(x.to(cuda), block_rows=block_rows)
    codes, scales = codes64(x, block_rows)
    same_codes(q.codes, codes)
    assert torch.equal(q.scales.double().cpu(), scales)


def test_quantize_strides_and_leading_dims(wq, cuda) -> None:
    base = rand((40, 700), 3, torch.bfloat16)
    for x in (base[:, 3:300], base[::2, 8:264], base.t()[:256], base[:, ::2], base[5:6, 1:2], base[:, :1]):
        for br in (1, 128):
            q = wq.quantize_fp8(x, block_rows=br)
            codes, scales = codes64(x, br)
            same_codes(q.codes, codes)
            assert torch.equal(q.scales.double().cpu(), scales)
    x3 = base.reshape(4, 10, 700)
    assert torch.equal(wq.quantize_fp8(x3).codes.view(torch.uint8), wq.quantize_fp8(base).codes.view(torch.uint8))
    assert wq.quantize_fp8(base[0]).shape == (1, 700)
    assert wq.quantize_fp8(base[:0]).shape == (0, 700) and wq.quantize_fp8(base[:, :0]).shape == (40, 0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_column_sum(wq, cuda, dtype) -> None:
    """fp32 sums of m rows: each of at most m / 64 + 64 additions off by half a step of at most S = sum |x|."""
    for rows, cols in ((1, 1), (31, 63), (33, 200), (1000, 777), (0, 5)):
        x = rand((rows, cols), rows, dtype)
        for out in DTYPES:
            s = wq._kernels.column_sum(x, out)
            ref = x.double().sum(0)
            bound = torch.finfo(out).eps / 2 * ref.abs() + 2.0 ** -24 * (rows / 64 + 65) * x.double().abs().sum(0)
            assert bool(((s.double() - ref).abs() <= bound + LEAST[out]).all()), (rows, cols, out)
    wide = rand((64, 300), 5, dtype)
    assert torch.equal(wq._kernels.column_sum(wide[:, 1:200], torch.float32),
                       wq._kernels.column_sum(wide[:, 1:200].contiguous(), torch.float32))


# ---- the product --------------------------------------------------------------------

ROWS = (1, 2, 5, 8, 16, 17, 31, 33, 64, 65, 100, 128, 129, 200, 256, 257, 300, 513)


@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("rows", ROWS)
def test_product_rows(wq, cuda, rows: int, transpose: bool) -> None:
    """Every row count around the tiles' borders, ragged columns and inner dimension."""
    for K, N, dtype in ((256, 128, torch.float32), (300, 333, torch.bfloat16), (1031, 517, torch.float16)):
        a = wq.quantize_fp8(rand((rows, K), rows, torch.bfloat16))
        w = any_scales(rand((K, N) if transpose else (N, K), K, scale=0.02), wq)
        y = wq.fp8_gemm(a, w, transpose=transpose, out_dtype=dtype)
        w64 = values64(w)
        check_product(y, values64(a), w64 if transpose else w64.t(), what=f"{rows}x{N}x{K}")


@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("K,N", [(1, 1), (16, 7), (127, 129), (128, 128), (129, 2304), (768, 100), (4095, 640),
                                 (8192, 384), (2000, 5000)])
def test_product_sizes(wq, cuda, K: int, N: int, transpose: bool) -> None:
    for rows, dtype in ((1, torch.bfloat16), (37, torch.float32), (270, torch.float16), (1100, torch.bfloat16)):
        a = any_scales(rand((rows, K), rows, torch.float32), wq, 1)
        w = wq.quantize_fp8(rand((K, N) if transpose else (N, K), K, scale=0.02), block_rows=128)
        bias = rand((N,), 11, DTYPES[rows % 3])
        y = wq.fp8_gemm(a, w, transpose=transpose, out_dtype=dtype, bias=bias)
        w64 = values64(w)
        check_product(y, values64(a), w64 if transpose else w64.t(), bias, f"{rows}x{N}x{K}")


@pytest.mark.parametrize("rows", [1, 20, 50, 128, 200])
def test_product_long_runs(wq, cuda, rows: int) -> None:
    """Large enough that every block's pipeline wraps around many times, called back to back without waiting."""
    w = wq.quantize_fp8(rand((9000, 8000), 2, torch.bfloat16, 0.02), block_rows=128)
    x = rand((rows, 8000), rows, torch.bfloat16)
    prev = wq._kernels.set_fault_check(False)
    try:
        outs = [wq.fp8_gemm(x, w, out_dtype=torch.float32) for _ in range(6)]
    finally:
        wq._kernels.set_fault_check(prev)
    assert wq._kernels.fault_status() == 0
    check_product(outs[0], values64(wq.quantize_fp8(x)), values64(w).t())
    assert all(torch.equal(y, outs[0]) for y in outs)


@pytest.mark.parametrize("rows", [1, 4, 17, 64, 150, 600])
def test_product_of_a_tensor_equals_quantize_then_product(wq, cuda, rows: int) -> None:
    w = wq.quantize_fp8(rand((700, 1030), 2, scale=0.02), block_rows=128)
    for dtype in DTYPES:
        x = rand((rows, 1030), rows, dtype)
        y = wq.fp8_gemm(x, w)
        assert y.dtype == dtype
        check_product(y, values64(wq.quantize_fp8(x)), values64(w).t())
        x3 = x[:, None, :].expand(rows, 2, 1030)
        y3 = wq.fp8_gemm(x3, w)
        assert y3.shape == (rows, 2, 700)
        check_product(y3.reshape(-1, 700), values64(wq.quantize_fp8(x3)), values64(w).t())


def test_product_layouts(wq, cuda) -> None:
    """Codes at any stride and alignment, scales in either order, strided outputs whose gaps stay as they were."""
    a = wq.quantize_fp8(rand((70, 515), 1))
    w = wq.quantize_fp8(rand((260, 515), 2, scale=0.02), block_rows=128)
    y = wq.fp8_gemm(a, w, out_dtype=torch.float32)
    tight = wq.Fp8Blocks(a.codes.view(torch.uint8).contiguous().view(E4M3), a.scales.contiguous())
    odd = torch.zeros(260 * 515 + 3, dtype=torch.uint8, device=cuda)[3:].view(260, 515)
    odd.copy_(w.codes.view(torch.uint8))
    col = torch.zeros(515, 260, dtype=torch.uint8, device=cuda)
    col.copy_(w.codes.view(torch.uint8).t())
    for a2 in (a, tight):
        for codes in (w.codes, odd.view(E4M3), col.view(E4M3).t()):
            w2 = wq.Fp8Blocks(codes, w.scales.t().contiguous().t(), 128)
            assert torch.equal(wq.fp8_gemm(a2, w2, out_dtype=torch.float32), y)
    for rows in (70, 3, 400):
        ar = wq.quantize_fp8(rand((rows, 515), 4))
        want = wq.fp8_gemm(ar, w, out_dtype=torch.bfloat16)
        big = torch.full((rows + 2, 300), 7.0, dtype=torch.bfloat16, device=cuda)
        got = wq.fp8_gemm(ar, w, out=big[1:-1, 5:265])
        assert torch.equal(got, want) and got.data_ptr() == big[1:-1, 5:265].data_ptr()
        big[1:-1, 5:265] = 7.0
        assert bool((big == 7.0).all())
    with pytest.raises(ValueError, match="out must be"):
        wq.fp8_gemm(a, w, out=torch.empty(70, 259, device=cuda))
    with pytest.raises(ValueError, match="unit column stride"):
        wq.fp8_gemm(a, w, out=torch.empty(260, 70, device=cuda).t())


def test_product_empty_and_nan(wq, cuda) -> None:
    w = wq.quantize_fp8(rand((200, 384), 2), block_rows=128)
    assert wq.fp8_gemm(rand((0, 384), 1), w).shape == (0, 200)
    none = wq.quantize_fp8(torch.empty(200, 0, device=cuda), block_rows=128)
    bias = rand((200,), 1)
    for rows in (3, 300):
        y = wq.fp8_gemm(torch.empty(rows, 0, device=cuda), none, bias=bias)
        assert torch.equal(y, bias.expand(rows, 200))
        assert bool((wq.fp8_gemm(torch.empty(rows, 0, device=cuda), none) == 0).all())
    for rows in (5, 40, 300):
        x = rand((rows, 384), 3)
        y = wq.fp8_gemm(x, w)
        x2 = x.clone()
        x2[rows // 2, 200] = float("nan")
        x2[rows - 1, 10] = float("inf")
        y2 = wq.fp8_gemm(x2, w)
        bad = torch.zeros(rows, dtype=torch.bool, device=cuda)
        bad[[rows // 2, rows - 1]] = True
        assert bool(y2[bad].isnan().all()) and torch.equal(y2[~bad], y[~bad])
        x2[bad] = 0
        assert bool((wq.fp8_gemm(x2, w)[bad] == 0).all())


def test_product_scale_range(wq, cuda) -> None:
    """Scales far from 1 on both sides: products of scales down to 2^-140 and up to 2^120."""
    for rows in (4, 300):
        for sa, sw in ((2.0 ** -80, 2.0 ** -60), (2.0 ** 60, 2.0 ** 60), (2.0 ** 100, 2.0 ** -100)):
            a0, w0 = wq.quantize_fp8(rand((rows, 256), 1)), wq.quantize_fp8(rand((130, 256), 2), block_rows=128)
            a = wq.Fp8Blocks(a0.codes, a0.scales * sa)
            w = wq.Fp8Blocks(w0.codes, w0.scales * sw, 128)
            y = wq.fp8_gemm(a, w, out_dtype=torch.float32)
            ref, size = values64(a) @ values64(w).t(), values64(a).abs() @ values64(w).abs().t()
            # below 2^-126 each of the two blocks' terms may lose up to a step 2^-149 of its scale product
            bound = 2.0 ** -23 * (256 / 16 + 6) * size + 2.0 ** -149 * 448 * 448 * 128 * 2
            assert bool(((y.double() - ref).abs() <= bound).all()), (rows, sa, sw)


def test_offsets_past_32_bits(wq, cuda) -> None:
    """An operand of more than 2^31 codes: its last rows as by themselves, in the quantizer, the product and the
    weight gradient."""
    rows, cols = 263_000, 8200
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device=cuda)
    x[-300:] = rand((300, cols), 1, torch.bfloat16)
    q, last = wq.quantize_fp8(x), wq.quantize_fp8(x[-300:])
    assert rows * cols > 2 ** 31
    assert torch.equal(q.codes[-300:].view(torch.uint8), last.codes.view(torch.uint8))
    assert torch.equal(q.scales[-300:], last.scales) and bool((q.scales[:-300] == 1).all())
    del x
    w = wq.quantize_fp8(rand((100, cols), 2, torch.bfloat16, 0.02), block_rows=128)
    y = wq.fp8_gemm(q, w, out_dtype=torch.float32)
    check_product(y[-300:], values64(last), values64(w).t())
    assert bool((y[:-300] == 0).all())
    dy = torch.ones(rows, 9, dtype=torch.bfloat16, device=cuda)
    dw = wq.fp8_weight_grad(dy, q)
    check_product(dw, dy[-300:].double().t(), values64(last))


# ---- the weight gradient ---------------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 2, 15, 16, 63, 64, 65, 128, 200, 777])
def test_weight_grad(wq, cuda, rows: int, dtype) -> None:
    for N, K, out in ((1, 1, torch.float32), (128, 128, torch.float32), (130, 257, torch.bfloat16),
                      (333, 1030, torch.float16), (520, 300, torch.float32)):
        dy = rand((rows, N), rows + N, dtype, 1e-2)
        x = wq.quantize_fp8(rand((rows, K), K, torch.bfloat16))
        dw = wq.fp8_weight_grad(dy, x, out_dtype=out)
        check_product(dw, dy.double().t(), values64(x), what=f"{rows} {N}x{K}")


def test_weight_grad_long(wq, cuda) -> None:
    for dtype in DTYPES:
        dy = rand((5000, 256), 1, dtype, 1e-2)
        x = wq.quantize_fp8(rand((5000, 384), 2))
        dw = wq.fp8_weight_grad(dy, x)
        check_product(dw, dy.double().t(), values64(x))
        ref = dy.double().t() @ values64(x)
        # additions in fp32 over 5000 rows: well under a hundred steps of the result's size
        assert float((dw.double() - ref).norm() / ref.norm()) <= 100 * 2.0 ** -24


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", [(8192, 128, 128), (4100, 300, 520), (8192, 1, 1), (3001, 777, 130)])
def test_weight_grad_rows_in_parts(wq, cuda, M: int, N: int, K: int, dtype) -> None:
    """Many rows and few tiles: the rows are summed in parts by several pairs of SMs. Run twice, the same bits; a
    strided output that is added to; a replayed graph on new values."""
    dy = rand((M, N), 1, dtype, 1e-2)
    x = wq.quantize_fp8(rand((M, K), 2, torch.bfloat16))
    dw = wq.fp8_weight_grad(dy, x)
    check_product(dw, dy.double().t(), values64(x))
    for _ in range(20):
        assert torch.equal(wq.fp8_weight_grad(dy, x), dw)
    big = torch.full((N + 2, K + 9), 0.25, device=cuda)
    got = wq.fp8_weight_grad(dy, x, out=big[1:-1, 4:4 + K], accumulate=True)
    ref = dw.double() + 0.25
    assert bool(((got.double() - ref).abs() <= 2.0 ** -24 * ref.abs()).all())
    big[1:-1, 4:4 + K] = 0.25
    assert bool((big == 0.25).all())
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        again = wq.fp8_weight_grad(dy, x)
    for seed in (3, 4, 5):
        dy.copy_(rand((M, N), seed, dtype, 1e-2))
        graph.replay()
        assert torch.equal(again, wq.fp8_weight_grad(dy, x))


def test_weight_grad_layouts_and_accumulate(wq, cuda) -> None:
    base = rand((90, 400), 1, torch.bfloat16)
    x = wq.quantize_fp8(rand((90, 515), 2))
    for dy in (base[:, 3:300], base[:, ::2], base.reshape(9, 10, 400), base[:, :1].expand(90, 33)):
        d2 = dy.reshape(90, -1)
        check_product(wq.fp8_weight_grad(dy, x), d2.double().t(), values64(x))
    tight = wq.Fp8Blocks(x.codes.view(torch.uint8).contiguous().view(E4M3), x.scales.contiguous())
    assert torch.equal(wq.fp8_weight_grad(base, tight), wq.fp8_weight_grad(base, x))
    big = torch.full((402, 600), 0.5, device=cuda)
    dw = wq.fp8_weight_grad(base, x)
    got = wq.fp8_weight_grad(base, x, out=big[1:-1, 7:522], accumulate=True)
    ref = dw.double() + 0.5
    assert bool(((got.double() - ref).abs() <= 2.0 ** -24 * ref.abs()).all())
    big[1:-1, 7:522] = 0.5
    assert bool((big == 0.5).all())
    for dtype in DTYPES:
        g = rand((400, 515), 5, dtype)
        want = g.double() + base.double().t() @ values64(x)
        size = g.double().abs() + base.double().abs().t() @ values64(x).abs()
        wq.fp8_weight_grad(base, x, out=g, accumulate=True)
        bound = torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -23 * (90 / 16 + 90 / 128 + 5) * size
        assert bool(((g.double() - want).abs() <= bound).all())
    # no rows: nothing to add
    none = wq.quantize_fp8(torch.empty(0, 515, device=cuda))
    assert bool((wq.fp8_weight_grad(base[:0], none) == 0).all())
    keep = rand((400, 515), 6)
    assert torch.equal(wq.fp8_weight_grad(base[:0], none, out=keep.clone(), accumulate=True), keep)


def test_weight_grad_nan_stays_in_its_row_and_column(wq, cuda) -> None:
    xf, dy = rand((100, 256), 1), rand((100, 192), 2)
    xf[17, 33] = float("nan")
    dy[40, 50] = float("inf")
    dw = wq.fp8_weight_grad(dy, wq.quantize_fp8(xf))
    bad = torch.zeros(192, 256, dtype=torch.bool, device=cuda)
    bad[:, 33] = True
    assert bool(dw[:, 33].isnan().all())
    assert bool((~dw[50].isfinite()).any())
    bad[50] = True
    assert bool(dw[~bad].isfinite().all())


# ---- the layer ---------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_forward_and_gradients(wq, cuda, dtype) -> None:
    for lead, n_in, n_out in (((7,), 300, 130), ((3, 50), 256, 384), ((), 129, 65), ((2, 2, 100), 1000, 513)):
        x = rand((*lead, n_in), 1, dtype).requires_grad_()
        w = rand((n_out, n_in), 2, dtype, 0.02).requires_grad_()
        b = rand((n_out,), 3, dtype).requires_grad_()
        y = wq.fp8_linear(x, w, b)
        assert y.shape == (*lead, n_out) and y.dtype == dtype
        dy = rand(y.shape, 4, dtype, 1e-2)
        dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
        assert (dx.shape, dw.shape, db.shape) == (x.shape, w.shape, b.shape)
        assert dx.dtype == dw.dtype == db.dtype == dtype
        x64 = values64(wq.quantize_fp8(x))
        w64 = values64(wq.quantize_fp8(w, block_rows=128))
        d2 = dy.reshape(-1, n_out)
        check_product(y.reshape(-1, n_out), x64, w64.t(), b)
        check_product(dx.reshape(-1, n_in), values64(wq.quantize_fp8(d2)), w64)
        check_product(dw, d2.double().t(), x64)
        ones = torch.ones(1, d2.shape[0], dtype=torch.float64, device=cuda)
        check_product(db[None], ones, d2.double())


def test_linear_gradients_against_differences(wq, cuda) -> None:
    """The gradients are those of L = <dy, x8 w8^T + b> with respect to the 8-bit operands (the quantizers pass
    gradients through): central differences of L in fp64, exact up to fp64 since L is linear in each argument.
    dx uses dy in 8 bits, so dy here is made of e4m3 values and enters unchanged."""
    dy = wq.dequantize_fp8(wq.quantize_fp8(rand((20, 70), 4)))
    x = rand((20, 150), 1).requires_grad_()
    w = rand((70, 150), 2).requires_grad_()
    b = rand((70,), 3).requires_grad_()
    grads = torch.autograd.grad(wq.fp8_linear(x, w, b), (x, w, b), dy)
    x64, w64 = values64(wq.quantize_fp8(x)), values64(wq.quantize_fp8(w, block_rows=128))

    def loss(xa, wa, ba):  # type: ignore[no-untyped-def]
        return float(((xa @ wa.t() + ba) * dy.double()).sum())

    args = [x64, w64, b.detach().double()]
    g = torch.Generator().manual_seed(9)
    for i, grad in enumerate(grads):
        for _ in range(5):
            at = tuple(int(torch.randint(n, (1,), generator=g)) for n in args[i].shape)
            up, down = args[i].clone(), args[i].clone()
            up[at] += 0.5
            down[at] -= 0.5
            diff = loss(*[up if j == i else v for j, v in enumerate(args)]) - \
                loss(*[down if j == i else v for j, v in enumerate(args)])
            # the loss sums 20 * 70 terms in fp64; fp32 sums of at most 70 terms in the gradient
            assert abs(float(grad[at]) - diff) <= 2e-5 * (1 + abs(diff)), (i, at)


def test_linear_needs_only_what_is_asked(wq, cuda) -> None:
    x, w, b = rand((40, 256), 1), rand((128, 256), 2), rand((128,), 3)
    for mask in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 0), (0, 0, 0)):
        leaves = [t.clone().requires_grad_(bool(m)) for t, m in zip((x, w, b), mask)]
        y = wq.fp8_linear(*leaves)
        if not any(mask):
            assert not y.requires_grad
            continue
        y.sum().backward()
        assert [t.grad is not None for t in leaves] == [bool(m) for m in mask]
    y = wq.fp8_linear(x, w.requires_grad_())
    y.backward(torch.ones_like(y))
    assert w.grad is not None


def test_checkpoint_is_one_byte_per_value(wq, cuda) -> None:
    """What the graph keeps of a bf16 input: its codes and scales, half the input's bytes plus one fp32 per 128."""
    w = rand((256, 2048), 2, torch.bfloat16).requires_grad_()
    seen = []

    def pack(t: torch.Tensor) -> torch.Tensor:
        seen.append(t.numel() * t.element_size())
        return t

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        y = wq.fp8_linear(rand((4096, 2048), 1, torch.bfloat16), w)
    assert sorted(seen) == [4096 * 16 * 4, 4096 * 2048]
    y.backward(torch.ones_like(y))


class _Net(torch.nn.Module):
    def __init__(self) -> None:
        super().__init__()
        self.up = torch.nn.Linear(200, 333)
        self.down = torch.nn.Linear(333, 130, bias=False)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return self.down(torch.relu(self.up(x)))


def test_model_of_layers_together(wq, cuda) -> None:
    """A model swapped layer by layer: forward, backward, a gradient-accumulating second step, then frozen serving
    of one token, each against the same computation from the operands in fp64."""
    torch.manual_seed(0)
    net = _Net().to(cuda)
    names = dict(net.named_parameters())
    model = wq.fp8_model(net)
    assert model is net and all(dict(net.named_parameters())[n] is p for n, p in names.items())
    assert isinstance(net.up, wq.Fp8Linear) and isinstance(net.down, wq.Fp8Linear)
    x = rand((50, 200), 1)
    y = net(x)
    dy = rand(y.shape, 2)
    y.backward(dy)
    w1, w2 = (values64(wq.quantize_fp8(m.weight, block_rows=128)) for m in (net.up, net.down))
    h = wq.fp8_linear(x, net.up.weight, net.up.bias).detach()
    check_product(h, values64(wq.quantize_fp8(x)), w1.t(), net.up.bias)
    r8 = values64(wq.quantize_fp8(torch.relu(h)))
    check_product(y, r8, w2.t())
    check_product(net.down.weight.grad, dy.double().t(), r8)
    dr = wq.fp8_gemm(dy, wq.quantize_fp8(net.down.weight, block_rows=128), transpose=True)
    check_product(dr, values64(wq.quantize_fp8(dy)), w2)
    dh = dr * (h > 0)
    check_product(net.up.weight.grad, dh.double().t(), values64(wq.quantize_fp8(x)))
    first = net.up.weight.grad.clone()
    net(x).backward(dy)
    assert torch.allclose(net.up.weight.grad, 2 * first, rtol=2.0 ** -23, atol=0)
    with torch.no_grad():
        want = net(x[:1])
        for m in (net.up, net.down):
            m.freeze()
        assert torch.equal(net(x[:1]), want)
        net.half()
        assert net.up.codes.dtype == E4M3 and net.up.scales.dtype == torch.float32
        assert net(x[:1].half()).dtype == torch.float16
    with pytest.raises(RuntimeError, match="no backward pass"):
        net.up(x.half().requires_grad_())


# ---- streams, graphs, repetition ------------------------------------------------------------


def test_same_bits_on_every_call_and_on_another_stream(wq, cuda) -> None:
    w = wq.quantize_fp8(rand((1000, 2000), 2, scale=0.02), block_rows=128)
    side = torch.cuda.Stream()
    for rows in (1, 20, 200, 1500):
        x = rand((rows, 2000), rows, torch.bfloat16)
        dy = rand((rows, 1000), rows + 1, torch.bfloat16)
        q = wq.quantize_fp8(x)
        y, dw = wq.fp8_gemm(x, w), wq.fp8_weight_grad(dy, q)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            outs = [(wq.fp8_gemm(x, w), wq.fp8_weight_grad(dy, q)) for _ in range(3)]
        torch.cuda.current_stream().wait_stream(side)
        for y2, dw2 in outs:
            assert torch.equal(y, y2) and torch.equal(dw, dw2)


def test_two_calls_at_once(wq, cuda) -> None:
    """Two streams run the same kinds of call on different operands, many times over: each has its own workspace."""
    jobs = []
    for seed, rows in ((1, 24), (2, 300)):
        x = rand((rows, 1500), seed, torch.bfloat16)
        w = wq.quantize_fp8(rand((900, 1500), seed + 5, scale=0.02), block_rows=128)
        dy = rand((rows, 900), seed + 9, torch.bfloat16)
        q = wq.quantize_fp8(x)
        jobs.append((x, w, dy, q, wq.fp8_gemm(x, w), wq.fp8_weight_grad(dy, q)))
    torch.cuda.synchronize()
    prev = wq._kernels.set_fault_check(False)
    try:
        streams = [torch.cuda.Stream() for _ in jobs]
        outs = [[], []]
        for _ in range(20):
            for i, (s, (x, w, dy, q, _, _)) in enumerate(zip(streams, jobs)):
                with torch.cuda.stream(s):
                    outs[i].append((wq.fp8_gemm(x, w), wq.fp8_weight_grad(dy, q)))
        torch.cuda.synchronize()
    finally:
        wq._kernels.set_fault_check(prev)
    assert wq._kernels.fault_status() == 0
    for got, job in zip(outs, jobs):
        for y, dw in got:
            assert torch.equal(y, job[4]) and torch.equal(dw, job[5])


def test_captured_and_replayed(wq, cuda) -> None:
    w = wq.quantize_fp8(rand((700, 1024), 2, scale=0.02), block_rows=128)
    for rows in (1, 30, 400):
        x = rand((rows, 1024), 1, torch.bfloat16)
        dy = rand((rows, 700), 2, torch.bfloat16)

        def step():  # type: ignore[no-untyped-def]
            q = wq.quantize_fp8(x)
            return wq.fp8_gemm(q, w), wq.fp8_gemm(x, w), wq.fp8_gemm(dy, w, transpose=True), wq.fp8_weight_grad(dy, q)

        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            step()
        torch.cuda.synchronize()
        graphs, outs = [], []
        for _ in range(2):   # two graphs over the same inputs, replayed in turn
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                outs.append(step())
            graphs.append(g)
        for seed in (5, 6):
            x.copy_(rand(x.shape, seed, x.dtype))
            dy.copy_(rand(dy.shape, seed + 1, dy.dtype))
            want = step()
            for g in graphs:
                g.replay()
            torch.cuda.synchronize()
            for out in outs:
                for a, b in zip(out, want):
                    assert torch.equal(a, b)
    assert wq._kernels.fault_status() == 0


def test_backward_in_a_graph(wq, cuda) -> None:
    """A whole step captured; no eager graph of the same leaves is alive meanwhile."""
    x = rand((96, 512), 1, torch.bfloat16).requires_grad_()
    w = rand((256, 512), 2, torch.bfloat16, 0.02).requires_grad_()
    dy = rand((96, 256), 3, torch.bfloat16)
    want = torch.autograd.grad(wq.fp8_linear(x, w), (x, w), dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(wq.fp8_linear(x, w), (x, w), dy)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = torch.autograd.grad(wq.fp8_linear(x, w), (x, w), dy)
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
