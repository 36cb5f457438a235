"""The 8-bit floating-point layer in a model: conversion, freezing, devices, mixed precision, memory."""

from __future__ import annotations

import copy

import pytest
import torch
import torch.utils.checkpoint
from torch import nn

from test_fp8_gpu import DTYPES, E4M3, check_product, rand, values64

pytestmark = pytest.mark.gpu


def net(cuda) -> nn.Module:  # type: ignore[no-untyped-def]
    torch.manual_seed(0)
    return nn.Sequential(nn.Linear(200, 333), nn.ReLU(), nn.Linear(333, 130)).to(cuda)


# ---- freezing ------------------------------------------------------------------------


def test_freezing_a_converted_model(wq, cuda) -> None:
    """Convert, train a step, convert again with freeze: every layer keeps its 8-bit tiles alone and answers as it
    did."""
    model = wq.fp8_model(net(cuda))
    x = rand((20, 200), 1)
    model(x).sum().backward()
    with torch.no_grad():
        want = model(x)
        assert wq.fp8_model(model, freeze=True) is model
        layers = [m for m in model.modules() if isinstance(m, wq.Fp8Linear)]
        assert len(layers) == 2 and all(m.weight is None and m.codes is not None for m in layers)
        assert torch.equal(model(x), want)
    one = wq.Fp8Linear(rand((64, 200), 2))
    assert wq.fp8_model(one, freeze=True) is one and one.weight is None
    mixed = nn.Sequential(wq.Fp8Linear(rand((64, 200), 2)), nn.Linear(64, 32, device=cuda))
    wq.fp8_model(mixed, freeze=True)
    assert all(isinstance(m, wq.Fp8Linear) and m.weight is None for m in mixed)


# ---- shared modules ------------------------------------------------------------------


def test_a_module_under_two_names(wq, cuda) -> None:
    """A layer that the model holds twice is replaced in both places, by one layer."""
    model = nn.Module()
    model.first = nn.Linear(64, 64, device=cuda)
    model.inner = nn.Sequential(nn.ReLU(), model.first)
    wq.fp8_model(model)
    assert isinstance(model.first, wq.Fp8Linear) and model.inner[1] is model.first


# ---- a frozen layer's rows -------------------------------------------------------------


@pytest.mark.parametrize("move", ["device", "copy", "assign", "operand"])
def test_moved_codes_keep_rows_that_the_products_read(wq, cuda, move: str) -> None:
    """A width that is no multiple of 16: after a way over the host, or a load that takes the state's tensors as they
    are, the codes lie in padded rows again, and a product allocates no copy of them."""
    layer = wq.Fp8Linear(rand((4096, 1001), 1, torch.bfloat16, 0.02)).freeze()
    x = rand((4, 1001), 2, torch.bfloat16)
    want = layer(x)
    if move == "device":
        layer = layer.cpu().to(cuda)
    elif move == "copy":
        layer = copy.deepcopy(layer)
    elif move == "assign":
        state = {k: v.contiguous() if v.dtype != E4M3 else v.view(torch.uint8).contiguous().view(E4M3)
                 for k, v in layer.state_dict().items()}
        assert state["codes"].stride(0) == 1001
        layer.load_state_dict(state, assign=True)
    else:
        q = layer.quantized_weight().to("cpu").to(cuda)
        assert torch.equal(wq.fp8_gemm(x, q), want)
        layer.codes = q.codes
    assert layer.codes.shape == (4096, 1001) and layer.codes.stride(0) % 16 == 0
    layer(x)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    y = layer(x)
    assert torch.equal(y, want)
    assert torch.cuda.max_memory_allocated() - before < 4096 * 1001


# ---- mixed precision ---------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_autocast(wq, cuda, dtype) -> None:
    """Under autocast the layer takes and gives autocast's type, as nn.Linear does, and its fp32 weight is quantized
    as it is; gradients come in their parameters' types."""
    plain = net(cuda)
    model = wq.fp8_model(copy.deepcopy(plain))
    x = rand((20, 200), 1)
    with torch.autocast("cuda", dtype=dtype):
        assert plain(x).dtype == dtype
        y = model(x)
        assert y.dtype == dtype
    w = model[0].weight
    h = wq.fp8_linear(x.to(dtype), w, model[0].bias)
    with torch.autocast("cuda", dtype=dtype):
        assert torch.equal(wq.fp8_linear(x, w, model[0].bias), h)
        assert wq.fp8_linear(x.double().float(), w).dtype == dtype
    check_product(h.detach(), values64(wq.quantize_fp8(x.to(dtype))), values64(wq.quantize_fp8(w, block_rows=128)).t(),
                  model[0].bias)
    xg = x.clone().requires_grad_()
    with torch.autocast("cuda", dtype=dtype):
        y = wq.fp8_linear(xg, w)
    dy = rand(y.shape, 3, dtype, 1e-2)
    dx, dw = torch.autograd.grad(y, (xg, w), dy)
    assert dx.dtype == dw.dtype == torch.float32
    check_product(dw, dy.double().t(), values64(wq.quantize_fp8(x.to(dtype))))
    assert torch.equal(dx, wq.fp8_gemm(dy, wq.quantize_fp8(w, block_rows=128), transpose=True).float())
    with torch.no_grad(), torch.autocast("cuda", dtype=dtype):
        want = model(x)
        wq.fp8_model(model, freeze=True)
        assert torch.equal(model(x), want)
    with torch.autocast("cuda", dtype=dtype, enabled=False):
        assert wq.fp8_linear(x, w).dtype == torch.float32


def test_func_transforms_are_refused(wq, cuda) -> None:
    x, w = rand((4, 64), 1), rand((32, 64), 2)
    with pytest.raises(RuntimeError, match="functorch"):
        torch.func.grad(lambda v: wq.fp8_linear(x, v).sum())(w)


# ---- memory --------------------------------------------------------------------------------


def test_weight_grad_of_bf16_keeps_no_copy_of_dy(wq, cuda) -> None:
    """dy in bf16 whose rows TMA reads is read where it is: beside dw the call holds no more than the parts' sums
    (here none); other dy is copied, fp16 and fp32 as two and three bf16 terms."""
    M, N, K = 4096, 4096, 512
    x = wq.quantize_fp8(rand((M, K), 1, torch.bfloat16))
    dw = torch.empty(N, K, device=cuda)

    def held(dy: torch.Tensor) -> int:
        wq.fp8_weight_grad(dy, x, out=dw)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        wq.fp8_weight_grad(dy, x, out=dw)
        return torch.cuda.max_memory_allocated() - before

    assert wq._kernels.fp8_weight_grad_plan(M, N, K, torch.bfloat16)[1] == 1
    dy = rand((M, N), 2, torch.bfloat16, 1e-2)
    assert held(dy) == 0
    check_product(dw, dy.double().t(), values64(x))
    wide = torch.zeros(M, N + 3, dtype=torch.bfloat16, device=cuda)
    wide[:, 3:] = dy
    assert held(wide[:, 3:]) == M * N * 2     # rows that TMA cannot read
    check_product(dw, dy.double().t(), values64(x))
    for dtype, terms in ((torch.float16, 2), (torch.float32, 3)):
        d2 = rand((M, N), 2, dtype, 1e-2)
        assert held(d2) == M * N * 2 * terms
        check_product(dw, d2.double().t(), values64(x))


@pytest.mark.parametrize("M,N,K", [(8192, 128, 128), (4100, 304, 520)])
def test_weight_grad_in_parts_reads_bf16_where_it_is(wq, cuda, M: int, N: int, K: int) -> None:
    """The counters and sums of parts lie where the terms would begin: right with aligned and other rows, in turn."""
    assert wq._kernels.fp8_weight_grad_plan(M, N, K, torch.bfloat16)[1] > 1
    x = wq.quantize_fp8(rand((M, K), 2, torch.bfloat16))
    dy = rand((M, N), 1, torch.bfloat16, 1e-2)
    odd = torch.zeros(M, N + 1, dtype=torch.bfloat16, device=cuda)
    odd[:, 1:] = dy
    want = wq.fp8_weight_grad(dy, x)
    check_product(want, dy.double().t(), values64(x))
    for _ in range(5):
        assert torch.equal(wq.fp8_weight_grad(odd[:, 1:], x), want)
        assert torch.equal(wq.fp8_weight_grad(dy, x), want)


# ---- one rounding -----------------------------------------------------------------------------


def test_dequantize_rounds_once(wq, cuda) -> None:
    """code * scale for scales that are no powers of two, rounded once to the type: for products that lie just beside
    the middle of two 16-bit values a rounding to fp32 before would fall on the middle itself."""
    codes = torch.arange(256, dtype=torch.uint8, device=cuda).view(E4M3)
    c64 = codes.double()
    fine = c64.isfinite() & (c64 != 0)
    g = torch.Generator(device="cuda").manual_seed(1)
    scales = torch.exp2(torch.rand(4096, generator=g, device=cuda) * 20 - 10)
    # scales next to those at which a code's value is the middle of two bf16 or fp16 numbers
    odd = (torch.arange(1024, device=cuda).double() * 2 + 1)
    near = []
    for bits in (8, 11):
        mid = 1 + odd[: 2 ** (bits - 1)] * 2.0 ** -bits
        for c in (1.125, 1.25, 1.375, 1.5, 1.75):
            s = (mid / c).float()
            near += [s, torch.nextafter(s, torch.full_like(s, 9.0)), torch.nextafter(s, torch.zeros_like(s))]
    scales = torch.cat([scales, *near])
    q = wq.Fp8Blocks(codes.view(torch.uint8).expand(scales.numel(), 256).contiguous().view(E4M3), scales[:, None].expand(-1, 2).contiguous())
    exact = c64 * scales.double()[:, None]     # 4 and 24 bits: exact in 64
    for dtype in DTYPES:
        got = wq.dequantize_fp8(q, dtype=dtype)[:, fine].double()
        want = exact[:, fine]
        # from half a step past the largest number, (2 - eps) 2^e, the nearest is infinity
        eps = torch.finfo(dtype).eps
        over = want.abs() >= torch.finfo(dtype).max * (1 + eps / 2 / (2 - eps))
        assert torch.equal(got.isinf(), over)
        got, want = got[~over], want[~over]
        # nearest: no neighbour of the result lies closer to the exact value (a tie may go either way here)
        up = torch.nextafter(got.to(dtype), torch.full_like(got, float("inf")).to(dtype)).double()
        down = torch.nextafter(got.to(dtype), torch.full_like(got, -float("inf")).to(dtype)).double()
        err = (got - want).abs()
        assert bool((err <= (up - want).abs()).all()) and bool((err <= (down - want).abs()).all()), dtype


# ---- sides of no length, scales of no stride, recomputation ---------------------------------------


def test_layer_without_rows_or_sides(wq, cuda) -> None:
    """No rows: gradients of zeros. No outputs, no inputs: what is left of the sums."""
    w, b = rand((64, 96), 1).requires_grad_(), rand((64,), 2).requires_grad_()
    for lead in ((0,), (3, 0)):
        x = torch.empty(*lead, 96, device=cuda, requires_grad=True)
        y = wq.fp8_linear(x, w, b)
        assert y.shape == (*lead, 64)
        dx, dw, db = torch.autograd.grad(y.sum(), (x, w, b))
        assert dx.shape == x.shape and bool((dw == 0).all()) and bool((db == 0).all())
    x, none = rand((5, 96), 3).requires_grad_(), torch.empty(0, 96, device=cuda, requires_grad=True)
    y = wq.fp8_linear(x, none)
    dx, dw = torch.autograd.grad(y.sum(), (x, none))
    assert y.shape == (5, 0) and bool((dx == 0).all()) and dw.shape == (0, 96)
    x, none = torch.empty(5, 0, device=cuda, requires_grad=True), torch.empty(64, 0, device=cuda, requires_grad=True)
    y = wq.fp8_linear(x, none, b)
    dx, dw, db = torch.autograd.grad(y.sum(), (x, none, b))
    assert torch.equal(y, b.expand(5, 64)) and dx.shape == (5, 0) and dw.shape == (64, 0) and bool((db == 5).all())


def test_one_scale_for_all_blocks(wq, cuda) -> None:
    """Scales without strides: one value stands for every block."""
    one = torch.full((1, 1), 0.375, device=cuda)
    q, w8 = wq.quantize_fp8(rand((40, 700), 1)), wq.quantize_fp8(rand((260, 700), 2), block_rows=128)
    a, w = wq.Fp8Blocks(q.codes, one.expand(40, 6)), wq.Fp8Blocks(w8.codes, one.expand(3, 6), 128)
    assert torch.equal(wq.dequantize_fp8(a).double(), q.codes.double() * 0.375)
    check_product(wq.fp8_gemm(a, w, out_dtype=torch.float32), values64(a), values64(w).t())
    dy = rand((40, 33), 3)
    # 0.375 has two bits: code * scale is exact in bf16
    check_product(wq.fp8_weight_grad(dy, a), dy.double().t(), values64(a))


def test_recomputed_forward(wq, cuda) -> None:
    """Activation checkpointing runs the forward again: the same gradients, bit for bit."""
    w, x = rand((64, 96), 1).requires_grad_(), rand((7, 96), 2).requires_grad_()

    def part(v: torch.Tensor) -> torch.Tensor:
        return torch.relu(wq.fp8_linear(v, w))

    want = torch.autograd.grad(part(x).square().sum(), (x, w))
    y = torch.utils.checkpoint.checkpoint(part, x, use_reentrant=False)
    got = torch.autograd.grad(y.square().sum(), (x, w))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
