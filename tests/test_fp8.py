"""Blocks of 8-bit floating point without a GPU: operand checks, refusals of the
C ABI and of the Python entry points, all before any CUDA call."""

from __future__ import annotations

import ctypes

import pytest
import torch

E4M3 = torch.float8_e4m3fn
P = ctypes.c_void_p(256)   # a non-null pointer that no refused call follows


def test_operand_checks(wq) -> None:
    codes = torch.zeros(130, 300, dtype=torch.uint8).view(E4M3)
    assert wq.Fp8Blocks(codes, torch.ones(130, 3)).shape == (130, 300)
    assert wq.Fp8Blocks(codes, torch.ones(2, 3), 128).block_rows == 128
    with pytest.raises(ValueError, match="block_rows must be 1 or 128"):
        wq.Fp8Blocks(codes, torch.ones(130, 3), 64)
    with pytest.raises(ValueError, match="codes must be a float8_e4m3fn matrix"):
        wq.Fp8Blocks(codes.view(torch.uint8), torch.ones(130, 3))
    with pytest.raises(ValueError, match="codes must be a float8_e4m3fn matrix"):
        wq.Fp8Blocks(codes[0], torch.ones(1, 3))
    for bad in (torch.ones(130, 2), torch.ones(2, 3), torch.ones(130, 3, dtype=torch.float64), torch.ones(390)):
        with pytest.raises(ValueError, match="scales must be float32"):
            wq.Fp8Blocks(codes, bad)
    with pytest.raises(ValueError, match="scales must be float32"):
        wq.Fp8Blocks(codes, torch.ones(130, 3), 128)


def test_python_refusals(wq) -> None:
    a = wq.Fp8Blocks(torch.zeros(4, 256, dtype=torch.uint8).view(E4M3), torch.ones(4, 2))
    w = wq.Fp8Blocks(torch.zeros(8, 256, dtype=torch.uint8).view(E4M3), torch.ones(1, 2), 128)
    x = torch.zeros(4, 256)
    with pytest.raises(ValueError, match="block_rows must be 1 or 128"):
        wq.quantize_fp8(x, block_rows=2)
    with pytest.raises(ValueError, match="x must be float32, float16 or bfloat16"):
        wq.quantize_fp8(x.double())
    with pytest.raises(ValueError, match="must be CUDA tensors"):
        wq.quantize_fp8(x)
    with pytest.raises(ValueError, match="must be CUDA tensors"):
        wq.dequantize_fp8(a)
    with pytest.raises(ValueError, match="dtype must be float32, float16 or bfloat16"):
        wq.dequantize_fp8(a, dtype=torch.int32)
    with pytest.raises(ValueError, match="weight must have one scale per 128 x 128 tile"):
        wq.fp8_gemm(a, a)
    with pytest.raises(ValueError, match="a must have one scale per 128 values of a row"):
        wq.fp8_gemm(w, w)
    with pytest.raises(ValueError, match="trailing dim 255, weight expects 256"):
        wq.fp8_gemm(x[:, :255], w)
    with pytest.raises(ValueError, match="trailing dim 256, weight expects 8"):
        wq.fp8_gemm(x, w, transpose=True)
    with pytest.raises(ValueError, match="must be CUDA tensors"):
        wq.fp8_gemm(x, w)
    with pytest.raises(ValueError, match="must be CUDA tensors"):
        wq.fp8_gemm(a, w)
    with pytest.raises(ValueError, match="out_dtype must be float32"):
        wq.fp8_gemm(a, w, out_dtype=torch.float64)
    with pytest.raises(ValueError, match="block_rows=1"):
        wq.fp8_weight_grad(x, w)
    with pytest.raises(ValueError, match="accumulate adds to out, which is missing"):
        wq.fp8_weight_grad(x, a, accumulate=True)
    with pytest.raises(ValueError, match="must be CUDA tensors"):
        wq.fp8_weight_grad(x, a)
    with pytest.raises(ValueError, match="trailing dim 256, weight expects 8"):
        wq.fp8_linear(x, torch.zeros(16, 8))
    with pytest.raises(ValueError, match="x must be a CUDA tensor"):
        wq.fp8_linear(x, torch.zeros(16, 256))
    with pytest.raises(ValueError, match="bias does not match out_features"):
        wq.fp8_linear(x, torch.zeros(16, 256), torch.zeros(15))
    with pytest.raises(ValueError, match=r"weight must have shape \[out, in\]"):
        wq.Fp8Linear(torch.zeros(16))
    with pytest.raises(ValueError, match="bias does not match out_features"):
        wq.Fp8Linear(torch.zeros(16, 8), torch.zeros(8))
    with pytest.raises(ValueError, match="expected in_features=8, got 9"):
        wq.Fp8Linear(torch.zeros(16, 8))(torch.zeros(2, 9))
    with pytest.raises(RuntimeError, match="expects CUDA parameters"):
        wq.fp8_model(torch.nn.Linear(4, 4))


def test_layer_shares_the_linear_parameters(wq) -> None:
    lin = torch.nn.Linear(8, 16)
    layer = wq.Fp8Linear.from_linear(lin)
    assert layer.weight is lin.weight and layer.bias is lin.bias
    assert {n for n, _ in layer.named_parameters()} == {"weight", "bias"}
    assert (layer.in_features, layer.out_features) == (8, 16)


def test_quantize_c_refusals(wq) -> None:
    lib = wq._kernels.library()

    def q(x=P, t=2, rows=4, cols=256, ldx=256, br=1, codes=P, ld=256, sc=P, sr=1, s_c=4):  # type: ignore[no-untyped-def]
        return lib.wq_fp8_quantize(x, t, rows, cols, ldx, br, codes, ld, sc, sr, s_c, None)

    assert q(t=3) == 23 and q(t=-1) == 23
    assert q(br=64) == 24 and q(br=0) == 24
    assert q(rows=-1) == 5 and q(cols=-1) == 5
    assert q(ldx=255) == 25 and q(ld=255) == 25 and q(sr=-1) == 25 and q(s_c=-1) == 25
    assert q(rows=1 << 31) == 13 and q(cols=1 << 23, ldx=1 << 23, ld=1 << 23) == 13
    assert q(x=None) == 11 and q(codes=None) == 11 and q(sc=None) == 11
    assert q(rows=0, x=None) == 0 and q(cols=0, x=None) == 0
    d = lib.wq_fp8_dequantize
    assert d(P, 4, 256, 256, 1, P, 1, 4, P, 9, 256, None) == 23
    assert d(P, 4, 256, 256, 3, P, 1, 4, P, 0, 256, None) == 24
    assert d(P, 4, 256, 256, 1, P, 1, 4, P, 0, 255, None) == 25
    assert d(None, 4, 256, 256, 1, P, 1, 4, P, 0, 256, None) == 11
    assert d(None, 0, 256, 256, 1, P, 1, 4, P, 0, 256, None) == 0
    c = lib.wq_column_sum
    assert c(P, 5, 4, 8, 8, P, 0, None) == 23 and c(P, 0, 4, 8, 8, P, 5, None) == 23
    assert c(P, 0, -4, 8, 8, P, 0, None) == 5 and c(P, 0, 4, 8, 7, P, 0, None) == 25
    assert c(None, 0, 4, 8, 8, P, 0, None) == 11 and c(None, 0, 4, 0, 0, None, 0, None) == 0


def test_product_c_refusals(wq) -> None:
    lib = wq._kernels.library()

    def g(a=P, M=4, K=256, lda=256, sa=P, sr=1, sc=4, w=P, wr=8, wc=256, ldw=256, sw=P, wsr=2, wsc=1, tr=0, bias=None,
          bt=0, out=P, ot=2, ldo=8, ws=P, nws=1 << 40):  # type: ignore[no-untyped-def]
        return lib.wq_fp8_gemm(a, M, K, lda, sa, sr, sc, w, wr, wc, ldw, sw, wsr, wsc, tr, bias, bt, out, ot, ldo, ws,
                               nws, None)

    assert g(ot=3) == 23 and g(bias=P, bt=7) == 23
    assert g(M=-1) == 5 and g(wr=-1) == 5
    assert g(wc=240) == 27 and g(tr=1) == 27
    assert g(ldw=255) == 25 and g(lda=255) == 25 and g(sr=-1) == 25 and g(wsc=-1) == 25
    assert g(ldo=7) == 20
    assert g(ldw=264) == 26 and g(lda=264) == 26 and g(w=ctypes.c_void_p(8)) == 26 and g(a=ctypes.c_void_p(8)) == 26
    assert g(M=1 << 23) == 13
    assert g(out=None) == 11 and g(a=None) == 11 and g(sw=None) == 11
    assert g(M=0, a=None, out=None) == 0 and g(wr=0, out=None) == 0

    def lin(x=P, t=2, M=4, K=256, ldx=256, nws=1 << 40, ws=P):  # type: ignore[no-untyped-def]
        return lib.wq_fp8_linear(x, t, M, K, ldx, P, 8, 256, 256, P, 2, 1, 0, None, 0, P, 2, 8, ws, nws, None)

    assert lin(t=4) == 23 and lin(K=255) == 27 and lin(ldx=255) == 25 and lin(x=None) == 11
    assert lin(nws=0) == 12 and lin(ws=None) == 12 and lin(ws=ctypes.c_void_p(16)) == 12
    assert lin(M=0, x=None, ws=None, nws=0) == 0
    assert lib.wq_fp8_linear_workspace_bytes(4, 8, 256) >= 4 * 256 + 4 * 2 * 4
    assert lib.wq_fp8_linear_workspace_bytes(0, 8, 256) == 0

    def wg(dy=P, dt=2, M=4, N=8, ldy=8, codes=P, K=256, ld=256, sc=P, sr=1, s_c=4, dw=P, wt=0, ldw=256, nws=1 << 40):  # type: ignore[no-untyped-def]
        return lib.wq_fp8_weight_grad(dy, dt, M, N, ldy, codes, K, ld, sc, sr, s_c, dw, wt, ldw, 0, P, nws, None)

    assert wg(dt=3) == 23 and wg(wt=3) == 23 and wg(M=-1) == 5
    assert wg(ldy=7) == 25 and wg(ld=240) == 25 and wg(s_c=-1) == 25 and wg(ldw=255) == 20
    assert wg(ld=264) == 26 and wg(codes=ctypes.c_void_p(4)) == 26
    assert wg(M=1 << 23) == 13
    assert wg(dw=None) == 11 and wg(dy=None) == 11 and wg(sc=None) == 11
    assert wg(N=0, dw=None) == 0 and wg(K=0, dw=None) == 0


def test_workspace_alignment_c_refusals(wq) -> None:
    """Workspaces that are needed and not 256-byte aligned, or too small, are refused by each entry point."""
    lib = wq._kernels.library()
    need = lib.wq_fp8_gemm_workspace_bytes(1, 4096, 8192)
    assert need > 0

    def g(ws, nws=need):  # type: ignore[no-untyped-def]
        return lib.wq_fp8_gemm(P, 1, 8192, 8192, P, 64, 1, P, 4096, 8192, 8192, P, 64, 1, 0, None, 0, P, 2, 4096, ws,
                               nws, None)

    assert g(ctypes.c_void_p(256 + 16)) == 12 and g(None) == 12 and g(P, need - 1) == 12
    need_w = lib.wq_fp8_weight_grad_workspace_bytes(4, 8, 256, 0)
    assert need_w > 0

    def wg(ws, nws=need_w):  # type: ignore[no-untyped-def]
        return lib.wq_fp8_weight_grad(P, 0, 4, 8, 8, P, 256, 256, P, 2, 1, P, 0, 256, 0, ws, nws, None)

    assert wg(ctypes.c_void_p(256 + 128)) == 12 and wg(None) == 12 and wg(P, need_w - 1) == 12


def test_status_messages(wq) -> None:
    msg = wq._kernels.status_message
    assert msg(23) == "element type must be fp32, fp16 or bf16"
    assert msg(24) == "block_rows must be 1 or 128"
    assert "16-byte aligned" in msg(26) and msg(27) == "inner dimensions do not match"
