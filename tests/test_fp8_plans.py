"""Which kernel of the 8-bit floating-point operators sizes take, asked without a GPU (148 SMs are assumed then):
the sizes of test_fp8_paths_gpu.py take the kernels that they are there to test, and every kernel has some. What a
call asks of the library, on which device."""

from __future__ import annotations

import ctypes

import torch

from test_fp8_paths_gpu import GRADIENTS, PRODUCTS


def test_sizes_take_the_kernels_they_test(wq) -> None:
    for size, plan in PRODUCTS.items():
        assert wq._kernels.fp8_gemm_plan(*size) == plan, size
    kinds = {(k, t, p > 1) for k, t, p in PRODUCTS.values()}
    assert kinds == {("few rows", t, False) for t in (16, 32, 64)} | {("pairs", t, p) for t in (128, 256)
                                                                     for p in (False, True)}
    for size, plan in GRADIENTS.items():
        for dtype in (torch.bfloat16, torch.float16, torch.float32):
            assert wq._kernels.fp8_weight_grad_plan(*size, dtype) == plan, size


def test_the_faster_kernel_at_64_rows(wq) -> None:
    """Weights for which one of the two kernels was measured at least a tenth faster than the other."""
    for n, k in ((28672, 8192), (8192, 28672), (60000, 4000), (128256, 4096), (16384, 16384), (1024, 14336),
                 (20000, 8000), (4096, 11008)):
        for m in (33, 48, 64):
            assert wq._kernels.fp8_gemm_plan(m, n, k)[0] == "few rows", (m, n, k)
    for n, k in ((4096, 4096), (14336, 4096), (5120, 5120), (8192, 8192), (24000, 1000), (2304, 768), (50257, 768)):
        for m in (33, 48, 64):
            assert wq._kernels.fp8_gemm_plan(m, n, k)[0] == "pairs", (m, n, k)


def test_plan_c_refusals(wq) -> None:
    lib = wq._kernels.library()
    a, b, c = (ctypes.c_int() for _ in range(3))
    p = lib.wq_fp8_gemm_plan
    assert p(0, 8, 8, a, b, c) == 5 and p(8, -1, 8, a, b, c) == 5
    assert p(1 << 23, 8, 8, a, b, c) == 13
    assert p(8, 8, 8, None, b, c) == 11 and p(8, 8, 8, a, b, c) == 0
    g = lib.wq_fp8_weight_grad_plan
    assert g(8, 8, 0, 0, a, b) == 5 and g(8, 8, 8, 3, a, b) == 23 and g(8, 8, 8, 0, None, b) == 11
    assert g(8, 8, 1 << 23, 0, a, b) == 13 and g(8, 8, 8, 2, a, b) == 0


def test_weight_grad_workspace(wq) -> None:
    """bf16 rows that TMA reads need no terms; the query by type covers every dy of the type."""
    lib = wq._kernels.library()
    M, N, K = 8192, 28672, 4096
    assert wq._kernels.fp8_weight_grad_plan(M, N, K, torch.bfloat16)[1] == 1
    every, this = lib.wq_fp8_weight_grad_workspace_bytes, lib.wq_fp8_weight_grad_workspace_for
    at = ctypes.c_void_p
    assert this(at(256), 2, M, N, N, K) == 0
    for dy, ld in ((258, N), (256, N + 1)):
        assert this(at(dy), 2, M, N, ld, K) == M * N * 2 == every(M, N, K, 2)
    assert this(at(256), 1, M, N, N, K) == M * N * 2 * 2 == every(M, N, K, 1)
    assert this(at(256), 0, M, N, N, K) == M * N * 2 * 3 == every(M, N, K, 0)
    # in parts: the counters and sums, with or without the terms
    assert wq._kernels.fp8_weight_grad_plan(8192, 128, 128, torch.bfloat16)[1] > 1
    parts = this(at(256), 2, 8192, 128, 128, 128)
    assert parts > 0 and this(at(256), 2, 8192, 128, 129, 128) == parts + 8192 * 128 * 2
    assert this(at(256), 2, 0, N, N, K) == 0
    # the call asks for what its dy needs
    p, big = at(256), 1 << 40

    def call(dy, ld, ws, nws):  # type: ignore[no-untyped-def]
        return lib.wq_fp8_weight_grad(dy, 2, M, N, ld, p, K, K, p, 1, M, p, 0, K, 0, ws, nws, None)

    assert call(at(258), N, None, 0) == 12 and call(p, N + 1, p, M * N * 2 - 1) == 12
    assert call(at(258), N, at(128), big) == 12


class _Held:
    """What the calls ask of a tensor, of one that lies on a device that is not here."""

    is_cuda = True

    def __init__(self, dtype: torch.dtype, *shape: int, device: int = 1) -> None:
        self.dtype, self.shape, self.ndim = dtype, shape, len(shape)
        self.device = torch.device("cuda", device)

    def stride(self, i: int | None = None):  # type: ignore[no-untyped-def]
        s = (self.shape[1], 1)
        return s if i is None else s[i]

    def numel(self) -> int:
        return self.shape[0] * self.shape[1]

    def data_ptr(self) -> int:
        return 4096


def test_sizes_are_asked_for_the_operands_device(wq, monkeypatch) -> None:
    """With operands on a device that is not the current one, workspaces are sized, and kernels launched, with theirs
    current; the current device is what it was afterwards."""
    k = wq._kernels
    now, seen = [0], []

    class Library:
        def __getattr__(self, name: str):  # type: ignore[no-untyped-def]
            def call(*args):  # type: ignore[no-untyped-def]
                seen.append((name, now[0]))
                return 0
            return call

    monkeypatch.setattr(k, "library", Library)
    monkeypatch.setattr(k, "_fault_check", False)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: now[0])
    monkeypatch.setattr(torch.cuda, "set_device", lambda d: now.__setitem__(0, d if isinstance(d, int) else d.index))
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 0, raising=False)
    e4m3, f32, bf16 = torch.float8_e4m3fn, torch.float32, torch.bfloat16
    a, w = _Held(e4m3, 4, 256), _Held(e4m3, 8, 256)
    out = _Held(bf16, 4, 8)
    for device in (1, 0):
        for t in (a, w, out):
            t.device = torch.device("cuda", device)
        sa, sw = _Held(f32, 4, 2, device=device), _Held(f32, 1, 2, device=device)
        k.fp8_gemm(a, sa, w, sw, False, None, bf16, out)
        k.fp8_gemm(_Held(bf16, 4, 256, device=device), None, w, sw, False, None, bf16, out)
        k.fp8_weight_grad(_Held(bf16, 4, 8, device=device), a, sa, f32, _Held(f32, 8, 256, device=device), False)
        assert len(seen) == 6 and {d for _, d in seen} == {device}, seen
        assert now == [0]
        seen.clear()
