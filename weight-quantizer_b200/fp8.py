"""Blocks of 8-bit floating point: quantization, the matrix product of two such
operands, and a linear layer that computes, and remembers its input, in 8 bits.

An operand (``Fp8Blocks``) holds e4m3 codes and one fp32 scale per block and
stands for ``code * scale``. Activations and gradients carry a scale per 128
values of a row (``block_rows=1``), weights one per 128 x 128 tile
(``block_rows=128``):

    y[m, n] = sum_b sa[m, b] * sw[n // 128, b] * sum_{k in block b} a[m, k] * w[n, k]

``quantize_fp8`` makes such operands (its scales are powers of two, so dividing
by one loses nothing); the products take operands with other scales too, such as
a checkpoint's, as long as ``sa * sw`` is a normal fp32 number or 0 (it is
computed first). ``fp8_linear`` is the differentiable layer: its forward product
reads the input in 8 bits, and the same codes, one byte per value instead of
two or four, are all that it keeps of the input for the weight's gradient:

    x8, w8 = quantize(x), quantize(w)          y  = x8 w8^T + bias
    dx = quantize(dy) w8                       dw = dy^T x8        db = sum_m dy

(the quantizers count as the identity for the gradients). None of this has a
counterpart in ptqkit. Inputs are CUDA tensors; results are written on the
current CUDA stream and returned without a host synchronization.
"""

from __future__ import annotations

from collections.abc import Callable
from dataclasses import dataclass
from typing import Any

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _kernels

FP8_BLOCK = _kernels.FP8_BLOCK
_BLOCK_ROWS = (1, FP8_BLOCK)


@dataclass(frozen=True)
class Fp8Blocks:
    """A [rows, cols] matrix as e4m3 codes and one scale per block.

    ``codes`` is float8_e4m3fn [rows, cols]; ``scales`` is float32
    [ceil(rows / block_rows), ceil(cols / 128)]. Any strides; the products
    read codes without a copy when the columns are contiguous, the first code
    is 16-byte aligned and rows lie a multiple of 16 bytes apart, as
    ``quantize_fp8`` lays them out. The last block of a row or column may be short.
    """

    codes: torch.Tensor
    scales: torch.Tensor
    block_rows: int = 1

    def __post_init__(self) -> None:
        if self.block_rows not in _BLOCK_ROWS:
            raise ValueError("block_rows must be 1 or 128")
        if self.codes.ndim != 2 or self.codes.dtype != torch.float8_e4m3fn:
            raise ValueError("codes must be a float8_e4m3fn matrix")
        rows, cols = self.codes.shape
        want = (-(-rows // self.block_rows), -(-cols // FP8_BLOCK))
        if self.scales.dtype != torch.float32 or self.scales.shape != want:
            raise ValueError(f"scales must be float32 {list(want)}, one per block of {self.block_rows} x {FP8_BLOCK}")

    @property
    def shape(self) -> tuple[int, int]:
        return int(self.codes.shape[0]), int(self.codes.shape[1])

    def to(self, device: torch.device | str) -> Fp8Blocks:
        """Copy of this operand with both tensors on ``device`` (codes in padded rows on a GPU)."""
        return Fp8Blocks(_kernels.fp8_padded(self.codes.to(device)), self.scales.to(device), self.block_rows)


def _flat(x: torch.Tensor) -> torch.Tensor:
    """x [..., cols] as [rows, cols]."""
    return x if x.ndim == 2 else x.reshape(x.shape[:-1].numel(), x.shape[-1])


def quantize_fp8(x: torch.Tensor, *, block_rows: int = 1) -> Fp8Blocks:
    """Quantize ``x`` [..., cols] (float32, float16 or bfloat16; leading dims are
    flattened to rows) to e4m3 codes with one scale per ``block_rows`` x 128 block.

    A block's scale is the least power of two s >= 2^-117 with max|x| <= 448 s
    over its finite values (1 for a block of zeros); a code is the e4m3 value
    nearest to x / s, ties to even. NaN and infinities become the NaN code.
    (From 2^128 (1 - 2^-5) on a value's code stands for 2^128, beyond float32.)
    """
    if block_rows not in _BLOCK_ROWS:
        raise ValueError("block_rows must be 1 or 128")
    if x.ndim < 1:
        raise ValueError("x must have shape [..., cols]")
    return Fp8Blocks(*_kernels.fp8_quantize(_flat(x), block_rows), block_rows)


def dequantize_fp8(q: Fp8Blocks, *, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The dense [rows, cols] matrix ``code * scale``, rounded once to ``dtype``."""
    return _kernels.fp8_dequantize(q.codes, q.scales, q.block_rows, dtype)


def fp8_gemm(
    a: Fp8Blocks | torch.Tensor,
    w: Fp8Blocks,
    *,
    transpose: bool = False,
    bias: torch.Tensor | None = None,
    out_dtype: torch.dtype | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """``a @ w^T (+ bias)``, or with ``transpose`` ``a @ w`` (the input gradient of
    the layer whose stored weight is ``w`` [out, in]).

    ``a``: an operand with ``block_rows=1``, or a 16- or 32-bit tensor
    [..., cols] that the call quantizes as ``quantize_fp8`` would. ``w``: an
    operand with ``block_rows=128``. Blocks are summed in fp32 and the result
    rounded once to ``out_dtype`` (default: a tensor ``a``'s own type, bfloat16
    for an operand). ``out`` may be a preallocated [rows, columns] matrix.
    """
    if w.block_rows != FP8_BLOCK:
        raise ValueError("the weight must have one scale per 128 x 128 tile (block_rows=128)")
    if isinstance(a, Fp8Blocks):
        if a.block_rows != 1:
            raise ValueError("a must have one scale per 128 values of a row (block_rows=1)")
        dt = torch.bfloat16 if out_dtype is None else out_dtype
        return _kernels.fp8_gemm(a.codes, a.scales, w.codes, w.scales, transpose, bias,
                                 out.dtype if out is not None and out_dtype is None else dt, out)
    if a.ndim < 1:
        raise ValueError("a must have shape [..., cols]")
    n_in = w.codes.shape[0 if transpose else 1]
    if a.shape[-1] != n_in:
        raise ValueError(f"a has trailing dim {a.shape[-1]}, weight expects {n_in}")
    lead = a.shape[:-1]
    dt = out_dtype if out_dtype is not None else (out.dtype if out is not None else a.dtype)
    y = _kernels.fp8_gemm(_flat(a), None, w.codes, w.scales, transpose, bias, dt, out)
    return y if len(lead) == 1 else y.reshape(*lead, y.shape[1])


def fp8_weight_grad(
    dy: torch.Tensor,
    x: Fp8Blocks,
    *,
    out_dtype: torch.dtype = torch.float32,
    out: torch.Tensor | None = None,
    accumulate: bool = False,
) -> torch.Tensor:
    """``dy^T @ x``: the gradient of a layer's weight [out, in] from the gradient of
    its output ``dy`` [..., out] and the 8-bit checkpoint of its input ``x``
    [rows, in] (``block_rows=1``).

    With ``quantize_fp8``'s scales no operand is rounded (x's values are exact in
    bfloat16, and a 16- or 32-bit ``dy`` enters the product as a sum of bfloat16
    terms, down to bits of 2^-133);
    other scales' ``code * scale`` is rounded to bfloat16. ``accumulate`` adds to
    ``out``, in ``out``'s type.
    """
    if x.block_rows != 1:
        raise ValueError("x must have one scale per 128 values of a row (block_rows=1)")
    if dy.ndim < 1:
        raise ValueError("dy must have shape [..., out]")
    if accumulate and out is None:
        raise ValueError("accumulate adds to out, which is missing")
    return _kernels.fp8_weight_grad(_flat(dy), x.codes, x.scales, out.dtype if out is not None else out_dtype, out,
                                    accumulate)


class _Fp8LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None) -> torch.Tensor:
        xc, xs = _kernels.fp8_quantize(_flat(x), 1)
        wc, ws = _kernels.fp8_quantize(weight, FP8_BLOCK)
        y = _kernels.fp8_gemm(xc, xs, wc, ws, False, bias, x.dtype, None)
        needs_x, needs_w, _ = ctx.needs_input_grad
        ctx.save_for_backward(*((xc, xs) if needs_w else (None, None)), *((wc, ws) if needs_x else (None, None)))
        ctx.x_shape, ctx.x_dtype, ctx.w_dtype = x.shape, x.dtype, weight.dtype
        ctx.b_dtype = None if bias is None else bias.dtype
        return y if x.ndim == 2 else y.reshape(*x.shape[:-1], weight.shape[0])

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, dy: torch.Tensor) -> tuple[torch.Tensor | None, ...]:
        xc, xs, wc, ws = ctx.saved_tensors
        dy2 = _flat(dy)
        dx = dw = db = None
        if ctx.needs_input_grad[0]:
            dx = _kernels.fp8_gemm(dy2, None, wc, ws, True, None, ctx.x_dtype, None)
            dx = dx if len(ctx.x_shape) == 2 else dx.reshape(ctx.x_shape)
        if ctx.needs_input_grad[1]:
            dw = _kernels.fp8_weight_grad(dy2, xc, xs, ctx.w_dtype, None, False)
        if ctx.needs_input_grad[2]:
            db = _kernels.column_sum(dy2, ctx.b_dtype)
        return dx, dw, db


def _autocast(x: torch.Tensor) -> torch.Tensor:
    """x in the type that a linear layer takes it in: under autocast autocast's, otherwise its own."""
    if torch.is_autocast_enabled("cuda") and x.is_cuda and x.dtype in _kernels.FP8_INPUTS:
        return x.to(torch.get_autocast_dtype("cuda"))
    return x


def fp8_linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None) -> torch.Tensor:
    """``x @ weight^T + bias`` from 8-bit operands, differentiable (see the module docstring).

    ``x`` [..., in], ``weight`` [out, in] and ``bias`` [out] are float32, float16
    or bfloat16; the result has x's type, each gradient its input's. Of ``x`` the
    graph keeps the 8-bit codes and their scales, of ``weight`` its 8-bit tiles.
    Under ``torch.autocast`` x is cast to autocast's type first, as a linear layer's
    input is, and the result has that type; weight and bias are read as they are.
    (``torch.func`` transforms refuse it.)
    """
    if weight.ndim != 2:
        raise ValueError("weight must have shape [out, in]")
    if x.ndim < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"x has trailing dim {x.shape[-1] if x.ndim else None}, weight expects {weight.shape[1]}")
    if bias is not None and tuple(bias.shape) != (weight.shape[0],):
        raise ValueError("bias does not match out_features")
    for name, t in (("x", x), ("weight", weight), ("bias", bias)):
        if t is not None and t.device.type != "cuda":
            raise ValueError(f"{name} must be a CUDA tensor")
    return _Fp8LinearFn.apply(_autocast(x), weight, bias)


class Fp8Linear(nn.Module):
    """A linear layer over ``fp8_linear``: 8-bit operands in the forward product and
    in the input gradient, an 8-bit checkpoint of the input for the weight gradient.

    ``freeze()`` replaces the trainable weight by its 8-bit tiles (one byte per
    weight, buffers ``codes`` and ``scales``), after which a forward quantizes
    its input alone and the layer serves without gradients.
    """

    weight: torch.Tensor | None
    bias: torch.Tensor | None
    codes: torch.Tensor | None
    scales: torch.Tensor | None

    def __init__(self, weight: torch.Tensor, bias: torch.Tensor | None = None) -> None:
        super().__init__()
        if weight.ndim != 2:
            raise ValueError("weight must have shape [out, in]")
        if bias is not None and int(bias.numel()) != int(weight.shape[0]):
            raise ValueError("bias does not match out_features")
        self.out_features, self.in_features = int(weight.shape[0]), int(weight.shape[1])
        self.weight = weight if isinstance(weight, nn.Parameter) else nn.Parameter(weight.detach())
        if bias is None or isinstance(bias, nn.Parameter):
            self.bias = bias
        else:
            self.bias = nn.Parameter(bias.detach().reshape(-1))
        self.register_buffer("codes", None)
        self.register_buffer("scales", None)

    @classmethod
    def from_linear(cls, module: nn.Linear) -> Fp8Linear:
        """The layer over ``module``'s own parameters (shared, not copied)."""
        return cls(module.weight, module.bias)

    def freeze(self) -> Fp8Linear:
        """Keep the weight as 8-bit tiles only, for serving."""
        if self.weight is not None:
            q = quantize_fp8(self.weight, block_rows=FP8_BLOCK)
            self.codes, self.scales = q.codes, q.scales
            self.weight = None
            if self.bias is not None:
                self.bias.requires_grad_(False)
        return self

    def _apply(self, fn: Callable[..., Any], recurse: bool = True) -> Fp8Linear:
        # a cast (half(), to(dtype)) is for the parameters: codes and scales only move, and
        # a copy of rows that do not fill their pitch comes without the padding
        codes, scales = self.codes, self.scales
        super()._apply(fn, recurse=recurse)  # type: ignore[no-untyped-call]
        if codes is not None and scales is not None and self.scales is not None:
            dev = self.scales.device
            self.codes, self.scales = _kernels.fp8_padded(codes.to(dev)), scales.to(dev)
        return self

    def _load_from_state_dict(self, *args: Any, **kwargs: Any) -> None:
        super()._load_from_state_dict(*args, **kwargs)  # type: ignore[no-untyped-call]
        if self.codes is not None:   # (with assign=True the state's own tensors)
            self.codes = _kernels.fp8_padded(self.codes)

    def quantized_weight(self) -> Fp8Blocks:
        """The weight as the products read it."""
        if self.weight is not None:
            return quantize_fp8(self.weight, block_rows=FP8_BLOCK)
        assert self.codes is not None and self.scales is not None
        return Fp8Blocks(self.codes, self.scales, FP8_BLOCK)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.shape[-1] != self.in_features:
            raise ValueError(f"expected in_features={self.in_features}, got {x.shape[-1]}")
        if self.weight is not None:
            return fp8_linear(x, self.weight, self.bias)
        if torch.is_grad_enabled() and x.requires_grad:
            raise RuntimeError("a frozen Fp8Linear has no backward pass; call it under torch.no_grad()")
        return fp8_gemm(_autocast(x), self.quantized_weight(), bias=self.bias)

    def extra_repr(self) -> str:
        return (f"in={self.in_features}, out={self.out_features}, block={FP8_BLOCK}, "
                f"frozen={self.weight is None}")
