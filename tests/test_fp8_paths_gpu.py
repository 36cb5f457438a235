"""The kernels of the 8-bit floating-point operators that large layers, few rows and long inner dimensions take,
against plain 64-bit computations, by the bounds of test_fp8_gpu.py.
"""

from __future__ import annotations

import pytest
import torch

from test_fp8_gpu import DTYPES, check_product, rand, values64

pytestmark = pytest.mark.gpu


# ---- the weight gradient -----------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
def test_weight_grad_operand_of_the_other_cta(wq, cuda, dtype) -> None:
    """Half of each tile's columns come from an operand that the pair's other CTA made in its own shared memory: many
    tiles and steps, many times over while the card is busy, every result with the same bits and right."""
    x = wq.quantize_fp8(rand((1000, 4096), 1, torch.bfloat16))
    dy = rand((1000, 4096), 2, dtype, 1e-2)
    dw = wq.fp8_weight_grad(dy, x)
    check_product(dw, dy.double().t(), values64(x))
    out = torch.empty_like(dw)
    for _ in range(40):
        out.fill_(float("nan"))
        wq.fp8_weight_grad(dy, x, out=out)
        assert torch.equal(out, dw)
