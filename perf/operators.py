"""The 8-bit floating-point operators, as a user's program calls them.

Blocks of 8-bit floating point (e4m3, one scale per 128 values of a row, or per 128 x 128 values
of a weight), the matrix product of two such operands, its two gradients (the input's from 8-bit
operands, the weight's from the 8-bit checkpoint of the layer's input), and the linear layer made
of them. ``own`` selects the framework's calls or the plain form in elementary torch operations.
"""

import importlib
import math

import torch

own = False

BLOCK = 128
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


# ---- the cases ---------------------------------------------------------------


def listed():
    return [
        # one token's activations on their way into a decode step: a launch's latency
        {"name": "quantize 1x8192", "op": "quantize", "tiles": False, "rows": 1, "cols": 8192, "dtype": "bf16"},
        # a prefill batch (or a training micro-batch) of activations
        {"name": "quantize 4096x8192", "op": "quantize", "tiles": False, "rows": 4096, "cols": 8192, "dtype": "bf16"},
        # a layer's fp32 master weight, after an optimizer step or at load time
        {"name": "quantize tiles 28672x8192", "op": "quantize", "tiles": True, "rows": 28672, "cols": 8192,
         "dtype": "fp32"},
        # decode: one token through the largest layer, straight from its 16-bit activations
        {"name": "product 1x28672x8192", "op": "linear", "rows": 1, "outs": 28672, "ins": 8192, "dtype": "bf16",
         "bias": False},
        # a small batch of requests on the layer with an odd input width, in fp32, with a bias
        {"name": "product 32x4096x4095", "op": "linear", "rows": 32, "outs": 4096, "ins": 4095, "dtype": "fp32",
         "bias": True},
        # prefill: the operands are in 8 bits already
        {"name": "product 4096x28672x8192", "op": "product", "rows": 4096, "outs": 28672, "ins": 8192,
         "dtype": "bf16"},
        # the input's gradient of a short sequence, ragged
        {"name": "input gradient 333x11008x4096", "op": "dgrad", "rows": 333, "outs": 11008, "ins": 4096,
         "dtype": "fp16"},
        # the input's gradient of a training micro-batch
        {"name": "input gradient 4096x11008x4096", "op": "dgrad", "rows": 4096, "outs": 11008, "ins": 4096,
         "dtype": "bf16"},
        # the weight's gradient of a small layer over a ragged batch, in fp32 throughout
        {"name": "weight gradient 777x2304x768", "op": "wgrad", "rows": 777, "outs": 2304, "ins": 768,
         "dtype": "fp32", "grad": "fp32"},
        # the weight's gradient of a large layer, added up in fp32 for the optimizer
        {"name": "weight gradient 8192x11008x4096", "op": "wgrad", "rows": 8192, "outs": 11008, "ins": 4096,
         "dtype": "bf16", "grad": "fp32"},
        # forward and backward of a small layer on a short sequence
        {"name": "step 64x2304x768", "op": "step", "rows": 64, "outs": 2304, "ins": 768, "dtype": "fp32",
         "bias": True},
        # forward and backward of a large layer on a training micro-batch
        {"name": "step 4096x11008x4096", "op": "step", "rows": 4096, "outs": 11008, "ins": 4096, "dtype": "bf16",
         "bias": True},
    ]


def _log(rng, low, high):
    """A whole number from low to high, spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["quantize", "linear", "product", "dgrad", "wgrad", "step"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "quantize":
        return {"op": op, "tiles": rng.random() < 0.4, "rows": _log(rng, 1, 16384), "cols": _log(rng, 16, 12288),
                "dtype": dtype}
    # no drawn case computes more than the largest listed product; a step has three products
    rows = _log(rng, 16 if op == "wgrad" else 1, {"linear": 64, "step": 2048}.get(op, 8192))
    outs, ins = _log(rng, 128, 14336), _log(rng, 128, 8192)
    case = {"op": op, "rows": rows, "outs": outs, "ins": ins, "dtype": dtype}
    if op in ("linear", "step"):
        case["bias"] = rng.random() < 0.5
    if op == "wgrad":
        case["grad"] = rng.choice([dtype, "fp32"])
    return case


# ---- what is in hand before the call --------------------------------------------


def _generator(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(1000003 * seed + 7919 * case["rows"] + case.get("ins", case.get("cols", 0)))
    return g


def _activations(g, rows, cols, dtype):
    """Normal values, one channel in a hundred twenty times as large, and the all-zero rows of padding."""
    x = torch.randn(rows, cols, generator=g, device="cuda")
    loud = torch.rand(cols, generator=g, device="cuda") < 0.01
    x = torch.where(loud, x * 20.0, x)
    pad = (torch.arange(rows, device="cuda") % 97 == 5).unsqueeze(1)
    return x.masked_fill_(pad, 0.0).to(dtype)


def _upstream(g, rows, cols, dtype):
    """A loss's gradient: small, and of another size for each token."""
    size = torch.exp(torch.randn(rows, 1, generator=g, device="cuda")) * 1e-2
    return (torch.randn(rows, cols, generator=g, device="cuda") * size).to(dtype)


def _weight(g, outs, ins, dtype=torch.float32):
    return (torch.randn(outs, ins, generator=g, device="cuda") * 0.02).to(dtype)


def _stored(codes, scales, tiles):
    """Codes and scales as the framework keeps them: rows of codes 16 bytes or a multiple apart, the scales of
    single rows with one block's values of all rows side by side."""
    rows, cols = codes.shape
    pitch = (cols + 15) // 16 * 16
    kept = torch.zeros(rows, pitch, dtype=codes.dtype, device=codes.device)
    kept.view(torch.uint8)[:, :cols] = codes.view(torch.uint8)
    if not tiles:
        scales = scales.t().contiguous().t()
    return kept[:, :cols], scales


def prepare(case, seed):
    g = _generator(case, seed)
    op, dt = case["op"], DTYPES[case["dtype"]]
    s = {"case": case}
    if op == "quantize":
        s["x"] = (_weight if case["tiles"] else _activations)(g, case["rows"], case["cols"], dt)
        return s
    rows, outs, ins = case["rows"], case["outs"], case["ins"]
    if op in ("linear", "product", "dgrad"):
        w = _weight(g, outs, ins)
        # a loaded checkpoint's scales are any numbers, not only powers of two
        s["w"] = _stored(*_any_scales(w), True)
    if op == "linear":
        s["x"] = _activations(g, rows, ins, dt)
        s["bias"] = torch.randn(outs, generator=g, device="cuda") if case["bias"] else None
    elif op == "product":
        s["a"] = _stored(*_quantize(_activations(g, rows, ins, dt), False), False)
    elif op == "dgrad":
        s["a"] = _stored(*_quantize(_upstream(g, rows, outs, dt), False), False)
    elif op == "wgrad":
        s["a"] = _stored(*_quantize(_activations(g, rows, ins, dt), False), False)
        s["dy"] = _upstream(g, rows, outs, dt)
    elif op == "step":
        s["x"] = _activations(g, rows, ins, dt).requires_grad_()
        s["w"] = _weight(g, outs, ins, dt).requires_grad_()
        s["bias"] = torch.randn(outs, generator=g, device="cuda").to(dt).requires_grad_() if case["bias"] else None
        s["dy"] = _upstream(g, rows, outs, dt)
    return s


def _any_scales(w):
    """128 x 128 tiles with the scale max / 448, as other programs' checkpoints hold them."""
    rows, cols = w.shape
    br, bc = -(-rows // BLOCK), -(-cols // BLOCK)
    padded = torch.nn.functional.pad(w, (0, bc * BLOCK - cols, 0, br * BLOCK - rows))
    tiles = padded.view(br, BLOCK, bc, BLOCK)
    scales = tiles.abs().amax(dim=(1, 3)).clamp_min(1e-12) / 448.0
    codes = (tiles / scales[:, None, :, None]).clamp(-448.0, 448.0).view(br * BLOCK, bc * BLOCK)[:rows, :cols]
    return codes.to(torch.float8_e4m3fn), scales


# ---- the plain form -----------------------------------------------------------------


def _blocks(x, tiles):
    """x in fp32, padded to whole blocks: [row blocks, rows of a block, column blocks, 128]."""
    rows, cols = x.shape
    br = BLOCK if tiles else 1
    nr, nc = -(-rows // br), -(-cols // BLOCK)
    padded = torch.nn.functional.pad(x.float(), (0, nc * BLOCK - cols, 0, nr * br - rows))
    return padded.view(nr, br, nc, BLOCK)


def _quantize(x, tiles):
    """e4m3 codes and the scale of each block: the least power of two, not below 2^-117, by which the largest
    magnitude is at most 448 (1 for a block of zeros)."""
    rows, cols = x.shape
    b = _blocks(x, tiles)
    mant, expo = torch.frexp(b.abs().amax(dim=(1, 3)))
    expo = torch.where(mant <= 0.875, expo - 9, expo - 8).clamp_min(-117)
    scales = torch.where(mant == 0.0, torch.ones_like(mant), torch.ldexp(torch.ones_like(mant), expo))
    codes = (b / scales[:, None, :, None]).flatten(2).flatten(0, 1)[:rows, :cols].to(torch.float8_e4m3fn)
    return codes, scales


def _values(codes, scales, tiles):
    """The fp32 matrix that codes and scales stand for."""
    rows, cols = codes.shape
    b = _blocks(codes, tiles)
    return (b * scales[:, None, :, None]).flatten(2).flatten(0, 1)[:rows, :cols]


def _plain(s):
    case = s["case"]
    op, dt = case["op"], DTYPES[case["dtype"]]
    if op == "quantize":
        return _quantize(s["x"], case["tiles"])
    if op == "linear":
        y = _values(*_quantize(s["x"], False), False) @ _values(*s["w"], True).t()
        return (y if s["bias"] is None else y + s["bias"]).to(dt)
    if op == "product":
        return (_values(*s["a"], False) @ _values(*s["w"], True).t()).to(dt)
    if op == "dgrad":
        return (_values(*s["a"], False) @ _values(*s["w"], True)).to(dt)
    if op == "wgrad":
        return (s["dy"].float().t() @ _values(*s["a"], False)).to(DTYPES[case["grad"]])
    with torch.no_grad():
        x = _values(*_quantize(s["x"], False), False)
        w = _values(*_quantize(s["w"], True), True)
        y = x @ w.t()
        if s["bias"] is not None:
            y = y + s["bias"].float()
        dx = _values(*_quantize(s["dy"], False), False) @ w
        dw = s["dy"].float().t() @ x
        grads = [dx.to(dt), dw.to(dt)]
        if s["bias"] is not None:
            grads.append(s["dy"].float().sum(dim=0).to(dt))
        return [y.to(dt), *grads]


# ---- the framework's calls ------------------------------------------------------------


def _own(s):
    wq = importlib.import_module("weight-quantizer_b200")
    case = s["case"]
    op, dt = case["op"], DTYPES[case["dtype"]]
    if op == "quantize":
        q = wq.quantize_fp8(s["x"], block_rows=BLOCK if case["tiles"] else 1)
        return q.codes, q.scales
    if op == "linear":
        return wq.fp8_gemm(s["x"], wq.Fp8Blocks(*s["w"], block_rows=BLOCK), bias=s["bias"], out_dtype=dt)
    if op == "product":
        return wq.fp8_gemm(wq.Fp8Blocks(*s["a"]), wq.Fp8Blocks(*s["w"], block_rows=BLOCK), out_dtype=dt)
    if op == "dgrad":
        return wq.fp8_gemm(wq.Fp8Blocks(*s["a"]), wq.Fp8Blocks(*s["w"], block_rows=BLOCK), transpose=True,
                           out_dtype=dt)
    if op == "wgrad":
        return wq.fp8_weight_grad(s["dy"], wq.Fp8Blocks(*s["a"]), out_dtype=DTYPES[case["grad"]])
    y = wq.fp8_linear(s["x"], s["w"], s["bias"])
    leaves = [s["x"], s["w"]] + ([] if s["bias"] is None else [s["bias"]])
    return [y.detach(), *torch.autograd.grad(y, leaves, s["dy"])]


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without ---------------------------------------------------


def _held(rows, cols, tiles):
    """Bytes of an 8-bit operand: its codes and its scales."""
    return rows * cols + 4 * (-(-rows // BLOCK) if tiles else rows) * -(-cols // BLOCK)


def work(case):
    op, n = case["op"], BYTES[case["dtype"]]
    if op == "quantize":
        rows, cols = case["rows"], case["cols"]
        return {"bytes": rows * cols * n + _held(rows, cols, case["tiles"]), "flops": 2 * rows * cols}
    rows, outs, ins = case["rows"], case["outs"], case["ins"]
    mm = 2 * rows * outs * ins
    if op == "linear":
        return {"bytes": rows * ins * n + _held(outs, ins, True) + rows * outs * n + (4 * outs if case["bias"] else 0),
                "flops": mm}
    if op == "product":
        return {"bytes": _held(rows, ins, False) + _held(outs, ins, True) + rows * outs * n, "flops": mm}
    if op == "dgrad":
        return {"bytes": _held(rows, outs, False) + _held(outs, ins, True) + rows * ins * n, "flops": mm}
    if op == "wgrad":
        return {"bytes": _held(rows, ins, False) + rows * outs * n + outs * ins * BYTES[case["grad"]], "flops": mm}
    # x, w, b, dy in; y, dx, dw, db out
    vectors = 2 * outs * n if case["bias"] else 0
    return {"bytes": n * (2 * rows * ins + 2 * rows * outs + 2 * outs * ins) + vectors, "flops": 3 * mm}


# ---- the definition in 64 bits ----------------------------------------------------------


def _e4m3(v):
    """The nearest e4m3 value of each v (|v| <= 448), ties to the even one: steps of 2^(e-3), e >= -6."""
    e = torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -40))).clamp_min(-6.0)
    # log2 next to a power of two may fall on its other side
    e = torch.where(v.abs() >= torch.exp2(e + 1.0), e + 1.0, e)
    e = torch.where((v.abs() < torch.exp2(e)) & (e > -6.0), e - 1.0, e)
    step = torch.exp2(e - 3.0)
    return torch.round(v / step) * step


def _block_max(x, height):
    rows, cols = x.shape
    out = torch.zeros(-(-rows // height), -(-cols // BLOCK), dtype=torch.float64, device=x.device)
    for j in range(out.shape[1]):
        strip = x[:, j * BLOCK:(j + 1) * BLOCK].abs().amax(dim=1).double()
        full = torch.zeros(out.shape[0] * height, dtype=torch.float64, device=x.device)
        full[:rows] = strip
        out[:, j] = full.view(-1, height).amax(dim=1)
    return out


def _spread(scales, rows, cols, height):
    return scales.double().repeat_interleave(height, dim=0)[:rows].repeat_interleave(BLOCK, dim=1)[:, :cols]


def _exact_quantize(x, height):
    """(e4m3 values, scales) in 64 bits."""
    top = _block_max(x, height)
    scales = torch.ones_like(top)
    some = top > 0
    k = torch.ceil(torch.log2(top[some] / 448.0))
    k = torch.where(top[some] <= 448.0 * torch.exp2(k - 1.0), k - 1.0, k)
    k = torch.where(top[some] > 448.0 * torch.exp2(k), k + 1.0, k)
    scales[some] = torch.exp2(k.clamp_min(-117.0))
    return _e4m3(x.double() / _spread(scales, *x.shape, height)), scales


def _exact_values(x, height):
    codes, scales = _exact_quantize(x, height)
    return codes * _spread(scales, *x.shape, height)


def _exact_stored(pair, height):
    codes, scales = pair
    return codes.to(torch.float64) * _spread(scales, *codes.shape, height)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    with torch.no_grad():
        if op == "quantize":
            return _exact_quantize(s["x"], BLOCK if case["tiles"] else 1)
        if op == "linear":
            y = _exact_values(s["x"], 1) @ _exact_stored(s["w"], BLOCK).t()
            return y if s["bias"] is None else y + s["bias"].double()
        if op == "product":
            return _exact_stored(s["a"], 1) @ _exact_stored(s["w"], BLOCK).t()
        if op == "dgrad":
            return _exact_stored(s["a"], 1) @ _exact_stored(s["w"], BLOCK)
        if op == "wgrad":
            return s["dy"].double().t() @ _exact_stored(s["a"], 1)
        x, w = _exact_values(s["x"], 1), _exact_values(s["w"], BLOCK)
        y = x @ w.t()
        out = [_exact_values(s["dy"], 1) @ w, s["dy"].double().t() @ x]
        if s["bias"] is not None:
            y = y + s["bias"].double()
            out.append(s["dy"].double().sum(dim=0))
        return [y, *out]
