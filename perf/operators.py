"""Cases for the microscaled operators: quantisation to blocks of 32 with a power-of-two scale
(mxfp8: e4m3 elements, mxfp4: e2m1 elements, e8m0 scales), the norm that leaves its rows in that
form, and the projections that take both of their operands in it.

``run`` computes every operator in elementary tensor operations, or, where ``own`` is true,
through the package's entry points.  The container is the package's: element codes row by row
(rows padded with zeros to a multiple of 128 elements, two e2m1 codes to a byte, the even element
in the low nibble) and the scales in tiles of 128 rows by 128 elements,
``scales[row // 128, k // 128, row % 32, row // 32 % 4, k // 32 % 4]``.
"""

from __future__ import annotations

import math

import torch

own = False

BLOCK = 32
STEP = 128
# largest element, and its exponent and leading digits: largest = digits * 2**exponent
LARGEST = {"mxfp4": (6.0, 2, 1.5), "mxfp8": (448.0, 8, 1.75)}
TYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ------------------------------------------------------------------------------------- cases

def listed():
    return [
        # a layer's fused gate/up weight, quantised once when a model is loaded (read back as values)
        dict(name="quantize_weight", op="quantize", rows=11264, cols=2048, dtype="bfloat16", format="mxfp4"),
        # the attention readers' float32 output of one decode step of sixteen sequences
        dict(name="quantize_step", op="quantize", rows=16, cols=2048, dtype="float32", format="mxfp8"),
        # the gated activations of eight prompts of 2048 tokens
        dict(name="quantize_prompts", op="quantize", rows=16384, cols=5632, dtype="bfloat16", format="mxfp8"),
        # the first norm of a decode step of one sequence: latency
        dict(name="norm_one_row", op="norm", rows=1, cols=2048, dtype="bfloat16", form="plain"),
        # the two norms between attention and MLP of a decode step of sixteen sequences
        dict(name="norm_step", op="norm", rows=16, cols=2048, dtype="bfloat16", form="sandwich"),
        # the same for sixteen prompts of 2048 tokens
        dict(name="norm_prompts", op="norm", rows=32768, cols=2048, dtype="bfloat16", form="sandwich"),
        # residual added before the norm, float16, a width that fills no block
        dict(name="norm_odd", op="norm", rows=771, cols=1001, dtype="float16", form="added"),
        # the fused Q/K/V projection of a decode step of sixteen sequences
        dict(name="linear_step", op="linear", rows=16, cols=2048, features=6144, x_format="mxfp8",
             w_format="mxfp4", out="bfloat16"),
        # a ragged product: short prompt, odd sizes, 8-bit weight, float32 out
        dict(name="linear_odd", op="linear", rows=77, cols=1000, features=1337, x_format="mxfp8",
             w_format="mxfp8", out="float32"),
        # the down projection of sixteen prompts of 2048 tokens
        dict(name="linear_prompts", op="linear", rows=32768, cols=5632, features=2048, x_format="mxfp8",
             w_format="mxfp4", out="bfloat16"),
        # gate/up projection and gated activation of a decode step, left quantised for the down projection
        dict(name="swiglu_step", op="swiglu", rows=16, cols=2048, features=5632, x_format="mxfp8",
             w_format="mxfp4", out="mxfp8"),
        # the same for eight prompts of 2048 tokens, in bfloat16
        dict(name="swiglu_prompts", op="swiglu", rows=16384, cols=2048, features=5632, x_format="mxfp8",
             w_format="mxfp4", out="bfloat16"),
    ]


def _size(rng, low, high):
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return n if rng.random() < 0.5 else min(high, -(-n // 64) * 64)


def draw(rng):
    op = rng.choice(("quantize", "norm", "linear", "swiglu"))
    rows, cols = int(round(math.exp(rng.uniform(0.0, math.log(32768))))), _size(rng, 32, 8192)
    dtype = rng.choice(("bfloat16", "bfloat16", "float16", "float32"))
    if op == "quantize":
        rows = max(1, min(rows, 16384 * 5632 // cols))
        return dict(op=op, rows=rows, cols=cols, dtype=dtype, format=rng.choice(("mxfp4", "mxfp8")))
    if op == "norm":
        rows = max(1, min(rows, 32768 * 2048 // cols))
        return dict(op=op, rows=rows, cols=cols, dtype=dtype, form=rng.choice(("plain", "added", "sandwich")))
    features = _size(rng, 32, 12288)
    most = 32768 * 5632 * 2048 if op == "linear" else 16384 * 2048 * 5632
    rows = max(1, min(rows, most // (cols * features)))
    formats = dict(x_format=rng.choice(("mxfp8", "mxfp8", "mxfp4")), w_format=rng.choice(("mxfp4", "mxfp4", "mxfp8")))
    out = rng.choice(("bfloat16", "float16", "float32") if op == "linear" else ("bfloat16", "float32", "mxfp8"))
    return dict(op=op, rows=rows, cols=cols, features=features, out=out, **formats)


def _padded(cols):
    return -(-cols // STEP) * STEP


def _mx_bytes(rows, cols, fmt):
    return rows * cols * (1.0 if fmt == "mxfp8" else 0.5) + rows * (-(-cols // BLOCK))


def work(case):
    rows, cols = case["rows"], case["cols"]
    if case["op"] == "quantize":
        size = TYPES[case["dtype"]].itemsize
        # mxfp4 codes are read back as bfloat16 values
        back = 0 if case["format"] == "mxfp8" else rows * cols * 2
        return {"bytes": rows * cols * size + _mx_bytes(rows, cols, case["format"]) + back, "flops": 4 * rows * cols}
    if case["op"] == "norm":
        size = TYPES[case["dtype"]].itemsize
        streams = {"plain": 1, "added": 3, "sandwich": 3}[case["form"]]
        weights = 2 if case["form"] == "sandwich" else 1
        return {"bytes": size * cols * (rows * streams + weights) + _mx_bytes(rows, cols, "mxfp8"),
                "flops": rows * cols * (16 if case["form"] == "sandwich" else 8)}
    n = case["features"]
    pair = 2 if case["op"] == "swiglu" else 1
    out = _mx_bytes(rows, n, "mxfp8") if case["out"] == "mxfp8" else rows * n * TYPES[case["out"]].itemsize
    return {"bytes": _mx_bytes(rows, cols, case["x_format"]) + pair * _mx_bytes(n, cols, case["w_format"]) + out,
            "flops": 2.0 * pair * rows * cols * n}


# ------------------------------------------------------------------------- the plain form

def _quantize(x, fmt):
    """float32 [rows, cols] -> element values [rows, padded] and scale exponents [rows, padded / 32]:
    the smallest power of two that keeps a block's elements in range, each element rounded to the
    nearest of the format, ties to the even code."""

    rows, cols = x.shape
    _, top, digits = LARGEST[fmt]
    x = torch.nn.functional.pad(x, (0, _padded(cols) - cols)).view(rows, -1, BLOCK)
    amax = x.abs().amax(-1)
    mantissa, exponent = torch.frexp(amax)
    exponent = exponent - 1 - top + (2 * mantissa > digits).to(exponent.dtype)
    exponent = torch.where(amax > 0, exponent, -127).clamp(-127, 127)
    scaled = torch.ldexp(x, -exponent[..., None])
    if fmt == "mxfp8":
        values = scaled.to(torch.float8_e4m3fn).float()
    else:
        step = torch.where(scaled.abs() < 2, 0.5, torch.where(scaled.abs() < 4, 1.0, 2.0))
        values = torch.round(scaled / step) * step
    return values.view(rows, -1), exponent


def _codes(values, fmt):
    if fmt == "mxfp8":
        return values.to(torch.float8_e4m3fn).view(torch.uint8)
    magnitude = torch.searchsorted(torch.tensor(E2M1, device=values.device), values.abs())
    code = (magnitude + 8 * torch.signbit(values)).to(torch.uint8)
    return code[:, 0::2] | (code[:, 1::2] << 4)


def _tile(exponent):
    """[rows, blocks] scale exponents -> the scale bytes in tiles; rows past the last have byte 0."""

    rows, blocks = exponent.shape
    byte = torch.nn.functional.pad((exponent + 127).to(torch.uint8), (0, 0, 0, -(-rows // 128) * 128 - rows))
    return byte.view(-1, 4, 32, blocks // 4, 4).permute(0, 3, 2, 1, 4).contiguous()


def _values(codes, scales, fmt, rows):
    """codes and scale tiles -> float32 [rows, padded]."""

    if fmt == "mxfp8":
        v = codes.view(torch.float8_e4m3fn).float()
    else:
        table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=codes.device)
        v = torch.stack((table[(codes & 15).int()], table[(codes >> 4).int()]), dim=-1).view(rows, -1)
    byte = scales.permute(0, 3, 2, 1, 4).reshape(-1, scales.shape[1] * 4)[:rows]
    return (v.view(rows, -1, BLOCK) * torch.ldexp(torch.ones_like(byte, dtype=torch.float32), byte.int() - 127)[..., None]).view(rows, -1)


def _held(values, exponent):
    """What an mxfp8 result is compared as: its elements and its scales, in their own types."""

    return {"codes": values.to(torch.float8_e4m3fn), "scales": _tile(exponent).view(torch.float8_e8m0fnu)}


def _normed(x, weight, eps):
    return weight * (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps))


# ------------------------------------------------------------------------------- the inputs

def _activations(gen, rows, cols, dtype=torch.float32):
    """Normal values with a few wide channels, as hidden states have them."""

    x = torch.randn(rows, cols, generator=gen, device="cuda")
    wide = torch.rand(cols, generator=gen, device="cuda") < 0.01
    return torch.where(wide, 8 * x, x).to(dtype)


def _operand(values, fmt):
    q, exponent = _quantize(values, fmt)
    codes, scales = _codes(q, fmt), _tile(exponent)
    state = {"codes": codes, "scales": scales, "format": fmt, "rows": values.shape[0], "cols": values.shape[1]}
    if own:
        from flashloop_b200 import MXTensor

        state["handle"] = MXTensor(codes, scales, tuple(values.shape), fmt)
    return state


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rows, cols = case["rows"], case["cols"]
    if case["op"] == "quantize":
        x = _activations(gen, rows, cols) if case["format"] == "mxfp8" else 0.02 * torch.randn(rows, cols, generator=gen, device="cuda")
        return {"case": case, "x": x.to(TYPES[case["dtype"]])}
    if case["op"] == "norm":
        dtype = TYPES[case["dtype"]]
        weights = [(1 + 0.1 * torch.randn(cols, generator=gen, device="cuda")).to(dtype) for _ in range(2)]
        return {"case": case, "x": _activations(gen, rows, cols, dtype), "other": _activations(gen, rows, cols, dtype),
                "weights": weights, "eps": 1e-6}
    x = _operand(_activations(gen, rows, cols), case["x_format"])
    weights = [_operand(torch.randn(case["features"], cols, generator=gen, device="cuda") * cols ** -0.5, case["w_format"])
               for _ in range(2 if case["op"] == "swiglu" else 1)]
    return {"case": case, "x": x, "weights": weights}


# --------------------------------------------------------------------------------- one pass

def _own(state):
    from flashloop_b200 import mx_linear, mx_linear_swiglu, mx_quantize, mx_rmsnorm

    case = state["case"]
    if case["op"] == "quantize":
        q = mx_quantize(state["x"], case["format"])
        return q.dequantize(torch.bfloat16) if case["format"] == "mxfp4" else _views(q)
    if case["op"] == "norm":
        w, eps, form = state["weights"], state["eps"], case["form"]
        if form == "plain":
            return _views(mx_rmsnorm(state["x"], w[0], eps)[0])
        if form == "added":
            q, _, total = mx_rmsnorm(state["x"], w[0], eps, addend=state["other"], want_sum=True)
            return {**_views(q), "sum": total}
        q, hidden, _ = mx_rmsnorm(state["x"], w[0], eps, residual=state["other"], weight2=w[1], eps2=eps)
        return {**_views(q), "hidden": hidden}
    weights = [w["handle"] for w in state["weights"]]
    if case["op"] == "linear":
        return mx_linear(state["x"]["handle"], weights[0], out_dtype=TYPES[case["out"]])
    if case["out"] == "mxfp8":
        return _views(mx_linear_swiglu(state["x"]["handle"], *weights, out_format="mxfp8"))
    return mx_linear_swiglu(state["x"]["handle"], *weights, out_dtype=TYPES[case["out"]])


def _views(q):
    return {"codes": q.codes.view(torch.float8_e4m3fn), "scales": q.scales.view(torch.float8_e8m0fnu)}


def run(state):
    if own:
        return _own(state)
    case = state["case"]
    if case["op"] == "quantize":
        values, exponent = _quantize(state["x"].float(), case["format"])
        if case["format"] == "mxfp8":
            return _held(values, exponent)
        back = torch.ldexp(values.view(case["rows"], -1, BLOCK), exponent[..., None]).view(case["rows"], -1)
        return back[:, :case["cols"]].to(torch.bfloat16)
    if case["op"] == "norm":
        dtype, (w, w2), eps = TYPES[case["dtype"]], state["weights"], state["eps"]
        x = state["x"].float()
        if case["form"] == "plain":
            return _held(*_quantize(_normed(x, w.float(), eps), "mxfp8"))
        other = state["other"].float()
        if case["form"] == "added":
            total = (other + x).to(dtype)
            return {**_held(*_quantize(_normed(total.float(), w.float(), eps), "mxfp8")), "sum": total}
        hidden = (other + _normed(x, w.float(), eps)).to(dtype)
        return {**_held(*_quantize(_normed(hidden.float(), w2.float(), eps), "mxfp8")), "hidden": hidden}
    x, *weights = (_values(t["codes"], t["scales"], t["format"], t["rows"]) for t in (state["x"], *state["weights"]))
    y = x @ weights[0].t()
    if case["op"] == "swiglu":
        y = y * torch.sigmoid(y) * (x @ weights[1].t())
        if case["out"] == "mxfp8":
            return _held(*_quantize(y, "mxfp8"))
    return y.to(TYPES[case["out"]])


# ------------------------------------------------------------------------- in 64 bits, apart

def _grid(fmt):
    """The format's magnitudes, ascending: code i stands for grid[i]."""

    if fmt == "mxfp4":
        return [m * 2.0 ** -1 if e == 0 else (2 + m) * 2.0 ** (e - 2) for e in range(4) for m in range(2)]
    return [m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10) for e in range(16) for m in range(8)][:127]


def _exact_quantize(x, fmt):
    """float64 [rows, cols] -> element values [rows, padded], scales [rows, blocks], both float64."""

    rows, cols = x.shape
    grid = torch.tensor(_grid(fmt), dtype=torch.float64, device=x.device)
    blocks = torch.zeros(rows, _padded(cols), dtype=torch.float64, device=x.device)
    blocks[:, :cols] = x
    blocks = blocks.view(rows, -1, BLOCK)
    ratio = blocks.abs().amax(-1) / grid[-1]
    scale = torch.exp2(torch.ceil(torch.log2(ratio)))
    scale = torch.where(ratio > scale, 2 * scale, torch.where(ratio <= scale / 2, scale / 2, scale))  # log2's last bit
    scale = scale.clamp(2.0 ** -127, 2.0 ** 127)
    unit = blocks / scale[..., None]
    # boundary i separates codes i and i + 1; on it, the even one of the two
    middle = (grid[1:] + grid[:-1]) / 2
    middle[1::2] = torch.nextafter(middle[1::2], torch.zeros_like(middle[1::2]))
    values = torch.copysign(grid[torch.bucketize(unit.abs(), middle)], unit)
    return values.view(rows, -1), scale


def _exact_held(x):
    values, scale = _exact_quantize(x, "mxfp8")
    rows, blocks = scale.shape
    tiles = torch.full((-(-rows // 128), blocks // 4, 32, 4, 4), 2.0 ** -127, dtype=torch.float64, device=x.device)
    r = torch.arange(rows, device=x.device)[:, None]
    b = torch.arange(blocks, device=x.device)[None, :]
    tiles[r // 128, b // 4, r % 32, r // 32 % 4, b % 4] = scale
    return {"codes": values, "scales": tiles}


def _exact_operand(t):
    rows, cols = t["rows"], t["cols"]
    grid = torch.tensor(_grid(t["format"]) + [math.nan] * (t["format"] == "mxfp8"), dtype=torch.float64, device="cuda")
    grid = torch.cat((grid, -grid))
    codes = t["codes"].long()
    if t["format"] == "mxfp4":
        codes = torch.stack((codes % 16, codes // 16), dim=-1).view(rows, -1)
    r = torch.arange(rows, device="cuda")[:, None]
    b = torch.arange(codes.shape[1] // BLOCK, device="cuda")[None, :]
    scale = torch.exp2(t["scales"][r // 128, b // 4, r % 32, r // 32 % 4, b % 4].double() - 127)
    return (grid[codes] * scale.repeat_interleave(BLOCK, 1))[:, :cols]


def _exact_norm(x, weight, eps):
    return x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + eps) * weight.double()


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "quantize":
        x = state["x"].double()
        if case["format"] == "mxfp8":
            return _exact_held(x)
        values, scale = _exact_quantize(x, case["format"])
        return (values * scale.repeat_interleave(BLOCK, 1))[:, :case["cols"]]
    if case["op"] == "norm":
        x, other, dtype, eps = state["x"].double(), state["other"].double(), TYPES[case["dtype"]], state["eps"]
        w, w2 = state["weights"]
        if case["form"] == "plain":
            return _exact_held(_exact_norm(x, w, eps))
        if case["form"] == "added":  # the norm is of the sum as it is stored
            return {**_exact_held(_exact_norm((x + other).to(dtype).double(), w, eps)), "sum": x + other}
        hidden = other + _exact_norm(x, w, eps)
        return {**_exact_held(_exact_norm(hidden.to(dtype).double(), w2, eps)), "hidden": hidden}
    x = _exact_operand(state["x"])
    y = x @ _exact_operand(state["weights"][0]).t()
    if case["op"] == "swiglu":
        y = y / (1 + torch.exp(-y)) * (x @ _exact_operand(state["weights"][1]).t())
        if case["out"] == "mxfp8":
            return _exact_held(y)
    return y
