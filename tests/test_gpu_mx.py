"""The microscaled operators against their definition in 64 bits."""

from __future__ import annotations

import copy
import math
import threading
import zlib

import pytest
import torch

import flashloop_b200 as fl
from flashloop_b200.mx import codes_shape, mx_status, scales_shape
from tests import mx_reference as ref

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
ELEMENT_HALF_STEP = {"mxfp8": 2.0 ** -4, "mxfp4": 2.0 ** -2}  # of a normal element, relative
SMALLEST_HALF = {"mxfp8": 2.0 ** -10, "mxfp4": 2.0 ** -2}      # of a subnormal element, in scales


def _gen(*seed):
    return torch.Generator(device="cuda").manual_seed(zlib.crc32(repr(seed).encode()) & 0x7fffffff)


def _random(rows, cols, dtype, *seed):
    """Normal values over blocks of very different sizes."""

    g = _gen(rows, cols, *seed)
    x = torch.randn(rows, cols, generator=g, device="cuda")
    return (x * torch.exp2(torch.randint(-6, 7, (rows, cols), generator=g, device="cuda").float())).to(dtype)


def _check_exact(q, x, fmt):
    """Codes and scales bit for bit; padding zero."""

    rows, cols = x.shape
    want, want_byte = ref.quantize(x, fmt)
    byte = ref.scale_bytes(q.scales, rows)
    assert torch.equal(byte[:rows], want_byte) and not byte[rows:].any()
    padded = want.shape[1]
    got = ref.decode(q.codes, q.scales, fmt, rows, padded)
    torch.testing.assert_close(got, want, rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 32), (3, 31), (2, 33), (17, 128), (128, 129), (129, 1000), (5, 2048), (300, 264)])
def test_quantize_is_exact(rows, cols, dtype, fmt):
    x = _random(rows, cols, dtype, fmt)
    q = fl.mx_quantize(x, fmt)
    assert q.shape == (rows, cols) and q.format == fmt
    _check_exact(q, x, fmt)
    for out in (torch.float32, torch.bfloat16, torch.float16):
        want = ref.decode(q.codes, q.scales, fmt, rows, cols).to(torch.float32).to(out)
        assert torch.equal(q.dequantize(out).cpu(), want)


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
def test_quantize_boundaries(fmt):
    """Ties, largest elements, powers of two, zeros, subnormals, the ends of the scale's range."""

    g = ref.grid(fmt)
    middles = (g[1:] + g[:-1]) / 2
    points = torch.cat((g, middles, torch.nextafter(middles.float(), torch.tensor(0.0)).double(),
                        torch.nextafter(middles.float(), torch.tensor(1e9)).double()))
    rows = []
    for exponent in (-130, -127, -126, -100, -1, 0, 1, 60, 118):
        for sign in (1, -1):
            block = torch.zeros(-(-len(points) // 31) * 32, dtype=torch.float64).view(-1, 32)
            block[:, 0] = g[-1]  # fixes the scale
            block[:, 1:] = torch.nn.functional.pad(points, (0, block.shape[0] * 31 - len(points))).view(-1, 31)
            rows.append(sign * block.flatten() * 2.0 ** exponent)
    x = torch.stack(rows).float().cuda()
    _check_exact(fl.mx_quantize(x, fmt), x, fmt)
    top = 3.4e38
    edge = torch.tensor([[0.0] * 32, [-0.0] * 32, [1e-45] * 32, [top] * 32, [g[-1].item()] * 32,
                         [math.nextafter(g[-1].item(), 1e9) * (1 + 2 ** -23)] * 32], device="cuda")
    _check_exact(fl.mx_quantize(edge, fmt), edge, fmt)


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
def test_quantize_keeps_what_is_not_finite_in_its_block(fmt):
    x = _random(5, 300, torch.float32, fmt)
    x[1, 40], x[3, 0], x[4, 299] = float("nan"), float("inf"), float("-inf")
    q = fl.mx_quantize(x, fmt)
    _check_exact(q, x, fmt)
    bad = torch.isnan(q.dequantize(torch.float32))
    want = torch.zeros_like(bad)
    want[1, 32:64] = want[3, :32] = want[4, 288:] = True
    assert torch.equal(bad, want)


def test_quantize_strides_and_leading_dimensions():
    base = _random(40, 500, torch.bfloat16, "strides")
    for x in (base[:, 3:203], base[::2, :128], base[:, :256].view(8, 5, 256), base.t()[:64], base[:, ::2],
              base[:1].expand(6, 500), base[5, :77], base[:0]):
        q = fl.mx_quantize(x, "mxfp8")
        flat = x.reshape(-1, x.shape[-1])
        assert q.shape == tuple(x.shape)
        if flat.numel():
            _check_exact(q, flat, "mxfp8")
        assert q.dequantize().shape == x.shape
    assert torch.equal(fl.mx_quantize(base, "mxfp4").view(4, 10, 500).dequantize(),
                       fl.mx_quantize(base, "mxfp4").dequantize().view(4, 10, 500))


def _norm64(x, w, eps):
    return w.double() * x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)


def _check_codes(q, n64, fmt):
    """Every element within half a step of the norm in 64 bits (and float32's error of the norm), under a scale at
    most one power of two off the definition's; nearly all codes are the definition's own."""

    rows, width = n64.shape
    got = q.dequantize(torch.float32).double()
    blocks = torch.nn.functional.pad(n64, (0, -width % 32)).view(rows, -1, 32)
    scale = (2 * blocks.abs().amax(-1) / ref.LARGEST[fmt]).repeat_interleave(32, 1)[:, :width]
    # norm in float32: the sum of `width` squares, a root and three products, below 2^-24 * (width + 8)
    slack = n64.abs() * 2.0 ** -24 * (width + 8)
    bound = torch.maximum(ELEMENT_HALF_STEP[fmt] * n64.abs(), SMALLEST_HALF[fmt] * 2 * scale) + slack + 1e-38
    assert bool(((got - n64).abs() <= bound).all()), float(((got - n64).abs() - bound).max())
    want, _ = ref.quantize(n64.float(), fmt)
    # a code differs where float32 puts the value on the other side of a boundary: a share of about
    # 2 * slack / step, below 1e-3 for the widths here
    assert float((got.cpu() != want[:, :width]).double().mean()) <= 1e-3 + 1.0 / n64.numel()
    byte = ref.scale_bytes(q.scales, rows)
    assert not byte[rows:].any()


@pytest.mark.parametrize("dtype,fmt", [(torch.bfloat16, "mxfp8"), (torch.float16, "mxfp8"), (torch.float32, "mxfp8"),
                                       (torch.bfloat16, "mxfp4")])
@pytest.mark.parametrize("rows,width", [(1, 1), (1, 2048), (16, 2048), (130, 96), (3, 1001), (2, 8192), (257, 64), (7, 5632)])
def test_norm(rows, width, dtype, fmt):
    g = _gen(rows, width)
    x = torch.randn(rows, width, generator=g, device="cuda").to(dtype)
    a, r = (torch.randn(rows, width, generator=g, device="cuda").to(dtype) for _ in range(2))
    w1, w2 = ((1 + 0.1 * torch.randn(width, generator=g, device="cuda")).to(dtype) for _ in range(2))

    q, hidden, total = fl.mx_rmsnorm(x, w1, 1e-6, format=fmt)
    assert hidden is None and total is None
    _check_codes(q, _norm64(x.double(), w1, 1e-6), fmt)

    q, _, total = fl.mx_rmsnorm(x, w1, 1e-6, addend=a, want_sum=True, format=fmt)
    assert torch.equal(total, (x.float() + a.float()).to(dtype))
    _check_codes(q, _norm64(total.double(), w1, 1e-6), fmt)
    same, _, none = fl.mx_rmsnorm(x, w1, 1e-6, addend=a, format=fmt)
    assert none is None and torch.equal(same.codes, q.codes) and torch.equal(same.scales, q.scales)

    for residual, addend in ((r, None), (None, a), (r, a)):
        q, hidden, _ = fl.mx_rmsnorm(x, w1, 1e-6, residual=residual, weight2=w2, eps2=1e-5, addend=addend, format=fmt)
        s = x.double() if addend is None else (x.float() + a.float()).to(dtype).double()
        n = _norm64(s, w1, 1e-6)
        want = n if residual is None else residual.double() + n
        # rounded once to the stored type, after float32's own error
        bound = HALF_STEP[dtype] * want.abs() + 2.0 ** -24 * (width + 8) * (n.abs() + want.abs()) + 2.0 ** -25
        assert bool(((hidden.double() - want).abs() <= bound).all())
        _check_codes(q, _norm64(hidden.double(), w2, 1e-5), fmt)


def test_norm_takes_strided_rows_and_leading_dimensions():
    base = _random(12, 600, torch.bfloat16, "strided")
    w = torch.ones(300, device="cuda", dtype=torch.bfloat16)
    x, r = base[:, ::2], base[:1, 300:].expand(12, 300)
    q, hidden, _ = fl.mx_rmsnorm(x, w, 1e-6, residual=r, weight2=w, eps2=1e-6)
    same, other, _ = fl.mx_rmsnorm(x.contiguous().view(3, 4, 300), w, 1e-6, residual=r.contiguous().view(3, 4, 300), weight2=w,
                                   eps2=1e-6)
    assert same.shape == other.shape == (3, 4, 300) and torch.equal(other.view(12, 300), hidden)
    assert torch.equal(q.codes, same.codes) and torch.equal(q.scales, same.scales)
    one = fl.mx_rmsnorm(x[0], w, 1e-6)[0]
    assert one.shape == (300,) and torch.equal(one.codes[0], fl.mx_rmsnorm(x, w, 1e-6)[0].codes[0])
    empty, nothing, _ = fl.mx_rmsnorm(x[:0], w, 1e-6, weight2=w)
    assert empty.shape == nothing.shape == (0, 300)


def test_copies_hold_their_own_tensors():
    q = fl.mx_quantize(_random(5, 200, torch.bfloat16, "copy"), "mxfp4")
    twin = copy.deepcopy(q)
    want = q.dequantize()
    q.codes.zero_()
    assert torch.equal(twin.dequantize(), want) and not q.dequantize().any()


def test_norm_of_rows_that_are_zero_or_not_finite():
    x = _random(4, 256, torch.bfloat16, "norm")
    x[1] = 0
    x[2, 17] = float("nan")
    w = torch.ones(256, device="cuda", dtype=torch.bfloat16)
    y = fl.mx_rmsnorm(x, w, 1e-6)[0].dequantize()
    assert not y[1].any() and torch.isnan(y[2]).all() and torch.isfinite(y[[0, 3]]).all()
    narrow = fl.mx_rmsnorm(x[:, :40].contiguous(), w[:40], 1e-6)[0]  # row 2 holds the NaN: its padding stays zero
    byte = ref.scale_bytes(narrow.scales, 4)
    assert byte[2].tolist() == [255, 255, 0, 0] and not byte[4:].any() and not narrow.codes[:, 40:].any()


def _operands(rows, cols, features, x_format, w_format, weights=1):
    x = fl.mx_quantize(_random(rows, cols, torch.float32, "x"), x_format)
    ws = [fl.mx_quantize(_random(features, cols, torch.float32, "w", i) * cols ** -0.5, w_format) for i in range(weights)]
    return x, ws


def _product64(x, w):
    """The product in 64 bits and the sum of its terms' magnitudes."""

    a = ref.decode(x.codes, x.scales, x.format, x.rows, x.cols).cuda()
    b = ref.decode(w.codes, w.scales, w.format, w.rows, w.cols).cuda()
    return a @ b.t(), a.abs() @ b.abs().t()


def _accumulation(cols):
    """Relative to the sum of magnitudes: `cols` float32 additions, each off by a last place at most."""

    return 2.0 ** -23 * (cols + 4)


SIZES = [(1, 1, 1), (1, 32, 128), (2, 128, 130), (16, 2048, 2048), (15, 1000, 1337), (17, 129, 64), (33, 300, 257),
         (64, 512, 384), (65, 4096, 256), (128, 128, 127), (129, 640, 513), (300, 2048, 640), (1000, 160, 4999),
         (2500, 264, 3000), (3, 20000, 200), (19500, 96, 100), (9800, 300, 200)]


@pytest.mark.parametrize("rows,cols,features", SIZES)
@pytest.mark.parametrize("x_format,w_format", [("mxfp8", "mxfp4"), ("mxfp8", "mxfp8"), ("mxfp4", "mxfp4"), ("mxfp4", "mxfp8")])
def test_linear(rows, cols, features, x_format, w_format):
    x, (w,) = _operands(rows, cols, features, x_format, w_format)
    want, magnitude = _product64(x, w)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        got = fl.mx_linear(x, w, out_dtype=dtype)
        assert got.shape == (rows, features) and got.dtype == dtype
        bound = HALF_STEP[dtype] * want.abs() + _accumulation(cols) * magnitude
        if dtype == torch.float16:
            bound += 2.0 ** -25  # its subnormals
        error = (got.double() - want).abs()
        assert bool((error <= bound).all()), (dtype, float(error.max()), float((error - bound).max()))
    assert mx_status() == 0


@pytest.mark.parametrize("rows,cols,features", SIZES)
@pytest.mark.parametrize("x_format,w_format", [("mxfp8", "mxfp4"), ("mxfp4", "mxfp8"), ("mxfp4", "mxfp4")])
def test_linear_swiglu(rows, cols, features, x_format, w_format):
    x, (gate, up) = _operands(rows, cols, features, x_format, w_format, weights=2)
    g, g_magnitude = _product64(x, gate)
    u, u_magnitude = _product64(x, up)
    s = torch.sigmoid(g)
    want = g * s * u
    dg, du = _accumulation(cols) * g_magnitude, _accumulation(cols) * u_magnitude
    # the derivative of silu is within [-0.1, 1.1]; expf and the divisions are within a few last places
    slack = 1.1 * dg * (u.abs() + du) + (g * s).abs() * du + 2.0 ** -20 * want.abs() + 1e-38
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        got = fl.mx_linear_swiglu(x, gate, up, out_dtype=dtype)
        bound = HALF_STEP[dtype] * want.abs() + slack + (2.0 ** -25 if dtype == torch.float16 else 0)
        fits = want.abs() < 60000 if dtype == torch.float16 else torch.ones_like(want, dtype=torch.bool)
        error = (got.double() - want).abs()
        assert bool((error <= bound)[fits].all()), (dtype, float(error[fits].max()))
    for fmt in ("mxfp8", "mxfp4"):
        q = fl.mx_linear_swiglu(x, gate, up, out_format=fmt)
        assert q.shape == (rows, features) and q.format == fmt
        # what the float32 result quantises to, bit for bit: the same sums, the same activation
        direct = fl.mx_quantize(fl.mx_linear_swiglu(x, gate, up, out_dtype=torch.float32), fmt)
        assert torch.equal(q.codes, direct.codes) and torch.equal(q.scales, direct.scales)
    assert mx_status() == 0


def test_linear_quantises_a_plain_tensor_and_keeps_leading_dimensions():
    x = _random(6, 200, torch.bfloat16, "plain").view(2, 3, 200)
    w = fl.mx_quantize(_random(70, 200, torch.bfloat16, "w"), "mxfp4")
    got = fl.mx_linear(x, w)
    assert got.shape == (2, 3, 70)
    assert torch.equal(got, fl.mx_linear(fl.mx_quantize(x, "mxfp8"), w))
    assert fl.mx_linear(x[:0], w).shape == (0, 3, 70)
    assert fl.mx_linear_swiglu(x[:0], w, w, out_format="mxfp8").shape == (0, 3, 70)


@pytest.mark.parametrize("rows", [5, 200, 19500])
@pytest.mark.parametrize("x_format", ["mxfp8", "mxfp4"])
def test_linear_blocks_that_are_not_finite(rows, x_format):
    x = torch.randn(rows, 300, generator=_gen("nan", rows), device="cuda")
    w = torch.randn(140, 300, generator=_gen("nan", rows + 1), device="cuda")
    x[3, 100] = float("inf")
    w[131, 299] = float("nan")
    y = fl.mx_linear(fl.mx_quantize(x, x_format), fl.mx_quantize(w, "mxfp4"))
    bad = torch.zeros(rows, 140, dtype=torch.bool, device="cuda")
    bad[3], bad[:, 131] = True, True
    assert torch.equal(torch.isnan(y), bad)


def test_linear_of_extreme_scales():
    """Scales near both ends of their range whose products are ordinary, and zero rows."""

    for rows, x_format in ((20, "mxfp8"), (20, "mxfp4"), (19500, "mxfp8"), (19500, "mxfp4")):
        x = torch.randn(rows, 256, generator=_gen("extreme"), device="cuda")
        w = torch.randn(30, 256, generator=_gen("extreme", 1), device="cuda")
        small, large = fl.mx_quantize(x * 2.0 ** -100, x_format), fl.mx_quantize(w * 2.0 ** 110, "mxfp4")
        plain = fl.mx_linear(fl.mx_quantize(x, x_format), fl.mx_quantize(w, "mxfp4"), out_dtype=torch.float32)
        assert torch.equal(fl.mx_linear(small, large, out_dtype=torch.float32), plain * 2.0 ** 10)
    zero = fl.mx_linear(torch.zeros_like(x), fl.mx_quantize(w, "mxfp4"))
    assert not zero.any()


def test_operators_together_as_a_layer_uses_them():
    """norm -> gate/up -> down, each in the form the previous one leaves, against float64 over the same weights."""

    rows, hidden, inner = 16, 256, 640
    g = _gen("together")
    stream = torch.randn(rows, 1, hidden, generator=g, device="cuda").to(torch.bfloat16)
    delta = torch.randn(rows, 1, hidden, generator=g, device="cuda").to(torch.bfloat16)
    n1, n2 = ((1 + 0.1 * torch.randn(hidden, generator=g, device="cuda")).to(torch.bfloat16) for _ in range(2))
    gate, up, down = (fl.mx_quantize(torch.randn(*s, generator=g, device="cuda") * s[1] ** -0.5, "mxfp4")
                      for s in ((inner, hidden), (inner, hidden), (hidden, inner)))
    q, new_stream, _ = fl.mx_rmsnorm(delta, n1, 1e-6, residual=stream, weight2=n2, eps2=1e-6)
    inner_q = fl.mx_linear_swiglu(q, gate, up, out_format="mxfp8")
    y = fl.mx_linear(inner_q, down)
    assert y.shape == (rows, 1, hidden) and y.dtype == torch.bfloat16
    w = [t.dequantize(torch.float32).double() for t in (gate, up, down)]
    x = _norm64(new_stream.double(), n2, 1e-6)
    a = torch.nn.functional.silu(x @ w[0].t()) * (x @ w[1].t())
    want = a @ w[2].t()
    # two roundings of e4m3 elements, 2^-4 at most and about 0.026 each in the root mean square
    assert float((y.double() - want).norm() / want.norm()) < 2 * 2.0 ** -4
    # and step by step against the values each stage received
    exact = inner_q.dequantize(torch.float32).double() @ w[2].t()
    assert float((y.double() - exact).norm() / exact.norm()) < 2.0 ** -8


def test_captured_calls_replay_on_new_values():
    g = _gen("graph")
    x = torch.randn(16, 512, generator=g, device="cuda").to(torch.bfloat16)
    weight = torch.ones(512, device="cuda", dtype=torch.bfloat16)
    w = fl.mx_quantize(torch.randn(384, 512, generator=g, device="cuda"), "mxfp4")

    def step():
        q = fl.mx_rmsnorm(x, weight, 1e-6)[0]
        return fl.mx_linear(fl.mx_linear_swiglu(q, w, w, out_format="mxfp8"), down)

    down = fl.mx_quantize(torch.randn(100, 384, generator=g, device="cuda"), "mxfp4")
    step()
    graphs, outs = [], []
    torch.cuda.synchronize()
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step())
        graphs.append(graph)
    for i in range(3):
        x.copy_(torch.randn(16, 512, generator=g, device="cuda"))
        for graph in graphs:
            graph.replay()
        want = step()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


def test_two_streams_and_repeats_agree():
    """The same products on two streams at once, many times: every result has the same bits."""

    x, (w,) = _operands(16, 2048, 1024, "mxfp8", "mxfp4")
    big_x, _ = _operands(700, 2048, 1, "mxfp8", "mxfp4")
    want, big = fl.mx_linear(x, w, out_dtype=torch.float32), fl.mx_linear(big_x, w, out_dtype=torch.float32)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for i in range(20):
        for s, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got.append((fl.mx_linear(x, w, out_dtype=torch.float32), want) if (i + s) % 2 else
                           (fl.mx_linear(big_x, w, out_dtype=torch.float32), big))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in got)
    assert mx_status() == 0


def test_chains_without_waiting():
    """The kernels of a chain overlap and its buffers are reused at once: the results are those of the same
    calls made one by one, for few rows and for many, and with other kernels in between."""

    for rows, width in ((16, 1024), (3, 640), (2000, 512)):
        g = _gen("chain", rows)
        inputs = [torch.randn(rows, width, generator=g, device="cuda").to(torch.bfloat16) for _ in range(6)]
        weight = torch.ones(width, device="cuda", dtype=torch.bfloat16)
        w = [torch.randn(width, width, generator=g, device="cuda") * width ** -0.5 for _ in range(3)]
        x = torch.empty_like(inputs[0])

        def chain(values, wait):
            x.copy_(values)
            done = lambda t: torch.cuda.synchronize() if wait else None
            gate, up, down = (fl.mx_quantize(t, "mxfp4") for t in w)  # used by the very next kernels
            done(gate)
            out = x
            for _ in range(4):
                q, hidden, _ = fl.mx_rmsnorm(out, weight, 1e-6, residual=x, weight2=weight, eps2=1e-6)
                done(q)
                inner = fl.mx_linear_swiglu(q, gate, up, out_format="mxfp8")
                done(inner)
                out = fl.mx_linear(inner, down)
                done(out)
                out = out + hidden  # a kernel of another kind
                done(out)
            x.zero_()  # written while the chain may still run, were it not in order
            return out

        want = [chain(v, True) for v in inputs]
        torch.cuda.synchronize()
        for _ in range(5):
            got = [chain(v, False) for v in inputs]
            assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("captured", [False, True])
def test_inputs_from_another_stream(captured):
    """What another stream writes before an event is there for the call after it, although the kernel may
    start before the one in front of it in its own stream has ended."""

    g = _gen("stream")
    w = fl.mx_quantize(torch.randn(256, 512, generator=g, device="cuda"), "mxfp4")
    x, fresh = (torch.randn(16, 512, generator=g, device="cuda") for _ in range(2))
    old, held = x.clone(), fl.mx_quantize(torch.randn(16, 512, generator=g, device="cuda"))
    want = fl.mx_linear(fl.mx_quantize(fresh), w)
    side = torch.cuda.Stream()

    def step():
        main = torch.cuda.current_stream()
        fl.mx_linear(held, w)
        side.wait_stream(main)
        with torch.cuda.stream(side):
            torch.cuda._sleep(2_000_000)  # about a millisecond
            x.copy_(fresh)
            back = fl.mx_quantize(x)
        fl.mx_linear(held, w)  # runs meanwhile
        main.wait_stream(side)
        return fl.mx_linear(fl.mx_quantize(x), w), fl.mx_linear(back, w)

    run = step
    if captured:
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        run = lambda: (graph.replay(), outs)[1]
    for _ in range(3):
        x.copy_(old)
        torch.cuda.synchronize()
        a, b = run()
        torch.cuda.synchronize()
        assert torch.equal(a, want) and torch.equal(b, want)


def test_long_rows():
    """More steps of K than a wait has tries, in both kernels."""

    for rows, cols, features, x_format, one in ((2, 400_000, 130, "mxfp4", 0x22), (200 * 192, 140_000, 130, "mxfp8", 0x38),
                                                (200 * 192, 140_000, 130, "mxfp4", 0x22)):
        x = fl.MXTensor(torch.full(codes_shape(rows, cols, x_format), one, dtype=torch.uint8, device="cuda"),
                        torch.full(scales_shape(rows, cols), 127, dtype=torch.uint8, device="cuda"), (rows, cols), x_format)
        w = fl.mx_quantize(torch.ones(features, cols, device="cuda", dtype=torch.bfloat16), "mxfp4")
        y = fl.mx_linear(x, w, out_dtype=torch.float32)  # ones times ones, exact in float32
        assert bool((y == cols).all())
        del x, w, y
    assert mx_status() == 0


def test_calls_from_several_threads():
    g = _gen("threads")
    w = fl.mx_quantize(torch.randn(512, 512, generator=g, device="cuda"), "mxfp4")
    inputs = [torch.randn(rows, 512, generator=g, device="cuda") for rows in (1, 16, 90, 9000)]
    want = [fl.mx_linear(x, w) for x in inputs]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(30):
                if not torch.equal(fl.mx_linear(inputs[i], w), want[i]):
                    wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong and mx_status() == 0


def test_gradients_are_refused():
    x = torch.randn(2, 64, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError, match="no gradient"):
        fl.mx_quantize(x)
    with pytest.raises(RuntimeError, match="no gradient"):
        fl.mx_rmsnorm(x, torch.ones(64, device="cuda"), 1e-6)
    with torch.no_grad():
        fl.mx_quantize(x)


def test_refusals():
    x = torch.randn(2, 64, device="cuda")
    w = fl.mx_quantize(torch.randn(8, 64, device="cuda"), "mxfp4")
    other = fl.mx_quantize(torch.randn(8, 96, device="cuda"), "mxfp4")
    with pytest.raises(ValueError, match="do not match"):
        fl.mx_linear(x, other)
    with pytest.raises(ValueError, match="agree"):
        fl.mx_linear_swiglu(x, w, fl.mx_quantize(torch.randn(9, 64, device="cuda"), "mxfp4"))
    with pytest.raises(ValueError, match="agree"):
        fl.mx_linear_swiglu(x, w, fl.mx_quantize(torch.randn(8, 64, device="cuda"), "mxfp8"))
    with pytest.raises(TypeError):
        fl.mx_linear(x, w, out_dtype=torch.float64)
    with pytest.raises(ValueError, match="unknown microscaled format"):
        fl.mx_quantize(x, "int8")
    with pytest.raises(ValueError, match="column"):
        fl.mx_quantize(x[:, :0])
    with pytest.raises(ValueError, match="residual"):
        fl.mx_rmsnorm(x, torch.ones(64, device="cuda"), 1e-6, residual=x)
    with pytest.raises(ValueError, match="addend"):
        fl.mx_rmsnorm(x, torch.ones(64, device="cuda"), 1e-6, want_sum=True)
    with pytest.raises(ValueError, match="weight"):
        fl.mx_rmsnorm(x, torch.ones(63, device="cuda"), 1e-6)
    with pytest.raises(ValueError, match="weight"):
        fl.mx_rmsnorm(x, torch.ones(64, device="cuda", dtype=torch.bfloat16), 1e-6)
    with pytest.raises(ValueError, match="wide"):
        fl.mx_rmsnorm(torch.zeros(1, 8193, device="cuda"), torch.ones(8193, device="cuda"), 1e-6)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        fl.mx_rmsnorm(x, torch.ones(64), 1e-6)
