"""The microscaled norm and quantiser on every path: each width's share of threads, each alignment, rows enough
that a CTA takes several, and the scales themselves against the definition."""

from __future__ import annotations

import zlib

import pytest
import torch

import flashloop_b200 as fl
from tests import mx_device_reference as dref

pytestmark = pytest.mark.gpu

BITS = {torch.bfloat16: 8, torch.float16: 11, torch.float32: 24}
HALF_STEP = {"mxfp8": (2.0 ** -4, 2.0 ** -10), "mxfp4": (2.0 ** -2, 2.0 ** -2)}  # of a normal element, of a subnormal one


def _gen(*seed):
    return torch.Generator(device="cuda").manual_seed(zlib.crc32(repr(seed).encode()) & 0x7fffffff)


def _tensor(g, rows, cols, dtype, offset=0):
    """Normal values whose first element lies `offset` elements past an aligned address."""

    flat = torch.empty(rows * cols + offset, dtype=dtype, device="cuda")
    x = flat[offset:].view(rows, cols)
    x.copy_(torch.randn(rows, cols, generator=g, device="cuda"))
    return x


def _check_norm(q, n64, width):
    """float32's norm is within `slack` of the one in 64 bits (a sum of `width` squares, a root and three
    products: 2^-24 * (width + 8), relative), so each block's scale lies between those of its largest value less
    and plus that, and each element within half a step of the scaled value, and the slack."""

    slack = 2.0 ** -24 * (width + 8)
    byte, got = dref.check_container(q)
    blocks = dref.blocks_of(n64)
    amax = blocks.abs().amax(-1)
    low, high = (dref.scale_byte(amax * f, q.format) for f in (1 - slack, 1 + slack))
    assert bool(((byte >= low) & (byte <= high)).all())
    assert float((high != low).double().mean()) < 0.02  # the bytes of nearly all blocks are fixed by this
    scale = dref.powers(byte.device)[byte][..., None]
    value, element = blocks.abs(), (got.view_as(blocks) * scale)
    relative, subnormal = HALF_STEP[q.format]
    bound = torch.maximum(relative * value * (1 + slack), subnormal * scale) + slack * value
    assert bool(((element - blocks).abs() <= bound).all())


def _norm64(s, w, eps):
    s = s.double()
    return w.double() * s * torch.rsqrt(s.square().mean(-1, keepdim=True) + eps)


def _check_forms(rows, width, dtype, fmt, offset):
    g = _gen(rows, width, str(dtype), offset)
    x, a, r = (_tensor(g, rows, width, dtype, offset) for _ in range(3))
    w, w2 = ((1 + 0.1 * _tensor(g, 1, width, torch.float32)[0]).to(dtype) for _ in range(2))
    q, none, _ = fl.mx_rmsnorm(x, w, 1e-6, format=fmt)
    assert none is None
    _check_norm(q, _norm64(x, w, 1e-6), width)
    q, _, total = fl.mx_rmsnorm(x, w, 1e-6, addend=a, want_sum=True, format=fmt)
    assert torch.equal(total, (x.float() + a.float()).to(dtype))
    _check_norm(q, _norm64(total, w, 1e-6), width)
    for residual, addend in ((r, None), (r, a), (None, None)):
        q, hidden, total = fl.mx_rmsnorm(x, w, 1e-6, residual=residual, weight2=w2, eps2=1e-5, addend=addend,
                                         want_sum=addend is not None, format=fmt)
        s = x if addend is None else total
        n = _norm64(s, w, 1e-6)
        want = n if residual is None else residual.double() + n
        slack = 2.0 ** -24 * (width + 8)
        bound = 2.0 ** -BITS[dtype] * want.abs() + slack * (n.abs() + want.abs()) + 2.0 ** -25
        assert bool(((hidden.double() - want).abs() <= bound).all())
        _check_norm(q, _norm64(hidden, w2, 1e-5), width)


# rows: past those that all CTAs of the device take at once (16 to an SM at most), and not a multiple of anything
WIDTHS = [(96, 40011), (200, 20011), (384, 11003), (1000, 6007), (2000, 5003), (2560, 3001), (6000, 2503)]


@pytest.mark.parametrize("rows_of", ["many", "few"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("width,rows", WIDTHS)
def test_norm_of_aligned_rows(width, rows, dtype, rows_of):
    _check_forms(rows if rows_of == "many" else 37, width, dtype, "mxfp8", 0)


@pytest.mark.parametrize("less", [1, 2, 6])  # two bytes, four and four of a 16-bit type
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("width,rows", WIDTHS)
def test_norm_of_ragged_widths(width, rows, dtype, less):
    _check_forms(rows, width - less, dtype, "mxfp8", 0)


@pytest.mark.parametrize("offset", [1, 2, 4])
@pytest.mark.parametrize("width,rows", WIDTHS)
def test_norm_of_bases_off_the_alignment_of_their_rows(width, rows, offset):
    _check_forms(rows, width, torch.float16 if offset == 2 else torch.bfloat16, "mxfp8", offset)


@pytest.mark.parametrize("less", [0, 1, 2])
@pytest.mark.parametrize("width,rows", WIDTHS)
def test_norm_to_four_bits(width, rows, less):
    _check_forms(rows, width - less, torch.bfloat16, "mxfp4", 0)


@pytest.mark.parametrize("width", [1, 8, 31, 33, 127, 128, 129, 255, 256, 257, 511, 512, 513, 1023, 1024, 1025, 2047, 2048,
                                   2049, 4095, 4096, 4097, 8191, 8192])
def test_norm_at_the_ends_of_the_widths(width):
    for rows in (1, 31, 33, 129):
        _check_forms(rows, width, torch.bfloat16, "mxfp8", 0)


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("cols,offset", [(704, 0), (704, 1), (702, 0), (704, 2), (701, 0), (701, 3)])
def test_many_rows_quantised_and_back(cols, offset, dtype, fmt):
    """Steps enough that a thread takes several: 16-, four- and two-byte loads and stores."""

    rows = 20011
    g = _gen(cols, offset, str(dtype), fmt)
    x = _tensor(g, rows, cols, dtype, offset)
    x *= torch.exp2(torch.randint(-6, 7, (rows, 1), generator=g, device="cuda").float()).to(dtype)
    for t in (x, x[:, :cols - 64], x[::2]):  # rows further apart than they are long
        q = fl.mx_quantize(t, fmt)
        dref.check_quantized(q, t)
        byte, e = dref.check_container(q)
        want = (e.view(q.rows, -1, 32) * dref.powers(e.device)[byte][..., None]).view(q.rows, -1)[:, :q.cols]
        for out in (torch.bfloat16, torch.float16, torch.float32):
            assert torch.equal(q.dequantize(out), want.float().to(out))  # both roundings: float32 holds the values


def test_rows_behind_the_last_one_stay_as_they_are():
    """A result that lies in a larger buffer: nothing past its rows is written."""

    from flashloop_b200 import _native

    lib, stream = _native.load(), torch.cuda.current_stream().cuda_stream
    for rows, cols in ((5, 300), (20011, 701)):
        g = _gen("behind", rows)
        x = _tensor(g, rows, cols, torch.bfloat16)
        one = torch.ones(cols, device="cuda", dtype=torch.bfloat16)
        steps, tiles = -(-cols // 128), -(-rows // 128)
        codes = torch.full((rows * steps * 128 + 4096,), 0xA5, dtype=torch.uint8, device="cuda")
        scales = torch.full((tiles * steps * 512 + 4096,), 0xA5, dtype=torch.uint8, device="cuda")
        hidden = torch.full((rows * cols + 2048,), 7.0, dtype=torch.bfloat16, device="cuda")
        assert lib.fl_mx_quantize(x.data_ptr(), 0, rows, cols, cols, 0, codes.data_ptr(), scales.data_ptr(), stream) == 0
        assert bool((codes[-4096:] == 0xA5).all()) and bool((scales[-4096:] == 0xA5).all())
        assert lib.fl_rmsnorm_mx(x.data_ptr(), None, None, one.data_ptr(), 1e-6, one.data_ptr(), 1e-6, 0, rows, cols, 0, None,
                                 hidden.data_ptr(), codes.data_ptr(), scales.data_ptr(), stream) == 0
        assert bool((codes[-4096:] == 0xA5).all()) and bool((scales[-4096:] == 0xA5).all())
        assert bool((hidden[-2048:] == 7).all())
        q = fl.mx_rmsnorm(x, one, 1e-6, weight2=one, eps2=1e-6)[0]
        assert torch.equal(codes[:-4096].view_as(q.codes), q.codes) and torch.equal(scales[:-4096].view_as(q.scales), q.scales)
