"""Microscaled operators without a GPU: refusals, the container's layout, and the test reference itself."""

from __future__ import annotations

import pytest
import torch

import flashloop_b200 as fl
from flashloop_b200 import _native, build_kernels, mx
from tests import mx_reference as ref


@pytest.fixture(scope="module")
def lib():
    build_kernels.build()
    return _native.load()


@pytest.mark.parametrize("rows,cols,fmt", [(1, 1, "mxfp8"), (128, 128, "mxfp4"), (129, 129, "mxfp8"), (300, 1000, "mxfp4")])
def test_shapes_agree_with_the_library(lib, rows, cols, fmt):
    r, c = mx.codes_shape(rows, cols, fmt)
    assert r * c == lib.fl_mx_codes_bytes(rows, cols, mx.FORMATS[fmt])
    assert torch.Size(mx.scales_shape(rows, cols)).numel() == lib.fl_mx_scales_bytes(rows, cols)
    assert lib.fl_mx_codes_bytes(-1, cols, 0) == lib.fl_mx_codes_bytes(rows, 0, 0) == lib.fl_mx_codes_bytes(rows, cols, 7) == 0


def test_reference_quantiser_on_known_blocks():
    x = torch.zeros(1, 64)
    x[0, :8] = torch.tensor([6.0, 5.0, 3.5, 2.5, 1.75, 1.25, 0.75, 0.25])  # ties go to the even code
    x[0, 32] = 6.5  # past the largest element: the next power of two
    values, byte = ref.quantize(x, "mxfp4")
    assert values[0, :8].tolist() == [6.0, 4.0, 4.0, 2.0, 2.0, 1.0, 1.0, 0.0]
    assert byte[0, :2].tolist() == [127, 128] and values[0, 32].item() == 6.0
    values, byte = ref.quantize(torch.tensor([[448.0] + [float(v) for v in (17, 19, 0.001)]]), "mxfp8")
    assert byte[0, 0] == 127 and values[0, :3].tolist() == [448.0, 16.0, 20.0]
    values, byte = ref.quantize(torch.tensor([[1.0, float("inf")]]), "mxfp8")
    assert byte[0, 0] == 255 and byte[0, 1] == 0 and torch.isnan(values[0, :32]).all()


def test_container_checks():
    codes, scales = torch.zeros(3, 128, dtype=torch.uint8), torch.zeros(1, 1, 32, 4, 4, dtype=torch.uint8)
    t = fl.MXTensor(codes, scales, (3, 100), "mxfp8")
    assert (t.rows, t.cols, t.nbytes()) == (3, 100, 3 * 128 + 512)
    assert t.view(1, 3, 100).shape == (1, 3, 100)
    with pytest.raises(ValueError):
        t.view(2, 3, 100)
    with pytest.raises(ValueError, match="codes"):
        fl.MXTensor(codes, scales, (3, 100), "mxfp4")
    with pytest.raises(ValueError, match="scales"):
        fl.MXTensor(codes, scales[:, :, :16].contiguous(), (3, 100), "mxfp8")
    with pytest.raises(ValueError, match="unknown microscaled format"):
        fl.MXTensor(codes, scales, (3, 100), "int4")
    with pytest.raises(TypeError):
        fl.MXTensor(codes.int(), scales, (3, 100), "mxfp8")
    with pytest.raises(TypeError):
        fl.MXTensor(torch.zeros(128, 3, dtype=torch.uint8).t(), scales, (3, 100), "mxfp8")
    with pytest.raises(ValueError):
        fl.MXTensor(codes, scales, (), "mxfp8")


@pytest.mark.parametrize("rows,cols,fmt", [(1, 1, "mxfp4"), (5, 33, "mxfp4"), (130, 200, "mxfp8"), (300, 257, "mxfp4"), (0, 64, "mxfp8")])
def test_plain_layout_of_a_checkpoint(rows, cols, fmt):
    g = torch.Generator().manual_seed(rows + cols)
    width = -(-cols // 2) if fmt == "mxfp4" else cols
    codes = torch.randint(0, 120, (rows, width), generator=g, dtype=torch.uint8)  # no NaN of e4m3
    scales = torch.randint(100, 150, (rows, -(-cols // 32)), generator=g, dtype=torch.uint8)
    t = fl.MXTensor.from_row_scales(codes, scales, (rows, cols), fmt)
    assert torch.equal(t.row_scales(), scales)
    values = codes.long()
    if fmt == "mxfp4":
        values = torch.stack((values & 15, values >> 4), -1).view(rows, -1)[:, :cols]
    half = 8 if fmt == "mxfp4" else 128
    grid = ref.grid(fmt)
    want = torch.where(values >= half, -1.0, 1.0) * grid[values % half]
    want = want * (2.0 ** (scales.double() - 127)).repeat_interleave(32, 1)[:, :cols]
    assert torch.equal(ref.decode(t.codes, t.scales, fmt, rows, cols), want)
    assert not ref.decode(t.codes, t.scales, fmt, rows, t.codes.shape[1] * (2 if fmt == "mxfp4" else 1))[:, cols:].any()
    assert not ref.scale_bytes(t.scales, rows)[rows:].any()
    with pytest.raises(ValueError, match="scales"):
        fl.MXTensor.from_row_scales(codes, scales[:, :-1], (rows, cols), fmt)


def test_rows_that_no_index_reaches_are_refused():
    wide = torch.zeros(1, dtype=torch.bfloat16).expand(2**32 + 64)  # one element of memory
    with pytest.raises(ValueError, match="columns"):
        _quantize_as_if_on_a_gpu(wide)
    with pytest.raises(ValueError, match="last dimension"):
        fl.MXTensor(torch.zeros(1, 128, dtype=torch.uint8), torch.zeros(1, 1, 32, 4, 4, dtype=torch.uint8), (1, 2**32 + 64), "mxfp8")
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        mx.mx_status("cpu")


def _quantize_as_if_on_a_gpu(x):
    keep, mx._values = mx._values, lambda *tensors: None
    try:
        return mx.mx_quantize(x)
    finally:
        mx._values = keep


def test_refusals_before_the_gpu():
    x = torch.zeros(2, 64)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        fl.mx_quantize(x)
    with pytest.raises(TypeError):
        fl.mx_quantize(x.int())
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        fl.mx_rmsnorm(x, torch.ones(64), 1e-6)
    with pytest.raises(TypeError):
        fl.mx_rmsnorm(x.double(), torch.ones(64), 1e-6)
    weight = fl.MXTensor(torch.zeros(8, 128, dtype=torch.uint8), torch.zeros(1, 1, 32, 4, 4, dtype=torch.uint8), (8, 64), "mxfp8")
    with pytest.raises(TypeError, match="MXTensor"):
        fl.mx_linear(weight, x)
    with pytest.raises(TypeError):
        fl.mx_linear([1.0], weight)
    with pytest.raises(ValueError, match="out_features"):
        fl.mx_linear(weight, weight.view(2, 4, 64))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        fl.mx_linear(weight, weight)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        weight.dequantize()
    with pytest.raises(TypeError):
        weight.dequantize(torch.float64)


def test_c_refusals(lib):
    def last():
        return lib.fl_last_error().decode()

    a = 1 << 20  # an aligned address nothing reads: every call below is refused on the host
    assert lib.fl_mx_quantize(a, 9, 1, 32, 32, 0, a, a, None) == -1 and "type or format" in last()
    assert lib.fl_mx_quantize(a, 0, 1, 32, 32, 2, a, a, None) == -1
    assert lib.fl_mx_quantize(a, 0, 2, 32, 31, 0, a, a, None) == -1 and "bad sizes" in last()
    assert lib.fl_mx_quantize(None, 0, 1, 32, 32, 0, a, a, None) == -1 and "null" in last()
    assert lib.fl_mx_quantize(a, 0, 1, 32, 32, 0, a + 8, a, None) == -1 and "aligned" in last()
    assert lib.fl_mx_quantize(a, 0, 0, 32, 32, 0, None, None, None) == 0
    assert lib.fl_mx_quantize(a, 0, 1 << 30, 1 << 20, 1 << 20, 0, a, a, None) == -1 and "too many" in last()
    assert lib.fl_mx_dequantize(a, a, 0, 1, 32, a, 7, None) == -1
    assert lib.fl_mx_dequantize(a, a, 0, 1, 32, None, 0, None) == -1
    norm = lambda **k: lib.fl_rmsnorm_mx(*{**dict(x=a, addend=None, residual=None, weight=a, eps=1e-6, weight2=None, eps2=0.0,
                                                  dtype=0, rows=1, width=64, format=0, sum_out=None, hidden=None, codes=a,
                                                  scales=a, stream=None), **k}.values())
    assert norm(width=8193) == -1 and "width" in last()
    assert norm(width=0) == -1
    assert norm(weight2=a) == -1 and "go together" in last()
    assert norm(residual=a) == -1 and "residual" in last()
    assert norm(sum_out=a) == -1 and "addend" in last()
    assert norm(x=None) == -1 and norm(codes=a + 4) == -1 and norm(dtype=3) == -1
    assert norm(rows=0, x=None) == 0
    assert lib.fl_mx_linear(a, a, 0, a, a, 1, 4, 64, 64, None, 0, None) == -1 and "out" in last()
    assert lib.fl_mx_linear(a, a, 0, a + 16, a, 1, 4, 64, 64, a, 0, None) == -1 and "32-byte" in last()
    assert lib.fl_mx_linear(a, a, 5, a, a, 1, 4, 64, 64, a, 0, None) == -1 and "format of x" in last()
    assert lib.fl_mx_linear(a, a, 0, a, a, 1, 4, 64, 64, a, 3, None) == -1 and "output type" in last()
    assert lib.fl_mx_linear(a, a, 0, a, a, 1, -1, 64, 64, a, 0, None) == -1
    assert lib.fl_mx_linear(a, a, 0, a, a, 1, 0, 64, 64, a, 0, None) == 0
    assert lib.fl_mx_linear_swiglu(a, a, 0, a, a, a, None, 1, 4, 64, 64, a, 0, 0, None, None) == -1 and "null" in last()
    assert lib.fl_mx_linear_swiglu(a, a, 0, a, a, a, a, 1, 4, 64, 64, a, 0, 4, a, None) == -1 and "output" in last()
    assert lib.fl_mx_status(None, 0, None) == -1


def test_engine_refusals_on_the_host():
    from tests.helpers import tiny_ouro_model

    with pytest.raises(RuntimeError, match="no CPU fallback"):
        fl.FlashLoopEngine(tiny_ouro_model(), validate_model=False, projection_format="mxfp4")
    with pytest.raises(ValueError, match="tensor parallelism"):
        fl.FlashLoopEngine(tiny_ouro_model(), validate_model=False, projection_format="mxfp4", tp_group=object())
