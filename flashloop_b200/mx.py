"""Microscaled operands: quantisation, the norm that writes them, and the projections that take them
(``csrc/fl_mx.cu``, ``csrc/fl_mx_norm.cu``, ``csrc/fl_mx_linear.cu``).

Thirty-two consecutive elements of a row share a power-of-two scale; the elements are e4m3
(``"mxfp8"``) or e2m1 (``"mxfp4"``).  The reference's projections are bfloat16
(flashloop/weights.py:74-117); these are what ``FlashLoopEngine(projection_format=...)`` runs
instead.  Inference only: no gradient is recorded, and inputs that require one, or carry a tangent, are refused.
"""

from __future__ import annotations

import ctypes as C
import math

import torch
from torch.autograd import forward_ad

from . import _native


def _stream_handle(index: int) -> int:
    return torch.cuda.current_stream(index).cuda_stream


# the handle alone where this PyTorch has that call: a Stream object costs 2 us
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _stream_handle)

FORMATS = {"mxfp8": 0, "mxfp4": 1}
_CODE_TYPES = ("float8_e4m3fn", "float4_e2m1fn_x2")  # by format code, where this PyTorch has them
MAX_NORM_WIDTH = 8192
MAX_COLUMNS = 2**31 - 256  # of a row: the kernels index a row in 32 bits


def _format_code(name: str) -> int:
    code = FORMATS.get(name) if isinstance(name, str) else None
    if code is None:
        raise ValueError(f"unknown microscaled format {name!r}: use one of {sorted(FORMATS)}")
    return code


def codes_shape(rows: int, cols: int, format: str) -> tuple[int, int]:
    """Shape of the codes of a [rows, cols] operand."""

    steps = -(-cols // 128)
    return rows, steps * (128 if _format_code(format) == 0 else 64)


def scales_shape(rows: int, cols: int) -> tuple[int, int, int, int, int]:
    """Shape of its scales: the scale of (row, k) is at [row // 128, k // 128, row % 32, row // 32 % 4, k // 32 % 4]."""

    return -(-rows // 128), -(-cols // 128), 32, 4, 4


class MXTensor:
    """A tensor whose last dimension is held in a microscaled format.

    ``codes`` uint8 (:func:`codes_shape`, elements past the last column zero) and ``scales`` uint8
    (:func:`scales_shape`, rows and blocks past the last zero; byte b stands for 2^(b - 127), 255 for NaN) of
    ``shape``, whose leading dimensions are the rows.  The tensors are held, not copied."""

    __slots__ = ("shape", "format", "rows", "cols", "device", "codes_ptr", "scales_ptr", "_code", "_codes", "_scales",
                 "_both")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, shape, format: str) -> None:
        shape = tuple(int(v) for v in shape)
        if not shape or min(shape) < 0 or not 0 < shape[-1] <= MAX_COLUMNS:
            raise ValueError(f"a microscaled tensor needs a last dimension of 1 to {MAX_COLUMNS}")
        rows = math.prod(shape[:-1])
        self._code = _format_code(format)
        for t, want, name in ((codes, codes_shape(rows, shape[-1], format), "codes"),
                              (scales, scales_shape(rows, shape[-1]), "scales")):
            if t.dtype != torch.uint8 or not t.is_contiguous():
                raise TypeError(f"{name} must be contiguous uint8")
            if tuple(t.shape) != want:
                raise ValueError(f"{name} of {shape} in {format} must be {want}, got {tuple(t.shape)}")
        if codes.device != scales.device:
            raise ValueError("codes and scales must be on one device")
        self.shape, self.format, self.rows, self.cols, self.device = shape, format, rows, shape[-1], codes.device
        self._codes, self._scales, self._both = codes, scales, None
        self.codes_ptr, self.scales_ptr = codes.data_ptr(), scales.data_ptr()

    @classmethod
    def _empty(cls, shape: tuple, rows: int, format: str, like: torch.Tensor) -> "MXTensor":
        """Uninitialised, on the device of ``like``: codes and then scales in one allocation."""

        self = object.__new__(cls)
        cols = shape[-1]
        code = self._code = _format_code(format)
        steps = (cols + 127) >> 7
        at = (rows * steps * (64 if code else 128) + 511) & ~511
        both = like.new_empty(at + ((rows + 127) >> 7) * steps * 512, dtype=torch.uint8)
        self.shape, self.format, self.rows, self.cols, self.device = shape, format, rows, cols, like.device
        self._codes = self._scales = None
        self._both = both
        self.codes_ptr = both.data_ptr()
        self.scales_ptr = self.codes_ptr + at
        return self

    @classmethod
    def from_row_scales(cls, codes: torch.Tensor, scales: torch.Tensor, shape, format: str) -> "MXTensor":
        """From the plain layout of a checkpoint: ``codes`` [rows, cols] (mxfp8) or [rows, ceil(cols / 2)] (mxfp4, the
        even element in the low nibble) and ``scales`` [rows, ceil(cols / 32)], as uint8, int8 or the types of just
        these bytes (float8_e4m3fn, float4_e2m1fn_x2, float8_e8m0fnu); padded and tiled once, by tensor operations
        on whatever device they are."""

        shape = tuple(int(v) for v in shape)
        if not shape or min(shape) < 0 or not 0 < shape[-1] <= MAX_COLUMNS:
            raise ValueError(f"a microscaled tensor needs a last dimension of 1 to {MAX_COLUMNS}")
        rows, cols, code = math.prod(shape[:-1]), shape[-1], _format_code(format)
        for t, want, name, own in ((codes, (rows, -(-cols // 2) if code else cols), "codes", _CODE_TYPES[code]),
                                   (scales, (rows, -(-cols // 32)), "scales", "float8_e8m0fnu")):
            if t.dtype not in (torch.uint8, torch.int8, getattr(torch, own, None)) or tuple(t.shape) != want:
                raise ValueError(f"{name} of {shape} in {format} must be uint8, int8 or {own}, {want}, "
                                 f"got {tuple(t.shape)} {t.dtype}")
        codes, scales = codes.view(torch.uint8), scales.view(torch.uint8)
        if code and cols % 2:
            codes = codes.clone()
            codes[:, -1] &= 15  # the element past the last column
        tiles, steps = -(-rows // 128), -(-cols // 128)
        pad = torch.nn.functional.pad
        codes = pad(codes, (0, codes_shape(rows, cols, format)[1] - codes.shape[1])).contiguous()
        scales = pad(scales, (0, steps * 4 - scales.shape[1], 0, tiles * 128 - rows))
        scales = scales.view(tiles, 4, 32, steps, 4).permute(0, 3, 2, 1, 4).contiguous()
        return cls(codes, scales, shape, format)

    def row_scales(self) -> torch.Tensor:
        """The scale bytes as [rows, ceil(cols / 32)]."""

        tiles, steps = scales_shape(self.rows, self.cols)[:2]
        plain = self.scales.permute(0, 3, 2, 1, 4).reshape(tiles * 128, steps * 4)
        return plain[:self.rows, :-(-self.cols // 32)].contiguous()

    def _any(self) -> torch.Tensor:
        """A tensor of this one's device, to allocate beside."""

        return self._codes if self._both is None else self._both

    @property
    def codes(self) -> torch.Tensor:
        codes = self._codes
        if codes is None:
            width = ((self.cols + 127) >> 7) * (64 if self._code else 128)
            codes = self._codes = self._both.as_strided((self.rows, width), (width, 1))
        return codes

    @property
    def scales(self) -> torch.Tensor:
        scales = self._scales
        if scales is None:
            steps = (self.cols + 127) >> 7
            scales = self._scales = self._both.as_strided(((self.rows + 127) >> 7, steps, 32, 4, 4),
                                                          (steps * 512, 512, 16, 4, 1), self.scales_ptr - self.codes_ptr)
        return scales

    def __reduce__(self):  # copies and pickles hold tensors of their own
        return MXTensor, (self.codes, self.scales, self.shape, self.format)

    def __repr__(self) -> str:
        return f"MXTensor(shape={self.shape}, format={self.format!r}, device={self.device})"

    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()

    def view(self, *shape) -> "MXTensor":
        """The same rows under other leading dimensions; the last one stays (what lies past it is zero)."""

        if not shape or int(shape[-1]) != self.cols:
            raise ValueError(f"a view keeps the last dimension, {self.cols}, got {shape}")
        return MXTensor(self.codes, self.scales, shape, self.format)

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """The values the codes and scales stand for, rounded to ``dtype``."""

        if dtype not in _native.DTYPE_CODES:
            raise TypeError("dequantize gives bfloat16, float16 or float32")
        _require_cuda(self.device)
        out = torch.empty(self.shape, dtype=dtype, device=self.device)
        _call(self.device, "fl_mx_dequantize", self.codes_ptr, self.scales_ptr, self._code, self.rows, self.cols,
              out.data_ptr(), _native.DTYPE_CODES[dtype])
        return out


def _require_cuda(device: torch.device) -> None:
    if device.type != "cuda":
        raise RuntimeError("flashloop_b200 kernels need CUDA tensors (there is no CPU fallback)")


def _call(device: torch.device, name: str, *args) -> None:
    """One entry point on the current stream of ``device`` (made the current device for the call)."""

    function = getattr(_native.load(), name)
    index = device.index
    if index == torch.cuda.current_device():
        status = function(*args, _raw_stream(index))
    else:
        with torch.cuda.device(device):
            status = function(*args, _raw_stream(index))
    if status:
        _native.check(status, name)


def _values(x: torch.Tensor, *others: torch.Tensor | None) -> None:
    """Floating-point CUDA inputs of one device that need no gradient."""

    if x.dtype not in _native.DTYPE_CODES:
        raise TypeError("microscaled operators take bfloat16, float16 or float32")
    if not x.is_cuda:
        _require_cuda(x.device)
    index = x.get_device()
    grad = torch.is_grad_enabled()
    for t in others:
        if t is not None:
            if t.get_device() != index:
                _require_cuda(t.device)
                raise ValueError("all operands must be on one device")
            if grad and t.requires_grad:
                raise RuntimeError(_NO_GRADIENT)
    if grad and x.requires_grad:
        raise RuntimeError(_NO_GRADIENT)
    if getattr(forward_ad, "_current_level", 0) >= 0:  # inside a dual level: asking every tensor takes 0.4 us each
        _refuse_duals(x, *others)


def _refuse_duals(*tensors: torch.Tensor | None) -> None:
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError("microscaled operators record no gradient: a dual tensor would lose its tangent")


_NO_GRADIENT = "microscaled operators record no gradient: call them under torch.no_grad()"


def mx_quantize(x: torch.Tensor, format: str = "mxfp8") -> MXTensor:
    """``x`` [..., cols] (bfloat16, float16 or float32; rows of unit inner stride, otherwise copied) in blocks
    of 32 along the last dimension: the scale is the smallest power of two that keeps the block in
    range, elements are rounded to nearest, ties to even.  A block with a NaN or an infinity reads
    as NaN."""

    _values(x)
    shape = tuple(x.shape)
    if not shape or not 0 < shape[-1] <= MAX_COLUMNS:
        raise ValueError(f"mx_quantize needs a last dimension of 1 to {MAX_COLUMNS} columns")
    cols = shape[-1]
    if x.ndim != 2 or x.stride(1) != 1 or (x.stride(0) < cols and shape[0] > 1):
        x = x.reshape(-1, cols)  # a view where the rows have one stride
        if (x.stride(1) != 1 and cols > 1) or (x.stride(0) < cols and x.shape[0] > 1):
            x = x.contiguous()
    rows = x.shape[0]
    q = MXTensor._empty(shape, rows, format, x)
    _call(x.device, "fl_mx_quantize", x.data_ptr(), _native.DTYPE_CODES[x.dtype], rows, cols, x.stride(0), q._code,
          q.codes_ptr, q.scales_ptr)
    return q


def mx_rmsnorm(x: torch.Tensor, weight: torch.Tensor, eps: float, *, residual: torch.Tensor | None = None,
               weight2: torch.Tensor | None = None, eps2: float = 0.0, addend: torch.Tensor | None = None,
               want_sum: bool = False, format: str = "mxfp8"):
    """RMSNorm with a microscaled result.  ``s = [addend +] x``; without ``weight2`` the result is
    ``RMSNorm(s)``, with it ``RMSNorm2(hidden)`` of ``hidden = [residual +] RMSNorm(s)``.  ``s`` and
    ``hidden`` are rounded to the type of ``x``, everything between is float32.  Returns (result
    :class:`MXTensor`, hidden or None, s or None): s only with ``want_sum``."""

    _values(x, weight, residual, weight2, addend)
    shape = tuple(x.shape)
    if not shape or not 0 < shape[-1] <= MAX_NORM_WIDTH:
        raise ValueError(f"rows must be 1 to {MAX_NORM_WIDTH} wide")
    width = shape[-1]
    for t in (weight, weight2):
        if t is not None and (t.numel() != width or t.dtype != x.dtype or not t.is_contiguous()):
            raise ValueError("weight does not match the rows")
    for t in (residual, addend):
        if t is not None and (t.shape != x.shape or t.dtype != x.dtype):
            raise ValueError("addend / residual do not match the rows")
    if residual is not None and weight2 is None:
        raise ValueError("a residual needs weight2: the stream it is added to is what weight2 normalises")
    if want_sum and addend is None:
        raise ValueError("want_sum needs an addend")
    x = x.contiguous()
    if residual is not None:
        residual = residual.contiguous()
    if addend is not None:
        addend = addend.contiguous()
    rows = x.numel() // width
    q = MXTensor._empty(shape, rows, format, x)
    hidden = None if weight2 is None else torch.empty_like(x)
    total = torch.empty_like(x) if want_sum else None
    ptr = _native.ptr
    _call(x.device, "fl_rmsnorm_mx", x.data_ptr(), ptr(addend), ptr(residual), weight.data_ptr(), eps, ptr(weight2), eps2,
          _native.DTYPE_CODES[x.dtype], rows, width, q._code, ptr(total), ptr(hidden), q.codes_ptr,
          q.scales_ptr)
    return q, hidden, total


def _operand(x, weight: MXTensor) -> MXTensor:
    if not isinstance(weight, MXTensor):
        raise TypeError("the weight must be an MXTensor (mx_quantize)")
    if len(weight.shape) != 2 or weight.rows > MAX_COLUMNS:
        raise ValueError("the weight must be [out_features, in_features]")
    if isinstance(x, torch.Tensor):
        x = mx_quantize(x, "mxfp8")
    elif not isinstance(x, MXTensor):
        raise TypeError("x must be an MXTensor or a tensor to quantise")
    if x.cols != weight.cols:
        raise ValueError("x and weight do not match")
    _require_cuda(x.device)
    if x.device != weight.device:
        _require_cuda(weight.device)
        raise ValueError("all operands must be on one device")
    return x


def mx_linear(x, weight: MXTensor, *, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``x @ weight.T`` of microscaled operands on the tensor cores, float32 accumulation, rounded once
    to ``out_dtype``.  ``x`` is an :class:`MXTensor` of either format or a tensor, which is then
    quantised to mxfp8 first; ``weight`` [out_features, in_features] of either format."""

    x = _operand(x, weight)
    if out_dtype not in _native.DTYPE_CODES:
        raise TypeError("out_dtype is bfloat16, float16 or float32")
    features = weight.rows
    out = x._any().new_empty((*x.shape[:-1], features), dtype=out_dtype)
    if x.rows and features:
        _call(x.device, "fl_mx_linear", x.codes_ptr, x.scales_ptr, x._code, weight.codes_ptr, weight.scales_ptr,
              weight._code, x.rows, features, x.cols, out.data_ptr(), _native.DTYPE_CODES[out_dtype])
    return out


def mx_linear_swiglu(x, gate: MXTensor, up: MXTensor, *, out_dtype: torch.dtype = torch.bfloat16,
                     out_format: str | None = None):
    """``silu(x @ gate.T) * (x @ up.T)`` in one launch, as :func:`mx_linear` takes its operands (gate and
    up of one shape and format).  The activation is float32 and rounded once: to ``out_dtype``, or
    with ``out_format`` to an :class:`MXTensor`, which the down projection takes as it is."""

    x = _operand(x, gate)
    _operand(x, up)
    if gate.shape != up.shape or gate.format != up.format:
        raise ValueError("gate and up must agree in shape and format")
    features = gate.rows
    shape = (*x.shape[:-1], features)
    if out_format is not None:
        if features == 0:
            raise ValueError("a microscaled result needs at least one feature")
        out = MXTensor._empty(shape, x.rows, out_format, x._any())
        target, dtype, fmt, scales = out.codes_ptr, 0, out._code, out.scales_ptr
    else:
        if out_dtype not in _native.DTYPE_CODES:
            raise TypeError("out_dtype is bfloat16, float16 or float32")
        out = x._any().new_empty(shape, dtype=out_dtype)
        target, dtype, fmt, scales = out.data_ptr(), _native.DTYPE_CODES[out_dtype], 0, None
    if x.rows and features:
        _call(x.device, "fl_mx_linear_swiglu", x.codes_ptr, x.scales_ptr, x._code, gate.codes_ptr, gate.scales_ptr,
              up.codes_ptr, up.scales_ptr, gate._code, x.rows, features, x.cols, target, dtype, fmt, scales)
    return out


def mx_status(device: torch.device | str = "cuda", *, reset: bool = False) -> int:
    """0, or 1 after a bounded wait inside a microscaled projection ran out on ``device`` (its result was
    not valid).  Synchronises the current stream."""

    flag = C.c_int32(-1)
    device = torch.device(device)
    _require_cuda(device)
    if device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    with torch.cuda.device(device):
        _native.check(_native.load().fl_mx_status(C.byref(flag), int(bool(reset)), _native.current_stream(device)),
                      "fl_mx_status")
    return int(flag.value)
