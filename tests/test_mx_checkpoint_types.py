"""The plain layout of a checkpoint in the types it may come in: what other bytes mean is not guessed."""

from __future__ import annotations

import pytest
import torch

import flashloop_b200 as fl


@pytest.mark.parametrize("fmt,width", [("mxfp8", 64), ("mxfp4", 32)])
def test_types_of_codes_and_scales(fmt, width):
    codes, scales = torch.full((3, width), 0x22, dtype=torch.uint8), torch.full((3, 2), 127, dtype=torch.uint8)
    want = fl.MXTensor.from_row_scales(codes, scales, (3, 64), fmt)
    own = torch.float8_e4m3fn if fmt == "mxfp8" else getattr(torch, "float4_e2m1fn_x2", None)
    for c in [codes.view(t) for t in (torch.uint8, torch.int8, own) if t is not None]:
        for s in (scales, scales.view(torch.int8), scales.view(torch.float8_e8m0fnu)):
            t = fl.MXTensor.from_row_scales(c, s, (3, 64), fmt)
            assert torch.equal(t.codes, want.codes) and torch.equal(t.scales, want.scales)
    others = [torch.float8_e5m2, torch.float8_e4m3fnuz, torch.float8_e5m2fnuz, torch.float8_e8m0fnu, torch.bool]
    others.append(torch.float8_e4m3fn if fmt == "mxfp4" else torch.float8_e8m0fnu)
    for t in others:
        with pytest.raises(ValueError, match="codes"):
            fl.MXTensor.from_row_scales(codes.view(t), scales, (3, 64), fmt)
    for t in (torch.float8_e4m3fn, torch.float8_e5m2, torch.bool):
        with pytest.raises(ValueError, match="scales"):
            fl.MXTensor.from_row_scales(codes, scales.view(t), (3, 64), fmt)
    with pytest.raises(ValueError, match="codes"):
        fl.MXTensor.from_row_scales(codes.half(), scales, (3, 64), fmt)
