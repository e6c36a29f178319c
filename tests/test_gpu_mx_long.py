"""Products so long that a wait sits through more steps than it has tries of its own."""

from __future__ import annotations

import torch
import pytest

import flashloop_b200 as fl
from flashloop_b200.mx import codes_shape, mx_status, scales_shape

pytestmark = pytest.mark.gpu


def test_a_share_of_many_steps():
    """400,000 steps to each of eight CTAs, whose epilogues wait for the last one (2^15 tries are about 50 ms).
    Ones here and there, so that every sum is exact."""

    cols, features = 400_000 * 8 * 128, 3

    def sparse(rows):
        codes = torch.zeros(codes_shape(rows, cols, "mxfp4"), dtype=torch.uint8, device="cuda")
        codes[:, ::8192] = 0x02  # 1.0 in the low nibble
        scales = torch.full(scales_shape(rows, cols), 127, dtype=torch.uint8, device="cuda")
        return fl.MXTensor(codes, scales, (rows, cols), "mxfp4")

    x, w = sparse(1), sparse(features)
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    start.record()
    y = fl.mx_linear(x, w, out_dtype=torch.float32)
    end.record()
    assert bool((y == cols // 2 // 8192).all())
    print(f"{start.elapsed_time(end):.1f} ms")
    assert mx_status() == 0
