"""The microscaled norm at the ends of float32's range: a sum of squares that is infinite, zero or a NaN."""

from __future__ import annotations

import pytest
import torch

import flashloop_b200 as fl
from flashloop_b200 import step_ops
from tests import mx_reference as ref

pytestmark = pytest.mark.gpu


def _blocks(bad: torch.Tensor) -> torch.Tensor:
    """Elements whose block of 32 holds a True."""

    rows, width = bad.shape
    padded = torch.nn.functional.pad(bad, (0, -width % 32)).view(rows, -1, 32).any(-1)
    return padded.repeat_interleave(32, 1)[:, :width]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("width", [96, 1001, 2048, 5632])
@pytest.mark.parametrize("addend", [False, True])
def test_rows_whose_squares_are_infinite(width, dtype, addend):
    """The factor of such a row is 0: finite elements give 0 and only the block of an infinite one reads as NaN."""

    g = torch.Generator(device="cuda").manual_seed(width)
    x = torch.randn(6, width, generator=g, device="cuda")
    x[1] *= 1e25               # finite, its squares are not
    x[2, 40] = float("inf")
    x[3, 7] = -float("inf")
    x[4] = 3e38
    x = x.to(dtype)
    w = (1 + 0.1 * torch.randn(width, generator=g, device="cuda")).to(dtype)
    s = x
    more = {}
    if addend:
        more["addend"] = torch.zeros_like(x)
        s = x + more["addend"]
    q = fl.mx_rmsnorm(x, w, 1e-6, **more)[0]
    infinite = torch.isinf(s)
    got = q.dequantize(torch.float32)
    assert torch.equal(torch.isnan(got), _blocks(infinite))
    assert not got[1:5][~_blocks(infinite)[1:5]].any()
    byte = ref.scale_bytes(q.scales, 6)[:6]
    zero = ~_blocks(infinite)[:, ::32].cpu()
    assert not byte[1:5, :zero.shape[1]][zero[1:5]].any()
    # the rows beside them are those of the same call without them
    alone = fl.mx_rmsnorm(x[::5].contiguous(), w, 1e-6)[0]
    assert torch.equal(q.codes[::5], alone.codes)

    residual = torch.randn(6, width, generator=g, device="cuda").to(dtype)
    q, hidden, _ = fl.mx_rmsnorm(x, w, 1e-6, residual=residual, weight2=w, eps2=1e-6, **more)
    assert torch.equal(torch.isnan(hidden), infinite)
    finite = ~infinite[1:5]
    assert torch.equal(hidden[1:5][finite], residual[1:5][finite])  # nothing is added to it
    # the second norm is that of the stored stream
    plain = torch.isnan(fl.mx_rmsnorm(hidden, w, 1e-6)[0].dequantize(torch.float32))
    assert torch.equal(torch.isnan(q.dequantize(torch.float32)), plain)
    if dtype == torch.bfloat16 and width % 8 == 0:
        # and the norm that the framework had says the same
        other = step_ops.rmsnorm(s, w, 1e-6)
        assert torch.equal(torch.isnan(other), infinite) and not other[1:5][finite].any()


def test_an_infinite_stream_in_the_second_norm():
    x = torch.randn(3, 256, generator=torch.Generator().manual_seed(3)).cuda().to(torch.bfloat16)
    w = torch.ones(256, device="cuda", dtype=torch.bfloat16)
    residual = x.clone()
    residual[1] = 2e38
    residual[2, 5] = float("inf")
    q, hidden, _ = fl.mx_rmsnorm(x, w, 1e-6, residual=residual, weight2=w, eps2=1e-6)
    got = q.dequantize(torch.float32)
    assert not got[1].any() and torch.isnan(got[2, :32]).all() and not got[2, 32:].any() and torch.isfinite(got[0]).all()


def test_rows_of_zeros_without_an_epsilon_are_not_numbers():
    """0 * (1 / sqrt(0)), as the formula has it."""

    x = torch.zeros(2, 64, device="cuda")
    x[1] = 1
    got = fl.mx_rmsnorm(x, torch.ones(64, device="cuda"), 0.0)[0].dequantize(torch.float32)
    assert torch.isnan(got[0]).all() and bool((got[1] == 1).all())
