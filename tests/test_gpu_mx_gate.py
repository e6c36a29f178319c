"""How exact the gated activation of microscaled projections is, with sums that are exact."""

from __future__ import annotations

import pytest
import torch

import flashloop_b200 as fl

pytestmark = pytest.mark.gpu


def _parts(g: torch.Tensor):
    """g (at most twelve bits) as three values that the format holds: each the quantised value of what is left."""

    parts, left = [], g
    for _ in range(3):
        parts.append(fl.mx_quantize(left[:, None].contiguous()).dequantize(torch.float32)[:, 0])
        left = left - parts[-1]
    assert not left.any()
    return parts


@pytest.mark.parametrize("rows", [7, 40, 130, 30000])
def test_the_gate_over_its_range(rows):
    """x = (three parts of g, 1) in blocks of their own, so that x @ gate is g and x @ up is u without any rounding.

    The bound counts the roundings: exp within 2 + 1.173 |g| units, the sum with 1 half a unit, the quotient two,
    the product half a one; a unit is at most 2^-23 of the value."""

    features = 40
    generator = torch.Generator(device="cuda").manual_seed(rows)
    g = torch.randint(-110 * 8, 110 * 8, (rows,), generator=generator, device="cuda").float() / 8
    g[:7] = torch.tensor([0.0, -87.0, 87.0, -87.5, -88.0, -100.0, -20.0])
    x = torch.zeros(rows, 128, device="cuda")
    x[:, 0], x[:, 32], x[:, 64] = _parts(g)
    x[:, 96] = 1
    u = 2.0 ** torch.arange(-20, 20, device="cuda").double()
    u[1::2] *= -1
    u[0], u[5] = 2.0 ** 100, 0.0
    gate, up = (torch.zeros(features, 128, device="cuda") for _ in range(2))
    gate[:, 0] = gate[:, 32] = gate[:, 64] = 1
    up[:, 96] = u.float()
    got = fl.mx_linear_swiglu(fl.mx_quantize(x), fl.mx_quantize(gate), fl.mx_quantize(up), out_dtype=torch.float32).double()
    g64 = g.double()[:, None]
    want = g64 / (1 + torch.exp(-g64)) * u
    bound = (2 + 1.173 * g64.abs() + 3) * 2.0 ** -23 * want.abs() + 2.0 ** -149
    ordinary = (g64 >= -87.3).expand_as(want)
    error = (got - want).abs()
    assert bool((error <= bound)[ordinary].all()), float((error - bound)[ordinary].max())
    assert bool((error <= 1.1e-36 * u.abs() + 2.0 ** -149)[~ordinary].all())
    assert not got[0].any()


def test_gates_that_are_not_finite():
    """An infinite sum: silu(inf) = inf, silu(-inf) = -inf * 0, as the formula has it."""

    x = torch.zeros(3, 128, device="cuda")
    x[:, 0] = torch.tensor([1.0, -1.0, 1.0]) * 2.0 ** 100
    x[:, 32] = 1
    gate, up = torch.zeros(2, 128, device="cuda"), torch.zeros(2, 128, device="cuda")
    gate[0, 0] = 2.0 ** 100
    up[:, 32] = 2
    got = fl.mx_linear_swiglu(fl.mx_quantize(x), fl.mx_quantize(gate), fl.mx_quantize(up), out_dtype=torch.float32)
    assert got[0, 0] == float("inf") and torch.isnan(got[1, 0]) and got[0, 1] == 0
