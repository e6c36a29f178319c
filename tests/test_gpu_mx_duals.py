"""Forward-mode gradients are refused like the others."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

import flashloop_b200 as fl

pytestmark = pytest.mark.gpu


def test_dual_tensors_are_refused():
    x, one = torch.randn(3, 64, device="cuda"), torch.ones(64, device="cuda")
    w = fl.mx_quantize(torch.randn(8, 64, device="cuda"))
    want = fl.mx_linear(x, w)
    with forward_ad.dual_level():
        dual, dual_one = forward_ad.make_dual(x, torch.ones_like(x)), forward_ad.make_dual(one, one)
        for call in (lambda: fl.mx_quantize(dual), lambda: fl.mx_linear(dual, w), lambda: fl.mx_linear_swiglu(dual, w, w),
                     lambda: fl.mx_rmsnorm(dual, one, 1e-6), lambda: fl.mx_rmsnorm(x, dual_one, 1e-6),
                     lambda: fl.mx_rmsnorm(x, one, 1e-6, addend=dual),
                     lambda: fl.mx_rmsnorm(x, one, 1e-6, residual=dual, weight2=one),
                     lambda: fl.mx_rmsnorm(x, one, 1e-6, residual=x, weight2=dual_one), lambda: fl.mx_quantize(dual[:, ::2])):
            with pytest.raises(RuntimeError, match="no gradient"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="no gradient"):
                call()  # no_grad leaves forward mode as it is
        assert torch.equal(fl.mx_linear(x, w), want)  # ordinary tensors in a dual level
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: fl.mx_quantize(t).dequantize(torch.float32), (x,), (x,))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: fl.mx_quantize(t).dequantize(torch.float32))(x)
    assert torch.equal(fl.mx_linear(x, w), want)
