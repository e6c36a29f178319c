"""Views of a microscaled tensor keep its last dimension."""

from __future__ import annotations

import pytest
import torch

import flashloop_b200 as fl


@pytest.mark.parametrize("fmt,width", [("mxfp8", 128), ("mxfp4", 64)])
def test_a_view_of_another_width_is_refused(fmt, width):
    """Elements past the last column are zero, which products rely on: another width would show or hide some."""

    codes, scales = torch.zeros(6, width, dtype=torch.uint8), torch.zeros(1, 1, 32, 4, 4, dtype=torch.uint8)
    t = fl.MXTensor(codes, scales, (6, 100), fmt)
    for shape in ((6, 64), (6, 101), (6, 128), (2, 3, 99), (6, 1), (6,), (600,), ()):
        with pytest.raises(ValueError):
            t.view(*shape)
    for shape in ((5, 100), (2, 100), (7, 100)):
        with pytest.raises(ValueError):
            t.view(*shape)
    for shape in ((6, 100), (2, 3, 100), (1, 6, 1, 100), (torch.Size((3, 2, 100)))):
        v = t.view(*shape)
        assert v.shape == tuple(shape) and v.codes is t.codes and v.scales is t.scales
    row = fl.MXTensor(codes[:1].contiguous(), scales, (100,), fmt)
    assert row.view(1, 1, 100).view(100).shape == (100,)
