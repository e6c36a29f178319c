"""Addresses between two elements are refused on the host: a load from one would fault on the GPU."""

from __future__ import annotations

import pytest

from flashloop_b200 import _native, build_kernels

A = 1 << 20  # an aligned address that nothing reads


@pytest.fixture(scope="module")
def lib():
    build_kernels.build()
    return _native.load()


@pytest.mark.parametrize("dtype,offsets", [(0, (1, 3)), (1, (1, 7)), (2, (1, 2, 6))])
def test_addresses_between_elements(lib, dtype, offsets):
    for off in offsets:
        assert lib.fl_mx_quantize(A + off, dtype, 2, 32, 32, 0, A, A, None) == -1
        assert b"aligned to its elements" in lib.fl_last_error()
        names = ("x", "addend", "residual", "weight", "weight2", "sum_out", "hidden")
        for name in names:
            p = {n: A + (off if n == name else 0) for n in names}
            assert lib.fl_rmsnorm_mx(p["x"], p["addend"], p["residual"], p["weight"], 1e-6, p["weight2"], 1e-6, dtype, 2, 64, 0,
                                     p["sum_out"], p["hidden"], A, A, None) == -1
            assert b"aligned to their elements" in lib.fl_last_error(), name
