"""Waits of the microscaled projections that run out: the call ends by itself, the status word says so until it
is reset, and the next call is exact.

``fl_mx_give_up_at`` makes the wait for a given step fail: nothing on the device faults or waits for ever (what
waits for the missing products afterwards gives up after some 50 ms)."""

from __future__ import annotations

from concurrent.futures import ThreadPoolExecutor

import pytest
import torch

import flashloop_b200 as fl
from flashloop_b200 import _native
from flashloop_b200.mx import mx_status

pytestmark = pytest.mark.gpu


@pytest.fixture
def give_up_at():
    lib = _native.load()
    assert mx_status(reset=True) == 0

    def at(step: int) -> None:
        assert lib.fl_mx_give_up_at(step) == 0

    yield at
    at(-1)
    mx_status(reset=True)


def _operands(rows, cols, features, x_format, weights):
    g = torch.Generator(device="cuda").manual_seed(rows + cols + features)
    draw = lambda n: torch.randn(n, cols, generator=g, device="cuda")
    return fl.mx_quantize(draw(rows), x_format), [fl.mx_quantize(draw(features) * cols ** -0.5, "mxfp4") for _ in range(weights)]


def _run_out(call, give_up_at, steps):
    want = call()
    assert mx_status() == 0
    for step in steps:
        give_up_at(step)
        call()
        give_up_at(-1)
        assert mx_status() == 1, step
        assert mx_status(reset=True) == 1 and mx_status() == 0
        for _ in range(2):
            assert torch.equal(call(), want), step
        assert mx_status() == 0


# one and several rounds of the ring, one CTA and clusters to a tile, each height of a tile of few rows
@pytest.mark.parametrize("rows,cols,features,steps", [
    (1, 100, 130, (0,)), (16, 2048, 2048, (0, 1)), (3, 20000, 200, (0, 2, 11, 12, 18)), (16, 20000, 19000, (0, 7, 60, 156)),
    (30, 4096, 9000, (0, 9)), (64, 2048, 9000, (0, 5, 10, 15)), (64, 4096, 384, (0, 2)), (128, 1024, 500, (0,)),
    (100, 4096, 18000, (0, 4, 6, 9, 31)), (100, 4096, 19000, (0, 4, 6, 9, 31))])
def test_few_rows(rows, cols, features, steps, give_up_at):
    x, (w, up) = _operands(rows, cols, features, "mxfp8", 2)
    _run_out(lambda: fl.mx_linear(x, w, out_dtype=torch.float32), give_up_at, steps)
    _run_out(lambda: fl.mx_linear_swiglu(x, w, up, out_dtype=torch.float32), give_up_at, steps[:2])
    _run_out(lambda: fl.mx_linear_swiglu(x, w, up, out_format="mxfp8").dequantize(torch.float32), give_up_at, steps[:1])


# one tile to a pair of CTAs and several, so that the epilogue waits for products that never come
@pytest.mark.parametrize("x_format", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("rows,cols,features,steps", [(2500, 4096, 1000, (0, 3, 7, 12)), (20000, 300, 300, (0, 1)),
                                                      (3000, 1500, 4000, (5, 14, 17))])
def test_many_rows(rows, cols, features, steps, x_format, give_up_at):
    x, (w, up) = _operands(rows, cols, features, x_format, 2)
    _run_out(lambda: fl.mx_linear(x, w, out_dtype=torch.float32), give_up_at, steps)
    _run_out(lambda: fl.mx_linear_swiglu(x, w, up, out_dtype=torch.float32), give_up_at, steps[:2])
    _run_out(lambda: fl.mx_linear_swiglu(x, w, up, out_format="mxfp8").dequantize(torch.float32), give_up_at, steps[-1:])


def test_a_step_that_no_call_reaches(give_up_at):
    for rows in (4, 20000):
        x, (w,) = _operands(rows, 640, 200, "mxfp8", 1)
        want = fl.mx_linear(x, w)
        give_up_at(10 ** 6)
        assert torch.equal(fl.mx_linear(x, w), want)
        give_up_at(-1)
    assert mx_status() == 0


def test_other_threads_and_what_was_captured_before(give_up_at):
    x, (w,) = _operands(16, 1024, 512, "mxfp8", 1)
    want = fl.mx_linear(x, w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fl.mx_linear(x, w)
    give_up_at(0)
    graph.replay()
    with ThreadPoolExecutor(1) as pool:
        got = pool.submit(fl.mx_linear, x, w).result()
    give_up_at(-1)
    assert torch.equal(out, want) and torch.equal(got, want) and mx_status() == 0


def test_calls_after_one_that_gave_up_are_in_order(give_up_at):
    """Calls before and after it in the stream, without waiting in between."""

    x, (w,) = _operands(16, 4096, 2048, "mxfp8", 1)
    big, _ = _operands(5000, 4096, 1, "mxfp8", 1)
    want, many = fl.mx_linear(x, w), fl.mx_linear(big, w)
    torch.cuda.synchronize()
    for _ in range(5):
        before, before_many = fl.mx_linear(x, w), fl.mx_linear(big, w)
        give_up_at(1)
        fl.mx_linear(x, w), fl.mx_linear(big, w), fl.mx_linear(x, w)
        give_up_at(-1)
        after, after_many = fl.mx_linear(x, w), fl.mx_linear(big, w)
        assert mx_status(reset=True) == 1
        assert torch.equal(before, want) and torch.equal(after, want)
        assert torch.equal(before_many, many) and torch.equal(after_many, many)
