"""Microscaled operators as the first thing that a thread does on the GPU."""

from __future__ import annotations

from concurrent.futures import ThreadPoolExecutor

import pytest
import torch

import flashloop_b200 as fl
from flashloop_b200.mx import mx_status

pytestmark = pytest.mark.gpu


def _in_a_new_thread(call):
    """The call's result; what it raises is raised here."""

    with ThreadPoolExecutor(1) as pool:
        return pool.submit(call).result()


@pytest.mark.parametrize("rows", [1, 16, 50, 100, 9000])
def test_the_first_call_of_a_thread(rows):
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = torch.randn(rows, 512, generator=g, device="cuda")
    w, up = (fl.mx_quantize(torch.randn(384, 512, generator=g, device="cuda"), "mxfp4") for _ in range(2))
    q, one = fl.mx_quantize(x), torch.ones(512, device="cuda")
    calls = (lambda: fl.mx_linear(q, w), lambda: fl.mx_linear_swiglu(q, w, up),
             lambda: fl.mx_linear_swiglu(q, w, up, out_format="mxfp8").dequantize(),
             lambda: fl.mx_quantize(x).dequantize(), lambda: fl.mx_rmsnorm(x, one, 1e-6)[0].dequantize(),
             lambda: q.dequantize(torch.float32), lambda: fl.mx_linear(x, w))
    for call in calls:
        want = call()
        torch.cuda.synchronize()
        assert torch.equal(_in_a_new_thread(call), want)
    assert _in_a_new_thread(mx_status) == 0


def test_threads_at_once():
    """Every call of every thread counts, and so does every exception."""

    g = torch.Generator(device="cuda").manual_seed(1)
    w = fl.mx_quantize(torch.randn(512, 512, generator=g, device="cuda"), "mxfp4")
    inputs = [torch.randn(rows, 512, generator=g, device="cuda") for rows in (1, 16, 90, 9000)]
    want = [fl.mx_linear(x, w) for x in inputs]
    torch.cuda.synchronize()

    def work(i: int, own_stream: bool) -> int:
        stream = torch.cuda.Stream() if own_stream else torch.cuda.default_stream()
        with torch.cuda.stream(stream):
            return sum(torch.equal(fl.mx_linear(inputs[i], w), want[i]) for _ in range(30))

    for own_stream in (True, False):
        with ThreadPoolExecutor(4) as pool:
            assert [f.result() for f in [pool.submit(work, i, own_stream) for i in range(4)]] == [30] * 4
    assert mx_status() == 0


def test_streams_without_the_raw_handle(monkeypatch):
    """What a PyTorch without that call uses names the same stream."""

    from flashloop_b200 import mx

    x, out = torch.zeros(4, 256, device="cuda"), []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for handle in (mx._raw_stream, mx._stream_handle):
        monkeypatch.setattr(mx, "_raw_stream", handle)
        with torch.cuda.stream(side):
            assert handle(side.device_index) == side.cuda_stream
            torch.cuda._sleep(2_000_000)  # about a millisecond
            out.append(fl.mx_quantize(x.fill_(3.0)).dequantize())
            x.zero_()
        assert handle(0) == torch.cuda.current_stream().cuda_stream
    torch.cuda.synchronize()
    assert all(bool((o == 3).all()) for o in out)
