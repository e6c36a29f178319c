"""The engine on microscaled projections does not hand on what a product whose wait ran out has left."""

from __future__ import annotations

import pytest
import torch

from flashloop_b200 import FlashLoopConfig, FlashLoopEngine, _native, mx_status
from tests.helpers import tiny_ouro_model

pytestmark = pytest.mark.gpu


@pytest.fixture
def give_up_at():
    lib = _native.load()
    mx_status(reset=True)
    yield lib.fl_mx_give_up_at
    lib.fl_mx_give_up_at(-1)
    mx_status(reset=True)


def _engine(**kwargs):
    return FlashLoopEngine(tiny_ouro_model().cuda(), validate_model=False, max_new_tokens=16, projection_format="mxfp4",
                           config=FlashLoopConfig(enable_sparse_decode=False), **kwargs)


PROMPTS = torch.randint(0, 256, (2, 140), generator=torch.Generator().manual_seed(5))


def test_prefill_raises_and_can_be_repeated(give_up_at):
    prompts, engine = PROMPTS.cuda(), _engine()
    want = engine.prefill(prompts).logits
    engine.reset()
    give_up_at(0)
    with pytest.raises(RuntimeError, match="ran out"):
        engine.prefill(prompts)
    give_up_at(-1)
    with pytest.raises(RuntimeError, match="not initialized"):
        engine.decode(prompts[:, :1])
    with pytest.raises(RuntimeError, match="ran out"):  # until somebody has taken note
        engine.prefill(prompts)
    assert mx_status(reset=True) == 1
    assert torch.equal(engine.prefill(prompts).logits, want)


@pytest.mark.parametrize("graph", [False, True])
def test_generate_raises(graph, give_up_at):
    prompts, engine = PROMPTS.cuda(), _engine(use_cuda_graph=graph)
    plain = engine.decode

    def decode(tokens):  # the last steps of a generation
        if engine.state.next_position >= prompts.shape[1] + 3:
            give_up_at(0)
            engine._graph = None  # recorded before
        return plain(tokens)

    engine.decode = decode
    with pytest.raises(RuntimeError, match="ran out"):
        engine.generate(prompts, max_new_tokens=5, eos_token_id=-1)
    give_up_at(-1)
    del engine.decode
    assert mx_status(reset=True) == 1
    assert engine.generate(prompts, max_new_tokens=5).shape[0] == 2


@pytest.mark.parametrize("graph", [False, True])
def test_decode_raises_in_the_step_after(graph, give_up_at):
    prompts, engine = PROMPTS.cuda(), _engine(use_cuda_graph=graph)
    token = prompts[:, :1].contiguous()
    engine.prefill(prompts)
    engine.decode(token)
    torch.cuda.synchronize()
    engine.decode(token)
    give_up_at(0)
    engine._graph = None
    engine.decode(token).logits.cpu()
    give_up_at(-1)
    with pytest.raises(RuntimeError, match="ran out"):
        engine.decode(token)
    with pytest.raises(RuntimeError, match="not initialized"):
        engine.decode(token)
    assert mx_status(reset=True) == 1
    engine.prefill(prompts)
    engine.decode(token)


def test_every_engine_on_the_device_sees_it(give_up_at):
    prompts, one, other = PROMPTS.cuda(), _engine(), _engine()
    token = prompts[:, :1].contiguous()
    for engine in (one, other):
        engine.prefill(prompts)
    give_up_at(0)
    one.decode(token).logits.cpu()
    give_up_at(-1)
    for engine in (other, one):  # whoever looks first
        with pytest.raises(RuntimeError, match="ran out"):
            engine.decode(token)


def test_bfloat16_projections_do_not_look_at_it(give_up_at):
    from flashloop_b200 import mx_linear, mx_quantize

    give_up_at(0)
    x = torch.randn(4, 256, device="cuda")
    mx_linear(x, mx_quantize(x))
    give_up_at(-1)
    assert mx_status() == 1
    engine = FlashLoopEngine(tiny_ouro_model().cuda(), validate_model=False, max_new_tokens=16)
    assert engine.generate(PROMPTS.cuda(), max_new_tokens=3).shape == (2, 143)
    assert mx_status() == 1


def test_a_decode_step_can_be_captured_by_the_caller(give_up_at):
    prompts, engine = PROMPTS.cuda(), _engine()
    token = prompts[:, :1].contiguous()
    engine.prefill(prompts)
    engine.decode(token)
    torch.cuda.synchronize()
    position = torch.full((2, 1), engine.state.next_position, device="cuda", dtype=torch.long)
    graph = torch.cuda.CUDAGraph()
    with torch.inference_mode(), torch.cuda.graph(graph):
        engine._require_valid_products(token.device, wait=False)
        engine._decode_step(token, position)
    graph.replay()
    torch.cuda.synchronize()
    assert mx_status() == 0
