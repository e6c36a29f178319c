"""Replacing projection weights by microscaled ones is all or nothing: what is refused, or fails on the way,
leaves every layer as it was."""

from __future__ import annotations

import pytest
import torch

import flashloop_b200 as fl
from flashloop_b200 import mx, weights
from tests.helpers import tiny_ouro_model


class Quantiser:
    """Stands for ``mx_quantize`` without a GPU; may fail at a call."""

    def __init__(self, fails_at=None):
        self.calls, self.fails_at = 0, fails_at

    def __call__(self, x, format):
        if self.calls == self.fails_at:
            raise torch.OutOfMemoryError("no memory left")
        self.calls += 1
        shape = tuple(x.shape)
        return fl.MXTensor(torch.zeros(mx.codes_shape(*shape, format), dtype=torch.uint8),
                           torch.zeros(mx.scales_shape(*shape), dtype=torch.uint8), shape, format)


def _layers():
    layers = tiny_ouro_model().model.layers
    weights.repack_projection_weights(layers)
    return layers


def _is_whole(layers) -> bool:
    return all(layer.self_attn._flashloop_qkv_weight is not None and layer.mlp._flashloop_gate_up_weight is not None
               and layer.self_attn.o_proj.weight is not None and layer.mlp.down_proj.weight is not None
               and getattr(layer.self_attn, "_flashloop_mx_qkv", None) is None
               and getattr(layer.mlp, "_flashloop_mx_gate", None) is None for layer in layers)


@pytest.mark.parametrize("fails_at", range(10))
def test_an_allocation_that_fails(fails_at, monkeypatch):
    layers = _layers()
    assert len(layers) == 2  # five weights each
    monkeypatch.setattr(weights, "mx_quantize", Quantiser(fails_at))
    with pytest.raises(torch.OutOfMemoryError):
        weights.quantize_projection_weights(layers, "mxfp4")
    assert _is_whole(layers)
    monkeypatch.setattr(weights, "mx_quantize", Quantiser())
    weights.quantize_projection_weights(layers, "mxfp4")  # and can be done again
    for layer in layers:
        assert layer.self_attn._flashloop_qkv_weight is None and layer.mlp._flashloop_gate_up_weight is None
        assert layer.self_attn.o_proj.weight is None and layer.mlp.down_proj.weight is None
        assert layer.self_attn._flashloop_mx_qkv.shape == (768, 256) and layer.self_attn._flashloop_mx_value.shape == (256, 256)
        assert layer.mlp._flashloop_mx_down.shape == (256, 384)


def _bias(layer):
    layer.self_attn.o_proj.bias = torch.nn.Parameter(torch.zeros(256))


def _other_bias(layer):
    layer.mlp.down_proj.bias = torch.nn.Parameter(torch.zeros(256))


def _narrow_heads(layer):
    layer.self_attn._flashloop_qkv_splits = (192, 256, 256)


def _not_repacked(layer):
    del layer.mlp._flashloop_gate_up_weight


def _released(layer):
    layer.self_attn.o_proj.weight = None


@pytest.mark.parametrize("break_it", [_bias, _other_bias, _narrow_heads, _not_repacked, _released])
def test_a_later_layer_that_is_refused(break_it, monkeypatch):
    layers = _layers()
    quantise = Quantiser()
    monkeypatch.setattr(weights, "mx_quantize", quantise)
    break_it(layers[1])
    with pytest.raises(ValueError):
        weights.quantize_projection_weights(layers, "mxfp8")
    assert quantise.calls == 0 and _is_whole(layers[:1])


def test_formats(monkeypatch):
    layers = _layers()
    monkeypatch.setattr(weights, "mx_quantize", Quantiser())
    with pytest.raises(ValueError, match="unknown microscaled format"):
        weights.quantize_projection_weights(layers, "int4")
    assert _is_whole(layers)
    weights.quantize_projection_weights(layers[1:], "mxfp8")
    with pytest.raises(RuntimeError, match="already held in mxfp8"):
        weights.quantize_projection_weights(layers, "mxfp4")
    assert _is_whole(layers[:1])
    weights.quantize_projection_weights(layers, "mxfp8")  # what is held already stays
    assert layers[0].self_attn._flashloop_mx_qkv.format == "mxfp8" and not _is_whole(layers[:1])
