"""Fused projection weights (flashloop/weights.py:20-117): Q/K/V and gate/up are stored as one
buffer each so that a decode step issues one GEMM instead of three / two.  The GEMMs themselves
are library calls (cuBLAS through ``F.linear``), or the microscaled products of :mod:`.mx` once
:func:`quantize_projection_weights` has replaced the weights."""

from __future__ import annotations

from collections.abc import Sequence

import torch
from torch import nn
from torch.nn import functional as F

from .mx import MXTensor, _format_code, mx_linear, mx_linear_swiglu, mx_quantize


@torch.no_grad()
def repack_projection_weights(layers: Sequence[nn.Module]) -> None:
    """weights.py:20-71: concatenate the weights, register them as buffers, release the originals."""

    for layer in layers:
        attention, mlp = layer.self_attn, layer.mlp
        if hasattr(attention, "_flashloop_qkv_weight"):
            if not hasattr(mlp, "_flashloop_gate_up_weight"):
                raise RuntimeError("partially repacked FlashLoop layer")
            continue
        modules = {"q_proj": attention.q_proj, "k_proj": attention.k_proj, "v_proj": attention.v_proj,
                   "gate_proj": mlp.gate_proj, "up_proj": mlp.up_proj}
        for name, module in modules.items():
            if module.bias is not None:
                raise ValueError(f"FlashLoop fused projection requires biasless {name}")
            if module.weight is None:
                raise ValueError(f"{name} has already released its weight")
        attention._flashloop_qkv_splits = tuple(int(modules[n].out_features) for n in ("q_proj", "k_proj", "v_proj"))
        mlp._flashloop_gate_up_splits = (int(mlp.gate_proj.out_features), int(mlp.up_proj.out_features))
        attention.register_buffer("_flashloop_qkv_weight", torch.cat(
            [modules[n].weight for n in ("q_proj", "k_proj", "v_proj")], dim=0).detach(), persistent=False)
        mlp.register_buffer("_flashloop_gate_up_weight", torch.cat(
            [mlp.gate_proj.weight, mlp.up_proj.weight], dim=0).detach(), persistent=False)
        for module in modules.values():
            module.weight = None


@torch.no_grad()
def quantize_projection_weights(layers: Sequence[nn.Module], format: str) -> None:
    """Replace the repacked projection weights of every layer (Q/K/V, ``o_proj``, gate, up,
    ``down_proj``) by their microscaled form and release the bfloat16 tensors: all of them once every
    microscaled one is there, or none.  No counterpart in the reference, whose projections stay
    bfloat16 (flashloop/weights.py:20-117)."""

    _format_code(format)
    todo = []
    for layer in layers:  # what is refused is refused before anything changes
        attention, mlp = layer.self_attn, layer.mlp
        done = getattr(attention, "_flashloop_mx_qkv", None)
        if done is not None:
            if done.format != format:
                raise RuntimeError(f"the projections are already held in {done.format}")
            continue
        if (getattr(attention, "_flashloop_qkv_weight", None) is None
                or getattr(mlp, "_flashloop_gate_up_weight", None) is None):
            raise ValueError("microscaled projections need fused projection weights (repack_projection_weights)")
        for name, module in (("o_proj", attention.o_proj), ("down_proj", mlp.down_proj)):
            if module.bias is not None:
                raise ValueError(f"microscaled projections require biasless {name}")
            if module.weight is None:
                raise ValueError(f"{name} has already released its weight")
        if sum(attention._flashloop_qkv_splits[:2]) % 128:
            raise ValueError("microscaled projections need heads of 128 channels")
        todo.append((attention, mlp))
    made = []
    for attention, mlp in todo:  # which may run out of memory
        gate, up = mlp._flashloop_gate_up_weight.split(mlp._flashloop_gate_up_splits, dim=0)
        made.append([mx_quantize(w, format) for w in (attention._flashloop_qkv_weight, attention.o_proj.weight, gate, up,
                                                      mlp.down_proj.weight)])
    for (attention, mlp), (qkv, output, gate, up, down) in zip(todo, made):
        value_row = sum(attention._flashloop_qkv_splits[:2])
        attention._flashloop_mx_qkv = qkv
        attention._flashloop_mx_value = MXTensor(qkv.codes[value_row:], qkv.scales[value_row // 128:],
                                                 (attention._flashloop_qkv_splits[2], qkv.cols), format)
        attention._flashloop_mx_output = output
        mlp._flashloop_mx_gate, mlp._flashloop_mx_up, mlp._flashloop_mx_down = gate, up, down
        attention._flashloop_qkv_weight = mlp._flashloop_gate_up_weight = None
        attention.o_proj.weight = mlp.down_proj.weight = None


def project_qkv(attention: nn.Module, values):
    """weights.py:74-88; ``values`` may be an :class:`MXTensor` where the weights are."""

    weight = getattr(attention, "_flashloop_mx_qkv", None)
    if weight is not None:
        return tuple(mx_linear(values, weight).split(attention._flashloop_qkv_splits, dim=-1))
    weight = getattr(attention, "_flashloop_qkv_weight", None)
    if weight is None:
        return attention.q_proj(values), attention.k_proj(values), attention.v_proj(values)
    return tuple(F.linear(values, weight).split(attention._flashloop_qkv_splits, dim=-1))


def project_value(attention: nn.Module, values) -> torch.Tensor:
    """weights.py:91-105: only V, from the packed QKV weight without copying it."""

    weight = getattr(attention, "_flashloop_mx_value", None)
    if weight is not None:
        return mx_linear(values, weight)
    weight = getattr(attention, "_flashloop_qkv_weight", None)
    if weight is None:
        return attention.v_proj(values)
    q_features, k_features, v_features = attention._flashloop_qkv_splits
    return F.linear(values, weight.narrow(0, q_features + k_features, v_features))


def project_output(attention: nn.Module, values: torch.Tensor) -> torch.Tensor:
    """The ``o_proj`` call of flashloop/prefill.py and flashloop/engine.py:531."""

    weight = getattr(attention, "_flashloop_mx_output", None)
    return attention.o_proj(values) if weight is None else mx_linear(values, weight)


def fused_mlp(mlp: nn.Module, values) -> torch.Tensor:
    """weights.py:108-117; with microscaled weights the gated activation stays in mxfp8 on its way to
    the down projection."""

    gate = getattr(mlp, "_flashloop_mx_gate", None)
    if gate is not None:
        return mx_linear(mx_linear_swiglu(values, gate, mlp._flashloop_mx_up, out_format="mxfp8"),
                         mlp._flashloop_mx_down)
    weight = getattr(mlp, "_flashloop_gate_up_weight", None)
    if weight is None:
        return mlp(values)
    gate, up = F.linear(values, weight).split(mlp._flashloop_gate_up_splits, dim=-1)
    return mlp.down_proj(mlp.act_fn(gate) * up)
