"""The engine with microscaled projections against its definition in elementary operations, which round
where the operators round and nowhere else.

What is left between the two is the order and precision of sums.  It moves a bfloat16 result to the
next value now and then, that an element of the next operand by an e4m3 step, and the network amplifies it from
layer to layer.  How far is not for a constant to say: the definition is evaluated with its products and norms in
64 bits and in 32, which differ by the same mechanism, and the engine has to be within four times their
distance (the elements that move are random) and a bfloat16 step of the logits.  A wiring error (a norm,
a residual, a scale out of place) is of order one.  Selecting keys is a decision: where it falls the other
way a whole step differs, so with sparse decoding the median step is held to the bound.
"""

from __future__ import annotations

import pytest
import torch
from torch.nn import functional as F

from flashloop_b200 import FlashLoopConfig, FlashLoopEngine, mx_quantize
from flashloop_b200.mx import mx_status
from flashloop_b200.prefill import apply_rope
from tests.helpers import tiny_ouro_model

pytestmark = pytest.mark.gpu
STEP = 2.0 ** -8


def _held(x, format="mxfp8"):
    """The values of x in the format (which test_gpu_mx holds to the definition bit for bit)."""

    return mx_quantize(x, format).dequantize(torch.float32)


def _norm(x, norm, precision):
    x = x.to(precision)
    return (norm.weight.to(precision) * (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + norm.eps))).float()


def _linear(x, weight, precision):
    return (x.to(precision) @ weight.to(precision).t()).to(torch.bfloat16)


class Weights:
    """The rounded weights of a layer, from a model that nothing has repacked."""

    def __init__(self, layer, format):
        a, m = layer.self_attn, layer.mlp
        self.qkv = torch.cat([_held(p.weight.detach(), format) for p in (a.q_proj, a.k_proj, a.v_proj)])
        self.out, self.gate, self.up, self.down = (
            _held(p.weight.detach(), format) for p in (a.o_proj, m.gate_proj, m.up_proj, m.down_proj))


def _mlp(x, w, precision):
    gate, up = (x.to(precision) @ t.to(precision).t() for t in (w.gate, w.up))
    return _linear(_held((F.silu(gate) * up).float()), w.down, precision)


def _reference_prefill(model, weights, prompts, precision):
    """Four dense loops; the logits of the last token."""

    backbone = model.model
    hidden = backbone.embed_tokens(prompts)
    batch, tokens, _ = hidden.shape
    cos, sin = backbone.rotary_emb(hidden, torch.arange(tokens, device="cuda")[None].expand(batch, -1))
    future = torch.ones(tokens, tokens, dtype=torch.bool, device="cuda").triu(1)
    mask = torch.zeros(batch, 1, tokens, tokens, dtype=hidden.dtype, device="cuda").masked_fill_(future, float("-inf"))
    for loop in range(4):
        # the late loops attend under an explicit mask, as their rows need not be all of the prompt
        how = dict(is_causal=True) if loop < 2 else dict(attn_mask=mask)
        for layer, w in zip(backbone.layers, weights):
            rows = _held(_norm(hidden, layer.input_layernorm, precision))
            q, k, v = (t.view(batch, tokens, -1, 128).transpose(1, 2) for t in _linear(rows, w.qkv, precision).chunk(3, -1))
            q, k = apply_rope(q, k, cos, sin)
            out = F.scaled_dot_product_attention(q, k.contiguous(), v.contiguous(), **how)
            out = _linear(_held(out.transpose(1, 2).reshape(batch, tokens, -1)), w.out, precision)
            hidden = (hidden.float() + _norm(out, layer.input_layernorm_2, precision)).to(torch.bfloat16)
            m = _mlp(_held(_norm(hidden, layer.post_attention_layernorm, precision)), w, precision)
            hidden = hidden + layer.post_attention_layernorm_2(m)
        hidden = backbone.norm(hidden)
    return model.lm_head(hidden[:, -1]).float()


class ReferenceDecode(FlashLoopEngine):
    """The engine with its decode step in elementary operations (but for the cache's own calls)."""

    def _decode_step_microscaled(self, token_ids, position_ids):
        batch, layers, precision = token_ids.shape[0], self.layers, self.precision
        hidden = self.backbone.embed_tokens(token_ids)
        cos, sin = self.backbone.rotary_emb(hidden, position_ids)
        keys, values = ([[None] * 4 for _ in layers] for _ in range(2))
        sources = [None] * len(layers)
        for loop in range(4):
            for i, (layer, w) in enumerate(zip(layers, self.reference_weights)):
                rows = _held(_norm(hidden, layer.input_layernorm, precision))
                q, k, v = (t.view(batch, 1, -1, 128).transpose(1, 2).contiguous() for t in _linear(rows, w.qkv, precision).chunk(3, -1))
                q, k = (t.contiguous() for t in apply_rope(q, k, cos, sin))
                if loop >= 2 and self._reuse:
                    q, k = None, keys[i][1]
                keys[i][loop], values[i][loop] = k, v
                out, addend, keep = self._attend(loop, i, q, k, v, float(layer.self_attn.scaling), sources,
                                                 lambda t, w=w: _linear(_held(t), w.out, precision), batch, convert=False)
                if keep:
                    sources[i][0] = out
                if addend is not None:
                    out = (addend.float() + out.float()).to(torch.bfloat16)
                hidden = (hidden.float() + _norm(out, layer.input_layernorm_2, precision)).to(torch.bfloat16)
                m = _mlp(_held(_norm(hidden, layer.post_attention_layernorm, precision)), w, precision)
                if i + 1 < len(layers):
                    hidden = (hidden.float() + _norm(m, layer.post_attention_layernorm_2, precision)).to(torch.bfloat16)
                else:
                    hidden = hidden + layer.post_attention_layernorm_2(m)
            hidden = self.backbone.norm(hidden)
        for i in range(len(layers)):
            self.state.cache.layers[i].append_decode_token(keys[i], values[i])
        return self.model.lm_head(hidden[:, -1]).float()


def _off(got, want):
    return float((got - want).norm() / want.norm())


@pytest.mark.parametrize("format,batch", [("mxfp4", 2), ("mxfp8", 3)])
def test_microscaled_prefill(format, batch):
    prompts = torch.randint(0, 256, (batch, 150), generator=torch.Generator().manual_seed(batch)).cuda()
    model = tiny_ouro_model().cuda()
    with torch.inference_mode():
        weights = [Weights(layer, format) for layer in model.model.layers]
        want, other = (_reference_prefill(model, weights, prompts, p) for p in (torch.float64, torch.float32))
        engine = FlashLoopEngine(model, validate_model=False, max_new_tokens=16, projection_format=format,
                                 config=FlashLoopConfig(enable_token_sparse_prefill=False))
        off = _off(engine.prefill(prompts).logits, want)
        spread = _off(other, want)
        assert off <= 4 * spread + STEP and spread < 0.1, (off, spread)
    assert mx_status() == 0
    layer = engine.layers[0]
    assert layer.self_attn._flashloop_qkv_weight is None and layer.mlp.down_proj.weight is None


@pytest.mark.parametrize("format,batch,config", [
    ("mxfp4", 2, dict(enable_sparse_decode=False)), ("mxfp8", 3, dict(enable_sparse_decode=False)),
    ("mxfp4", 19, dict(enable_sparse_decode=False)), ("mxfp4", 2, {}), ("mxfp8", 2, dict(reuse_selected_probabilities=True))])
def test_microscaled_decode(format, batch, config):
    g = torch.Generator().manual_seed(batch)
    prompts = torch.randint(0, 256, (batch, 150), generator=g).cuda()
    tokens = [torch.randint(0, 256, (batch, 1), generator=g).cuda() for _ in range(7)]
    logits = []
    with torch.inference_mode():
        weights = [Weights(layer, format) for layer in tiny_ouro_model().cuda().model.layers]
        for kind, precision in ((FlashLoopEngine, None), (ReferenceDecode, torch.float64), (ReferenceDecode, torch.float32)):
            engine = kind(tiny_ouro_model().cuda(), validate_model=False, max_new_tokens=16, projection_format=format,
                          config=FlashLoopConfig(**config))
            engine.reference_weights, engine.precision = weights, precision
            engine.prefill(prompts)
            logits.append([engine.decode(t).logits for t in tokens])
    got, want, other = logits
    off, spread = (torch.tensor([_off(a, b) for a, b in zip(t, want)]) for t in (got, other))
    middle = config.get("enable_sparse_decode", True)
    off, spread = (float(t.median() if middle else t.max()) for t in (off, spread))
    assert off <= 4 * spread + STEP and spread < 0.1, (off, spread)
    assert mx_status() == 0


def test_microscaled_decode_in_a_graph_and_generation():
    prompts = torch.randint(0, 256, (2, 140), generator=torch.Generator().manual_seed(5)).cuda()
    outs, logits = [], []
    for graph in (False, True):
        engine = FlashLoopEngine(tiny_ouro_model().cuda(), validate_model=False, max_new_tokens=16, use_cuda_graph=graph,
                                 projection_format="mxfp4")
        outs.append(engine.generate(prompts, max_new_tokens=6))
        engine.reset()
        engine.prefill(prompts)
        tokens = torch.arange(6, device="cuda")[:, None, None].expand(6, 2, 1)
        logits.append(torch.stack([engine.decode(t.contiguous()).logits for t in tokens]))
    assert outs[0].shape == outs[1].shape == (2, 146)
    # the same launches; the readers merge their partial sums in arrival order
    torch.testing.assert_close(logits[0], logits[1], rtol=0, atol=0.25)
    assert float((logits[0] - logits[1]).abs().median()) < 1e-3


def test_microscaled_engine_refusals():
    with pytest.raises(ValueError, match="unknown microscaled format"):
        FlashLoopEngine(tiny_ouro_model().cuda(), validate_model=False, projection_format="int4")
    with pytest.raises(ValueError, match="fused projection weights"):
        FlashLoopEngine(tiny_ouro_model().cuda(), validate_model=False, projection_format="mxfp4", fuse_decode_ops=False)
    with pytest.raises(ValueError, match="fused projection weights"):
        FlashLoopEngine(tiny_ouro_model().cuda(), validate_model=False, projection_format="mxfp4",
                        config=FlashLoopConfig(fuse_projection_weights=False))
    model = tiny_ouro_model().cuda()
    FlashLoopEngine(model, validate_model=False, projection_format="mxfp4")
    FlashLoopEngine(model, validate_model=False, projection_format="mxfp4")  # holds them already
    with pytest.raises(RuntimeError, match="already held"):
        FlashLoopEngine(model, validate_model=False, projection_format="mxfp8")
    with pytest.raises(ValueError, match="microscaled"):
        FlashLoopEngine(model, validate_model=False)
