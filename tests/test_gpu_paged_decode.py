"""Decoder layers over a paged cache, prompt and steps, against the dense layers' oracle run over each sample's whole sequence."""
from __future__ import annotations

import dataclasses

import pytest
import torch

from aginfer_b200.recipes import paged_decode
from aginfer_b200.recipes.decoder_layer import LayerConfig
from aginfer_b200.recipes.package import build_aim, describe
from oracle import decoder_layer as oracle_layer
from oracle import ops

pytestmark = pytest.mark.gpu


def dense(cfg, weights, hidden):
    """All layers of ``cfg`` over one sequence."""
    layer = dataclasses.replace(cfg.layer, tokens=hidden.shape[0])
    for i in range(cfg.layers):
        mine = {n.replace(f"layers.{i}.", "layers.0."): t for n, t in weights.items() if f"layers.{i}." in n}
        hidden = oracle_layer.forward(layer, mine, hidden)
    return hidden


def run(tmp_path, cfg, prompt, steps):
    weights = paged_decode.synthetic_weights(cfg, seed=4)
    serving = paged_decode.Serving(build_aim(tmp_path, weights, paged_decode.build_recipe(cfg, describe(weights))), cfg)
    out = [serving.prompt(prompt.cuda()).cpu()]
    for s in steps:
        out.append(serving.step(s.cuda()).cpu())
    assert serving.status() == 0
    return weights, out


@pytest.mark.parametrize("heads,kv_heads,d,page,tokens,window", [(4, 2, 64, 16, 70, 0), (7, 1, 128, 32, 288, 0), (4, 2, 64, 16, 80, 4096)], ids=str)
def test_steps_continue_the_prompt(tmp_path, heads, kv_heads, d, page, tokens, window):
    """A window longer than the sequences shows everything, so all of these are dense causal attention."""
    cfg = paged_decode.ServeConfig(layer=LayerConfig(hidden=256, heads=heads, kv_heads=kv_heads, head_dim=d, intermediate=704, tokens=tokens),
                                   layers=2, sequences=3, page=page, new_tokens=5, window=window, sinks=4 if window else 0)
    g = torch.Generator().manual_seed(2)
    prompt = torch.randn(tokens, 256, generator=g).to(torch.bfloat16)
    steps = [torch.randn(3, 256, generator=g).to(torch.bfloat16) for _ in range(5)]
    weights, out = run(tmp_path, cfg, prompt, steps)
    # 2e-2, the BF16 tier's bound for a layer's output
    assert ops.max_rel_err(out[0], dense(cfg, weights, prompt)) < 2e-2
    for b in range(3):
        whole = dense(cfg, weights, torch.cat([prompt, *[s[b:b + 1] for s in steps]]))
        got = torch.stack([o[b] for o in out[1:]])
        assert ops.max_rel_err(got, whole[tokens:]) < 2e-2, b


def test_a_sample_stops_at_its_pages(tmp_path):
    cfg = paged_decode.ServeConfig(layer=LayerConfig(hidden=256, heads=4, kv_heads=2, head_dim=64, intermediate=704, tokens=16), layers=1,
                                   sequences=2, page=16, new_tokens=1)
    x = torch.zeros(2, 256, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        run(tmp_path, cfg, torch.zeros(16, 256, dtype=torch.bfloat16), [x, x])
