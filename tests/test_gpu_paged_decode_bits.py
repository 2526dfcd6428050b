"""Decoder layers served with 4-bit weights and a cache in 8 bits, against the dense oracle with the weights that the codes stand for and keys
and values that go through the cache's rounding."""
from __future__ import annotations

import dataclasses

import pytest
import torch

from aginfer_b200.recipes import paged_decode
from aginfer_b200.recipes.decoder_layer import LayerConfig
from aginfer_b200.recipes.layout import unpack_w4
from aginfer_b200.recipes.package import build_aim, describe
from oracle import decoder_layer as oracle_layer
from oracle import ops
from tests.paged_e4m3_util import rounded

pytestmark = pytest.mark.gpu


def dense_weights(cfg, weights):
    """What a 4-bit checkpoint stands for, under the names of the dense layers."""
    if cfg.weight_bits == 16:
        return weights
    c, out = cfg.layer, dict(weights)
    rows = {"self_attn.qkv_proj": (("q_proj", c.q_dim), ("k_proj", c.kv_dim), ("v_proj", c.kv_dim)), "self_attn.o_proj": (("o_proj", c.hidden),),
            "mlp.gate_up_proj": (("gate_proj", c.intermediate), ("up_proj", c.intermediate)), "mlp.down_proj": (("down_proj", c.hidden),)}
    for i in range(cfg.layers):
        for name, parts in rows.items():
            at, row, total = f"model.layers.{i}.{name}", 0, sum(n for _, n in parts)
            w = unpack_w4(out.pop(f"{at}.weight").view(torch.int32), out.pop(f"{at}.weight_scale"), total)
            bias = out.pop(f"{at}.bias", None)
            for part, n in parts:
                to = f"model.layers.{i}.{name.split('.')[0]}.{part}"
                out[f"{to}.weight"] = w[row:row + n]
                if bias is not None:
                    out[f"{to}.bias"] = bias[row:row + n]
                row += n
    return out


def dense(cfg, weights, x):
    layer = dataclasses.replace(cfg.layer, tokens=x.shape[0])
    for i in range(cfg.layers):
        x = oracle_layer.forward(layer, {n.replace(f"layers.{i}.", "layers.0."): t for n, t in weights.items() if f"layers.{i}." in n}, x)
    return x


def hidden(rows: int, seed: int) -> torch.Tensor:
    return torch.randn(rows, 256, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16)


@pytest.mark.parametrize("weight_bits,cache_bits,tokens,window,heads", [
    (4, 16, 20, 0, (4, 2, 64)), (16, 8, 70, 0, (4, 2, 64)), (4, 8, 70, 0, (7, 1, 128)), (4, 8, 32, 4096, (4, 2, 64)), (4, 8, 40, 0, (4, 4, 64))], ids=str)
def test_prompt_and_steps(tmp_path, monkeypatch, weight_bits, cache_bits, tokens, window, heads):
    layer = LayerConfig(hidden=256, heads=heads[0], kv_heads=heads[1], head_dim=heads[2], intermediate=704, tokens=tokens)
    cfg = paged_decode.ServeConfig(layer=layer, layers=2, sequences=3, page=16, new_tokens=6, window=window, sinks=4 if window else 0,
                                   weight_bits=weight_bits, cache_bits=cache_bits)
    weights = {n: (t.float() * 6).to(t.dtype) if "o_proj" in n or "v_proj" in n else t for n, t in paged_decode.synthetic_weights(cfg, seed=4).items()}
    if weight_bits == 4:
        weights = paged_decode.quantize_weights(cfg, weights)
    serving = paged_decode.Serving(build_aim(tmp_path, weights, paged_decode.build_recipe(cfg, describe(weights))), cfg)
    exact = ops.attention
    if cache_bits == 8:      # keys and values as the cache holds them
        monkeypatch.setattr(ops, "attention", lambda q, k, v, mask: exact(q, rounded(k.to(torch.bfloat16)).float(), rounded(v.to(torch.bfloat16)).float(), mask=mask))
    plain = dense_weights(cfg, weights)
    # As for FP8 blocks: a rounding of the hidden states in front of a quantisation may be another code, so two right answers differ by more than
    # the 2e-2 of layers in bf16.
    bound = ops.FP8_BLOCK_TOL if cache_bits == 8 else 2e-2
    for request in range(2):
        prompt, steps = hidden(tokens, 10 * request), [hidden(3, 10 * request + 1 + i) for i in range(6)]
        got = [serving.prompt(prompt.cuda()).cpu(), *[serving.step(s.cuda()).cpu() for s in steps]]
        assert serving.status() == 0
        assert ops.max_rel_err(got[0], dense(cfg, plain, prompt)) < bound
        for b in range(3):
            whole = dense(cfg, plain, torch.cat([prompt, *[s[b:b + 1] for s in steps]]))
            assert ops.max_rel_err(torch.stack([o[b] for o in got[1:]]), whole[tokens:]) < bound, (request, b)


def test_a_replayed_step_and_a_fresh_one_agree(tmp_path):
    """Steps are replays of one graph: the second request's answer is bit for bit that of a server that has seen nothing before."""
    layer = LayerConfig(hidden=256, heads=4, kv_heads=2, head_dim=64, intermediate=704, tokens=38)
    cfg = paged_decode.ServeConfig(layer=layer, layers=2, sequences=3, page=16, new_tokens=5, weight_bits=4, cache_bits=8)
    weights = paged_decode.quantize_weights(cfg, paged_decode.synthetic_weights(cfg, seed=1))

    def answer(serving, request):
        out = [serving.prompt(hidden(38, request).cuda()).cpu(), *[serving.step(hidden(3, 100 * request + i).cuda()).cpu() for i in range(5)]]
        assert serving.status() == 0
        return out

    def server(name):
        (tmp_path / name).mkdir()
        return paged_decode.Serving(build_aim(tmp_path / name, weights, paged_decode.build_recipe(cfg, describe(weights))), cfg)

    kept = server("kept")
    answer(kept, 1)
    assert all(torch.equal(a, b) for a, b in zip(answer(kept, 2), answer(server("fresh"), 2)))
