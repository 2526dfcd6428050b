"""``paged_decode.Serving`` over more than one request, under windows that hide something, and at its limits, against a dense oracle that
runs every sample's whole sequence."""
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

BOUND = 2e-2        # the BF16 tier's bound for a layer's output


def served(tmp_path, **kw):
    tmp_path.mkdir(exist_ok=True)
    tokens, window = kw.pop("tokens", 32), kw.pop("window", 0)
    layer = LayerConfig(hidden=256, heads=4, kv_heads=2, head_dim=64, intermediate=704, tokens=tokens)
    cfg = paged_decode.ServeConfig(layer=layer, sequences=3, page=16, window=window, **kw)
    # attention weighs as much as the rest of a layer does, so that a wrong token in sight shows
    weights = {n: (t.float() * 6).to(t.dtype) if "o_proj" in n or "v_proj" in n else t for n, t in paged_decode.synthetic_weights(cfg, seed=4).items()}
    return cfg, weights, paged_decode.Serving(build_aim(tmp_path, weights, paged_decode.build_recipe(cfg, describe(weights))), cfg)


def hidden(rows: int, seed: int) -> torch.Tensor:
    return torch.randn(rows, 256, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16)


def dense(cfg, weights, x):
    layer = dataclasses.replace(cfg.layer, tokens=x.shape[0])
    for i in range(cfg.layers):
        x = oracle_layer.forward(layer, {n.replace(f"layers.{i}.", "layers.0."): t for n, t in weights.items() if f"layers.{i}." in n}, x)
    return x


@pytest.mark.parametrize("tokens,window", [(38, 0), (32, 4096)], ids=str)
def test_a_second_prompt_is_answered_as_if_it_were_the_first(tmp_path, tokens, window):
    """The second request would still fit behind the first one's answer; with the third there are more steps than one has pages for."""
    kw = dict(tokens=tokens, window=window, sinks=4 if window else 0, layers=2, new_tokens=18)
    cfg, weights, serving = served(tmp_path / "kept", **kw)
    for request, count in enumerate((3, 12, 18)):
        prompt, steps = hidden(tokens, 10 * request), [hidden(3, 10 * request + 1 + i) for i in range(count)]

        def answer(server):
            out = [server.prompt(prompt.cuda()).cpu(), *[server.step(s.cuda()).cpu() for s in steps]]
            assert server.status() == 0
            return out

        got, fresh = answer(serving), answer(served(tmp_path / f"fresh{request}", **kw)[2])
        assert all(torch.equal(a, b) for a, b in zip(got, fresh)), request
        assert ops.max_rel_err(got[0], dense(cfg, weights, prompt)) < BOUND
        for b in range(3):
            whole = dense(cfg, weights, torch.cat([prompt, *[s[b:b + 1] for s in steps]]))
            assert ops.max_rel_err(torch.stack([o[b] for o in got[1:]]), whole[tokens:]) < BOUND, (request, b)


def test_a_window_that_hides_most_of_the_prompt(tmp_path, monkeypatch):
    """Shared pages in the samples' tables, first tokens inside the prompt, a window that begins in the prompt and leaves it."""
    window, sinks = 12, 3
    cfg, weights, serving = served(tmp_path, tokens=48, window=window, sinks=sinks, layers=2, new_tokens=20)
    prompt, steps = hidden(48, 1), [hidden(3, 2 + i) for i in range(20)]
    got = [serving.prompt(prompt.cuda()).cpu(), *[serving.step(s.cuda()).cpu() for s in steps]]
    assert serving.status() == 0
    samples = [torch.cat([prompt, *[s[b:b + 1] for s in steps]]) for b in range(3)]
    everything = [dense(cfg, weights, x) for x in samples]

    def windowed(q, k, v, *, mask):
        assert mask == "causal"
        i, j = torch.arange(q.shape[0])[:, None], torch.arange(k.shape[0])[None, :]
        seen = (j <= i) & ((i - j < window) | (j < sinks))
        k, v = (t.float().repeat_interleave(q.shape[1] // t.shape[1], dim=1) for t in (k, v))
        score = torch.einsum("ihd,jhd->hij", q.float() * q.shape[2] ** -0.5, k).masked_fill(~seen, float("-inf"))
        return ops.bf16_round(torch.einsum("hij,jhd->ihd", torch.softmax(score, dim=-1), v))

    monkeypatch.setattr(ops, "attention", windowed)
    for b in range(3):
        want, answer = dense(cfg, weights, samples[b]), torch.cat([got[0], *[o[b:b + 1] for o in got[1:]]])
        assert ops.max_rel_err(answer, want) < BOUND, b
        assert ops.max_rel_err(everything[b][window:], want[window:]) > 5 * BOUND        # the window does hide something


def test_a_sample_stops_at_its_pages_and_not_before(tmp_path):
    _, _, serving = served(tmp_path, tokens=16, layers=1, new_tokens=2)
    x = hidden(3, 1).cuda()
    serving.prompt(hidden(16, 0).cuda())
    serving.step(x)
    serving.step(x)
    with pytest.raises(ValueError, match="a sample generates at most 2 tokens"):
        serving.step(x)
    assert serving.status() == 0
