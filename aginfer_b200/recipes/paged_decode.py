"""Decoder layers served token by token over a paged K/V cache: a prompt that fills pages once, then steps of a batch of samples
that go on from it.

    python -m aginfer_b200.recipes.paged_decode [--layers 2] [--sequences 8] [--tokens 288] [--steps 64] [--window 0]

The layers are those of ``decoder_layer`` (BF16; same checkpoint names, ``model.layers.{i}``).  Two profiles share the package:

* ``prompt``  the prompt's tokens, one sequence: ``kv_append``, ``paged_attention`` over what it has just appended;
* ``step``    one new token of every sample: ``kv_append`` with the prompt's length as the rotary offset, then ``prefix_attention``
              (the prompt's pages are read once for all samples).  With ``window`` the samples' tables begin with the prompt's
              pages instead, and ``paged_attention`` keeps the last ``window`` tokens and the first ``sinks``.

The pools are tensors of the caller, bound as outputs of both profiles: a profile writes into its pages and leaves the rest.
``Serving`` keeps pools, tables and lengths on the device and runs both profiles on them.
"""
from __future__ import annotations

import argparse
import json
import tempfile
from dataclasses import dataclass, field
from pathlib import Path

from .builder import PagedCache, RecipeBuilder, Tensor, Weight, ceil_div, io
from .decoder_layer import LayerConfig, linear_shapes

BF = 2


@dataclass(frozen=True)
class ServeConfig:
    layer: LayerConfig = field(default_factory=LayerConfig)      # ``layer.tokens``: tokens of the prompt
    layers: int = 2
    sequences: int = 8
    page: int = 64
    new_tokens: int = 64             # the most that a sample generates
    window: int = 0
    sinks: int = 0

    def __post_init__(self) -> None:
        if self.layer.fp8:
            raise ValueError("the paged decoder has BF16 layers")
        if self.window and self.layer.tokens % self.page:
            raise ValueError("samples that share the prompt's pages in their tables need a prompt of whole pages")

    @property
    def prompt_pages(self) -> int:
        return ceil_div(self.layer.tokens, self.page)

    @property
    def own_pages(self) -> int:
        return ceil_div(self.new_tokens, self.page)

    @property
    def table_pages(self) -> int:
        return self.own_pages + (self.prompt_pages if self.window else 0)

    @property
    def pages(self) -> int:
        return self.prompt_pages + self.sequences * self.own_pages

    @property
    def pool_shape(self) -> list[int]:
        c = self.layer
        return [self.pages, c.kv_heads, c.head_dim // 64, self.page, 64]


def synthetic_weights(cfg: ServeConfig, seed: int = 0) -> dict:
    from . import decoder_layer
    out = {}
    for i in range(cfg.layers):
        for name, t in decoder_layer.synthetic_weights(cfg.layer, seed + i).items():
            out[name.replace("layers.0.", f"layers.{i}.")] = t
    return out


def _layer(r: RecipeBuilder, cfg: ServeConfig, i: int, x, y, rows: int, cache: PagedCache, append, attend) -> None:
    """Layer i over ``rows`` rows, ``x`` -> ``y``; ``append`` and ``attend`` are the operators' arguments that the profiles differ in."""
    c, H, I = cfg.layer, cfg.layer.hidden, cfg.layer.intermediate
    w = lambda name: Weight(f"model.layers.{i}.{name}")  # noqa: E731
    qkv_dim, mark = c.q_dim + 2 * c.kv_dim, r.mark()
    normed, qkv, q = r.alloc(rows * H * BF), r.alloc(rows * qkv_dim * BF), r.alloc(rows * c.q_dim * BF)
    attn, resid, gate_up, act = r.alloc(rows * c.q_dim * BF), r.alloc(rows * H * BF), r.alloc(rows * 2 * I * BF), r.alloc(rows * I * BF)
    r.rmsnorm(x, w("input_layernorm.weight"), normed, rows, H, c.eps)
    col = 0
    for name, width in (("q_proj", c.q_dim), ("k_proj", c.kv_dim), ("v_proj", c.kv_dim)):
        r.gemm(normed, w(f"self_attn.{name}.weight"), qkv + col * BF if col else qkv, rows, width, H, bias=w(f"self_attn.{name}.bias"), ldy=qkv_dim)
        col += width
    r.kv_append(qkv, q, cache, rows=rows, q_heads=c.heads, theta=c.theta, **append)
    attend(q, attn)
    r.gemm(attn, w("self_attn.o_proj.weight"), resid, rows, H, c.q_dim, residual=x)
    r.rmsnorm(resid, w("post_attention_layernorm.weight"), normed, rows, H, c.eps)
    r.gemm(normed, w("mlp.gate_proj.weight"), gate_up, rows, I, H, ldy=2 * I)
    r.gemm(normed, w("mlp.up_proj.weight"), gate_up + I * BF, rows, I, H, ldy=2 * I)
    r.swiglu(gate_up, gate_up + I * BF, act, rows, I, 2 * I)
    r.gemm(act, w("mlp.down_proj.weight"), y, rows, H, I, residual=resid)
    r.release(mark)


def build_recipe(cfg: ServeConfig, weights) -> RecipeBuilder:
    """``weights``: name -> (dtype, shape) as from ``package.describe``."""
    c = cfg.layer
    r = RecipeBuilder(weights)
    hidden = [r.alloc(max(c.tokens, cfg.sequences) * c.hidden * BF) for _ in range(2)]
    pools = [io(f"{kind}{i}", "BF16", cfg.pool_shape) for i in range(cfg.layers) for kind in "kv"]

    def profile(name: str, rows: int, sequences: int, table_pages: int, shared: bool) -> None:
        extra = [io("prefix_table", "I32", [cfg.prompt_pages]), io("prefix_length", "I32", [1])] if shared else []
        r.begin_profile(name, [io("hidden_in", "BF16", [rows, c.hidden]), io("starts", "I32", [sequences + 1]), io("lengths", "I32", [sequences]),
                               io("table", "I32", [sequences, table_pages]), *extra],
                        [io("hidden_out", "BF16", [rows, c.hidden]), *pools, io("status", "I32", [1])])
        at = Tensor("hidden_in")
        for i in range(cfg.layers):
            cache = PagedCache(k=Tensor(f"k{i}"), v=Tensor(f"v{i}"), table=Tensor("table"), lengths=Tensor("lengths"), starts=Tensor("starts"),
                               sequences=sequences, pages=cfg.pages, page=cfg.page, pages_per_sequence=table_pages, kv_heads=c.kv_heads,
                               head_dim=c.head_dim)
            longest = rows if sequences == 1 else 1

            def attend(q, o, cache=cache, longest=longest):
                if shared:
                    r.prefix_attention(q, o, cache, Tensor("prefix_table"), Tensor("prefix_length"), prefix_pages=cfg.prompt_pages, rows=rows,
                                       q_heads=c.heads, longest=longest)
                else:
                    r.paged_attention(q, o, cache, rows=rows, q_heads=c.heads, longest=longest, window=cfg.window, sinks=cfg.sinks)

            to = Tensor("hidden_out") if i == cfg.layers - 1 else hidden[i % 2]
            _layer(r, cfg, i, at, to, rows, cache, {"offset": Tensor("prefix_length")} if shared else {}, attend)
            at = to
        r.export_status(Tensor("status"))

    profile("prompt", c.tokens, 1, cfg.prompt_pages, False)
    profile("step", cfg.sequences, cfg.sequences, cfg.table_pages, not cfg.window)
    return r


class Serving:
    """A packaged ``build_recipe`` with its pools, tables and lengths on the current device."""

    def __init__(self, aim: Path, cfg: ServeConfig):
        import torch

        from .. import runtime as rt
        from ..runner import Runner
        self.cfg = cfg
        self.runners = {p: Runner(aim, profile=p, flags=rt.PROGRAMMATIC_LAUNCH) for p in ("prompt", "step")}
        self.pools = {f"{kind}{i}": torch.zeros(cfg.pool_shape, dtype=torch.bfloat16, device="cuda") for i in range(cfg.layers) for kind in "kv"}
        ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        c, B, own, prompt = cfg.layer, cfg.sequences, cfg.own_pages, list(range(cfg.prompt_pages))
        pages = [[cfg.prompt_pages + b * own + j for j in range(own)] for b in range(B)]
        self.batch = {"prompt": {"starts": ints([0, c.tokens]), "lengths": ints([c.tokens]), "table": ints([prompt])},
                      "step": {"starts": ints(list(range(B + 1))), "lengths": ints([c.tokens if cfg.window else 0] * B),
                               "table": ints([(prompt if cfg.window else []) + p for p in pages])}}
        if not cfg.window:
            self.batch["step"] |= {"prefix_table": ints(prompt), "prefix_length": ints([c.tokens])}
        self.steps = 0
        self.out = {p: {"hidden_out": torch.empty(rows, c.hidden, dtype=torch.bfloat16, device="cuda"), **self.pools,
                        "status": torch.zeros(1, dtype=torch.int32, device="cuda")} for p, rows in (("prompt", c.tokens), ("step", B))}

    def _run(self, profile: str, hidden):
        self.runners[profile].run({"hidden_in": hidden, **self.batch[profile]}, self.out[profile])
        return self.out[profile]["hidden_out"]

    def prompt(self, hidden):
        """Hidden states [tokens, hidden] of the prompt -> those behind the last layer (the buffer of the next call too).  The
        samples begin anew behind it: what they generated from the prompt before is not looked at any more."""
        self.steps = 0
        self.batch["step"]["lengths"].fill_(self.cfg.layer.tokens if self.cfg.window else 0)      # in place: the graphs keep its address
        return self._run("prompt", hidden)

    def step(self, hidden):
        """Hidden states [sequences, hidden] of every sample's next token -> those behind the last layer."""
        if self.steps >= self.cfg.new_tokens:
            raise ValueError(f"a sample generates at most {self.cfg.new_tokens} tokens")
        self.steps += 1
        self.batch["step"]["lengths"] += 1
        return self._run("step", hidden)

    def status(self) -> int:
        """The status words of both profiles' last runs (0: nothing to report); waits for them."""
        return max(int(o["status"].item()) for o in self.out.values())


def main() -> None:
    import torch

    from .package import build_aim, describe
    ap = argparse.ArgumentParser()
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--sequences", type=int, default=8)
    ap.add_argument("--tokens", type=int, default=288)
    ap.add_argument("--steps", type=int, default=64)
    ap.add_argument("--page", type=int, default=32)
    ap.add_argument("--window", type=int, default=0)
    ap.add_argument("--sinks", type=int, default=0)
    args = ap.parse_args()
    cfg = ServeConfig(layer=LayerConfig(tokens=args.tokens), layers=args.layers, sequences=args.sequences, page=args.page,
                      new_tokens=2 * args.steps + 3, window=args.window, sinks=args.sinks)
    weights = synthetic_weights(cfg)
    with tempfile.TemporaryDirectory(prefix="agi_paged_") as tmp:
        serving = Serving(build_aim(Path(tmp), weights, build_recipe(cfg, describe(weights))), cfg)
    g = torch.Generator(device="cuda").manual_seed(1)
    randn = lambda rows: torch.randn(rows, cfg.layer.hidden, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
    timed = {}
    hidden, step = randn(args.tokens), randn(args.sequences)
    for name, call, count in (("prompt", lambda: serving.prompt(hidden), 8), ("step", lambda: serving.step(step), args.steps)):
        for _ in range(3):
            call()
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        for _ in range(count):
            call()
        end.record()
        torch.cuda.synchronize()
        timed[name] = start.elapsed_time(end) / count
    print(json.dumps({"workload": f"{cfg.layers} decoder layers, prompt of {args.tokens}, {args.sequences} samples, window {args.window}",
                      "ms_per_prompt": timed["prompt"], "ms_per_step": timed["step"], "tokens_per_s": args.sequences / timed["step"] * 1e3,
                      "launches_per_step": int(serving.runners["step"].stats()["launches_per_enqueue"]), "status": serving.status()}))


if __name__ == "__main__":
    main()
