"""Paged K/V caches for the tests: a batch whose pages lie in no order in a pool that holds NaN wherever no token is."""
from __future__ import annotations

from dataclasses import dataclass, field

import torch

from aginfer_b200 import runtime as rt
from aginfer_b200.recipes import PagedCache, RecipeBuilder, Tensor
from aginfer_b200.recipes.layout import pack_kv_pages
from aginfer_b200.recipes.package import build_aim, describe
from aginfer_b200.runner import Runner
from oracle import paged
from tests.gpu_util import spec

BF = torch.bfloat16
# Of sum p |v|: half a bf16 step (2^-8) where the weights are rounded before they meet the values, as much where the output is,
# and scores of 128 products in 32 bits are off by less than 2^-10.
BOUND = 2.0 ** -7 + 2.0 ** -10


@dataclass
class Batch:
    new: list
    total: list
    page: int = 16
    heads: tuple = (4, 2, 64)            # query heads, key heads, width
    prefix: int = 0
    spare_rows: int = 0                  # rows of no sequence behind the others
    sharp: float = 1.0                   # factor on the queries
    seed: int = 0
    extra: dict = field(default_factory=dict)

    def __post_init__(self):
        hq, hk, d = self.heads
        g = torch.Generator().manual_seed(self.seed)
        randn = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
        self.rows = sum(self.new) + self.spare_rows
        self.longest = max(1, *self.new)
        counts = [-(-t // self.page) for t in self.total]
        self.width = max(1, *counts)
        self.prefix_pages = max(1, -(-self.prefix // self.page))
        self.pages = sum(counts) + self.prefix_pages + 3
        order = torch.randperm(self.pages, generator=g).tolist()
        self.prefix_table = torch.tensor(order[:self.prefix_pages], dtype=torch.int32)
        at, self.table = self.prefix_pages, torch.full((len(self.new), self.width), -7, dtype=torch.int32)
        k = torch.full((self.pages, self.page, hk, d), float("nan"))
        v = torch.full((self.pages, self.page, hk, d), float("nan"))
        self.keys, self.values = [], []
        for b, (t, n) in enumerate(zip(self.total, counts)):
            mine = order[at:at + n]
            at += n
            self.table[b, :n] = torch.tensor(mine, dtype=torch.int32)
            self.keys.append(self._fill(k, mine, t, randn))
            self.values.append(self._fill(v, mine, t, randn))
        self.prefix_kv = None
        if self.prefix:
            self.prefix_kv = tuple(self._fill(pool, order[:self.prefix_pages], self.prefix, randn) for pool in (k, v))
        self.k, self.v = pack_kv_pages(k.to(BF)), pack_kv_pages(v.to(BF))
        self.starts = torch.tensor([sum(self.new[:b]) for b in range(len(self.new) + 1)], dtype=torch.int32)
        self.lengths = torch.tensor(self.total, dtype=torch.int32)
        self.q = (self.sharp * randn(self.rows, hq * d)).to(BF)

    def _fill(self, pool, pages, tokens, randn):
        t = randn(max(tokens, 0), *pool.shape[2:]).to(BF)
        for j in range(tokens):
            pool[pages[j // self.page], j % self.page] = t[j].float()
        return t

    def index(self, b: int, i: int) -> int:
        return self.total[b] - self.new[b] + i

    def expected(self, window: int = 0, sinks: int = 0, scale=None):
        """(o, mass) [rows, heads * head_dim] in 64 bits; rows of no sequence are NaN."""
        hq, _, d = self.heads
        o = torch.full((self.rows, hq * d), float("nan"), dtype=torch.float64)
        mass = torch.zeros_like(o)
        for b, n in enumerate(self.new):
            for i in range(n):
                row = int(self.starts[b]) + i
                one, m = paged.attention(self.q[row].view(hq, d), self.keys[b], self.values[b], self.index(b, i), window, sinks, scale,
                                         self.prefix_kv)
                o[row], mass[row] = one.reshape(-1), m.reshape(-1)
        return o, mass

    def cache(self, **names) -> PagedCache:
        hq, hk, d = self.heads
        p = {n: Tensor(n) for n in ("k", "v", "table", "lengths", "starts")} | names
        return PagedCache(**p, sequences=len(self.new), pages=self.pages, page=self.page, pages_per_sequence=self.width, kv_heads=hk,
                          head_dim=d)

    def inputs(self) -> dict:
        x = {"q": self.q, "k": self.k, "v": self.v, "table": self.table, "lengths": self.lengths, "starts": self.starts}
        if self.prefix:
            x |= {"prefix_table": self.prefix_table, "prefix_length": torch.tensor([self.prefix], dtype=torch.int32)}
        return x | self.extra

    def attend(self, r: RecipeBuilder, **kw) -> None:
        """The launches of the batch's attention in ``r``."""
        common = dict(rows=self.rows, q_heads=self.heads[0]) | kw
        if self.prefix:
            r.prefix_attention(Tensor("q"), Tensor("o"), self.cache(), Tensor("prefix_table"), Tensor("prefix_length"),
                               prefix_pages=self.prefix_pages, **common)
        else:
            r.paged_attention(Tensor("q"), Tensor("o"), self.cache(), **common)
        r.export_status(Tensor("status"))


def packaged(tmp_path, inputs: dict, outputs: dict, body, flags: int = rt.PROGRAMMATIC_LAUNCH):
    """(runner, device inputs, device outputs) of a one-profile recipe; ``outputs`` are the tensors that the buffers start as."""
    weights = {"unused.pad": torch.zeros(8, dtype=BF)}
    r = RecipeBuilder(describe(weights))
    r.begin_profile("default", [spec(n, t) for n, t in inputs.items()], [spec(n, t) for n, t in outputs.items()])
    body(r)
    runner = Runner(build_aim(tmp_path, weights, r), flags=flags)
    return runner, {n: t.cuda() for n, t in inputs.items()}, {n: t.cuda() for n, t in outputs.items()}


def attention_outputs(batch: Batch) -> dict:
    return {"o": torch.full((batch.rows, batch.heads[0] * batch.heads[2]), 77.0).to(BF), "status": torch.zeros(1, dtype=torch.int32)}


def check(batch: Batch, got: torch.Tensor, window: int = 0, sinks: int = 0, scale=None) -> None:
    want, mass = batch.expected(window, sinks, scale)
    live = ~want.isnan()
    error = (got.double() - want).abs()
    assert bool((got[~live] == 77.0).all()), "rows of no sequence were written"
    assert bool(got[live].isfinite().all())
    worst = (error - BOUND * mass)[live]
    assert worst.numel() == 0 or worst.max() <= 0, f"{worst.max():.3g} over the bound, largest error {error[live].max():.3g}"
