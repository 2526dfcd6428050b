"""Paged caches in 8 bits for the tests: the batches of ``paged_util`` with their tokens rounded to codes, any byte and a scale of NaN wherever no
token is."""
from __future__ import annotations

from dataclasses import dataclass

import torch

from aginfer_b200.recipes import PagedCache, Tensor
from aginfer_b200.recipes.layout import quantize_kv_pages, read_kv_pages, unpack_kv_pages
from tests.paged_util import BF, Batch

POOLS = ("k", "v", "k_scale", "v_scale")


def rounded(t: torch.Tensor) -> torch.Tensor:
    """Tokens [tokens, kv_heads, head_dim] as the cache holds them (their codes times their scales, exact in bf16)."""
    return read_kv_pages(*quantize_kv_pages(t[None])).squeeze(0).to(BF) if t.shape[0] else t


@dataclass
class Batch8(Batch):
    spread: int = 0                      # tokens and heads of unequal size: factors 2^-spread .. 2^spread

    def __post_init__(self):
        super().__post_init__()
        g = torch.Generator().manual_seed(self.seed + 1000)
        self.pools = {}
        held = None
        for name in "kv":
            t = unpack_kv_pages(getattr(self, name)).float()
            held = ~t[..., 0].isnan()
            if self.spread:
                t = torch.ldexp(t, torch.randint(-self.spread, self.spread + 1, t.shape[:3], generator=g)[..., None])
            codes, scales = quantize_kv_pages(t.to(BF))
            noise = torch.randint(0, 256, codes.shape, generator=g).to(torch.uint8)
            gone = ~held.permute(0, 2, 1)
            self.pools[name] = torch.where(gone[..., None], noise, codes).contiguous()
            self.pools[name + "_scale"] = scales.contiguous()
            tokens = read_kv_pages(codes, scales).to(BF)
            pick = lambda pages, count: torch.stack([tokens[pages[j // self.page], j % self.page] for j in range(count)]) if count > 0 else tokens[0, :0]  # noqa: B023,E731
            lists = [pick(self.table[b].tolist(), t) for b, t in enumerate(self.total)]
            if name == "k":
                self.keys = lists
            else:
                self.values = lists
            if self.prefix:
                shared = pick(self.prefix_table.tolist(), self.prefix)
                self.prefix_kv = (shared, None) if name == "k" else (self.prefix_kv[0], shared)

    def cache(self, **names) -> PagedCache:
        hq, hk, d = self.heads
        p = {n: Tensor(n) for n in (*POOLS, "table", "lengths", "starts")} | names
        return PagedCache(**p, sequences=len(self.new), pages=self.pages, page=self.page, pages_per_sequence=self.width, kv_heads=hk, head_dim=d)

    def inputs(self) -> dict:
        return super().inputs() | self.pools
