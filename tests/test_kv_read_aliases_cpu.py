"""What bringing the pages of a cache in 8 bits back writes shares no memory with what it reads, in the arena too, where pointers may differ and ranges
meet all the same."""
from __future__ import annotations

import pytest

from aginfer_b200.recipes import Arena, PagedCache, RecipeBuilder, Tensor, io

KV, DIM, PAGES, PAGE, SEQUENCES, WIDTH = 2, 128, 9, 16, 3, 4
POOL, SCALES, WIDE = PAGES * KV * PAGE * DIM, PAGES * KV * PAGE * 2, SEQUENCES * WIDTH * KV * PAGE * DIM * 2       # bytes
AT = Arena(1 << 24)


def read(**kw) -> None:
    r = RecipeBuilder({"w": ("BF16", (8,))})
    codes, scales = [PAGES, KV, PAGE, DIM], [PAGES, KV, PAGE]
    r.begin_profile("default", [io("k", "F8_E4M3", codes), io("v", "F8_E4M3", codes), io("ks", "BF16", scales), io("vs", "BF16", scales),
                                io("table", "I32", [SEQUENCES, WIDTH]), io("lengths", "I32", [SEQUENCES]), io("starts", "I32", [SEQUENCES + 1])],
                    [io("k16", "BF16", [12, KV, 2, PAGE, 64]), io("v16", "BF16", [12, KV, 2, PAGE, 64]), io("table16", "I32", [SEQUENCES, WIDTH])])
    p = {n: Tensor(n) for n in ("k", "v", "ks", "vs", "k16", "v16", "table", "table16", "lengths", "starts")} | kw
    shape = dict(sequences=SEQUENCES, page=PAGE, pages_per_sequence=WIDTH, kv_heads=KV, head_dim=DIM, lengths=p["lengths"], starts=p["starts"])
    r.kv_read(PagedCache(k=p["k"], v=p["v"], k_scale=p["ks"], v_scale=p["vs"], table=p["table"], pages=PAGES, **shape),
              PagedCache(k=p["k16"], v=p["v16"], table=p["table16"], pages=12, **shape), rows=1)


@pytest.mark.parametrize("kw", [
    dict(k=AT, k16=AT + 16), dict(k=AT, k16=AT + (POOL - 16)), dict(k16=AT, v=AT + (WIDE - 16)), dict(k16=AT, v16=AT + (WIDE - 16)), dict(v16=AT, k16=AT + (WIDE - 16)),
    dict(ks=AT, v16=AT + (SCALES - 16)), dict(vs=AT, k16=AT + 16), dict(table=AT, table16=AT + 4), dict(table16=AT, table=AT + (SEQUENCES * WIDTH * 4 - 4)),
    dict(k16=AT, table16=AT + (WIDE - 4)), dict(starts=AT, table16=AT + SEQUENCES * 4), dict(lengths=AT, v16=AT), dict(k16=Tensor("v16")),
], ids=str)
def test_what_meets_is_refused(kw):
    with pytest.raises(ValueError, match="tensors of their own"):
        read(**kw)


@pytest.mark.parametrize("kw", [
    {}, dict(k=AT, k16=AT + POOL), dict(k16=AT, v=AT + WIDE), dict(k16=AT, v16=AT + WIDE), dict(ks=AT, vs=AT + SCALES, table16=AT + 2 * SCALES),
    dict(table=AT, table16=AT + SEQUENCES * WIDTH * 4),
], ids=str)
def test_what_lies_side_by_side_is_taken(kw):
    read(**kw)
