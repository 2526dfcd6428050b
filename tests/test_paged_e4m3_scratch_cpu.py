"""What attention of many rows over a cache in 8 bits takes of the arena: bf16 pages for its table's places or for the pool's pages, whichever are
fewer by half."""
from __future__ import annotations

import pytest

from aginfer_b200.recipes import PagedCache, RecipeBuilder, Tensor, io
from aginfer_b200.recipes import builder as B


def recipe(sequences: int, width: int, pages: int, prefix_pages: int = 0, page=64, heads=4, d=128) -> tuple[RecipeBuilder, list, int]:
    """The recipe, its launches of ``kv_read`` and the bytes that its arena grew by."""
    r = RecipeBuilder({"w": ("BF16", (8,))})
    codes, scales = [pages, heads, page, d], [pages, heads, page]
    r.begin_profile("default", [io("q", "BF16", [100, heads * d]), io("table", "I32", [sequences, width]), io("lengths", "I32", [sequences]),
                                io("starts", "I32", [sequences + 1]), io("k", "F8_E4M3", codes), io("v", "F8_E4M3", codes), io("ks", "BF16", scales),
                                io("vs", "BF16", scales), io("shared", "I32", [max(prefix_pages, 1)]), io("at", "I32", [1])], [io("o", "BF16", [100, heads * d])])
    cache = PagedCache(k=Tensor("k"), v=Tensor("v"), k_scale=Tensor("ks"), v_scale=Tensor("vs"), table=Tensor("table"), lengths=Tensor("lengths"),
                       starts=Tensor("starts"), sequences=sequences, pages=pages, page=page, pages_per_sequence=width, kv_heads=heads, head_dim=d)
    before = r.arena_bytes
    kw = dict(rows=100, q_heads=heads)
    if prefix_pages:
        r.prefix_attention(Tensor("q"), Tensor("o"), cache, Tensor("shared"), Tensor("at"), prefix_pages=prefix_pages, **kw)
    else:
        r.paged_attention(Tensor("q"), Tensor("o"), cache, **kw)
    return r, [l for l in r._profile.launches if l["kernel"] == "agi_kv_read_e4m3"], r.arena_bytes - before


def flags(launch) -> int:
    return launch["arguments"][-1]["scalar_u32"]


@pytest.mark.parametrize("sequences,width,pages", [(64, 512, 4096), (256, 512, 8192), (64, 512, 16384)], ids=str)
def test_scratch_is_not_the_rectangle_of_the_table(sequences, width, pages):
    r, (read,), grown = recipe(sequences, width, pages)
    pool = 2 * pages * 4 * 64 * 128 * 2
    assert pool <= grown <= pool + (256 << 20), "bf16 pages of the pool, and what the attention kernels join their parts in"
    assert flags(read) == B.KV_READ_FRESH_ONLY | B.KV_READ_BY_PAGE
    many = next(l for l in r._profile.launches if l["kernel"] == "agi_paged_many_bf16_d128")
    assert [many["arguments"][i] for i in (2, 3)] == [read["arguments"][i] for i in (7, 8)]
    assert many["arguments"][6] == {"tensor": "table"} and many["arguments"][16] == {"scalar_u32": pages}, "pages are where the batch's own table says"


def test_few_places_are_read_in_the_order_of_the_table():
    _, (read,), grown = recipe(2, 100, 4096)
    assert flags(read) == B.KV_READ_FRESH_ONLY and grown <= 2 * 200 * 4 * 64 * 128 * 2 + (256 << 20)


@pytest.mark.parametrize("prefix_pages,by_page", [(100, False), (127, False), (128, True), (1000, True)], ids=str)
def test_the_place_of_a_prefix(prefix_pages, by_page):
    r, reads, _ = recipe(1, 8, 64, prefix_pages)
    assert flags(reads[0]) == B.KV_READ_NO_STARTS | (B.KV_READ_BY_PAGE if by_page else 0)
    behind = next(l for l in r._profile.launches if l["kernel"] == "agi_paged_prefix_bf16_d128")
    assert (behind["arguments"][7] == {"tensor": "shared"}) == by_page
    assert behind["arguments"][16] == {"scalar_u32": 64 if by_page else prefix_pages}
