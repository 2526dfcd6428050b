"""How the many-row kernel's CTAs share out key tiles, restated: every tile of every item is taken once, parts of an item lie in neighbouring
CTAs, and a small launch has as many CTAs as it has tiles."""
from __future__ import annotations

import random

import pytest

from aginfer_b200.recipes import Arena, PagedCache
from aginfer_b200.recipes.builder import SM_COUNT, paged_many_tiling

ITEM_COST = 3


def runs(items: list[int], grid: int, least: int, snap: int):
    """(per, [(first tile, last + 1, CTA) of every item]), as the kernel walks them."""
    total = sum(items) + ITEM_COST * len(items)
    per, parts = max(-(-total // grid), least), [[] for _ in items]
    for cta in range(grid):
        begin, end, first = min(per * cta, total), min(per * cta + per, total), 0
        for which, count in enumerate(items):
            tiles_at, after = first + ITEM_COST, first + ITEM_COST + count

            def cut(at):
                if at >= after:
                    return after
                return tiles_at if at <= tiles_at + snap else after if at + snap >= after else at

            if begin < end and first < end and after > begin and cut(begin) < cut(end):
                parts[which].append((cut(begin) - tiles_at, cut(end) - tiles_at, cta))
            first = after
    return per, parts


@pytest.mark.parametrize("snap", [0, 1])
def test_every_tile_is_taken_once_and_parts_are_neighbours(snap):
    rng = random.Random(snap)
    for _ in range(3000):
        longest = rng.choice([1, 2, 3, 6, 20, 200])
        items = [rng.randint(1, longest) for _ in range(rng.choice([1, 1, 2, 3, 5, 20, 150]))]
        least = rng.choice([1, 2, 3])
        grid = rng.choice([SM_COUNT, min(SM_COUNT, -(-sum(items) // least)), rng.randint(1, SM_COUNT)])
        per, parts = runs(items, grid, least, snap)
        slots, first = set(), 0
        for count, mine in zip(items, parts):
            assert mine[0][0] == 0 and mine[-1][1] == count
            assert all(a[1] == b[0] and a[2] + 1 == b[2] for a, b in zip(mine, mine[1:]))
            if len(mine) > 1:
                tiles_at = first + ITEM_COST
                assert (tiles_at + count - snap - 1) // per - (tiles_at + snap) // per + 1 == len(mine)       # what the note for the join says
                for begin, _, cta in mine:       # a slot for the item that a CTA goes on with, one for the item that it leaves open
                    assert (cta, begin > 0) not in slots
                    slots.add((cta, begin > 0))
            first += ITEM_COST + count


@pytest.mark.parametrize("tokens,blocks,kv_heads", [(64, 2, 4), (150, 2, 2), (288, 5, 4), (1500, 3, 2)])
def test_a_small_launch_has_a_cta_for_every_tile(tokens, blocks, kv_heads):
    at = Arena(0)
    cache = PagedCache(k=at, v=at, table=at, lengths=at, starts=at, sequences=1, pages=100, page=16, pages_per_sequence=-(-tokens // 16),
                       kv_heads=kv_heads, head_dim=128)
    t = paged_many_tiling(cache, blocks, tokens)
    assert t["grid"] == min(SM_COUNT, blocks * kv_heads * -(-tokens // 128)) and t["least"] == 1
