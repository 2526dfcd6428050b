"""Attention of many rows over a cache in 8 bits whose table has far more places than its pool has pages: pages come back under their own numbers."""
from __future__ import annotations

import pytest
import torch

from tests.paged_e4m3_util import Batch8
from tests.paged_util import BOUND, check
from tests.test_gpu_paged_e4m3 import attend

pytestmark = pytest.mark.gpu

NEW, TOTAL = [70, 40, 1, 0, 3, 0, 0, 90], [700, 300, 290, 5, 100, 0, 1, 333]


def batch_of(page=16, heads=(4, 2, 64), shared=0, **kw) -> Batch8:
    """Sequences of unequal length; with ``shared`` those that are long enough begin with as many pages of the first one."""
    batch = Batch8(NEW, TOTAL, page, heads, seed=page + shared, **kw)
    for b, total in enumerate(TOTAL):
        if b and total > shared * page:
            batch.table[b, :shared] = batch.table[0, :shared]
            for lists in (batch.keys, batch.values):
                lists[b][:shared * page] = lists[0][:shared * page]
    assert len(NEW) * batch.width >= 2 * batch.pages
    return batch


@pytest.mark.parametrize("kw", [{}, dict(window=50), dict(window=100, sinks=20), dict(window=1000, sinks=3)], ids=str)
@pytest.mark.parametrize("page,heads,shared", [(16, (4, 2, 64), 0), (16, (4, 2, 64), 4), (32, (7, 1, 128), 2), (64, (8, 2, 64), 1)], ids=str)
def test_pages_of_the_pool(tmp_path, page, heads, shared, kw):
    batch = batch_of(page, heads, shared)
    got, status, mask = attend(tmp_path, batch, repeats=2, longest=90, **kw)
    assert status == 0
    check(batch, got, **mask)


@pytest.mark.parametrize("new,total", [([1, 1], [9, 80]), ([50, 1], [60, 30])], ids=["few", "chunk"])
def test_a_prefix_with_a_long_table(tmp_path, new, total):
    batch = Batch8(new, total, 16, (4, 2, 64), prefix=130, seed=4)
    wide = torch.full((2 * batch.pages + 5,), -9, dtype=torch.int32)
    wide[:batch.prefix_pages] = batch.prefix_table
    batch.prefix_table, batch.prefix_pages = wide, wide.numel()
    got, status, _ = attend(tmp_path, batch, repeats=2, longest=max(new))
    assert status == 0
    check(batch, got)


@pytest.mark.parametrize("page_id", [-1, None])
def test_a_page_outside_the_pool_is_reported_and_not_followed(tmp_path, page_id):
    batch = batch_of()
    got, status, _ = attend(tmp_path, batch, longest=90, change=lambda x: x["table"][1, 3].fill_(batch.pages if page_id is None else page_id))
    assert status == 0x400
    want, mass = batch.expected()
    rows = [*range(70), *range(110, batch.rows)]      # the other sequences are what they are
    assert bool(((got[rows].double() - want[rows]).abs() <= BOUND * mass[rows]).all())
