"""Beside a page outside the pool, or a length beyond the table, every other page comes back as ever."""
from __future__ import annotations

import pytest
import torch

from aginfer_b200.recipes.layout import unpack_kv_pages
from tests.paged_e4m3_util import Batch8
from tests.test_gpu_paged_e4m3 import check_read, read

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page,heads", [(16, (2, 2, 64)), (32, (2, 1, 128))], ids=str)
@pytest.mark.parametrize("place", [(1, 0), (1, 2), (2, 1)], ids=str)
@pytest.mark.parametrize("outside", [True, False])
def test_a_page_outside_the_pool(tmp_path, page, heads, place, outside):
    batch = Batch8([1, 1, 1], [30, 100, 100], page, heads, seed=page)
    got = read(tmp_path, batch, change=lambda x: x["table"][place].fill_(batch.pages if outside else -1))
    at, tokens = place[0] * batch.width + place[1], slice(place[1] * page, (place[1] + 1) * page)
    assert int(got["status"]) == 0x400 and int(got["table16"][place]) == -1
    for name, lists in (("k16", batch.keys), ("v16", batch.values)):
        assert bool((got[name][at] == 77.0).all())
        lists[place[0]][tokens] = 77.0       # the page was left as it was; everything else is checked below
    got["table16"][place] = at
    got["status"].zero_()
    check_read(batch, got)


@pytest.mark.parametrize("length", [113, 2 ** 31 - 1])
def test_a_length_beyond_the_table(tmp_path, length):
    """It is cut to the table: the places that there are come back, and nothing behind them."""
    batch = Batch8([1, 1, 1], [30, 100, 100], 16, (2, 2, 64), seed=2)
    got = read(tmp_path, batch, change=lambda x: x["lengths"][1].fill_(length))
    assert int(got["status"]) == 0x500
    got["status"].zero_()
    last = batch.width + 6      # behind token 99 the pool holds any codes under scales of NaN
    for name in ("k16", "v16"):
        tokens = unpack_kv_pages(got[name][last:last + 1])[0]
        assert bool(tokens[4:].isnan().all())
        got[name][last][:, :, 4:] = 77.0
    check_read(batch, got)
