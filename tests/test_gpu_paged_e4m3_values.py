"""Values of any size in a paged cache in 8 bits: scales that lie hundreds of binades apart beside each other, few and many rows."""
from __future__ import annotations

import pytest
import torch

from tests.paged_e4m3_util import Batch8
from tests.paged_util import BOUND, check
from tests.test_gpu_paged_e4m3 import attend

pytestmark = pytest.mark.gpu

LONGEST = pytest.mark.parametrize("longest", [1, 4, 70])      # a row, drafts, and more rows than the kernel of few takes
HEADS = pytest.mark.parametrize("heads", [(4, 2, 64), (8, 1, 128)], ids=str)


def of_one_size(longest: int, heads: tuple, spread: int = 0) -> Batch8:
    """Keys of one size, or one key would take everything; values that differ by 2^-spread .. 2^spread."""
    batch = Batch8([longest, 1], [150, 90], 16, heads, seed=longest, spread=spread)
    keys = Batch8([longest, 1], [150, 90], 16, heads, seed=longest)
    batch.keys, batch.pools = keys.keys, batch.pools | {n: keys.pools[n] for n in ("k", "k_scale")}
    return batch


def times(batch: Batch8, factor: float, b: int, tokens) -> None:
    for j in tokens:
        batch.pools["v_scale"][batch.table[b, j // 16], :, j % 16] *= factor
        batch.values[b][j] *= factor


def attend_and_check(tmp_path, batch: Batch8, longest: int) -> None:
    got, status, _ = attend(tmp_path, batch, longest=longest)
    assert status == 0
    check(batch, got)


@LONGEST
@HEADS
def test_sizes_side_by_side(tmp_path, longest, heads):
    attend_and_check(tmp_path, of_one_size(longest, heads, spread=100), longest)


@LONGEST
@HEADS
@pytest.mark.parametrize("exponent", [-100, -75, 64, 75, 100])
def test_all_of_one_far_size(tmp_path, longest, heads, exponent):
    batch = of_one_size(longest, heads)
    for b, total in enumerate(batch.total):
        times(batch, 2.0 ** exponent, b, range(total))
    attend_and_check(tmp_path, batch, longest)


@LONGEST
@pytest.mark.parametrize("place", [3, 149])
def test_one_huge_value(tmp_path, longest, place):
    """A single token of up to 2^118 among ordinary ones: behind it, in front of rows that do not see it yet."""
    batch = of_one_size(longest, (4, 2, 64))
    times(batch, 2.0 ** 116, 0, [place])
    attend_and_check(tmp_path, batch, longest)


@LONGEST
def test_a_huge_value_whose_weight_vanishes(tmp_path, longest):
    """Scores some hundreds below the others': in 32 bits their weights are zero, in 64 too little to be seen beside the rest."""
    batch = of_one_size(longest, (4, 2, 64))
    for b, total in enumerate(batch.total):
        for head in range(2):
            # of the token's key only its first column is left, against queries that are positive there
            for j in (5, 40):
                batch.pools["k"][batch.table[b, j // 16], head, j % 16] = 0
                chunk = j >> 1 & 3      # where the first 16 columns of the token lie
                batch.pools["k"][batch.table[b, j // 16], head, j % 16, chunk * 16] = 0xfe      # -448
                batch.pools["k_scale"][batch.table[b, j // 16], head, j % 16] = 16.0
                batch.keys[b][j, head] = 0.0
                batch.keys[b][j, head, 0] = -448.0 * 16.0
        times(batch, 2.0 ** 80, b, [5, 40])
    q = batch.q.view(batch.rows, 4, 64)
    q[..., 0] = q[..., 0].abs() + 1.0
    attend_and_check(tmp_path, batch, longest)


@pytest.mark.parametrize("heads", [(4, 2, 64), (8, 1, 128)], ids=str)
@pytest.mark.parametrize("new,total,unseen", [([4, 1], [100, 90], [(0, 99)]), ([3, 2], [66, 18], [(0, 65), (0, 64), (1, 17)])], ids=str)
def test_rows_that_do_not_see_a_draft_are_not_touched_by_it(tmp_path, new, total, unseen, heads):
    """Later drafts whose keys and values are not finite: earlier rows are what they are without them, the others NaN."""
    batch = Batch8(new, total, 16, heads, seed=5)
    for b, j in unseen:
        for name in ("k_scale", "v_scale"):
            batch.pools[name][batch.table[b, j // 16], :, j % 16] = float("nan")
    got, status, _ = attend(tmp_path, batch, longest=max(new))
    assert status == 0
    want, mass = batch.expected()
    row = 0
    for b, n in enumerate(new):
        first = min((j for c, j in unseen if c == b), default=total[b])
        for i in range(n):
            if batch.index(b, i) < first:
                assert bool(((got[row].double() - want[row]).abs() <= BOUND * mass[row]).all()), (b, i)
            else:
                assert bool(got[row].isnan().all()), (b, i)
            row += 1
