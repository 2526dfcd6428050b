"""A declared tensor whose rows are not the ones that a launch would read (a pitch left out or taken from another tensor) is refused; a
tensor that says the same memory in another shape is not."""
from __future__ import annotations

import pytest

from aginfer_b200.recipes import PagedCache, RecipeBuilder, Tensor, io

HEADS, KV, DIM, ROWS, SEQS = 8, 2, 128, 5, 3
QKV, Q = (HEADS + 2 * KV) * DIM, HEADS * DIM


def build(call, *, table=(SEQS, 4), x=(ROWS, QKV), o=(ROWS, Q), axes=None, rows=ROWS, sequences=SEQS, **kw):
    """``axes``: the shape of three-axis positions."""
    r = RecipeBuilder({"w": ("BF16", (8,))})
    pool = [9, KV, DIM // 64, 16, 64]
    r.begin_profile("default", [io("x", "BF16", list(x)), io("table", "I32", list(table)), io("lengths", "I32", [SEQS]), io("starts", "I32", [SEQS + 1]),
                                io("positions", "I32", list(axes or (3, rows)))],
                    [io("o", "BF16", list(o)), io("k", "BF16", pool), io("v", "BF16", pool)])
    cache = PagedCache(k=Tensor("k"), v=Tensor("v"), table=Tensor("table"), lengths=Tensor("lengths"), starts=Tensor("starts"), sequences=sequences,
                       pages=9, page=16, pages_per_sequence=4, kv_heads=KV, head_dim=DIM)
    if call == "append":
        if axes:
            kw |= dict(positions=Tensor("positions"), sections=(16, 24, 24))
        r.kv_append(Tensor("x"), Tensor("o"), cache, rows=rows, q_heads=HEADS, theta=1e6, **kw)
    else:
        r.paged_attention(Tensor("x"), Tensor("o"), cache, rows=rows, q_heads=HEADS, **{"q_stride": QKV} | kw)


@pytest.mark.parametrize("call,kw", [
    *[(call, kw) for call in ("append", "attend") for kw in (dict(table=(SEQS, 8)), dict(table=(SEQS, 5)), dict(o=(ROWS, Q + 8)), dict(o=(ROWS, 2 * Q)),
                                                            dict(x=(ROWS, QKV + 64)))],
    ("attend", dict(q_stride=None)), ("append", dict(axes=(3, ROWS + 1)))], ids=str)
def test_rows_of_another_width_are_refused(call, kw):
    with pytest.raises(ValueError, match="apart"):
        build(call, **kw)


@pytest.mark.parametrize("call,kw", [
    *[(call, kw) for call in ("append", "attend") for kw in (
        {}, dict(table=(SEQS * 4,)), dict(table=(SEQS + 2, 4)), dict(table=(2 * SEQS, 2)), dict(table=(1, 30), sequences=1), dict(o=(ROWS * HEADS, DIM)),
        dict(o=(ROWS, HEADS, DIM)), dict(o=(ROWS + 3, Q)), dict(x=(ROWS, HEADS + 2 * KV, DIM)), dict(o=(1, 5 * Q), rows=1), dict(o=(ROWS * 2 * Q,)))],
    ("attend", dict(x=(ROWS, Q), q_stride=None)), ("append", dict(axes=(3, ROWS))), ("append", dict(axes=(3 * ROWS,)))], ids=str)
def test_the_same_rows_in_another_shape_are_taken(call, kw):
    build(call, **kw)
