"""What the outputs of a product with 4-bit weights may share memory with: the residual, place for place, and nothing else that is read."""
from __future__ import annotations

import pytest

from aginfer_b200.recipes import Arena, RecipeBuilder, Tensor, io

N, K, G = 40, 128, 64
AT = Arena(1 << 20)
CODES, SCALES = 3 * K * 8, 3 * (K // G) * 32       # bytes


def product(m: int, **kw) -> None:
    r = RecipeBuilder({"w": ("BF16", (8,))})
    r.begin_profile("default", [io("x", "BF16", [m, K]), io("c", "I32", [3, 2, 32, 4]), io("s", "BF16", [3, 2, 8, 2]), io("residual", "BF16", [m, N])],
                    [io("y", "BF16", [m, N]), io("row", "BF16", [m, N]), io("units", "BF16", [3, 2, 8, 2])])
    p = dict(x=Tensor("x"), w=Tensor("c"), s=Tensor("s"), y=Tensor("y")) | {n: kw.pop(n) for n in ("x", "w", "s", "y") if n in kw}
    r.gemm_w4(p["x"], p["w"], p["s"], p["y"], m, N, K, group=G, **kw)


@pytest.mark.parametrize("m", [3, 40, 410])
@pytest.mark.parametrize("kw", [
    dict(w=AT, y=AT), dict(w=AT, y=AT + (CODES - 2)), dict(w=AT + 16, y=AT), dict(s=AT, y=AT + (SCALES - 2)), dict(s=AT + 64, y=AT),
    dict(bias=AT, y=AT), dict(bias=AT + 2 * N, y=AT), dict(bias=AT, y=AT + (2 * N - 2)),
    dict(residual=AT, y=AT + 2), dict(residual=AT + 2 * N, y=AT), dict(residual=AT, y=AT + 2 * N), dict(residual=AT, y=AT + 48, ldy=N + 24),
], ids=str)
def test_outputs_over_what_is_still_read_are_refused(m, kw):
    with pytest.raises(ValueError, match="still read"):
        product(m, **kw)


def test_tensors_over_what_is_still_read_are_refused():
    for kw in (dict(s=Tensor("units"), y=Tensor("units")), dict(bias=Tensor("y"))):
        with pytest.raises(ValueError, match="still read"):
            product(1, **kw)


@pytest.mark.parametrize("m", [3, 40, 410])
@pytest.mark.parametrize("kw", [
    dict(w=AT, s=AT + CODES, y=AT + CODES + SCALES), dict(w=AT + 2 * 410 * N, y=AT),
    dict(residual=AT, y=AT), dict(residual=AT, y=AT, ldy=N + 24), dict(residual=AT, y=AT + 2 * N, ldy=2 * N), dict(residual=Tensor("row"), y=Tensor("row")),
    dict(residual=AT + 2 * 410 * N, y=AT), dict(bias=AT + 2 * 410 * N, y=AT),
], ids=str)
def test_outputs_beside_what_is_read_are_taken(m, kw):
    product(m, **kw)
