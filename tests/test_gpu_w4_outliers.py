"""Products with 4-bit weights of tokens that hold a few values thousands of times the others', as decoders' hidden states do.  Where the weights of
those columns are zero the outputs are the other columns' alone, and their digits have to be there: the bound is that of the tokens without
their outliers, half a unit of 2^-13 of the largest value left in 64 columns, and what bf16 outputs and sums in 32 bits are off by."""
from __future__ import annotations

import pytest
import torch

from tests.test_gpu_w4 import BF, Case, packaged

pytestmark = pytest.mark.gpu


def with_outliers(m: int, n: int, k: int, group: int, size: float, places, seed: int = 0, rest=None) -> tuple[Case, Case]:
    """The product to be run, of which every second row of weights is zero where the tokens are large, and that of the tokens without outliers."""
    clean = Case(m, n, k, group, seed=seed, x=rest)
    g = torch.Generator().manual_seed(seed + 17)
    columns = torch.tensor(sorted(places))
    clean.x = clean.x.clone()
    clean.x[:, columns] = 0
    clean.codes[::2, columns] = 8
    from aginfer_b200.recipes.layout import pack_w4
    clean.words, clean.units = pack_w4(clean.codes, clean.scales)
    full = Case(m, n, k, group, seed=seed, x=clean.x.clone())
    full.codes, full.scales, full.words, full.units = clean.codes, clean.scales, clean.words, clean.units
    sign = torch.randint(0, 2, (m, len(columns)), generator=g) * 2 - 1
    full.x[:, columns] = (sign * size * (1 + torch.rand(m, len(columns), generator=g))).to(BF)
    return full, clean


def run_and_check(tmp_path, full: Case, clean: Case) -> None:
    runner, x, out = packaged(tmp_path, full)
    got = []
    for _ in range(2):
        out["y"].fill_(77.0)
        runner.run(x, out)
        got.append(out["y"].cpu())
    assert int(out["status"].cpu()) == 0
    assert torch.equal(got[0].view(torch.int16), got[1].view(torch.int16)), "runs of one input differ"
    full.check(got[0])
    want, bound = clean.expected()
    error, bound = (got[0].double() - want).abs()[:, ::2], bound[:, ::2]
    assert bool((error <= bound).all()), f"{(error / bound).max():.3g} times the bound of the tokens without outliers"


@pytest.mark.parametrize("size", [30.0, 100.0, 1000.0, 10000.0, 1e6, 1e30])
@pytest.mark.parametrize("m", [1, 3, 8, 13, 17])
def test_one_column(tmp_path, m, size):
    run_and_check(tmp_path, *with_outliers(m, 130, 1024, 64, size, [333]))


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,n,k", [(1, 70, 1152), (4, 33, 2176), (9, 120, 1408), (12, 16400, 2048), (2, 640, 11008), (16, 48, 128)], ids=str)
def test_every_block(tmp_path, m, n, k, group):
    """One to five columns of each 64, in both halves."""
    g = torch.Generator().manual_seed(k + group)
    places = {block * 64 + int(torch.randint(0, 64, (), generator=g)) for block in range(k // 64) for _ in range(1 + block % 5)}
    run_and_check(tmp_path, *with_outliers(m, n, k, group, 3000.0, places, seed=group))


@pytest.mark.parametrize("m", [1, 6])
def test_of_unequal_size(tmp_path, m):
    """Among the rest, too, some are thousands of times the others: blocks of 2^-20 .. 2^20, and tokens that are zero but for three values."""
    g = torch.Generator().manual_seed(m)
    rest = torch.ldexp(torch.randn(m, 1024, generator=g), torch.randint(-20, 21, (1, 16), generator=g).repeat_interleave(64, 1))
    run_and_check(tmp_path, *with_outliers(m, 90, 1024, 64, 2.0 ** 40, range(7, 1024, 64), rest=rest.to(BF)))
    sparse = torch.zeros(m, 1024)
    sparse[:, [5, 40, 700]] = torch.randn(m, 3, generator=g)
    (tmp_path / "sparse").mkdir()
    run_and_check(tmp_path / "sparse", *with_outliers(m, 90, 1024, 64, 1000.0, [6, 701], rest=sparse.to(BF)))


@pytest.mark.parametrize("group", [32, 64, 128])
def test_every_geometry(tmp_path, monkeypatch, group):
    """Ways, parts, copies and depths of the ring over a product some of whose blocks are of integers and some are not."""
    from aginfer_b200.recipes import builder as B
    k, blocks = 2816, 44
    places = [block * 64 + (block * 37) % 64 for block in range(blocks) if block % 5 in (0, 1, 3)]
    full, clean = with_outliers(6, 1003, k, group, 2000.0, places, seed=group)
    for i, (eights, splits, ways, chunk, stages, ctas) in enumerate(((1, 1, 1, 4, 2, 3), (1, 1, 8, 8, 2, 1), (2, 1, 2, 4, 3, 5), (1, 5, 4, 4, 2, 7), (2, 3, 1, 8, 2, 2), (1, 44, 8, 4, 5, 3))):
        groups, per = -(-full.m // (4 * eights)), -(-blocks // splits)
        tiling = {"eights": eights, "splits": splits, "ways": ways, "chunk": chunk, "stages": stages, "grid": (ctas, groups, splits),
                  "shared_bytes": 16 * stages * chunk * 576 + per * eights * (672 if group == 32 else 608)}
        assert tiling["shared_bytes"] + B.W4_STATIC_BYTES <= B.MAX_DYNAMIC_SHARED
        monkeypatch.setattr(B, "w4_tiling", lambda *a, tiling=tiling: tiling)
        where = tmp_path / str(i)
        where.mkdir()
        run_and_check(where, full, clean)


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_beside_a_token_that_is_not_finite(tmp_path, value):
    full, clean = with_outliers(7, 90, 512, 64, 5000.0, [3, 77, 300])
    runner, x, out = packaged(tmp_path, full)
    x["x"][2, 70] = value
    x["x"][5, 400] = value
    runner.run(x, out)
    got = out["y"].cpu()
    assert int(out["status"].cpu()) == 0 and bool(got[[2, 5]].isnan().all())
    want, bound = clean.expected()
    kept = [0, 1, 3, 4, 6]
    assert bool(((got[kept].double() - want[kept]).abs()[:, ::2] <= bound[kept][:, ::2]).all())
