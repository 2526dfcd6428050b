"""Paged K/V cache where operands, orders and sizes meet the edges of what the entry points promise, against the definitions in 64 bits."""
from __future__ import annotations

import pytest
import torch

from aginfer_b200.recipes import PagedCache, Tensor
from oracle import paged
from tests.paged_util import BF, Batch, attention_outputs, check, packaged
from tests.test_gpu_paged import check_append, run_and_check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new,total,heads", [([700, 1, 300], [700, 40, 333], (8, 2, 128)), ([5], [5], (4, 2, 64))], ids=str)
def test_append_in_place_without_a_pitch(tmp_path, new, total, heads):
    """Queries | keys | values side by side, the queries turned where they stand."""
    batch = Batch(new, total, 16, heads, seed=31)
    hq, hk, d = heads
    x = torch.randn(batch.rows, (hq + 2 * hk) * d, generator=torch.Generator().manual_seed(1)).to(BF)
    inputs = {n: t for n, t in batch.inputs().items() if n in ("table", "lengths", "starts")}
    outputs = {"k": batch.k, "v": batch.v, "x": x, "status": torch.zeros(1, dtype=torch.int32)}

    def body(r):
        r.kv_append(Tensor("x"), Tensor("x"), batch.cache(), rows=batch.rows, q_heads=hq, theta=1e6)
        r.export_status(Tensor("status"))

    runner, dev, out = packaged(tmp_path, inputs, outputs, body)
    runner.run(dev, out)
    got = {n: t.cpu() for n, t in out.items()}
    assert torch.equal(got["x"][:, hq * d:], x[:, hq * d:])
    got["q_out"] = got["x"][:, :hq * d]
    q, k, v = (t.reshape(batch.rows, -1, d) for t in x.split([hq * d, hk * d, hk * d], dim=1))
    index = torch.tensor([batch.index(b, i) for b, n in enumerate(batch.new) for i in range(n)])
    angles = paged.rotary_angles(index, 1e6, d)
    turned = lambda t: (paged.turn(t, angles), t.double().abs())  # noqa: E731
    check_append(batch, got, turned(q), turned(k), v)


# rows of an item that end inside a warp, where that warp's lanes part: whole items, items that CTAs share, both streams on the same rows
@pytest.mark.parametrize("new,total,heads,prefix,spare", [
    ([45], [2000], (4, 2, 64), 0, 0), ([45, 300], [100, 1500], (3, 1, 128), 0, 5), ([141], [141], (1, 1, 128), 0, 0),
    ([5, 0, 8], [60, 2, 700], (5, 1, 64), 300, 3), ([1] * 37, list(range(1, 38)), (4, 1, 128), 2500, 4), ([70, 1], [70, 90], (3, 1, 128), 40, 7)], ids=str)
def test_rows_that_end_inside_a_warp(tmp_path, new, total, heads, prefix, spare):
    batch = Batch(new, total, 32, heads, prefix=prefix, spare_rows=spare, seed=41)
    run_and_check(tmp_path, batch, repeats=3, longest=max(new))


def test_more_sequences_than_the_queries_memory_holds(tmp_path):
    """The schedule of 2600 sequences lies in the ring of keys as well (64-wide heads)."""
    lengths = torch.randint(1, 40, (2600,), generator=torch.Generator().manual_seed(5)).tolist()
    new = [0 if i % 19 == 7 else 1 for i in range(2600)]
    new[2000], lengths[2000], new[0], lengths[0] = 150, 700, 60, 60
    run_and_check(tmp_path, Batch(new, lengths, 16, (2, 1, 64), seed=42), repeats=3, longest=150)


# rows of three sequences (or, below, of many) that are not in order: they end before they begin, lie outside the launch, leave a gap to fall into
DISORDER = ([5, 0, -3, 2], [0, 2 ** 31 - 1, -2 ** 31, 3], [-1, -1, -1, -1], [0, 2, 1, 3], [0, 1, 2, 90000], [-1, 1, 2, 3], [2, 1, 0, 0])


@pytest.mark.parametrize("sequences,at", [(3, 0), (40, 0), (40, 36), (400, 33), (400, 396)], ids=str)
def test_append_with_rows_out_of_order_does_nothing_and_says_so(tmp_path, sequences, at):
    batch = Batch([1] * sequences, [20 + i % 30 for i in range(sequences)], 16, (4, 2, 64), seed=43)
    hq, hk, d = batch.heads
    inputs = {n: t for n, t in batch.inputs().items() if n in ("table", "lengths", "starts")}
    inputs["x"] = torch.randn(batch.rows, (hq + 2 * hk) * d, generator=torch.Generator().manual_seed(2)).to(BF)
    outputs = {"k": batch.k, "v": batch.v, "q_out": torch.full((batch.rows, hq * d), 77.0).to(BF), "status": torch.zeros(1, dtype=torch.int32)}

    def body(r):
        r.kv_append(Tensor("x"), Tensor("q_out"), batch.cache(), rows=batch.rows, q_heads=hq, theta=1e6)
        r.export_status(Tensor("status"))

    runner, dev, out = packaged(tmp_path, inputs, outputs, body)
    good = dev["starts"].clone()
    for disorder in DISORDER:
        dev["starts"].copy_(good)
        shifted = [min(s + (at if disorder[0] >= 0 else 0), 2 ** 31 - 1) for s in disorder]
        dev["starts"][at:at + 4] = torch.tensor(shifted, dtype=torch.int32)
        runner.run(dev, out)
        assert int(out["status"].cpu()) == 0x500, disorder
        assert bool((out["q_out"] == 77.0).all()), disorder
        for name, before in (("k", batch.k), ("v", batch.v)):
            assert torch.equal(out[name].cpu().view(torch.int16), before.view(torch.int16)), disorder
    dev["starts"].copy_(good)
    runner.run(dev, out)
    assert int(out["status"].cpu()) == 0 and not bool((out["q_out"] == 77.0).any())


@pytest.mark.parametrize("prefix", [0, 90], ids=["", "prefix"])
@pytest.mark.parametrize("longest,sequences,at", [(1, 3, 0), (80, 3, 0), (1, 450, 440), (80, 450, 440)], ids=str)
def test_attention_with_rows_out_of_order_does_nothing_and_says_so(tmp_path, prefix, longest, sequences, at):
    new, total = [1] * sequences, [20 + i % 30 for i in range(sequences)]
    new[1], total[1] = longest, 100
    batch = Batch(new, total, 16, (4, 2, 64), prefix=prefix, seed=44)
    runner, x, out = packaged(tmp_path, batch.inputs(), attention_outputs(batch), lambda r: batch.attend(r, longest=longest))
    good = x["starts"].clone()
    runner.run(x, out)            # parts of an earlier pass lie in the workspace from here on
    assert int(out["status"].cpu()) == 0
    for disorder in DISORDER:
        x["starts"].copy_(good)
        shifted = [min(s + (at if disorder[0] >= 0 else 0), 2 ** 31 - 1) for s in disorder]
        x["starts"][at:at + 4] = torch.tensor(shifted, dtype=torch.int32)
        if bool((x["starts"] == good).all()):
            continue
        out["o"].fill_(77.0)
        runner.run(x, out)
        assert int(out["status"].cpu()) == 0x500, disorder
        assert bool((out["o"] == 77.0).all()), disorder
    x["starts"].copy_(good)
    runner.run(x, out)
    assert int(out["status"].cpu()) == 0
    check(batch, out["o"].cpu())


@pytest.mark.parametrize("new,total,heads,kw", [
    ([1], [9000], (4, 1, 64), {}), ([1], [20000], (2, 2, 128), {}), ([2, 1, 0], [30, 15000, 7], (4, 1, 128), {}), ([1, 4], [12000, 50], (16, 2, 64), {}),
    ([1], [17000], (2, 1, 64), dict(window=12000, sinks=70)), ([1, 1], [11, 40], (2, 1, 64), {})], ids=str)
def test_one_long_sequence(tmp_path, new, total, heads, kw):
    """An item in more parts than a short one is ever cut into."""
    run_and_check(tmp_path, Batch(new, total, 64, heads, seed=45), repeats=3, longest=max(new), **kw)


def test_one_long_sequence_has_the_whole_card(tmp_path):
    """As many keys in one sequence as in twelve: about the same time, since what CTAs share out are tiles of keys (with an item cut
    into at most twelve parts it took three times as long)."""
    def microseconds(sequences: int, keys: int) -> float:
        pages = sequences * keys // 64
        specs = {"q": torch.randn(sequences, 16 * 128).to(BF), "starts": torch.arange(sequences + 1, dtype=torch.int32),
                 "lengths": torch.full((sequences,), keys, dtype=torch.int32), "table": torch.randperm(pages).to(torch.int32).view(sequences, -1),
                 "k": torch.zeros(pages, 2, 2, 64, 64, dtype=BF), "v": torch.zeros(pages, 2, 2, 64, 64, dtype=BF)}
        names = {n: Tensor(n) for n in ("k", "v", "table", "lengths", "starts")}
        cache = PagedCache(**names, sequences=sequences, pages=pages, page=64, pages_per_sequence=keys // 64, kv_heads=2, head_dim=128)
        where = tmp_path / str(sequences)
        where.mkdir()
        runner, x, out = packaged(where, specs, {"o": torch.zeros(sequences, 16 * 128).to(BF)},
                                  lambda r: r.paged_attention(Tensor("q"), Tensor("o"), cache, rows=sequences, q_heads=16, longest=1))
        times = []
        for _ in range(6):
            begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            begin.record()
            for _ in range(20):
                runner.run(x, out)
            end.record()
            torch.cuda.synchronize()
            times.append(begin.elapsed_time(end) * 50)
        return min(times)

    many, one = microseconds(12, 64 * 170), microseconds(1, 64 * 170 * 12)
    assert one < 1.8 * many, (one, many)


# Enough key tiles a CTA that every slot of the rings is used again (five stages with 64-wide heads, two with 128), in long items and in
# many short ones whose last tile is zeroed behind the sequence's end
@pytest.mark.parametrize("new,total,page,heads,prefix,kw", [
    ([2000], [2000], 64, (16, 2, 64), 0, {}), ([300], [13000], 32, (8, 2, 64), 0, {}), ([300], [13000], 128, (4, 2, 128), 0, {}),
    ([33] * 300, [33 + 7 * i % 260 for i in range(300)], 16, (4, 2, 64), 0, {}), ([33] * 150, [33 + 7 * i % 260 for i in range(150)], 16, (4, 2, 128), 0, {}),
    ([600], [9000], 64, (12, 2, 64), 0, dict(window=3000, sinks=130)), ([4] * 64, [4 + i for i in range(64)], 64, (32, 4, 64), 4100, {}),
    ([2] * 64, [2 + i for i in range(64)], 32, (28, 4, 128), 3001, {})], ids=lambda v: str(v)[:24])
def test_rings_that_go_round(tmp_path, new, total, page, heads, prefix, kw):
    run_and_check(tmp_path, Batch(new, total, page, heads, prefix=prefix, seed=46), repeats=3, longest=max(new), **kw)
