"""Paged K/V cache: appending with rotation, and attention over the pages, against the definitions in 64 bits."""
from __future__ import annotations

import pytest
import torch

from aginfer_b200.recipes import Tensor
from aginfer_b200.recipes.layout import unpack_kv_pages
from oracle import paged
from tests.paged_util import BF, BOUND, Batch, attention_outputs, check, packaged

pytestmark = pytest.mark.gpu


def attend(tmp_path, batch: Batch, repeats: int = 1, change=None, **kw):
    mask = {n: kw[n] for n in ("window", "sinks", "scale") if n in kw}
    runner, x, out = packaged(tmp_path, batch.inputs(), attention_outputs(batch), lambda r: batch.attend(r, **kw))
    if change is not None:
        change(x)
    first = None
    for _ in range(repeats):
        out["o"].fill_(77.0)
        runner.run(x, out)
        if first is not None:
            assert torch.equal(first.view(torch.int16), out["o"].view(torch.int16)), "runs of one input differ"
        first = out["o"].clone()
    return out["o"].cpu(), int(out["status"].cpu()), mask


def run_and_check(tmp_path, batch: Batch, **kw):
    got, status, mask = attend(tmp_path, batch, **kw)
    assert status == 0
    check(batch, got, **mask)


# new tokens and lengths of the sequences: one token, page ends on, before and behind a tile's, sequences without new tokens,
# without any, and rows in front of their sequence's beginning (they see nothing)
SINGLE = ([1, 1, 1, 1, 1, 1], [1, 16, 17, 63, 64, 65])
RAGGED = ([3, 0, 1, 2, 0, 5], [3, 40, 129, 66, 0, 300])
BEFORE = ([4, 1, 2], [2, 0, 1])


@pytest.mark.parametrize("new,total", [SINGLE, RAGGED, BEFORE, ([1], [1]), ([1], [1000]), ([0, 1], [0, 7])], ids=lambda v: str(len(v)))
@pytest.mark.parametrize("page,heads", [(16, (4, 2, 64)), (32, (7, 1, 128)), (64, (16, 2, 128)), (128, (3, 3, 64))], ids=str)
def test_few_tokens(tmp_path, new, total, page, heads):
    batch = Batch(new, total, page, heads, seed=page + len(new))
    run_and_check(tmp_path, batch, longest=max(1, *new))


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 3), (16, 16), (64, 0), (64, 70), (100, 4), (1000, 10), (130, 129)])
@pytest.mark.parametrize("new,total,page,heads", [([1, 2, 1], [200, 70, 333], 16, (6, 2, 64)), ([1, 1, 40], [1, 129, 190], 64, (4, 1, 128))],
                         ids=["few", "chunk"])
def test_windows(tmp_path, window, sinks, new, total, page, heads):
    batch = Batch(new, total, page, heads, seed=window)
    run_and_check(tmp_path, batch, longest=max(new), window=window, sinks=sinks)


@pytest.mark.parametrize("new,total,page,heads", [
    ([37], [37], 16, (2, 1, 64)), ([128], [128], 128, (2, 2, 128)), ([129, 1, 200], [129, 300, 513], 64, (4, 2, 128)),
    ([65, 0, 3, 64], [65, 9, 500, 64], 32, (8, 2, 64)), ([300], [301], 16, (7, 1, 128)), ([40, 30], [20, 30], 16, (5, 1, 128)),
    ([70], [777], 128, (16, 2, 128))], ids=str)
def test_chunks(tmp_path, new, total, page, heads):
    batch = Batch(new, total, page, heads, seed=sum(new))
    run_and_check(tmp_path, batch, longest=max(new))


@pytest.mark.parametrize("new,total", [([1, 1, 1], [5, 70, 1]), ([6, 50, 1], [300, 60, 20])], ids=["few", "chunk"])
@pytest.mark.parametrize("heads", [(32, 1, 64), (40, 2, 128)], ids=str)
def test_many_queries_share_a_key_head(tmp_path, new, total, heads):
    batch = Batch(new, total, 32, heads, seed=9)
    run_and_check(tmp_path, batch, longest=max(new))


@pytest.mark.parametrize("new,total,longest", [([1, 3, 2], [50, 200, 7], None), ([40, 3, 2], [50, 200, 7], 1), ([1, 1], [400, 30], 2)], ids=str)
def test_the_longest_sequence_is_a_hint(tmp_path, new, total, longest):
    batch = Batch(new, total, 16, (4, 2, 128), seed=4)
    run_and_check(tmp_path, batch, longest=longest)


@pytest.mark.parametrize("new,total,page,heads,prefix", [
    ([1, 1, 1], [1, 17, 64], 16, (4, 2, 64), 100), ([1] * 8, [3, 1, 64, 65, 2, 9, 30, 130], 64, (16, 2, 128), 288),
    ([2, 0, 3, 1], [2, 0, 90, 33], 32, (7, 1, 128), 129), ([1] * 20, list(range(1, 21)), 16, (14, 2, 128), 1000),
    ([1], [1], 128, (4, 4, 128), 1), ([50, 1, 20], [60, 1, 20], 64, (6, 3, 64), 200), ([3, 1], [1, 0], 16, (4, 2, 64), 30)], ids=str)
def test_a_shared_prefix(tmp_path, new, total, page, heads, prefix):
    batch = Batch(new, total, page, heads, prefix=prefix, seed=prefix)
    run_and_check(tmp_path, batch, longest=max(new))


@pytest.mark.parametrize("prefix", [0, 90], ids=str)
@pytest.mark.parametrize("sequences,long", [(33, 1), (70, 1), (130, 3), (450, 40), (450, 1)], ids=str)
def test_more_sequences_than_a_warp_or_a_block_looks_at(tmp_path, sequences, long, prefix):
    lengths = torch.randint(1, 50, (sequences,), generator=torch.Generator().manual_seed(sequences)).tolist()
    new = [0 if i % 17 == 3 else 1 for i in range(sequences)]
    new[sequences - 2], lengths[sequences - 2] = long, 150
    batch = Batch(new, lengths, 16, (2, 1, 64), prefix=prefix, seed=long)
    run_and_check(tmp_path, batch, longest=long)


@pytest.mark.parametrize("new,total", [([1, 1], [9, 80]), ([50, 1], [60, 30])], ids=["few", "chunk"])
def test_prefixes_that_are_empty_too_long_or_not_in_the_pool(tmp_path, new, total):
    batch = Batch(new, total, 16, (4, 2, 128), prefix=40, seed=21)
    got, status, _ = attend(tmp_path, batch, change=lambda x: x["prefix_length"].zero_(), longest=max(new))
    batch.prefix_kv = None
    assert status == 0
    check(batch, got)
    for code, change in ((0x500, lambda x: x["prefix_length"].fill_(49)), (0x400, lambda x: x["prefix_table"].fill_(batch.pages))):
        assert attend(tmp_path, batch, change=change, longest=max(new))[1] == code


def test_a_prefix_without_programmatic_launch(tmp_path):
    batch = Batch([1, 2, 1], [30, 70, 1], 32, (8, 2, 128), prefix=300, seed=22)
    runner, x, out = packaged(tmp_path, batch.inputs(), attention_outputs(batch), lambda r: batch.attend(r, longest=2), flags=0)
    for _ in range(2):
        runner.run(x, out)
    assert int(out["status"].cpu()) == 0
    check(batch, out["o"].cpu())


@pytest.mark.parametrize("new,total,prefix", [([1, 2], [90, 300], 0), ([70], [300], 0), ([1, 1], [9, 80], 70)], ids=str)
def test_sharp_scores(tmp_path, new, total, prefix):
    """Scores up to a few hundred: one key takes (almost) all, the rest underflows."""
    batch = Batch(new, total, 32, (4, 2, 128), prefix=prefix, sharp=60.0, seed=5)
    # a score of 300 in 32 bits is off by up to 128 * 2^-24 * 300 < 2^-8, as much again as the other roundings
    got, status, _ = attend(tmp_path, batch, longest=max(new))
    want, mass = batch.expected()
    assert status == 0 and bool(((got.double() - want).abs() <= 2.0 ** -6 * mass + 2.0 ** -9).all())


@pytest.mark.parametrize("new,total,prefix", [([1, 1], [200, 40], 0), ([80, 4], [200, 40], 0), ([1, 2], [20, 40], 90)], ids=str)
def test_infinite_scores_and_rows_without_weight(tmp_path, new, total, prefix):
    """A key of minus infinity in the direction of every query takes no weight; a row that sees only such keys is zero."""
    batch = Batch(new, total, 16, (2, 1, 64), prefix=prefix, seed=6)
    batch.q = batch.q.abs() + 0.01
    dead = [range(0, total[0], 3), range(total[1])] if not prefix else [range(0, total[0], 3), []]
    pool = unpack_kv_pages(batch.k)
    for b, which in enumerate(dead):
        for j in which:
            batch.keys[b][j] = float("-inf")
            pool[batch.table[b, j // 16], j % 16] = float("-inf")
    from aginfer_b200.recipes.layout import pack_kv_pages
    batch.k = pack_kv_pages(pool)
    got, status, _ = attend(tmp_path, batch, longest=max(new))
    for b in range(2):       # the oracle without the dead keys
        for i in range(new[b]):
            index = batch.index(b, i)
            live = [j for j in range(index + 1) if j not in dead[b]]
            row = int(batch.starts[b]) + i
            want, mass = paged.attention(batch.q[row].view(2, 64), batch.keys[b][live], batch.values[b][live], len(live) - 1, prefix=batch.prefix_kv)
            assert bool(((got[row].double() - want.reshape(-1)).abs() <= BOUND * mass.reshape(-1)).all())
    assert status == 0


@pytest.mark.parametrize("longest", [1, 70])
def test_strides_scale_and_rows_of_no_sequence(tmp_path, longest):
    batch = Batch([1, 0, 1] if longest == 1 else [70, 0, 1], [30, 4, 100] if longest == 1 else [75, 4, 100], 16, (4, 2, 64), spare_rows=3, seed=7)
    wide = torch.full((batch.rows, 4 * 64 + 24), float("nan")).to(BF)
    wide[:, :256] = batch.q
    batch.extra = {"q": wide}
    out = {"o": torch.full((batch.rows, 256 + 8), 77.0).to(BF), "status": torch.zeros(1, dtype=torch.int32)}
    runner, x, out = packaged(tmp_path, batch.inputs(), out, lambda r: batch.attend(r, longest=longest, q_stride=280, o_stride=264, scale=0.3))
    runner.run(x, out)
    got = out["o"].cpu()
    assert int(out["status"].cpu()) == 0 and bool((got[:, 256:] == 77.0).all())
    check(batch, got[:, :256], scale=0.3)


@pytest.mark.parametrize("new,total,prefix", [([1, 1, 1], [700, 30, 90], 0), ([90, 2], [700, 30], 0), ([1, 1, 2], [40, 1, 90], 500)], ids=str)
def test_runs_repeat_bit_for_bit_and_follow_lengths_changed_in_place(tmp_path, new, total, prefix):
    batch = Batch(new, total, 32, (8, 2, 128), prefix=prefix, seed=8)
    runner, x, out = packaged(tmp_path, batch.inputs(), attention_outputs(batch), lambda r: batch.attend(r, longest=max(new)))
    side, results = torch.cuda.Stream(), []
    for _ in range(4):
        out["o"].fill_(77.0)
        side.wait_stream(torch.cuda.current_stream())
        runner.run(x, out, stream=side)
        torch.cuda.current_stream().wait_stream(side)
        results.append(out["o"].cpu())
    assert all(torch.equal(results[0].view(torch.int16), r.view(torch.int16)) for r in results)
    check(batch, results[0])
    shorter = [max(n, t - 11) for n, t in zip(new, total)]       # the same graph, other lengths
    x["lengths"].copy_(torch.tensor(shorter, dtype=torch.int32))
    out["o"].fill_(77.0)
    runner.run(x, out)
    batch.total = shorter
    check(batch, out["o"].cpu())
    assert int(out["status"].cpu()) == 0


@pytest.mark.parametrize("longest", [1, 80])
def test_what_a_table_must_not_say_is_reported_and_not_followed(tmp_path, longest):
    new, total = ([1, 1, 1], [50, 60, 200]) if longest == 1 else ([1, 80, 1], [50, 90, 200])
    batch = Batch(new, total, 16, (4, 2, 64), seed=3)
    for code, change in ((0x400, lambda x: x["table"][1].fill_(batch.pages)), (0x400, lambda x: x["table"][1].fill_(-1)),
                         (0x500, lambda x: x["lengths"][1].fill_(batch.width * 16 + 1)), (0x500, lambda x: x["lengths"][1].fill_(2 ** 31 - 1))):
        got, status, _ = attend(tmp_path, batch, change=change, longest=longest)
        assert status & ~0xff == code
        want, mass = batch.expected()
        for row in (0, batch.rows - 1):      # the other sequences are what they are
            assert bool(((got[row].double() - want[row]).abs() <= BOUND * mass[row]).all())


@pytest.mark.parametrize("longest", [1, 80])
def test_starts_in_disorder_stay_inside(tmp_path, longest):
    batch = Batch([1, 1, 1] if longest == 1 else [1, 80, 1], [50, 100, 200], 16, (4, 2, 64), seed=3)
    for starts in ([5, 0, -3, 2], [0, 2 ** 31 - 1, -2 ** 31, 3], [-1, -1, -1, -1]):
        attend(tmp_path, batch, change=lambda x: x["starts"].copy_(torch.tensor(starts, dtype=torch.int32)), longest=longest)


@pytest.mark.parametrize("name", ["q", "k", "v"])
@pytest.mark.parametrize("longest", [1, 80])
def test_a_tensor_off_its_boundary_is_reported(tmp_path, name, longest):
    batch = Batch([longest], [100], 16, (4, 2, 64), seed=3)

    def shift(x):
        flat = torch.zeros(x[name].numel() + 1, dtype=BF, device="cuda")
        x[name] = flat[1:].view(x[name].shape)

    _, status, _ = attend(tmp_path, batch, change=shift, longest=longest)
    assert status & ~0xff == 0x600


@pytest.mark.parametrize("longest", [1, 40])
def test_offsets_beyond_32_bits(tmp_path, longest):
    """A pool of 9 GB: pages behind the first 2^32 elements."""
    batch = Batch([longest], [150], 64, (4, 2, 128), seed=2)
    pages = 2 ** 32 // (64 * 2 * 128) + 64
    small_k, small_v, table = batch.k, batch.v, batch.table
    batch.pages = pages
    inputs = batch.inputs() | {"k": torch.empty(0), "v": torch.empty(0)}
    from aginfer_b200.recipes import RecipeBuilder, io
    from aginfer_b200.recipes.package import build_aim, describe
    from aginfer_b200.runner import Runner
    weights = {"unused.pad": torch.zeros(8, dtype=BF)}
    r = RecipeBuilder(describe(weights))
    specs = [io(n, "I32" if t.dtype == torch.int32 else "BF16", [pages, *small_k.shape[1:]] if n in "kv" else t.shape) for n, t in inputs.items()]
    r.begin_profile("default", specs, [io("o", "BF16", [longest, 512]), io("status", "I32", [1])])
    batch.attend(r, longest=longest)
    runner = Runner(build_aim(tmp_path, weights, r))
    x = {n: t.cuda() for n, t in inputs.items()}
    for n, small in (("k", small_k), ("v", small_v)):
        x[n] = torch.empty(pages, *small_k.shape[1:], dtype=BF, device="cuda")
        x[n][-small.shape[0]:] = small.cuda()
    x["table"] = (table + (pages - small_k.shape[0])).cuda()
    out = {"o": torch.full((longest, 512), 77.0, dtype=BF, device="cuda"), "status": torch.zeros(1, dtype=torch.int32, device="cuda")}
    runner.run(x, out)
    assert int(out["status"].cpu()) == 0
    check(batch, out["o"].cpu())


# ---- appending ------------------------------------------------------------------------------------------

def append(tmp_path, batch: Batch, *, axes=0, sections=None, theta=1e6, ladder=None, offset=None, apart=False, in_place=False, at=None, seed=1):
    """The outputs of kv_append over ``batch`` and what they have to be: (got, want q, turned keys, values)."""
    hq, hk, d = batch.heads
    g = torch.Generator().manual_seed(seed)
    rows = batch.rows
    x = torch.randn(rows, (hq + 2 * hk) * d, generator=g).to(BF)
    q, k, v = x.split([hq * d, hk * d, hk * d], dim=1)
    index = torch.tensor([batch.index(b, i) for b, n in enumerate(batch.new) for i in range(n)] + [0] * batch.spare_rows)
    positions = index + (offset or 0)
    inputs = {n: t for n, t in batch.inputs().items() if n in ("table", "lengths", "starts")}
    if axes:
        shape = (rows,) if axes == 1 else (3, rows)
        positions = torch.randint(0, at or 5000, shape, generator=g, dtype=torch.int32)
        inputs["positions"] = positions
    if offset is not None:
        inputs["offset"] = torch.tensor([offset], dtype=torch.int32)
    pools = {"k": batch.k, "v": batch.v, "status": torch.zeros(1, dtype=torch.int32)}
    kw = dict(rows=rows, q_heads=hq, theta=theta, sections=sections, ladder=ladder, positions=Tensor("positions") if axes else None,
              offset=Tensor("offset") if offset is not None else None)
    outputs = pools | {"q_out": torch.full((rows, hq * d), 77.0).to(BF)}
    if in_place:
        outputs = pools | {"x": x}
        call = lambda r: r.kv_append(Tensor("x"), Tensor("x"), batch.cache(), out_stride=x.shape[1], **kw)  # noqa: E731
    elif apart:
        inputs |= {"q": q.contiguous(), "key": torch.nn.functional.pad(k, (0, 16)), "value": torch.nn.functional.pad(v, (0, 16))}
        call = lambda r: r.kv_append(Tensor("q"), Tensor("q_out"), batch.cache(), k=Tensor("key"), v=Tensor("value"),  # noqa: E731
                                     kv_stride=hk * d + 16, **kw)
    else:
        inputs["x"] = x
        call = lambda r: r.kv_append(Tensor("x"), Tensor("q_out"), batch.cache(), **kw)  # noqa: E731

    def body(r):
        call(r)
        r.export_status(Tensor("status"))

    runner, dev, out = packaged(tmp_path, inputs, outputs, body)
    runner.run(dev, out)
    got = {n: t.cpu() for n, t in out.items()}
    if in_place:
        assert torch.equal(got["x"][:, hq * d:], x[:, hq * d:])
        got["q_out"] = got["x"][:, :hq * d]
    angles = paged.rotary_angles(positions, theta, d, sections, ladder)
    turn = lambda t, h: (paged.turn(t.reshape(rows, h, d), angles), t.reshape(rows, h, d).double().abs())  # noqa: E731
    return got, turn(q, hq), turn(k, hk), v.reshape(rows, hk, d)


def near(got, want, size):
    """A rounding to bf16 (half a step: at most 2^-8) and, in 32 bits, two products and their sum of values up to |a| + |b| with
    sine and cosine."""
    half = size.shape[-1] // 2
    both = size[..., :half] + size[..., half:]
    slack = torch.cat([both, both], dim=-1) * 2.0 ** -20
    assert bool(((got.double() - want).abs() <= want.abs() * 2.0 ** -8 + slack).all())


def check_append(batch: Batch, got, q, keys, values):
    hq, hk, d = batch.heads
    live = sum(batch.new)
    assert int(got["status"]) == 0
    near(got["q_out"][:live].reshape(live, hq, d), q[0][:live], q[1][:live])
    k, v = unpack_kv_pages(got["k"]), unpack_kv_pages(got["v"])
    k0, v0 = unpack_kv_pages(batch.k), unpack_kv_pages(batch.v)
    row = 0
    for b, n in enumerate(batch.new):
        for i in range(n):
            j = batch.index(b, i)
            if j >= 0:
                page, token = int(batch.table[b, j // batch.page]), j % batch.page
                near(k[page, token], keys[0][row], keys[1][row])
                assert torch.equal(v[page, token], values[row])
                k[page, token], v[page, token] = k0[page, token], v0[page, token]
            row += 1
    for pool, before in ((k, k0), (v, v0)):      # nothing else was touched, bit for bit
        assert torch.equal(pool.view(torch.int16), before.view(torch.int16))


@pytest.mark.parametrize("new,total", [SINGLE, RAGGED, BEFORE, ([300], [300]), ([1], [1])], ids=lambda v: str(len(v)))
@pytest.mark.parametrize("page,heads", [(16, (4, 2, 64)), (32, (7, 1, 128)), (64, (16, 2, 128)), (128, (3, 3, 64))], ids=str)
def test_append(tmp_path, new, total, page, heads):
    batch = Batch(new, total, page, heads, seed=page)
    check_append(batch, *append(tmp_path, batch))


@pytest.mark.parametrize("kw", [dict(axes=1), dict(axes=3, sections=(16, 24, 24)), dict(axes=3, sections=(0, 0, 64), theta=1e4), dict(offset=1234),
                                dict(axes=3, sections=(20, 22, 22), ladder=32), dict(apart=True), dict(in_place=True), dict(axes=1, at=2 ** 30),
                                dict(offset=10 ** 6, theta=5e5)], ids=str)
def test_append_forms(tmp_path, kw):
    batch = Batch([5, 1, 33], [20, 300, 33], 16, (6, 2, 128), spare_rows=0 if kw.get("in_place") else 2, seed=11)
    got, *want = append(tmp_path, batch, **kw)
    if batch.spare_rows:
        assert bool((got["q_out"][-2:] == 77.0).all())
    check_append(batch, got, *want)


def test_append_more_rows_than_blocks(tmp_path):
    batch = Batch([1500, 1, 700], [1500, 40, 900], 64, (2, 1, 64), seed=12)
    check_append(batch, *append(tmp_path, batch, axes=3, sections=(8, 12, 12)))


@pytest.mark.parametrize("code,change", [(0x400, lambda x, b: x["table"][1].fill_(b.pages)), (0x400, lambda x, b: x["table"][1].fill_(-2)),
                                         (0x500, lambda x, b: x["lengths"][1].fill_(b.width * 16 + 2)),
                                         (0x500, lambda x, b: x["lengths"][1].fill_(2 ** 31 - 1))])
def test_append_does_not_follow_what_a_table_must_not_say(tmp_path, code, change):
    batch = Batch([1, 2, 1], [30, 40, 200], 16, (2, 1, 64), seed=13)
    hq, hk, d = batch.heads
    x = torch.randn(batch.rows, (hq + 2 * hk) * d).to(BF)
    inputs = {"x": x, "table": batch.table, "lengths": batch.lengths, "starts": batch.starts}
    outputs = {"q_out": torch.zeros(batch.rows, hq * d).to(BF), "k": batch.k, "v": batch.v, "status": torch.zeros(1, dtype=torch.int32)}

    def body(r):
        r.kv_append(Tensor("x"), Tensor("q_out"), batch.cache(), rows=batch.rows, q_heads=hq, theta=1e4)
        r.export_status(Tensor("status"))

    runner, dev, out = packaged(tmp_path, inputs, outputs, body)
    change(dev, batch)
    runner.run(dev, out)
    assert int(out["status"].cpu()) == code
    before, after = unpack_kv_pages(batch.k), unpack_kv_pages(out["k"].cpu())
    changed = (before.view(torch.int16) != after.view(torch.int16)).flatten(1).any(1).nonzero().flatten().tolist()
    assert sorted(changed) == sorted({int(batch.table[0, 29 // 16]), int(batch.table[2, 199 // 16])})


def test_append_then_attend(tmp_path):
    """A step as it is served: the launches of one recipe, the second reading what the first one has just written."""
    batch = Batch([1, 4, 1], [60, 64, 1], 16, (4, 2, 64), seed=14)
    hq, hk, d = batch.heads
    x = torch.randn(batch.rows, (hq + 2 * hk) * d, generator=torch.Generator().manual_seed(3)).to(BF)
    inputs = {"x": x, "table": batch.table, "lengths": batch.lengths, "starts": batch.starts}
    outputs = {**attention_outputs(batch), "k": batch.k, "v": batch.v}

    def body(r):
        turned = r.alloc(batch.rows * hq * d * 2)
        r.kv_append(Tensor("x"), turned, batch.cache(), rows=batch.rows, q_heads=hq, theta=1e4)
        r.paged_attention(turned, Tensor("o"), batch.cache(), rows=batch.rows, q_heads=hq, longest=4)
        r.export_status(Tensor("status"))

    runner, dev, out = packaged(tmp_path, inputs, outputs, body)
    for _ in range(3):
        runner.run(dev, out)
    k = unpack_kv_pages(out["k"].cpu())
    row = 0
    for b, n in enumerate(batch.new):
        for i in range(n):
            j = batch.index(b, i)
            batch.keys[b][j] = k[int(batch.table[b, j // 16]), j % 16]
            batch.values[b][j] = x[row, (hq + hk) * d:].view(hk, d)
            angles = paged.rotary_angles(torch.tensor([j]), 1e4, d)
            turned = paged.turn(x[row, :hq * d].view(1, hq, d), angles)
            batch.q[row] = turned.reshape(-1).to(BF)
            near(batch.keys[b][j], paged.turn(x[row, hq * d:(hq + hk) * d].view(1, hk, d), angles)[0],
                 x[row, hq * d:(hq + hk) * d].view(hk, d).double().abs())
            row += 1
    # the queries here are rounded from 64 bits: one of them may round the other way, 2^-8 of a score of less than 4
    want, mass = batch.expected()
    assert bool(((out["o"].cpu().double() - want).abs() <= 2.0 ** -6 * mass).all()) and int(out["status"].cpu()) == 0
