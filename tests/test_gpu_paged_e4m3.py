"""Paged caches in 8 bits: appending, bringing pages back, attention over the codes, against the definitions in 64 bits."""
from __future__ import annotations

import pytest
import torch

from aginfer_b200.recipes import PagedCache, Tensor
from aginfer_b200.recipes.layout import quantize_kv_pages, read_kv_pages, unpack_kv_pages
from oracle import paged
from tests.paged_e4m3_util import POOLS, Batch8, rounded
from tests.paged_util import BF, BOUND, attention_outputs, check, packaged
from tests.test_gpu_paged import near

pytestmark = pytest.mark.gpu

SINGLE = ([1, 1, 1, 1, 1, 1], [1, 16, 17, 63, 64, 65])
RAGGED = ([3, 0, 1, 2, 0, 5], [3, 40, 129, 66, 0, 300])
BEFORE = ([4, 1, 2], [2, 0, 1])
SHAPES = [(16, (4, 2, 64)), (32, (7, 1, 128)), (64, (16, 2, 128)), (128, (3, 3, 64))]


def attend(tmp_path, batch: Batch8, repeats: int = 1, change=None, **kw):
    mask = {n: kw[n] for n in ("window", "sinks", "scale") if n in kw}
    runner, x, out = packaged(tmp_path, batch.inputs(), attention_outputs(batch), lambda r: batch.attend(r, **kw))
    if change is not None:
        change(x)
    first = None
    for _ in range(repeats):
        out["o"].fill_(77.0)
        runner.run(x, out)
        assert first is None or torch.equal(first.view(torch.int16), out["o"].view(torch.int16)), "runs of one input differ"
        first = out["o"].clone()
    return out["o"].cpu(), int(out["status"].cpu()), mask


def run_and_check(tmp_path, batch: Batch8, **kw):
    got, status, mask = attend(tmp_path, batch, **kw)
    assert status == 0
    check(batch, got, **mask)


# ---- bringing pages back ----------------------------------------------------------------------------------

def read(tmp_path, batch: Batch8, change=None, **kw):
    hk, d, slots = batch.heads[1], batch.heads[2], len(batch.new) * batch.width
    inputs = {n: t for n, t in batch.inputs().items() if n in (*POOLS, "table", "lengths", "starts")}
    outputs = {"k16": torch.full((slots, hk, d // 64, batch.page, 64), 77.0).to(BF), "v16": torch.full((slots, hk, d // 64, batch.page, 64), 77.0).to(BF),
               "table16": torch.full((len(batch.new), batch.width), -9, dtype=torch.int32), "status": torch.zeros(1, dtype=torch.int32)}
    to = PagedCache(k=Tensor("k16"), v=Tensor("v16"), table=Tensor("table16"), lengths=Tensor("lengths"), starts=Tensor("starts"), sequences=len(batch.new),
                    pages=slots, page=batch.page, pages_per_sequence=batch.width, kv_heads=hk, head_dim=d)

    def body(r):
        r.kv_read(batch.cache(), to, rows=batch.rows, **kw)
        r.export_status(Tensor("status"))

    runner, x, out = packaged(tmp_path, inputs, outputs, body)
    if change is not None:
        change(x)
    for _ in range(2):
        runner.run(x, out)
    return {n: t.cpu() for n, t in out.items()}


def check_read(batch: Batch8, got, window=0, sinks=0):
    assert int(got["status"]) == 0
    for b, total in enumerate(batch.total):
        start = max(0, total - batch.new[b] - window + 1) if window else 0
        for slot in range(batch.width):
            at, tokens = b * batch.width + slot, range(slot * batch.page, min((slot + 1) * batch.page, total))
            seen = any(j >= start or j < sinks for j in tokens)
            assert int(got["table16"][b, slot]) == (at if seen else -9), (b, slot)
            for name, lists in (("k16", batch.keys), ("v16", batch.values)):
                page = unpack_kv_pages(got[name][at:at + 1])[0]
                count = len(tokens) if seen else 0
                if count:
                    assert torch.equal(page[:count].view(torch.int16), lists[b][tokens.start:tokens.stop].view(torch.int16)), (b, slot, name)
                assert bool((page[count:] == 77.0).all()), (b, slot, name)


@pytest.mark.parametrize("new,total", [SINGLE, RAGGED, ([1], [1]), ([1], [1000]), ([0, 1], [0, 7]), ([0], [0])], ids=lambda v: str(len(v)))
@pytest.mark.parametrize("page,heads", SHAPES, ids=str)
def test_read(tmp_path, new, total, page, heads):
    batch = Batch8(new, total, page, heads, spare_rows=1, seed=page, spread=3)
    check_read(batch, read(tmp_path, batch))


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (20, 3), (64, 70), (100, 4), (1000, 10), (130, 129)])
def test_read_what_a_window_leaves(tmp_path, window, sinks):
    batch = Batch8([1, 0, 40, 1], [200, 333, 190, 64], 16, (2, 2, 64), seed=window)
    check_read(batch, read(tmp_path, batch, window=window, sinks=sinks), window, sinks)


@pytest.mark.parametrize("sequences", [40, 300, 4096])
def test_read_many_sequences(tmp_path, sequences):
    lengths = torch.randint(0, 40, (sequences,), generator=torch.Generator().manual_seed(sequences)).tolist()
    batch = Batch8([1 if t else 0 for t in lengths], lengths, 16, (1, 1, 64), seed=1)
    got = read(tmp_path, batch)
    assert int(got["status"]) == 0
    for b in (0, 31, 32, sequences // 2, sequences - 1):
        tokens = unpack_kv_pages(got["k16"][b * batch.width:(b + 1) * batch.width]).flatten(0, 1)[:lengths[b]]
        assert torch.equal(tokens, batch.keys[b])
    want = torch.tensor([[b * batch.width + i if i * 16 < lengths[b] else -9 for i in range(batch.width)] for b in range(sequences)], dtype=torch.int32)
    assert torch.equal(got["table16"], want)


def test_read_does_not_follow_what_a_table_must_not_say(tmp_path):
    for n, (code, change) in enumerate(((0x400, lambda x, b: x["table"][1, 2].fill_(b.pages)), (0x400, lambda x, b: x["table"][1, 2].fill_(-1)),
                                        (0x500, lambda x, b: x["lengths"][1].fill_(b.width * 16 + 1)), (0x500, lambda x, b: x["starts"][1].fill_(9)))):
        where = tmp_path / str(n)
        where.mkdir()
        batch = Batch8([1, 1, 1], [30, 100, 100], 16, (2, 2, 64), seed=n)
        got = read(where, batch, change=lambda x: change(x, batch))
        assert int(got["status"]) == code
        if code == 0x400:
            assert int(got["table16"][1, 2]) == -1 and bool((got["k16"][batch.width + 2] == 77.0).all())
            got["status"].zero_()
            got["table16"][1, 2] = batch.width + 2
            got["k16"][batch.width + 2], got["v16"][batch.width + 2] = (
                torch.cat([t[1][32:48] for _ in (0,)]).view(1, 16, 2, 64).permute(0, 2, 1, 3).unsqueeze(2)[0] for t in (batch.keys, batch.values))
        if n == 3:
            assert bool((got["k16"] == 77.0).all()) and bool((got["table16"] == -9).all())


@pytest.mark.parametrize("name", POOLS)
def test_read_reports_a_pool_off_its_boundary(tmp_path, name):
    def shift(x):
        flat = torch.zeros(x[name].numel() + 8, dtype=x[name].dtype, device="cuda")
        x[name] = flat[1:1 + x[name].numel()].view(x[name].shape)

    got = read(tmp_path, Batch8([1], [30], 16, (2, 2, 64)), change=shift)
    assert int(got["status"]) == 0x600 and bool((got["k16"] == 77.0).all())


# ---- appending ----------------------------------------------------------------------------------------------

def append(tmp_path, batch: Batch8, *, axes=0, sections=None, theta=1e6, offset=None, apart=False, in_place=False, size=None, seed=1):
    hq, hk, d = batch.heads
    g = torch.Generator().manual_seed(seed)
    rows = batch.rows
    x = torch.randn(rows, (hq + 2 * hk) * d, generator=g)
    x = (x if size is None else torch.ldexp(x.view(rows, -1, d), torch.randint(-size, size, (rows, hq + 2 * hk, 1), generator=g)).view(rows, -1)).to(BF)
    q, k, v = x.split([hq * d, hk * d, hk * d], dim=1)
    index = torch.tensor([batch.index(b, i) for b, n in enumerate(batch.new) for i in range(n)] + [0] * batch.spare_rows)
    positions = index + (offset or 0)
    inputs = {n: t for n, t in batch.inputs().items() if n in ("table", "lengths", "starts")}
    if axes:
        positions = torch.randint(0, 5000, (rows,) if axes == 1 else (3, rows), generator=g, dtype=torch.int32)
        inputs["positions"] = positions
    if offset is not None:
        inputs["offset"] = torch.tensor([offset], dtype=torch.int32)
    outputs = batch.pools | {"status": torch.zeros(1, dtype=torch.int32)}
    kw = dict(rows=rows, q_heads=hq, theta=theta, sections=sections, positions=Tensor("positions") if axes else None,
              offset=Tensor("offset") if offset is not None else None)
    if in_place:
        outputs |= {"x": x}
        call = lambda r: r.kv_append(Tensor("x"), Tensor("x"), batch.cache(), **kw)  # noqa: E731
    elif apart:
        outputs |= {"q_out": torch.full((rows, hq * d), 77.0).to(BF)}
        inputs |= {"q": q.contiguous(), "key": torch.nn.functional.pad(k, (0, 16)), "value": torch.nn.functional.pad(v, (0, 16))}
        call = lambda r: r.kv_append(Tensor("q"), Tensor("q_out"), batch.cache(), k=Tensor("key"), v=Tensor("value"), kv_stride=hk * d + 16, **kw)  # noqa: E731
    else:
        outputs |= {"q_out": torch.full((rows, hq * d), 77.0).to(BF)}
        inputs["x"] = x
        call = lambda r: r.kv_append(Tensor("x"), Tensor("q_out"), batch.cache(), **kw)  # noqa: E731

    def body(r):
        call(r)
        r.export_status(Tensor("status"))

    runner, dev, out = packaged(tmp_path, inputs, outputs, body)
    runner.run(dev, out)
    got = {n: t.cpu() for n, t in out.items()}
    if in_place:
        assert torch.equal(got["x"][:, hq * d:].view(torch.int16), x[:, hq * d:].view(torch.int16))
        got["q_out"] = got["x"][:, :hq * d]
    angles = paged.rotary_angles(positions, theta, d, sections)
    turn = lambda t, h: (paged.turn(t.reshape(rows, h, d), angles), t.reshape(rows, h, d).double().abs())  # noqa: E731
    return got, turn(q, hq), turn(k, hk), v.reshape(rows, hk, d)


def check_append(batch: Batch8, got, q, keys, values):
    hq, hk, d = batch.heads
    live = sum(batch.new)
    assert int(got["status"]) == 0
    near(got["q_out"][:live].reshape(live, hq, d), q[0][:live], q[1][:live])
    after = {n: got[n].clone() for n in POOLS}
    tokens = {n: read_kv_pages(got[n], got[n + "_scale"]).double() for n in "kv"}
    codes, scales = quantize_kv_pages(values[None])          # one long page of every row's values
    value = read_kv_pages(codes, scales)[0].double()
    row = 0
    for b, n in enumerate(batch.new):
        for i in range(n):
            j = batch.index(b, i)
            if j >= 0:
                page, token = int(batch.table[b, j // batch.page]), j % batch.page
                assert torch.equal(tokens["v"][page, token], value[row]) and torch.equal(got["v_scale"][page, :, token], scales[0, :, row])
                want, half = keys[0][row], d // 2
                size = keys[1][row][:, :half] + keys[1][row][:, half:]
                slack = torch.cat([size, size], dim=-1) * 2.0 ** -20          # rotation in 32 bits, as in `near`
                scale = got["k_scale"][page, :, token].double()[:, None]
                # a code is off by half a step, 2^-4 of the value, or 2^-10 of the scale where codes are subnormal
                assert bool(((tokens["k"][page, token] - want).abs() <= (want.abs() * 2.0 ** -4).clamp_min(scale * 2.0 ** -10) + 1.0625 * slack).all())
                peak = want.abs().amax(dim=-1)
                assert bool((torch.frexp(scale)[0] == 0.5).all())
                reach = slack.amax(dim=-1)
                assert bool((peak - reach <= 448 * scale[:, 0]).all()) and bool((peak + reach > 224 * scale[:, 0]).logical_or(peak == 0).all())
                for name in "kv":
                    after[name][page, :, token] = batch.pools[name][page, :, token]
                    after[name + "_scale"][page, :, token] = batch.pools[name + "_scale"][page, :, token]
            row += 1
    for name in POOLS:      # nothing else was touched, bit for bit
        assert torch.equal(after[name].view(torch.uint8), batch.pools[name].view(torch.uint8)), name


@pytest.mark.parametrize("new,total", [SINGLE, RAGGED, BEFORE, ([300], [300]), ([1], [1])], ids=lambda v: str(len(v)))
@pytest.mark.parametrize("page,heads", SHAPES, ids=str)
def test_append(tmp_path, new, total, page, heads):
    batch = Batch8(new, total, page, heads, seed=page)
    check_append(batch, *append(tmp_path, batch))


@pytest.mark.parametrize("kw", [dict(axes=1), dict(axes=3, sections=(16, 24, 24)), dict(offset=1234), dict(apart=True), dict(in_place=True), dict(size=30),
                                dict(offset=10 ** 6, theta=5e5)], ids=str)
@pytest.mark.parametrize("heads", [(6, 2, 128), (20, 20, 128)], ids=str)
def test_append_forms(tmp_path, kw, heads):
    batch = Batch8([5, 1, 33], [20, 300, 33], 16, heads, spare_rows=0 if kw.get("in_place") else 2, seed=11)
    got, *want = append(tmp_path, batch, **kw)
    if batch.spare_rows:
        assert bool((got["q_out"][-2:] == 77.0).all())
    check_append(batch, got, *want)


def test_append_tokens_of_zeros_infinities_and_nan(tmp_path):
    batch = Batch8([6], [6], 16, (2, 2, 64), seed=3)
    x = torch.ones(6, 6 * 64).to(BF)
    x[0] = 0.0
    x[1, 130], x[2, 260], x[3, 195], x[4, 383] = float("nan"), float("inf"), float("-inf"), float("nan")
    x[5] *= 2.0 ** -130
    inputs = {"x": x, "table": batch.table, "lengths": batch.lengths, "starts": batch.starts}
    outputs = {"q_out": torch.zeros(6, 128).to(BF), "status": torch.zeros(1, dtype=torch.int32)} | batch.pools

    def body(r):
        r.kv_append(Tensor("x"), Tensor("q_out"), batch.cache(), rows=6, q_heads=2, theta=1e4)
        r.export_status(Tensor("status"))

    runner, dev, out = packaged(tmp_path, inputs, outputs, body)
    runner.run(dev, out)
    page = int(batch.table[0, 0])
    tokens = {n: read_kv_pages(out[n].cpu(), out[n + "_scale"].cpu())[page, :6] for n in "kv"}
    assert bool((tokens["k"][0] == 0).all()) and bool((tokens["v"][0] == 0).all()) and bool((out["k_scale"][page, :, 0] == 1).all())
    gone = {"k": [(1, 0), (3, 1)], "v": [(2, 0), (4, 1)]}
    for name, places in gone.items():
        for token in range(1, 5):
            for head in range(2):
                assert bool(tokens[name][token, head].isnan().all()) == ((token, head) in places), (name, token, head)
    # 2^-130 is 2^-4 of the least scale, a code as it is; turned keys lie below
    assert bool((out["v_scale"][page, :, 5].float() == 2.0 ** -126).all()) and bool((tokens["v"][5] == 2.0 ** -130).all())


@pytest.mark.parametrize("code,change", [(0x400, lambda x, b: x["table"][1].fill_(b.pages)), (0x500, lambda x, b: x["lengths"][1].fill_(2 ** 31 - 1)),
                                         (0x500, lambda x, b: x["starts"][2].fill_(0))])
def test_append_does_not_follow_what_a_table_must_not_say(tmp_path, code, change):
    batch = Batch8([1, 2, 1], [30, 40, 200], 16, (2, 1, 64), seed=13)
    x = torch.randn(batch.rows, 4 * 64).to(BF)
    inputs = {"x": x, "table": batch.table, "lengths": batch.lengths, "starts": batch.starts}
    outputs = {"q_out": torch.full((batch.rows, 128), 77.0).to(BF), "status": torch.zeros(1, dtype=torch.int32)} | batch.pools

    def body(r):
        r.kv_append(Tensor("x"), Tensor("q_out"), batch.cache(), rows=batch.rows, q_heads=2, theta=1e4)
        r.export_status(Tensor("status"))

    runner, dev, out = packaged(tmp_path, inputs, outputs, body)
    change(dev, batch)
    runner.run(dev, out)
    assert int(out["status"].cpu()) == code
    ordered = bool((dev["starts"].diff() >= 0).all())
    for name in POOLS:
        changed = (batch.pools[name].view(torch.uint8) != out[name].cpu().view(torch.uint8)).flatten(1).any(1).nonzero().flatten().tolist()
        pages = {int(batch.table[0, 29 // 16]), int(batch.table[2, 199 // 16])}
        assert (pages >= set(changed) if "scale" in name else sorted(changed) == sorted(pages)) if ordered else not changed


# ---- attention ----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("new,total", [SINGLE, RAGGED, BEFORE, ([1], [1]), ([1], [1000]), ([0, 1], [0, 7])], ids=lambda v: str(len(v)))
@pytest.mark.parametrize("page,heads", SHAPES, ids=str)
def test_few_tokens(tmp_path, new, total, page, heads):
    run_and_check(tmp_path, Batch8(new, total, page, heads, seed=page + len(new)), longest=max(1, *new), repeats=2)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 3), (16, 16), (64, 0), (64, 70), (100, 4), (1000, 10), (130, 129)])
@pytest.mark.parametrize("new,total,page,heads", [([1, 2, 1], [200, 70, 333], 16, (6, 2, 64)), ([1, 1, 40], [1, 129, 190], 64, (4, 1, 128)),
                                                  ([8, 1, 4], [300, 129, 190], 32, (8, 2, 128))], ids=["few", "chunk", "drafts"])
def test_windows(tmp_path, window, sinks, new, total, page, heads):
    run_and_check(tmp_path, Batch8(new, total, page, heads, seed=window), longest=max(new), window=window, sinks=sinks)


@pytest.mark.parametrize("new,total,page,heads", [
    ([37], [37], 16, (2, 1, 64)), ([129, 1, 200], [129, 300, 513], 64, (4, 2, 128)), ([65, 0, 3, 64], [65, 9, 500, 64], 32, (8, 2, 64)),
    ([300], [301], 16, (7, 1, 128)), ([40, 30], [20, 30], 16, (5, 1, 128)), ([70], [777], 128, (16, 2, 128))], ids=str)
def test_chunks(tmp_path, new, total, page, heads):
    run_and_check(tmp_path, Batch8(new, total, page, heads, seed=sum(new)), longest=max(new), repeats=2)


@pytest.mark.parametrize("new,total,page,heads,prefix", [
    ([1, 1, 1], [1, 17, 64], 16, (4, 2, 64), 100), ([1] * 8, [3, 1, 64, 65, 2, 9, 30, 130], 64, (16, 2, 128), 288),
    ([2, 0, 3, 1], [2, 0, 90, 33], 32, (7, 1, 128), 129), ([1], [1], 128, (4, 4, 128), 1), ([50, 1, 20], [60, 1, 20], 64, (6, 3, 64), 200),
    ([3, 1], [1, 0], 16, (4, 2, 64), 30)], ids=str)
def test_a_shared_prefix(tmp_path, new, total, page, heads, prefix):
    run_and_check(tmp_path, Batch8(new, total, page, heads, prefix=prefix, seed=prefix), longest=max(new), repeats=3)


@pytest.mark.parametrize("new,total", [([1, 1], [9, 80]), ([50, 1], [60, 30])], ids=["few", "chunk"])
def test_prefixes_that_are_empty_too_long_or_not_in_the_pool(tmp_path, new, total):
    batch = Batch8(new, total, 16, (4, 2, 128), prefix=40, seed=21)
    got, status, _ = attend(tmp_path, batch, change=lambda x: x["prefix_length"].zero_(), longest=max(new))
    kept, batch.prefix_kv = batch.prefix_kv, None
    assert status == 0
    check(batch, got)
    batch.prefix_kv = kept
    for code, change in ((0x500, lambda x: x["prefix_length"].fill_(49)), (0x400, lambda x: x["prefix_table"].fill_(batch.pages))):
        assert attend(tmp_path, batch, change=change, longest=max(new))[1] == code


@pytest.mark.parametrize("prefix", [0, 90], ids=str)
@pytest.mark.parametrize("sequences,long", [(33, 1), (130, 3), (450, 40)], ids=str)
def test_more_sequences_than_a_warp_or_a_block_looks_at(tmp_path, sequences, long, prefix):
    lengths = torch.randint(1, 50, (sequences,), generator=torch.Generator().manual_seed(sequences)).tolist()
    new = [0 if i % 17 == 3 else 1 for i in range(sequences)]
    new[sequences - 2], lengths[sequences - 2] = long, 150
    run_and_check(tmp_path, Batch8(new, lengths, 16, (2, 1, 64), prefix=prefix, seed=long), longest=long)


@pytest.mark.parametrize("new,total,heads,kw", [([1], [9000], (4, 1, 64), {}), ([2, 1, 0], [30, 15000, 7], (4, 1, 128), {}), ([1, 4], [12000, 50], (16, 2, 64), {}),
                                                ([1], [17000], (2, 1, 64), dict(window=12000, sinks=70))], ids=str)
def test_one_long_sequence(tmp_path, new, total, heads, kw):
    run_and_check(tmp_path, Batch8(new, total, 64, heads, seed=45), repeats=3, longest=max(new), **kw)


@pytest.mark.parametrize("new,total,heads", [([1, 1, 1], [5, 70, 1], (32, 1, 64)), ([6, 50, 1], [300, 60, 20], (40, 2, 128))], ids=str)
def test_many_queries_share_a_key_head(tmp_path, new, total, heads):
    run_and_check(tmp_path, Batch8(new, total, 32, heads, seed=9), longest=max(new))


@pytest.mark.parametrize("longest", [1, 70])
def test_tokens_and_rows_of_unequal_size(tmp_path, longest):
    """Values, and below them queries, that differ by powers of two up to 2^40: scales meet weights of any size.  Keys of one size, or one key would
    take everything."""
    batch = Batch8([longest, 1], [120, 90], 16, (4, 2, 64), seed=31, spread=20)
    keys = Batch8([longest, 1], [120, 90], 16, (4, 2, 64), seed=31)
    batch.keys, batch.pools = keys.keys, batch.pools | {n: keys.pools[n] for n in ("k", "k_scale")}
    factor = torch.tensor([2.0 ** -20, 1.0, 2.0 ** -60, 2.0 ** 3]).repeat_interleave(64)
    batch.q = (batch.q.float() * factor).to(BF)
    got, status, _ = attend(tmp_path, batch, longest=longest)
    assert status == 0
    check(batch, got)


@pytest.mark.parametrize("new,total,prefix", [([1, 2], [90, 300], 0), ([70], [300], 0), ([1, 1], [9, 80], 70)], ids=str)
def test_sharp_scores(tmp_path, new, total, prefix):
    """Scores up to a few hundred: one key takes (almost) all, the rest underflows."""
    batch = Batch8(new, total, 32, (4, 2, 128), prefix=prefix, sharp=60.0, seed=5)
    got, status, _ = attend(tmp_path, batch, longest=max(new))
    want, mass = batch.expected()
    # a score of 300 in 32 bits is off by up to 128 * 2^-24 * 300 < 2^-8, as much again as the other roundings
    assert status == 0 and bool(((got.double() - want).abs() <= 2.0 ** -6 * mass + 2.0 ** -9).all())


def test_hidden_tokens_that_are_not_finite(tmp_path):
    """Tokens behind a window, which no row sees, may be anything, in a tile with tokens that are seen as well."""
    batch = Batch8([1, 1], [100, 64], 16, (4, 2, 64), seed=8)
    for b, hidden in ((0, range(4, 90)), (1, range(4, 54))):
        for j in hidden:
            batch.pools["k_scale"][batch.table[b, j // 16], :, j % 16] = float("nan")
            batch.pools["v_scale"][batch.table[b, j // 16], :, j % 16] = float("nan")
            batch.pools["v"][batch.table[b, j // 16], :, j % 16] = 0x7f
    run_and_check(tmp_path, batch, longest=1, window=10, sinks=4)


@pytest.mark.parametrize("longest", [1, 70])
def test_strides_scale_and_rows_of_no_sequence(tmp_path, longest):
    batch = Batch8([1, 0, 1] if longest == 1 else [70, 0, 1], [30, 4, 100] if longest == 1 else [75, 4, 100], 16, (4, 2, 64), spare_rows=3, seed=7)
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
    batch = Batch8(new, total, 32, (8, 2, 128), prefix=prefix, seed=8)
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
    batch = Batch8(new, total, 16, (4, 2, 64), seed=3)
    for code, change in ((0x400, lambda x: x["table"][1].fill_(batch.pages)), (0x400, lambda x: x["table"][1].fill_(-1)),
                         (0x500, lambda x: x["lengths"][1].fill_(batch.width * 16 + 1)), (0x500, lambda x: x["lengths"][1].fill_(2 ** 31 - 1))):
        got, status, _ = attend(tmp_path, batch, change=change, longest=longest)
        assert status & ~0xff == code
        want, mass = batch.expected()
        for row in (0, batch.rows - 1):      # the other sequences are what they are
            assert bool(((got[row].double() - want[row]).abs() <= BOUND * mass[row]).all())


@pytest.mark.parametrize("prefix", [0, 90], ids=["", "prefix"])
@pytest.mark.parametrize("longest", [1, 80])
def test_rows_out_of_order_leave_no_work(tmp_path, prefix, longest):
    batch = Batch8([1, longest, 1], [20, 100, 30], 16, (4, 2, 64), prefix=prefix, seed=44)
    runner, x, out = packaged(tmp_path, batch.inputs(), attention_outputs(batch), lambda r: batch.attend(r, longest=longest))
    good = x["starts"].clone()
    for disorder in ([5, 0, -3, 2], [0, 2 ** 31 - 1, -2 ** 31, 3], [0, 2, 1, 3], [-1, 1, 2, 3]):
        x["starts"].copy_(torch.tensor(disorder, dtype=torch.int32))
        out["o"].fill_(77.0)
        runner.run(x, out)
        assert int(out["status"].cpu()) == 0x500 and bool((out["o"] == 77.0).all()), disorder
    x["starts"].copy_(good)
    runner.run(x, out)
    assert int(out["status"].cpu()) == 0
    check(batch, out["o"].cpu())


@pytest.mark.parametrize("name", ["q", *POOLS])
@pytest.mark.parametrize("longest", [1, 80])
def test_a_tensor_off_its_boundary_is_reported(tmp_path, name, longest):
    batch = Batch8([longest], [100], 16, (4, 2, 64), seed=3)

    def shift(x):
        flat = torch.zeros(x[name].numel() + 8, dtype=x[name].dtype, device="cuda")
        x[name] = flat[1:1 + x[name].numel()].view(x[name].shape)

    assert attend(tmp_path, batch, change=shift, longest=longest)[1] & ~0xff == 0x600


@pytest.mark.parametrize("longest", [1, 40])
def test_offsets_beyond_32_bits(tmp_path, longest):
    """Pools of 4.5 GB: pages behind the first 2^32 bytes."""
    batch = Batch8([longest], [150], 64, (4, 2, 128), seed=2)
    pages = 2 ** 32 // (64 * 2 * 128) + 64
    small, table = dict(batch.pools), batch.table
    batch.pages = pages
    from aginfer_b200.recipes import RecipeBuilder, io
    from aginfer_b200.recipes.package import build_aim, describe
    from aginfer_b200.runner import Runner
    weights = {"unused.pad": torch.zeros(8, dtype=BF)}
    r = RecipeBuilder(describe(weights))
    kinds = {torch.int32: "I32", torch.uint8: "F8_E4M3", BF: "BF16"}
    inputs = {n: t for n, t in batch.inputs().items() if n in ("q", "table", "lengths", "starts", *POOLS)}
    r.begin_profile("default", [io(n, kinds[t.dtype], [pages, *t.shape[1:]] if n in POOLS else t.shape) for n, t in inputs.items()],
                    [io("o", "BF16", [longest, 512]), io("status", "I32", [1])])
    batch.attend(r, longest=longest)
    runner = Runner(build_aim(tmp_path, weights, r))
    x = {n: t.cuda() for n, t in inputs.items() if n not in POOLS}
    for n, t in small.items():
        x[n] = torch.empty(pages, *t.shape[1:], dtype=t.dtype, device="cuda")
        x[n][-t.shape[0]:] = t.cuda()
    x["table"] = (table + (pages - small["k"].shape[0])).cuda()
    out = {"o": torch.full((longest, 512), 77.0, dtype=BF, device="cuda"), "status": torch.zeros(1, dtype=torch.int32, device="cuda")}
    runner.run(x, out)
    assert int(out["status"].cpu()) == 0
    check(batch, out["o"].cpu())


@pytest.mark.parametrize("new,total,longest", [([1, 4, 1], [60, 64, 1], 4), ([40, 1], [50, 30], 40)], ids=str)
def test_append_then_attend(tmp_path, new, total, longest):
    """A step as it is served: the launches of one recipe, the second reading what the first one has just written."""
    batch = Batch8(new, total, 16, (4, 2, 64), seed=14)
    hq, hk, d = batch.heads
    x = torch.randn(batch.rows, (hq + 2 * hk) * d, generator=torch.Generator().manual_seed(3)).to(BF)
    inputs = {"x": x, "table": batch.table, "lengths": batch.lengths, "starts": batch.starts}
    outputs = {**attention_outputs(batch), **batch.pools, "turned": torch.zeros(batch.rows, hq * d).to(BF)}

    def body(r):
        r.kv_append(Tensor("x"), Tensor("turned"), batch.cache(), rows=batch.rows, q_heads=hq, theta=1e4)
        r.paged_attention(Tensor("turned"), Tensor("o"), batch.cache(), rows=batch.rows, q_heads=hq, longest=longest)
        r.export_status(Tensor("status"))

    runner, dev, out = packaged(tmp_path, inputs, outputs, body)
    for _ in range(3):
        runner.run(dev, out)
    batch.q = out["turned"].cpu()
    tokens = {n: read_kv_pages(out[n].cpu(), out[n + "_scale"].cpu()).to(BF) for n in "kv"}
    row = 0
    for b, n in enumerate(batch.new):
        for i in range(n):
            j = batch.index(b, i)
            page = int(batch.table[b, j // 16])
            batch.keys[b][j], batch.values[b][j] = tokens["k"][page, j % 16], tokens["v"][page, j % 16]
            turned = paged.turn(x[row, hq * d:(hq + hk) * d].view(1, hk, d), paged.rotary_angles(torch.tensor([j]), 1e4, d))[0]
            assert bool(((batch.keys[b][j].double() - turned).abs() <= turned.abs() * 2.0 ** -4 + 2.0 ** -8).all())
            assert torch.equal(batch.values[b][j], rounded(x[row:row + 1, (hq + hk) * d:].view(1, hk, d))[0])
            row += 1
    assert int(out["status"].cpu()) == 0
    check(batch, out["o"].cpu())
