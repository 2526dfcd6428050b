"""Paged K/V cache without a GPU: the pool's layout, what the entry points refuse, and that a recipe of them packages."""
from __future__ import annotations

import pytest
import torch

from aginfer_b200.recipes import Arena, PagedCache, RecipeBuilder, Tensor, io
from aginfer_b200.recipes.layout import pack_kv_pages, unpack_kv_pages

CACHE = dict(k=Tensor("k"), v=Tensor("v"), table=Tensor("table"), lengths=Tensor("lengths"), starts=Tensor("starts"), sequences=3, pages=9, page=16,
             pages_per_sequence=4, kv_heads=2, head_dim=128)
ROWS, HEADS = 5, 8


def builder() -> RecipeBuilder:
    r = RecipeBuilder({"w": ("BF16", (8,))})
    pool = [9, 2, 2, 16, 64]
    r.begin_profile("default", [io("q", "BF16", [ROWS, HEADS * 128]), io("qkv", "BF16", [ROWS, (HEADS + 4) * 128]), io("table", "I32", [3, 4]),
                                io("lengths", "I32", [3]), io("starts", "I32", [4]), io("positions", "I32", [3, ROWS]), io("at", "I32", [1]),
                                io("pages", "I32", [6]), io("k_in", "BF16", pool)],
                    [io("o", "BF16", [ROWS, HEADS * 128]), io("k", "BF16", pool), io("v", "BF16", pool)])
    return r


def append(r, **kw):
    cache = PagedCache(**CACHE | kw.pop("cache", {}))
    r.kv_append(kw.pop("x", Tensor("qkv")), kw.pop("out", Tensor("o")), cache, **dict(rows=ROWS, q_heads=HEADS, theta=1e6) | kw)


def attend(r, **kw):
    cache = PagedCache(**CACHE | kw.pop("cache", {}))
    r.paged_attention(kw.pop("q", Tensor("q")), kw.pop("o", Tensor("o")), cache, **dict(rows=ROWS, q_heads=HEADS) | kw)


def share(r, **kw):
    cache = PagedCache(**CACHE | kw.pop("cache", {}))
    r.prefix_attention(Tensor("q"), Tensor("o"), cache, kw.pop("table", Tensor("pages")), kw.pop("length", Tensor("at")),
                       **dict(rows=ROWS, q_heads=HEADS, prefix_pages=6) | kw)


def test_pages_pack_and_unpack():
    for page, heads, d in ((16, 2, 64), (128, 1, 128)):
        t = torch.arange(3 * page * heads * d).reshape(3, page, heads, d).to(torch.int16)
        p = pack_kv_pages(t)
        assert p.shape == (3, heads, d // 64, page, 64) and torch.equal(unpack_kv_pages(p), t)
        token, column = 13, d - 3       # one element by hand
        chunk = (column % 64 // 8) ^ (token & 7)
        assert p[2, heads - 1, column // 64, token, chunk * 8 + column % 8] == t[2, token, heads - 1, column]


def test_the_operators_package_together():
    r = builder()
    append(r)
    append(r, positions=Tensor("positions"), sections=(16, 24, 24))
    append(r, offset=Tensor("at"))
    attend(r)
    attend(r, window=100, sinks=4, longest=2, scale=0.1)
    share(r)
    share(r, longest=1)
    plan = r.plan()
    assert [t["op"] for t in r.tactic_database()["tactics"] if t["op"] != "prologue"] and plan["shape_dispatch"][0]["launches"]


@pytest.mark.parametrize("change", [dict(page=8), dict(page=48), dict(head_dim=80), dict(head_dim=256), dict(sequences=0), dict(pages=0),
                                    dict(pages_per_sequence=0), dict(kv_heads=0), dict(sequences=5000), dict(pages_per_sequence=1 << 27)], ids=str)
def test_caches_that_are_refused(change):
    with pytest.raises(ValueError):
        PagedCache(**CACHE | change)


@pytest.mark.parametrize("kw", [
    dict(rows=0), dict(rows=1 << 24), dict(q_heads=7), dict(q_heads=0), dict(rows=6), dict(cache=dict(pages=8)), dict(cache=dict(page=32)),
    dict(cache=dict(kv_heads=1)), dict(cache=dict(sequences=4)), dict(cache=dict(pages_per_sequence=5)), dict(cache=dict(k=Tensor("lengths"))),
    dict(cache=dict(k=Tensor("nothing"))), dict(cache=dict(lengths=Tensor("q")))], ids=str)
@pytest.mark.parametrize("call", [append, attend, share])
def test_batches_that_are_refused(call, kw):
    with pytest.raises(ValueError):
        call(builder(), **kw)


@pytest.mark.parametrize("kw", [
    dict(row_stride=1000), dict(row_stride=(HEADS + 4) * 128 + 4), dict(out_stride=1000), dict(k=Tensor("q")), dict(kv_stride=256),
    dict(sections=(16, 24, 24)), dict(positions=Tensor("positions"), sections=(16, 24, 25)), dict(positions=Tensor("positions"), sections=(64,)),
    dict(positions=Tensor("positions"), sections=(-1, 1, 64)), dict(positions=Tensor("lengths")), dict(offset=Tensor("q")),
    dict(positions=Tensor("positions"), offset=Tensor("at")), dict(theta=0.0), dict(ladder=65), dict(cache=dict(k=Tensor("k_in"))),
    dict(x=Tensor("q")), dict(x=Arena(8)), dict(out=Tensor("qkv"))], ids=str)
def test_appends_that_are_refused(kw):
    with pytest.raises(ValueError):
        append(builder(), **kw)


@pytest.mark.parametrize("kw", [dict(longest=0), dict(longest=6), dict(window=-1), dict(sinks=3), dict(window=4, sinks=-1), dict(q_stride=1025),
                                dict(o_stride=512), dict(q=Arena(24)), dict(o=Tensor("lengths")), dict(window=1 << 30), dict(scale=0.0),
                                dict(scale=-1.0)], ids=str)
def test_attention_that_is_refused(kw):
    with pytest.raises(ValueError):
        attend(builder(), **kw)


@pytest.mark.parametrize("kw", [dict(prefix_pages=0), dict(prefix_pages=7), dict(prefix_pages=1 << 28), dict(table=Tensor("q")), dict(length=Tensor("q"))], ids=str)
def test_prefixes_that_are_refused(kw):
    with pytest.raises(ValueError):
        share(builder(), **kw)


def test_every_kernel_of_the_paged_decoder_is_an_entry_point():
    from aginfer_b200.build import build_all
    from aginfer_b200.recipes import paged_decode
    from aginfer_b200.recipes.decoder_layer import LayerConfig
    from aginfer_b200.recipes.package import describe
    from tests.test_cubin_symbols_cpu import function_symbols
    entry_points = function_symbols(build_all()[1].read_bytes())
    for window, heads in ((0, (4, 2, 64)), (64, (7, 1, 128)), (0, (64, 1, 64))):
        layer = LayerConfig(hidden=256, heads=heads[0], kv_heads=heads[1], head_dim=heads[2], intermediate=704, tokens=64)
        cfg = paged_decode.ServeConfig(layer=layer, layers=2, sequences=3, page=16, new_tokens=40, window=window)
        plan = paged_decode.build_recipe(cfg, describe(paged_decode.synthetic_weights(cfg))).plan()
        used = {l["kernel"] for p in plan["shape_dispatch"] for l in p["launches"]}
        assert used <= entry_points, sorted(used - entry_points)
        assert {p["profile"] for p in plan["shape_dispatch"]} == {"prompt", "step"}


@pytest.mark.parametrize("kw", [dict(window=64, tokens=70), dict(fp8=True)], ids=str)
def test_paged_decoders_that_are_refused(kw):
    from aginfer_b200.recipes import paged_decode
    from aginfer_b200.recipes.decoder_layer import LayerConfig
    with pytest.raises(ValueError):
        paged_decode.ServeConfig(layer=LayerConfig(tokens=kw.get("tokens", 64), fp8=kw.get("fp8", False)), window=kw.get("window", 0))


def test_more_key_tiles_than_a_launch_numbers_are_refused():
    r = RecipeBuilder({"w": ("BF16", (8,))})
    r.begin_profile("default", [], [])
    at = Arena(1 << 20)
    cache = PagedCache(k=at, v=at, table=at, lengths=at, starts=at, sequences=4096, pages=1 << 20, page=128, pages_per_sequence=1 << 14, kv_heads=8,
                       head_dim=128)
    r.paged_attention(at, at, cache, rows=4, q_heads=8)
    with pytest.raises(ValueError):
        r.paged_attention(at, at, cache, rows=4096, q_heads=64)


def test_tilings_stay_inside_what_an_sm_and_the_scratch_hold():
    from aginfer_b200.recipes.builder import SM_COUNT, TC_COUNTER_BYTES, TC_SCRATCH_BYTES, paged_few_tiling, paged_many_tiling
    for d in (64, 128):
        for page in (16, 128):
            cache = PagedCache(**CACHE | dict(head_dim=d, page=page, sequences=4096, pages_per_sequence=1000))
            for rows in range(1, 33):
                t = paged_few_tiling(cache, 4096, 1, rows)
                assert t["rows"] >= min(rows, 32) and t["stages"] >= 2 and t["grid"] * 4 <= TC_COUNTER_BYTES
                per_sm = 1 if t["rows"] == 32 and d == 128 else 2
                static = {8: 384, 16: 640, 32: 1152}[t["rows"]]      # barriers, maxima and weights of the warps
                assert per_sm * (t["shared_bytes"] + static + 1024) <= 228 * 1024
                assert t["grid"] * 2 * t["rows"] * (d + 2) * 4 <= TC_SCRATCH_BYTES
            t = paged_many_tiling(cache, 100, 128000)
            assert t["grid"] <= SM_COUNT and 2 <= t["stages"] <= 6 and t["shared_bytes"] + 2048 <= 227 * 1024


def test_no_cta_waits_for_one_that_may_lack_tensor_memory():
    """The order that tests/test_tensor_memory_cpu.py reads off the other kernels, for the paged one."""
    from tests.test_tensor_memory_cpu import body_events
    events = body_events("paged_many.cuh")
    assert events.count("tmem_alloc") == events.count("tmem_free") == 1 and "cluster_wait" not in events
    assert all(events.index("tmem_alloc") < i for i, e in enumerate(events) if "grid_dependency" in e)
