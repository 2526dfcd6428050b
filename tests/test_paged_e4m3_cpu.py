"""Paged caches in 8 bits without a GPU: layout and rounding of the pools, what the entry points refuse, and what they launch."""
from __future__ import annotations

import math

import pytest
import torch

from aginfer_b200.recipes import Arena, PagedCache, RecipeBuilder, Tensor, io
from aginfer_b200.recipes.layout import quantize_kv_pages, read_kv_pages

ROWS, HEADS, KV, DIM, PAGES, PAGE = 5, 8, 2, 128, 9, 16
NAMES = dict(k=Tensor("k"), v=Tensor("v"), k_scale=Tensor("ks"), v_scale=Tensor("vs"), table=Tensor("table"), lengths=Tensor("lengths"), starts=Tensor("starts"))
SHAPE = dict(sequences=3, pages=PAGES, page=PAGE, pages_per_sequence=4, kv_heads=KV, head_dim=DIM)
WIDE = dict(k=Tensor("k16"), v=Tensor("v16"), table=Tensor("table16"), lengths=Tensor("lengths"), starts=Tensor("starts"))


def builder() -> RecipeBuilder:
    r = RecipeBuilder({"w": ("BF16", (8,))})
    codes, scales, wide = [PAGES, KV, PAGE, DIM], [PAGES, KV, PAGE], [12, KV, DIM // 64, PAGE, 64]
    r.begin_profile("default", [io("q", "BF16", [ROWS, HEADS * DIM]), io("qkv", "BF16", [ROWS, (HEADS + 2 * KV) * DIM]), io("table", "I32", [3, 4]),
                                io("lengths", "I32", [3]), io("starts", "I32", [4]), io("at", "I32", [1]), io("pages", "I32", [6]),
                                io("codes_in", "F8_E4M3", codes), io("scales_in", "BF16", scales)],
                    [io("o", "BF16", [ROWS, HEADS * DIM]), io("k", "F8_E4M3", codes), io("v", "F8_E4M3", codes), io("ks", "BF16", scales),
                     io("vs", "BF16", scales), io("k16", "BF16", wide), io("v16", "BF16", wide), io("table16", "I32", [3, 4]),
                     io("bf16_pool", "BF16", [PAGES, KV, PAGE, DIM]), io("narrow", "BF16", [PAGES, KV, PAGE // 2])])
    return r


def cache(**kw) -> PagedCache:
    return PagedCache(**NAMES | SHAPE | kw)


def wide(**kw) -> PagedCache:
    return PagedCache(**WIDE | SHAPE | dict(pages=12) | kw)


def append(r, **kw):
    r.kv_append(Tensor("qkv"), Tensor("o"), cache(**kw.pop("cache", {})), **dict(rows=ROWS, q_heads=HEADS, theta=1e6) | kw)


def attend(r, **kw):
    r.paged_attention(Tensor("q"), Tensor("o"), cache(**kw.pop("cache", {})), **dict(rows=ROWS, q_heads=HEADS) | kw)


def share(r, **kw):
    r.prefix_attention(Tensor("q"), Tensor("o"), cache(**kw.pop("cache", {})), Tensor("pages"), Tensor("at"), **dict(rows=ROWS, q_heads=HEADS, prefix_pages=6) | kw)


def read(r, **kw):
    r.kv_read(cache(**kw.pop("cache", {})), wide(**kw.pop("to", {})), **dict(rows=ROWS) | kw)


@pytest.mark.parametrize("page,heads,d", [(16, 2, 64), (128, 1, 128), (32, 3, 128)], ids=str)
def test_tokens_are_rounded_once_to_codes_and_a_power_of_two(page, heads, d):
    g = torch.Generator().manual_seed(d + page)
    t = torch.ldexp(torch.randn(3, page, heads, d, generator=g), torch.randint(-30, 30, (3, page, heads, 1), generator=g))
    t[0, 3], t[1, 5, 0, 7] = 0.0, 448.0 * 2 ** 40
    codes, scales = quantize_kv_pages(t)
    assert codes.shape == (3, heads, page, d) and codes.dtype == torch.uint8 and scales.shape == (3, heads, page)
    s = scales.double().permute(0, 2, 1)
    assert bool((torch.frexp(s)[0] == 0.5).all()) and bool((s[0, 3] == 1).all())
    peak = t.double().abs().amax(-1)
    assert bool((peak <= 448 * s).all()) and bool(((peak > 224 * s) | (peak == 0)).all())
    back = read_kv_pages(codes, scales).double()
    assert bool(((back - t.double()).abs() <= (t.double().abs() * 2.0 ** -4).clamp_min(s[..., None] * 2.0 ** -10)).all())
    assert torch.equal(back.to(torch.bfloat16).double(), back), "codes times scales are bf16 numbers"
    token, column = page - 3, d - 5       # one code by hand
    chunk = (column // 16) ^ (token & 7 if d == 128 else (token >> 1) & 3)
    value = float(codes.view(torch.float8_e4m3fn)[2, heads - 1, token, chunk * 16 + column % 16]) * float(s[2, token, heads - 1])
    assert value == float(back[2, token, heads - 1, column])


@pytest.mark.parametrize("peak,exponent", [(448.0, 0), (448.0001, 1), (224.0, -1), (224.0001, 0), (1.0, -8), (1.75, -8), (1.7500001, -7), (2.0 ** -118, -126),
                                           (2.0 ** -140, -126), (3.3e38, 120)], ids=str)
def test_the_scale_of_a_largest_value(peak, exponent):
    t = torch.zeros(1, 16, 1, 64)
    t[0, 4, 0, 9] = -peak
    scale = float(quantize_kv_pages(t)[1][0, 0, 4])
    assert scale == 2.0 ** exponent


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_a_token_that_is_not_finite_is_nan(value):
    t = torch.ones(1, 16, 2, 64)
    t[0, 4, 1, 9] = value
    codes, scales = quantize_kv_pages(t)
    back = read_kv_pages(codes, scales)
    assert bool(back[0, 4, 1].isnan().all()) and bool((back[0, 4, 0] == 1).all()) and int(back.isnan().sum()) == 64
    assert bool((codes[0, 1, 4] == 0).all())


def test_the_operators_package_together():
    r = builder()
    append(r)
    append(r, offset=Tensor("at"))
    attend(r)
    attend(r, longest=2)
    attend(r, window=100, sinks=4, longest=2, scale=0.1)
    share(r)
    share(r, longest=1)
    read(r)
    read(r, window=40, sinks=3)
    names = [l["kernel"] for l in r._profile.launches[1:]]
    assert names == ["agi_kv_append_e4m3"] * 2 + ["agi_paged_few_e4m3_d128_r32"] + ["agi_paged_few_e4m3_d128_r8"] * 2 + \
        ["agi_kv_read_e4m3", "agi_paged_few_e4m3_d128_r32", "agi_paged_prefix_bf16_d128", "agi_paged_join_prefix_bf16_d128"] + \
        ["agi_kv_read_e4m3", "agi_paged_few_e4m3_d128_r8", "agi_paged_prefix_bf16_d128", "agi_paged_join_prefix_bf16_d128"] + ["agi_kv_read_e4m3"] * 2
    assert r.plan()["shape_dispatch"][0]["launches"] == r._profile.launches


def test_many_rows_read_the_pages_back_first():
    r = RecipeBuilder({"w": ("BF16", (8,))})
    r.begin_profile("default", [io("q", "BF16", [100, HEADS * DIM]), io("table", "I32", [3, 4]), io("lengths", "I32", [3]), io("starts", "I32", [4]),
                                io("k", "F8_E4M3", [PAGES, KV, PAGE, DIM]), io("v", "F8_E4M3", [PAGES, KV, PAGE, DIM]), io("ks", "BF16", [PAGES, KV, PAGE]),
                                io("vs", "BF16", [PAGES, KV, PAGE]), io("pages", "I32", [6]), io("at", "I32", [1])], [io("o", "BF16", [100, HEADS * DIM])])
    before = r.mark()
    attend(r, rows=100)
    share(r, rows=100)
    assert r.mark() == before
    names = [l["kernel"] for l in r._profile.launches[1:]]
    own = ["agi_paged_many_bf16_d128", "agi_paged_join_bf16_d128"]
    assert names == ["agi_kv_read_e4m3", *own, "agi_kv_read_e4m3", "agi_kv_read_e4m3", *own, "agi_paged_prefix_bf16_d128", "agi_paged_join_prefix_bf16_d128"]
    read_back, many = r._profile.launches[1], r._profile.launches[2]
    # the kernel reads what was brought back: pools, table, page count
    assert [many["arguments"][i] for i in (2, 3, 6)] == [read_back["arguments"][i] for i in (7, 8, 9)]
    assert many["arguments"][16] == {"scalar_u32": 12}


@pytest.mark.parametrize("call,kw,match", [
    (append, dict(cache=dict(k_scale=None)), "both held in 8 bits"),
    (append, dict(cache=dict(k=Tensor("bf16_pool"))), "F8_E4M3"),
    (append, dict(cache=dict(v_scale=Tensor("narrow"))), "scales of values"),
    (append, dict(cache=dict(k=Tensor("codes_in"))), "output of the profile"),
    (append, dict(cache=dict(k_scale=Tensor("scales_in"))), "output of the profile"),
    (append, dict(cache=dict(k_scale=Arena(1 << 20 | 8))), "16-byte"),
    (attend, dict(cache=dict(head_dim=96)), "heads"),
    (attend, dict(cache=dict(pages=8)), "keys"),
    (share, dict(cache=dict(v_scale=Tensor("no"))), "no tensor"),
    (read, dict(to=dict(k_scale=Tensor("ks"), v_scale=Tensor("vs"))), "goes from"),
    (read, dict(cache=dict(k_scale=None, v_scale=None)), "goes from"),
    (read, dict(to=dict(sequences=2)), "same batch"),
    (read, dict(to=dict(lengths=Tensor("at"))), "same batch"),
    (read, dict(to=dict(page=32)), "same batch"),
    (read, dict(to=dict(pages=11)), "do not fit"),
    (read, dict(sinks=4), "go with a window"),
    (read, dict(window=-1), "counts of tokens"),
    (read, dict(rows=0), "rows"),
    (read, dict(to=dict(table=Tensor("table"))), "output of the profile"),
    (read, dict(to=dict(k=Tensor("v16"))), "tensors of their own"),
], ids=lambda v: getattr(v, "__name__", None) or str(v)[:60])
def test_what_does_not_fit_is_refused(call, kw, match):
    with pytest.raises(ValueError, match=match):
        call(builder(), **kw)


def test_a_table_with_more_pages_than_a_launch_numbers_is_refused():
    r = RecipeBuilder({"w": ("BF16", (8,))})
    sequences, width = 4096, 1 << 18
    r.begin_profile("default", [io("table", "I32", [sequences, width]), io("lengths", "I32", [sequences]), io("starts", "I32", [sequences + 1])],
                    [io("t16", "I32", [sequences, width])])
    shape = dict(sequences=sequences, pages_per_sequence=width, page=64, kv_heads=8, head_dim=64, lengths=Tensor("lengths"), starts=Tensor("starts"))
    at = Arena(1 << 20)
    with pytest.raises(ValueError, match="launch numbers"):
        r.kv_read(PagedCache(k=at, v=at + 16, k_scale=at + 32, v_scale=at + 48, table=Tensor("table"), pages=9, **shape),
                  PagedCache(k=at + 64, v=at + 80, table=Tensor("t16"), pages=sequences * width, **shape), rows=1)
