"""4-bit weights without a GPU: codes and scales, the packed layout, launch geometry, what the entry point refuses and what it launches."""
from __future__ import annotations

import random

import pytest
import torch

from aginfer_b200.recipes import Arena, RecipeBuilder, Tensor, Weight, io
from aginfer_b200.recipes import builder as B
from aginfer_b200.recipes.layout import pack_w4, quantize_w4, unpack_w4

M, N, K, G = 3, 40, 128, 64
SHAPES = {"codes": ("I32", [3, 2, 32, 4]), "scales": ("BF16", [3, 2, 8, 2])}


@pytest.mark.parametrize("group", [32, 64, 128])
def test_weights_are_off_by_half_a_step(group):
    w = torch.randn(37, 384, generator=torch.Generator().manual_seed(group)) * torch.logspace(-30, 30, 37)[:, None]
    w[5, :group] = 0.0
    codes, scales = quantize_w4(w, group)
    assert codes.dtype == torch.uint8 and int(codes.max()) <= 15 and scales.shape == (37, 384 // group) and float(scales[5, 0]) == 0
    back = (codes.double() - 8) * scales.double().repeat_interleave(group, 1)
    assert bool(((back - w.double()).abs() <= 0.5001 * scales.double().repeat_interleave(group, 1)).all())
    assert torch.equal(codes[5, :group], torch.full((group,), 8, dtype=torch.uint8))


@pytest.mark.parametrize("rows,group", [(37, 32), (16, 64), (1, 128), (48, 64)], ids=str)
def test_codes_pack_and_unpack(rows, group):
    g = torch.Generator().manual_seed(rows)
    codes = torch.randint(0, 16, (rows, 256), generator=g).to(torch.uint8)
    scales = torch.rand(rows, 256 // group, generator=g).to(torch.bfloat16)
    words, units = pack_w4(codes, scales)
    tiles = -(-rows // 16)
    assert words.dtype == torch.int32 and words.shape == (tiles, 4, 32, 4) and units.shape == (tiles, 256 // group, 8, 2)
    assert torch.equal(unpack_w4(words, units, rows), (codes.float() - 8) * scales.float().repeat_interleave(group, 1))
    for row, column in ((rows - 1, 200), (0, 0), (rows // 2, 255), (rows - 1, 97)):      # by hand
        tile, r, block, c = row // 16, row % 16, column // 64, column % 64
        lane, word = 4 * (r % 8) + c % 32 // 8, 2 * (c // 32) + c % 8 // 4
        bits = 4 * (r // 8 + 2 * (c % 4 // 2) + 4 * (c % 2))
        assert int(words[tile, block, lane, word]) >> bits & 15 == int(codes[row, column])
        assert units[tile, column // group, r % 8, r // 8] == scales[row, column // group]


@pytest.mark.parametrize("call", [lambda: quantize_w4(torch.zeros(4, 96), 64), lambda: pack_w4(torch.zeros(4, 96), torch.zeros(4, 3)),
                                  lambda: pack_w4(torch.zeros(4, 128), torch.zeros(3, 2)), lambda: pack_w4(torch.zeros(4, 128), torch.zeros(4, 3))])
def test_what_does_not_pack_is_refused(call):
    with pytest.raises(ValueError):
        call()


def test_every_geometry_fits():
    """Shared memory, scratch, counters, and that all blocks, tiles and tokens are somebody's."""
    rng = random.Random(7)
    for _ in range(3000):
        m, n, k, group = rng.randint(1, 32), int(10 ** rng.uniform(0, 5.3)), 64 * int(10 ** rng.uniform(0, 3.6)), rng.choice((32, 64, 128))
        t = B.w4_tiling(m, max(n, 1), max(k, 128), group)
        if t is None:
            continue
        tiles, blocks, (ctas, groups, splits) = -(-max(n, 1) // 16), max(k, 128) // 64, t["grid"]
        per = -(-blocks // splits)
        assert 2 <= t["stages"] <= 8 and t["chunk"] % 4 == 0 and t["ways"] in (1, 2, 4, 8)
        assert t["shared_bytes"] == 16 * t["stages"] * t["chunk"] * 576 + per * t["eights"] * (672 if group == 32 else 608)
        assert t["shared_bytes"] + B.W4_STATIC_BYTES <= B.MAX_DYNAMIC_SHARED
        assert groups * 4 * t["eights"] >= m and (splits - 1) * per < blocks <= splits * per and 1 <= ctas * groups * splits <= B.SM_COUNT
        assert splits == 1 or (tiles * groups * splits * 16 * 4 * t["eights"] * 4 <= B.TC_SCRATCH_BYTES and tiles * groups * 4 <= B.TC_COUNTER_BYTES)
        assert B.w4_tiling(m, max(n, 1), max(k, 128), group) is t


def builder(**weights) -> RecipeBuilder:
    r = RecipeBuilder({"w": ("BF16", (8,)), "codes": ("F32", (3, 2, 32, 4)), "scales": ("BF16", (3, 2, 8, 2)), **weights})
    r.begin_profile("default", [io("x", "BF16", [M, K]), io("wide", "BF16", [M, K + 8]), io("bias", "BF16", [N]), io("residual", "BF16", [M, N]),
                                io("c", *SHAPES["codes"]), io("s", *SHAPES["scales"]), io("s32", "BF16", [3, 4, 8, 2])],
                    [io("y", "BF16", [M, N]), io("y_wide", "BF16", [M, N + 24]), io("c_out", *SHAPES["codes"]), io("xy", "BF16", [M, K])])
    return r


def product(r, x=Tensor("x"), w=Tensor("c"), s=Tensor("s"), y=Tensor("y"), m=M, n=N, k=K, **kw):
    r.gemm_w4(x, w, s, y, m, n, k, **dict(group=G) | kw)
    return r._profile.launches[-1]


def early(launch) -> int:
    return launch["arguments"][-1]["scalar_u32"]


def test_forms():
    r = builder()
    assert product(r)["kernel"] == "agi_gemm_w4_g64_t1" and early(product(r)) == 1
    assert early(product(r, w=Weight("codes"), s=Weight("scales"))) == 1
    assert early(product(r, w=Tensor("c_out"))) == 0 and early(product(r, w=Arena(1 << 20))) == 0      # an earlier launch may have written them
    assert product(r, x=Tensor("wide"), ldx=K + 8, y=Tensor("y_wide"), ldy=N + 24, bias=Tensor("bias"), act="silu")["kernel"] == "agi_gemm_w4_g64_t1"
    assert product(r, s=Tensor("s32"), group=32)["kernel"] == "agi_gemm_w4_g32_t1"
    assert product(r, residual=Tensor("residual"))["kernel"] == "agi_gemm_w4_g64_t1"
    r.plan()


def recipe(m: int) -> RecipeBuilder:
    r = RecipeBuilder({"w": ("BF16", (8,))})
    r.begin_profile("default", [io("x", "BF16", [m, K]), io("c", *SHAPES["codes"]), io("s", *SHAPES["scales"])], [io("y", "BF16", [m, N]), io("s_out", *SHAPES["scales"])])
    return r


@pytest.mark.parametrize("m", [17, 400])
def test_more_tokens_are_tiles_of_converted_weights(m):
    r = recipe(m)
    launch = product(r, m=m)
    assert launch["kernel"].startswith("agi_gemm_tk_w4") and len(r._profile.launches) == 2
    late = lambda: r._profile.launches[-1]["arguments"][7]["scalar_u32"] & B.FLAG_LATE_WEIGHTS  # noqa: E731
    assert not late()
    product(r, m=m, w=Arena(1 << 20))
    assert late()
    product(r, m=m, s=Tensor("s_out"))
    assert late()


def test_many_tokens_go_through_bf16_weights_in_scratch():
    r = recipe(401)
    before = r.mark()
    product(r, m=401)
    first, second = r._profile.launches[-2:]
    assert first["kernel"] == "agi_dequantize_w4_bf16" and second["kernel"].startswith("agi_gemm_tk_bf16") and r.mark() == before
    assert second["arguments"][15] == first["arguments"][2], "the product's weights are those that were brought out"
    assert second["arguments"][9]["scalar_u32"] & B.FLAG_LATE_WEIGHTS, "and not asked for before that"


def test_tiles_of_converted_weights_fit():
    rng = random.Random(8)
    for _ in range(300):
        m, n, k = rng.choice((rng.randint(17, 400), rng.randint(1, 400))), int(10 ** rng.uniform(0, 4.8)), 64 * int(10 ** rng.uniform(0, 2.6))
        t = B.w4_tk_tiling(m, max(n, 1), max(k, 64))
        assert t["NB"] % 16 == 0 and 16 <= t["NB"] <= 128 and t["C"] in (1, 2, 4, 8) and t["stages"] >= 2 and t["shared_bytes"] <= B.TK_SMEM_BUDGET
        assert t["tiles"] * t["NB"] >= n and t["groups"] * t["tg"] >= m


@pytest.mark.parametrize("kw,match", [
    (dict(group=16), "groups of"), (dict(group=96), "groups of"), (dict(k=96), "multiple"), (dict(k=64, group=128), "multiple"), (dict(k=0), "multiple"),
    (dict(m=0), "below 1"), (dict(n=0), "below 1"), (dict(m=1 << 24), "below 1"),
    (dict(ldx=K - 8), "rows of"), (dict(ldx=K + 4), "rows of"), (dict(ldy=N - 1), "rows of"),
    (dict(m=M + 1), "x"), (dict(m=1, k=192, w=Arena(1 << 21), s=Weight("scales")), "weight 'scales'"), (dict(n=49), "y"),
    (dict(w=Tensor("s")), "codes"), (dict(s=Tensor("s32")), "scales"), (dict(w=Weight("w")), "weight 'w'"), (dict(s=Weight("codes")), "weight 'codes'"),
    (dict(bias=Tensor("nobody")), "no tensor"), (dict(residual=Tensor("bias")), "residual"), (dict(x=Arena((1 << 20) + 8)), "16-byte"),
    (dict(w=Arena((1 << 20) + 4)), "16-byte"), (dict(y=Tensor("residual")), "output of the profile"), (dict(x=Tensor("xy"), y=Tensor("xy"), n=K, w=Arena(1 << 21), s=Arena(1 << 22)), "still read"),
    (dict(x=Arena(1 << 20), y=Arena((1 << 20) + 2 * K)), "still read"), (dict(ldx=K + 8), "x"),
], ids=str)
def test_what_does_not_fit_is_refused(kw, match):
    with pytest.raises(ValueError, match=match):
        product(builder(), **kw)


def test_a_served_decoder_of_fewer_bits_packages():
    from aginfer_b200.recipes import paged_decode
    from aginfer_b200.recipes.decoder_layer import LayerConfig
    from aginfer_b200.recipes.package import describe
    layer = LayerConfig(hidden=256, heads=4, kv_heads=2, head_dim=64, intermediate=704, tokens=48)
    for window in (0, 128):
        cfg = paged_decode.ServeConfig(layer=layer, layers=2, sequences=3, page=16, new_tokens=6, window=window, weight_bits=4, cache_bits=8)
        weights = paged_decode.quantize_weights(cfg, paged_decode.synthetic_weights(cfg))
        assert not any(".q_proj" in n or ".gate_proj" in n for n in weights) and weights["model.layers.1.self_attn.qkv_proj.bias"].shape == (512,)
        plan = paged_decode.build_recipe(cfg, describe(weights)).plan()
        prompt, step = ([l["kernel"] for l in p["launches"]] for p in plan["shape_dispatch"])
        assert sum("gemm_tk_w4" in k for k in prompt) == 8 and step.count("agi_gemm_w4_g64_t1") == 8      # 48 tokens, three
        assert prompt.count("agi_kv_append_e4m3") == step.count("agi_kv_append_e4m3") == 2
        assert step.count("agi_paged_few_e4m3_d64_r8") == 2 and step.count("agi_kv_read_e4m3") == (0 if window else 2)


@pytest.mark.parametrize("kw", [dict(weight_bits=8), dict(cache_bits=4), dict(weight_bits=0)], ids=str)
def test_served_decoders_that_are_refused(kw):
    from aginfer_b200.recipes import paged_decode
    with pytest.raises(ValueError, match="bits"):
        paged_decode.ServeConfig(**kw)
