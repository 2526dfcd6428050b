"""Operands that an earlier launch of the recipe writes: attention over keys and values, and products of tokens, read what that launch has just left, in every
run, whatever the runs before read at the same place."""
from __future__ import annotations

import pytest
import torch

from aginfer_b200 import runtime as rt
from aginfer_b200.recipes import U32, RecipeBuilder, Tensor, Weight, io
from aginfer_b200.recipes.package import build_aim, describe
from aginfer_b200.runner import Runner

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def runs(tmp_path, rows: int, columns: int, weights, outputs, body, check) -> None:
    """Several runs over tokens that change, each moved into the arena by a launch in front of ``body``."""
    r = RecipeBuilder(describe(weights))
    r.begin_profile("default", [io("x", "BF16", [rows, columns])], [*outputs, io("status", "I32", [1])])
    x = r.alloc(rows * columns * 2)
    r.launch("agi_copy_u32", (-(-rows * columns // 512), 1, 1), (256, 1, 1), [Tensor("x"), x, U32(rows * columns // 2)])
    body(r, x)
    r.export_status(Tensor("status"))
    runner = Runner(build_aim(tmp_path, weights, r), flags=rt.PROGRAMMATIC_LAUNCH)
    kinds = {"BF16": BF, "I32": torch.int32}
    out = {t["name"]: torch.zeros(t["shape"], dtype=kinds[t["dtype"]], device="cuda") for t in outputs}
    out["status"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    g = torch.Generator().manual_seed(rows + columns)
    x = {"x": torch.zeros(rows, columns, dtype=BF, device="cuda")}
    for _ in range(10):
        fresh = torch.randn(rows, columns, generator=g).to(BF)
        x["x"].copy_(fresh)
        runner.run(x, out)
        assert int(out["status"].cpu()) == 0
        check(fresh.double(), out)


@pytest.mark.parametrize("algorithm,kernel", [("key_split", "agi_attention_rows_bf16"), ("keys_in_smem", "agi_attention_smem_bf16"), ("warp_per_row", "agi_attention_bf16"),
                                              ("auto", "agi_attention_mma_bf16")])
@pytest.mark.parametrize("rows,heads,d", [(8, 4, 64), (30, 2, 32)], ids=str)
def test_keys_and_values(tmp_path, rows, heads, d, algorithm, kernel):
    wide = 3 * heads * d

    def body(r, x):
        r.attention(x, x + 2 * heads * d, x + 4 * heads * d, Tensor("o"), q_rows=rows, kv_rows=rows, q_heads=heads, kv_heads=heads, head_dim=d, q_stride=wide,
                    k_stride=wide, v_stride=wide, o_stride=heads * d, mask="causal", algorithm=algorithm)
        assert r._profile.launches[-1]["kernel"] == kernel

    def check(x, out):
        q, k, v = (t.view(rows, heads, d).transpose(0, 1) for t in x.split(heads * d, dim=1))
        s = (q @ k.transpose(1, 2) * d ** -0.5).masked_fill(torch.ones(rows, rows).triu(1).bool(), float("-inf"))
        want = (s.softmax(-1) @ v).transpose(0, 1).reshape(rows, heads * d)
        # weights and outputs are rounded to bf16, half a step 2^-8 each, of values below 5
        assert float((out["o"].cpu().double() - want).abs().max()) <= 5 * 2.0 ** -7

    runs(tmp_path, rows, wide, {"unused.pad": torch.zeros(8, dtype=BF)}, [io("o", "BF16", [rows, heads * d])], body, check)


@pytest.mark.parametrize("tactic", ["skinny", "stream", "tcgen05_plan", "simt"])
@pytest.mark.parametrize("m,n,k", [(5, 64, 256), (30, 200, 1024)], ids=str)
def test_tokens_of_a_product(tmp_path, m, n, k, tactic):
    weights = {"w": torch.randn(n, k, generator=torch.Generator().manual_seed(n)).to(BF)}

    def check(x, out):
        w = weights["w"].double()
        want, mass = x @ w.t(), x.abs() @ w.abs().t()
        assert bool(((out["y"].cpu().double() - want).abs() <= want.abs() * 2.0 ** -8 + mass * 2.0 ** -18).all())

    runs(tmp_path, m, k, weights, [io("y", "BF16", [m, n])], lambda r, x: r.gemm(x, Weight("w"), Tensor("y"), m, n, k, tactic=tactic), check)
