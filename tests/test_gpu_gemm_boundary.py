"""Tokens off a 16-byte boundary: the tcgen05 products, which copy rows in pieces of 16 bytes, say so and read and write nothing."""
from __future__ import annotations

import pytest
import torch

from aginfer_b200.recipes import RecipeBuilder, Tensor, Weight
from aginfer_b200.recipes.package import build_aim, describe
from aginfer_b200.runner import Runner
from tests.gpu_util import spec
from tests.test_gpu_w4 import BF, Case, packaged

pytestmark = pytest.mark.gpu


def off_its_boundary(t: torch.Tensor) -> torch.Tensor:
    flat = torch.zeros(t.numel() + 8, dtype=t.dtype, device="cuda")
    flat[1:1 + t.numel()].copy_(t.flatten())
    return flat[1:1 + t.numel()].view(t.shape)


@pytest.mark.parametrize("m,n,k", [(401, 64, 128), (450, 300, 1152), (700, 40, 4096)], ids=str)
def test_many_tokens_of_a_product_with_4_bit_weights(tmp_path, m, n, k):
    case = Case(m, n, k)
    runner, x, out = packaged(tmp_path, case)
    runner.run(x | {"x": off_its_boundary(x["x"])}, out)
    assert int(out["status"].cpu()) == 0x600 and bool((out["y"] == 77.0).all())
    runner.run(x, out)       # and the next call is as ever
    assert int(out["status"].cpu()) == 0
    case.check(out["y"].cpu())


@pytest.mark.parametrize("m", [40, 100, 1000])
def test_a_product(tmp_path, m):
    g = torch.Generator().manual_seed(m)
    weights = {"w": torch.randn(256, 1024, generator=g).to(BF)}
    inputs = {"x": torch.randn(m, 1024, generator=g).to(BF)}
    outputs = {"y": torch.full((m, 256), 77.0).to(BF), "status": torch.zeros(1, dtype=torch.int32)}
    r = RecipeBuilder(describe(weights))
    r.begin_profile("default", [spec(n, t) for n, t in inputs.items()], [spec(n, t) for n, t in outputs.items()])
    r.gemm(Tensor("x"), Weight("w"), Tensor("y"), m, 256, 1024)
    assert r._profile.launches[-1]["kernel"].startswith("agi_gemm_tk_bf16")
    r.export_status(Tensor("status"))
    runner = Runner(build_aim(tmp_path, weights, r))
    x, out = {"x": inputs["x"].cuda()}, {n: t.cuda() for n, t in outputs.items()}
    runner.run({"x": off_its_boundary(x["x"])}, out)
    assert int(out["status"].cpu()) == 0x600 and bool((out["y"] == 77.0).all())
    runner.run(x, out)
    assert int(out["status"].cpu()) == 0
    want = x["x"].cpu().double() @ weights["w"].double().t()
    mass = x["x"].cpu().double().abs() @ weights["w"].double().abs().t()
    assert bool(((out["y"].cpu().double() - want).abs() <= want.abs() * 2.0 ** -8 + mass * 2.0 ** -18).all())
