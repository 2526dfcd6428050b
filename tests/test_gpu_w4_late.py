"""4-bit weights that an earlier launch of the recipe writes: every run multiplies by what that launch has just left, whatever the runs before it read."""
from __future__ import annotations

import pytest
import torch

from aginfer_b200 import runtime as rt
from aginfer_b200.recipes import U32, RecipeBuilder, Tensor, io
from aginfer_b200.recipes.layout import pack_w4
from aginfer_b200.recipes.package import build_aim, describe
from aginfer_b200.runner import Runner
from tests.gpu_util import spec
from tests.test_gpu_w4 import BF, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,k,group", [(128, 128, 64), (300, 1152, 32), (2000, 2048, 128)], ids=str)
@pytest.mark.parametrize("m", [2, 12, 40, 200, 410])
def test_codes_and_scales_that_change_from_run_to_run(tmp_path, m, n, k, group):
    case = Case(m, n, k, group)
    inputs = {"x": case.x, "c": case.words, "s": case.units}
    weights = {"unused.pad": torch.zeros(8, dtype=BF)}
    r = RecipeBuilder(describe(weights))
    r.begin_profile("default", [spec(name, t) for name, t in inputs.items()], [io("y", "BF16", [m, n]), io("status", "I32", [1])])
    codes, scales = r.alloc(case.words.numel() * 4), r.alloc(case.units.numel() * 2)
    for name, to, words in (("s", scales, case.units.numel() // 2), ("c", codes, case.words.numel())):
        r.launch("agi_copy_u32", (-(-words // 256), 1, 1), (256, 1, 1), [Tensor(name), to, U32(words)])
    r.gemm_w4(Tensor("x"), codes, scales, Tensor("y"), m, n, k, group=group)
    r.export_status(Tensor("status"))
    runner = Runner(build_aim(tmp_path, weights, r), flags=rt.PROGRAMMATIC_LAUNCH)
    x = {name: t.cuda() for name, t in inputs.items()}
    out = {"y": torch.zeros(m, n, dtype=BF, device="cuda"), "status": torch.zeros(1, dtype=torch.int32, device="cuda")}
    g = torch.Generator().manual_seed(m + n)
    for _ in range(3):
        runner.run(x, out)
    for _ in range(8):
        case.codes = torch.randint(0, 16, (n, k), generator=g).to(torch.uint8)
        case.scales = (torch.exp(torch.randn(n, k // group, generator=g)) * 0.1).to(BF)
        case.words, case.units = pack_w4(case.codes, case.scales)
        x["c"].copy_(case.words)
        x["s"].copy_(case.units)
        out["y"].fill_(77.0)
        runner.run(x, out)
        assert int(out["status"].cpu()) == 0
        case.check(out["y"].cpu())
