"""Products with 4-bit weights against the definition in 64 bits."""
from __future__ import annotations

import pytest
import torch

from aginfer_b200 import runtime as rt
from aginfer_b200.recipes import RecipeBuilder, Tensor, Weight, io
from aginfer_b200.recipes.layout import pack_w4
from aginfer_b200.recipes.package import build_aim, describe
from aginfer_b200.runner import Runner
from tests.gpu_util import spec

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
ACT = {None: lambda v: v, "silu": lambda v: v * torch.sigmoid(v), "gelu_tanh": lambda v: torch.nn.functional.gelu(v, approximate="tanh"), "relu": torch.relu}


class Case:
    """A product and its definition.  ``bound`` follows from the roundings: of the output, half a bf16 step (2^-8); of a token, half a unit, of which
    the largest value of its 64 columns has at least 2^13: 2^-14 of that, or 2^-127, as the unit is at least 2^-126 (or, behind bf16 weights, half a step of
    each); of sums in 32 bits 2^-20 of sum |x| |w|."""

    def __init__(self, m: int, n: int, k: int, group: int = 64, seed: int = 0, bias=False, residual=False, act=None, x=None, ldx=None, ldy=None):
        g = torch.Generator().manual_seed(seed + m + n + k)
        self.m, self.n, self.k, self.group, self.act, self.ldx, self.ldy = m, n, k, group, act, ldx or k, ldy or n
        self.x = torch.randn(m, k, generator=g).to(BF) if x is None else x
        self.codes = torch.randint(0, 16, (n, k), generator=g).to(torch.uint8)
        self.scales = (torch.exp(torch.randn(n, k // group, generator=g)) * 0.1).to(BF)
        self.words, self.units = pack_w4(self.codes, self.scales)
        self.bias = torch.randn(n, generator=g).to(BF) if bias else None
        self.residual = torch.randn(m, self.ldy, generator=g).to(BF) if residual else None

    def inputs(self) -> dict:
        wide = torch.full((self.m, self.ldx), float("nan")).to(BF)
        wide[:, :self.k] = self.x
        x = {"x": wide, "codes": self.words, "scales": self.units, "bias": self.bias, "residual": self.residual}
        return {name: t for name, t in x.items() if t is not None}

    def launch(self, r: RecipeBuilder, w=Tensor("codes"), s=Tensor("scales"), y=Tensor("y")) -> None:
        r.gemm_w4(Tensor("x"), w, s, y, self.m, self.n, self.k, group=self.group, bias=Tensor("bias") if self.bias is not None else None,
                  residual=Tensor("residual") if self.residual is not None else None, act=self.act, ldx=self.ldx, ldy=self.ldy)

    def expected(self) -> tuple[torch.Tensor, torch.Tensor]:
        w = (self.codes.double() - 8) * self.scales.double().repeat_interleave(self.group, 1)
        x = self.x.double()
        y, mass = x @ w.t(), x.abs() @ w.abs().t()
        largest = x.abs().view(self.m, -1, 64).amax(2).repeat_interleave(64, 1)
        slack = mass * 2.0 ** -8 if self.m > 16 or self.k > 400000 else (largest * 2.0 ** -14).clamp_min(2.0 ** -127) @ w.abs().t()
        if self.bias is not None:
            y = y + self.bias.double()
        y, slack = ACT[self.act](y), 1.13 * (slack + (mass + y.abs()) * 2.0 ** -20)       # gelu is as steep as 1.13
        if self.act is not None:
            slack = slack + (y.abs() + 1) * 2.0 ** -18
        if self.residual is not None:
            y = y + self.residual[:, :self.n].double()
        return y, slack + y.abs() * 2.0 ** -8

    def check(self, got: torch.Tensor) -> None:
        want, bound = self.expected()
        y = got[:, :self.n].double()
        error = (y - want).abs()
        # what the bound lets lie beyond the largest bf16 may be infinite: that is what it rounds to
        beyond = (want.abs() + bound > torch.finfo(BF).max) & (y == want.sign() * float("inf"))
        assert bool((beyond | (error <= bound)).all()), f"{(error / bound)[~beyond].nan_to_num().max():.3g} times the bound"
        assert bool((got[:, self.n:] == 77.0).all()), "columns behind the row were written"


def packaged(tmp_path, case: Case, body=None, weights=None, flags=rt.PROGRAMMATIC_LAUNCH):
    weights = weights or {"unused.pad": torch.zeros(8, dtype=BF)}
    inputs = {n: t for n, t in case.inputs().items() if n not in weights}
    outputs = {"y": torch.full((case.m, case.ldy), 77.0).to(BF), "status": torch.zeros(1, dtype=torch.int32)}
    r = RecipeBuilder(describe(weights))
    r.begin_profile("default", [spec(n, t) for n, t in inputs.items()], [spec(n, t) for n, t in outputs.items()])
    (body or case.launch)(r)
    r.export_status(Tensor("status"))
    runner = Runner(build_aim(tmp_path, weights, r), flags=flags)
    return runner, {n: t.cuda() for n, t in inputs.items()}, {n: t.cuda() for n, t in outputs.items()}


def run_and_check(tmp_path, case: Case, repeats: int = 2) -> None:
    runner, x, out = packaged(tmp_path, case)
    first = None
    for _ in range(repeats):
        out["y"].fill_(77.0)
        runner.run(x, out)
        got = out["y"].cpu()
        assert first is None or torch.equal(first.view(torch.int16), got.view(torch.int16)), "runs of one input differ"
        first = got
    assert int(out["status"].cpu()) == 0
    case.check(first)


@pytest.mark.parametrize("n,k", [(1, 128), (16, 128), (17, 384), (300, 640), (2049, 128), (40, 8192)], ids=str)
@pytest.mark.parametrize("m", [1, 2, 4, 5, 8, 13, 16, 17, 100, 300, 401])
def test_sizes(tmp_path, m, n, k):
    run_and_check(tmp_path, Case(m, n, k))


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,n,k", [(1, 500, 1152), (3, 33, 2176), (9, 120, 1408), (33, 70, 384), (200, 300, 1152), (450, 70, 384)], ids=str)
def test_groups(tmp_path, m, n, k, group):
    run_and_check(tmp_path, Case(m, n, k, group))


def test_a_single_block_of_columns(tmp_path):
    run_and_check(tmp_path, Case(2, 50, 64, 32))


@pytest.mark.parametrize("m,n,k,group", [(1, 2560, 2048, 64), (8, 11000, 2048, 128), (12, 18000, 2048, 64), (1, 640, 18944, 32), (4, 2048, 11008, 64), (40, 2048, 1024, 64), (48, 2048, 11008, 32), (288, 4000, 2048, 64), (64, 300, 18944, 128),
                                          (2, 16, 512000, 128)], ids=str)
def test_sizes_of_decoders(tmp_path, m, n, k, group):
    """Several rounds a team, sets of one, two and eight warps, parts of K that meet."""
    run_and_check(tmp_path, Case(m, n, k, group), repeats=3)


def test_every_geometry_gives_the_same(tmp_path, monkeypatch):
    """All ways, parts, copies and depths of the ring over one product: rings that go round, warps without columns, tiles that not all warps have."""
    from aginfer_b200.recipes import builder as B
    case = Case(6, 1003, 2752, 64)
    for i, (eights, splits, ways, chunk, stages, ctas) in enumerate(((1, 1, 1, 4, 2, 3), (1, 1, 8, 8, 2, 1), (2, 1, 2, 4, 3, 5), (1, 5, 4, 4, 2, 7), (2, 3, 1, 8, 2, 2), (1, 43, 8, 4, 5, 3), (2, 2, 8, 4, 2, 2))):
        groups, per = -(-case.m // (4 * eights)), -(-43 // splits)
        tiling = {"eights": eights, "splits": splits, "ways": ways, "chunk": chunk, "stages": stages, "grid": (ctas, groups, splits),
                  "shared_bytes": 16 * stages * chunk * 576 + per * eights * 608}
        assert ctas * groups * splits <= 148 * 2 and tiling["shared_bytes"] + B.W4_STATIC_BYTES <= B.MAX_DYNAMIC_SHARED
        monkeypatch.setattr(B, "w4_tiling", lambda *a, tiling=tiling: tiling)
        where = tmp_path / str(i)
        where.mkdir()
        run_and_check(where, case, repeats=3)


def test_every_tile_of_converted_weights_gives_the_same(tmp_path, monkeypatch):
    """All clusters, heights and groups of tokens over one product: rings that go round, tiles of which part is no weight, ranks without columns."""
    from aginfer_b200.recipes import builder as B
    case = Case(150, 1003, 2752, 32)
    for i, (C, NB) in enumerate(((1, 16), (1, 128), (2, 48), (4, 80), (8, 112), (8, 32))):
        t = B.tk_tiling(150, (1003,), 2752, 2, clusters=(C,), rows_per_tile=NB, must_fit=False)
        monkeypatch.setattr(B, "w4_tk_tiling", lambda *a, t=t: t)
        where = tmp_path / str(i)
        where.mkdir()
        run_and_check(where, case, repeats=3)


@pytest.mark.parametrize("m", [1, 7, 40, 410])
@pytest.mark.parametrize("kw", [dict(bias=True), dict(residual=True), dict(bias=True, act="silu"), dict(bias=True, residual=True, act="gelu_tanh"), dict(act="relu"),
                                dict(ldx=520, ldy=144, bias=True, residual=True)], ids=str)
def test_epilogues_and_pitches(tmp_path, m, kw):
    run_and_check(tmp_path, Case(m, 133, 512, **kw))


@pytest.mark.parametrize("m", [3, 40, 410])
def test_weights_of_the_checkpoint(tmp_path, m):
    case = Case(m, 200, 512, 32)
    weights = {"l.weight": case.words.view(torch.float32), "l.weight_scale": case.units, "a": torch.zeros(3, dtype=BF)}
    runner, x, out = packaged(tmp_path, case, lambda r: case.launch(r, Weight("l.weight"), Weight("l.weight_scale")), weights)
    runner.run({"x": x["x"]} | {n: t for n, t in x.items()}, out)
    case.check(out["y"].cpu())


def test_tokens_of_unequal_size(tmp_path):
    """Tokens, and blocks and columns of a token, that differ by powers of two; zeros; one value a thousand times its neighbours."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(8, 1024, generator=g)
    x[0] *= 2.0 ** -100
    x[1] *= 2.0 ** 60
    x[2] = 0.0
    x[3] *= torch.logspace(-6, 6, 16).repeat_interleave(64)
    x[4, 5::64] *= 1000.0
    x[5, :960] = 0.0
    x[6] = x[6].abs()
    x[7, 100] = 3.0e38
    run_and_check(tmp_path, Case(8, 100, 1024, x=x.to(BF)))
    (tmp_path / "tiny").mkdir()
    run_and_check(tmp_path / "tiny", Case(1, 100, 1024, 128, x=(torch.randn(1, 1024, generator=g) * 2.0 ** -131).to(BF)))


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_a_token_that_is_not_finite_keeps_to_itself(tmp_path, value):
    case = Case(5, 70, 512)
    runner, x, out = packaged(tmp_path, case)
    x["x"][3, 77] = value
    runner.run(x, out)
    got = out["y"].cpu()
    assert bool(got[3].isnan().all())
    got[3] = case.expected()[0][3].to(BF)
    case.check(got)


@pytest.mark.parametrize("m", [2, 40, 410])
def test_what_the_codes_are_is_read_when_the_launch_runs(tmp_path, m):
    """Weights that an earlier launch of the recipe writes, and outputs of one product that are the next one's tokens."""
    case, second = Case(m, 128, 128, 64), Case(m, 60, 128, 32, seed=5)
    weights = {"codes": second.words.view(torch.float32), "scales": second.units}
    inputs = {"x": case.x, "c": case.words, "s": case.units}

    def body(r):
        middle, copied = r.alloc(m * 128 * 2), r.alloc(case.words.numel() * 4)
        r.launch("agi_copy_u32", (1, 1, 1), (32, 1, 1), [Tensor("c"), copied, _u32(case.words.numel())])
        r.gemm_w4(Tensor("x"), copied, Tensor("s"), middle, m, 128, 128, group=64)
        r.gemm_w4(middle, Weight("codes"), Weight("scales"), Tensor("y"), m, 60, 128, group=32)

    from aginfer_b200.recipes import U32 as _u32
    r = RecipeBuilder(describe(weights))
    r.begin_profile("default", [spec(n, t) for n, t in inputs.items()], [io("y", "BF16", [m, 60])])
    body(r)
    runner, out = Runner(build_aim(tmp_path, weights, r), flags=rt.PROGRAMMATIC_LAUNCH), {"y": torch.zeros(m, 60, dtype=BF, device="cuda")}
    x = {n: t.cuda() for n, t in inputs.items()}
    for _ in range(3):
        runner.run(x, out)
    middle = case.expected()
    second.x = middle[0].to(BF)
    want, bound = second.expected()
    w = (second.codes.double() - 8).abs() * second.scales.double().repeat_interleave(32, 1)
    assert bool(((out["y"].cpu().double() - want).abs() <= bound + (middle[1] + middle[0].abs() * 2.0 ** -8) @ w.t()).all())
    x["c"].copy_(torch.randint(-2 ** 31, 2 ** 31 - 1, x["c"].shape, dtype=torch.int32))
    before = out["y"].clone()
    runner.run(x, out)
    assert not torch.equal(before, out["y"])


@pytest.mark.parametrize("m", [3, 40, 410])
def test_two_streams_and_replays(tmp_path, m):
    case = Case(m, 2000, 4096, 64)
    runner, x, out = packaged(tmp_path, case)
    side = torch.cuda.Stream()
    for _ in range(3):
        side.wait_stream(torch.cuda.current_stream())
        runner.run(x, out, stream=side)
        torch.cuda.current_stream().wait_stream(side)
        runner.run(x, out)
    case.check(out["y"].cpu())


@pytest.mark.parametrize("name", ["x", "codes", "scales"])
@pytest.mark.parametrize("m", [2, 40, 410])
def test_a_tensor_off_its_boundary_is_reported(tmp_path, name, m):
    case = Case(m, 64, 128)
    runner, x, out = packaged(tmp_path, case)
    if m > 400 and name == "x":
        return       # `gemm` takes the tokens there, which says nothing of them
    flat = torch.zeros(x[name].numel() + 8, dtype=x[name].dtype, device="cuda")
    x[name] = flat[1:1 + x[name].numel()].view(x[name].shape)
    runner.run(x, out)
    assert int(out["status"].cpu()) == 0x600
