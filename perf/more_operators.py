"""What the operators of decoding in fewer bytes are measured on: one pass is one recipe of a single operator.

Operators (``op``):

* ``append``     rotates the queries and keys of the step's new tokens by their positions, writes the queries out, and keys and values in
                 8 bits, with a power of two for each token and head, into the pages of an E4M3 cache;
* ``read``       brings the pages of a batch back as bf16;
* ``attention``  causal attention over the pages of an E4M3 cache, over everything or a sliding window with a few first tokens that stay
                 visible; single tokens, chunks of prompts;
* ``prefix``     attention of a batch whose sequences share a long prefix, held once in the same cache;
* ``linear``     a product with 4-bit weights that have a scale for each group along K.

A cache case says how many sequences there are, how many tokens each brings (``new_low`` .. ``new_high``) and how many it holds already
(``held_low`` .. ``held_high``); both are spread over their logarithm from ``lengths`` as a seed, so that they belong to the case.
Heads and widths are those of the repository's decoder configurations (16 | 2 and 28 | 4 heads of 128, 8 | 4 of the action expert) and
generic 64-wide ones, matrices those of its 2048- and 3584-wide decoders.

Cache layout: pools [pages, kv_heads, page, head_dim] of E4M3 codes, scales [pages, kv_heads, page] of bf16.  The 16-byte chunk c of
token t lies at position c ^ (t & 7) of its row where rows have eight chunks, at c ^ ((t >> 1) & 3) where they have four.

Weight layout: codes [N / 16, K / 64, 32, 4] of 32-bit words, scales [N / 16, K / group, 8, 2] of bf16, N rounded up to 16 rows.  The
four bits from 4 p of word j of lane 4 g + t are the code of row g + 8 (p & 1), column 32 (j >> 1) + 8 t + 4 (j & 1) + 2 ((p & 2) >> 1) + (p >> 2)
of the tile; a weight is (code - 8) times its row's and group's scale; scale [g, h] belongs to row g + 8 h.
"""
from __future__ import annotations

import math
import random
from collections import OrderedDict

import torch

own = False

THETA = 1e6
SECTIONS = {64: (8, 12, 12), 128: (16, 24, 24)}      # rotary pairs of the time, height and width axes
MAX_LOADED = 24                                      # recipes kept loaded, as a serving process keeps them
GROUPS = (32, 64, 128)


def _cached(name: str, op: str, seqs: int, heads: tuple[int, int, int], page: int, new: tuple[int, int], held: tuple[int, int], *,
            window: int = 0, sinks: int = 0, axes: int = 0, prefix: int = 0, lengths: int = 1) -> dict:
    case = {"op": op, "seqs": seqs, "q_heads": heads[0], "kv_heads": heads[1], "head_dim": heads[2], "page": page,
            "new_low": new[0], "new_high": new[1], "held_low": held[0], "held_high": held[1], "window": window,
            "sinks": sinks, "axes": axes, "prefix": prefix, "lengths": lengths}
    return {"name": name, **case} if name else case


def _linear(name: str, rows: int, out: int, k: int, group: int, bias: bool = False, residual: bool = False) -> dict:
    case = {"op": "linear", "rows": rows, "out": out, "k": k, "group": group, "bias": bias, "residual": residual}
    return {"name": name, **case} if name else case


SMALL, WIDE, EXPERT = (16, 2, 128), (28, 4, 128), (8, 4, 128)
NARROW = (16, 4, 64)


def listed() -> list[dict]:
    return [
        # one request, one token: the latency of a decoding step's append
        _cached("append_e4m3_1tok", "append", 1, SMALL, 64, (1, 1), (300, 300)),
        # a mixed step of a busy server: single tokens beside chunks of prompts, small pages, positions of their own
        _cached("append_e4m3_mixed", "append", 24, WIDE, 16, (1, 1024), (1, 8192), axes=1, lengths=3),
        # what a few requests hold, some of it hidden behind a window, narrow heads
        _cached("read_window", "read", 6, NARROW, 32, (32, 1024), (1, 8192), window=1024, sinks=4, lengths=6),
        # the whole cache of a batch of long requests, as it leaves for a layer that computes in bf16
        _cached("read_long", "read", 24, WIDE, 64, (1, 1), (2000, 16000), lengths=5),
        # one request, one token, some 1500 keys: latency of a decoding step
        _cached("decode_e4m3_1", "attention", 1, SMALL, 64, (1, 1), (1499, 1499)),
        # a large decoding batch over long contexts: the cache is read at the rate of memory
        _cached("decode_e4m3_long", "attention", 64, WIDE, 64, (1, 1), (2000, 32000), lengths=5),
        # chunks of prompts of unequal length over what their requests hold already
        _cached("chunks_e4m3_mixed", "attention", 6, WIDE, 32, (32, 1024), (1, 8192), lengths=6),
        # a batch behind one long instruction
        _cached("prefix_e4m3_long", "prefix", 64, WIDE, 64, (1, 1), (1, 1024), prefix=16384, lengths=8),
        # the Q | K | V projection of one token
        _linear("w4_qkv_1tok", 1, 2560, 2048, 64, bias=True),
        # the gate | up projection of eight samples, 7B-wide, large groups
        _linear("w4_gate_up_8tok", 8, 37888, 3584, 128),
        # the down projection of a batch of drafts, long K, small groups
        _linear("w4_down_48tok", 48, 2048, 11008, 32, residual=True),
        # the gate | up projection of the 288-token prompt
        _linear("w4_gate_up_288", 288, 22016, 2048, 64),
    ]


def _log(rng, low: int, high: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng) -> dict:
    """Sizes over the ranges of the listed cases, no larger in all than the largest of them."""
    while True:
        op = rng.choice(("append", "read", "attention", "attention", "prefix", "linear", "linear"))
        if op == "linear":
            k = 64 * _log(rng, 4, 296)
            group = rng.choice([g for g in GROUPS if k % g == 0])
            case = _linear("", rng.choice((1, _log(rng, 1, 512))), _log(rng, 200, 38000), k, group, rng.choice((False, True)), rng.choice((False, True)))
            if case["out"] * k <= 1.4e8 and work(case)["flops"] <= 2.6e10:
                return case
            continue
        heads = rng.choice((SMALL, WIDE, EXPERT, NARROW))
        page, seed = rng.choice((16, 32, 64, 128)), rng.randrange(1 << 30)
        window = rng.choice((0, _log(rng, 16, 4096)))
        sinks = rng.choice((0, rng.randint(1, 130))) if window else 0
        if op == "append":
            high = _log(rng, 1, 2048)
            case = _cached("", op, _log(rng, 1, 48), heads, page, (rng.choice((1, high)), high), (1, _log(rng, 1, 8192)),
                           axes=rng.choice((0, 1, 3)), lengths=seed)
        elif op == "read":
            high = rng.choice((1, _log(rng, 1, 1024)))
            case = _cached("", op, _log(rng, 1, 48), heads, page, (1, high), (1, _log(rng, 16, 16000)), window=window, sinks=sinks, lengths=seed)
        elif op == "attention":
            high = rng.choice((1, rng.randint(2, 6), _log(rng, 16, 4096)))
            case = _cached("", op, _log(rng, 1, 64 if high < 16 else 8), heads, page, (rng.choice((1, high)), high),
                           (1, _log(rng, 16, 32000 if high < 16 else 8192)), window=window, sinks=sinks, lengths=seed)
        else:
            high = rng.choice((1, rng.randint(2, 8)))
            case = _cached("", op, _log(rng, 2, 96), heads, page, (1, high), (1, _log(rng, 1, 2048)), prefix=_log(rng, 64, 32000),
                           lengths=seed)
        s, w = _sizes(case), work(case)
        if w["bytes"] <= 6e8 and w["flops"] <= 2.0e11 and s["rows"] <= 9000 and (op in ("append", "read") or s["padded_scores"] <= 1.8e9):
            return case


# ---- lengths of a cache case ------------------------------------------------------------------------------

def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """(new tokens, tokens held once they are in) of every sequence."""
    rng = random.Random(case["lengths"])
    new = [_log(rng, case["new_low"], case["new_high"]) for _ in range(case["seqs"])]
    held = [0 if case["held_high"] == 0 else _log(rng, case["held_low"], case["held_high"]) for _ in range(case["seqs"])]
    return new, [n + h for n, h in zip(new, held)]


def _sizes(case: dict) -> dict:
    new, total = _lengths(case)
    pages = [-(-t // case["page"]) for t in total]
    prefix_pages = -(-case["prefix"] // case["page"])
    width = -(-max(total) // case["page"])
    return {"rows": sum(new), "longest": max(new), "width": width, "pages": sum(pages) + prefix_pages + 3,
            "prefix_pages": prefix_pages,
            "padded_scores": case["seqs"] * case["q_heads"] * max(new) * (width * case["page"] + case["prefix"])}


def _hidden(case: dict, new: int, total: int) -> tuple[int, int]:
    """Keys [first, last) that no row of a sequence sees."""
    start = max(0, total - new - case["window"] + 1) if case["window"] else 0
    return min(case["sinks"], start), start


def _read_tokens(case: dict, new: int, total: int) -> int:
    """Tokens of the pages that some row of a sequence sees a token of."""
    first, last = _hidden(case, new, total)
    gone = max(0, last // case["page"] - -(-first // case["page"]))
    return total - gone * case["page"]


def _visible(case: dict, new: int, total: int) -> tuple[int, int]:
    """(pairs of a row and a key that it sees, keys that any row sees) of one sequence."""
    window, sinks = case["window"] or total, case["sinks"]
    pairs = sum(min(p + 1, window) + min(sinks, max(0, p + 1 - window)) for p in range(total - new, total))
    first, last = _hidden(case, new, total)
    return pairs, total - (last - first)


def work(case: dict) -> dict:
    """Bytes: inputs and outputs once, of a cache what any row sees (codes and scales), page numbers and lengths.  Flops: products of
    attention over visible pairs, six operations a rotated pair, products of a matrix."""
    if case["op"] == "linear":
        m, n, k = case["rows"], case["out"], case["k"]
        return {"bytes": n * k // 2 + 2 * n * k // case["group"] + 2 * m * k + 2 * m * n * (2 if case["residual"] else 1) + 2 * n * case["bias"],
                "flops": 2 * m * n * k}
    new, total = _lengths(case)
    heads, kv, d, rows = case["q_heads"], case["kv_heads"], case["head_dim"], sum(new)
    if case["op"] == "append":
        return {"bytes": 4 * rows * heads * d + 2 * rows * kv * (3 * d + 2) + 4 * rows * case["axes"] + 4 * (rows + 2 * len(new) + 1),
                "flops": 3 * rows * (heads + kv) * d}
    tables = 4 * (sum(-(-t // case["page"]) for t in total) + 2 * len(new) + 1)
    if case["op"] == "read":
        tokens = sum(_read_tokens(case, n, t) for n, t in zip(new, total))
        return {"bytes": 2 * tokens * kv * (3 * d + 2) + tables, "flops": 2 * tokens * kv * d}
    seen = [_visible(case, n, t) for n, t in zip(new, total)]
    pairs, keys = sum(p for p, _ in seen) + rows * case["prefix"], sum(k for _, k in seen) + case["prefix"]
    return {"bytes": 4 * rows * heads * d + 2 * keys * kv * (d + 2) + tables, "flops": 4 * heads * d * pairs}


# ---- a request ------------------------------------------------------------------------------------------

_loaded: OrderedDict = OrderedDict()


def _runner(case: dict):
    """The loaded recipe of a case.  It holds sizes alone: what a serving process compiles once for a batch shape."""
    import tempfile
    from pathlib import Path

    from aginfer_b200 import runtime as rt
    from aginfer_b200.recipes import RecipeBuilder
    from aginfer_b200.recipes.package import build_aim, describe
    from aginfer_b200.runner import Runner

    key = tuple(v for k, v in case.items() if k not in ("name", "lengths", "new_low", "new_high", "held_low", "held_high"))
    if case["op"] != "linear":
        s = _sizes(case)
        key += (s["rows"], s["longest"], s["width"], s["pages"])
    if key in _loaded:
        _loaded.move_to_end(key)
        return _loaded[key]
    weights = {"unused.pad": torch.zeros(8, dtype=torch.bfloat16)}
    r = RecipeBuilder(describe(weights))
    (_linear_recipe if case["op"] == "linear" else _cache_recipe)(r, case)
    while len(_loaded) >= MAX_LOADED:
        _loaded.popitem(last=False)
    with tempfile.TemporaryDirectory(prefix="agi_perf_") as tmp:
        _loaded[key] = Runner(build_aim(Path(tmp), weights, r), flags=rt.PROGRAMMATIC_LAUNCH)
    return _loaded[key]


def _linear_recipe(r, case: dict) -> None:
    from aginfer_b200.recipes import Tensor, io
    m, n, k, group = case["rows"], case["out"], case["k"], case["group"]
    tiles = -(-n // 16)
    extra = ([io("bias", "BF16", [n])] if case["bias"] else []) + ([io("residual", "BF16", [m, n])] if case["residual"] else [])
    r.begin_profile("default", [io("x", "BF16", [m, k]), io("codes", "I32", [tiles, k // 64, 32, 4]), io("scales", "BF16", [tiles, k // group, 8, 2]), *extra],
                    [io("y", "BF16", [m, n])])
    r.gemm_w4(Tensor("x"), Tensor("codes"), Tensor("scales"), Tensor("y"), m, n, k, group=group, bias=Tensor("bias") if case["bias"] else None,
              residual=Tensor("residual") if case["residual"] else None)


def _cache_recipe(r, case: dict) -> None:
    from aginfer_b200.recipes import PagedCache, Tensor, io
    s, op = _sizes(case), case["op"]
    heads, kv, d, page, rows, seqs = (case["q_heads"], case["kv_heads"], case["head_dim"], case["page"], s["rows"], case["seqs"])
    batch = [io("starts", "I32", [seqs + 1]), io("lengths", "I32", [seqs]), io("table", "I32", [seqs, s["width"]])]
    pools = [io("k_cache", "F8_E4M3", [s["pages"], kv, page, d]), io("v_cache", "F8_E4M3", [s["pages"], kv, page, d]),
             io("k_scale", "BF16", [s["pages"], kv, page]), io("v_scale", "BF16", [s["pages"], kv, page])]
    shape = dict(sequences=seqs, page=page, pages_per_sequence=s["width"], kv_heads=kv, head_dim=d, lengths=Tensor("lengths"), starts=Tensor("starts"))
    cache = PagedCache(k=Tensor("k_cache"), v=Tensor("v_cache"), k_scale=Tensor("k_scale"), v_scale=Tensor("v_scale"), table=Tensor("table"),
                       pages=s["pages"], **shape)
    if op == "append":
        positions = [io("positions", "I32", [rows] if case["axes"] == 1 else [3, rows])] if case["axes"] else []
        r.begin_profile("default", [io("qkv", "BF16", [rows, (heads + 2 * kv) * d]), *batch, *positions],
                        [io("q", "BF16", [rows, heads * d]), *pools])
        r.kv_append(Tensor("qkv"), Tensor("q"), cache, rows=rows, q_heads=heads, theta=THETA,
                    positions=Tensor("positions") if positions else None, sections=SECTIONS[d] if case["axes"] == 3 else None)
    elif op == "read":
        out = [seqs * s["width"], kv, d // 64, page, 64]
        r.begin_profile("default", [*pools, *batch], [io("k", "BF16", out), io("v", "BF16", out), io("pages", "I32", [seqs, s["width"]])])
        r.kv_read(cache, PagedCache(k=Tensor("k"), v=Tensor("v"), table=Tensor("pages"), pages=out[0], **shape), rows=rows,
                  window=case["window"], sinks=case["sinks"])
    else:
        shared = [io("prefix_table", "I32", [s["prefix_pages"]]), io("prefix_length", "I32", [1])] if op == "prefix" else []
        r.begin_profile("default", [io("q", "BF16", [rows, heads * d]), *pools, *batch, *shared], [io("o", "BF16", [rows, heads * d])])
        if op == "prefix":
            r.prefix_attention(Tensor("q"), Tensor("o"), cache, Tensor("prefix_table"), Tensor("prefix_length"),
                               prefix_pages=s["prefix_pages"], rows=rows, longest=s["longest"], q_heads=heads)
        else:
            r.paged_attention(Tensor("q"), Tensor("o"), cache, rows=rows, longest=s["longest"], q_heads=heads,
                              window=case["window"], sinks=case["sinks"])


def _places(tokens: int, d: int, device="cuda") -> torch.Tensor:
    """[tokens, d]: where column j of a token lies in its stored row."""
    column, token = torch.arange(d, device=device)[None, :], torch.arange(tokens, device=device)[:, None]
    turn = token & 7 if d == 128 else (token >> 1) & 3
    return ((column // 16) ^ turn) * 16 + column % 16


def _quantised(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(E4M3 codes, scales) of [..., d]: the least power of two that brings a row to 448 or less, one for a row of zeros."""
    peak = x.abs().amax(dim=-1)
    fraction, exponent = torch.frexp(peak)                                   # peak = fraction 2^exponent, fraction in [0.5, 1)
    exponent = torch.where(peak > 0, exponent - 9 + (fraction > 0.875), 0)   # 448 = 0.875 * 2^9
    scale = torch.ldexp(torch.ones_like(peak), exponent)
    return (x / scale[..., None]).to(torch.float8_e4m3fn), scale.to(torch.bfloat16)


def _pool(values: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes as bytes, scales) of [pages, kv heads, page, d], stored."""
    codes, scale = _quantised(values)
    page, d = values.shape[-2:]
    stored = codes.view(torch.uint8).gather(-1, _places(page, d).expand(values.shape))       # exchanging chunks is its own inverse
    return stored, scale


def _cache_inputs(case: dict, seed: int) -> dict:
    """Tensors of a request: a pool whose pages lie in no order, projections ~ N(0, 1) with channels of unequal size, as
    keys have them (scores then spread with a standard deviation of 1.5 or so)."""
    new, total = _lengths(case)
    s = _sizes(case)
    heads, kv, d, page, rows, seqs = (case["q_heads"], case["kv_heads"], case["head_dim"], case["page"], s["rows"], case["seqs"])
    g = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    channel = torch.exp(0.4 * randn(kv, 1, d))
    x = {}
    x["k_cache"], x["k_scale"] = _pool(randn(s["pages"], kv, page, d) * channel)
    x["v_cache"], x["v_scale"] = _pool(randn(s["pages"], kv, page, d))
    order = torch.randperm(s["pages"], generator=g, device="cuda").to(torch.int32).cpu()
    table, at = torch.zeros(seqs, s["width"], dtype=torch.int32), s["prefix_pages"]
    for b, t in enumerate(total):
        n = -(-t // page)
        table[b, :n] = order[at:at + n]
        at += n
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    x["table"] = table.cuda()
    x["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    x["lengths"] = torch.tensor(total, dtype=torch.int32, device="cuda")
    if case["op"] == "append":
        x["qkv"] = randn(rows, (heads + 2 * kv) * d).to(torch.bfloat16)
        if case["axes"]:
            index = torch.cat([torch.arange(t - n, t, dtype=torch.int32) for n, t in zip(new, total)])
            if case["axes"] == 1:      # an image took fewer positions than tokens
                x["positions"] = (index - index // 4).cuda()
            else:                      # patches of a 16-wide grid, every fifth token text behind them
                text = index % 5 == 4
                x["positions"] = torch.stack([torch.where(text, index, index // 256), torch.where(text, index, index // 16),
                                              torch.where(text, index, index % 16)]).to(torch.int32).contiguous().cuda()
    elif case["op"] != "read":
        x["q"] = (1.25 * randn(rows, heads * d)).to(torch.bfloat16)
        if case["op"] == "prefix":
            x["prefix_table"] = order[:s["prefix_pages"]].clone().cuda()
            x["prefix_length"] = torch.tensor([case["prefix"]], dtype=torch.int32, device="cuda")
    return x


def _linear_inputs(case: dict, seed: int) -> dict:
    """Activations ~ N(0, 1), codes as a normal weight has them, scales that make outputs of size one."""
    m, n, k, group = case["rows"], case["out"], case["k"], case["group"]
    tiles = -(-n // 16)
    g = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    codes = (2.7 * randn(8, tiles, k // 64, 32, 4)).round_().clamp_(-8, 7).to(torch.int32) + 8
    words = torch.zeros_like(codes[0])
    for p in range(8):
        words |= codes[p] << (4 * p)
    x = {"x": randn(m, k).to(torch.bfloat16), "codes": words,
         "scales": (torch.exp(0.3 * randn(tiles, k // group, 8, 2)) * (0.35 * k ** -0.5)).to(torch.bfloat16)}
    if case["bias"]:
        x["bias"] = randn(n).to(torch.bfloat16)
    if case["residual"]:
        x["residual"] = randn(m, n).to(torch.bfloat16)
    return x


def _inputs(case: dict, seed: int) -> dict:
    return _linear_inputs(case, seed) if case["op"] == "linear" else _cache_inputs(case, seed)


def prepare(case: dict, seed: int) -> dict:
    x = _inputs(case, seed)
    state = {"case": case, "x": x}
    empty = lambda *shape: torch.empty(*shape, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    if case["op"] == "linear":
        state["out"] = {"y": empty(case["rows"], case["out"])}
    else:
        s = state["sizes"] = _sizes(case)
        if case["op"] == "append":
            state["out"] = {"q": empty(s["rows"], case["q_heads"] * case["head_dim"]),
                            **{n: x.pop(n) for n in ("k_cache", "v_cache", "k_scale", "v_scale")}}
        elif case["op"] == "read":
            shape = (case["seqs"] * s["width"], case["kv_heads"], case["head_dim"] // 64, case["page"], 64)
            state["out"] = {"k": empty(shape).zero_(), "v": empty(shape).zero_(),
                            "pages": torch.zeros(case["seqs"], s["width"], dtype=torch.int32, device="cuda")}
        else:
            state["out"] = {"o": torch.empty_like(x["q"])}
    if own:
        state["runner"] = _runner(case)
    return state


def run(state: dict) -> dict:
    if own:
        out = state["runner"].run(state["x"], state["out"])
    else:
        out = {"append": _plain_append, "read": _plain_read, "linear": _plain_linear}.get(state["case"]["op"], _plain_attention)(state)
    if state["case"]["op"] == "append":
        out = {n: t.view(torch.float8_e4m3fn) if t.dtype == torch.uint8 else t for n, t in out.items()}
    return out


# ---- the plain form: elementary operations in 32 bits (angles in 64) ---------------------------------------

def _plain_sequences(state: dict) -> tuple[torch.Tensor, torch.Tensor]:
    """(sequence, cache index) of every row."""
    starts, lengths = state["x"]["starts"].long(), state["x"]["lengths"].long()
    row = torch.arange(state["sizes"]["rows"], device="cuda")
    seq = torch.searchsorted(starts, row, right=True) - 1
    return seq, lengths[seq] - (starts[seq + 1] - row)


def _plain_append(state: dict) -> dict:
    case, x, out = state["case"], state["x"], state["out"]
    heads, kv, d, page, rows = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"], state["sizes"]["rows"]
    half = d // 2
    seq, index = _plain_sequences(state)
    frequency = torch.exp2(-math.log2(THETA) * torch.arange(half, device="cuda", dtype=torch.float64) / half)
    if case["axes"] == 3:
        axis = torch.repeat_interleave(torch.arange(3, device="cuda"), torch.tensor(SECTIONS[d], device="cuda"), output_size=half)
        position = x["positions"].double()[axis].t()
    else:
        position = (x["positions"] if case["axes"] else index).double()[:, None]
    angle = position * frequency
    c, s = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    qkv = x["qkv"].view(rows, heads + 2 * kv, d).float()
    lo, hi = qkv[:, :heads + kv, :half], qkv[:, :heads + kv, half:]
    turned = torch.cat([lo * c - hi * s, hi * c + lo * s], dim=2)
    out["q"].copy_(turned[:, :heads].reshape(rows, heads * d))
    slot, token = x["table"].long()[seq, index // page], index % page
    places = _places(page, d)[token][:, None].expand(rows, kv, d)
    for name, values in (("k", turned[:, heads:]), ("v", qkv[:, heads + kv:])):
        codes, scale = _quantised(values)
        out[name + "_cache"][slot, :, token] = codes.view(torch.uint8).gather(2, places)
        out[name + "_scale"][slot, :, token] = scale
    return out


def _plain_pages(x: dict, which: str, pages: torch.Tensor) -> torch.Tensor:
    """[..., n, kv heads, page, head_dim] in 32 bits of the pages numbered ``pages`` [..., n]."""
    codes, scale = x[which + "_cache"][pages.long()], x[which + "_scale"][pages.long()]
    at = _places(*codes.shape[-2:]).expand(codes.shape)
    return codes.gather(-1, at).view(torch.float8_e4m3fn).float() * scale.float()[..., None]


def _plain_tokens(x: dict, which: str, pages: torch.Tensor) -> torch.Tensor:
    """[..., tokens, kv heads, head_dim] of the same."""
    t = _plain_pages(x, which, pages).transpose(-3, -2)
    return t.reshape(*pages.shape[:-1], -1, *t.shape[-2:])


def _plain_read(state: dict) -> dict:
    case, x, out = state["case"], state["x"], state["out"]
    kv, d, page, seqs, width = case["kv_heads"], case["head_dim"], case["page"], case["seqs"], state["sizes"]["width"]
    starts, lengths = x["starts"].long(), x["lengths"].long()[:, None]
    first = lengths - (starts[1:] - starts[:-1])[:, None]
    from_token = (first - case["window"] + 1).clamp_min(0) if case["window"] else torch.zeros_like(first)
    token = torch.arange(width * page, device="cuda")[None, :]
    held = token < lengths
    seen = held & ((token >= from_token) | (token < case["sinks"]))
    pages_seen = seen.view(seqs, width, page).any(dim=2)
    live = (held.view(seqs, width, page) & pages_seen[:, :, None]).view(seqs * width, 1, 1, page, 1)
    column, row = torch.arange(64, device="cuda")[None, :], torch.arange(page, device="cuda")[:, None]
    at = (((column // 8) ^ (row & 7)) * 8 + column % 8).expand(seqs * width, kv, d // 64, page, 64)
    for which in "kv":
        t = _plain_pages(x, which, x["table"]).view(seqs * width, kv, page, d // 64, 64).transpose(2, 3)
        out[which].copy_(torch.where(live, t.gather(-1, at), out[which].float()))
    number = torch.arange(seqs * width, dtype=torch.int32, device="cuda").view(seqs, width)
    out["pages"].copy_(torch.where(pages_seen, number, out["pages"]))
    return out


def _plain_attention(state: dict) -> dict:
    case, x, s = state["case"], state["x"], state["sizes"]
    heads, kv, d, seqs, rows = case["q_heads"], case["kv_heads"], case["head_dim"], case["seqs"], s["rows"]
    group, most = heads // kv, s["longest"]
    seq, index = _plain_sequences(state)
    place = torch.arange(rows, device="cuda") - x["starts"].long()[seq]
    q = torch.zeros(seqs, most, kv, group, d, device="cuda")
    q[seq, place] = x["q"].view(rows, kv, group, d).float() * d ** -0.5
    q = q.permute(0, 2, 3, 1, 4).reshape(seqs, kv, group * most, d)
    k, v = (_plain_tokens(x, which, x["table"]).permute(0, 2, 1, 3) for which in "kv")               # [seqs, kv, keys, d]
    score = (q @ k.transpose(2, 3)).view(seqs, kv, group, most, -1)
    p = torch.full((seqs, most), -1, device="cuda")
    p[seq, place] = index
    key = torch.arange(score.shape[-1], device="cuda")
    seen = key <= p[:, :, None]
    if case["window"]:
        seen &= (p[:, :, None] - key < case["window"]) | (key < case["sinks"])
    score.masked_fill_(~seen[:, None, None], -math.inf)
    if case["op"] == "prefix":
        pk, pv = (_plain_tokens(x, which, x["prefix_table"])[:case["prefix"]].permute(1, 0, 2) for which in "kv")
        score = torch.cat([score, (q @ pk.transpose(1, 2)).view(seqs, kv, group, most, -1)], dim=-1)
    peak = score.amax(dim=-1, keepdim=True)
    weight = torch.exp(score.sub_(torch.where(peak > -math.inf, peak, 0.0)))
    total = weight.sum(dim=-1, keepdim=True)
    weight = weight.view(seqs, kv, group * most, -1)
    o = weight[..., :key.numel()] @ v
    if case["op"] == "prefix":
        o += weight[..., key.numel():] @ pv
    o = o.view(seqs, kv, group, most, d) / torch.where(total > 0, total, 1.0)
    state["out"]["o"].copy_(o.permute(0, 3, 1, 2, 4)[seq, place].reshape(rows, heads * d))
    return state["out"]


def _plain_linear(state: dict) -> dict:
    case, x = state["case"], state["x"]
    n, k, group = case["out"], case["k"], case["group"]
    tiles = -(-n // 16)
    shift = 4 * torch.arange(8, device="cuda", dtype=torch.int32)
    code = ((x["codes"][..., None] >> shift) & 15).view(tiles, k // 64, 8, 4, 2, 2, 2, 2, 2)
    # axes: tile, block, g, t, half of the block, quarter of a lane's eight, column's lowest bit, its next one, row half
    w = code.permute(0, 8, 2, 1, 4, 3, 5, 7, 6).reshape(tiles * 16, k // group, group).float() - 8
    w = w * x["scales"].float().permute(0, 3, 2, 1).reshape(tiles * 16, k // group, 1)
    y = x["x"].float() @ w.view(tiles * 16, k)[:n].t()
    if case["bias"]:
        y += x["bias"].float()
    if case["residual"]:
        y += x["residual"].float()
    state["out"]["y"].copy_(y)
    return state["out"]


# ---- the definition in 64 bits ------------------------------------------------------------------------------

def _exact_scale(peak: torch.Tensor) -> torch.Tensor:
    tight = torch.exp2(torch.ceil(torch.log2(peak / 448)))
    tight = torch.where(tight * 224 >= peak, tight / 2, tight)          # where the logarithm was rounded up to the next number
    tight = torch.where(tight * 448 < peak, tight * 2, tight)
    return torch.where(peak > 0, tight, 1.0)


def _exact_tokens(x: dict, which: str, pages: list[int], count: int) -> torch.Tensor:
    """The first ``count`` tokens held in ``pages``, [tokens, kv heads, head_dim] in 64 bits."""
    codes = x[which + "_cache"][pages].view(torch.float8_e4m3fn)
    n, kv, page, d = codes.shape
    tokens = codes.to(torch.float64).permute(0, 2, 1, 3).reshape(n * page, kv, d // 16, 16)[:count]
    scale = x[which + "_scale"][pages].double().permute(0, 2, 1).reshape(n * page, kv)[:count]
    rows = torch.empty_like(tokens)
    period = 8
    for j in range(period):                       # tokens j, j + 8, ... keep their chunks in the same order
        for c in range(d // 16):
            rows[j::period, :, c] = tokens[j::period, :, c ^ (j if d == 128 else j // 2)]
    return rows.reshape(-1, kv, d) * scale[:, :, None]


def _exact_append(case: dict, x: dict) -> dict:
    heads, kv, d, page = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"]
    half = d // 2
    new, total = _lengths(case)
    out = {n: (x[n].view(torch.float8_e4m3fn) if "cache" in n else x[n]).to(torch.float64) for n in ("k_cache", "v_cache", "k_scale", "v_scale")}
    table, q_all, row = x["table"].tolist(), [], 0
    frequency = THETA ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
    for b, (n, t) in enumerate(zip(new, total)):
        part = x["qkv"][row:row + n].double().view(n, heads + 2 * kv, d)
        if case["axes"] == 3:
            s0, s1, s2 = SECTIONS[d]
            at = x["positions"][:, row:row + n].double()
            position = torch.cat([at[0][:, None].expand(n, s0), at[1][:, None].expand(n, s1), at[2][:, None].expand(n, s2)], dim=1)
        elif case["axes"] == 1:
            position = x["positions"][row:row + n].double()[:, None]
        else:
            position = torch.arange(t - n, t, dtype=torch.float64, device="cuda")[:, None]
        wave = torch.polar(torch.ones_like(position * frequency), position * frequency)[:, None]
        pairs = torch.complex(part[:, :heads + kv, :half].contiguous(), part[:, :heads + kv, half:].contiguous()) * wave
        turned = torch.cat([pairs.real, pairs.imag], dim=2)
        q_all.append(turned[:, :heads].reshape(n, heads * d))
        index = range(t - n, t)
        for name, values in (("k", turned[:, heads:]), ("v", part[:, heads + kv:])):
            scale = _exact_scale(values.abs().amax(dim=2))
            codes = (values / scale[:, :, None]).view(n, kv, d // 16, 16)
            for j in range(8):
                mine = [i for i in range(n) if index[i] % 8 == j]
                if not mine:
                    continue
                pages, tokens = [table[b][index[i] // page] for i in mine], [index[i] % page for i in mine]
                out[name + "_scale"][pages, :, tokens] = scale[mine]
                for c in range(d // 16):
                    to = 16 * (c ^ (j if d == 128 else j // 2))
                    out[name + "_cache"][pages, :, tokens, to:to + 16] = codes[mine][:, :, c]
        row += n
    return {"q": torch.cat(q_all), **out}


def _exact_read(case: dict, x: dict) -> dict:
    kv, d, page, seqs = case["kv_heads"], case["head_dim"], case["page"], case["seqs"]
    new, total = _lengths(case)
    width, table = _sizes(case)["width"], x["table"].tolist()
    out = {n: torch.zeros(seqs * width, kv, d // 64, page, 64, dtype=torch.float64, device="cuda") for n in "kv"}
    numbers = torch.zeros(seqs, width, dtype=torch.int32)
    for b, (n, t) in enumerate(zip(new, total)):
        first, last = _hidden(case, n, t)
        count = -(-t // page)
        seen = [i for i in range(count) if not (i * page >= first and min((i + 1) * page, t) <= last)]
        numbers[b, seen] = torch.tensor([b * width + i for i in seen], dtype=torch.int32)
        for which in "kv":
            tokens = torch.zeros(count * page, kv, d, dtype=torch.float64, device="cuda")
            tokens[:t] = _exact_tokens(x, which, table[b][:count], t)
            pages = tokens.view(count, page, kv, d // 64, 8, 8).permute(0, 2, 3, 1, 4, 5)
            stored = torch.empty_like(pages)
            for j in range(8):
                for c in range(8):
                    stored[:, :, :, j::8, c ^ j] = pages[:, :, :, j::8, c]
            out[which][[b * width + i for i in seen]] = stored.reshape(count, kv, d // 64, page, 64)[seen]
    return {**out, "pages": numbers.cuda()}


def _exact_attention(case: dict, x: dict) -> dict:
    heads, kv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    group, row, out = heads // kv, 0, []
    new, total = _lengths(case)
    table = x["table"].tolist()
    shared = None
    if case["op"] == "prefix":
        pages = x["prefix_table"].tolist()
        shared = [_exact_tokens(x, which, pages, case["prefix"]) for which in "kv"]
    for b, (n, t) in enumerate(zip(new, total)):
        pages = table[b][:-(-t // case["page"])]
        k, v = (_exact_tokens(x, which, pages, t) for which in "kv")
        q = x["q"][row:row + n].double().view(n, kv, group, d)
        for first in range(0, n, 512):
            part = q[first:first + 512]
            p = torch.arange(t - n + first, t - n + first + part.shape[0], device="cuda")[:, None]
            j = torch.arange(t, device="cuda")[None, :]
            hidden = j > p
            if case["window"]:
                hidden = hidden | ((p - j >= case["window"]) & (j >= case["sinks"]))
            answer = torch.empty_like(part)
            for h in range(kv):
                score = torch.einsum("ngd,kd->gnk", part[:, h], k[:, h]) / math.sqrt(d)
                score = score.masked_fill(hidden, -math.inf)
                values = v[:, h]
                if shared is not None:
                    score = torch.cat([score, torch.einsum("ngd,kd->gnk", part[:, h], shared[0][:, h]) / math.sqrt(d)], dim=2)
                    values = torch.cat([values, shared[1][:, h]])
                answer[:, h] = torch.einsum("gnk,kd->ngd", torch.softmax(score, dim=2), values)
            out.append(answer.reshape(-1, heads * d))
        row += n
    return {"o": torch.cat(out)}


def _exact_linear(case: dict, x: dict) -> dict:
    n, k, group = case["out"], case["k"], case["group"]
    tiles = -(-n // 16)
    w = torch.empty(tiles, 16, k // 64, 64, dtype=torch.float64, device="cuda")
    for p in range(8):
        code = torch.bitwise_and(x["codes"].div(1 << (4 * p), rounding_mode="floor"), 15).double().view(tiles, k // 64, 8, 4, 4)      # [.., g, t, j]
        for t in range(4):
            for j in range(4):
                column = 32 * (j // 2) + 8 * t + 4 * (j % 2) + 2 * (p // 2 % 2) + p // 4
                w[:, 8 * (p % 2):8 * (p % 2) + 8, :, column] = code[:, :, :, t, j].transpose(1, 2) - 8.0
    scale = torch.cat([x["scales"][..., 0], x["scales"][..., 1]], dim=2).double()                                                     # [tile, group, row]
    w = (w.view(tiles, 16, k // group, group) * scale.transpose(1, 2)[..., None]).reshape(tiles * 16, k)[:n]
    y = x["x"].double() @ w.t()
    y = y + x["bias"].double() if case["bias"] else y
    return {"y": y + x["residual"].double() if case["residual"] else y}


def exact(case: dict, seed: int):
    x = _inputs(case, seed)
    return {"append": _exact_append, "read": _exact_read, "linear": _exact_linear}.get(case["op"], _exact_attention)(case, x)
