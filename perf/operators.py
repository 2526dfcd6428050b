"""What the paged-cache operators are measured on: one pass is one recipe of a single operator over a batch of sequences.

Operators (``op``):

* ``append``     rotates the queries and keys of the step's new tokens by their positions, writes the queries out and keys and
                 values into the pages of a K/V cache;
* ``attention``  causal attention of those queries over the pages, over everything or over a sliding window with a few first
                 tokens that stay visible; single tokens, chunks of prompts, whole prompts;
* ``prefix``     attention of a batch whose sequences share a long prefix, held once, and go on with tokens of their own.

A case says how many sequences there are, how many tokens each brings (``new_low`` .. ``new_high``) and how many it holds
already (``held_low`` .. ``held_high``); both are spread over their logarithm from ``lengths`` as a seed, so that they belong
to the case.  Heads and widths are those of the repository's decoder configurations (16 | 2 and 28 | 4 heads of 128, 8 | 4
of the action expert) and generic 64-wide ones.
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


def _case(name: str, op: str, seqs: int, heads: tuple[int, int, int], page: int, new: tuple[int, int], held: tuple[int, int], *,
          window: int = 0, sinks: int = 0, axes: int = 0, prefix: int = 0, lengths: int = 1) -> dict:
    case = {"op": op, "seqs": seqs, "q_heads": heads[0], "kv_heads": heads[1], "head_dim": heads[2], "page": page,
            "new_low": new[0], "new_high": new[1], "held_low": held[0], "held_high": held[1], "window": window,
            "sinks": sinks, "axes": axes, "prefix": prefix, "lengths": lengths}
    return {"name": name, **case} if name else case


SMALL, WIDE, EXPERT = (16, 2, 128), (28, 4, 128), (8, 4, 128)
NARROW = (16, 4, 64)


def listed() -> list[dict]:
    return [
        # one request, one token: the latency of a decoding step's append
        _case("append_1tok", "append", 1, SMALL, 64, (1, 1), (300, 300)),
        # the 288-token image-and-text prompt with time, height and width positions
        _case("append_prompt_288", "append", 1, SMALL, 64, (288, 288), (0, 0), axes=3),
        # a mixed step of a busy server: single tokens beside chunks of prompts, small pages
        _case("append_mixed", "append", 24, WIDE, 16, (1, 1024), (1, 8192), axes=1, lengths=3),
        # one request, one token, some 1500 keys: latency of a decoding step
        _case("decode_1", "attention", 1, SMALL, 64, (1, 1), (1499, 1499)),
        # a decoding batch that keeps a window of 1024 keys and the first four, small pages
        _case("decode_window", "attention", 48, WIDE, 16, (1, 1), (200, 16000), window=1024, sinks=4, lengths=4),
        # a large decoding batch over long contexts: the cache is read at the rate of memory
        _case("decode_long", "attention", 64, WIDE, 64, (1, 1), (2000, 32000), lengths=5),
        # the 288-token prompt, causal
        _case("prompt_288", "attention", 1, SMALL, 64, (288, 288), (0, 0)),
        # a long prompt under a window with sinks
        _case("prompt_window_8192", "attention", 1, WIDE, 64, (8192, 8192), (0, 0), window=2048, sinks=4),
        # chunks of prompts of unequal length over what their requests hold already
        _case("chunks_mixed", "attention", 6, WIDE, 32, (32, 1024), (1, 8192), lengths=6),
        # eight samples from one 288-token prompt, a few tokens into their answers
        _case("prefix_8", "prefix", 8, SMALL, 64, (1, 1), (1, 64), prefix=288, lengths=7),
        # a batch behind one long instruction
        _case("prefix_long", "prefix", 64, WIDE, 64, (1, 1), (1, 1024), prefix=16384, lengths=8),
        # several drafted tokens a sequence, narrow heads, small pages
        _case("prefix_drafts", "prefix", 24, NARROW, 16, (2, 8), (1, 500), prefix=4001, lengths=9),
    ]


def _log(rng, low: int, high: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng) -> dict:
    """Sizes over the ranges of the listed cases, no larger in all than the largest of them."""
    while True:
        op = rng.choice(("append", "attention", "attention", "prefix"))
        heads = rng.choice((SMALL, WIDE, EXPERT, NARROW))
        page, seed = rng.choice((16, 32, 64, 128)), rng.randrange(1 << 30)
        if op == "append":
            high = _log(rng, 1, 2048)
            case = _case("", op, _log(rng, 1, 48), heads, page, (rng.choice((1, high)), high), (1, _log(rng, 1, 8192)),
                         axes=rng.choice((0, 1, 3)), lengths=seed)
        elif op == "attention":
            window = rng.choice((0, _log(rng, 16, 4096)))
            sinks = rng.choice((0, rng.randint(1, 130))) if window else 0
            high = rng.choice((1, rng.randint(2, 6), _log(rng, 16, 8192)))
            case = _case("", op, _log(rng, 1, 64 if high < 16 else 8), heads, page, (rng.choice((1, high)), high),
                         (1, _log(rng, 16, 32000 if high < 16 else 8192)), window=window, sinks=sinks, lengths=seed)
        else:
            high = rng.choice((1, rng.randint(2, 8)))
            case = _case("", op, _log(rng, 2, 96), heads, page, (1, high), (1, _log(rng, 1, 2048)), prefix=_log(rng, 64, 32000),
                         lengths=seed)
        s, w = _sizes(case), work(case)
        if w["bytes"] <= 1.2e9 and w["flops"] <= 2.0e11 and s["rows"] <= 9000 and (op == "append" or s["padded_scores"] <= 1.8e9):
            return case


# ---- lengths of a case ----------------------------------------------------------------------------------

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


def _visible(case: dict, new: int, total: int) -> tuple[int, int]:
    """(pairs of a row and a key that it sees, keys that any row sees) of one sequence."""
    window, sinks = case["window"] or total, case["sinks"]
    first = total - new
    pairs = sum(min(p + 1, window) + min(sinks, max(0, p + 1 - window)) for p in range(first, total))
    start = max(0, first - window + 1)
    return pairs, total - start + min(sinks, start)


def work(case: dict) -> dict:
    """Bytes: queries, outputs and every key and value that any row sees, once; page numbers and lengths.  Flops: the two
    products of attention over visible pairs, six operations a rotated pair."""
    new, total = _lengths(case)
    heads, kv, d, rows = case["q_heads"], case["kv_heads"], case["head_dim"], sum(new)
    tables = 4 * (sum(-(-t // case["page"]) for t in total) + 2 * len(new) + 1)
    if case["op"] == "append":
        return {"bytes": 4 * rows * (heads + 2 * kv) * d + 4 * rows * case["axes"] + 4 * (rows + 2 * len(new) + 1),
                "flops": 3 * rows * (heads + kv) * d}
    seen = [_visible(case, n, t) for n, t in zip(new, total)]
    pairs, keys = sum(p for p, _ in seen) + rows * case["prefix"], sum(k for _, k in seen) + case["prefix"]
    return {"bytes": 4 * rows * heads * d + 4 * keys * kv * d + tables, "flops": 4 * heads * d * pairs}


# ---- a request ------------------------------------------------------------------------------------------

_loaded: OrderedDict = OrderedDict()


def _runner(case: dict):
    """The loaded recipe of a case.  It holds sizes alone: what a serving process compiles once for a batch shape."""
    import tempfile
    from pathlib import Path

    from aginfer_b200 import runtime as rt
    from aginfer_b200.recipes import PagedCache, RecipeBuilder, Tensor, io
    from aginfer_b200.recipes.package import build_aim, describe
    from aginfer_b200.runner import Runner

    s, op = _sizes(case), case["op"]
    heads, kv, d, page, rows, seqs = (case["q_heads"], case["kv_heads"], case["head_dim"], case["page"], s["rows"], case["seqs"])
    key = (op, rows, s["longest"], s["width"], s["pages"], *(case[k] for k in ("seqs", "q_heads", "kv_heads", "head_dim", "page", "window",
                                                                               "sinks", "axes", "prefix")))
    if key in _loaded:
        _loaded.move_to_end(key)
        return _loaded[key]
    weights = {"unused.pad": torch.zeros(8, dtype=torch.bfloat16)}
    pool = [s["pages"], kv, d // 64, page, 64]
    batch = [io("starts", "I32", [seqs + 1]), io("lengths", "I32", [seqs]), io("table", "I32", [seqs, s["width"]])]
    pools = [io("k_cache", "BF16", pool), io("v_cache", "BF16", pool)]
    cache = PagedCache(k=Tensor("k_cache"), v=Tensor("v_cache"), table=Tensor("table"), lengths=Tensor("lengths"), starts=Tensor("starts"),
                       sequences=seqs, pages=s["pages"], page=page, pages_per_sequence=s["width"], kv_heads=kv, head_dim=d)
    r = RecipeBuilder(describe(weights))
    if op == "append":
        positions = [io("positions", "I32", [rows] if case["axes"] == 1 else [3, rows])] if case["axes"] else []
        r.begin_profile("default", [io("qkv", "BF16", [rows, (heads + 2 * kv) * d]), *batch, *positions],
                        [io("q", "BF16", [rows, heads * d]), *pools])
        r.kv_append(Tensor("qkv"), Tensor("q"), cache, rows=rows, q_heads=heads, theta=THETA,
                    positions=Tensor("positions") if positions else None, sections=SECTIONS[d] if case["axes"] == 3 else None)
    else:
        shared = [io("prefix_table", "I32", [s["prefix_pages"]]), io("prefix_length", "I32", [1])] if op == "prefix" else []
        r.begin_profile("default", [io("q", "BF16", [rows, heads * d]), *pools, *batch, *shared], [io("o", "BF16", [rows, heads * d])])
        if op == "prefix":
            r.prefix_attention(Tensor("q"), Tensor("o"), cache, Tensor("prefix_table"), Tensor("prefix_length"),
                               prefix_pages=s["prefix_pages"], rows=rows, longest=s["longest"], q_heads=heads)
        else:
            r.paged_attention(Tensor("q"), Tensor("o"), cache, rows=rows, longest=s["longest"], q_heads=heads,
                              window=case["window"], sinks=case["sinks"])
    while len(_loaded) >= MAX_LOADED:
        _loaded.popitem(last=False)
    with tempfile.TemporaryDirectory(prefix="agi_perf_") as tmp:
        _loaded[key] = Runner(build_aim(Path(tmp), weights, r), flags=rt.PROGRAMMATIC_LAUNCH)
    return _loaded[key]


def _inputs(case: dict, seed: int) -> dict:
    """Tensors of a request: a pool whose pages lie in no order, projections ~ N(0, 1) with channels of unequal size, as
    keys have them (scores then spread with a standard deviation of 1.5 or so)."""
    new, total = _lengths(case)
    s = _sizes(case)
    heads, kv, d, page, rows, seqs = (case["q_heads"], case["kv_heads"], case["head_dim"], case["page"], s["rows"], case["seqs"])
    g = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    channel = torch.exp(0.4 * randn(kv, d // 64, 1, 64))
    x = {"k_cache": (randn(s["pages"], kv, d // 64, page, 64) * channel).to(torch.bfloat16),
         "v_cache": randn(s["pages"], kv, d // 64, page, 64).to(torch.bfloat16)}
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
    else:
        x["q"] = (1.25 * randn(rows, heads * d)).to(torch.bfloat16)
        if case["op"] == "prefix":
            x["prefix_table"] = order[:s["prefix_pages"]].clone().cuda()
            x["prefix_length"] = torch.tensor([case["prefix"]], dtype=torch.int32, device="cuda")
    return x


def prepare(case: dict, seed: int) -> dict:
    x = _inputs(case, seed)
    state = {"case": case, "x": x, "sizes": _sizes(case)}
    if case["op"] == "append":
        state["out"] = {"q": torch.empty(state["sizes"]["rows"], case["q_heads"] * case["head_dim"], dtype=torch.bfloat16, device="cuda"),
                        "k_cache": x.pop("k_cache"), "v_cache": x.pop("v_cache")}
    else:
        state["out"] = {"o": torch.empty_like(x["q"])}
    if own:
        state["runner"] = _runner(case)
    return state


def run(state: dict) -> dict:
    if own:
        return state["runner"].run(state["x"], state["out"])
    return _plain_append(state) if state["case"]["op"] == "append" else _plain_attention(state)


# ---- the plain form: elementary operations in 32 bits -----------------------------------------------------

def _columns(page: int, device) -> torch.Tensor:
    """[page, 64]: where column j of a token's 64-column block lies in its stored row (16-byte chunks are swizzled)."""
    column, token = torch.arange(64, device=device)[None, :], torch.arange(page, device=device)[:, None]
    return ((column // 8) ^ (token % 8)) * 8 + column % 8


def _plain_rows(state: dict) -> tuple[torch.Tensor, torch.Tensor]:
    """(sequence, cache index) of every row."""
    starts, lengths = state["x"]["starts"].long(), state["x"]["lengths"].long()
    row = torch.arange(state["sizes"]["rows"], device="cuda")
    seq = torch.searchsorted(starts, row, right=True) - 1
    return seq, lengths[seq] - (starts[seq + 1] - row)


def _plain_append(state: dict) -> dict:
    case, x, out = state["case"], state["x"], state["out"]
    heads, kv, d, page, rows = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"], state["sizes"]["rows"]
    half = d // 2
    seq, index = _plain_rows(state)
    frequency = torch.exp2(-math.log2(THETA) * torch.arange(half, device="cuda", dtype=torch.float32) / half)
    if case["axes"] == 3:
        axis = torch.repeat_interleave(torch.arange(3, device="cuda"), torch.tensor(SECTIONS[d], device="cuda"), output_size=half)
        position = x["positions"].float()[axis].t()
    else:
        position = (x["positions"] if case["axes"] else index).float()[:, None]
    angle = position * frequency
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    qkv = x["qkv"].view(rows, heads + 2 * kv, d)
    lo, hi = qkv[:, :heads + kv, :half].float(), qkv[:, :heads + kv, half:].float()
    turned = torch.cat([lo * c - hi * s, hi * c + lo * s], dim=2).to(torch.bfloat16)
    out["q"].copy_(turned[:, :heads].reshape(rows, heads * d))
    slot = x["table"].long()[seq, index // page]
    token = index % page
    columns = _columns(page, "cuda")[token]                                             # [rows, 64]
    blocks = lambda t: t.reshape(rows, kv, d // 64, 64).gather(3, columns[:, None, None].expand(rows, kv, d // 64, 64))  # noqa: E731
    out["k_cache"][slot, :, :, token] = blocks(turned[:, heads:])
    out["v_cache"][slot, :, :, token] = blocks(qkv[:, heads + kv:])
    return out


def _plain_pages(pool: torch.Tensor, pages: torch.Tensor) -> torch.Tensor:
    """[..., tokens, kv heads, head_dim] in 32 bits of the pages numbered ``pages`` [..., n]."""
    _, kv, blocks, page, _ = pool.shape
    at = _columns(page, pool.device).expand(*pages.shape, kv, blocks, page, 64)
    t = pool[pages.long()].gather(-1, at).float()                                       # [..., n, kv, blocks, page, 64]
    t = t.movedim(-2, -4)                                                               # [..., n, page, kv, blocks, 64]
    return t.reshape(*pages.shape[:-1], pages.shape[-1] * page, kv, blocks * 64)


def _plain_attention(state: dict) -> dict:
    case, x, s = state["case"], state["x"], state["sizes"]
    heads, kv, d, seqs, rows = case["q_heads"], case["kv_heads"], case["head_dim"], case["seqs"], s["rows"]
    group, most = heads // kv, s["longest"]
    seq, index = _plain_rows(state)
    place = torch.arange(rows, device="cuda") - x["starts"].long()[seq]
    q = torch.zeros(seqs, most, kv, group, d, device="cuda")
    q[seq, place] = x["q"].view(rows, kv, group, d).float() * d ** -0.5
    q = q.permute(0, 2, 3, 1, 4).reshape(seqs, kv, group * most, d)
    k, v = (_plain_pages(x[n], x["table"]).permute(0, 2, 1, 3) for n in ("k_cache", "v_cache"))      # [seqs, kv, keys, d]
    score = (q @ k.transpose(2, 3)).view(seqs, kv, group, most, -1)
    p = torch.full((seqs, most), -1, device="cuda")
    p[seq, place] = index
    key = torch.arange(score.shape[-1], device="cuda")
    seen = key <= p[:, :, None]
    if case["window"]:
        seen &= (p[:, :, None] - key < case["window"]) | (key < case["sinks"])
    score.masked_fill_(~seen[:, None, None], -math.inf)
    if case["op"] == "prefix":
        pk, pv = (_plain_pages(x[n], x["prefix_table"])[:case["prefix"]].permute(1, 0, 2) for n in ("k_cache", "v_cache"))
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


# ---- the definition in 64 bits, sequence by sequence ------------------------------------------------------

def _exact_tokens(pool: torch.Tensor, pages: list[int], count: int) -> torch.Tensor:
    """The first ``count`` tokens held in ``pages``, [tokens, kv heads, head_dim] in 64 bits."""
    page = pool.shape[3]
    out = []
    for j in range(8):                       # tokens j, j + 8, ... of a page keep their chunks in the same order
        rows = pool[pages][:, :, :, j::8].double()                           # [n, kv, blocks, page / 8, 64]
        chunks = [rows[..., 8 * (c ^ j):8 * (c ^ j) + 8] for c in range(8)]
        out.append(torch.cat(chunks, dim=-1))
    tokens = torch.stack(out, dim=4)                                         # [n, kv, blocks, page / 8, 8, 64]
    n, kv, blocks = tokens.shape[:3]
    return tokens.reshape(n, kv, blocks, page, 64).permute(0, 3, 1, 2, 4).reshape(n * page, kv, blocks * 64)[:count]


def _exact_append(case: dict, x: dict) -> dict:
    heads, kv, d, page = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"]
    half = d // 2
    new, total = _lengths(case)
    k_cache, v_cache = x["k_cache"].double(), x["v_cache"].double()
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
        index = torch.arange(t - n, t)
        for j in range(8):
            mine = [i for i in range(n) if int(index[i]) % page % 8 == j]
            if not mine:
                continue
            pages = [table[b][int(index[i]) // page] for i in mine]
            tokens = [int(index[i]) % page for i in mine]
            for c in range(8):
                for pool, values in ((k_cache, turned[:, heads:]), (v_cache, part[:, heads + kv:])):
                    source = values[mine].view(len(mine), kv, d // 64, 64)[..., 8 * c:8 * c + 8]
                    pool[pages, :, :, tokens, 8 * (c ^ j):8 * (c ^ j) + 8] = source
        row += n
    return {"q": torch.cat(q_all), "k_cache": k_cache, "v_cache": v_cache}


def _exact_attention(case: dict, x: dict) -> dict:
    heads, kv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    group, row, out = heads // kv, 0, []
    new, total = _lengths(case)
    table = x["table"].tolist()
    shared = None
    if case["op"] == "prefix":
        pages = x["prefix_table"].tolist()
        shared = [_exact_tokens(x[n], pages, case["prefix"]) for n in ("k_cache", "v_cache")]
    for b, (n, t) in enumerate(zip(new, total)):
        pages = table[b][:-(-t // case["page"])]
        k, v = (_exact_tokens(x[name], pages, t) for name in ("k_cache", "v_cache"))
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


def exact(case: dict, seed: int):
    x = _inputs(case, seed)
    return _exact_append(case, x) if case["op"] == "append" else _exact_attention(case, x)
