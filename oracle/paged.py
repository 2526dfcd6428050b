"""Paged K/V cache oracles in 64 bits: tokens are kept as plain [tokens, kv_heads, head_dim] tensors per sequence, row by row."""
from __future__ import annotations

import math

import torch


def rotary_angles(positions: torch.Tensor, theta: float, head_dim: int, sections=None, ladder: int | None = None) -> torch.Tensor:
    """[rows, head_dim / 2] angles of positions [rows], or [3, rows] with ``sections``."""
    half, ladder = head_dim // 2, ladder or head_dim // 2
    pair = torch.arange(half)
    frequency = float(theta) ** (-(pair % ladder).double() / ladder)
    if sections is None:
        return positions.double()[:, None] * frequency
    axis = torch.tensor([0] * sections[0] + [1] * sections[1] + [2] * sections[2])
    return positions.double()[axis].t() * frequency


def turn(x: torch.Tensor, angles: torch.Tensor) -> torch.Tensor:
    """x [rows, heads, head_dim], half-split pairs, in 64 bits."""
    half = x.shape[-1] // 2
    a, b = x[..., :half].double(), x[..., half:].double()
    c, s = angles.cos()[:, None], angles.sin()[:, None]
    return torch.cat([a * c - b * s, b * c + a * s], dim=-1)


def attention(q, keys, values, index: int, window: int = 0, sinks: int = 0, scale: float | None = None, prefix=None):
    """One row: q [heads, head_dim] at ``index`` of a sequence whose tokens are keys / values [tokens, kv_heads, head_dim];
    ``prefix``: (keys, values) that every row sees first.  Returns (o, mass): the output and sum_j p_j |v_j|, what the weights'
    rounding is relative to."""
    heads, d = q.shape
    seen = [j for j in range(min(index + 1, keys.shape[0])) if window == 0 or index - j < window or j < sinks] if index >= 0 else []
    k, v = keys[seen].double(), values[seen].double()
    if prefix is not None:
        k, v = torch.cat([prefix[0].double(), k]), torch.cat([prefix[1].double(), v])
    if k.shape[0] == 0:
        return torch.zeros(heads, d, dtype=torch.float64), torch.zeros(heads, d, dtype=torch.float64)
    group = heads // k.shape[1]
    kv_head = torch.arange(heads) // group
    score = torch.einsum("hd,khd->hk", q.double(), k[:, kv_head]) * (scale if scale is not None else 1.0 / math.sqrt(d))
    p = torch.softmax(score, dim=1)
    return torch.einsum("hk,khd->hd", p, v[:, kv_head]), torch.einsum("hk,khd->hd", p, v[:, kv_head].abs())
