"""Packed operand layout of the bulk-copy tensor-core GEMM: "K-block-major, swizzled".

A matrix [R, K] of 1- or 2-byte elements is cut into 128-byte K blocks.  Block kb of row r is stored at byte
offset ``(kb * R_padded + r) * 128``, and inside it the 16-byte chunk c sits at position ``c ^ (r & 7)``: exactly
the image of a 128-byte-swizzled K-major shared-memory tile.  A tile of consecutive rows of one K block is
therefore ONE contiguous run of global memory, which a single bulk copy (no tensor map needed) drops into
shared memory ready for ``tcgen05.mma``.  Weights are packed once when the model is packaged (this module, on
the CPU); activations are written in this layout by the quantisation kernel.
"""
from __future__ import annotations

WEIGHT_ROW_PAD = 256        # packed weights are padded to whole 256-row tiles (zero rows)


def padded_weight_rows(n: int) -> int:
    return (n + WEIGHT_ROW_PAD - 1) // WEIGHT_ROW_PAD * WEIGHT_ROW_PAD


def padded_token_rows(m: int) -> int:
    """Rows reserved for a packed activation matrix: any token tile of up to 256 rows stays inside."""
    return (m + 255) // 256 * 256 + 256


def pack_kblock_swizzled(t, rows_padded: int | None = None):
    """[R, K] tensor (1- or 2-byte dtype, K bytes a multiple of 128) -> same dtype, shape
    [K bytes / 128, R_padded, 128 / element size]."""
    import torch
    rows, _ = t.shape
    elem = t.element_size()
    raw = t.contiguous().view(torch.uint8).reshape(rows, -1)
    k_bytes = raw.shape[1]
    if k_bytes % 128:
        raise ValueError("K must be a whole number of 128-byte blocks")
    rp = rows_padded if rows_padded is not None else padded_weight_rows(rows)
    padded = torch.zeros(rp, k_bytes, dtype=torch.uint8)
    padded[:rows] = raw
    blocks = padded.reshape(rp, k_bytes // 128, 8, 16).permute(1, 0, 2, 3)          # [kb, r, chunk, 16]
    source_chunk = torch.arange(8)[None, :] ^ (torch.arange(rp) % 8)[:, None]       # position p holds chunk p ^ (r & 7)
    index = source_chunk[None, :, :, None].expand(blocks.shape[0], rp, 8, 16)
    out = torch.gather(blocks, 2, index).contiguous()
    return out.reshape(k_bytes // 128, rp, 128).view(t.dtype).reshape(k_bytes // 128, rp, 128 // elem)


def unpack_kblock_swizzled(p, rows: int):
    """Inverse of ``pack_kblock_swizzled`` (drops the padding rows)."""
    import torch
    kb, rp, _ = p.shape
    raw = p.contiguous().view(torch.uint8).reshape(kb, rp, 8, 16)
    source_pos = torch.arange(8)[None, :] ^ (torch.arange(rp) % 8)[:, None]          # chunk c sits at position c ^ (r & 7)
    index = source_pos[None, :, :, None].expand(kb, rp, 8, 16)
    blocks = torch.gather(raw, 2, index)
    flat = blocks.permute(1, 0, 2, 3).reshape(rp, kb * 128)[:rows].contiguous()
    return flat.view(p.dtype)


def quantize_w4(t, group: int = 64):
    """A weight matrix [N, K] -> (codes [N, K] from 0 to 15 as uint8, scales [N, K / group] in bf16): the weight is (code - 8) * scale.  The
    scale is the largest |weight| of the group over 7, rounded up to a bf16 where rounding down would take it below (none is
    clipped then); a group of zeros has the scale zero, one that is not finite the scale NaN."""
    import torch
    n, k = t.shape
    if k % group:
        raise ValueError(f"{k} columns do not fall into groups of {group}")
    x = t.float().reshape(n, k // group, group)
    least = x.abs().amax(dim=-1) / 7
    scale = least.to(torch.bfloat16)
    scale = torch.where(scale.float() < least, torch.nextafter(scale, torch.full_like(scale, float("inf"))), scale)
    scale = torch.where(least.isfinite(), scale, torch.full_like(scale, float("nan")))
    codes = torch.where(scale[..., None] > 0, (x / scale.float()[..., None]).round().clamp(-8, 7) + 8, 8.0)
    return codes.to(torch.uint8).reshape(n, k), scale


def pack_w4(codes, scales):
    """Codes [N, K] from 0 to 15 and scales [N, K / group] that are bf16 numbers (``quantize_w4``, or a checkpoint's own) as ``gemm_w4`` takes them: int32
    [N / 16, K / 64, 32, 4] and bf16 [N / 16, K / group, 8, 2], N rounded up to 16 rows (a checkpoint stores the codes' bits as F32).
    The four bits from 4 p of word j of lane 4 g + t are the code of row g + 8 (p & 1), column 32 (j >> 1) + 8 t + 4 (j & 1) + (p & 2) + (p >> 2)
    of a tile of 16 rows and 64 columns: a lane's words are its operands of four matrix products, and its columns are eight in a row."""
    import torch
    n, k = codes.shape
    if k % 64 or k % scales.shape[1] or scales.shape[0] != n:
        raise ValueError(f"codes {list(codes.shape)} and scales {list(scales.shape)}: K is a multiple of 64 and of the group")
    if codes.numel() and not (0 <= int(codes.min()) and int(codes.max()) <= 15):
        raise ValueError(f"codes from {int(codes.min())} to {int(codes.max())}: they have four bits")
    if not torch.equal(scales.to(torch.bfloat16).double().nan_to_num(), scales.double().nan_to_num()):
        raise ValueError(f"scales ({scales.dtype}) that bf16 does not hold: round them, and make the codes for the rounded ones")
    tiles, groups = (n + 15) // 16, scales.shape[1]
    padded = torch.full((tiles * 16, k), 8, dtype=torch.int64, device=codes.device)
    padded[:n] = codes
    units = torch.zeros(tiles * 16, groups, dtype=torch.bfloat16, device=codes.device)
    units[:n] = scales
    # row: half h, g; column: j >> 1, t, j & 1, p & 2, p >> 2
    c = padded.reshape(tiles, 2, 8, k // 64, 2, 4, 2, 2, 2).permute(0, 3, 2, 5, 4, 6, 8, 7, 1)      # [tile, block, g, t, j, j, p >> 2, p & 2, p & 1]
    shift = 4 * torch.arange(8, device=codes.device)
    words = (c.reshape(tiles, k // 64, 32, 4, 8) << shift).sum(dim=-1)
    words = torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)
    return words, units.reshape(tiles, 2, 8, groups).permute(0, 3, 2, 1).contiguous()


def unpack_w4(words, scales, rows: int):
    """Inverse of ``pack_w4``, with the scales applied: the weights [rows, K] in fp32, exact."""
    import torch
    tiles, blocks = words.shape[:2]
    groups = scales.shape[1]
    shift = 4 * torch.arange(8, device=words.device, dtype=torch.int32)
    c = (words.view(torch.int32)[..., None] >> shift & 15).reshape(tiles, blocks, 8, 4, 2, 2, 2, 2, 2)
    c = c.permute(0, 8, 2, 1, 4, 3, 5, 7, 6).reshape(tiles * 16, groups, blocks * 64 // groups)
    units = scales.permute(0, 3, 2, 1).reshape(tiles * 16, groups, 1)
    return ((c - 8).float() * units.float()).reshape(tiles * 16, blocks * 64)[:rows]


def pack_kv_pages(t):
    """Keys or values [pages, page, kv_heads, head_dim] (2-byte dtype, head_dim a multiple of 64) -> the pool of a paged cache,
    [pages, kv_heads, head_dim / 64, page, 64]: 16-byte chunk c of a token's 64 columns sits at position ``c ^ (token & 7)``, so
    that consecutive tokens of a page, head and block are the image of a 128-byte-swizzled shared-memory tile."""
    pages, page, heads, d = t.shape
    blocks = t.reshape(pages, page, heads, d // 64, 8, 8).permute(0, 2, 3, 1, 4, 5)       # [..., token, chunk, 8]
    return _swap_chunks(blocks).reshape(pages, heads, d // 64, page, 64)


def unpack_kv_pages(p):
    """Inverse of ``pack_kv_pages``."""
    pages, heads, blocks, page, _ = p.shape
    t = _swap_chunks(p.reshape(pages, heads, blocks, page, 8, 8))
    return t.permute(0, 3, 1, 2, 4, 5).reshape(pages, page, heads, blocks * 64)


def quantize_kv_pages(t):
    """Keys or values [pages, page, kv_heads, head_dim] (head_dim 64 or 128) -> (codes, scales) of a paged cache in 8 bits: E4M3 codes
    [pages, kv_heads, page, head_dim] as uint8, in which 16-byte chunk c of token t sits at position ``c ^ (t & 7)``, or at
    ``c ^ ((t >> 1) & 3)`` of a row of 64; scales [pages, kv_heads, page] in bf16, the least power of two that brings the largest |value|
    of a token and head to 448 or less (one for zeros, 2^-126 at the least, NaN, with codes of zero, where a value is not finite)."""
    import torch
    x = t.permute(0, 2, 1, 3).float()
    peak = x.abs().amax(dim=-1)
    finite = x.isfinite().all(dim=-1)
    fraction, exponent = torch.frexp(torch.where(finite, peak, 1.0))        # fraction in [0.5, 1); 448 = 0.875 * 2^9
    exponent = torch.where(peak > 0, (exponent - 9 + (fraction > 0.875).int()).clamp_min(-126), 0)
    scale = torch.where(finite, torch.ldexp(torch.ones_like(peak), exponent), float("nan"))
    codes = torch.where(finite[..., None], x / scale[..., None], 0.0).clamp(-448, 448).to(torch.float8_e4m3fn)
    return _swap_code_chunks(codes.view(torch.uint8)), scale.to(torch.bfloat16)


def read_kv_pages(codes, scales):
    """Inverse of ``quantize_kv_pages`` but for the rounding: [pages, page, kv_heads, head_dim] in fp32."""
    import torch
    t = _swap_code_chunks(codes.view(torch.uint8)).view(torch.float8_e4m3fn).float() * scales.float()[..., None]
    return t.permute(0, 2, 1, 3).contiguous()


def _swap_code_chunks(t):
    """[..., page, head_dim] bytes with the 16-byte chunks of every token exchanged (its own inverse)."""
    import torch
    page, d = t.shape[-2:]
    if d not in (64, 128):
        raise ValueError(f"a cache in 8 bits holds heads 64 or 128 wide, not {d}")
    token = torch.arange(page, device=t.device)[:, None]
    source = torch.arange(d // 16, device=t.device)[None, :] ^ (token % 8 if d == 128 else token // 2 % 4)
    chunks = t.reshape(*t.shape[:-1], d // 16, 16)
    return torch.gather(chunks, -2, source[:, :, None].expand(chunks.shape)).reshape(t.shape).contiguous()


def _swap_chunks(t):
    """[..., token, chunk, 8] with chunk c of token r exchanged with chunk c ^ (r & 7) (its own inverse)."""
    import torch
    tokens = torch.arange(t.shape[-3], device=t.device)
    source = torch.arange(8, device=t.device)[None, :] ^ (tokens % 8)[:, None]
    return torch.gather(t, -2, source[:, :, None].expand(t.shape)).contiguous()
