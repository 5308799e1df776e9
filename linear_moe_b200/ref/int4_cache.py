"""Eager definition of the paged cache of 4 bits a number (layout: :mod:`linear_moe_b200.ops.int4_cache`)."""
from __future__ import annotations

import torch

UNIT = 32
FIFTEENTH = float(torch.tensor(1.0 / 15.0))               # in 32 bits


def place(n: int, rows: torch.Tensor) -> torch.Tensor:
    """Where the groups of the given rows of a page lie, ``[rows, n]``."""
    at = torch.arange(n, device=rows.device)[None]
    return at ^ (rows[:, None] // 2 % 4) if n == 4 else at ^ (rows[:, None] // 4 % 2) if n == 2 else at.expand(rows.shape[0], n)


def encode(x: torch.Tensor):
    """``x [..., D]`` -> codes ``[..., D / 32, 32]`` (uint8), lows and sizes ``[..., D / 32]`` (bf16)."""
    g = x.float().unflatten(-1, (-1, UNIT))
    finite = g.isfinite().all(-1)
    g = torch.where(finite[..., None], g, 0.0)
    least = g.amin(-1)
    bits = torch.where(least == 0, 0.0, least).view(torch.int32)                          # of zeros the positive one
    low = (torch.where(bits < 0, bits + 0xffff, bits) & -65536).view(torch.float32)
    size = ((((g.amax(-1) - low) * FIFTEENTH).abs().view(torch.int32) + 0xffff) & -65536).view(torch.float32)      # (never -0)
    finite = finite & low.isfinite() & size.isfinite()
    code = torch.round((g - low[..., None]) / torch.where(size > 0, size, 1.0)[..., None]).clamp(0, 15)
    code = torch.where((finite & (size > 0))[..., None], code, 0.0)
    def upper(x, other):                                  # bf16 from its bits: how NaN is rounded follows the device
        return torch.where(finite, x.view(torch.int32) >> 16, other).to(torch.int16).view(torch.bfloat16)
    return code.to(torch.uint8), upper(low, 0x7fc0), upper(size, 0)


def _parts(pool: torch.Tensor, D: int):
    """Codes ``[P, G, page, D / 32, 16]`` and scales ``[P, G, page, D / 8]`` of a pool, as views."""
    P, G, n = pool.shape
    page = 8 * n // (5 * D)
    return pool[..., : page * D // 2].view(P, G, page, D // UNIT, 16), pool[..., page * D // 2:].view(P, G, page, D // 8)


def write(pool: torch.Tensor, pages: torch.Tensor, rows: torch.Tensor, x: torch.Tensor):
    """Row i of ``x [n, G, D]`` to row ``rows[i]`` of page ``pages[i]``."""
    codes, scales = _parts(pool, x.shape[-1])
    code, low, size = encode(x)
    packed = code[..., 0::2] | code[..., 1::2] << 4
    at = place(low.shape[-1], rows)[:, None, :, None].expand(packed.shape)
    codes[pages, :, rows] = torch.empty_like(packed).scatter_(2, at, packed)
    scales[pages, :, rows] = torch.cat([low, size], -1).view(torch.uint8)


def read(pool: torch.Tensor, pages: torch.Tensor, rows: torch.Tensor, D: int) -> torch.Tensor:
    """Rows ``rows`` of the pages ``pages`` (both ``[n]``), fp32 ``[n, G, D]``."""
    codes, scales = _parts(pool, D)
    n = D // UNIT
    packed = codes[pages, :, rows]
    packed = packed.gather(2, place(n, rows)[:, None, :, None].expand(packed.shape))
    s = scales[pages, :, rows].contiguous().view(torch.bfloat16).float()
    code = torch.stack([packed & 15, packed >> 4], -1).flatten(-2).float()
    return (s[..., :n, None] + s[..., n:, None] * code).flatten(-2)


def _rows(table, b, keys, page, pages, capacity, n):
    if not 0 <= n <= capacity:
        raise ValueError(f"request {b}: a length of {n} in a table of {table.shape[1]} pages of {page}")
    at = table[b].long()[keys // page]
    if at.numel() and not 0 <= int(at.min()) <= int(at.max()) < pages:
        raise ValueError(f"request {b}: a page outside the {pages} that there are")
    return at


def store_rows(k_new, v_new, k_pool, v_pool, table, lengths):
    B, T, G, D = k_new.shape
    page = 8 * k_pool.shape[2] // (5 * D)
    for b, n in enumerate(lengths.tolist()):
        keys = torch.arange(max(n - T, 0), max(n, 0), device=k_new.device)
        at = _rows(table, b, keys, page, k_pool.shape[0], table.shape[1] * page, n)
        for pool, new in ((k_pool, k_new), (v_pool, v_new)):
            write(pool, at, keys % page, new[b, T - len(keys):])


def read_rows(k_pool, v_pool, table, lengths, n, D, dtype):
    B, G = table.shape[0], k_pool.shape[1]
    page = 8 * k_pool.shape[2] // (5 * D)
    out = torch.zeros(2, B, n, G, D, dtype=dtype, device=k_pool.device)
    for b, length in enumerate(lengths.tolist()):
        keys = torch.arange(max(0, min(n, length)), device=k_pool.device)
        at = _rows(table, b, keys, page, k_pool.shape[0], table.shape[1] * page, length)
        for i, pool in enumerate((k_pool, v_pool)):
            out[i, b, : len(keys)] = read(pool, at, keys % page, D).to(dtype)
    return out[0], out[1]


def paged_attention(q, k_pool, v_pool, table, lengths, scale=None, window=None, softcap=None, slopes=None):
    B, H, D = q.shape
    G, page = k_pool.shape[1], 8 * k_pool.shape[2] // (5 * D)
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(B, H, D, dtype=q.dtype, device=q.device)
    for b, n in enumerate(lengths.tolist()):
        keys = torch.arange(max(0, n - window) if window is not None else 0, max(n, 0), device=q.device)
        at = _rows(table, b, keys, page, k_pool.shape[0], table.shape[1] * page, n)
        if n == 0:
            continue
        k, v = (read(pool, at, keys % page, D) for pool in (k_pool, v_pool))
        x = torch.einsum("grd,jgd->grj", q[b].float().reshape(G, H // G, D) * scale, k)
        if softcap is not None:
            x = softcap * torch.tanh(x / softcap)
        if slopes is not None:
            x = x - slopes.float().reshape(G, H // G, 1) * (n - 1 - keys).float()
        out[b] = torch.einsum("grj,jgd->grd", torch.softmax(x, -1), v).reshape(H, D).to(q.dtype)
    return out
