"""Attention of one new token per request over a paged cache (the one-token form of :mod:`.scored_attn`).

    x_j = cap tanh(scale q k_j / cap) - slope_h (n - 1 - j),   o = sum_j softmax_j(x_j) v_j   over  max(0, n - window) <= j < n

The cache is a pool of pages ``[P, page, heads, dim]`` for keys and one for values (:class:`~linear_moe_b200.infer.kv_cache.LayerPages`); a request's keys lie on the pages of
its row of ``table``, in order.  ``lengths`` (on the device, so captured steps go on growing) counts the new token, whose row ``k_new`` / ``v_new`` is stored at its place by the
same call.  bf16 and fp16 with heads of up to 128, in multiples of 8, run ``csrc/paged_step.cu``, split over the cache's length and joined; the rest of what CUDA tensors can be runs
``csrc/paged_step_any.cu`` and CPU tensors the eager definition.

A length outside the table is clipped and a page number outside the pool hides its keys (nothing is read or stored there); on CUDA both set the kernels' error word
(``ops.gemm.check_error``), on the CPU they raise.  Two requests may share pages, but not the row that one of them stores."""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from ..ref import ops as R
from .scored_attn import _check_scores, on_device

GROUP, MIN_GROUPS = 16, 16                     # csrc/paged_step.cuh


class _Args(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p) for n in ("q", "k_new", "v_new", "k", "v", "out", "part", "ml", "slopes", "table", "lengths")] +
                [(n, ctypes.c_longlong) for n in ("q_b", "q_h", "n_b", "n_h", "m_b", "m_h", "k_page", "k_row", "k_head", "v_page", "v_row", "v_head", "table_ld")] +
                [(n, ctypes.c_int) for n in ("B", "H", "G", "D", "page", "pages", "table_n", "window", "splits")] +
                [("scale", ctypes.c_float), ("cap", ctypes.c_float), ("err", ctypes.c_void_p)])


_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _check(q, k, v, table, lengths, scale, window, softcap, slopes, k_new, v_new):
    if q.dim() != 3 or k.dim() != 4 or v.shape != k.shape or k.shape[3] != q.shape[2]:
        raise ValueError("paged attention takes q [B, H, D] and pages [P, page, heads, D] of keys and of values")
    B, H, D = q.shape
    if k.shape[2] == 0 or H % k.shape[2] or k.shape[1] == 0:
        raise ValueError(f"{H} query heads do not share {k.shape[2]} key/value heads evenly, or pages of {k.shape[1]} rows")
    if q.dtype not in _TYPES or not q.dtype == k.dtype == v.dtype:
        raise ValueError("queries and pages have one type: fp32, bf16 or fp16")
    if D > 512 or D == 0:
        raise ValueError(f"heads of {D} numbers (up to 512)")
    if table.dtype != torch.int32 or table.dim() != 2 or table.shape[0] != B or lengths.dtype != torch.int32 or lengths.shape != (B,):
        raise ValueError(f"the table is int32 [{B}, pages] and the lengths int32 [{B}]")
    if (k_new is None) != (v_new is None):
        raise ValueError("the new token's key and value come together")
    for t in (k_new, v_new):
        if t is not None and (t.shape != (B, k.shape[2], D) or t.dtype != q.dtype):
            raise ValueError(f"the new rows are [B, heads, D] = [{B}, {k.shape[2]}, {D}] of the queries' type")
    if any(t is not None and t.device != q.device for t in (k, v, table, lengths, k_new, v_new)):
        raise ValueError("the tensors lie on one device")
    if window is not None and window < 1:
        raise ValueError(f"a window of {window}")
    if k.stride(3) != 1 or v.stride(3) != 1 or any(s < 0 for s in k.stride() + v.stride()):
        raise ValueError("a page's rows have unit stride along the head")
    if B > 65535 or table.shape[1] * k.shape[1] >= (1 << 31) - 16:
        raise ValueError("more requests or longer tables than the kernels count")
    _check_scores(q, H, scale, softcap, slopes)


def splits_of(B: int, G: int, heads: int, keys: int) -> int:
    """CTAs that share a key head of a request of up to ``keys`` keys."""
    from . import cuda as K
    work = B * G * (1 if heads <= 8 else -(-heads // 16))
    return max(1, min(-(-20 * K.num_sms() // work), -(-keys // (GROUP * MIN_GROUPS))))


def paged_attention(q, k_pages, v_pages, table, lengths, scale: Optional[float] = None, window: Optional[int] = None, *, softcap: Optional[float] = None,
                    slopes: Optional[torch.Tensor] = None, k_new=None, v_new=None):
    """``[B, H, D]``; see the module.  Forward only."""
    _check(q, k_pages, v_pages, table, lengths, scale, window, softcap, slopes, k_new, v_new)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k_pages, v_pages, k_new, v_new)):
        raise ValueError("one-token attention has no backward pass: use ops.softmax_attention")
    if not q.is_cuda:
        return R.paged_attention(q, k_pages, v_pages, table, lengths, scale, window, softcap, slopes, k_new, v_new)
    from . import cuda as K
    from . import gemm
    B, H, D = q.shape
    P, page, G = k_pages.shape[:3]
    out = torch.empty(B, H, D, dtype=q.dtype, device=q.device)
    if out.numel() == 0:
        return out
    flat = lambda t: t if t is None or t.stride(2) == 1 or D == 1 else t.contiguous()      # noqa: E731
    q, k_new, v_new = flat(q), flat(k_new), flat(v_new)
    table = table if table.stride(1) == 1 or table.shape[1] <= 1 else table.contiguous()
    lengths = lengths if lengths.is_contiguous() else lengths.contiguous()
    slopes = slopes if slopes is None or slopes.is_contiguous() else slopes.contiguous()
    a = _Args()
    a.q, a.q_b, a.q_h, a.out = q.data_ptr(), q.stride(0), q.stride(1), out.data_ptr()
    a.k, a.k_page, a.k_row, a.k_head = k_pages.data_ptr(), k_pages.stride(0), k_pages.stride(1), k_pages.stride(2)
    a.v, a.v_page, a.v_row, a.v_head = v_pages.data_ptr(), v_pages.stride(0), v_pages.stride(1), v_pages.stride(2)
    if k_new is not None:
        a.k_new, a.n_b, a.n_h, a.v_new, a.m_b, a.m_h = k_new.data_ptr(), k_new.stride(0), k_new.stride(1), v_new.data_ptr(), v_new.stride(0), v_new.stride(1)
    a.slopes, a.table, a.lengths, a.table_ld = K._ptr(slopes), table.data_ptr(), lengths.data_ptr(), table.stride(0)
    a.B, a.H, a.G, a.D, a.page, a.pages, a.table_n = B, H, G, D, page, P, table.shape[1]
    a.window, a.scale, a.cap, a.splits = int(window or 0), float(scale) if scale is not None else D ** -0.5, float(softcap or 0.0), 1
    a.err = gemm._err(q.device).data_ptr()
    # 16-byte rows (of q and the new token too: misaligned ones are rare and small, but a copy of the cache is out of the question)
    vec = (q.dtype != torch.float32 and D % 8 == 0 and D <= 128 and page % GROUP == 0 and
           all(x % 8 == 0 for x in (a.q_b, a.q_h, a.n_b, a.n_h, a.m_b, a.m_h, a.k_page, a.k_row, a.k_head, a.v_page, a.v_row, a.v_head)) and
           all((x or 0) % 16 == 0 for x in (a.q, a.k, a.v, a.k_new, a.v_new)))
    with on_device(q):
        if not vec:
            K._check(K.lib().lmoe_paged_step_any(ctypes.byref(a), ctypes.c_int(_TYPES[q.dtype]), K._st()), "paged_step_any")
            return out
        a.splits = splits_of(B, G, H // G, table.shape[1] * page)
        if a.splits > 1:
            work = torch.empty(B * H * a.splits * (D + 2), dtype=torch.float32, device=q.device)
            a.part, a.ml = work.data_ptr(), work.data_ptr() + B * H * a.splits * D * 4
        K._check(K.lib().lmoe_paged_step(ctypes.byref(a), ctypes.c_int(int(q.dtype == torch.float16)), K._st()), "paged_step", 1 if a.splits == 1 else 2)
    return out
