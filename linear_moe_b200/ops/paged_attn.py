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
from typing import Dict, Optional, Tuple

import torch

from ..ref import ops as R
from .scored_attn import _check_scores, on_device

GROUP, MIN_GROUPS, MAX_CLUSTER = 16, 8, 8     # csrc/paged_step.cuh, .cu


class _Args(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p) for n in ("q", "k_new", "v_new", "k", "v", "out", "part", "ml", "slopes", "table", "lengths")] +
                [(n, ctypes.c_longlong) for n in ("q_b", "q_h", "n_b", "n_h", "m_b", "m_h", "k_page", "k_row", "k_head", "v_page", "v_row", "v_head", "table_ld")] +
                [(n, ctypes.c_int) for n in ("B", "H", "G", "D", "page", "pages", "table_n", "window", "splits", "sorted")] +
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


def splits_of(B: int, G: int, heads: int, D: int, keys: int) -> Tuple[int, int]:
    """(CTAs that share a key head of a request of up to ``keys`` keys, are the longest requests to come first).

    One wave: as many parts as give every slot of the GPU a CTA, of 128 keys at least (300 keys in three parts 5.4 us, in two or one 6.9).  Eight requests of up to 2048 keys, 8 heads of 64: 25 us in one part, 8.9 in eight; one
    of 65536, 8 heads of 128: 112 in 8 parts, 48 in 32, 54 in 64.  Requests that fill more than half of the slots by themselves, but not four waves, go in two parts each, so that the end
    of the longest ones is shared (32 requests of up to 3000 keys, 8 heads of 128: 48 -> 39), and with more CTAs than slots the longest ones first (64 of up to 8192: 200 -> 187)."""
    from . import cuda as K
    work, slots = B * G * (1 if heads <= 8 else -(-heads // 16)), (4 if D <= 64 else 2) * K.num_sms()
    n = slots // work if 2 * work <= slots else 2 if work < 4 * slots else 1
    n = min(n, -(-keys // (GROUP * MIN_GROUPS)))
    n = 8 if MAX_CLUSTER < n < 16 else max(n, 1)            # a cluster joins eight parts in the same launch (1024 keys: 6.3 us, in 16 parts and two launches 6.9)
    return n, int(1 < B <= 128 and work * n > slots)


class _Plan:
    """What follows from shapes, strides and types alone: the arguments without their addresses, and the launch."""
    __slots__ = ("args", "align", "flat", "work", "part", "launch", "name", "count")


def _plan(q, k, v, table, lengths, scale, window, softcap, slopes, k_new, v_new) -> _Plan:
    from . import cuda as K
    _check(q, k, v, table, lengths, scale, window, softcap, slopes, k_new, v_new)
    B, H, D = q.shape
    P, page, G = k.shape[:3]
    p, a = _Plan(), _Args()
    a.q_b, a.q_h = q.stride(0), q.stride(1)
    a.k_page, a.k_row, a.k_head = _dense(k)
    a.v_page, a.v_row, a.v_head = _dense(v)
    if k_new is not None:
        a.n_b, a.n_h, a.m_b, a.m_h = k_new.stride(0), k_new.stride(1), v_new.stride(0), v_new.stride(1)
    a.B, a.H, a.G, a.D, a.page, a.pages, a.table_n, a.table_ld = B, H, G, D, page, P, table.shape[1], table.stride(0)
    a.window, a.scale, a.cap, a.splits = min(int(window or 0), (1 << 31) - 1), float(scale) if scale is not None else D ** -0.5, float(softcap or 0.0), 1
    p.flat = all(t is None or t.stride(-1) == 1 or t.shape[-1] <= 1 for t in (q, k_new, v_new, table, lengths, slopes))
    # 16-byte rows (of q and the new token too: misaligned ones are rare and small, but a copy of the cache is out of the question)
    vec = (q.dtype != torch.float32 and D % 8 == 0 and D <= 128 and page % GROUP == 0 and P > 0 and
           all(x % 8 == 0 for x in (a.q_b, a.q_h, a.n_b, a.n_h, a.m_b, a.m_h)) and
           all(x % 8 == 0 and 0 < x < 1 << 38 for x in (a.k_page, a.k_row, a.k_head, a.v_page, a.v_row, a.v_head)))
    p.align = 15 if vec else 0
    p.work = p.part = 0
    if vec:
        a.splits, a.sorted = splits_of(B, G, H // G, D, table.shape[1] * page)
        if a.splits > MAX_CLUSTER:
            p.part = B * H * a.splits * D * 4
            p.work = B * H * a.splits * (D + 2)
        p.launch, p.name, p.count = K.lib().lmoe_paged_step, "paged_step", 1 if a.splits <= MAX_CLUSTER else 2
    p.args = bytes(a)
    return p


def _dense(t: torch.Tensor):
    """Strides of a pool; those of dimensions of one, which say nothing, as in a dense tensor."""
    out, dense = [0, 0, 0], t.shape[3]
    for i in (2, 1, 0):
        out[i] = t.stride(i) if t.shape[i] > 1 else dense
        dense *= t.shape[i]
    return out


_PLANS: Dict[tuple, _Plan] = {}
_KIND = {torch.bfloat16: 0, torch.float16: 1}


def paged_attention(q, k_pages, v_pages, table, lengths, scale: Optional[float] = None, window: Optional[int] = None, *, softcap: Optional[float] = None,
                    slopes: Optional[torch.Tensor] = None, k_new=None, v_new=None):
    """``[B, H, D]``; see the module.  Forward only."""
    if torch.is_grad_enabled() and (q.requires_grad or k_pages.requires_grad or v_pages.requires_grad or (k_new is not None and k_new.requires_grad)
                                    or (v_new is not None and v_new.requires_grad)):
        raise ValueError("one-token attention has no backward pass: use ops.softmax_attention")
    if not q.is_cuda:
        _check(q, k_pages, v_pages, table, lengths, scale, window, softcap, slopes, k_new, v_new)
        return R.paged_attention(q, k_pages, v_pages, table, lengths, scale, window, softcap, slopes, k_new, v_new)
    from . import cuda as K
    dev = q.device
    # the host's share of a short step is as long as the kernel: checks, strides and the launch's shape are worked out once per layout
    key = (q.shape, q.stride(), q.dtype, dev, k_pages.shape, k_pages.stride(), k_pages.dtype, k_pages.device, v_pages.shape, v_pages.stride(), v_pages.dtype,
           v_pages.device, table.shape, table.stride(), table.dtype, table.device, lengths.shape, lengths.stride(), lengths.dtype, lengths.device, scale, window, softcap,
           slopes if slopes is None else (slopes.shape, slopes.stride(), slopes.dtype, slopes.device, slopes.requires_grad),
           k_new if k_new is None else (k_new.shape, k_new.stride(), k_new.dtype, k_new.device),
           v_new if v_new is None else (v_new.shape, v_new.stride(), v_new.dtype, v_new.device))
    p = _PLANS.get(key)
    if p is None:
        if len(_PLANS) >= 4096:
            _PLANS.clear()
        p = _PLANS[key] = _plan(q, k_pages, v_pages, table, lengths, scale, window, softcap, slopes, k_new, v_new)
    if not p.flat:
        flat = lambda t: t if t is None or t.stride(-1) == 1 else t.contiguous()      # noqa: E731
        return paged_attention(flat(q), k_pages, v_pages, flat(table), flat(lengths), scale, window, softcap=softcap, slopes=flat(slopes), k_new=flat(k_new),
                               v_new=flat(v_new))
    out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    if out.numel() == 0:
        return out
    a = _Args.from_buffer_copy(p.args)
    a.q, a.k, a.v, a.out = qp, kp, vp, a_out = q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), out.data_ptr()
    a.table, a.lengths = table.data_ptr(), lengths.data_ptr()
    bits = qp | kp | vp | a_out
    if k_new is not None:
        a.k_new, a.v_new = kn, vn = k_new.data_ptr(), v_new.data_ptr()
        bits |= kn | vn
    if slopes is not None:
        a.slopes = slopes.data_ptr()
    a.err = K.error_word(dev)
    with on_device(q):
        if not p.align or bits & p.align:
            a.splits, a.sorted = 1, 0
            K._check(K.lib().lmoe_paged_step_any(ctypes.byref(a), _TYPES[q.dtype], K._st()), "paged_step_any")
            return out
        if p.work:
            work = torch.empty(p.work, dtype=torch.float32, device=dev)
            a.part = base = work.data_ptr()
            a.ml = base + p.part
        K._check(p.launch(ctypes.byref(a), _KIND[q.dtype], K._st()), p.name, p.count)
    return out
