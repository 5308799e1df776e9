"""A paged cache of 4 bits a number: rows into it, rows out of it, and attention of one new token per request over it (CUDA: ``csrc/int4_cache.cu``, ``csrc/int4_step.cu``; CPU tensors run the eager
definition).

A row of a head goes in groups of 32 numbers, ``x = low + size * code`` with codes of 0 to 15: ``low`` is the least number of the group, rounded down to bf16, ``size`` a fifteenth of what is left up to the
greatest one, rounded up to bf16, so that a number comes back within half a size.  That is 5/8 byte a number, 80 bytes a row of 128 where bf16 has 256.  A group with a number that is not finite, or with a
range that 32 bits do not hold, comes back as NaN.

A pool is one uint8 tensor ``[pages, heads, page * 5 D / 8]`` (:func:`int4_pages`) for keys and one for values; ``copy_pages_`` copies its pages like any other's.  Per page and head it holds the codes of its rows
(``D / 2`` bytes each, the lower half of a byte first) and then every row's lows and sizes; ``csrc/int4_cache.cuh`` says in which order a row's groups lie.  A request's rows are on the pages of its row of ``table``, in order;
``lengths`` (on the device, so captured steps go on growing) counts the rows that a call brings.

A length outside the table is clipped (:func:`store_rows_int4` then leaves the request out) and a page number outside the pool hides its rows (nothing is read or stored there); on CUDA both set the kernels' error word
(``ops.gemm.check_error``), on the CPU they raise.  Two requests may share pages, but not the rows that one of them stores."""
from __future__ import annotations

import ctypes
from typing import Dict, Optional, Tuple

import torch

from ..ref import int4_cache as R
from .scored_attn import _check_scores, on_device

UNIT, GROUP, WIDEST, MOST_ROWS = R.UNIT, 16, 256, 1 << 16


class _Rows(ctypes.Structure):
    _fields_ = [("x", ctypes.c_void_p * 2), ("pool", ctypes.c_void_p * 2), ("table", ctypes.c_void_p), ("lengths", ctypes.c_void_p), ("x_b", ctypes.c_longlong * 2), ("x_t", ctypes.c_longlong * 2),
                ("x_g", ctypes.c_longlong * 2), ("table_ld", ctypes.c_longlong)] + [(n, ctypes.c_int) for n in ("B", "T", "G", "D", "page", "pages", "table_n", "page_bits")] + [("err", ctypes.c_void_p)]


class _Step(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p) for n in ("q", "k", "v", "out", "part", "ml", "slopes", "table", "lengths")] + [(n, ctypes.c_longlong) for n in ("q_b", "q_h", "table_ld")] +
                [(n, ctypes.c_int) for n in ("B", "H", "G", "D", "page", "pages", "table_n", "window", "splits", "q_rows", "sorted")] +
                [("scale", ctypes.c_float), ("cap", ctypes.c_float), ("err", ctypes.c_void_p)])


_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def int4_pages(pages: int, heads: int, dim: int, page: int = 64, device=None) -> torch.Tensor:
    """An empty pool of ``pages`` pages of ``page`` rows (a multiple of 16) of ``heads`` heads of ``dim`` numbers (a multiple of 32, up to 256)."""
    if dim % UNIT or not 0 < dim <= WIDEST or page % GROUP or not 0 < page <= MOST_ROWS:
        raise ValueError(f"heads of {dim} numbers (a multiple of {UNIT} up to {WIDEST}), pages of {page} rows (a multiple of {GROUP} up to {MOST_ROWS})")
    return torch.zeros(pages, heads, page * 5 * dim // 8, dtype=torch.uint8, device=device)


def _check_pools(k_pages, v_pages, table, lengths, B: int, G: Optional[int], D: int) -> int:
    """Rows of a page."""
    if D % UNIT or not 0 < D <= WIDEST:
        raise ValueError(f"heads of {D} numbers (a multiple of {UNIT} up to {WIDEST})")
    for p in (k_pages, v_pages):
        if p.dtype != torch.uint8 or p.dim() != 3 or p.shape != k_pages.shape or not p.is_contiguous() or p.data_ptr() % 16:
            raise ValueError("a pool of 4 bits a number is uint8 [pages, heads, page bytes], dense, from a 16-byte boundary on")
    if G is not None and k_pages.shape[1] != G:
        raise ValueError(f"rows of {G} heads for pages of {k_pages.shape[1]}")
    n = k_pages.shape[2]
    page = 8 * n // (5 * D)
    if page == 0 or page % GROUP or page > MOST_ROWS or page * 5 * D != 8 * n:
        raise ValueError(f"{n} bytes are no whole pages of a multiple of {GROUP} rows (up to {MOST_ROWS}) of {D} numbers")
    if table.dtype != torch.int32 or table.dim() != 2 or table.shape[0] != B or lengths.dtype != torch.int32 or lengths.shape != (B,):
        raise ValueError(f"the table is int32 [{B}, pages] and the lengths int32 [{B}]")
    if any(t.device != k_pages.device for t in (v_pages, table, lengths)):
        raise ValueError("the tensors lie on one device")
    if B > 65535 or table.shape[1] * page >= (1 << 31) - 4096:
        raise ValueError("more requests or longer tables than the kernels count")
    return page


def _key(t: Optional[torch.Tensor]):
    return t if t is None else (t.shape, t.stride(), t.dtype, t.device)


_PLANS: Dict[tuple, object] = {}


def _planned(key: tuple, make):
    p = _PLANS.get(key)
    if p is None:
        if len(_PLANS) >= 4096:
            _PLANS.clear()
        p = _PLANS[key] = make()
    return p


def _flat(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def _rows_args(table, page, pages, G, D, T) -> _Rows:
    return _Rows(table_ld=table.stride(0), B=table.shape[0], T=T, G=G, D=D, page=page, pages=pages, table_n=table.shape[1], page_bits=page.bit_length() - 1 if page & (page - 1) == 0 else -1)


# ---- rows into the cache ----------------------------------------------------------------------------------------------------------
def _store_plan(k_new, v_new, k_pages, v_pages, table, lengths):
    if k_new.dim() != 4 or v_new.shape != k_new.shape or k_new.dtype not in _TYPES or v_new.dtype != k_new.dtype or k_new.device != k_pages.device or v_new.device != k_pages.device:
        raise ValueError("rows are [B, T, heads, D], keys and values alike, in fp32, bf16 or fp16, where the pools lie")
    B, T, G, D = k_new.shape
    page = _check_pools(k_pages, v_pages, table, lengths, B, G, D)
    if T >= 1 << 30 or G > 32767:
        raise ValueError(f"{T} rows of {G} heads are more than the kernel counts")
    a = _rows_args(table, page, k_pages.shape[0], G, D, T)
    rows = True                                             # strides of the rows as they are: 16-byte steps
    for i, t in enumerate((k_new, v_new)):
        a.x_b[i], a.x_t[i], a.x_g[i] = t.stride()[:3]
        rows = rows and (t.stride(3) == 1 or D == 1) and all(s * t.element_size() % 16 == 0 for s in t.stride()[:3])
    return bytes(a), rows


def store_rows_int4(k_new: torch.Tensor, v_new: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor):
    """Rows ``k_new``, ``v_new`` ``[B, T, heads, D]`` become the last T of the ``lengths[b]`` rows of request b; those that would lie in front of the first one (padding on the left, a
    request of no rows) are left out.  No gradient: what is stored is the rows' values."""
    if not k_new.is_cuda:
        _store_plan(k_new, v_new, k_pages, v_pages, table, lengths)
        with torch.no_grad():
            return R.store_rows(k_new, v_new, k_pages, v_pages, table, lengths)
    from . import cuda as K
    plan, rows = _planned(("store", _key(k_new), _key(v_new), _key(k_pages), _key(v_pages), _key(table), _key(lengths), (k_pages.data_ptr() | v_pages.data_ptr()) % 16),
                          lambda: _store_plan(k_new, v_new, k_pages, v_pages, table, lengths))
    if not rows or (k_new.data_ptr() | v_new.data_ptr()) % 16:
        k_new, v_new = (t.clone(memory_format=torch.contiguous_format) for t in (k_new.detach(), v_new.detach()))
        plan, _ = _store_plan(k_new, v_new, k_pages, v_pages, table, lengths)
    if k_new.numel() == 0:
        return
    table, lengths = _flat(table), _flat(lengths)
    a = _Rows.from_buffer_copy(plan)
    a.table_ld = table.stride(0)
    a.x[0], a.x[1], a.pool[0], a.pool[1] = k_new.data_ptr(), v_new.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr()
    a.table, a.lengths, a.err = table.data_ptr(), lengths.data_ptr(), K.error_word(k_pages.device)
    with on_device(k_pages):
        K._check(K.lib().lmoe_int4_rows(ctypes.byref(a), _TYPES[k_new.dtype], 0, K._st()), "int4_store")


# ---- rows out of the cache --------------------------------------------------------------------------------------------------------
def _read_plan(k_pages, v_pages, table, lengths, n, dim, dtype):
    if dtype not in _TYPES or n < 0:
        raise ValueError(f"{n} rows in {dtype}: fp32, bf16 or fp16")
    if table.dim() != 2:
        raise ValueError("the table is int32 [B, pages]")
    page = _check_pools(k_pages, v_pages, table, lengths, table.shape[0], None, dim)
    if n >= 1 << 30 or k_pages.shape[1] > 32767:
        raise ValueError(f"{n} rows of {k_pages.shape[1]} heads are more than the kernel counts")
    return bytes(_rows_args(table, page, k_pages.shape[0], k_pages.shape[1], dim, n))


def read_rows_int4(k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, n: int, dim: int, dtype: torch.dtype) -> Tuple[torch.Tensor, torch.Tensor]:
    """The first ``n`` rows of every request, keys and values ``[B, n, heads, dim]`` in ``dtype``; rows behind a request's length are zeros."""
    if not k_pages.is_cuda:
        _read_plan(k_pages, v_pages, table, lengths, n, dim, dtype)
        return R.read_rows(k_pages, v_pages, table, lengths, n, dim, dtype)
    from . import cuda as K
    plan = _planned(("read", _key(k_pages), _key(v_pages), _key(table), _key(lengths), n, dim, dtype, (k_pages.data_ptr() | v_pages.data_ptr()) % 16),
                    lambda: _read_plan(k_pages, v_pages, table, lengths, n, dim, dtype))
    shape = (table.shape[0], n, k_pages.shape[1], dim)
    k, v = torch.empty(shape, dtype=dtype, device=k_pages.device), torch.empty(shape, dtype=dtype, device=k_pages.device)
    if k.numel() == 0:
        return k, v
    table, lengths = _flat(table), _flat(lengths)
    a = _Rows.from_buffer_copy(plan)
    a.table_ld = table.stride(0)
    a.x[0], a.x[1], a.pool[0], a.pool[1] = k.data_ptr(), v.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr()
    a.table, a.lengths, a.err = table.data_ptr(), lengths.data_ptr(), K.error_word(k_pages.device)
    with on_device(k_pages):
        K._check(K.lib().lmoe_int4_rows(ctypes.byref(a), _TYPES[dtype], 1, K._st()), "int4_read")
    return k, v


# ---- attention of one token -------------------------------------------------------------------------------------------------------
HEADS, MAX_CLUSTER, MIN_GROUPS = 8, 8, 8                  # csrc/int4_step.cu, .cuh


def splits_of(B: int, G: int, heads: int, D: int, keys: int) -> Tuple[int, int]:
    """(CTAs that share a key head of a request of up to ``keys`` keys, are the longest requests to come first).

    One wave: as many parts as give every slot of the GPU a CTA, of 128 keys at least (300 keys in three parts 8.3 us, in one 10.3, replayed).  Two of up to 100001 keys, 2 heads of 64: 77 us in 16 parts, 43 in 32, 25 in
    111, 23 in 148.  Requests that fill more than half of the slots by themselves, but not four waves, go in two parts each, the longest ones first (64 of up to 8192 keys, 8 heads of 128: 113 us, in one part each 156, in four 130; in
    two unsorted 144).  The host knows how many pages a request's table has, not how long the request is: a short one with a wide table has parts without keys, and a second launch where there are more than eight."""
    from . import cuda as K
    work, slots = max(1, B * G * -(-heads // HEADS)), 4 * K.num_sms()
    n = slots // work if 2 * work <= slots else 2 if work < 4 * slots else 1
    n = min(n, -(-keys // (GROUP * MIN_GROUPS)))
    n = MAX_CLUSTER if MAX_CLUSTER < n < 16 else max(n, 1)
    return n, int(1 < B <= 128 and work * n > slots)


def _step_plan(q, k_pages, v_pages, table, lengths, scale, window, softcap, slopes):
    """(Arguments without their addresses, floats of the parts' outputs and of their maxima and sums; on the tensor cores?)"""
    if q.dim() != 3 or q.dtype not in _TYPES or q.device != k_pages.device:
        raise ValueError("queries are [B, H, D] in fp32, bf16 or fp16, where the pools lie")
    B, H, D = q.shape
    page = _check_pools(k_pages, v_pages, table, lengths, B, None, D)
    G = k_pages.shape[1]
    if G == 0 or H % G:
        raise ValueError(f"{H} query heads do not share {G} key/value heads evenly")
    if window is not None and window < 1:
        raise ValueError(f"a window of {window}")
    _check_scores(q, H, scale, softcap, slopes)
    a = _Step(q_b=q.stride(0), q_h=q.stride(1), table_ld=table.stride(0), B=B, H=H, G=G, D=D, page=page, pages=k_pages.shape[0], table_n=table.shape[1],
              window=min(int(window or 0), (1 << 31) - 1), splits=1, sorted=0, scale=float(scale) if scale is not None else D ** -0.5, cap=float(softcap or 0.0))
    tensor = q.dtype != torch.float32 and D <= 128 and G * -(-(H // G) // HEADS) <= 65535
    part = 0
    if tensor and q.is_cuda:
        a.splits, a.sorted = splits_of(B, G, H // G, D, table.shape[1] * page)
        part = B * H * a.splits * D if a.splits > MAX_CLUSTER else 0
    return bytes(a), part, tensor, a.splits


def paged_attention_int4(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, scale: Optional[float] = None, window: Optional[int] = None, *,
                         softcap: Optional[float] = None, slopes: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``[B, H, D]``: ``ops.paged_attention`` over pools of 4 bits a number, into which the new token's row has been stored (:func:`store_rows_int4`).  Forward only.

    On CUDA 16-bit queries of up to 128 numbers a head run on the tensor cores: sums in 32 bits, weights times the sizes of values to 22 bits and times their lows to 16 (the error against 64 bits is that of 32-bit
    arithmetic and one rounding), queries but for what is below 2^-35 of a head's largest number.  Others are computed in 32 bits throughout by a simpler kernel (64 requests of up to 8192 keys, 32 over 8 heads of 128:
    111 us and, with queries in fp32, 4990)."""
    if torch.is_grad_enabled() and q.requires_grad:
        raise ValueError("one-token attention has no backward pass: use ops.softmax_attention")
    if not q.is_cuda:
        _step_plan(q, k_pages, v_pages, table, lengths, scale, window, softcap, slopes)
        return R.paged_attention(q, k_pages, v_pages, table, lengths, scale, window, softcap, slopes)
    from . import cuda as K
    plan, part, tensor, splits = _planned(("step", _key(q), _key(k_pages), _key(v_pages), _key(table), _key(lengths), scale, window, softcap, _key(slopes), slopes is not None and slopes.requires_grad,
                     (k_pages.data_ptr() | v_pages.data_ptr()) % 16), lambda: _step_plan(q, k_pages, v_pages, table, lengths, scale, window, softcap, slopes))
    q, table, lengths = _flat(q), _flat(table), _flat(lengths)
    slopes = slopes if slopes is None else _flat(slopes)
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if out.numel() == 0:
        return out
    a = _Step.from_buffer_copy(plan)
    a.q_b, a.q_h, a.table_ld = q.stride(0), q.stride(1), table.stride(0)
    a.q_rows = int(q.stride(0) % 8 == 0 and q.stride(1) % 8 == 0 and q.data_ptr() % 16 == 0)
    a.q, a.k, a.v, a.out = q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), out.data_ptr()
    a.table, a.lengths, a.slopes, a.err = table.data_ptr(), lengths.data_ptr(), K._ptr(slopes), K.error_word(q.device)
    with on_device(q):
        if not tensor:
            K._check(K.lib().lmoe_int4_step_any(ctypes.byref(a), _TYPES[q.dtype], K._st()), "int4_step_any")
            return out
        if part:
            work = torch.empty(part + 2 * (part // q.shape[2]), dtype=torch.float32, device=q.device)
            a.part = work.data_ptr()
            a.ml = a.part + 4 * part
        K._check(K.lib().lmoe_int4_step(ctypes.byref(a), int(q.dtype == torch.float16), K._st()), "int4_step", 1 if splits <= MAX_CLUSTER else 2)
    return out
