"""Softmax attention with capped scores, a bias by distance and a range of visible keys per query.

    x_ij = cap tanh(scale q_i k_j / cap) - slope_h |p_i - j|        p_i = q_offset + i
    o_i  = sum_j softmax_j(x_ij) v_j   over the keys  key_first_i <= j < key_stop_i  that causality and the window leave too

A query that sees no key gives zeros and passes no gradient.  One interval per query describes packed documents
(:func:`document_first`), prefixes that see themselves whole and padded batches (:func:`prefix_stop`).

bf16 and fp16 CUDA tensors with heads of up to 128, in multiples of 8, run the tcgen05 kernels of ``csrc/flash_attn_scored.cuh``; others (fp32, CPU,
wider heads, more than 2^20 queries or 1023 query heads) run the eager definition :func:`linear_moe_b200.ref.ops.softmax_attention`.  Slopes and ranges get no gradient.  Hidden keys and
values have to be finite, as for the eager form: a weight of zero times NaN is NaN.
"""
from __future__ import annotations

import contextlib
import ctypes
from typing import Dict, Optional, Sequence

import torch

from ..ref import ops as R

MAX_QUERIES, MAX_HEADS = 1 << 20, 1023        # what the dk / dv kernel's list of query tiles holds; heads for which a sequence's rows stay below 2^31


def on_device(t: torch.Tensor):
    """Launches go to the current device's stream: makes it the tensor's device."""
    return contextlib.nullcontext() if t.device.index == torch.cuda.current_device() else torch.cuda.device(t.device)


# ---- ranges ---------------------------------------------------------------------------------------------------------------------
def document_first(tokens: torch.Tensor, end_token: int) -> torch.Tensor:
    """First token of every position's document, int32 ``[B, T]``, where ``end_token`` closes a document (its own position belongs to the
    document that it ends): ``key_first`` of causal attention inside documents."""
    T = tokens.shape[-1]
    at = torch.arange(T, device=tokens.device, dtype=torch.int32)
    starts = torch.where(tokens == end_token, at + 1, torch.zeros_like(at))
    first = torch.cummax(starts, dim=-1).values
    return torch.cat([torch.zeros_like(first[..., :1]), first[..., :-1]], dim=-1).contiguous()


def prefix_stop(T: int, prefix: Sequence[int], lengths: Optional[Sequence[int]] = None, device=None) -> torch.Tensor:
    """Key behind the last visible one, int32 ``[B, T]``, for sequences whose first ``prefix[b]`` tokens see one another and whose later tokens
    are causal (``causal=False``, the range says it all).  Positions from ``lengths[b]`` on are padding: they see nothing and nobody sees
    them."""
    at = torch.arange(T, device=device, dtype=torch.int32)[None]
    p = torch.as_tensor(prefix, dtype=torch.int32, device=device)[:, None]
    stop = torch.maximum(at + 1, p)
    if lengths is not None:
        n = torch.as_tensor(lengths, dtype=torch.int32, device=device)[:, None]
        stop = torch.where(at < n, torch.minimum(stop, n), torch.zeros_like(stop))
    return stop.contiguous()


def alibi_slopes(heads: int) -> torch.Tensor:
    """Slopes of the distance bias, fp32 ``[heads]`` (Press et al., "Train Short, Test Long"): a geometric series from 2^(-8/n) on for n heads, a power of two; other
    numbers of heads take the series of the next lower power and every second slope of the next higher one's."""
    n = 1 << (heads.bit_length() - 1)
    s = [2.0 ** (-8.0 * (i + 1) / n) for i in range(n)] + [2.0 ** (-8.0 * (i + 1) / (2 * n)) for i in range(0, 2 * n, 2)]
    return torch.tensor(s[:heads], dtype=torch.float32)


def _check_options(q, k, v, scale, causal, q_offset, window, softcap, slopes, key_first, key_stop):
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("attention takes q [B, Tq, Hq, D], k and v [B, Tk, Hkv, D]")
    if k.shape[:3] != v.shape[:3] or k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3]:
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not go together")
    if k.shape[2] == 0 or q.shape[2] % k.shape[2]:
        raise ValueError(f"{q.shape[2]} query heads do not share {k.shape[2]} key/value heads evenly")
    if not q.dtype == k.dtype == v.dtype or not q.device == k.device == v.device:
        raise ValueError("q, k and v have one type and lie on one device")
    _check_scores(q, q.shape[2], scale, softcap, slopes)
    if window is not None and not (causal and window >= 1):
        raise ValueError("a window is a positive number of keys of causal attention")
    if not abs(q_offset) < 1 << 30 or max(q.shape[1], k.shape[1]) >= 1 << 30:
        raise ValueError(f"positions beyond 2^30: {q.shape[1]} queries from {q_offset} on, {k.shape[1]} keys")
    for name, r in (("key_first", key_first), ("key_stop", key_stop)):
        if r is None:
            continue
        if r.dtype != torch.int32 or r.shape != q.shape[:2] or r.device != q.device:
            raise ValueError(f"{name} is an int32 tensor [B, Tq] = {tuple(q.shape[:2])} on {q.device}")


def _check_scores(q, heads, scale, softcap, slopes):
    if scale is not None and not 1e-30 < scale < 1e30:           # what fp32 holds, and its quotient with a cap
        raise ValueError(f"scale {scale}")
    if softcap is not None and not 1e-7 < softcap < 1e7:
        raise ValueError(f"soft cap {softcap}")
    if slopes is not None and (slopes.dtype != torch.float32 or slopes.shape != (heads,) or slopes.device != q.device or slopes.requires_grad):
        raise ValueError(f"slopes are {heads} fp32 numbers on {q.device} without a gradient, one per query head")


# ---- binding --------------------------------------------------------------------------------------------------------------------
class _Ranges(ctypes.Structure):
    _fields_ = ([("first", ctypes.c_void_p), ("stop", ctypes.c_void_p), ("first_b", ctypes.c_longlong), ("stop_b", ctypes.c_longlong)] +
                [("slopes", ctypes.c_void_p), ("low", ctypes.c_void_p), ("tiles", ctypes.c_void_p), ("cap", ctypes.c_float), ("causal", ctypes.c_int), ("d", ctypes.c_int)])


_SIZES = [(n, ctypes.c_int) for n in ("B", "Tq", "Tk", "Hq", "Hkv", "q_offset", "window")] + [("scale", ctypes.c_float), ("err", ctypes.c_void_p), ("x", _Ranges)]


class _Args(ctypes.Structure):
    _fields_ = [("out", ctypes.c_void_p), ("lse", ctypes.c_void_p)] + _SIZES


class _BwdArgs(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("lse", "delta", "dq", "dk", "dv")] + _SIZES


def _strides(t: torch.Tensor):
    """Element strides (batch, token, head) of a tensor that a tensor map can describe, or None.  The stride of a dimension of one is
    never used, whatever the tensor says: it gets the one of a dense tensor."""
    if t.stride(3) != 1:
        return None
    out, dense = [0, 0, 0], t.shape[3]
    for i in (2, 1, 0):
        s = t.stride(i) if t.shape[i] > 1 else dense
        if s <= 0 or s % 8 or s >= 1 << 38:
            return None
        out[i], dense = s, dense * t.shape[i]
    return (ctypes.c_longlong * 3)(*out)


def _laid_out(t: torch.Tensor) -> torch.Tensor:
    """The tensor, or a dense copy where no tensor map can describe it."""
    return t if _strides(t) is not None and t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


class _Plan:
    """What follows from shapes, strides, types and options alone: the arguments without their addresses."""
    __slots__ = ("eager", "args", "bwd", "qs", "ks", "vs", "ranges", "lse", "tiles", "low", "fwd_fn", "bwd_fn", "copy")


_PLANS: Dict[tuple, _Plan] = {}


def _plan(q, k, v, scale, causal, q_offset, window, softcap, slopes, first, stop) -> _Plan:
    from . import cuda as K
    _check_options(q, k, v, scale, causal, q_offset, window, softcap, slopes, first, stop)
    p, (B, Tq, Hq, D) = _Plan(), q.shape
    p.eager = (not q.is_cuda or q.dtype not in (torch.bfloat16, torch.float16) or v.shape[3] != D or D > 128 or D % 8 != 0 or Tq > MAX_QUERIES or Hq > MAX_HEADS
               or min(q.numel(), k.numel()) == 0)
    if p.eager:
        return p
    p.qs, p.ks, p.vs = _strides(q), _strides(k), _strides(v)
    p.ranges = all(r is None or r.stride(-1) == 1 or r.shape[-1] == 1 for r in (first, stop, slopes))
    p.copy = None in (p.qs, p.ks, p.vs) or not p.ranges
    fwd, bwd = _Args(), _BwdArgs()
    for a in (fwd, bwd):
        a.B, a.Tq, a.Hq, a.Tk, a.Hkv = B, Tq, Hq, k.shape[1], k.shape[2]
        a.q_offset, a.window, a.scale = int(q_offset), min(int(window or 0), (1 << 31) - 1), float(scale) if scale is not None else D ** -0.5
        a.x.cap, a.x.causal, a.x.d = float(softcap or 0.0), int(bool(causal)), D
        a.x.first_b, a.x.stop_b = (0 if r is None else r.stride(0) for r in (first, stop))
    p.args, p.bwd = bytes(fwd), bytes(bwd)
    p.lse, p.tiles, p.low = B * Hq * Tq * 4, B * -(-Tq // 128) * 16, B * Tq * Hq * _round16(D)      # bytes
    half = q.dtype == torch.float16
    p.fwd_fn = K.lib().lmoe_scored_attn_fwd_fp16 if half else K.lib().lmoe_scored_attn_fwd
    p.bwd_fn = K.lib().lmoe_scored_attn_bwd_fp16 if half else K.lib().lmoe_scored_attn_bwd
    return p


def _addresses(a, dev, first, stop, slopes, stats: int, low: int, tiles: int):
    """What a launch reads beside q, k and v: ranges, slopes, and the forward kernel's notes (row statistics, next bits of the output, intervals of the query tiles)."""
    from . import cuda as K
    x = a.x
    if first is not None:
        x.first = first.data_ptr()
    if stop is not None:
        x.stop = stop.data_ptr()
    if slopes is not None:
        x.slopes = slopes.data_ptr()
    a.lse, x.low, x.tiles, a.err = stats, low, tiles, K.error_word(dev)


def _round16(n: int) -> int:
    return (n + 15) & ~15


class ScoredAttention(torch.autograd.Function):
    """q, k and v as tensor maps take them (``_Plan.copy`` is false, bases on 16-byte boundaries)."""

    @staticmethod
    def forward(ctx, q, k, v, first, stop, slopes, p):
        from . import cuda as K
        dev = q.device
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
        train = any(ctx.needs_input_grad[:3])
        at_tiles = _round16(p.lse)
        at_low = at_tiles + p.tiles
        notes = torch.empty(at_low + (p.low if train else 0), dtype=torch.uint8, device=dev)
        base = notes.data_ptr()
        a = _Args.from_buffer_copy(p.args)
        a.out = out.data_ptr()
        _addresses(a, dev, first, stop, slopes, base, base + at_low if train else 0, base + at_tiles)
        with on_device(q):
            K._check(p.fwd_fn(K._p(q), p.qs, K._p(k), p.ks, K._p(v), p.vs, ctypes.byref(a), K._st()), "scored_attn_fwd")
        if train:
            ctx.save_for_backward(q, k, v, first, stop, slopes, out, notes)
            ctx.plan = p
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_out):
        from . import cuda as K
        q, k, v, first, stop, slopes, out, notes = ctx.saved_tensors
        p, dev = ctx.plan, q.device
        d_out = d_out.contiguous()
        if d_out.data_ptr() % 16:
            d_out = d_out.clone()
        dq = torch.empty_like(out)
        dk, dv = torch.empty(k.shape, dtype=k.dtype, device=dev), torch.empty(k.shape, dtype=k.dtype, device=dev)
        delta = torch.empty(p.lse, dtype=torch.uint8, device=dev)
        base, at_tiles = notes.data_ptr(), _round16(p.lse)
        a = _BwdArgs.from_buffer_copy(p.bwd)
        a.dq, a.dk, a.dv = dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
        _addresses(a, dev, first, stop, slopes, base, base + at_tiles + p.tiles, base + at_tiles)
        with on_device(q):
            K._check(p.bwd_fn(K._p(q), p.qs, K._p(k), p.ks, K._p(v), p.vs, K._p(out), K._p(d_out), K._p(delta), ctypes.byref(a), K._st()), "scored_attn_bwd", 3)
        return dq, dk, dv, None, None, None, None


def _meta(t):
    return None if t is None else (t.shape, t.stride(), t.dtype, t.device, t.requires_grad)


def scored_attention(q, k, v, scale=None, causal: bool = True, q_offset: int = 0, window: Optional[int] = None, softcap: Optional[float] = None,
                     slopes: Optional[torch.Tensor] = None, key_first: Optional[torch.Tensor] = None, key_stop: Optional[torch.Tensor] = None):
    """See the module; what ``ops.softmax_attention`` calls when it is given one of the last four."""
    # checks, strides and sizes are worked out once per layout
    key = (q.shape, q.stride(), q.dtype, q.device, k.shape, k.stride(), k.dtype, k.device, v.shape, v.stride(), v.dtype, v.device, scale, causal, q_offset, window, softcap,
           _meta(slopes), _meta(key_first), _meta(key_stop))
    p = _PLANS.get(key)
    if p is None:
        p = _plan(q, k, v, scale, causal, q_offset, window, softcap, slopes, key_first, key_stop)
        if len(_PLANS) >= 4096:
            _PLANS.clear()
        _PLANS[key] = p
    if p.eager:
        return R.softmax_attention(q, k, v, scale, causal, q_offset, window, softcap, slopes, key_first, key_stop)
    if p.copy or (q.data_ptr() | k.data_ptr() | v.data_ptr()) % 16:
        row = lambda r: None if r is None else r.contiguous()       # noqa: E731
        return scored_attention(_laid_out(q), _laid_out(k), _laid_out(v), scale, causal, q_offset, window, softcap, row(slopes), row(key_first), row(key_stop))
    return ScoredAttention.apply(q, k, v, key_first, key_stop, slopes, p)
