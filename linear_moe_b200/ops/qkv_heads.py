"""Queries, keys and values out of a fused projection, normed and turned in one pass (``csrc/qkv_heads.cu``; CPU tensors run the eager definition).

    y = w x / sqrt(mean x^2 + eps)   per query and key head,   (a, b) -> (a cos - b sin, a sin + b cos)   over the pairs of its first R numbers

A token's row of the projection holds, group by group, the r query heads that share a key head, the key and the value: ``[B, T, G, r + 2, D]``.  The cosines and sines come from tables in fp32
``[tokens, R / 2]``, whose row is a token's place in its sequence or what ``positions [B, T]`` says (on the device, so captured steps go on).  Everything between the projection and the results is
computed in 32 bits and rounded once.  The backward pass gives the projection's gradient in one tensor and those of the norms' weights, summed in an order that the sizes alone decide.  (On CUDA
there are no second derivatives and no forward mode: both raise.)

A position outside the tables raises on the CPU; on CUDA it sets the kernels' error word (``ops.gemm.check_error``) and the nearest row is taken."""
from __future__ import annotations

import ctypes
from typing import Dict, Optional

import torch

from ..ref import ops as R
from .scored_attn import on_device


class _Args(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p) for n in ("x", "wq", "wk", "q", "k", "v", "cos", "sin", "at", "dq", "dk", "dv", "dx", "dwq", "dwk", "part")] +
                [(n, ctypes.c_longlong) for n in ("x_b", "x_t", "rows")] +
                [(n, ctypes.c_int) for n in ("T", "G", "r", "D", "R", "tokens", "interleaved", "at_wide", "w_type", "parts")] + [("div", ctypes.c_uint * 8)] + [(n, ctypes.c_int) for n in ("vectors", "parts_q", "parts_k")] +
                [("eps", ctypes.c_float), ("err", ctypes.c_void_p)])


_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MOST = 1024                               # numbers of a head


def _check(qkv, q_weight, k_weight, eps, cos, sin, positions):
    if qkv.dim() != 5 or qkv.shape[3] < 3:
        raise ValueError("a projection is [B, T, groups, query heads + key + value, D]")
    if qkv.dtype not in _TYPES:
        raise ValueError("a projection in fp32, bf16 or fp16")
    B, T, G, S, D = qkv.shape
    if not 1 <= D <= MOST:
        raise ValueError(f"heads of {D} numbers (up to {MOST})")
    for w in (q_weight, k_weight):
        if w is not None and (w.shape != (D,) or w.dtype not in _TYPES or w.device != qkv.device):
            raise ValueError(f"a norm's weight is [{D}], in fp32, bf16 or fp16, where the projection lies")
    if q_weight is not None and k_weight is not None and q_weight.dtype != k_weight.dtype:
        raise ValueError("the norms' weights have one type")
    if not eps >= 0:
        raise ValueError(f"an epsilon of {eps}")
    if (cos is None) != (sin is None):
        raise ValueError("cosines and sines come together")
    if cos is None:
        if positions is not None:
            raise ValueError("positions without tables")
        return
    if cos.dim() != 2 or cos.shape != sin.shape or cos.dtype != torch.float32 or sin.dtype != torch.float32 or 2 * cos.shape[1] > D:
        raise ValueError(f"the tables are fp32 [tokens, R / 2] with R up to {D}")
    if cos.requires_grad or sin.requires_grad:
        raise ValueError("the tables get no gradient")
    if any(t is not None and t.device != qkv.device for t in (cos, sin, positions)):
        raise ValueError("the tensors lie on one device")
    if positions is None and cos.shape[0] < T:
        raise ValueError(f"tables of {cos.shape[0]} rows for {T} tokens")
    if positions is not None and (positions.shape != (B, T) or positions.dtype not in (torch.int32, torch.int64)):
        raise ValueError(f"positions are int32 or int64 [{B}, {T}]")
    if cos.shape[0] >= 1 << 31 or (cos.shape[0] == 0 and B * T > 0):
        raise ValueError(f"tables of {cos.shape[0]} rows")


def _key(t: Optional[torch.Tensor]):
    return t if t is None else (t.shape, t.stride(), t.dtype, t.device)


class _Plan:
    """What follows from shapes, strides and types alone: the arguments without their addresses, forward and backward."""
    __slots__ = ("forward", "backward", "type", "vectors", "rows", "parts", "shapes")


_PLANS: Dict[tuple, _Plan] = {}


def _plan(qkv, q_weight, k_weight, eps, cos, sin, positions, interleaved) -> _Plan:
    from . import cuda as K
    _check(qkv, q_weight, k_weight, eps, cos, sin, positions)
    B, T, G, S, D = qkv.shape
    w = q_weight if q_weight is not None else k_weight
    a = _Args(x_b=qkv.stride(0), x_t=qkv.stride(1), rows=B * T, T=T, G=G, r=S - 2, D=D, R=0 if cos is None else 2 * cos.shape[1], tokens=0 if cos is None else cos.shape[0],
              interleaved=int(interleaved), at_wide=int(positions is not None and positions.dtype == torch.int64), w_type=0 if w is None else _TYPES[w.dtype], parts=0, eps=eps)
    for i, d in enumerate((a.G * a.r, a.G, a.r, a.T)):
        a.div[2 * i:2 * i + 2] = _divisor(max(d, 1))
    p, size = _Plan(), qkv.element_size()
    p.type, p.shapes = _TYPES[qkv.dtype], ((B, T, G * (S - 2), D), (B, T, G, D))
    # Heads that divide into 16 bytes a thread; what does not lie on 16-byte boundaries is copied for them, so that the result is the same wherever a tensor lies.
    e = 16 // size
    p.vectors = a.D % (2 * e) == 0 and a.D <= 64 * e and a.R % (2 * e) == 0 and a.rows * a.G * a.r < 1 << 31
    p.rows = not p.vectors or all(s * size % 16 == 0 for s in qkv.stride()[:2])
    a.vectors = int(p.vectors)
    if p.vectors:
        _blocks(a, size, 4 * K.num_sms())
    p.forward = bytes(a)
    if p.vectors:
        _blocks(a, size, 2 * K.num_sms())
        p.parts = a.parts_q + a.parts_k
    else:
        a.parts = max(1, min(-(-a.rows * a.G * S // 8), 8 * K.num_sms()))
        p.parts = 2 * a.parts
    p.backward = bytes(a)
    return p


def _blocks(a: _Args, size: int, most: int):
    """Blocks of the vectors' kernels: of queries, keys and values by their number, up to what the GPU holds at once (four per SM forward, two backward)."""
    threads = 4
    while threads * 2 * (16 // size) < a.D:
        threads *= 2
    share = max(1, min(-(-a.rows * a.G * threads // 256), most // (a.r + 2)))
    a.parts_k, a.parts_q = share, max(1, min(-(-a.rows * a.G * a.r * threads // 256), most - 2 * share))
    a.parts = a.parts_q + 2 * share


def _divisor(d: int):
    """Multiplier and shift of a division by d (``over`` in csrc/qkv_heads.cu): floor(2^32 (2^s - d) / d) + 1 with s = ceil(log2 d)."""
    s = (d - 1).bit_length()
    return (((1 << s) - d << 32) // d + 1) & 0xffffffff, s


def _dense_heads(t: torch.Tensor) -> bool:
    """Are a token's heads one dense block?"""
    return t[0, 0].is_contiguous() if t.numel() else True


def _forward(qkv, wq, wk, plan, cos, sin, at):
    from . import cuda as K
    dev, dt = qkv.device, qkv.dtype
    heads, keys = plan.shapes
    q, k, v = torch.empty(heads, dtype=dt, device=dev), torch.empty(keys, dtype=dt, device=dev), torch.empty(keys, dtype=dt, device=dev)
    a = _Args.from_buffer_copy(plan.forward)
    a.x, a.q, a.k, a.v, a.err = qkv.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), K.error_word(dev)
    _inputs(a, wq, wk, cos, sin, at)
    with on_device(qkv):
        K._check(K.lib().lmoe_qkv_heads(ctypes.byref(a), plan.type, 0, K._st()), "qkv_heads")
    return q, k, v


def _inputs(a: _Args, wq, wk, cos, sin, at):
    if wq is not None:
        a.wq = wq.data_ptr()
    if wk is not None:
        a.wk = wk.data_ptr()
    if cos is not None:
        a.cos, a.sin = cos.data_ptr(), sin.data_ptr()
        if at is not None:
            a.at = at.data_ptr()


class _QkvHeads(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, wq, wk, plan, cos, sin, at):
        ctx.save_for_backward(qkv, wq, wk, cos, sin, at)
        ctx.plan = plan
        ctx.set_materialize_grads(False)
        return _forward(qkv, wq, wk, plan, cos, sin, at)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq, dk, dv):
        from . import cuda as K
        qkv, wq, wk, cos, sin, at = ctx.saved_tensors
        dev, plan = qkv.device, ctx.plan
        a = _Args.from_buffer_copy(plan.backward)
        grads = [g if g is None or (g.is_contiguous() and not (plan.vectors and g.data_ptr() % 16)) else g.clone(memory_format=torch.contiguous_format) for g in (dq, dk, dv)]
        a.dq, a.dk, a.dv = (K._ptr(g) for g in grads)
        dx = torch.empty(qkv.shape, dtype=qkv.dtype, device=dev)
        dws = [torch.empty_like(w) if w is not None and need else None for w, need in zip((wq, wk), ctx.needs_input_grad[1:3])]
        a.x, a.dx, a.dwq, a.dwk, a.err = qkv.data_ptr(), dx.data_ptr(), K._ptr(dws[0]), K._ptr(dws[1]), K.error_word(dev)
        _inputs(a, wq, wk, cos, sin, at)
        work = None
        if dws[0] is not None or dws[1] is not None:
            work = torch.empty(plan.parts * a.D, dtype=torch.float32, device=dev)
            a.part = work.data_ptr()
        with on_device(qkv):
            K._check(K.lib().lmoe_qkv_heads(ctypes.byref(a), plan.type, 1, K._st()), "qkv_heads backward", 1 if work is None else 2)
        return (dx, *dws, None, None, None, None)


def qkv_heads(qkv: torch.Tensor, q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6, cos: Optional[torch.Tensor] = None,
              sin: Optional[torch.Tensor] = None, *, positions: Optional[torch.Tensor] = None, interleaved: bool = False):
    """``qkv [B, T, G, r + 2, D]`` -> ``(q [B, T, G r, D], k [B, T, G, D], v [B, T, G, D])``; see the module.  A head without a weight is not normed, without tables nothing is turned."""
    if not qkv.is_cuda:
        _check(qkv, q_weight, k_weight, eps, cos, sin, positions)
        return R.qkv_heads(qkv, q_weight, k_weight, eps, cos, sin, positions, interleaved)
    # the host's share of a short call is as long as the kernels: checks, strides and the launch's shape are worked out once per layout
    key = (_key(qkv), _key(q_weight), _key(k_weight), eps, _key(cos), _key(sin), _key(positions), interleaved, cos is not None and (cos.requires_grad or sin.requires_grad))
    plan = _PLANS.get(key)
    if plan is None:
        if len(_PLANS) >= 4096:
            _PLANS.clear()
        if not all(t is None or t.is_contiguous() for t in (q_weight, k_weight, cos, sin, positions)) or not _dense_heads(qkv):
            _check(qkv, q_weight, k_weight, eps, cos, sin, positions)
            flat = lambda t: t if t is None else t.contiguous()      # noqa: E731
            return qkv_heads(qkv if _dense_heads(qkv) else qkv.contiguous(), flat(q_weight), flat(k_weight), eps, flat(cos), flat(sin), positions=flat(positions), interleaved=interleaved)
        plan = _PLANS[key] = _plan(qkv, q_weight, k_weight, eps, cos, sin, positions, interleaved)
    if qkv.numel() == 0:
        return R.qkv_heads(qkv, q_weight, k_weight, eps, cos, sin, positions, interleaved)
    if plan.vectors and (not plan.rows or (qkv.data_ptr() | (0 if cos is None else cos.data_ptr() | sin.data_ptr())) % 16):
        qkv = qkv if plan.rows and not qkv.data_ptr() % 16 else qkv.clone(memory_format=torch.contiguous_format)
        cos, sin = (t if t is None or not t.data_ptr() % 16 else t.clone() for t in (cos, sin))
        return qkv_heads(qkv, q_weight, k_weight, eps, cos, sin, positions=positions, interleaved=interleaved)
    from . import cuda as K
    if K._unwatched() and (not torch.is_grad_enabled() or not (qkv.requires_grad or (q_weight is not None and q_weight.requires_grad) or (k_weight is not None and k_weight.requires_grad))):
        return _forward(qkv, q_weight, k_weight, plan, cos, sin, positions)
    return _QkvHeads.apply(qkv, q_weight, k_weight, plan, cos, sin, positions)
