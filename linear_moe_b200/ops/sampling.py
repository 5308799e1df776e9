"""The next token of every request out of its logits and one random number (``csrc/sample.cu``; CPU tensors run the eager form).

    w_i = exp((x_i - max x) / temperature)

Tokens are put in the order of falling logits, equal ones by their number.  A token is kept while fewer than ``top_k`` come before it, while the weight of those before it is below ``top_p`` of the whole, and
if ``w_i >= min_p``; the first one always is.  The token drawn is the first one, in the order of the vocabulary, up to which the kept weights exceed ``draw`` times their sum.  Given the random numbers, the result is
a function of the logits: sums are exact in units of 2^-44 of the largest weight (weights below half of that are never drawn), so it does not depend on how a row is shared out.  (More than 2^19 logits, which the
eager form takes on CUDA too: in units of 2^-43, one bit less for every doubling, so that the sums stay within 2^63.)

NaN logits count as minus infinity; tokens at plus infinity share the whole weight.  A row of nothing but minus infinity gives token 0 and a log-probability of minus infinity.  A temperature that is not
above zero takes the largest logit; ``top_k`` below 1 and ``top_p`` of 1 or more cut nothing off, nor do a ``top_p`` and a ``min_p`` of NaN in a tensor."""
from __future__ import annotations

import ctypes
from typing import Dict, Tuple, Union

import torch

from .scored_attn import on_device

MOST, PART = 1 << 19, 1 << 16                              # logits of a row, and of a CTA (csrc/sample.cu)
_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
Setting = Union[int, float, torch.Tensor]


class _Args(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p) for n in ("logits", "draw", "temperature", "top_p", "min_p", "top_k", "token", "logp")] + [("ld", ctypes.c_longlong)] +
                [(n, ctypes.c_int) for n in ("B", "V", "parts", "len", "k")] + [(n, ctypes.c_float) for n in ("t", "p", "least")])


def _check(logits, draw, temperature, top_k, top_p, min_p):
    if logits.dim() != 2 or logits.dtype not in _TYPES or logits.shape[1] == 0:
        raise ValueError("sampling takes logits [B, V] in fp32, bf16 or fp16")
    B = logits.shape[0]
    if draw.shape != (B,) or draw.dtype != torch.float32 or draw.device != logits.device:
        raise ValueError(f"the random numbers are fp32 [{B}], where the logits lie")
    for name, x, dtype, good in (("temperature", temperature, torch.float32, lambda v: v >= 0), ("top_k", top_k, torch.int32, lambda v: v >= 0 and v == int(v)),
                                 ("top_p", top_p, torch.float32, lambda v: v >= 0), ("min_p", min_p, torch.float32, lambda v: 0 <= v <= 1)):
        if torch.is_tensor(x):
            if x.shape != (B,) or x.dtype != dtype or x.device != logits.device:
                raise ValueError(f"{name} is a number or {dtype} [{B}], where the logits lie")
        elif not good(x):
            raise ValueError(f"{name} of {x}")


def _eager(logits, draw, temperature, top_k, top_p, min_p):
    B, V = logits.shape
    dev = logits.device

    def setting(x):
        return (x if torch.is_tensor(x) else torch.full((B,), float(x), dtype=torch.float32, device=dev))[:, None].double()
    t, k, p, least = (setting(x) for x in (temperature, top_k, top_p, min_p))
    p = torch.nan_to_num(p, nan=1.0)
    x = torch.nan_to_num(logits.double(), nan=float("-inf"), posinf=float("inf"), neginf=float("-inf"))
    x, order = torch.sort(x, dim=-1, descending=True, stable=True)
    top = x[:, :1]
    greedy = ~(t > 0)
    y = torch.where(x == top, 0.0, (x - top) / torch.where(greedy, 1.0, t))
    unit = 2.0 ** min(44, 63 - (V - 1).bit_length())                                        # V of them: 2^63 at most
    w = torch.where((x == float("-inf")) | y.isnan(), 0.0, (y.exp() * unit).round()).to(torch.int64)               # (NaN: minus infinity over an endless temperature)
    before, whole, _ = _sums(w)
    limit = (torch.where(p >= 1, 0.0, p) * whole).ceil().clamp_min(1).to(torch.int64)
    keep = (torch.arange(V, device=dev) < torch.where(greedy, 1, torch.where(k >= 1, k, V))) & ((before < limit) | (p >= 1))
    keep &= (w >= (torch.nan_to_num(least, nan=0.0).clamp(0, 1) * unit).ceil().to(torch.int64)) | (x == top)
    kept = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, 0))
    before, whole, last = _sums(kept)
    u = torch.nan_to_num(draw, nan=0.0).clamp_min(0)[:, None].double()
    goal = torch.where(u < 1, torch.minimum((u * whole).to(torch.int64), last), last)
    some = last[:, 0] >= 0
    token = torch.where(some, (before <= goal).sum(-1) - 1, 0)                               # the last one that the goal reaches
    share = kept.gather(1, token[:, None]).double() / whole
    return token, torch.where(some, share[:, 0].log(), float("-inf")).float()


def _sums(w):
    """What comes before every weight, the whole as a 64-bit number, and the whole less one: 2^63 itself 63 bits do not hold."""
    before = torch.nn.functional.pad(w[:, :-1].cumsum(-1), (1, 0))
    last = before[:, -1:] + (w[:, -1:] - 1)
    return before, (last.clamp_max((1 << 63) - 2) + 1).double(), last


def _shares(V: int) -> Tuple[int, int]:
    """(CTAs of a row, logits of each): as many as a cluster has, of 2048 logits at least (one row of 32000: 38 us in one part, 26 in two, 18 in four, 15 in eight; 128 rows of 128256 in fp32, top-p: 181 in two,
    175 in four, 149 in eight; nothing cut off: 90, 98, 86; 20 calls in a graph).  Full batches with a top-k alone would do better in four (bf16, the 50 largest: 121, 101, 119): the rule does not look at the settings, which may
    lie on the device."""
    parts = 1
    while parts < 8 and parts * 2048 < V:
        parts *= 2
    return parts, -(-V // (parts * 128)) * 128


def _key(x):
    return (x.shape, x.stride(), x.dtype, x.device) if isinstance(x, torch.Tensor) else x


class _Plan:
    """What follows from shapes, strides, types and the numbers among the settings: the arguments without their addresses."""
    __slots__ = ("args", "type", "flat", "tensors")


_PLANS: Dict[tuple, _Plan] = {}


def _plan(logits, draw, temperature, top_k, top_p, min_p) -> _Plan:
    _check(logits, draw, temperature, top_k, top_p, min_p)
    B, V = logits.shape
    parts, length = _shares(V)
    settings = (temperature, top_k, top_p, min_p)
    t, k, share, least = (0 if isinstance(x, torch.Tensor) else x for x in settings)
    p = _Plan()
    p.args = bytes(_Args(ld=logits.stride(0), B=B, V=V, parts=parts, len=length, k=min(int(k), MOST), t=t, p=min(float(share), 2.0), least=least))
    p.type = _TYPES[logits.dtype]
    p.flat = all(not isinstance(x, torch.Tensor) or x.stride(-1) == 1 or x.shape[-1] <= 1 for x in (logits, draw, *settings))
    p.tensors = [(name, i) for i, (name, x) in enumerate(zip(("temperature", "top_k", "top_p", "min_p"), settings)) if isinstance(x, torch.Tensor)]
    return p


def sample_tokens(logits: torch.Tensor, draw: torch.Tensor, temperature: Setting = 1.0, top_k: Setting = 0, top_p: Setting = 1.0, min_p: Setting = 0.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """``logits [B, V]``, ``draw [B]`` fp32 in [0, 1): ``(token int64 [B], log-probability fp32 [B])``, the latter among the kept tokens.  Each setting is a number or a tensor with one for every
    request (``top_k`` int32, the others fp32).  No gradient."""
    if not logits.is_cuda or logits.shape[-1] > MOST or logits.shape[0] > 65535:
        _check(logits, draw, temperature, top_k, top_p, min_p)
        with torch.no_grad():
            return _eager(logits, draw, temperature, top_k, top_p, min_p)
    from . import cuda as K
    key = (_key(logits), _key(draw), _key(temperature), _key(top_k), _key(top_p), _key(min_p))
    plan = _PLANS.get(key)
    if plan is None:
        if len(_PLANS) >= 4096:
            _PLANS.clear()
        plan = _PLANS[key] = _plan(logits, draw, temperature, top_k, top_p, min_p)
    settings = (temperature, top_k, top_p, min_p)
    if not plan.flat:
        return sample_tokens(*(t.contiguous() if isinstance(t, torch.Tensor) and t.stride(-1) != 1 else t for t in (logits, draw, *settings)))
    B, dev = logits.shape[0], logits.device
    token, logp = torch.empty(B, dtype=torch.int64, device=dev), torch.empty(B, dtype=torch.float32, device=dev)
    if B == 0:
        return token, logp
    a = _Args.from_buffer_copy(plan.args)
    a.logits, a.draw, a.token, a.logp = logits.data_ptr(), draw.data_ptr(), token.data_ptr(), logp.data_ptr()
    for name, i in plan.tensors:
        setattr(a, name, settings[i].data_ptr())
    with on_device(logits):
        K._check(K.lib().lmoe_sample(ctypes.byref(a), plan.type, K._st()), "sample")
    return token, logp
