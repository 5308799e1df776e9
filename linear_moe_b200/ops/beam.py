"""One step of a beam search: the best continuations, and the beams' states in their new order (``csrc/beam.cu``; CPU tensors run the eager form).

:func:`beam_select` takes the best ``n`` of ``scores[b] + log_softmax(logits[b])[t]`` over beams and vocabulary of every prompt, ties to the lowest ``b V + t``.  Candidates of one beam
are compared by their logits; those of different beams by scores in 64 bits (rounded once for the result) whose log-sums are sums of 32-bit exponentials, some 1e-7 off: nearer ones can come in
either order on CUDA, equal rows with equal scores in the order of their beams.  NaN logits count as minus infinity.  :func:`reorder_states` gives the rows ``parents`` of every state, all of them in one launch;
:func:`copy_pages_` copies pages inside their pools."""
from __future__ import annotations

import ctypes
from typing import List, Sequence, Tuple

import torch

from .scored_attn import on_device

CHUNK, MOST, TENSORS = 4096, 128, 64                      # csrc/beam.cu
PLACES = (1 << 31) - (1 << 14)                            # places of beam and token: a part's last chunk ends behind them, still below 2^31
_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


class _Args(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p) for n in ("logits", "scores", "out", "beam", "token", "key", "top", "at", "sum")] +
                [(n, ctypes.c_longlong) for n in ("s_n", "s_k", "c_n", "c_k")] + [(n, ctypes.c_int) for n in ("N", "K", "V", "n", "parts", "length")])


class _Rows(ctypes.Structure):
    _fields_ = [("src", ctypes.c_void_p * TENSORS), ("dst", ctypes.c_void_p * TENSORS), ("bytes", ctypes.c_longlong * TENSORS), ("rows", ctypes.c_longlong * TENSORS),
                ("from_", ctypes.c_void_p), ("to", ctypes.c_void_p), ("count", ctypes.c_longlong), ("tensors", ctypes.c_int), ("err", ctypes.c_void_p)]


def _eager_select(logits, scores, n):
    x = torch.nan_to_num(logits.double(), nan=float("-inf"), posinf=float("inf"), neginf=float("-inf"))
    x = x - x.amax(-1, keepdim=True)                       # NaN in beams of nothing but minus infinity
    # rows padded to begin alike: how a row's sum is grouped follows its place, and equal rows have equal sums
    sums = torch.nn.functional.pad(x, (0, -x.shape[2] % 64), value=float("-inf")).exp().sum(-1, keepdim=True)
    total = x + (scores.double()[..., None] - sums.log())
    total = torch.nan_to_num(total, nan=float("-inf"), posinf=float("inf"), neginf=float("-inf")).flatten(1)
    V = logits.shape[2]
    best, at = torch.empty(len(total), n, dtype=torch.float64, device=x.device), torch.empty(len(total), n, dtype=torch.int64, device=x.device)
    for i, row in enumerate(total):
        place = (row >= row.topk(n).values[-1]).nonzero()[:, 0]          # in order of place, so that a stable sort leaves ties there
        s, o = torch.sort(row[place], descending=True, stable=True)
        best[i], at[i] = s[:n], place[o[:n]]
    return best.float(), at // V, at % V


def _held(N: int, K: int, V: int, n: int) -> bool:
    """Do the kernels hold a search of this size?"""
    return 0 < N and n <= MOST and K <= MOST and N * K <= 65535 and K * V <= PLACES


def _shares(N: int, K: int, V: int, slots: int) -> Tuple[int, int]:
    """(parts of a beam's row, logits of a part): a chunk to a part, or parts for one wave."""
    parts = max(1, min(-(-V // CHUNK), slots // (N * K)))
    return parts, -(-V // (parts * 8)) * 8


def beam_select(logits: torch.Tensor, scores: torch.Tensor, n: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``logits [N, K, V]`` (fp32, bf16 or fp16) and ``scores [N, K]`` (fp32) of N prompts with K beams: ``(scores fp32, beam int64, token int64)``, each ``[N, n]``,
    best first.  No gradient."""
    kind, shape, dev = _TYPES.get(logits.dtype), logits.shape, logits.device
    if len(shape) != 3 or scores.shape != shape[:2] or kind is None or scores.dtype != torch.float32:
        raise ValueError("beam selection takes logits [N, K, V] in fp32, bf16 or fp16 and fp32 scores [N, K]")
    if scores.device != dev:
        raise ValueError("logits and scores lie on one device")
    N, K, V = shape
    if not 1 <= n <= K * V:
        raise ValueError(f"{n} continuations of {K} beams over a vocabulary of {V}")
    if not logits.is_cuda or not _held(N, K, V, n):
        with torch.no_grad():
            return _eager_select(logits, scores, n)
    from . import cuda as Kn
    s_n, s_k, s_v = logits.stride()
    if s_v != 1 and V > 1:
        logits = logits.contiguous()
        s_n, s_k, s_v = logits.stride()
    out, beam, token = torch.empty((N, n), dtype=torch.float32, device=dev), torch.empty((N, n), dtype=torch.int64, device=dev), torch.empty((N, n), dtype=torch.int64, device=dev)
    parts, length = _shares(N, K, V, 4 * Kn.num_sms())                           # four CTAs per SM
    rows = N * K * parts
    work = torch.empty(rows * (3 + 2 * n), dtype=torch.float32, device=dev)      # sums (64 bits), maxima, candidates
    p = work.data_ptr()
    c_n, c_k = scores.stride()
    a = _Args(logits.data_ptr(), scores.data_ptr(), out.data_ptr(), beam.data_ptr(), token.data_ptr(), p + rows * 12, p + rows * 8, p + rows * (12 + 4 * n), p, s_n, s_k,
              c_n, c_k, N, K, V, n, parts, length)
    with on_device(logits):
        Kn._check(Kn.lib().lmoe_beam_select(ctypes.byref(a), kind, Kn._st()), "beam_select", 2)
    return out, beam, token


def _copy_rows(src: Sequence[torch.Tensor], dst: Sequence[torch.Tensor], rows: int, from_, to):
    from . import cuda as K
    a = _Rows()
    a.from_, a.to, a.count, a.err = from_.data_ptr(), K._ptr(to), rows, K.error_word(from_.device)
    with on_device(from_):
        for first in range(0, len(src), TENSORS):
            some = src[first:first + TENSORS]
            n = len(some)
            a.src[:n], a.dst[:n] = [t.data_ptr() for t in some], [t.data_ptr() for t in dst[first:first + TENSORS]]
            a.rows[:n] = [t.shape[0] for t in some]
            a.bytes[:n] = [t.nbytes // t.shape[0] for t in dst[first:first + TENSORS]]
            a.tensors = n
            K._check(K.lib().lmoe_copy_rows(ctypes.byref(a), K._st()), "copy_rows")


def reorder_states(states: Sequence[torch.Tensor], parents: torch.Tensor) -> List[torch.Tensor]:
    """``[t[parents] for t in states]`` for states with one row per beam and ``parents`` int64 ``[rows]``.  A number that is no row raises on the CPU; on CUDA its row is left
    undefined and the kernels' error word is set.  No gradient."""
    if parents.dtype != torch.int64 or parents.dim() != 1:
        raise ValueError("parents is an int64 tensor [rows]")
    dev, n = parents.device, parents.shape[0]
    for t in states:
        if t.dim() < 1 or t.device != dev:
            raise ValueError("a state has a row per beam and lies where the parents are")
    if not parents.is_cuda:
        with torch.no_grad():
            return [t.index_select(0, parents) for t in states]
    states = [t if t.is_contiguous() else t.contiguous() for t in states]
    out = [torch.empty_like(t) if t.shape[0] == n else torch.empty((n, *t.shape[1:]), dtype=t.dtype, device=dev) for t in states]
    some = [(t, o) for t, o in zip(states, out) if o.numel()]
    if some:
        _copy_rows([t for t, _ in some], [o for _, o in some], n, parents if parents.is_contiguous() else parents.contiguous(), None)
    return out


def copy_pages_(pools: Sequence[torch.Tensor], src: Sequence[int], dst: Sequence[int]):
    """``pool[dst[i]] = pool[src[i]]`` in every pool ``[pages, ...]``.  The pages written are all different and none of them is read."""
    if len(src) != len(dst) or len(set(dst)) != len(dst) or set(dst) & set(src):
        raise ValueError("pages are copied to as many other ones, each once")
    for t in pools:
        if not t.is_contiguous() or t.device != pools[0].device:
            raise ValueError("pools of pages are contiguous and lie on one device")
        if any(not 0 <= p < t.shape[0] for p in (*src, *dst)):
            raise ValueError(f"a page outside the {t.shape[0]} of its pool")
    pools = [t for t in pools if t.numel()]
    if not src or not pools:
        return
    at = torch.tensor([list(src), list(dst)], dtype=torch.int64, device=pools[0].device)
    if not pools[0].is_cuda:
        with torch.no_grad():
            for t in pools:
                t[at[1]] = t[at[0]]
        return
    _copy_rows(pools, pools, len(src), at[0], at[1])
