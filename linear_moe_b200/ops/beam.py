"""One step of a beam search: the best continuations, and the beams' states in their new order (``csrc/beam.cu``; CPU tensors run the eager form).

:func:`beam_select` takes the best ``n`` of ``scores[b] + log_softmax(logits[b])[t]`` over beams and vocabulary of every prompt, ties to the lowest ``b V + t``; the scores are
compared in 64 bits and rounded once.  NaN logits count as minus infinity.  :func:`reorder_states` gives the rows ``parents`` of every state, all of them in one launch;
:func:`copy_pages_` copies pages inside their pools."""
from __future__ import annotations

import ctypes
from typing import List, Sequence, Tuple

import torch

from .scored_attn import on_device

PART, MOST, TENSORS = 4096, 128, 64                       # csrc/beam.cu
_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


class _Args(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p) for n in ("logits", "scores", "out", "beam", "token", "key", "top", "at", "sum")] +
                [(n, ctypes.c_longlong) for n in ("s_n", "s_k", "c_n", "c_k")] + [(n, ctypes.c_int) for n in ("N", "K", "V", "n", "parts")])


class _Rows(ctypes.Structure):
    _fields_ = [("src", ctypes.c_void_p * TENSORS), ("dst", ctypes.c_void_p * TENSORS), ("bytes", ctypes.c_longlong * TENSORS), ("rows", ctypes.c_longlong * TENSORS),
                ("from_", ctypes.c_void_p), ("to", ctypes.c_void_p), ("count", ctypes.c_longlong), ("tensors", ctypes.c_int), ("err", ctypes.c_void_p)]


def _eager_select(logits, scores, n):
    x = torch.nan_to_num(logits.double(), nan=float("-inf"), posinf=float("inf"), neginf=float("-inf"))
    x = x - x.amax(-1, keepdim=True)                       # NaN in beams of nothing but minus infinity
    total = x + (scores.double()[..., None] - x.exp().sum(-1, keepdim=True).log())
    total = torch.nan_to_num(total, nan=float("-inf"), posinf=float("inf"), neginf=float("-inf")).flatten(1)
    V = logits.shape[2]
    best, at = torch.empty(len(total), n, dtype=torch.float64, device=x.device), torch.empty(len(total), n, dtype=torch.int64, device=x.device)
    for i, row in enumerate(total):
        place = (row >= row.topk(n).values[-1]).nonzero()[:, 0]          # in order of place, so that a stable sort leaves ties there
        s, o = torch.sort(row[place], descending=True, stable=True)
        best[i], at[i] = s[:n], place[o[:n]]
    return best.float(), at // V, at % V


@torch.no_grad()
def beam_select(logits: torch.Tensor, scores: torch.Tensor, n: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``logits [N, K, V]`` (fp32, bf16 or fp16) and ``scores [N, K]`` (fp32) of N prompts with K beams: ``(scores fp32, beam int64, token int64)``, each ``[N, n]``,
    best first."""
    if logits.dim() != 3 or scores.shape != logits.shape[:2] or logits.dtype not in _TYPES or scores.dtype != torch.float32:
        raise ValueError("beam selection takes logits [N, K, V] in fp32, bf16 or fp16 and fp32 scores [N, K]")
    if scores.device != logits.device:
        raise ValueError("logits and scores lie on one device")
    N, K, V = logits.shape
    if not 1 <= n <= K * V:
        raise ValueError(f"{n} continuations of {K} beams over a vocabulary of {V}")
    if not logits.is_cuda or n > MOST or K > MOST or N * K > 65535 or K * V >= 1 << 31 or N == 0:      # wider searches than the kernels hold
        return _eager_select(logits, scores, n)
    from . import cuda as Kn
    dev = logits.device
    logits = logits if logits.stride(2) == 1 or V == 1 else logits.contiguous()
    out, ids = torch.empty(N, n, dtype=torch.float32, device=dev), torch.empty(2, N, n, dtype=torch.int64, device=dev)
    parts = -(-(V + 7) // PART)                            # rows may begin up to seven numbers behind a 16-byte boundary
    rows = N * K * parts
    work = torch.empty(rows * 3 + rows * n * 2, dtype=torch.float32, device=dev)      # sums (64 bits), maxima, candidates
    a, p = _Args(), work.data_ptr()
    a.logits, a.scores, a.out, a.beam, a.token = logits.data_ptr(), scores.data_ptr(), out.data_ptr(), ids.data_ptr(), ids[1].data_ptr()
    a.sum, a.top, a.key, a.at = p, p + rows * 8, p + rows * 12, p + rows * (12 + 4 * n)
    a.s_n, a.s_k, a.c_n, a.c_k = logits.stride(0), logits.stride(1), scores.stride(0), scores.stride(1)
    a.N, a.K, a.V, a.n, a.parts = N, K, V, n, parts
    with on_device(logits):
        Kn._check(Kn.lib().lmoe_beam_select(ctypes.byref(a), ctypes.c_int(_TYPES[logits.dtype]), Kn._st()), "beam_select", 2)
    return out, ids[0], ids[1]


def _copy_rows(src: Sequence[torch.Tensor], dst: Sequence[torch.Tensor], rows: int, from_, to):
    from . import cuda as K
    from . import gemm
    a = _Rows()
    a.from_, a.to, a.count, a.err = from_.data_ptr(), K._ptr(to), rows, gemm._err(from_.device).data_ptr()
    with on_device(from_):
        for first in range(0, len(src), TENSORS):
            some = src[first:first + TENSORS]
            for i, (s, d) in enumerate(zip(some, dst[first:first + TENSORS])):
                a.src[i], a.dst[i], a.rows[i] = s.data_ptr(), d.data_ptr(), s.shape[0]
                a.bytes[i] = s.numel() // max(s.shape[0], 1) * s.element_size()
            a.tensors = len(some)
            K._check(K.lib().lmoe_copy_rows(ctypes.byref(a), K._st()), "copy_rows")


@torch.no_grad()
def reorder_states(states: Sequence[torch.Tensor], parents: torch.Tensor) -> List[torch.Tensor]:
    """``[t[parents] for t in states]`` for states with one row per beam and ``parents`` int64 ``[rows]``.  A number that is no row raises on the CPU; on CUDA its row is left
    undefined and the kernels' error word is set."""
    if parents.dtype != torch.int64 or parents.dim() != 1:
        raise ValueError("parents is an int64 tensor [rows]")
    for t in states:
        if t.dim() < 1 or t.device != parents.device:
            raise ValueError("a state has a row per beam and lies where the parents are")
    if not parents.is_cuda:
        return [t.index_select(0, parents) for t in states]
    out = [torch.empty(parents.shape[0], *t.shape[1:], dtype=t.dtype, device=t.device) for t in states]
    work = [(t if t.is_contiguous() else t.contiguous(), o) for t, o in zip(states, out) if o.numel()]
    if work:
        _copy_rows([s for s, _ in work], [d for _, d in work], parents.shape[0], parents.contiguous(), None)
    return out


@torch.no_grad()
def copy_pages_(pools: Sequence[torch.Tensor], src: Sequence[int], dst: Sequence[int]):
    """``pool[dst[i]] = pool[src[i]]`` in every pool ``[pages, ...]``.  The pages written are all different and none of them is read."""
    if len(src) != len(dst) or len(set(dst)) != len(dst) or set(dst) & set(src):
        raise ValueError("pages are copied to as many other ones, each once")
    for t in pools:
        if not t.is_contiguous():
            raise ValueError("a pool of pages is contiguous")
        if any(not 0 <= p < t.shape[0] for p in (*src, *dst)):
            raise ValueError(f"a page outside the {t.shape[0]} of its pool")
    pools = [t for t in pools if t.numel()]
    if not src or not pools:
        return
    at = torch.tensor([list(src), list(dst)], dtype=torch.int64, device=pools[0].device)
    if not pools[0].is_cuda:
        for t in pools:
            t[at[1]] = t[at[0]]
        return
    _copy_rows(pools, pools, len(src), at[0], at[1])
