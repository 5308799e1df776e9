"""Decoding caches of a model whose softmax layers keep their keys and values in pages.

A :class:`PagedCache` is the list of per-layer dicts that ``CausalLM.forward`` takes.  The linear layers' dicts are filled by the layers themselves, as ever.  A softmax layer's holds its two
pools ``k_pages`` / ``v_pages`` ``[pages, PAGE, heads, dim]`` and, the same tensors in every layer, the requests' page ``table [rows, n]``, their ``lengths [rows]`` (the tokens of the running call
counted) and the rotary tables.  Nothing moves or grows while requests are decoded, so one-token steps can be captured in a CUDA graph; the dense cache is concatenated anew for every token.

All rows are at the same position, as in ``generate_tokens``.  :meth:`advance` comes before the forward pass of every call.  :meth:`reorder` makes row i go on from row ``parents[i]`` (beam search):
whole pages are shared, and a row that would write into a page that another one uses gets a copy of it."""
from __future__ import annotations

from typing import Dict, List, Optional, Sequence

import torch

from .. import ops
from ..ref import ops as R
from .kv_cache import PAGE


class PagedCache(list):
    def __init__(self, model, rows: int, tokens: int, live: Optional[int] = None):
        """Room for ``rows`` requests of up to ``tokens`` tokens; ``live``: rows of the first calls (default: all; :meth:`reorder` sets their number)."""
        if not self.supported(model):
            raise ValueError("a paged cache is for softmax layers on one context-parallel rank (no latent attention, no layer-list designs)")
        super().__init__({} for _ in model.specs)
        dev = next(model.parameters()).device
        cfg = model.cfg
        width = -(-max(tokens, 1) // PAGE)
        self.rows, self.tokens, self.length = rows, tokens, 0
        self.free: List[int] = list(range(rows * width + rows))[::-1]
        self.owned: List[List[int]] = [[] for _ in range(rows if live is None else live)]
        self.uses: Dict[int, int] = {}
        self._host = torch.zeros(rows, width, dtype=torch.int32)
        self._table = self._host.to(dev)
        self._lengths = torch.zeros(rows, dtype=torch.int32, device=dev)
        self.paged = [i for i, s in enumerate(model.specs) if s.mixer == "attn"]
        rope = None
        for i in self.paged:
            att = model.decoder.layers[i]._mixer()
            if att.rope is not None and rope is None:
                rope = R.rope_freqs(width * PAGE, int(att.D * cfg.rotary_percent), cfg.rotary_base, 0, dev, cfg.rotary_seq_len_interpolation_factor)
            for name in ("k_pages", "v_pages"):
                self[i][name] = torch.zeros(len(self.free), PAGE, att.Gl, att.D, dtype=att.linear_qkv.weight.dtype, device=dev)
            if rope is not None:
                self[i]["cos"], self[i]["sin"] = rope
        self._bind()

    @staticmethod
    def supported(model) -> bool:
        return (not getattr(model, "packed_rows", False) and model.mesh["cp"].is_trivial and model.specs is not None
                and all(s.mixer != "mla" for s in model.specs))

    def _bind(self):
        for i in self.paged:
            self[i]["table"], self[i]["lengths"] = self._table[: len(self.owned)], self._lengths[: len(self.owned)]

    def _page(self) -> int:
        p = self.free.pop()
        self.uses[p] = 1
        return p

    def _drop(self, p: int):
        self.uses[p] -= 1
        if self.uses[p] == 0:
            del self.uses[p]
            self.free.append(p)

    def _upload(self):
        for b, pages in enumerate(self.owned):
            self._host[b, : len(pages)] = torch.tensor(pages, dtype=torch.int32)
        self._table.copy_(self._host)

    def advance(self, n: int):
        """Room for ``n`` more tokens of every row."""
        end = self.length + n
        if end > self.tokens:
            raise ValueError(f"{end} tokens in a cache for {self.tokens}")
        need = -(-end // PAGE)
        grown = [pages for pages in self.owned if len(pages) < need] if self.paged else []
        for pages in grown:
            while len(pages) < need:
                pages.append(self._page())
        if grown:
            self._upload()
        self.length = end
        self._lengths.fill_(end)

    def expect(self, rows: int, tokens: int, position_offset: int):
        """What a forward pass asks of its cache: as many rows, and room for its tokens (a captured step comes without its offset)."""
        if self.paged and rows != len(self.owned):
            raise ValueError(f"{rows} rows of tokens on a cache of {len(self.owned)} rows")
        if self.paged and position_offset + tokens > self.length:
            raise ValueError(f"tokens up to {position_offset + tokens} on a cache with room for {self.length}: advance() comes first")

    def reorder(self, parents: Sequence[int]):
        """Row i goes on from row ``parents[i]``; linear layers' states too.  Entries have to be tensors with a row per request (:meth:`reorderable`)."""
        n = len(self.owned)
        if not 1 <= len(parents) <= self.rows or any(not 0 <= p < n for p in parents):
            raise ValueError(f"rows {list(parents)} of {n}, {self.rows} at most")
        states = [(c, k) for i, c in enumerate(self) if i not in self.paged for k in c]
        if states:
            at = torch.tensor(list(parents), dtype=torch.int64, device=self._table.device)
            for (c, k), t in zip(states, ops.reorder_states([c[k] for c, k in states], at)):
                c[k] = t
        if not self.paged:
            self.owned = [[] for _ in parents]
            return
        new = [list(self.owned[p]) for p in parents]
        for pages in new:
            for p in pages:
                self.uses[p] += 1
        for pages in self.owned:
            for p in pages:
                self._drop(p)
        self.owned = new
        if self.length % PAGE:                             # the page that the next token goes to
            src, dst = [], []
            for pages in self.owned:
                if self.uses[pages[-1]] > 1:
                    src.append(pages[-1])
                    self._drop(pages[-1])
                    pages[-1] = self._page()
                    dst.append(pages[-1])
            ops.copy_pages_([self[i][name] for i in self.paged for name in ("k_pages", "v_pages")], src, dst)
        self._upload()
        self._bind()

    def reorderable(self) -> bool:
        """After a call: has every linear layer kept tensors with a row per request, and nothing else?"""
        return all(torch.is_tensor(t) and t.dim() > 0 and t.shape[0] == len(self.owned)
                   for i, c in enumerate(self) if i not in self.paged for t in c.values())
