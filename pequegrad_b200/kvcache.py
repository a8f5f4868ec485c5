"""Paged key / value cache of a model: pages, which sequence holds them, and the plans of its calls.

The reference generates by running the whole model over all tokens again for every new one
(examples/gpt2.py:406-438); here each token's keys and values are kept. All layers share the
bookkeeping: a page number is good for every layer's cache. Storing, reading and attending are
the calls `kv_write`, `kv_read` and `paged_attention` of `kernels`.
"""
from __future__ import annotations

from typing import Sequence

import torch

from . import kernels as K


class KVPlan:
    """One step of some sequences: row offsets, lengths and page table on the device (see `kernels.kv_write`), and the
    position of every row. `rows` is their number, `last` the row of each sequence's last new token (-1 without one), `fewest` the
    smallest number of new tokens of a sequence, `longest` the longest context."""

    def __init__(self, new: Sequence[int], ctx: Sequence[int], tables: Sequence[Sequence[int]], device):
        start = [0]
        for n in new:
            start.append(start[-1] + n)
        width = max((len(t) for t in tables), default=0)
        # one upload: offsets, lengths, last rows, positions, table
        flat = start + list(ctx) + [s - 1 if n else -1 for s, n in zip(start[1:], new)]
        for n, c in zip(new, ctx):
            flat.extend(range(c - n, c))
        for t in tables:
            flat.extend(list(t) + [-1] * (width - len(t)))
        B, self.rows, self.longest, self.fewest = len(new), start[-1], max(ctx, default=0), min(new, default=1)
        dev = torch.tensor(flat, dtype=torch.int32).to(device)
        at = 0

        def take(n):
            nonlocal at
            at += n
            return dev[at - n:at]

        self.q_start, self.ctx_len, self.last, self.positions = take(B + 1), take(B), take(B), take(self.rows)
        self.page_table = take(B * width).view(B, width)


class PagedKVCache:
    """Keys and values of `n_layer` layers in `n_pages` pages of `page_size` tokens, in `dtype` (float16, bfloat16, or int8
    with a scale per token and head). Heads lie outermost in a page: a head's tokens are contiguous."""

    def __init__(self, n_layer: int, n_head: int, head_dim: int, n_pages: int, page_size: int = 16, dtype=torch.float16, device="cuda"):
        shape = (n_layer, n_pages, n_head, page_size, head_dim)
        self.page_size, self.dtype, self.device = page_size, dtype, torch.device(device)
        self.k, self.v = (torch.zeros(shape, dtype=dtype, device=device) for _ in range(2))
        self.k_scale = self.v_scale = None
        if dtype == torch.int8:
            self.k_scale, self.v_scale = (torch.zeros(shape[:-1], dtype=torch.float32, device=device) for _ in range(2))
        self._free = list(range(n_pages - 1, -1, -1))
        self._pages, self._len, self._next = {}, {}, 0

    def open(self) -> int:
        """A new sequence without tokens; its handle."""
        self._next += 1
        self._pages[self._next], self._len[self._next] = [], 0
        return self._next

    def close(self, seq: int) -> None:
        """Gives a sequence's pages back. Work that was enqueued on them comes before what their next owner enqueues."""
        self._free.extend(reversed(self._pages.pop(seq)))
        del self._len[seq]

    def length(self, seq: int) -> int:
        return self._len[seq]

    def free_pages(self) -> int:
        return len(self._free)

    def extend(self, seqs: Sequence[int], new: Sequence[int]) -> KVPlan:
        """Makes room for `new` tokens of each sequence and returns the plan of the step that stores them. Every layer of the
        model then writes and attends with this plan. Raises before anything changes if the pages do not suffice."""
        if len(set(seqs)) != len(seqs) or len(seqs) != len(new) or any(n < 0 for n in new):
            raise ValueError("extend: each sequence once, with a number of new tokens")
        need = [-(-(self._len[s] + n) // self.page_size) - len(self._pages[s]) for s, n in zip(seqs, new)]
        if sum(need) > len(self._free):
            raise RuntimeError(f"extend: {sum(need)} pages are needed and {len(self._free)} are free")
        for s, n, p in zip(seqs, new, need):
            self._pages[s].extend(self._free.pop() for _ in range(p))
            self._len[s] += n
        return KVPlan(new, [self._len[s] for s in seqs], [self._pages[s] for s in seqs], self.device)

    def _layer(self, i: int) -> dict:
        return dict(k_scale=None, v_scale=None) if self.k_scale is None else dict(k_scale=self.k_scale[i], v_scale=self.v_scale[i])

    def write(self, layer: int, k: torch.Tensor, v: torch.Tensor, plan: KVPlan) -> None:
        """Stores the step's keys and values [rows, heads, head dim] of one layer. Rows behind the plan's are padding."""
        if len(k) < plan.rows:
            raise ValueError(f"write: {len(k)} rows for a plan of {plan.rows}")
        K.kv_write(k, v, self.k[layer], self.v[layer], plan.q_start, plan.ctx_len, plan.page_table, **self._layer(layer))

    def attend(self, layer: int, q: torch.Tensor, plan: KVPlan, scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
        """Causal attention of the step's queries [rows, query heads, head dim] over all that is stored of their sequences."""
        if len(q) < plan.rows:
            raise ValueError(f"attend: {len(q)} rows for a plan of {plan.rows}")
        return K.paged_attention(q, self.k[layer], self.v[layer], plan.q_start, plan.ctx_len, plan.page_table, scale, out=out, **self._layer(layer))

    def read(self, layer: int, seqs: Sequence[int], out_dtype=None):
        """(k, v) of the sequences, packed one after another [tokens, heads, head dim]; an int8 cache as `out_dtype`."""
        n = [self._len[s] for s in seqs]
        plan = KVPlan(n, n, [self._pages[s] for s in seqs], self.device)
        return K.kv_read(self.k[layer], self.v[layer], plan.q_start, plan.page_table, plan.rows, out_dtype=out_dtype, **self._layer(layer))
