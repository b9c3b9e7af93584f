"""Paged KV cache of a decoder: the pools of all layers, and the account on the host of which sequence has which pages.

Sequences of any lengths share the pools, so a batch takes the memory of the keys that it holds (plus a part of a page for each sequence), not of
its longest sequence times its size. The reference keeps no keys at all (ghostflow-nn/src/gpt.rs:402-422).
"""
from __future__ import annotations

from dataclasses import dataclass

import torch


@dataclass
class PagedBatch:
    """What :func:`ops.rope_qkv_to_pages` and :func:`ops.paged_attention` are told of a batch (the same for all layers)."""
    table: torch.Tensor            # int32 [B, pages of the longest]
    lens: torch.Tensor             # int32 [B]: keys with the new ones
    cu: torch.Tensor | None        # int32 [B + 1]: first new token of each; None: one each
    longest: int                   # keys of the longest

    def advance(self) -> None:
        """To the next token of every sequence of a batch of one token each, whose pages were reserved."""
        self.lens.add_(1)
        self.longest += 1


class PagedKVCache:
    """``num_pages`` pages of ``page_size`` rows (a power of two from 16 for the kernels) for the keys and values of ``layers`` layers."""

    def __init__(self, layers: int, num_pages: int, page_size: int, kv_heads: int, head_dim: int, device=None, dtype=None):
        shape = (num_pages, page_size, kv_heads, head_dim)
        self.page_size = page_size
        self.pools = [(torch.zeros(shape, device=device, dtype=dtype), torch.zeros(shape, device=device, dtype=dtype)) for _ in range(layers)]
        self.device = self.pools[0][0].device if layers else torch.device(device or "cpu")
        self._free = list(range(num_pages - 1, -1, -1))
        self._pages: dict = {}

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def reserve(self, sequence, length: int) -> None:
        """Pages for ``length`` keys of a sequence (any hashable name), those it has among them; all or none are taken."""
        have = self._pages.get(sequence, [])
        more = -(-length // self.page_size) - len(have)
        if more > len(self._free):
            raise RuntimeError(f"{more} pages of {self.page_size} rows are needed and {len(self._free)} are free")
        self._pages[sequence] = have + [self._free.pop() for _ in range(more)]

    def release(self, sequence) -> None:
        """Gives a sequence's pages back."""
        self._free.extend(reversed(self._pages.pop(sequence)))

    def batch(self, sequences, lens, new=None) -> PagedBatch:
        """The batch of ``sequences`` with ``lens`` keys each, of which the last ``new`` (one, without it) are new tokens. Their pages have to be
        reserved. A sequence may come more than once (parts of a prompt; any number of empty slots), but no position of it be new twice."""
        sequences, lens = list(sequences), [int(n) for n in lens]
        new = None if new is None else [int(n) for n in new]
        if len(sequences) != len(lens) or (new is not None and len(new) != len(lens)):
            raise ValueError(f"{len(sequences)} sequences, {len(lens)} lengths and {None if new is None else len(new)} numbers of new tokens")
        pages, written = [self._pages.get(s, []) for s in sequences], {}
        for s, n, m, have in zip(sequences, lens, [min(n, 1) for n in lens] if new is None else new, pages):
            if n > len(have) * self.page_size:
                raise ValueError(f"sequence {s!r} has {len(have)} pages of {self.page_size} rows, not room for {n} keys")
            if not 0 <= m <= n:
                raise ValueError(f"sequence {s!r} has {n} keys, {m} of them new")
            if m > 0:
                spans = written.setdefault(s, [])
                if any(n - m < end and start < n for start, end in spans):
                    raise ValueError(f"sequence {s!r} is there more than once with new tokens at the same positions")
                spans.append((n - m, n))
        B, width = len(lens), max(map(len, pages), default=0)
        ints = [p for have in pages for p in (*have, *[-1] * (width - len(have)))] + lens
        if new is not None:
            ints.append(0)
            for n in new:
                ints.append(ints[-1] + n)
        t = torch.tensor(ints, dtype=torch.int32, device=self.device)            # one copy
        return PagedBatch(t[:B * width].view(B, width), t[B * width:B * width + B], t[B * width + B:] if new is not None else None,
                          max(lens, default=0))
