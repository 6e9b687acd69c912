"""Paged key/value cache of a model and the batches that are decoded over it.

:class:`PagedKVCache` owns the page pools of every layer (``ops.functional.KVPages``) and hands out pages
to sequences.  :class:`CacheBatch` is one step's device-side description of the batch (block table, cached
lengths, row starts) that the cache-writing and attention kernels read.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import List, Optional, Sequence

import torch

from .config import ModelConfig

CACHE_DTYPES = {"bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}


@dataclass
class CacheBatch:
    """The new tokens of one step: ``rows[b]`` tokens of sequence b, the last of ``lens[b]`` cached ones."""

    block_table: torch.Tensor
    kv_lens: torch.Tensor
    q_starts: Optional[torch.Tensor]
    max_q_len: int
    positions: torch.Tensor


class PagedKVCache:
    """Page pools of all layers of a model, shared by the sequences that hold pages of them.

    ``dtype`` is ``bf16``, ``e4m3`` or ``int8`` (8-bit codes with one scale per token and head).  Pages are
    handed out by :meth:`extend` and returned by :meth:`release`; a page belongs to one sequence.
    """

    def __init__(self, cfg: ModelConfig, n_pages: int, page_size: int = 64, dtype: str = "bf16",
                 device: Optional[torch.device] = None) -> None:
        if dtype not in CACHE_DTYPES:
            raise ValueError(f"unknown cache dtype {dtype!r}; expected one of {sorted(CACHE_DTYPES)}")
        if page_size not in (16, 32, 64, 128):
            raise ValueError(f"page_size must be 16, 32, 64 or 128, got {page_size}")
        if n_pages < 1:
            raise ValueError(f"n_pages must be positive, got {n_pages}")
        from ..ops.functional import KVPages

        self.cfg = cfg
        self.page_size = page_size
        self.device = torch.device("cuda" if device is None else device)
        self.layers: List[KVPages] = []
        shape = (n_pages, cfg.n_kv_heads, page_size, cfg.head_dim)
        for _ in range(cfg.n_layers):
            pools = [torch.zeros(shape, dtype=CACHE_DTYPES[dtype], device=self.device) for _ in range(2)]
            scales = [None, None]
            if dtype != "bf16":
                scales = [torch.zeros(shape[:3], dtype=torch.float32, device=self.device) for _ in range(2)]
            self.layers.append(KVPages(pools[0], pools[1], scales[0], scales[1]))
        self._free = list(range(n_pages - 1, -1, -1))
        self._pages: List[List[int]] = []
        self._lens: List[int] = []

    @classmethod
    def for_batch(cls, cfg: ModelConfig, batch: int, max_tokens: int, page_size: int = 64, dtype: str = "bf16",
                  device: Optional[torch.device] = None) -> "PagedKVCache":
        """A cache that holds ``batch`` sequences of up to ``max_tokens`` tokens, with the sequences added."""
        cache = cls(cfg, batch * max(1, -(-max_tokens // page_size)), page_size, dtype, device)
        for _ in range(batch):
            cache.add_sequence()
        return cache

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def add_sequence(self) -> int:
        """A new empty sequence; returns its number."""
        self._pages.append([])
        self._lens.append(0)
        return len(self._lens) - 1

    def _check(self, seqs: Sequence[int]) -> None:
        for s in seqs:
            if not 0 <= s < len(self._lens):
                raise IndexError(f"the cache has no sequence {s}, only 0 to {len(self._lens) - 1}")

    def length(self, seq: int) -> int:
        self._check([seq])
        return self._lens[seq]

    def release(self, seq: int) -> None:
        """Returns the sequence's pages; it is empty afterwards."""
        self._check([seq])
        self._free.extend(reversed(self._pages[seq]))
        self._pages[seq] = []
        self._lens[seq] = 0

    def extend(self, seqs: Sequence[int], rows: Sequence[int]) -> CacheBatch:
        """Makes room for ``rows[i]`` more tokens of sequence ``seqs[i]`` and describes the step that adds them.
        Nothing is changed if the pool has too few pages."""
        if len(seqs) != len(rows) or len(set(seqs)) != len(seqs):
            raise ValueError("extend: one row count for each of a set of different sequences")
        self._check(seqs)
        if any(n < 0 for n in rows):
            raise ValueError("extend: row counts must not be negative")
        need = [max(0, -(-(self._lens[s] + n) // self.page_size) - len(self._pages[s])) for s, n in zip(seqs, rows)]
        if sum(need) > len(self._free):
            raise RuntimeError(f"the cache is out of pages: {sum(need)} needed, {len(self._free)} free")
        # described first, taken when nothing can fail any more
        left = len(self._free)
        pages, lens = [], []
        for s, n, count in zip(seqs, rows, need):
            pages.append(self._pages[s] + self._free[left - count:left][::-1])
            lens.append(self._lens[s] + n)
            left -= count
        table = torch.zeros(len(seqs), max([len(p) for p in pages] + [1]), dtype=torch.int32)
        for i, p in enumerate(pages):
            table[i, :len(p)] = torch.tensor(p, dtype=torch.int32)
        starts = torch.zeros(len(seqs) + 1, dtype=torch.int32)
        starts[1:] = torch.cumsum(torch.tensor(list(rows), dtype=torch.int32), 0)
        positions = torch.cat([torch.arange(end - n, end) for end, n in zip(lens, rows)])
        single = all(n == 1 for n in rows)
        batch = CacheBatch(table.to(self.device), torch.tensor(lens, dtype=torch.int32).to(self.device),
                           None if single else starts.to(self.device), max(max(rows), 1), positions.to(self.device))
        for s, p, n in zip(seqs, pages, lens):
            self._pages[s], self._lens[s] = p, n
        del self._free[left:]
        return batch

    def retract(self, seqs: Sequence[int], rows: Sequence[int]) -> None:
        """Takes the last ``rows[i]`` tokens off sequence ``seqs[i]``: undoes an :meth:`extend` whose step failed."""
        self._check(seqs)
        if len(seqs) != len(rows) or len(set(seqs)) != len(seqs):
            raise ValueError("retract: one row count for each of a set of different sequences")
        if any(not 0 <= n <= self._lens[s] for s, n in zip(seqs, rows)):
            raise ValueError("retract: a sequence has fewer tokens")
        for s, n in reversed(list(zip(seqs, rows))):
            self._lens[s] -= n
            while len(self._pages[s]) > -(-self._lens[s] // self.page_size):
                self._free.append(self._pages[s].pop())
