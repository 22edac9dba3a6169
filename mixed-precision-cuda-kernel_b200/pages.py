"""Which pages of a pool (`quant_cuda.KVPages`) the sequences of a batch hold: the host's side of a paged KV cache.

The reference keeps one cache of the full length per sequence (llama/modeling_llama_quant.py:371-419 of the reference project).
"""
from __future__ import annotations

from typing import Dict

import torch


class PageTable:
    """Table (sequences, width) int32 of pages, -1 where there is none; pages come from a list of free ones and go back to it."""

    def __init__(self, sequences: int, slots: int, pages: int, page_size: int):
        if sequences < 1 or slots < 1 or pages < 1 or page_size < 1:
            raise ValueError("sequences, slots, pages and page_size must be positive")
        self.page_size, self.pages = page_size, pages
        self.host = torch.full((sequences, -(-slots // page_size)), -1, dtype=torch.int32)
        self.held = [0] * sequences                      # pages of each sequence
        self.free = list(range(pages - 1, -1, -1))

    def reserve(self, slots: Dict[int, int]) -> bool:
        """Pages for the first slots[s] slots of every sequence s named, for all of them or for none (ValueError).  True where the
        table has changed."""
        more = {s: -(-n // self.page_size) - self.held[s] for s, n in slots.items()}
        for s, n in slots.items():
            if n > self.host.shape[1] * self.page_size:
                raise ValueError(f"{n} slots do not fit the {self.host.shape[1]} pages of a sequence")
        need = sum(m for m in more.values() if m > 0)
        if need > len(self.free):
            raise ValueError(f"{need} more pages are needed, {len(self.free)} of {self.pages} are free")
        for s, m in more.items():
            for _ in range(m):
                self.host[s, self.held[s]] = self.free.pop()
                self.held[s] += 1
        return need > 0

    def release(self, sequence: int) -> None:
        """All pages of a sequence are free again."""
        self.free += self.host[sequence, :self.held[sequence]].flip(0).tolist()
        self.host[sequence] = -1
        self.held[sequence] = 0
