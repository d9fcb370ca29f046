"""A key/value cache in pages, for generation with sequences of different length.

The pages of a layer are two tensors [pages, kv heads, page_size, D] (:class:`PagedKVCache`), bf16 or e4m3 with a power of
two per row at half the bytes.  Which pages a sequence has, in which order, says one table for all layers
(:class:`PageTable`).  The device side - writing, reading back, attention of few new tokens - is ``kernels.paged_*``; the
methods here only pass the tensors on.

A contiguous cache (``kernels.qkv_prologue`` with its [B, H, cap, D] buffers) holds the longest sequence's length for all of
them; pages hold what each has, and a sequence that ends gives its pages to the next.
"""
from __future__ import annotations

from typing import List, Optional, Tuple

import torch

from . import kernels as K


class PageTable:
    """Which pages ``batch`` sequences of up to ``max_tokens`` tokens have, out of ``num_pages`` (default: enough for all of
    them at full length).  Bookkeeping is on the host; ``table`` is the int32 [batch, pages per sequence] tensor that the
    kernels take, updated in place (its address stays, for captured graphs), -1 where a sequence has no page."""

    def __init__(self, batch: int, max_tokens: int, page_size: int = 64, num_pages: Optional[int] = None, device="cuda"):
        if batch < 1 or max_tokens < 1:
            raise ValueError("batch and max_tokens must be positive")
        if page_size < 16 or page_size > 512 or page_size % 16:
            raise ValueError(f"page_size must be a multiple of 16 up to 512, got {page_size}")
        self.batch, self.page_size = batch, page_size
        self.per_sequence = -(-max_tokens // page_size)
        self.num_pages = batch * self.per_sequence if num_pages is None else num_pages
        self._free: List[int] = list(range(self.num_pages - 1, -1, -1))
        self._owned: List[List[int]] = [[] for _ in range(batch)]
        self._host = torch.full((batch, self.per_sequence), -1, dtype=torch.int32)
        self.table = self._host.to(device)

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def _check(self, sequence: int) -> None:
        if not 0 <= sequence < self.batch:
            raise IndexError(f"sequence {sequence} is none of 0 .. {self.batch - 1}")

    def pages_of(self, sequence: int) -> List[int]:
        self._check(sequence)
        return list(self._owned[sequence])

    def reserve(self, sequence: int, tokens: int) -> None:
        """Gives the sequence pages for its first ``tokens`` tokens; those it has stay.  Raises, and changes nothing, where
        there is no such sequence, it would be too long or the pages do not suffice."""
        self.reserve_all({sequence: tokens})

    def reserve_all(self, tokens: dict) -> None:
        """:meth:`reserve` for several sequences {sequence: tokens} with one update of ``table``."""
        need = {}
        for s, n in tokens.items():
            self._check(s)
            want = -(-n // self.page_size)
            if want > self.per_sequence:
                raise RuntimeError(f"sequence {s}: {n} tokens exceed {self.per_sequence} pages of {self.page_size}")
            need[s] = max(0, want - len(self._owned[s]))
        if sum(need.values()) > len(self._free):
            raise RuntimeError(f"out of pages: {sum(need.values())} wanted, {len(self._free)} of {self.num_pages} free")
        for s, n in need.items():
            for _ in range(n):
                page = self._free.pop()
                self._host[s, len(self._owned[s])] = page
                self._owned[s].append(page)
        if any(need.values()):
            self.table.copy_(self._host)

    def release(self, sequence: int) -> None:
        """Takes the sequence's pages back.  Work already submitted on other streams must be done with them."""
        self._check(sequence)
        if self._owned[sequence]:
            self._free.extend(reversed(self._owned[sequence]))
            self._owned[sequence] = []
            self._host[sequence] = -1
            self.table.copy_(self._host)


class PagedKVCache:
    """One layer's pages: ``k``, ``v`` [num_pages, heads, page_size, head_dim] of bf16, or (``dtype=torch.float8_e4m3fn``)
    e4m3 with ``scales`` uint8 [num_pages, heads, page_size, 2].  ``start``, ``lens``, ``count``: int32 [batch] on the
    device; ``table``: :attr:`PageTable.table`."""

    def __init__(self, num_pages: int, heads: int, head_dim: int, page_size: int = 64, dtype: torch.dtype = torch.bfloat16,
                 device="cuda"):
        if dtype not in (torch.bfloat16, torch.float8_e4m3fn):
            raise ValueError(f"dtype must be bfloat16 or float8_e4m3fn, got {dtype}")
        if head_dim not in (64, 128):
            raise ValueError(f"head_dim must be 64 or 128, got {head_dim}")
        shape = (num_pages, heads, page_size, head_dim)
        self.k = torch.zeros(shape, dtype=torch.uint8 if dtype != torch.bfloat16 else dtype, device=device).view(dtype)
        self.v = torch.zeros_like(self.k)
        self.scales = None
        if dtype == torch.float8_e4m3fn:
            self.scales = torch.zeros((num_pages, heads, page_size, 2), dtype=torch.uint8, device=device)

    @property
    def nbytes(self) -> int:
        return self.k.nbytes + self.v.nbytes + (0 if self.scales is None else self.scales.nbytes)

    def append(self, k, v, table, start, *, count=None, status=None) -> None:
        """:func:`kernels.paged_kv_append`."""
        K.paged_kv_append(k, v, self.k, self.v, table, start, scales=self.scales, count=count, status=status)

    def prologue(self, q, k, v, table, start, **kw) -> torch.Tensor:
        """:func:`kernels.paged_qkv_prologue`."""
        return K.paged_qkv_prologue(q, k, v, self.k, self.v, table, start, scales=self.scales, **kw)

    def read(self, table, lens, n: int, *, start: int = 0, out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None, status=None):
        """:func:`kernels.paged_kv_read`."""
        return K.paged_kv_read(self.k, self.v, table, lens, n, scales=self.scales, start=start, out=out, status=status)

    def attend(self, q, table, lens, scale: Optional[float] = None, **kw):
        """:func:`kernels.paged_attn_fwd`."""
        return K.paged_attn_fwd(q, self.k, self.v, table, lens, scale, scales=self.scales, **kw)
