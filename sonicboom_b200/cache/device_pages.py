"""Page lists on the device: what `Cache` does for full-attention groups with lists on the host, as tensors and kernels, so that
a captured step can take the pages it needs by itself.

Beyond the reference, whose cache sets belong to one conversation and are sized when it is opened
(core/include/sonicboom/planner/kv_cache.h:96-170)."""
from __future__ import annotations

import torch

from .. import ops
from .kv import PAGE_SIZE
from .pages import CacheError


class DevicePages:
    """`n_slots` sequences of up to `pages_per_slot` pages each out of `n_pages`.

    A step is three calls, any or all of them in a captured graph: `plan` makes its tables, the step's kernels read them (they are a
    plan as `ops.attention_e4m3` takes it), `advance` records it.  `release` ends sequences.  Nothing here waits for the device:
    a request that cannot be met shows in `tables.status` (`tables.check()`), and its step has no rows."""

    def __init__(self, n_slots: int, n_pages: int, pages_per_slot: int, device, page_size: int = PAGE_SIZE):
        if min(n_slots, n_pages, pages_per_slot, page_size) <= 0:
            raise CacheError(f"{n_slots} slots, {n_pages} pages, {pages_per_slot} pages a slot of {page_size} tokens")
        self.page_size, self.n_pages, self.pages_per_slot = page_size, n_pages, pages_per_slot
        self.lengths = torch.zeros(n_slots, dtype=torch.int32, device=device)
        self.table = torch.full((n_slots, pages_per_slot), -1, dtype=torch.int32, device=device)
        self.free = torch.arange(n_pages - 1, -1, -1, dtype=torch.int32, device=device)      # the lowest page on top
        self.n_free = torch.full((1,), n_pages, dtype=torch.int32, device=device)

    def tables(self, max_seqs: int, max_rows: int, max_pages: int | None = None) -> ops.PageTables:
        """Room for a step's tables: `max_seqs` requests, `max_rows` rows of all of them and `max_pages` pages (as many as the
        requests can have)."""
        most = min(self.n_pages, max_seqs * self.pages_per_slot)
        return ops.PageTables(max_seqs, max_rows, most if max_pages is None else max_pages, self.lengths.device, self.page_size)

    def _check(self, tables: ops.PageTables) -> None:
        if tables.page_size != self.page_size:
            raise CacheError(f"tables for pages of {tables.page_size} tokens, these have {self.page_size}")

    def plan(self, slots: torch.Tensor, new: torch.Tensor, tables: ops.PageTables, max_new: int, max_len: int = 0) -> ops.PageTables:
        """The tables of a step in which the sequence in `slots[i]` gets `new[i]` tokens (see `ops.page_tables`)."""
        self._check(tables)
        return ops.page_tables(slots, new, self.lengths, self.table, self.free, self.n_free, tables, max_new,
                               max_len or self.pages_per_slot * self.page_size)

    def advance(self, slots: torch.Tensor, new: torch.Tensor, tables: ops.PageTables) -> None:
        """That step has run."""
        self._check(tables)
        ops.page_advance(slots, new, self.lengths, self.n_free, tables)

    def release(self, slots: torch.Tensor) -> None:
        """The sequences in `slots` end."""
        ops.page_release(slots, self.lengths, self.table, self.free, self.n_free, self.page_size)
