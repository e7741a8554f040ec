"""An engine: one bound model, its cache, and the step function over them."""
from __future__ import annotations

import torch

from ..cache.kv import E4M3, PAGE_SIZE, Cache
from .step import StepEntry, step


def _cache_dtype(model, cache_dtype):
    """The type of the cache's keys and values; refuses a model with a mixer that does not take it."""
    if cache_dtype is None:
        return model.dtype
    if cache_dtype not in ("e4m3", E4M3):
        raise ValueError(f"cache_dtype must be None (the model's own) or 'e4m3', got {cache_dtype!r}")
    for i, e in enumerate(model.spec.schedule):
        block = model.blocks[e.layer]
        if block.kv_need() is not None and not getattr(getattr(block, "mixer", None), "takes_e4m3", False):
            raise ValueError(f"layer {e.layer} (schedule entry {i}): its mixer does not take a cache held in 8 bits")
    return E4M3


class Engine:
    """Owns the cache of a model and runs steps on it.

    `max_tokens` is the most tokens live sequences may hold together, each sequence's count
    rounded up to a whole cache page (64 tokens); it sizes the cache.  `cache_dtype` "e4m3" keeps keys and values in 8 bits
    with a power-of-two scale for each page and head (models whose layers all mix by plain attention): half the bytes of
    bfloat16, three bits behind a number's first one."""

    PAGE_SIZE = PAGE_SIZE

    def __init__(self, model, max_tokens: int, n_slots: int | None = None, cache_dtype=None):
        self.model = model
        self.use_decode_loop = True
        self.cache = Cache(model.kv_needs(), model.state_needs(), max_tokens,
                           dtype=model.dtype, device=model.device, n_slots=n_slots,
                           model_state=model.model_state_needs(), kv_dtype=_cache_dtype(model, cache_dtype))

    def open(self) -> int:
        """A slot for a new sequence."""
        return self.cache.open()

    def close(self, slot: int) -> None:
        """Gives the sequence's slot and pages back."""
        self.cache.close(slot)

    def length(self, slot: int) -> int:
        return self.cache.length(slot)

    @property
    def page_size(self) -> int:
        return self.cache.page_size

    def free_pages(self) -> int:
        """Pages every group can still hand out."""
        return min((g.pool.free_count for g in self.cache.groups), default=0)

    def free_slots(self) -> int:
        return self.cache.slots.free_count

    def decode_loop(self, slots, budgets, samplings):
        """The captured decode step for these live sequences, or None when it cannot serve
        them (penalties need each sequence's token history on the host).  `budgets`: the most
        tokens each of them will still be asked for; each gets pages for its own budget.  A
        windowed cache group holds those pages for the life of the loop and gives back the
        ones its window has left behind when the loop is closed."""
        from .decode import DecodeLoop
        if not self.use_decode_loop or any(s.penalizes for s in samplings):
            return None
        return DecodeLoop(self, slots, budgets, samplings)

    def step(self, entries) -> torch.Tensor:
        """entries: StepEntry items or (slot, tokens, want) tuples."""
        entries = [e if isinstance(e, StepEntry) else StepEntry(e[0], list(e[1]), list(e[2]))
                   for e in entries]
        return step(self.model, self.cache, entries)
