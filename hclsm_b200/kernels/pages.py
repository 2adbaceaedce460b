"""Page tables of a state cache that many sequences share, kept on the device.

The pages of a pool are handed out and taken back as sequences grow and end.
Lengths are device tensors and no call reads them on the host, so a rollout
step (pages, slots, write, attention) captures into a CUDA graph.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch
from torch import Tensor

from .. import _lib

__all__ = ["PageTable", "pages_resize", "page_slots"]


@dataclass
class PageTable:
    """table (B, M) int32: each entry's pages in order, -1 behind them; free (P,) int32: a stack whose first
    ``n_free`` (1,) int32 places are the free pages; page: tokens of a page, a power of two."""

    table: Tensor
    free: Tensor
    n_free: Tensor
    page: int = 32

    @classmethod
    def empty(cls, batch: int, max_tokens: int, pages: int, *, page: int = 32, device="cuda") -> "PageTable":
        """No entry has a page; room for ``max_tokens`` tokens (rounded up to whole pages) an entry, page 0 on top of
        the stack of all ``pages``."""
        _check_page(page)
        if max_tokens < 0 or pages < 0:
            raise ValueError(f"max_tokens {max_tokens}, pages {pages}")

        def full(*shape):
            return torch.full(shape, -1, dtype=torch.int32, device=device)

        return cls(full(batch, (max_tokens + page - 1) // page),
                   torch.arange(pages - 1, -1, -1, dtype=torch.int32, device=device),
                   torch.full((1,), pages, dtype=torch.int32, device=device), page)


def _check_page(page):
    if page < 1 or page & (page - 1):
        raise ValueError(f"page must be a power of two, got {page}")


def _state(t, dim, name, dev):
    """A tensor that a call changes in place."""
    if t.dtype != torch.int32 or t.dim() != dim or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of {dim} dims, got {t.dtype} {tuple(t.shape)}")
    if t.device != dev:
        raise ValueError(f"{name} must be on {dev}")
    return t


def pages_resize(pages: PageTable, old_lens: Tensor, new_lens: Tensor) -> None:
    """Entries that held ``old_lens`` (B,) tokens hold ``new_lens`` (B,) from now on, in place.

    The pages this releases go onto the stack, the first (entries, then places ascending) on top; then the pages that
    are wanted come off its top in the same order, so giving up what was just taken puts all back as it was.
    A request that cannot be met (a length outside the table, too few free pages, a page outside the
    pool, a wanted place that holds a page already, as where ``old_lens`` is not what an entry has) changes nothing and
    sets the device error word."""
    dev = _lib.require_cuda(pages.table)
    table, free = _state(pages.table, 2, "table", dev), _state(pages.free, 1, "free", dev)
    n_free = _state(pages.n_free, 1, "n_free", dev)
    if n_free.numel() != 1:
        raise ValueError("n_free must have one element")
    _check_page(pages.page)
    B, M = table.shape
    old = _lib.index32(old_lens, (B,), "old_lens", dev)
    new = _lib.index32(new_lens, (B,), "new_lens", dev)
    if old is None or new is None:
        raise ValueError("old_lens and new_lens are required")
    lib, ws = _lib.load(), None
    n = lib.hclsm_pages_resize_workspace_size(B, M)
    if n:
        ws = table.new_empty(n, dtype=torch.uint8)
    _lib.check(lib.hclsm_pages_resize(table.data_ptr(), B, M, free.data_ptr(), n_free.data_ptr(), free.numel(), pages.page,
                                      old.data_ptr(), new.data_ptr(), _lib.ptr(ws), n, _lib.stream_ptr(dev)),
               "hclsm_pages_resize")
    _lib.changed(table, free, n_free)


def page_slots(table: Tensor, start: Tensor, n: int, *, count: Tensor | None = None, page: int = 32) -> Tensor:
    """Slots (B, n) int32 of tokens start[b], start[b] + 1, ...: page number * page + place in the page; -1
    behind the first ``count[b]`` (default n) of them and where the table (B, M) has no page; 2^31 - 1, behind every cache,
    for a page number that no slot holds."""
    dev = _lib.require_cuda(table)
    if table.dim() != 2:
        raise ValueError("table must be (B, M)")
    _check_page(page)
    if n < 0:
        raise ValueError(f"n must not be negative, got {n}")
    B, M = table.shape
    table = _lib.index32(table, (B, M), "table", dev)
    start = _lib.index32(start, (B,), "start", dev)
    if start is None:
        raise ValueError("start is required")
    count = _lib.index32(count, (B,), "count", dev)
    slots = table.new_empty((B, n))
    _lib.check(_lib.load().hclsm_page_slots(table.data_ptr(), B, M, page, start.data_ptr(), _lib.ptr(count), n,
                                            slots.data_ptr(), _lib.stream_ptr(dev)), "hclsm_page_slots")
    return slots
