"""Sequences and pages of the 8-bit cache moved about (csrc/kv8_pages_kernels.cuh).

``Kv8Cache.create`` gives each slot pages of its own.  With ``Kv8Pages`` the
pages are one pool: sequences with a common beginning share pages
(``sm100_kv8_fork``: samples of one prompt, beams), a slot whose request has
ended gives its pages back (``sm100_kv8_free``), pages are taken when tokens
come (``sm100_kv8_reserve``), and those in use are brought together
(``sm100_kv8_compact``), to be saved or sent as one piece of each layer.

    cache = Kv8Cache.create(slots=64, max_tokens=32768, pages=4096, ...)
    pages = Kv8Pages(cache)
    missing, _ = sm100_kv8_reserve(pages, 1)      # before a step of one token each
    ...                                           # sm100_kv8_append, sm100_kv8_attention
    cache.advance(1)
    sm100_kv8_fork(pages, source, target)         # between steps
    sm100_kv8_free(pages, ended)

Everything is decided on the device from the lengths and the table as they
are there, and nothing is read back, so the calls can be captured.  They change the
cache's ``page_table``, ``lengths``, ``tail`` and (compaction) ``codes`` and ``scales``
in place: calls on one pool follow one another on one stream, or are ordered by events.
"""

from __future__ import annotations

import ctypes

import torch

from .. import _native
from ._common import TensorHandle, binding, require
from .kv_cache import Kv8Cache

SM100_KV8_FORK_BACKEND = "sm100_kv8_fork"
SM100_KV8_RESERVE_BACKEND = "sm100_kv8_reserve"
SM100_KV8_COMPACT_BACKEND = "sm100_kv8_compact"
KV8_POOL_ROWS = 2048  # sequences of a call


class Kv8Pages(TensorHandle):
    """The pages of a cache as one pool.

    ``refs`` int32 ``[pages]`` counts the entries of the cache's ``page_table`` that hold a page; a
    page with none is free.  Counted from the table where it is not given; who
    changes the table by other means calls ``recount``.

    A cache has one pool: a further handle of it shares the counts.  One that is made with other
    ``refs`` takes their place, and calls on the handles before it are refused.
    """

    def __init__(self, cache: Kv8Cache, refs: torch.Tensor | None = None) -> None:
        counted = refs is None
        if counted:
            refs = torch.zeros(cache.pages, dtype=torch.int32, device=cache.device) if cache._pool is None else cache._pool[0]
        require(
            refs.dtype == torch.int32 and tuple(refs.shape) == (cache.pages,) and refs.is_contiguous()
            and refs.device == cache.device and refs.data_ptr() % 16 == 0,
            "refs must be a contiguous, 16-byte aligned int32 [pages] tensor on the cache's device",
        )
        if cache._pool is None or cache._pool[0].data_ptr() != refs.data_ptr():
            cache._pool = (refs, torch.zeros(_native.kv8_pool_scratch(cache.pages), dtype=torch.int32, device=cache.device))
        refs, scratch = cache._pool
        self.cache = cache
        self.refs = refs
        self._scratch = scratch
        self._struct = _native.Kv8PoolView(
            cache._views[0], cache.layers, refs.data_ptr(), self._scratch.data_ptr()
        )
        # what the binding takes: the struct's address and a tensor on the pool's device
        self._handle = (ctypes.addressof(self._struct), refs)
        if counted:
            self.recount()

    @property
    def handle(self) -> tuple[int, torch.Tensor]:
        """For the binding; RuntimeError where the cache's pages go by other counts since this was made."""

        if self.cache._pool[0] is not self.refs:
            raise RuntimeError("the cache's pages go by other counts: a Kv8Pages was made with refs of its own after this one")
        return self._handle

    def recount(self) -> None:
        """Count the table's entries anew."""

        self.handle  # noqa: B018 - refuses
        with torch.inference_mode():  # where the counts were made in that mode too
            flat = self.cache.page_table.reshape(-1).long()
            held = (flat >= 0) & (flat < self.cache.pages)
            self.refs.zero_().index_add_(0, torch.where(held, flat, 0), held.to(torch.int32))

    @property
    def free(self) -> int:
        """Free pages (read from the device)."""

        return int((self.refs <= 0).sum())


def sm100_kv8_fork(pages: Kv8Pages, source: torch.Tensor, target: torch.Tensor) -> tuple[torch.Tensor, str]:
    """Slot ``target[i]`` becomes what slot ``source[i]`` was before the call, for all pairs
    at once (int32 ``[n]``, ``n`` up to 2048): it shares the pages of the full blocks, gets a copy of the
    open block in its tail, and the length; the pages that it held are given up.  A slot may be one
    pair's source and another's target.  Tokens that are appended but not counted are
    forgotten in the targets.

    A source below 0 leaves the slot empty.  A pair with one slot twice, with a target that is none or a
    source past the slots does nothing; of pairs with one target the last counts.  Returns
    the lengths."""

    binding().kv8_fork(pages.handle, source, target)
    return pages.cache.lengths, SM100_KV8_FORK_BACKEND


def sm100_kv8_free(pages: Kv8Pages, slots: torch.Tensor) -> tuple[torch.Tensor, str]:
    """Empties the slots (int32 ``[n]``) and gives up their pages; those that no other
    slot shares are free.  A fork from nothing; returns the lengths."""

    binding().kv8_fork(pages.handle, None, slots)
    return pages.cache.lengths, SM100_KV8_FORK_BACKEND


def sm100_kv8_reserve(
    pages: Kv8Pages,
    tokens: int,
    *,
    slots: torch.Tensor | None = None,
    counts: torch.Tensor | None = None,
) -> tuple[torch.Tensor, str]:
    """Pages for the blocks that the next ``tokens`` of each sequence (``counts[b]`` of them where
    given, up to ``tokens``) may fill; rows and ``slots`` as in ``sm100_kv8_append``, which comes next with
    the same ones.  A block without a page, or with one that another sequence holds too, takes the lowest free page,
    in the order of rows and blocks.

    Returns ``missing`` int32 ``[B]``: the blocks that got none, as no page was free or the table
    ends before them (what is appended there is not stored, and reads as NaN).  Of rows with one slot
    the first counts."""

    return binding().kv8_reserve(pages.handle, tokens, slots, counts), SM100_KV8_RESERVE_BACKEND


def sm100_kv8_compact(pages: Kv8Pages) -> tuple[torch.Tensor, str]:
    """Brings the ``n`` pages in use to the front: the k-th one from page ``n`` on moves to the k-th
    free page below, in all layers, and the table and ``refs`` follow.  ``codes[:, :n]`` and ``scales[:, :n]`` hold all
    full blocks then; what a page held that moved stays behind in it.  Returns ``n``, int32
    ``[1]``."""

    return binding().kv8_compact(pages.handle), SM100_KV8_COMPACT_BACKEND


__all__ = [
    "KV8_POOL_ROWS",
    "Kv8Pages",
    "SM100_KV8_COMPACT_BACKEND",
    "SM100_KV8_FORK_BACKEND",
    "SM100_KV8_RESERVE_BACKEND",
    "sm100_kv8_compact",
    "sm100_kv8_fork",
    "sm100_kv8_free",
    "sm100_kv8_reserve",
]
