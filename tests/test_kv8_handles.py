"""The 8-bit cache's handle without a GPU."""

from __future__ import annotations

import pytest
import torch

from solution.kernels import Kv8Cache


def _cache() -> Kv8Cache:
    return Kv8Cache.create(slots=4, max_tokens=100, num_kv_heads=2, head_dim=64, device="cpu")


@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_advance_counts_nothing_for_slots_that_are_none(kind: torch.dtype) -> None:
    """Rows without a sequence carry a slot outside the cache, as the kernels allow."""
    cache = _cache()
    slots = torch.tensor([2, -1, 0, 4, 1 << 30], dtype=torch.int32)
    cache.advance(3, slots)
    assert cache.lengths.tolist() == [3, 0, 3, 0]
    cache.advance(torch.tensor([1, 50, 2, 60, 70], dtype=kind), slots)
    assert cache.lengths.tolist() == [5, 0, 4, 0]
    cache.advance(7)
    cache.advance(torch.tensor([1, 2, 3, 4], dtype=kind))
    assert cache.lengths.tolist() == [13, 9, 14, 11]
