"""Handles of the decoding operators without a GPU."""

from __future__ import annotations

import pytest
import torch

from solution.kernels import Kv8Cache, RotaryTable, pack_w4


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


def test_tensors_of_a_handle_are_not_exchanged() -> None:
    """The kernels read them at the addresses taken when the handle was made."""
    table, weight = RotaryTable.create(16, 8, "cpu"), pack_w4(torch.randn(8, 64))
    for handle, names in (
        (_cache(), ("codes", "scales", "tail", "page_table", "lengths")),
        (table, ("cos", "sin")),
        (weight, ("packed", "scales")),
    ):
        for name in names:
            held = getattr(handle, name)
            with pytest.raises(AttributeError, match="in place"):
                setattr(handle, name, held.clone())
            with pytest.raises(AttributeError, match="in place"):
                setattr(handle, name, None)
            assert getattr(handle, name) is held
    cache = _cache()
    at = cache.lengths.data_ptr()
    cache.lengths += 5
    cache.lengths[1] = 2
    assert cache.lengths.tolist() == [5, 2, 5, 5] and cache.lengths.data_ptr() == at
