"""The registered form of a fork from nothing."""

from __future__ import annotations

from types import SimpleNamespace

import torch

from solution.kernels import Kv8Cache, kv_pages, ops


def test_registered_fork_from_nothing_frees(monkeypatch) -> None:  # noqa: ANN001
    """It passes no source: a free neither reads one nor asks whether the tails can be addressed."""
    calls = []
    monkeypatch.setattr(kv_pages, "binding", lambda: SimpleNamespace(kv8_fork=lambda *a: calls.append(a)))
    cache = Kv8Cache.create(slots=2, max_tokens=200, num_kv_heads=1, head_dim=32, pages=5, device="cpu")
    tensors = (cache.codes, cache.scales, cache.tail, cache.page_table, cache.lengths, torch.zeros(5, dtype=torch.int32))
    target = torch.tensor([1, 0], dtype=torch.int32)
    ops.kv8_fork._init_fn(*tensors, None, target)
    ops.kv8_fork._init_fn(*tensors, target, target)
    assert calls[0][1] is None and calls[0][2] is target and calls[1][1] is target
