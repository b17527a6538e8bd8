"""What the operators for many requests cannot run on is refused as such: at trace time too, and by the adapters' stack."""

from __future__ import annotations

import pytest
import torch

from solution.kernels import Kv8Cache, LowRankAdapters, ops  # noqa: F401 - registers the operators

B200 = torch.ops.b200tx
I32, F32 = torch.int32, torch.float32


def _meta(*shape, dtype=torch.bfloat16):  # noqa: ANN001, ANN002, ANN202
    return torch.empty(*shape, device="meta", dtype=dtype)


def _pool():  # noqa: ANN202
    cache = Kv8Cache.create(slots=3, max_tokens=256, num_kv_heads=1, head_dim=32, layers=2, device="cpu")
    tensors = (cache.codes, cache.scales, cache.tail, cache.page_table, cache.lengths, torch.zeros(cache.pages, dtype=I32))
    return [t.to("meta") for t in tensors]


@pytest.mark.parametrize(("rows", "inner", "outer"), [(5, 0, 40), (0, 64, 40), (5, 64, 0)])
def test_adapters_of_nothing(rows, inner, outer) -> None:  # noqa: ANN001
    with pytest.raises(ValueError):
        B200.low_rank_add(_meta(rows, inner), _meta(rows, outer), _meta(3, 8, inner), _meta(3, outer, 8), _meta(3, dtype=F32),
                          _meta(5, dtype=I32))


def test_pages_at_trace_time() -> None:
    pool = _pool()
    many = _meta(2049, dtype=I32)
    for call in (
        lambda: B200.kv8_fork(*pool, many, many),
        lambda: B200.kv8_fork(*pool, None, many),
        lambda: B200.kv8_reserve(*pool, -1),
        lambda: B200.kv8_reserve(*pool, 1, many),
        lambda: B200.kv8_reserve(*pool, 1, many[:0]),
        lambda: B200.kv8_reserve(*pool, 1, many[:2], many[:1]),
        lambda: B200.kv8_reserve(*pool, 1, None, many[:4]),
    ):
        with pytest.raises(ValueError):
            call()
    assert B200.kv8_fork(*pool, many[:2048], many[:2048]) is None
    assert tuple(B200.kv8_reserve(*pool, 0, many[:2048], many[:2048]).shape) == (2048,)
    assert tuple(B200.kv8_reserve(*pool, 0, None, many[:2]).shape) == (2,)


@pytest.mark.parametrize(("batch", "tokens", "vocab"), [(0, 2, 50), (2, 1025, 50), (2, 2, 0)])
def test_drafts_at_trace_time(batch, tokens, vocab) -> None:  # noqa: ANN001
    with pytest.raises(ValueError):
        B200.verify_draft(_meta(batch, tokens + 1, vocab), _meta(batch, tokens, dtype=I32), _meta(batch, tokens + 1, dtype=F32))


def test_a_stack_of_what_is_no_adapter() -> None:
    good = (torch.zeros(4, 16), torch.zeros(10, 4), 1.0)
    for bad in ((torch.tensor(1.0), good[1], 1.0), (good[0], torch.zeros(10), 1.0), (torch.zeros(2, 4, 16), good[1], 1.0),
                (torch.zeros(200, 16), torch.zeros(10, 4), 1.0)):
        for order in ([good, bad], [bad, good]):
            with pytest.raises(ValueError):
                LowRankAdapters.stack(order)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1024, 1025])
def test_drafts_of_too_many_tokens(tokens) -> None:  # noqa: ANN001
    from solution.kernels import can_use_sm100_verify_draft, sm100_verify_draft

    target = torch.full((2, tokens + 1, 8), 0.125, device="cuda")
    drafted = torch.zeros(2, tokens, dtype=torch.int64, device="cuda")
    uniform = torch.zeros(2, tokens + 1, device="cuda")
    if tokens == 1024:
        assert can_use_sm100_verify_draft(target, drafted)
        got, accepted, _ = sm100_verify_draft(target, drafted, uniform)
        assert accepted.tolist() == [1024, 1024] and not got.any()
        return
    assert not can_use_sm100_verify_draft(target, drafted)
    with pytest.raises(RuntimeError):
        sm100_verify_draft(target, drafted, uniform)
