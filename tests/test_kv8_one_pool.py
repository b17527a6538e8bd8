"""A cache's pages are one pool, whoever made the handle."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from solution.kernels import (
    Kv8Cache,
    Kv8Pages,
    sm100_kv8_compact,
    sm100_kv8_fork,
    sm100_kv8_free,
    sm100_kv8_reserve,
)
from solution.runtimes import CachedDecoder
from solution.transformer import UserOptimizedTransformer, copy_model_weights
from workloads import WorkloadConfig, seeded_state_dict

DEV = "cuda:0"


def _ints(values, device="cpu"):  # noqa: ANN001, ANN202
    return torch.tensor(values, dtype=torch.int32, device=device)


def _cache(device="cpu", pages=5):  # noqa: ANN001, ANN202
    return Kv8Cache.create(slots=2, max_tokens=200, num_kv_heads=1, head_dim=32, pages=pages, device=device)


def test_handles_of_one_cache_share_its_counts() -> None:
    cache = _cache()
    cache.page_table[0, :2] = _ints([4, 1])
    first = Kv8Pages(cache)
    cache.page_table[1, :1] = _ints([4])
    second = Kv8Pages(cache)  # counted anew, for both
    assert second.refs is first.refs and first.refs.tolist() == [0, 1, 0, 0, 2]
    assert Kv8Pages(cache, first.refs).refs is first.refs
    other = _cache()
    assert Kv8Pages(other).refs.tolist() == [0] * 5 and first.free == 3


def test_counts_of_the_callers_own_take_the_place_of_those_before() -> None:
    """Two handles that count apart would give out each other's pages: the last one made goes on, the one before is refused."""
    cache = _cache()
    before = Kv8Pages(cache)
    own = torch.ones(5, dtype=torch.int32)
    now = Kv8Pages(cache, own)
    one = _ints([0])
    for call in (lambda: sm100_kv8_fork(before, one, one), lambda: sm100_kv8_free(before, one), lambda: sm100_kv8_reserve(before, 1),
                 lambda: sm100_kv8_compact(before), before.recount):
        with pytest.raises(RuntimeError, match="other counts"):
            call()
    assert own.tolist() == [1] * 5
    now.recount()
    assert own.tolist() == [0] * 5
    assert Kv8Pages(cache).refs is own


def _model(config: WorkloadConfig) -> UserOptimizedTransformer:
    model = UserOptimizedTransformer(SimpleNamespace(**config.as_dict()))
    copy_model_weights(seeded_state_dict(config, 0), model)
    return model.to(DEV).eval()


def _randn(*shape: int, seed: int = 1) -> torch.Tensor:
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("graph", [True, False])
@pytest.mark.parametrize("made", ["before", "between", "decoder"])
def test_a_users_pool_beside_a_decoders(graph, made) -> None:  # noqa: ANN001
    """Slots that the user frees, forks and compacts by hand between a decoder's steps: bit for bit a decoder whose slots share
    nothing."""
    config = WorkloadConfig(4, 200, 128, 2, 256, 2)
    model = _model(config)
    shared = CachedDecoder(model, slots=4, max_tokens=256, weights="bf16", graph=graph)
    apart = CachedDecoder(model, slots=4, max_tokens=256, weights="bf16", graph=graph)
    pool = Kv8Pages(shared.cache) if made == "before" else None
    prompt = _randn(4, 130, 128)
    shared.prompt(prompt)
    if made != "before":
        shared.fork([1, 1, 2, 3])
        pool = shared.pages if made == "decoder" else Kv8Pages(shared.cache)
    else:
        sm100_kv8_fork(pool, _ints([1], DEV), _ints([0], DEV))
    apart.prompt(prompt[[1, 1, 2, 3]].contiguous())
    sm100_kv8_fork(pool, _ints([0, 3], DEV), _ints([3, 2], DEV))  # 1 1 3 1
    sm100_kv8_compact(pool)
    apart.prompt(prompt[[1, 1, 3, 1]].contiguous())

    def steps(n: int, seed: int, rows=(0, 1, 2, 3)) -> None:  # noqa: ANN001
        for i in range(n):
            x = _randn(4, 1, 128, seed=seed + i)
            got, want = shared.step(x), apart.step(x)
            assert torch.equal(got[list(rows)], want[list(rows)]), i

    steps(70, 100)
    refs = shared.pages.refs
    assert int(refs.max()) > 1 and torch.equal(refs, Kv8Pages(Kv8Cache(
        shared.cache.codes, shared.cache.scales, shared.cache.tail, shared.cache.page_table, shared.cache.lengths)).refs)
    # slots that share pages with others end, and fill pages again that must not be the others'
    sm100_kv8_free(pool, _ints([0], DEV))
    assert shared.cache.lengths.tolist() == [0, 200, 200, 200]
    sm100_kv8_compact(pool)
    steps(50, 300, (1, 2, 3))
    assert bool(shared.step(_randn(4, 1, 128))[0].isfinite().all())
    # the bound that the decoder keeps is looked up where slots may have ended
    sm100_kv8_free(pool, _ints([1, 2, 3], DEV))
    assert shared.step(_randn(4, 30, 128)).isfinite().all()


@pytest.mark.gpu
def test_a_pool_of_more_slots_than_a_call_takes() -> None:
    """Steps of a decoder that could not fork reserve their pages in several calls."""
    config = WorkloadConfig(2100, 8, 64, 2, 64, 1)
    model = _model(config)
    shared, apart = (CachedDecoder(model, slots=2100, max_tokens=128, weights="bf16") for _ in range(2))
    pool = Kv8Pages(shared.cache)
    sm100_kv8_free(pool, torch.arange(2048, dtype=torch.int32, device=DEV))
    sm100_kv8_free(pool, torch.arange(2048, 2100, dtype=torch.int32, device=DEV))
    assert pool.free == 4200
    for n, seed in ((40, 1), (40, 2), (1, 3)):
        x = _randn(2100, n, 64, seed=seed)
        assert torch.equal(shared.step(x), apart.step(x))
    assert pool.free == 2100 and int(pool.refs.max()) == 1


def test_the_same_counts_by_another_name() -> None:
    cache = _cache()
    first = Kv8Pages(cache)
    second = Kv8Pages(cache, first.refs.view(5, 1).view(5))
    assert second.refs is first.refs
    first.recount()
    second.recount()
    with pytest.raises(ValueError):
        Kv8Pages(cache, first.refs[:4])
    first.recount()
