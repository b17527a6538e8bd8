"""A decoder's slots that take requests one after the other."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch
from conftest import MAX_ABS_TOL

from solution.runtimes import CachedDecoder
from solution.transformer import UserOptimizedTransformer, copy_model_weights
from workloads import WorkloadConfig, seeded_state_dict

DEV = "cuda:0"


def _ints(values):  # noqa: ANN001, ANN202
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _model(config: WorkloadConfig) -> UserOptimizedTransformer:
    model = UserOptimizedTransformer(SimpleNamespace(**config.as_dict()))
    copy_model_weights(seeded_state_dict(config, 0), model)
    return model.to(DEV).eval()


def _randn(*shape: int, seed: int = 1) -> torch.Tensor:
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(DEV)


@pytest.mark.gpu
def test_a_slot_begins_anew_among_others() -> None:
    """A slot that is emptied reads a new request's tokens in steps that count nothing for the others."""
    config = WorkloadConfig(3, 100, 128, 2, 256, 2)
    model = _model(config)
    decoder = CachedDecoder(model, slots=3, max_tokens=192, weights="bf16")
    x = _randn(3, 100, 128)
    decoder.prompt(x[:, :80].contiguous())
    decoder.fork([0, -1, 2])
    request = _randn(1, 90, 128, seed=5)
    for begin, end in ((0, 64), (64, 90)):
        given = _randn(3, end - begin, 128, seed=6)  # what the others are given does not count
        given[1] = request[0, begin:end]
        decoder.step(given, advance=False)
        decoder.advance(_ints([0, end - begin, 0]))
    assert decoder.cache.lengths.tolist() == [80, 90, 80]
    alone = CachedDecoder(model, slots=3, max_tokens=192, weights="bf16")
    alone.prompt(x[:, :80].contiguous())
    fresh = CachedDecoder(model, slots=1, max_tokens=192, weights="bf16")
    for begin, end in ((0, 64), (64, 90)):
        fresh.step(request[:, begin:end].contiguous())
    for i in range(40):
        x = _randn(3, 1, 128, seed=20 + i)
        got, others, one = decoder.step(x), alone.step(x), fresh.step(x[1:2].contiguous())
        assert torch.allclose(got[[0, 2]], others[[0, 2]], atol=MAX_ABS_TOL, rtol=0) and torch.allclose(got[1:2], one, atol=MAX_ABS_TOL, rtol=0)
