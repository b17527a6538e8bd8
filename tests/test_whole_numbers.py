"""Slots' adapters and parents in every whole type that torch has, and in none besides."""

from __future__ import annotations

import pytest
import torch

from solution.runtimes import CachedDecoder
from solution.kernels import LowRankAdapters


def _decoder(slots: int = 3) -> CachedDecoder:
    """What ``set_adapters`` looks at, without a GPU."""
    decoder = object.__new__(CachedDecoder)
    decoder.slots, decoder.pending = slots, 0
    small, large = (
        LowRankAdapters(torch.zeros(n, 8, 8).bfloat16(), torch.zeros(n, 8, 8).bfloat16(), torch.ones(n)) for n in (2, 5)
    )
    decoder.adapters = [{"qkv": large}, {"out": small}]
    decoder.adapter_indices = torch.full((slots,), -1, dtype=torch.int32)
    return decoder


WHOLE = [torch.uint8, torch.uint16, torch.uint32, torch.uint64, torch.int8, torch.int16, torch.int32, torch.int64]


@pytest.mark.parametrize("dtype", WHOLE)
def test_adapters_of_slots(dtype) -> None:  # noqa: ANN001
    decoder = _decoder()
    decoder.set_adapters(torch.tensor([0, 1, 0], dtype=dtype))
    assert decoder.adapter_indices.tolist() == [0, 1, 0]
    with pytest.raises(ValueError, match="adapter 2 of 2"):
        decoder.set_adapters(torch.tensor([0, 1, 2], dtype=dtype))
    most = torch.iinfo(dtype).max
    with pytest.raises(ValueError, match="adapter"):
        decoder.set_adapters(torch.tensor([0, 1, 0], dtype=dtype).fill_(most))
    if dtype.is_signed:
        decoder.set_adapters(torch.tensor([0, torch.iinfo(dtype).min, -1], dtype=dtype))
        assert decoder.adapter_indices.tolist() == [0, -1, -1]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float8_e4m3fn, torch.bool, torch.complex64, torch.complex128])
def test_other_types_are_refused(dtype) -> None:  # noqa: ANN001
    decoder = _decoder()
    for call in (decoder.set_adapters, decoder.fork):
        with pytest.raises(ValueError, match="whole numbers"):
            call(torch.zeros(3).to(dtype))
    with pytest.raises(ValueError, match="whole numbers"):
        decoder.fork([0, 1j, 2])
    assert decoder.adapter_indices.tolist() == [-1, -1, -1]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.uint16, torch.uint32, torch.uint64])
def test_parents_in_unsigned_types(dtype) -> None:  # noqa: ANN001
    from types import SimpleNamespace

    from solution.transformer import UserOptimizedTransformer
    from workloads import WorkloadConfig

    config = WorkloadConfig(3, 40, 128, 2, 128, 1)
    model = UserOptimizedTransformer(SimpleNamespace(**config.as_dict())).to("cuda:0").eval()
    n, k = model.layers[0].attention.out_proj.weight.shape
    adapters = LowRankAdapters.stack([(torch.zeros(8, k), torch.zeros(n, 8), 1.0)] * 2, "cuda:0")
    decoder = CachedDecoder(model, slots=3, max_tokens=64, weights="bf16", adapters=[{"out": adapters}])
    decoder.prompt(torch.zeros(3, 5, 128, device="cuda:0"))
    decoder.step(torch.zeros(3, 1, 128, device="cuda:0"))
    decoder.set_adapters([0, 1, -1])
    for device in ("cpu", "cuda:0"):
        decoder.set_adapters(torch.tensor([0, 1, 1], dtype=dtype, device=device))
        decoder.fork(torch.tensor([1, 0, torch.iinfo(dtype).max], dtype=dtype, device=device))  # past the slots: it stays as it is
        assert decoder.adapter_indices.tolist() == [1, 0, 1] and decoder.cache.lengths.tolist() == [6, 6, 6]
