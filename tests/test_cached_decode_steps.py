"""Steps of ``CachedDecoder``: how often they are captured."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch
from conftest import MAX_ABS_TOL, REL_L2_TOL

from solution.runtimes import CachedDecoder, cuda_graph
from solution.transformer import UserOptimizedTransformer, copy_model_weights
from workloads import WorkloadConfig, seeded_state_dict

DEV = "cuda:0"


def _model(config: WorkloadConfig, device: str = DEV) -> UserOptimizedTransformer:
    model = UserOptimizedTransformer(SimpleNamespace(**config.as_dict()))
    copy_model_weights(seeded_state_dict(config, 0), model)
    return model.to(device).eval()


def _randn(*shape: int, seed: int = 1) -> torch.Tensor:
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(DEV)


def _near(got: torch.Tensor, want: torch.Tensor) -> None:
    diff = got.float() - want.float()
    rel = float(diff.norm() / want.float().norm())
    assert float(diff.abs().max()) <= MAX_ABS_TOL and rel <= REL_L2_TOL, (float(diff.abs().max()), rel)


@pytest.mark.gpu
def test_fresh_inputs_replay_one_graph(monkeypatch: pytest.MonkeyPatch) -> None:
    """Every token comes in a tensor of its own: one capture for each shape and dtype, and no
    more workspaces as the steps go on."""
    captures = []
    capture = cuda_graph.capture_program
    monkeypatch.setattr(cuda_graph, "capture_program", lambda *args: captures.append(args) or capture(*args))
    config = WorkloadConfig(2, 120, 128, 2, 256, 2)
    model = _model(config)
    x = _randn(2, 120, 128)
    with torch.inference_mode():
        want = model(x)
    decoder = CachedDecoder(model, slots=2, max_tokens=120, weights="bf16")
    tokens = [x[:, t : t + 1].contiguous() for t in range(80)]  # all alive: no address comes again
    outs = [decoder.step(token) for token in tokens[:3]]
    spaces = len(decoder.cache._workspaces)
    outs += [decoder.step(token) for token in tokens[3:]]
    assert len(captures) == 1 and len(decoder.cache._workspaces) == spaces
    assert len({out.data_ptr() for out in outs}) == len(outs)  # each output is the caller's
    _near(torch.cat(outs, 1), want[:, :80])
    kept = x[:, 80:81].contiguous()
    _near(decoder.step(kept), want[:, 80:81])
    _near(decoder.step(kept.copy_(x[:, 81:82])), want[:, 81:82])  # a buffer that is used again
    assert len(captures) == 1
    for t in (82, 86):
        _near(decoder.step(x[:, t : t + 4].contiguous()), want[:, t : t + 4])
    _near(decoder.step(x[:, 90:91].contiguous().bfloat16()), want[:, 90:91])
    assert len(captures) == 3
