"""``CachedDecoder``: prompt and steps against the model's own whole forward.

Tolerances.  With the model's own weights a step differs from the forward by
the cache's rounding: a code is off by at most half a step of max / 254, some
1/100 of a value's typical size, on keys and values alike; the attention's
part of the fp32 residual carries that, and the gate of the repository (max-abs
2e-2, rel-L2 1e-2) must still hold.  With 4-bit weights the model to compare
with is the one that has the packed weights' values.
"""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch
from conftest import MAX_ABS_TOL, REL_L2_TOL

from solution.kernels import RotaryTable, pack_w4, sm100_flash_attention, sm100_qk_norm_rope
from solution.runtimes import CachedDecoder
from solution.transformer import UserOptimizedTransformer
from workloads import WorkloadConfig, seeded_state_dict

DEV = "cuda:0"


def _model(config: WorkloadConfig, device: str = DEV, weights=None) -> UserOptimizedTransformer:  # noqa: ANN001
    from solution.transformer import copy_model_weights

    model = UserOptimizedTransformer(SimpleNamespace(**config.as_dict()))
    copy_model_weights(seeded_state_dict(config, 0), model)
    if weights is not None:
        with torch.no_grad():
            weights(model)
    return model.to(device).eval()


def _near(got: torch.Tensor, want: torch.Tensor) -> None:
    diff = (got.float() - want.float())
    rel = float(diff.norm() / want.float().norm())
    assert float(diff.abs().max()) <= MAX_ABS_TOL and rel <= REL_L2_TOL, (float(diff.abs().max()), rel)


def test_refusals_without_a_gpu() -> None:
    config = WorkloadConfig(1, 8, 128, 4, 128, 1)
    model = _model(config, "cpu")
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        CachedDecoder(model, slots=1, max_tokens=64)
    with pytest.raises(ValueError, match="head_dim"):
        CachedDecoder(_model(WorkloadConfig(1, 8, 128, 16, 128, 1), "cpu"), slots=1, max_tokens=64)
    with pytest.raises(ValueError, match="causal"):
        CachedDecoder(_model(WorkloadConfig(1, 8, 128, 4, 128, 1, False), "cpu"), slots=1, max_tokens=64)
    with pytest.raises(ValueError, match="weights"):
        CachedDecoder(model, slots=1, max_tokens=64, weights="int3")
    with pytest.raises(ValueError, match="qk_norms"):
        CachedDecoder(model, slots=1, max_tokens=64, qk_norms=[])


@pytest.mark.gpu
@pytest.mark.parametrize(
    ("config", "prompt", "graph"),
    [
        (WorkloadConfig(3, 150, 256, 4, 512, 2), 61, True),  # steps over two blocks' ends
        (WorkloadConfig(2, 140, 128, 4, 128, 3), 64, True),  # head_dim 32
        (WorkloadConfig(1, 80, 256, 2, 256, 2), 7, False),  # head_dim 128
        (WorkloadConfig(1, 70, 512, 2, 256, 1), 40, True),  # head_dim 256
    ],
)
def test_steps_match_the_whole_forward(config: WorkloadConfig, prompt: int, graph: bool) -> None:
    model = _model(config)
    x = torch.randn(config.batch_size, config.seq_len, config.d_model, generator=torch.Generator().manual_seed(1)).to(DEV)
    with torch.inference_mode():
        want = model(x)
    decoder = CachedDecoder(model, slots=config.batch_size, max_tokens=config.seq_len, weights="bf16", graph=graph)
    _near(decoder.prompt(x[:, :prompt].contiguous()), want[:, :prompt])
    buffer = torch.empty(config.batch_size, 1, config.d_model, device=DEV)
    for t in range(prompt, config.seq_len - 5):
        buffer.copy_(x[:, t : t + 1])
        _near(decoder.step(buffer), want[:, t : t + 1])
    # the last five at once, and again after they were not counted
    last = x[:, -5:].contiguous()
    first = decoder.step(last, advance=False)
    _near(first, want[:, -5:])
    assert torch.equal(decoder.step(last), first)
    with pytest.raises(ValueError, match="pass the cache"):
        decoder.step(last)
    decoder.reset()
    assert decoder.held == 0 and int(decoder.cache.lengths.sum()) == 0


@pytest.mark.gpu
def test_w4_steps_match_the_model_with_the_packed_weights() -> None:
    config = WorkloadConfig(2, 100, 256, 4, 512, 2)

    def quantise(model: UserOptimizedTransformer) -> None:
        for layer in model.layers:
            for linear in (layer.attention.qkv_proj, layer.attention.out_proj, layer.ffn_in, layer.ffn_out):
                linear.weight.copy_(pack_w4(linear.weight).dequantize())

    model = _model(config)
    same = _model(config, weights=quantise)
    x = torch.randn(2, 100, 256, generator=torch.Generator().manual_seed(1)).to(DEV)
    with torch.inference_mode():
        want = same(x)
    decoder = CachedDecoder(model, slots=2, max_tokens=128)
    got = torch.cat([decoder.step(x[:, t : t + 1].contiguous()) for t in range(0, 90)], 1)
    _near(got, want[:, :90])
    _near(decoder.step(x[:, 90:].contiguous()), want[:, 90:])  # 20 rows


@pytest.mark.gpu
def test_rotation_and_norms_in_prompt_and_steps() -> None:
    """A prompt at once and the same tokens one by one leave the same cache, and
    the steps' outputs agree with the prompt's."""
    config = WorkloadConfig(2, 90, 256, 4, 256, 2)
    model = _model(config)
    g = torch.Generator().manual_seed(5)
    norms = [tuple(1 + 0.1 * torch.randn(64, generator=g).to(DEV) for _ in range(2)) for _ in range(2)]
    rope = RotaryTable.create(128, 64, DEV)
    x = torch.randn(2, 90, 256, generator=g).to(DEV)
    whole = CachedDecoder(model, slots=2, max_tokens=128, weights="bf16", rope=rope, qk_norms=norms)
    steps = CachedDecoder(model, slots=2, max_tokens=128, weights="bf16", rope=rope, qk_norms=norms)
    want = whole.prompt(x)
    got = torch.cat([steps.step(x[:, t : t + 1].contiguous()) for t in range(90)], 1)
    _near(got, want)
    # the first layer's keys and values depend on the inputs alone
    assert torch.equal(steps.cache.codes[0, steps.cache.page_table[:, 0].long()], whole.cache.codes[0, whole.cache.page_table[:, 0].long()])
    # and the rotation does something: without it the outputs are others
    plain = CachedDecoder(model, slots=2, max_tokens=128, weights="bf16").prompt(x)
    assert float((plain - want).abs().max()) > 10 * MAX_ABS_TOL
    with torch.inference_mode():  # what the prompt attends to is the packed projection, turned in place
        qkv = torch.randn(1, 9, 3 * 256, generator=g).bfloat16().to(DEV)
        turned, _ = sm100_qk_norm_rope(qkv, 4, q_weight=norms[0][0], k_weight=norms[0][1], rope=rope)
        assert sm100_flash_attention(turned, 4)[0].shape == (1, 9, 256)
