"""Steps of ``CachedDecoder``: how often they are captured, which of their tokens
count, and which weights they run with."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch
from conftest import MAX_ABS_TOL, REL_L2_TOL

from solution.kernels import pack_w4
from solution.runtimes import CachedDecoder, cached_decode, cuda_graph
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


@pytest.mark.gpu
@pytest.mark.parametrize("graph", [False, True])
def test_advance_counts_what_can_be_counted(graph: bool) -> None:
    config = WorkloadConfig(2, 400, 128, 2, 256, 2)
    model = _model(config)
    x = _randn(2, 400, 128)
    with torch.inference_mode():
        want = model(x)
    decoder = CachedDecoder(model, slots=2, max_tokens=400, weights="bf16", graph=graph)

    def lengths() -> list[int]:
        return [decoder.held, *decoder.cache.lengths.tolist()]

    with pytest.raises(ValueError, match="counted"):
        decoder.advance(1)  # nothing has been appended
    decoder.prompt(x[:, :60].contiguous())
    for n in (-1, 1):
        with pytest.raises(ValueError, match="counted"):
            decoder.advance(n)
    decoder.advance(0)
    # a draft over a block's end: three of nine, then two more, then none of the rest
    _near(decoder.step(x[:, 60:69].contiguous(), advance=False), want[:, 60:69])
    for n in (-1, 10):
        with pytest.raises(ValueError, match="counted"):
            decoder.advance(n)
    decoder.advance(3)
    with pytest.raises(ValueError, match="counted"):
        decoder.advance(7)
    decoder.advance(2)
    assert lengths() == [65, 65, 65]
    _near(decoder.step(x[:, 65:66].contiguous()), want[:, 65:66])
    with pytest.raises(ValueError, match="counted"):
        decoder.advance(1)
    # more than 64 tokens: all or nothing else
    _near(decoder.step(x[:, 66:166].contiguous(), advance=False), want[:, 66:166])
    for n in (0, 50, 99, 101, -1):
        with pytest.raises(ValueError, match="counted"):
            decoder.advance(n)
    with pytest.raises(ValueError, match="taken back"):
        decoder.step(x[:, 66:67].contiguous())
    assert lengths() == [66, 66, 66]
    decoder.advance(100)
    assert lengths() == [166, 166, 166]
    _near(decoder.step(x[:, 166:167].contiguous()), want[:, 166:167])
    # forgetting everything is always possible
    decoder.step(x[:, 167:267].contiguous(), advance=False)
    decoder.reset()
    assert lengths() == [0, 0, 0]
    _near(decoder.step(x[:, :70].contiguous()), want[:, :70])
    decoder.step(x[:, 70:270].contiguous(), advance=False)
    _near(decoder.prompt(x[:, :30].contiguous()), want[:, :30])
    _near(decoder.step(x[:, 30:31].contiguous()), want[:, 30:31])


@pytest.mark.gpu
@pytest.mark.parametrize(("slots", "tokens"), [(1, 1), (33, 1), (64, 1), (65, 1), (130, 1), (4, 16), (4, 17), (2, 100)])
def test_steps_of_any_size_run_with_the_packed_weights(slots: int, tokens: int) -> None:
    """Within the gate of the model that has the packed weights' values, and outside it for
    the one that has its own: weights of unlike size in one group make the two differ."""
    config = WorkloadConfig(slots, 40 + 2 * tokens, 128, 2, 256, 2)
    linears = lambda model: [  # noqa: E731
        linear for layer in model.layers
        for linear in (layer.attention.qkv_proj, layer.attention.out_proj, layer.ffn_in, layer.ffn_out)
    ]
    model, same = _model(config), _model(config)
    with torch.no_grad():
        for linear, other in zip(linears(model), linears(same)):
            linear.weight[:, ::2] *= 0.06  # beside full weights these round to none or one step
            other.weight.copy_(pack_w4(linear.weight).dequantize())
    x = _randn(slots, config.seq_len, 128)
    with torch.inference_mode():
        want, plain = same(x), model(x)
    decoder = CachedDecoder(model, slots=slots, max_tokens=config.seq_len)
    for t in range(0, config.seq_len - tokens + 1, tokens):
        got = decoder.step(x[:, t : t + tokens].contiguous())
        _near(got, want[:, t : t + tokens])
    with pytest.raises(AssertionError):
        _near(got, plain[:, t : t + tokens])


@pytest.mark.gpu
def test_a_step_that_fails_on_its_way(monkeypatch: pytest.MonkeyPatch) -> None:
    """Up to 64 tokens nothing is lost; more may have taken the place of older ones in the
    layers that came first, so that the sequences are forgotten."""
    config = WorkloadConfig(2, 300, 128, 2, 256, 2)
    model = _model(config)
    x = _randn(2, 300, 128)
    with torch.inference_mode():
        want = model(x)
    decoder = CachedDecoder(model, slots=2, max_tokens=300, weights="bf16", graph=False)
    decoder.prompt(x[:, :60].contiguous())
    attend, calls = cached_decode.sm100_kv8_attention, []

    def failing(*args, **kwargs):  # noqa: ANN002, ANN003, ANN202
        calls.append(args)
        if len(calls) == 2:
            raise RuntimeError("second layer")
        return attend(*args, **kwargs)

    for tokens in (40, 140):
        calls.clear()
        monkeypatch.setattr(cached_decode, "sm100_kv8_attention", failing)
        with pytest.raises(RuntimeError, match="second layer"):
            decoder.step(x[:, 60 : 60 + tokens].contiguous())
        monkeypatch.setattr(cached_decode, "sm100_kv8_attention", attend)
        if tokens == 40:
            assert decoder.held == 60
            _near(decoder.step(x[:, 60:61].contiguous(), advance=False), want[:, 60:61])
    assert [decoder.held, decoder.pending, *decoder.cache.lengths.tolist()] == [0, 0, 0, 0]
    _near(decoder.prompt(x[:, :30].contiguous()), want[:, :30])
    _near(decoder.step(x[:, 30:31].contiguous()), want[:, 30:31])


@pytest.mark.gpu
def test_graphs_of_many_shapes_share_their_memory() -> None:
    """Steps of changing sizes in turn give what the whole forward gives, and another shape costs
    no memory pool of its own (at least 20 MB, the allocator's segment)."""
    config = WorkloadConfig(2, 300, 128, 2, 256, 2)
    model = _model(config)
    x = _randn(2, 300, 128)
    with torch.inference_mode():
        want = model(x)
    decoder = CachedDecoder(model, slots=2, max_tokens=300, weights="bf16")
    at = 0
    for sizes in ((1, 2, 3), range(4, 16), (3, 15, 1, 2, 9, 1, 14, 4)):
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        before = torch.cuda.memory_reserved()
        for tokens in sizes:
            draft = x[:, at : at + tokens].contiguous()
            _near(decoder.step(draft, advance=False), want[:, at : at + tokens])
            keep = (tokens + 1) // 2
            decoder.advance(keep)
            at += keep
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        if len(sizes) == 12:
            assert torch.cuda.memory_reserved() - before <= 60 << 20
    assert len(decoder._replays) == 15
