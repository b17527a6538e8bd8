"""Whose workspace an attention call over the 8-bit cache uses: calls on one
stream share one, a captured graph has its own."""

from __future__ import annotations

import threading

import pytest
import torch

from solution.kernels import Kv8Cache, sm100_kv8_append, sm100_kv8_attention

DEV = "cuda:0"


def _randn(*shape: int, seed: int) -> torch.Tensor:
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV)


def _filled(tokens: int) -> Kv8Cache:
    cache = Kv8Cache.create(slots=1, max_tokens=tokens, num_kv_heads=2, head_dim=64, device=DEV)
    sm100_kv8_append(cache, _randn(1, tokens, 6 * 64, seed=3).bfloat16(), 2)
    cache.advance(tokens - 1)
    return cache


def test_a_capture_has_a_workspace_of_its_own(monkeypatch: pytest.MonkeyPatch) -> None:
    """By stream outside of captures, by stream and capture inside; no GPU needed."""
    monkeypatch.setattr(Kv8Cache, "_new_workspace", lambda self: torch.zeros(16))
    cache = Kv8Cache.create(slots=1, max_tokens=64, num_kv_heads=1, head_dim=64, device="cpu")
    five, six = cache.workspace(5), cache.workspace(6)
    assert five is not six and cache.workspace(5) is five
    first = cache.workspace(5, 101)
    assert first is not five and cache.workspace(5, 101) is first
    fork = cache.workspace(6, 101)
    assert fork is not six and fork is not first and cache.workspace(5, 101) is first
    second = cache.workspace(5, 102)
    assert second is not first and second is not five and cache.workspace(5, 102) is second
    assert cache.workspace(5) is five and cache.workspace(6) is six


def test_workspaces_of_many_streams_are_given_up(monkeypatch: pytest.MonkeyPatch) -> None:
    """The oldest ones; a stream that comes back gets a new one; captures hold the last one's."""
    monkeypatch.setattr(Kv8Cache, "_new_workspace", lambda self: torch.zeros(16))
    cache = Kv8Cache.create(slots=1, max_tokens=64, num_kv_heads=1, head_dim=64, device="cpu")
    first = cache.workspace(1)
    for stream in range(2, 100):
        latest = cache.workspace(stream)
        assert cache.workspace(stream) is latest
        for capture in (2 * stream, 2 * stream + 1):
            cache.workspace(stream, capture)
        assert len(cache._workspaces) <= 8 and len(cache._captured) == 1
    assert cache.workspace(1) is not first


@pytest.mark.gpu
def test_a_replay_beside_calls_on_its_capture_stream() -> None:
    """A graph on one stream, calls on the stream that it was captured on, and another
    graph captured there on a third, all at once: each gives the bits that it gives alone."""
    with torch.inference_mode():
        cache = _filled(30000)  # one sequence over every SM: all tiles are split
        queries = [_randn(1, 1, 2, 64, seed=s).bfloat16() for s in range(3)]
        want = [sm100_kv8_attention(cache, q)[0].clone() for q in queries]
        capture, one, two = (torch.cuda.Stream() for _ in range(3))
        capture.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(capture):
            sm100_kv8_attention(cache, queries[0])
        torch.cuda.synchronize()
        graphs, outs = [], []
        for q in queries[:2]:
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=capture):
                # two calls of a capture share its workspace, as a model's layers do
                sm100_kv8_attention(cache, queries[2])
                outs.append(sm100_kv8_attention(cache, q)[0])
        for stream in (one, two, capture):
            stream.wait_stream(torch.cuda.current_stream())
        held = []
        for _ in range(50):
            for graph, stream in zip(graphs, (one, two)):
                with torch.cuda.stream(stream):
                    graph.replay()
            with torch.cuda.stream(capture):
                held.append(sm100_kv8_attention(cache, queries[2])[0])
        torch.cuda.synchronize()
        assert all(torch.equal(got, want[2]) for got in held)
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


@pytest.mark.gpu
def test_registered_operators_make_what_they_use(monkeypatch: pytest.MonkeyPatch) -> None:
    """Their handles live for one call: the append makes no workspace, the attention one,
    of which only the counters are cleared."""
    made = []
    make = Kv8Cache._new_workspace

    def counted(self: Kv8Cache) -> torch.Tensor:
        made.append(make(self))
        return made[-1]

    monkeypatch.setattr(Kv8Cache, "_new_workspace", counted)
    with torch.inference_mode():
        cache = _filled(300)
        parts = (cache.codes[0], cache.scales[0], cache.tail[0], cache.page_table, cache.lengths)
        made.clear()
        q = torch.ops.b200tx.kv8_append(*parts, _randn(1, 1, 6 * 64, seed=2).bfloat16(), 2)
        assert q.shape == (1, 1, 2, 64) and not made
        got = torch.ops.b200tx.kv8_attention(*parts, q)
        assert len(made) == 1 and torch.equal(got, sm100_kv8_attention(cache, q)[0])


@pytest.mark.gpu
def test_more_streams_than_workspaces() -> None:
    with torch.inference_mode():
        cache = _filled(30000)
        q = _randn(1, 1, 2, 64, seed=1).bfloat16()
        want = sm100_kv8_attention(cache, q)[0].clone()
        streams = [torch.cuda.Stream() for _ in range(12)]
        outs = []
        for stream in streams:
            stream.wait_stream(torch.cuda.current_stream())
        for _ in range(5):
            for stream in streams:
                with torch.cuda.stream(stream):
                    outs.append(sm100_kv8_attention(cache, q)[0])
        torch.cuda.synchronize()
        assert all(torch.equal(out, want) for out in outs)
        assert len(cache._workspaces) <= 8


@pytest.mark.gpu
def test_two_host_threads_on_one_cache() -> None:
    """Each on a stream of its own."""
    with torch.inference_mode():
        cache = _filled(30000)
        queries = [_randn(1, 1, 2, 64, seed=s).bfloat16() for s in range(2)]
        want = [sm100_kv8_attention(cache, q)[0].clone() for q in queries]
        torch.cuda.synchronize()
    wrong: list[object] = []

    def work(which: int) -> None:
        try:
            with torch.inference_mode(), torch.cuda.stream(torch.cuda.Stream()):
                outs = [sm100_kv8_attention(cache, queries[which])[0] for _ in range(100)]
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(out, want[which]) for out in outs):
                    wrong.append(which)
        except Exception as exc:  # noqa: BLE001 - told by the assertion below
            wrong.append(exc)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    assert not wrong
