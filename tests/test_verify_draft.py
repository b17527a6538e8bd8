"""Verification of drafted tokens against plain loops in 64 bits.  Sums in 64 bits differ by 2^-52 of themselves a
term, so at random numbers of 24 bits and these sizes no border is that near: tokens and counts are equal."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from solution import _native
from solution.kernels import can_use_sm100_verify_draft, sm100_verify_draft

gpu = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _inference():
    with torch.inference_mode():
        yield
    if torch.cuda.is_available():
        torch.cuda.synchronize()


def _plain(target, drafted, uniform, draft=None, counts=None):  # noqa: ANN001, ANN202
    target, uniform = target.double().cpu().numpy(), uniform.double().cpu().numpy()
    draft = None if draft is None else draft.double().cpu().numpy()
    tokens = drafted.cpu().numpy()
    batch, most = tokens.shape
    out, accepted = np.full((batch, most + 1), -1, dtype=np.int64), np.zeros(batch, dtype=np.int64)
    vocab = target.shape[2]
    for b in range(batch):
        n = most if counts is None else min(max(int(counts[b]), 0), most)
        t = 0
        while t < n:
            d = int(tokens[b, t])
            if not 0 <= d < vocab or not uniform[b, t] * (1.0 if draft is None else draft[b, t, d]) < target[b, t, d]:
                break
            out[b, t] = d
            t += 1
        mass = target[b, t].copy()
        if t < n:
            if draft is not None:
                mass = mass - draft[b, t]
            elif 0 <= int(tokens[b, t]) < vocab:
                mass[int(tokens[b, t])] = 0
            if not (mass > 0).any():
                mass = target[b, t].copy()
        mass = np.where(mass > 0, mass, 0)
        sums = np.cumsum(mass)
        past = np.flatnonzero(sums > max(uniform[b, -1], 0) * sums[-1])
        held = np.flatnonzero(mass)
        out[b, t] = past[0] if len(past) else held[-1] if len(held) else -1
        accepted[b] = t
    return out, accepted


def _check(target, drafted, uniform, draft=None, counts=None):  # noqa: ANN001, ANN202
    tokens, accepted, marker = sm100_verify_draft(target, drafted, uniform, draft=draft, counts=counts)
    want, many = _plain(target, drafted, uniform, draft, None if counts is None else counts.tolist())
    assert tokens.dtype == drafted.dtype and accepted.dtype == torch.int32 and marker == "sm100_verify_draft"
    assert accepted.tolist() == many.tolist()
    assert tokens.tolist() == want.tolist()
    return tokens, accepted


def _case(batch, tokens, vocab, seed, dtype=torch.float32, sharp=2.0):  # noqa: ANN001, ANN202
    g = torch.Generator(device="cuda").manual_seed(seed)
    logits = sharp * torch.randn(batch, tokens + 1, vocab, generator=g, device="cuda")
    target = torch.softmax(logits, -1).to(dtype)
    draft = torch.softmax(logits[:, :-1] + 0.5 * torch.randn(batch, tokens, vocab, generator=g, device="cuda"), -1).to(dtype)
    drafted = torch.multinomial(draft.float().flatten(0, 1), 1, generator=g).view(batch, tokens) if tokens else \
        torch.zeros(batch, 0, dtype=torch.int64, device="cuda")
    return target, draft, drafted, torch.rand(batch, tokens + 1, generator=g, device="cuda")


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize(
    ("batch", "tokens", "vocab"),
    [(1, 1, 1), (2, 3, 5), (3, 0, 17), (64, 4, 127), (5, 2, 1024), (17, 8, 4001), (2, 31, 32000), (4, 5, 65537), (3, 2, 300003)],
)
def test_verify_draft(dtype, batch, tokens, vocab) -> None:  # noqa: ANN001
    target, draft, drafted, uniform = _case(batch, tokens, vocab, vocab + tokens, dtype)
    counts = torch.randint(-1, tokens + 2, (batch,), device="cuda", dtype=torch.int32,
                           generator=torch.Generator(device="cuda").manual_seed(1))
    for kwargs in ({}, {"draft": draft}, {"counts": counts}, {"draft": draft, "counts": counts}):
        _check(target, drafted, uniform, **kwargs)
        _check(target, drafted.to(torch.int32), uniform, **kwargs)


@gpu
def test_borders() -> None:
    """u q = p refuses, u = 0 takes what has mass, u next to 1 the last with mass, one-hot rows, equal rows, nothing left."""
    low, high = 0.0, 1 - 2.0**-24
    target = torch.zeros(9, 2, 1000, device="cuda")
    draft = torch.zeros(9, 1, 1000, device="cuda")
    drafted = torch.full((9, 1), 7, device="cuda")
    uniform = torch.zeros(9, 2, device="cuda")
    target[:, 0, 7], target[:, 0, 900], draft[:, 0, 7] = 0.25, 0.75, 0.5
    target[:, 1, [3, 4, 999]] = torch.tensor([0.25, 0.5, 0.25], device="cuda")
    uniform[0] = torch.tensor([0.5, high])  # 0.25 < 0.25 is not so: refused; the rest is 0.75 at 900
    uniform[1] = torch.tensor([0.5 - 2.0**-25, 0.25])  # counts; at 0.25 of the last row the sum 0.25 does not pass
    uniform[2] = torch.tensor([0.0, low])
    uniform[3] = torch.tensor([0.0, high])
    uniform[4] = torch.tensor([0.9, low])
    draft[5], uniform[5] = target[5, 0], torch.tensor([high, 0.5])  # equal: always counts
    drafted[6, 0], draft[6] = 8, target[6, 0]  # refused, and nothing is left of max(p - q, 0): from p
    target[7], uniform[7] = 0, torch.tensor([0.3, 0.3])  # no mass at all
    uniform[8] = torch.tensor([0.4, 1.0])  # past the documented range: the last with mass
    tokens, accepted = _check(target, drafted, uniform, draft)
    assert accepted.tolist() == [0, 1, 1, 1, 0, 1, 0, 0, 1]
    assert tokens.tolist() == [[900, -1], [7, 4], [7, 3], [7, 999], [900, -1], [7, 4], [7, -1], [-1, -1], [7, 999]]
    _check(target, drafted, uniform)
    for bad in (-1, 1000, -(1 << 40), 1 << 40):
        drafted[:3] = bad
        _check(target, drafted, uniform, draft)
        _check(target, drafted, uniform)


@gpu
def test_values_that_are_no_probabilities() -> None:
    target, draft, drafted, uniform = _case(6, 2, 700, 3)
    target[0, 0, 100:300] = torch.nan  # no mass
    drafted[0, 0] = 150
    target[1] = torch.nan
    draft[2, :, ::2] = torch.nan
    draft[3] = torch.nan
    target[4, :, 5] = torch.inf
    target[5] *= 1000  # not normed
    target[5, :, 11] = -4
    drafted[4:, 0] = 9
    uniform[4:, 0] = 0.999
    with np.errstate(invalid="ignore"):
        _check(target, drafted, uniform)
        _check(target, drafted, uniform, draft)
    uniform[5] = torch.nan
    with np.errstate(invalid="ignore"):
        tokens, accepted, _ = sm100_verify_draft(target, drafted, uniform, draft=draft)
    assert int(accepted[5]) == 0  # a number that is none refuses, and draws as 0 does


@gpu
def test_many_small_masses() -> None:
    """A long flat row: the running sum of 64 bits finds the index, a sum of 32 bits would be off by tens."""
    vocab = 1 << 18
    target = torch.full((4, 1, vocab), 1.0 / 3, device="cuda")
    uniform = torch.tensor([[0.1], [0.5], [0.999999], [0.33333]], device="cuda")
    drafted = torch.zeros(4, 0, dtype=torch.int64, device="cuda")
    tokens, _ = _check(target, drafted, uniform)
    assert tokens[:, 0].tolist() == [int(float(u) * vocab) for u in uniform[:, 0]]


@gpu
def test_strides_streams_and_graphs() -> None:
    target, draft, drafted, uniform = _case(5, 4, 1000, 4)
    for pad, shift in ((24, 0), (24, 4), (3, 1), (1, 0)):  # padded vocabularies; rows that start anywhere
        wide = torch.full((5, 5, 1000 + pad), 7.0, device="cuda")
        view = wide[..., shift : shift + 1000]
        view.copy_(target)
        _check(view, drafted, uniform, draft)
        other = torch.full((5, 4, 1000 + pad), 7.0, device="cuda")[..., shift : shift + 1000]
        other.copy_(draft)
        _check(target, drafted, uniform, other)
    swapped = target.transpose(0, 1).contiguous().transpose(0, 1)
    _check(swapped, drafted, uniform, draft)
    _check(target[:1].expand(5, 5, 1000), drafted, uniform, draft[:1].expand(5, 4, 1000))
    want, many = _check(target, drafted, uniform, draft)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            tokens, accepted, _ = sm100_verify_draft(target, drafted, uniform, draft=draft)
        graph.replay()
    stream.synchronize()
    assert torch.equal(tokens, want) and torch.equal(accepted, many)
    uniform.copy_(uniform.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    again = _check(target, drafted, uniform, draft)
    assert torch.equal(tokens, again[0]) and torch.equal(accepted, again[1])


@gpu
def test_tokens_are_distributed_as_the_targets() -> None:
    """The token of the first place, drafted or drawn anew, has the target's probabilities: 200000 draws over 8 tokens, each
    share within 5 standard deviations (a seeded draw, so it does not vary from run to run)."""
    n, vocab = 200000, 8
    g = torch.Generator(device="cuda").manual_seed(11)
    p = torch.softmax(torch.randn(vocab, generator=g, device="cuda"), 0)
    q = torch.softmax(torch.randn(vocab, generator=g, device="cuda"), 0)
    drafted = torch.multinomial(q, n, replacement=True, generator=g)[:, None]
    uniform = torch.rand(n, 2, generator=g, device="cuda")
    tokens, _, _ = sm100_verify_draft(p.expand(n, 2, vocab), drafted, uniform, draft=q.expand(n, 1, vocab))
    share = torch.bincount(tokens[:, 0], minlength=vocab).double() / n
    assert bool(((share - p.double()).abs() <= 5 * (p.double() * (1 - p.double()) / n).sqrt()).all())


@gpu
def test_beyond_32_bit_offsets() -> None:
    target = torch.zeros(40, 2, 1 << 25, dtype=torch.bfloat16, device="cuda")  # 2.7e9 values
    drafted = torch.full((40, 1), (1 << 25) - 1, device="cuda")
    target[39, 0, -1], target[39, 1, 12345678] = 1.0, 0.5
    target[:39, 0, 5] = 1.0
    uniform = torch.full((40, 2), 0.5, device="cuda")
    tokens, accepted, _ = sm100_verify_draft(target, drafted, uniform)
    assert accepted.tolist() == [0] * 39 + [1]
    assert tokens[39].tolist() == [(1 << 25) - 1, 12345678] and tokens[:39].tolist() == [[5, -1]] * 39


def test_without_a_gpu() -> None:
    target, drafted = torch.zeros(2, 4, 9), torch.zeros(2, 3, dtype=torch.int64)
    assert not can_use_sm100_verify_draft(target, drafted)
    with pytest.raises(RuntimeError):  # no CPU form
        sm100_verify_draft(target, drafted, torch.zeros(2, 4))


@gpu
def test_refusals() -> None:
    target, draft, drafted, uniform = _case(3, 2, 40, 5)
    assert can_use_sm100_verify_draft(target, drafted)
    for bad_target, bad_drafted in (
        (target.double(), drafted), (target[:2], drafted), (target[:, :2], drafted), (target[..., ::2], drafted),
        (target, drafted.float()), (target, drafted.cpu()), (target[0], drafted), (target, drafted[0]), (target[..., :0], drafted),
        (target[:0], drafted[:0]), (target, drafted.t().contiguous().t()),
    ):
        assert not can_use_sm100_verify_draft(bad_target, bad_drafted)
        with pytest.raises(RuntimeError):
            sm100_verify_draft(bad_target, bad_drafted, uniform)
    for kwargs in (
        {"uniform": uniform.double()}, {"uniform": uniform[:, :2]}, {"uniform": uniform.cpu()}, {"uniform": uniform.t().contiguous().t()},
        {"draft": draft.bfloat16()}, {"draft": draft[..., :39]}, {"draft": draft[:2]}, {"draft": draft.cpu()}, {"draft": target},
        {"counts": torch.zeros(3, device="cuda")}, {"counts": torch.zeros(2, dtype=torch.int32, device="cuda")}, {"draft": 3},
    ):
        with pytest.raises(ValueError):
            sm100_verify_draft(**{"target": target, "drafted": drafted, "uniform": uniform, **kwargs})
    many = torch.zeros(1, 1025, dtype=torch.int64, device="cuda")
    with pytest.raises(RuntimeError):
        sm100_verify_draft(torch.zeros(1, 1026, 2, device="cuda"), many, torch.zeros(1, 1026, device="cuda"))
    _check(*(torch.rand(1, 1025, 3, device="cuda"), torch.ones(1, 1024, dtype=torch.int32, device="cuda"),
             torch.rand(1, 1025, device="cuda")))


def test_c_entry_refusals() -> None:
    lib = _native.load()

    def call(target=16, draft=None, dtype=0, drafted=16, uniform=16, batch=1, tokens=1, vocab=8, out=16, accepted=16):  # noqa: ANN001, ANN202
        return lib.b200tx_verify_draft(target, 16, 8, draft, 8, 8, dtype, drafted, 0, uniform, None, batch, tokens, vocab, out,
                                       accepted, None)

    for bad in ({"target": None}, {"drafted": None}, {"uniform": None}, {"out": None}, {"accepted": None}, {"dtype": 5},
                {"batch": 0}, {"tokens": -1}, {"tokens": 1025}, {"vocab": 0}, {"batch": 1 << 21}, {"vocab": 1 << 29}):
        assert call(**bad) < 0, bad
