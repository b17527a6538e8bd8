"""A batch of many requests over ``CachedDecoder``: adapters of each slot, forks, drafted tokens that are verified; and the
registered forms of the operators under it.

Tolerance: adapters make a model of other weights, ``W + s up down``, whose own forward (bf16 weights, so one rounding of each
more) the decoder is compared with, at the repository's gate (max-abs 2e-2, rel-L2 1e-2)."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch
from conftest import MAX_ABS_TOL, REL_L2_TOL
from torch._subclasses.fake_tensor import FakeTensorMode

from solution.kernels import Kv8Cache, Kv8Pages, LowRankAdapters, ops, sm100_low_rank_add, sm100_verify_draft
from solution.runtimes import CachedDecoder
from solution.transformer import UserOptimizedTransformer, copy_model_weights
from workloads import WorkloadConfig, seeded_state_dict

DEV = "cuda:0"
B200 = torch.ops.b200tx


def _model(config: WorkloadConfig, device: str = DEV, change=None) -> UserOptimizedTransformer:  # noqa: ANN001
    model = UserOptimizedTransformer(SimpleNamespace(**config.as_dict()))
    copy_model_weights(seeded_state_dict(config, 0), model)
    if change is not None:
        with torch.no_grad():
            change(model)
    return model.to(device).eval()


def _adapters(model: UserOptimizedTransformer, count: int, rank: int, names=("qkv", "out", "ffn_in", "ffn_out"),  # noqa: ANN001, ANN202
              device: str = DEV):
    g = torch.Generator().manual_seed(7)
    sets = []
    for layer in model.layers:
        given = {}
        for name, linear in CachedDecoder._linears(layer):
            if name in names:
                n, k = linear.weight.shape
                given[name] = LowRankAdapters.stack(
                    [(torch.randn(rank, k, generator=g) * k**-0.5, torch.randn(n, rank, generator=g) * 0.15, 0.5 + i)
                     for i in range(count)], device,
                )
        sets.append(given)
    return sets


def _near(got: torch.Tensor, want: torch.Tensor) -> None:
    diff = got.float() - want.float()
    rel = float(diff.norm() / want.float().norm())
    assert float(diff.abs().max()) <= MAX_ABS_TOL and rel <= REL_L2_TOL, (float(diff.abs().max()), rel)


def _randn(*shape: int, seed: int = 1) -> torch.Tensor:
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("graph", [True, False])
def test_each_slot_has_its_adapter(graph) -> None:  # noqa: ANN001
    config = WorkloadConfig(3, 90, 256, 4, 512, 2)
    model = _model(config)
    sets = _adapters(model, 2, 8)

    def merged(index: int):  # noqa: ANN202
        def change(other: UserOptimizedTransformer) -> None:
            for layer, given in zip(other.layers, sets):
                for name, linear in CachedDecoder._linears(layer):
                    a = given[name]
                    delta = (a.up[index].double() @ a.down[index].double() * float(a.scales[index])).float().cpu()
                    linear.weight.add_(delta)

        return _model(config, change=change)

    x = _randn(3, 90, 256)
    with torch.inference_mode():
        want = torch.stack([merged(1)(x)[0], model(x)[1], merged(0)(x)[2]])
        assert float((want - model(x)).abs()[[0, 2]].max()) > 10 * MAX_ABS_TOL  # the adapters do something
    decoder = CachedDecoder(model, slots=3, max_tokens=96, weights="bf16", adapters=sets, graph=graph)
    decoder.set_adapters([1, -1, 0])
    _near(decoder.prompt(x[:, :70].contiguous()), want[:, :70])
    for t in range(70, 80):
        _near(decoder.step(x[:, t : t + 1].contiguous()), want[:, t : t + 1])
    _near(decoder.step(x[:, 80:86].contiguous()), want[:, 80:86])
    # others, for the same graphs, from the next token on
    decoder.reset()
    decoder.set_adapters(torch.tensor([0, 0, -1]))
    with torch.inference_mode():
        want = torch.stack([merged(0)(x)[0], merged(0)(x)[1], model(x)[2]])
    _near(torch.cat([decoder.step(x[:, t : t + 1].contiguous()) for t in range(20)], 1), want[:, :20])


@pytest.mark.gpu
def test_without_an_adapter_the_projections_are_the_same() -> None:
    """Slots without an adapter: what a decoder without any gives, up to where the GELU's rounding falls."""
    config = WorkloadConfig(2, 40, 256, 4, 512, 2)
    model = _model(config)
    x = _randn(2, 40, 256)
    plain = CachedDecoder(model, slots=2, max_tokens=64)
    only = CachedDecoder(model, slots=2, max_tokens=64, adapters=_adapters(model, 3, 16, ("qkv", "out", "ffn_out")))
    assert torch.equal(plain.prompt(x[:, :30].contiguous()), only.prompt(x[:, :30].contiguous()))
    for t in range(30, 40):
        assert torch.equal(plain.step(x[:, t : t + 1].contiguous()), only.step(x[:, t : t + 1].contiguous()))


@pytest.mark.gpu
@pytest.mark.parametrize("graph", [True, False])
def test_forks_go_on_as_if_each_slot_had_read_it_all(graph) -> None:  # noqa: ANN001
    """One prompt for all slots, then beams: bit for bit the decoder whose slots read their own histories."""
    config = WorkloadConfig(4, 200, 128, 2, 256, 2)
    model = _model(config)
    g = torch.Generator().manual_seed(3)
    tokens = torch.randn(200, 128, generator=g).to(DEV)
    forked = CachedDecoder(model, slots=4, max_tokens=256, weights="bf16", graph=graph)
    plain = CachedDecoder(model, slots=4, max_tokens=256, weights="bf16", graph=graph)
    prompt = tokens[:100].expand(4, 100, 128).contiguous()
    # only slot 2 of the forked one has read the prompt: the others hold something else
    other = prompt.clone()
    other[[0, 1, 3]] = _randn(3, 100, 128, seed=9)
    forked.prompt(other)
    plain.prompt(prompt)
    forked.fork([2, 2, 2, 2])
    history = [[prompt[0]] for _ in range(4)]

    def step(n: int, seed: int) -> None:
        x = _randn(4, n, 128, seed=seed)
        assert torch.equal(forked.step(x), plain.step(x))
        for b in range(4):
            history[b].append(x[b])

    for i in range(40):
        step(1, 100 + i)
    step(17, 50)
    parents = [3, 0, 0, 1]
    forked.fork(torch.tensor(parents))
    history[:] = [list(history[p]) for p in parents]
    whole = torch.stack([torch.cat(h) for h in history])
    plain.reset()  # its slots read the new histories token by token, as the forked one's have
    plain.prompt(whole[:, :100].contiguous())
    for t in range(100, 140):
        plain.step(whole[:, t : t + 1].contiguous())
    plain.step(whole[:, 140:].contiguous())
    for i in range(30):
        step(1, 200 + i)
    assert int(forked._pages.refs.max()) > 1  # pages are shared
    with pytest.raises(ValueError, match="pass the cache"):
        forked.step(_randn(4, 100, 128))
    forked.prompt(prompt)  # from the beginning, on shared pages
    plain.prompt(prompt)
    step(1, 7)
    before = plain.cache.lengths.clone()
    forked.fork([0, -1, 2, 9])
    assert forked.cache.lengths.tolist() == [before[0], 0, before[2], before[3]]
    x = _randn(4, 1, 128, seed=8)
    got, want = forked.step(x), plain.step(x)
    assert torch.equal(got[[0, 2, 3]], want[[0, 2, 3]])


@pytest.mark.gpu
def test_drafted_tokens_that_are_verified() -> None:
    """Greedy drafting end to end: a vocabulary of inputs, the next token's probabilities from a fixed head; whatever is
    drafted, the tokens are those that steps of one token each give."""
    config = WorkloadConfig(3, 64, 128, 2, 256, 2)
    model = _model(config)
    vocab, length = 40, 60
    g = torch.Generator().manual_seed(4)
    table = torch.randn(vocab, 128, generator=g).to(DEV)
    head = torch.randn(128, vocab, generator=g).to(DEV) * 3

    def greedy(y: torch.Tensor) -> torch.Tensor:  # a one-hot row for each output
        return torch.nn.functional.one_hot((y @ head).argmax(-1), vocab).float()

    start = torch.tensor([1, 7, 30], device=DEV)
    plain = CachedDecoder(model, slots=3, max_tokens=128, weights="bf16")
    token, want = start, []
    for _ in range(length):
        token = greedy(plain.step(table[token][:, None]))[:, 0].argmax(-1)
        want.append(token)
    want = torch.stack(want, 1)

    drafting = CachedDecoder(model, slots=3, max_tokens=128, weights="bf16")
    got: list[list[int]] = [[] for _ in range(3)]
    token, rng = start, torch.Generator().manual_seed(5)
    steps = 0
    while min(len(row) for row in got) < length:
        # drafts that are right with some luck: the true ones, a random number of them spoilt
        n = 4
        drafted = torch.zeros(3, n, dtype=torch.int64)
        for b in range(3):
            right = want[b, len(got[b]) : len(got[b]) + n].cpu()
            drafted[b, : len(right)] = right
            spoil = int(torch.randint(0, n + 1, (1,), generator=rng))
            if spoil < n:
                drafted[b, spoil] = (drafted[b, spoil] + 1) % vocab
        drafted = drafted.to(DEV)
        x = torch.cat((table[token][:, None], table[drafted]), 1)
        y = drafting.step(x, advance=False)
        tokens, accepted = drafting.accept(greedy(y), drafted, torch.rand(3, n + 1, generator=rng).to(DEV))
        for b in range(3):
            got[b] += tokens[b, : int(accepted[b]) + 1].tolist()
        token = tokens.gather(1, accepted[:, None].long())[:, 0]
        steps += 1
        assert drafting.cache.lengths.tolist() == [len(row) for row in got]
    assert steps < length
    for b in range(3):
        assert got[b][:length] == want[b].tolist()
    # the bound that the decoder keeps is larger than what is held, and is looked up before it refuses
    assert drafting.held > int(drafting.cache.lengths.max())
    drafting.held = 127
    drafting.step(x, advance=False)
    with pytest.raises(ValueError, match="drafted"):
        drafting.accept(greedy(y), drafted[:, :2], torch.rand(3, 3).to(DEV))
    with pytest.raises(ValueError, match="drafted"):
        drafting.accept(greedy(y), drafted[:2], torch.rand(2, 5).to(DEV))


@pytest.mark.gpu
def test_all_of_it_together() -> None:
    """Adapters, forks and verified drafts over packed weights, as a server runs them: bit for bit what slots give that share
    nothing."""
    config = WorkloadConfig(4, 128, 256, 4, 512, 2)
    model = _model(config)
    sets = _adapters(model, 3, 24)
    vocab = 50
    g = torch.Generator().manual_seed(6)
    head = torch.randn(256, vocab, generator=g).to(DEV)
    prompt = _randn(4, 70, 256)
    shared = CachedDecoder(model, slots=4, max_tokens=160, adapters=sets)
    apart = CachedDecoder(model, slots=4, max_tokens=160, adapters=sets)
    shared.set_adapters([2, 0, 1, -1])
    shared.prompt(prompt)
    parents, mixed = [0, 0, 2, 3], [2, 2, 1, -1]
    shared.fork(parents)
    apart.set_adapters(mixed)
    apart.prompt(prompt[parents].contiguous())
    assert shared.adapter_indices.tolist() == mixed
    for turn in range(12):
        x = _randn(4, 5, 256, seed=20 + turn)
        drafted = torch.randint(0, vocab, (4, 4), generator=g).to(DEV)
        uniform = torch.rand(4, 5, generator=g).to(DEV) * 0.2  # so that some are accepted
        draft = torch.softmax(torch.randn(4, 4, vocab, generator=g), -1).to(DEV)
        results = []
        for decoder in (shared, apart):
            y = decoder.step(x, advance=False)
            target = torch.softmax(y @ head, -1)
            results.append((y, *decoder.accept(target, drafted, uniform, draft=draft)))
        for a, b in zip(*results):
            assert torch.equal(a, b)
        assert torch.equal(shared.cache.lengths, apart.cache.lengths)
    assert int(shared.cache.lengths.min()) < int(shared.cache.lengths.max())


@pytest.mark.gpu
def test_counts_of_each_slot_and_refusals() -> None:
    config = WorkloadConfig(2, 80, 128, 2, 128, 1)
    model = _model(config)
    decoder = CachedDecoder(model, slots=2, max_tokens=200, weights="bf16", adapters=_adapters(model, 2, 8, ("out",)))
    x = _randn(2, 5, 128)
    decoder.step(x, advance=False)
    decoder.advance(torch.tensor([2, 9], dtype=torch.int32, device=DEV))
    assert decoder.cache.lengths.tolist() == [2, 5] and decoder.pending == 0
    for bad in (torch.tensor([1, 1], device=DEV), torch.tensor([1], dtype=torch.int32, device=DEV), torch.tensor([1, 1], dtype=torch.int32)):
        with pytest.raises(ValueError):
            decoder.advance(bad)
    decoder.step(_randn(2, 70, 128), advance=False)
    for call in (lambda: decoder.advance(torch.tensor([1, 1], dtype=torch.int32, device=DEV)), lambda: decoder.fork([0, 1])):
        with pytest.raises(ValueError):
            call()
    decoder.advance(70)
    for call in (lambda: decoder.fork([0]), lambda: decoder.fork([0.0, 1.0]), lambda: decoder.set_adapters([0]),
                 lambda: decoder.set_adapters([0.5, 1.0]), lambda: decoder.set_adapters([0, 2])):
        with pytest.raises(ValueError):
            call()
    decoder.set_adapters([1, 0])
    decoder.fork([1 << 33, 1 << 32])  # past the slots: nothing
    assert decoder.adapter_indices.tolist() == [1, 0] and decoder.cache.lengths.tolist() == [72, 75]
    decoder.fork([1, 1])
    assert decoder.adapter_indices.tolist() == [0, 0] and decoder.cache.lengths.tolist() == [75, 75]
    decoder.set_adapters(torch.tensor([0, 5], device=DEV))
    y = decoder.step(_randn(2, 1, 128))
    assert bool(y[0].isfinite().all()) and bool(y[1].isnan().all())
    with pytest.raises(ValueError, match="without adapters"):
        CachedDecoder(model, slots=2, max_tokens=64).set_adapters([0, 0])
    for sets in ([], [{"middle": None}], [{"qkv": _adapters(model, 1, 8, ("out",))[0]["out"]}],
                 _adapters(model, 1, 8, ("out",), device="cpu")):
        with pytest.raises(ValueError):
            CachedDecoder(model, slots=2, max_tokens=64, adapters=sets)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64])
def test_slots_in_any_whole_type(dtype) -> None:  # noqa: ANN001
    config = WorkloadConfig(3, 40, 128, 2, 128, 1)
    model = _model(config)
    decoder = CachedDecoder(model, slots=3, max_tokens=100, adapters=_adapters(model, 2, 8, ("qkv",)))
    decoder.prompt(_randn(3, 10, 128))
    for device in ("cpu", DEV):
        decoder.set_adapters(torch.tensor([0, 1, 0], dtype=dtype, device=device))
        assert decoder.adapter_indices.tolist() == [0, 1, 0]
        decoder.fork(torch.tensor([1, 0, 100], dtype=dtype, device=device))
        assert decoder.adapter_indices.tolist() == [1, 0, 0] and decoder.cache.lengths.tolist() == [10, 10, 10]


def _meta(*shape, dtype=torch.bfloat16):  # noqa: ANN001, ANN002, ANN202
    return torch.empty(*shape, device="meta", dtype=dtype)


def _pool(device="meta", pages=9):  # noqa: ANN001, ANN202
    cache = Kv8Cache.create(slots=2, max_tokens=256, num_kv_heads=1, head_dim=32, layers=3, pages=pages, device="cpu")
    tensors = (cache.codes, cache.scales, cache.tail, cache.page_table, cache.lengths, torch.zeros(pages, dtype=torch.int32))
    return [t.to(device) for t in tensors]


def test_registered_forms_trace() -> None:
    i32, f32 = torch.int32, torch.float32
    y = B200.low_rank_add(_meta(2, 5, 64), _meta(2, 5, 40, dtype=f32), _meta(3, 8, 64), _meta(3, 40, 8), _meta(3, dtype=f32),
                          _meta(2, dtype=i32), True)
    assert (tuple(y.shape), y.dtype) == ((2, 5, 40), torch.bfloat16)
    tokens, accepted = B200.verify_draft(_meta(4, 6, 100), _meta(4, 5, dtype=i32), _meta(4, 6, dtype=f32), _meta(4, 5, 100))
    assert (tuple(tokens.shape), tokens.dtype, tuple(accepted.shape), accepted.dtype) == ((4, 6), i32, (4,), i32)
    pool = _pool()
    assert B200.kv8_fork(*pool, _meta(2, dtype=i32), _meta(2, dtype=i32)) is None
    assert tuple(B200.kv8_reserve(*pool, 5).shape) == (2,) and tuple(B200.kv8_reserve(*pool, 5, _meta(1, dtype=i32)).shape) == (1,)
    assert tuple(B200.kv8_compact(*pool).shape) == (1,)
    for call in (
        lambda: B200.low_rank_add(_meta(5, 64), _meta(5, 40), _meta(3, 12, 64), _meta(3, 40, 12), _meta(3, dtype=f32), _meta(5, dtype=i32)),
        lambda: B200.low_rank_add(_meta(5, 64), _meta(5, 40), _meta(3, 8, 64), _meta(3, 40, 8), _meta(3, dtype=f32), _meta(3, dtype=i32)),
        lambda: B200.verify_draft(_meta(4, 5, 100), _meta(4, 5, dtype=i32), _meta(4, 6, dtype=f32)),
        lambda: B200.kv8_fork(*pool[:5], _meta(8, dtype=i32), None, _meta(2, dtype=i32)),
    ):
        with pytest.raises(ValueError):
            call()
    with FakeTensorMode():
        y = B200.low_rank_add(torch.empty(5, 64, dtype=torch.bfloat16), torch.empty(5, 40), torch.empty(3, 8, 64, dtype=torch.bfloat16),
                              torch.empty(3, 40, 8, dtype=torch.bfloat16), torch.empty(3), torch.empty(5, dtype=i32))
        assert tuple(y.shape) == (5, 40)
    for name in ("low_rank_add", "kv8_fork", "kv8_reserve", "kv8_compact", "verify_draft"):
        assert name in ops.OPERATORS
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        B200.kv8_compact(*_pool("cpu"))


@pytest.mark.gpu
def test_registered_forms_give_the_wrappers_values() -> None:
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(6, 64, generator=g, device=DEV).bfloat16()
    base = torch.randn(6, 40, generator=g, device=DEV)
    adapters = LowRankAdapters(torch.randn(3, 8, 64, generator=g, device=DEV).bfloat16(),
                               torch.randn(3, 40, 8, generator=g, device=DEV).bfloat16(), torch.ones(3, device=DEV))
    indices = torch.tensor([0, 2, -1, 1, 1, 0], dtype=torch.int32, device=DEV)
    with torch.no_grad():
        want, _ = sm100_low_rank_add(x, base, adapters, indices, gelu=True, out_dtype=torch.bfloat16)
    got = B200.low_rank_add(x, base, adapters.down, adapters.up, adapters.scales, indices, True)
    assert torch.equal(got, want)
    target = torch.softmax(torch.randn(4, 3, 50, generator=g, device=DEV), -1)
    drafted = torch.randint(0, 50, (4, 2), generator=g, device=DEV)
    uniform = torch.rand(4, 3, generator=g, device=DEV)
    for a, b in zip(B200.verify_draft(target, drafted, uniform), sm100_verify_draft(target, drafted, uniform)):
        assert torch.equal(a, b)
    pool = _pool(DEV)
    assert B200.kv8_reserve(*pool, 130).tolist() == [0, 0]
    assert pool[3].tolist() == [[0, 1, -1, -1], [2, 3, -1, -1]] and pool[5].tolist() == [1] * 4 + [0] * 5
    pool[4].fill_(130)
    one = torch.tensor([0], dtype=torch.int32, device=DEV)
    B200.kv8_fork(*pool, one + 1, one)
    assert pool[3].tolist() == [[2, 3, -1, -1]] * 2 and pool[5].tolist() == [0, 0, 2, 2, 0, 0, 0, 0, 0]
    assert B200.kv8_compact(*pool).tolist() == [2] and pool[3].tolist() == [[0, 1, -1, -1]] * 2
    B200.kv8_fork(*pool, None, one)
    assert pool[4].tolist() == [0, 130] and Kv8Pages(Kv8Cache(*pool[:5])).free == 7
