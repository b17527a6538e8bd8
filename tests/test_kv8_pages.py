"""Forking, freeing, reserving and compacting the 8-bit cache's pages, against plain loops.
All results are whole numbers or copies, so they are equal."""

from __future__ import annotations

import random

import pytest
import torch

from solution import _native
from solution.kernels import (
    Kv8Cache,
    Kv8Pages,
    sm100_kv8_append,
    sm100_kv8_attention,
    sm100_kv8_compact,
    sm100_kv8_fork,
    sm100_kv8_free,
    sm100_kv8_gather,
    sm100_kv8_reserve,
)

gpu = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _inference():
    with torch.inference_mode():
        yield
    if torch.cuda.is_available():
        torch.cuda.synchronize()


def _ints(values, device="cuda"):  # noqa: ANN001, ANN202
    return torch.tensor(values, dtype=torch.int32, device=device)


class Plain:
    """The pool as lists on the host."""

    def __init__(self, pages: Kv8Pages) -> None:
        cache = pages.cache
        self.pages, self.max_blocks, self.slots = cache.pages, cache.max_blocks, cache.slots
        self.table = cache.page_table.tolist()
        self.lengths = cache.lengths.tolist()
        self.refs = pages.refs.tolist()
        self.tail = cache.tail.cpu().clone()
        self.codes = cache.codes.cpu().clone()
        self.scales = cache.scales.cpu().clone()

    def known(self, page: int) -> bool:
        return 0 <= page < self.pages

    def fork(self, source, target) -> None:  # noqa: ANN001
        lengths, table, tail = list(self.lengths), [list(r) for r in self.table], self.tail.clone()
        last = {t: i for i, t in enumerate(target)}
        for i, (s, t) in enumerate(zip(source, target)):
            if not 0 <= t < self.slots or s >= self.slots or s == t or last[t] != i:
                continue
            held = max(0, lengths[s]) if s >= 0 else 0
            full, rest = divmod(held, 64)
            for block in range(self.max_blocks):
                page = table[s][block] if s >= 0 and block < full and self.known(table[s][block]) else -1
                old = self.table[t][block]
                if old == page:
                    continue
                if self.known(old):
                    self.refs[old] -= 1
                if page >= 0:
                    self.refs[page] += 1
                self.table[t][block] = page
            self.lengths[t] = held
            if rest:
                self.tail[:, t, full % 2, :, :, :rest] = tail[:, s, full % 2, :, :, :rest]

    def reserve(self, tokens, slots, counts) -> list[int]:  # noqa: ANN001
        wanted, seen, missing = [], set(), [0] * len(slots)
        for b, slot in enumerate(slots):
            if not 0 <= slot < self.slots or slot in seen:
                continue
            seen.add(slot)
            held = max(0, self.lengths[slot])
            n = min(max(counts[b], 0), tokens)
            for block in range(held // 64, (held + n) // 64):
                if block >= self.max_blocks:
                    missing[b] += 1
                    continue
                page = self.table[slot][block]
                if not self.known(page) or self.refs[page] > 1:
                    wanted.append((b, slot, block, page))
        for _, _, _, page in wanted:
            if self.known(page):
                self.refs[page] -= 1
        free = [p for p in range(self.pages) if self.refs[p] <= 0][::-1]
        for b, slot, block, _ in wanted:
            if free:
                page = free.pop()
                self.refs[page] = 1
            else:
                page = -1
                missing[b] += 1
            self.table[slot][block] = page
        return missing

    def compact(self) -> int:
        used = sum(r > 0 for r in self.refs)
        holes = [p for p in range(used) if self.refs[p] <= 0]
        movers = [p for p in range(used, self.pages) if self.refs[p] > 0]
        where = {p: p for p in range(used) if self.refs[p] > 0}
        for to, of in zip(holes, movers):
            self.codes[:, to] = self.codes[:, of]
            self.scales[:, to] = self.scales[:, of]
            self.refs[to], self.refs[of] = self.refs[of], 0
            where[of] = to
        self.table = [[where.get(p, -1) for p in row] for row in self.table]
        return used

    def check(self, pages: Kv8Pages, codes: bool = False) -> None:
        cache = pages.cache
        assert cache.page_table.tolist() == self.table
        assert cache.lengths.tolist() == self.lengths
        assert pages.refs.tolist() == self.refs
        assert torch.equal(cache.tail.cpu(), self.tail)
        if codes:
            assert torch.equal(cache.codes.cpu(), self.codes) and torch.equal(cache.scales.cpu(), self.scales)


def _pool(slots=6, max_tokens=600, pages=40, layers=2, kv_heads=2, dim=32, seed=0):  # noqa: ANN001, ANN202
    """A pool whose slots hold sequences of their own, and whatever bytes."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    cache = Kv8Cache.create(slots=slots, max_tokens=max_tokens, num_kv_heads=kv_heads, head_dim=dim, layers=layers, pages=pages)
    cache.codes.copy_(torch.randint(0, 256, cache.codes.shape, generator=g, device="cuda", dtype=torch.uint8))
    cache.scales.copy_(torch.rand(cache.scales.shape, generator=g, device="cuda"))
    cache.tail.copy_(torch.randn(cache.tail.shape, generator=g, device="cuda").bfloat16())
    pages_of = Kv8Pages(cache)
    rng = random.Random(seed)
    lengths = [rng.choice((0, 1, 63, 64, 65, 127, 128, rng.randrange(max_tokens))) for _ in range(slots)]
    order = list(range(pages))
    rng.shuffle(order)
    for slot, held in enumerate(lengths):
        full = min(held // 64, len(order))
        lengths[slot] = min(held, full * 64 + held % 64)
        cache.page_table[slot, :full] = _ints([order.pop() for _ in range(full)])
    cache.lengths.copy_(_ints(lengths))
    pages_of.recount()
    return pages_of


@gpu
@pytest.mark.parametrize("seed", range(6))
@pytest.mark.parametrize(
    ("slots", "max_tokens", "pages", "layers", "kv_heads", "dim"),
    [(1, 64, 1, 1, 1, 32), (6, 600, 40, 2, 2, 64), (40, 1000, 700, 1, 3, 32), (5, 9000, 900, 1, 1, 256), (300, 130, 500, 1, 1, 32)],
)
def test_any_sequence_of_calls(seed, slots, max_tokens, pages, layers, kv_heads, dim) -> None:  # noqa: ANN001
    """Forks (beams in a new order, slots twice, slots that are none), frees, reservations with and without room, growth and
    compactions, in any order."""
    pool = _pool(slots, max_tokens, pages, layers, kv_heads, dim, seed)
    plain = Plain(pool)
    rng = random.Random(seed + 100)
    for _ in range(8):
        call = rng.choice(("fork", "permute", "free", "reserve", "reserve", "compact"))
        n = rng.randint(1, min(2 * slots, 70))
        some = [rng.randint(-1, slots) for _ in range(n)]
        if call == "fork":
            source = [rng.randint(-2, slots) for _ in range(n)]
            sm100_kv8_fork(pool, _ints(source), _ints(some))
            plain.fork(source, some)
        elif call == "permute":
            source = [rng.randrange(slots) for _ in range(slots)]
            lengths, _ = sm100_kv8_fork(pool, _ints(source), _ints(list(range(slots))))
            plain.fork(source, list(range(slots)))
            assert lengths is pool.cache.lengths
        elif call == "free":
            sm100_kv8_free(pool, _ints(some))
            plain.fork([-1] * n, some)
        elif call == "reserve":
            tokens = rng.choice((0, 1, 64, 200, max_tokens + 100))
            counts = [rng.randint(-3, tokens + 5) for _ in range(n)]
            plan = rng.choice(("all", "slots", "both"))
            if plan == "all":
                missing, _ = sm100_kv8_reserve(pool, tokens)
                want = plain.reserve(tokens, range(slots), [tokens] * slots)
                grown = [(slot, tokens) for slot in range(slots)]
            elif plan == "slots":
                missing, _ = sm100_kv8_reserve(pool, tokens, slots=_ints(some))
                want = plain.reserve(tokens, some, [tokens] * n)
                grown = []
            else:
                missing, _ = sm100_kv8_reserve(pool, tokens, slots=_ints(some), counts=_ints(counts))
                want = plain.reserve(tokens, some, counts)
                grown = []
            assert missing.tolist() == want
            for slot, count in grown:  # as after the append of a step, where every block has its page
                if want[slot] == 0:
                    plain.lengths[slot] += count
            pool.cache.lengths.copy_(_ints(plain.lengths))
        else:
            used, _ = sm100_kv8_compact(pool)
            assert used.tolist() == [plain.compact()]
            plain.check(pool, codes=True)
        plain.check(pool)
    again = pool.refs.clone()
    pool.recount()
    assert torch.equal(pool.refs, again)
    assert pool.free == sum(r == 0 for r in plain.refs)


@gpu
def test_pages_are_lowest_first_and_shared_ones_are_replaced() -> None:
    cache = Kv8Cache.create(slots=3, max_tokens=256, num_kv_heads=1, head_dim=32, pages=8)
    pool = Kv8Pages(cache)
    missing, _ = sm100_kv8_reserve(pool, 130, counts=_ints([130, 64, 63]))
    assert missing.tolist() == [0, 0, 0]
    assert cache.page_table.tolist() == [[0, 1, -1, -1], [2, -1, -1, -1], [-1] * 4]
    cache.advance(_ints([130, 64, 63]))
    sm100_kv8_fork(pool, _ints([0]), _ints([2]))
    assert cache.page_table[2].tolist() == [0, 1, -1, -1] and pool.refs.tolist() == [2, 2, 1, 0, 0, 0, 0, 0]
    # the caller goes back to the middle of a shared block: what is written there is the slot's own
    cache.lengths.copy_(_ints([130, 64, 70]))
    missing, _ = sm100_kv8_reserve(pool, 64)
    assert missing.tolist() == [0, 0, 0]
    assert cache.page_table.tolist() == [[0, 1, 3, -1], [2, 4, -1, -1], [0, 5, -1, -1]]
    assert pool.refs.tolist() == [2, 1, 1, 1, 1, 1, 0, 0]
    # a pool with too few pages: the first rows get them.  Blocks 2 to 4 of slot 0 (4 is past the table), 1 to 3 of the others
    missing, _ = sm100_kv8_reserve(pool, 192)
    assert missing.tolist() == [1, 1, 2] and cache.page_table.tolist() == [[0, 1, 3, 6], [2, 4, 7, -1], [0, 5, -1, -1]]


def _step(cache, pool, qkv, heads, slots=None):  # noqa: ANN001, ANN202
    missing, _ = sm100_kv8_reserve(pool, qkv.shape[1], slots=slots)
    assert not missing.any()
    outs = []
    for layer in range(cache.layers):
        q, _ = sm100_kv8_append(cache, qkv, heads, layer=layer, slots=slots)
        outs.append(sm100_kv8_attention(cache, q, layer=layer, slots=slots)[0])
    cache.advance(qkv.shape[1], slots)
    return torch.stack(outs)


@gpu
@pytest.mark.parametrize("dim", [32, 64, 128, 256])
def test_samples_of_a_prompt_attend_as_if_each_had_read_it(dim) -> None:  # noqa: ANN001
    """A prompt, forked, steps, beams in a new order, compaction, more steps: bit for bit what slots with the whole history of their own
    give."""
    kv_heads, heads, layers, slots = 2, 4, 2, 5
    g = torch.Generator(device="cuda").manual_seed(dim)

    def tokens(batch, n):  # noqa: ANN001, ANN202
        return torch.randn(batch, n, (heads + 2 * kv_heads) * dim, generator=g, device="cuda").bfloat16()

    pooled = Kv8Cache.create(slots=slots, max_tokens=400, num_kv_heads=kv_heads, head_dim=dim, layers=layers, pages=25)
    pool = Kv8Pages(pooled)
    prompt = tokens(1, 150)
    _step(pooled, pool, prompt, heads, _ints([3]))
    sm100_kv8_fork(pool, _ints([3] * 4), _ints([0, 1, 2, 4]))
    assert pool.free == 25 - 2
    history = [[prompt[0]] for _ in range(slots)]

    def check() -> None:
        own = Kv8Cache.create(slots=slots, max_tokens=400, num_kv_heads=kv_heads, head_dim=dim, layers=layers)
        new = tokens(slots, 1)
        got = _step(pooled, pool, new, heads)
        for b in range(slots):
            whole = torch.cat(history[b])[None]
            for layer in range(layers):
                sm100_kv8_append(own, whole, heads, layer=layer, slots=_ints([b]))
            own.advance(whole.shape[1], _ints([b]))
        want = []
        for layer in range(layers):
            q, _ = sm100_kv8_append(own, new, heads, layer=layer)
            want.append(sm100_kv8_attention(own, q, layer=layer)[0])
        assert torch.equal(got, torch.stack(want))
        own.advance(1)
        for layer in range(layers):
            for a, b in zip(sm100_kv8_gather(pooled, 400, layer=layer)[:2], sm100_kv8_gather(own, 400, layer=layer)[:2]):
                assert torch.equal(a, b)
        for b in range(slots):
            history[b].append(new[b])

    check()
    more = tokens(slots, 60)
    _step(pooled, pool, more, heads)
    for b in range(slots):
        history[b].append(more[b])
    check()
    parents = [1, 0, 0, 4, 2]  # beams 0 and 1 change places, 3 is dropped
    sm100_kv8_fork(pool, _ints(parents), _ints(list(range(slots))))
    history[:] = [list(history[p]) for p in parents]
    check()
    sm100_kv8_free(pool, _ints([2]))
    used, _ = sm100_kv8_compact(pool)
    assert int(used) == 25 - pool.free and not (pooled.page_table >= used).any()
    sm100_kv8_fork(pool, _ints([0]), _ints([2]))
    history[2] = list(history[0])
    for _ in range(70):
        new = tokens(slots, 1)
        _step(pooled, pool, new, heads)
        for b in range(slots):
            history[b].append(new[b])
    check()


@gpu
def test_captured_calls() -> None:
    """Reserve, free and fork in a graph, replayed: each replay goes on from the state that it finds."""
    pool, twin = _pool(seed=4), _pool(seed=4)
    plain = Plain(pool)
    source, target, ended = _ints([0, 1, 5]), _ints([1, 0, 2]), _ints([4])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            sm100_kv8_fork(pool, source, target)
            sm100_kv8_free(pool, ended)
            missing, _ = sm100_kv8_reserve(pool, 64)
            used, _ = sm100_kv8_compact(pool)
        for _ in range(3):
            graph.replay()
            sm100_kv8_fork(twin, source, target)
            sm100_kv8_free(twin, ended)
            lacking, _ = sm100_kv8_reserve(twin, 64)
            held, _ = sm100_kv8_compact(twin)
            plain.fork([0, 1, 5], [1, 0, 2])
            plain.fork([-1], [4])
            want = plain.reserve(64, range(6), [64] * 6)
            n = plain.compact()
            stream.synchronize()
            assert missing.tolist() == lacking.tolist() == want and used.tolist() == held.tolist() == [n]
            plain.check(pool, codes=True)
            plain.check(twin, codes=True)


@gpu
def test_counts_that_do_not_fit_the_table_are_survived() -> None:
    """Tables and lengths that a caller broke: nothing out of range is read or written, and a new count mends the rest."""
    pool = _pool(seed=7)
    cache = pool.cache
    cache.page_table[0, 0], cache.page_table[1, 1], cache.page_table[2, 0] = 1 << 30, -7, cache.pages
    cache.lengths.copy_(_ints([-5, 1 << 30, 2147483647, 600, 100, 64]))
    pool.recount()
    plain = Plain(pool)
    sm100_kv8_fork(pool, _ints([0, 1, 2]), _ints([3, 4, 5]))
    plain.fork([0, 1, 2], [3, 4, 5])
    plain.check(pool)
    missing, _ = sm100_kv8_reserve(pool, 1 << 26)
    assert missing.tolist() == plain.reserve(1 << 26, range(6), [1 << 26] * 6)
    plain.check(pool)
    pool.refs.zero_()  # nothing counts: every page is free, every entry goes
    used, _ = sm100_kv8_compact(pool)
    assert used.tolist() == [0] and not (cache.page_table >= 0).any()


@gpu
def test_as_many_sequences_as_a_call_takes() -> None:
    slots = 2048
    cache = Kv8Cache.create(slots=slots, max_tokens=192, num_kv_heads=1, head_dim=32, pages=3 * slots)
    pool = Kv8Pages(cache)
    cache.tail.copy_(torch.randn(cache.tail.shape, generator=torch.Generator(device="cuda").manual_seed(0), device="cuda"))
    missing, _ = sm100_kv8_reserve(pool, 150)
    assert not missing.any() and cache.page_table[:, :2].flatten().tolist() == list(range(2 * slots))
    cache.advance(150)
    before, tail = cache.page_table.clone(), cache.tail.clone()
    turned = torch.arange(slots, device="cuda").roll(1).to(torch.int32)
    sm100_kv8_fork(pool, turned, torch.arange(slots, device="cuda", dtype=torch.int32))
    assert torch.equal(cache.page_table, before[turned.long()])
    assert torch.equal(cache.tail[:, :, 0, :, :, :22], tail[:, turned.long(), 0, :, :, :22])
    assert torch.equal(cache.tail[:, :, 0, :, :, 22:], tail[:, :, 0, :, :, 22:]) and torch.equal(cache.tail[:, :, 1], tail[:, :, 1])
    assert pool.refs.tolist() == [1] * (2 * slots) + [0] * slots
    sm100_kv8_free(pool, turned)
    assert pool.free == 3 * slots and not cache.lengths.any()


@gpu
def test_pages_beyond_32_bit_offsets() -> None:
    """Compaction of codes of more than 2^31 bytes a layer, and forks of tails past 2^31 values."""
    cache = Kv8Cache.create(slots=2, max_tokens=64 * 8, num_kv_heads=8, head_dim=128, layers=2, pages=20000)
    pool = Kv8Pages(cache)
    cache.page_table[0, :3] = _ints([19999, 5, 18000])
    cache.lengths.copy_(_ints([200, 0]))
    cache.codes[:, 19999], cache.codes[:, 18000], cache.codes[:, 5] = 7, 9, 3
    cache.codes[1, 19999] = 8
    cache.scales[1, 18000] = 0.25
    pool.recount()
    used, _ = sm100_kv8_compact(pool)
    assert used.tolist() == [3]
    # pages in use from 3 on, in order: 5, 18000, 19999 go to 0, 1, 2
    assert cache.page_table[0, :3].tolist() == [2, 0, 1]
    assert [int(cache.codes[0, p].float().mean()) for p in range(3)] == [3, 9, 7] and int(cache.codes[1, 2].float().mean()) == 8
    assert float(cache.scales[1, 1].min()) == 0.25
    del cache, pool
    cache = Kv8Cache.create(slots=5000, max_tokens=64, num_kv_heads=16, head_dim=256, layers=1, pages=2)  # 5.2e9 values of tails
    pool = Kv8Pages(cache)
    cache.lengths[4999] = 63
    cache.tail[0, 4999] = 1.5
    sm100_kv8_fork(pool, _ints([4999]), _ints([4000]))
    assert bool((cache.tail[0, 4000, 0, :, :, :63] == 1.5).all()) and not cache.tail[0, 4000, 0, :, :, 63:].any()
    assert not cache.tail[0, 3999].any() and int(cache.lengths[4000]) == 63


def test_pool_without_a_gpu() -> None:
    cache = Kv8Cache.create(slots=2, max_tokens=200, num_kv_heads=1, head_dim=32, pages=5, device="cpu")
    assert cache.pages == 5 and cache.page_table.tolist() == [[-1] * 4] * 2
    cache.page_table[0, :2] = _ints([4, 1], "cpu")
    cache.page_table[1, :3] = _ints([4, -9, 70], "cpu")
    pool = Kv8Pages(cache)
    assert pool.refs.tolist() == [0, 1, 0, 0, 2] and pool.free == 3
    assert Kv8Pages(cache, torch.ones(5, dtype=torch.int32)).refs.tolist() == [1] * 5
    whole = Kv8Cache.create(slots=2, max_tokens=200, num_kv_heads=1, head_dim=32, device="cpu")
    assert Kv8Pages(whole).free == 0
    for refs in (torch.zeros(4, dtype=torch.int32), torch.zeros(5), torch.zeros(10, dtype=torch.int32)[::2],
                 torch.zeros(6, dtype=torch.int32)[1:]):
        with pytest.raises(ValueError):
            Kv8Pages(cache, refs)
    with pytest.raises(AttributeError):
        pool.refs = pool.refs.clone()
    one = _ints([0], "cpu")
    for call in (lambda: sm100_kv8_fork(pool, one, one), lambda: sm100_kv8_free(pool, one), lambda: sm100_kv8_reserve(pool, 1),
                 lambda: sm100_kv8_compact(pool)):
        with pytest.raises(RuntimeError):  # no CPU form
            call()


@gpu
def test_refusals() -> None:
    pool = _pool()
    plain = Plain(pool)
    one = _ints([1, 0])
    for source, target in (
        (one, one[:1]), (one.long(), one), (one, one.long()), (one.cpu(), one), (one, one.cpu()), (one[None], one[None]),
        (_ints([0, 1, 2, 3])[::2], one), (_ints([0] * 2049), _ints([0] * 2049)), (3, one), (one, None),
    ):
        with pytest.raises(ValueError):
            sm100_kv8_fork(pool, source, target)
    with pytest.raises(ValueError):
        sm100_kv8_free(pool, _ints([0] * 2049))
    for kwargs in (
        {"tokens": -1}, {"tokens": 1, "slots": one.long()}, {"tokens": 1, "slots": one, "counts": one[:1]},
        {"tokens": 1, "counts": _ints([1] * 7)}, {"tokens": 1, "slots": one[:0]}, {"tokens": 1, "slots": _ints([0] * 2049)},
        {"tokens": 1, "counts": one.long()},
    ):
        with pytest.raises(ValueError):
            sm100_kv8_reserve(pool, **kwargs)
    with pytest.raises(RuntimeError):
        sm100_kv8_reserve(pool, (1 << 26) + 1)
    none = _ints([])
    sm100_kv8_fork(pool, none, none)  # nothing to do
    sm100_kv8_free(pool, none)
    plain.check(pool)


def test_c_entry_refusals() -> None:
    import ctypes

    lib = _native.load()
    size = ctypes.c_int64()
    assert lib.b200tx_kv8_pool_scratch(0, ctypes.byref(size)) < 0 and lib.b200tx_kv8_pool_scratch(5, None) < 0
    assert lib.b200tx_kv8_pool_scratch(5, ctypes.byref(size)) == 0 and size.value >= 10

    def view(**changes):  # noqa: ANN003, ANN202
        cache = {"codes": 16, "scales": 16, "tail": 16, "page_table": 16, "lengths": 16, "pages": 4, "slots": 2, "max_blocks": 2,
                 "kv_heads": 1, "head_dim": 32}
        pool = {"layers": 1, "refs": 16, "scratch": 16}
        for name, value in changes.items():
            (cache if name in cache else pool)[name] = value
        return _native.Kv8PoolView(_native.Kv8CacheView(*cache.values()), *pool.values())

    calls = (
        lambda p: lib.b200tx_kv8_fork(p, 16, 16, 1, None),
        lambda p: lib.b200tx_kv8_reserve(p, None, None, 1, 1, 16, None),
        lambda p: lib.b200tx_kv8_compact(p, 16, None),
    )
    for call in calls:
        assert call(None) < 0
        for bad in ({"codes": None}, {"codes": 8}, {"tail": None}, {"tail": 24}, {"scales": None}, {"page_table": None},
                    {"lengths": None}, {"refs": None}, {"refs": 20}, {"scratch": None}, {"scratch": 8}, {"layers": 0}, {"pages": 0}, {"slots": 0},
                    {"head_dim": 48}, {"max_blocks": 0}, {"kv_heads": 0}):
            assert call(ctypes.byref(view(**bad))) < 0, bad
    good = ctypes.byref(view())
    assert lib.b200tx_kv8_fork(good, 16, 16, 2049, None) < 0 and lib.b200tx_kv8_fork(good, 16, None, 1, None) < 0
    assert lib.b200tx_kv8_fork(good, 16, 16, -1, None) < 0
    for tokens, rows, missing in ((-1, 1, 16), (1, 0, 16), (1, 2049, 16), (1, 3, 16), (1, 1, None), (1 << 27, 1, 16)):
        assert lib.b200tx_kv8_reserve(good, None, None, tokens, rows, missing, None) < 0
    assert lib.b200tx_kv8_compact(good, None, None) < 0
