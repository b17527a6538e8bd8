"""Attention over the 8-bit cache for batches whose sequences have different numbers of
new tokens: rows past a sequence's count are zero and cost next to nothing; and rows
that end before a block whose page is not in the table.

Tolerance as for the attention elsewhere: a bf16 result (2^-8 of its size) of
probabilities rounded to 11 bits (2^-11 of the largest value)."""

from __future__ import annotations

import pytest
import torch

from solution.kernels import KV8_BLOCK, Kv8Cache, sm100_kv8_append, sm100_kv8_attention, sm100_kv8_gather

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.fixture(autouse=True)
def _inference():
    with torch.inference_mode():
        yield
    torch.cuda.synchronize()


def _randn(*shape: int, seed: int) -> torch.Tensor:
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV)


def _filled(totals: list[int], kv_heads: int, dim: int, room: int) -> Kv8Cache:
    cache = Kv8Cache.create(slots=len(totals), max_tokens=room, num_kv_heads=kv_heads, head_dim=dim, device=DEV)
    counts = torch.tensor(totals, dtype=torch.int32, device=DEV)
    sm100_kv8_append(cache, _randn(len(totals), max(totals), 3 * kv_heads * dim, seed=dim).bfloat16(), kv_heads, counts=counts)
    cache.advance(counts)
    return cache


def _want(cache: Kv8Cache, slot: int, q: torch.Tensor, total: int) -> torch.Tensor:
    """q [n, H, D], the last n of `total` tokens, in 64 bits."""
    k, v, _ = sm100_kv8_gather(cache, total, slots=torch.tensor([slot], dtype=torch.int32, device=DEV),
                               counts=torch.tensor([q.shape[0]], dtype=torch.int32, device=DEV))
    n, heads, dim = q.shape
    full = total // KV8_BLOCK
    out = []
    for i, rounded in enumerate((k, v)):  # exact values of the full blocks
        pages = cache.page_table[slot, :full].long()
        coded = (cache.codes[0, pages, i].double() - 128) * cache.scales[0, pages, i].double()[..., None, None]
        out.append(torch.cat((coded.transpose(1, 2).flatten(0, 1), rounded[0, full * KV8_BLOCK :].double())))
    keys, values = (t.repeat_interleave(heads // t.shape[1], 1) for t in out)
    score = torch.einsum("thd,shd->hts", q.double(), keys) * dim**-0.5
    late = torch.ones(n, total, dtype=torch.bool, device=DEV).triu(total - n + 1)
    return torch.einsum("hts,shd->thd", torch.softmax(score.masked_fill(late, float("-inf")), -1), values)


def _check(cache, q, counts, slots, totals) -> None:  # noqa: ANN001
    """totals: after the call; None for a slot that is none."""
    tokens, heads, dim = q.shape[1:]
    got, _ = sm100_kv8_attention(
        cache, q, counts=torch.tensor(counts, dtype=torch.int32, device=DEV),
        slots=torch.tensor(slots, dtype=torch.int32, device=DEV),
        out=torch.full((len(counts), tokens, heads * dim), 7.0, dtype=torch.bfloat16, device=DEV),
    )
    for b, (n, slot, total) in enumerate(zip(counts, slots, totals)):
        if total is None:
            assert bool(got[b].isnan().all())
            continue
        n = min(max(n, 0), tokens)
        assert bool((got[b, n:] == 0).all())
        if n:
            want = _want(cache, slot, q[b, :n], total)
            off = (got[b, :n].view(n, heads, dim).double() - want).abs()
            assert bool((off <= 2.0**-8 * want.abs() + 2.0**-11 * 6).all()), (b, float(off.max()))


@pytest.mark.parametrize("wide", [False, True])  # a page table for which taller row tiles are taken
@pytest.mark.parametrize(("dim", "kv_heads", "group"), [(32, 3, 2), (64, 2, 4), (128, 2, 4), (256, 1, 3)])
def test_counts_far_apart(dim: int, kv_heads: int, group: int, wide: bool) -> None:
    totals, counts, tokens = [200, 3000, 64, 130, 700, 65, 1], [130, 1, 0, 64, 9, -5, 1], 130
    cache = _filled(totals, kv_heads, dim, 3200)
    cache.lengths.sub_(torch.tensor(counts, dtype=torch.int32, device=DEV).clamp(0, tokens))
    if wide:
        table = torch.full((cache.slots, 12500), -1, dtype=torch.int32, device=DEV)
        table[:, : cache.max_blocks] = cache.page_table
        cache = Kv8Cache(cache.codes, cache.scales, cache.tail, table, cache.lengths)
    q = _randn(8, tokens, kv_heads * group, dim, seed=2).bfloat16()
    _check(cache, q, counts + [130], [0, 1, 2, 3, 4, 5, 6, 99], totals + [None])
    # all rows in place: no counts, the same bits as with counts that say so
    cache.lengths.copy_(torch.full((7,), 5, dtype=torch.int32, device=DEV))
    full = torch.full((7,), tokens, dtype=torch.int32, device=DEV)
    assert torch.equal(sm100_kv8_attention(cache, q[:7], counts=full)[0], sm100_kv8_attention(cache, q[:7])[0])
    # nobody has a row
    assert bool((sm100_kv8_attention(cache, q[:7], counts=torch.zeros_like(full))[0] == 0).all())


def test_more_sequences_than_ctas() -> None:
    batch, dim, heads, tokens = 700, 64, 2, 3
    totals = [1 + (37 * b) % 130 for b in range(batch)]
    counts = [min(t, b % 4) for b, t in enumerate(totals)]  # 0 to 3 of 3
    cache = _filled(totals, heads, dim, 192)
    cache.lengths.sub_(torch.tensor(counts, dtype=torch.int32, device=DEV))
    slots = list(range(batch))
    slots[5], slots[600] = -1, batch
    _check(cache, _randn(batch, tokens, heads, dim, seed=2).bfloat16(), counts, slots,
           [None if not 0 <= s < batch else t for s, t in zip(slots, totals)])


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("dim", [32, 64, 128, 256])
def test_rows_before_a_block_without_a_page(dim: int, wide: bool) -> None:
    """New tokens over a block's end: the rows that do not see the block are what they are, the
    others NaN."""
    cache = _filled([192, 200], 2, dim, 256)
    cache.lengths.sub_(100)  # rows at 92..191 and 100..199; block 2 is tokens 128..191
    want = [None, None]
    q = _randn(2, 100, 4, dim, seed=3).bfloat16()
    for b, (total, seen) in enumerate(((192, 36), (200, 28))):
        want[b] = _want(cache, b, q[b], total)[:seen]
    if wide:
        table = torch.full((cache.slots, 12500), -1, dtype=torch.int32, device=DEV)
        table[:, : cache.max_blocks] = cache.page_table
        cache = Kv8Cache(cache.codes, cache.scales, cache.tail, table, cache.lengths)
    cache.page_table[0, 2], cache.page_table[1, 2] = -1, cache.pages
    got = sm100_kv8_attention(cache, q)[0].view(2, 100, 4, dim)
    for b, rows in enumerate(want):
        n = len(rows)
        off = (got[b, :n].double() - rows).abs()
        assert bool((off <= 2.0**-8 * rows.abs() + 2.0**-11 * 6).all())
        assert bool(got[b, n:].isnan().all())


def _time(call) -> float:  # noqa: ANN001
    for _ in range(5):
        call()
    times = []
    for _ in range(15):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        for _ in range(10):
            call()
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b))
    return sorted(times)[len(times) // 2]


def test_rows_past_the_counts_cost_little() -> None:
    """16 sequences of 8192 tokens with one new token each, in a call of 128: one pass over
    the cache (67 MB) and 16 MB of zeros, not one for each 8 or 16 rows.  And sequences without a
    new token: their zeros are written by all CTAs."""
    cache = Kv8Cache.create(slots=16, max_tokens=8400, num_kv_heads=4, head_dim=64, device=DEV)
    cache.lengths.fill_(8192)
    q = _randn(16, 128, 8, 64, seed=1).bfloat16()
    one = torch.ones(16, dtype=torch.int32, device=DEV)
    alone = _time(lambda: sm100_kv8_attention(cache, q[:, :1].contiguous()))
    padded = _time(lambda: sm100_kv8_attention(cache, q, counts=one))
    assert padded < 3 * alone, (padded, alone)
    cache.lengths.fill_(100)
    wide = _randn(2, 2048, 8, 64, seed=1).bfloat16()
    short = _time(lambda: sm100_kv8_attention(cache, wide[:, :1].contiguous()))
    empty = _time(lambda: sm100_kv8_attention(cache, wide, counts=torch.zeros_like(one[:2])))
    assert empty < 5 * short, (empty, short)
