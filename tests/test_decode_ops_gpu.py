"""Decoding operators against plain 64-bit implementations: norm + rotation of
queries and keys, the 8-bit cache (append, gather, attention), 4-bit linear.

Tolerances, from the number formats:
* a bf16 result (8 significant bits) carries one rounding, at most 2^-8 of its size;
* fp32 norm and rotation: a few roundings of 2^-24 and the square root's 2^-22;
* attention rounds probabilities to fp16 (11 significant bits, 2^-11 of each at
  most), so an output may be off by 2^-11 of the largest value beside its own
  rounding;
* a 4-bit product is summed in fp32: K / 16 MMA steps and K / 32 group sums, each
  off by at most 2^-23 of the sum of magnitudes.
"""

from __future__ import annotations

import math

import pytest
import torch

from solution import _native
from solution.kernels import (
    KV8_BLOCK,
    Kv8Cache,
    RotaryTable,
    can_use_sm100_kv8_attention,
    pack_w4,
    sm100_kv8_append,
    sm100_kv8_attention,
    sm100_kv8_gather,
    sm100_linear_w4,
    sm100_qk_norm_rope,
)

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
BF16_HALF_ULP = 2.0**-8  # of the value, at most


@pytest.fixture(autouse=True)
def _inference():
    with torch.inference_mode():
        yield
    torch.cuda.synchronize()


def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(*shape: int, seed: int) -> torch.Tensor:
    return torch.randn(*shape, generator=_gen(seed), device=DEV)


# ------------------------------------------------------------------ norm + rotation


def _norm_rope64(x, weight, eps, table, positions):  # noqa: ANN001, ANN202
    """x [B, T, heads, D] in float64."""
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()
    if table is None:
        return x
    cos = table.cos.double()[positions][:, :, None]
    sin = table.sin.double()[positions][:, :, None]
    r = table.rotary
    y = x.clone()
    if table.interleaved:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        y[..., 0:r:2], y[..., 1:r:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., : r // 2], x[..., r // 2 : r]
        y[..., : r // 2], y[..., r // 2 : r] = a * cos - b * sin, b * cos + a * sin
    return y


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize(
    ("batch", "tokens", "heads", "kv_heads", "dim", "rotary", "interleaved", "normed"),
    [
        (1, 1, 1, 1, 64, 64, False, True),
        (2, 5, 4, 2, 8, 8, False, True),
        (2, 7, 3, 1, 16, 8, True, True),
        (3, 33, 5, 5, 32, 24, False, True),  # rotary / 2 = 12 dims
        (2, 17, 12, 3, 64, 32, True, False),
        (1, 129, 7, 7, 128, 128, False, True),
        (2, 65, 6, 2, 128, 64, False, True),
        (2, 9, 3, 1, 256, 256, False, True),
        (1, 31, 2, 2, 256, 112, True, True),
        (1, 3001, 16, 4, 64, 64, False, True),  # a warp takes the whole token
    ],
)
def test_norm_rope(dtype, batch, tokens, heads, kv_heads, dim, rotary, interleaved, normed) -> None:  # noqa: ANN001
    total = heads + 2 * kv_heads
    qkv = (3 * _randn(batch, tokens, total * dim, seed=dim + tokens)).to(dtype)
    weights = [1 + 0.2 * _randn(dim, seed=s) for s in (1, 2)] if normed else [None, None]
    table = RotaryTable.create(4096, rotary, DEV, interleaved=interleaved)
    positions = torch.randint(0, 4096, (batch, tokens), generator=_gen(5), device=DEV)
    got, marker = sm100_qk_norm_rope(
        qkv, heads, kv_heads, q_weight=weights[0], k_weight=weights[1], eps=1e-5, rope=table, positions=positions
    )
    assert marker == "sm100_qk_norm_rope" and got.dtype == dtype
    x = qkv.double().reshape(batch, tokens, total, dim)
    want = torch.cat(
        (
            _norm_rope64(x[:, :, :heads], weights[0], 1e-5, table, positions),
            _norm_rope64(x[:, :, heads : heads + kv_heads], weights[1], 1e-5, table, positions),
            x[:, :, heads + kv_heads :],
        ),
        2,
    )
    diff = (got.double().reshape(want.shape) - want).abs()
    # a turned value is a difference of two: its error goes by the pair's size
    size = want.abs().amax(-1, keepdim=True)
    bound = 2.0**-20 * size + (BF16_HALF_ULP * want.abs() if dtype == torch.bfloat16 else 0)
    assert bool((diff <= bound).all()), float((diff / size).max())
    # values are copied bit for bit, int32 positions and in-place give the same bits
    assert torch.equal(got[..., (heads + kv_heads) * dim :], qkv[..., (heads + kv_heads) * dim :])
    again = qkv.clone()
    sm100_qk_norm_rope(
        again, heads, kv_heads, q_weight=weights[0], k_weight=weights[1], eps=1e-5, rope=table,
        positions=positions.int(), out=again,
    )
    assert torch.equal(again, got)


def test_norm_rope_defaults_strides_and_parts() -> None:
    heads, dim, tokens = 4, 64, 19
    wide = _randn(2, tokens, 3 * heads * dim + 64, seed=3).bfloat16()
    qkv = wide[..., 32 : 32 + 3 * heads * dim]  # 64 bytes in, a longer row
    table = RotaryTable.create(64, dim, DEV)
    got, _ = sm100_qk_norm_rope(qkv, heads, rope=table)
    same, _ = sm100_qk_norm_rope(
        qkv.contiguous(), heads, rope=table, positions=torch.arange(tokens, device=DEV, dtype=torch.int32)
    )
    assert torch.equal(got, same)
    # a norm on the keys alone, no rotation; one head group straddles q and k
    weight = 1 + 0.1 * _randn(dim, seed=9)
    keyed, _ = sm100_qk_norm_rope(qkv[..., : 3 * 64], 1, k_weight=weight)
    assert torch.equal(keyed[..., :64], qkv[..., :64]) and torch.equal(keyed[..., 128:], qkv[..., 128:192])
    want = _norm_rope64(qkv[..., 64:128].double()[:, :, None], weight, 1e-6, None, None)[:, :, 0]
    assert bool(((keyed[..., 64:128].double() - want).abs() <= 1.01 * BF16_HALF_ULP * want.abs()).all())
    # transposed batch and token
    flipped, _ = sm100_qk_norm_rope(qkv.transpose(0, 1), heads, rope=table, positions=torch.zeros(2, dtype=torch.int64, device=DEV))
    assert flipped.shape == (tokens, 2, 3 * heads * dim)
    assert torch.equal(flipped[..., : 2 * heads * dim], qkv.transpose(0, 1)[..., : 2 * heads * dim])  # position 0: no turn


def test_norm_rope_position_outside_the_table_is_nan() -> None:
    qkv = _randn(1, 4, 3 * 64, seed=4).bfloat16()
    table = RotaryTable.create(8, 32, DEV)
    positions = torch.tensor([0, 8, -1, 7], device=DEV)
    got, _ = sm100_qk_norm_rope(qkv, 1, rope=table, positions=positions)
    got = got.float()
    assert bool(got[0, 1:3, :32].isnan().all()) and bool(got[0, 1:3, 64:96].isnan().all())
    assert bool(got[0, [0, 3]].isfinite().all())


# ------------------------------------------------------------------ 8-bit cache


def _append64(qkv, heads, kv_heads, dim, start, q_weight, k_weight, table):  # noqa: ANN001, ANN202
    """q, k, v of one call, [B, T, heads, D]; k and v rounded to bf16 as they enter."""
    batch, tokens, _ = qkv.shape
    x = qkv.double().reshape(batch, tokens, heads + 2 * kv_heads, dim)
    positions = start[:, None] + torch.arange(tokens, device=DEV)
    q = _norm_rope64(x[:, :, :heads], q_weight, 1e-6, table, positions)
    k = _norm_rope64(x[:, :, heads : heads + kv_heads], k_weight, 1e-6, table, positions)
    return q, k, x[:, :, heads + kv_heads :]


def _check_quantised(got, want, total, slack):  # noqa: ANN001, ANN202
    """got, want [T, Hkv, D]: full blocks within half a step, the rest bf16."""
    full = total // KV8_BLOCK * KV8_BLOCK
    w = want[:total].double()
    g = got[:total].double()
    if full:
        blocks = w[:full].unflatten(0, (-1, KV8_BLOCK))
        peak = blocks.abs().amax((1, 3), keepdim=True)
        off = (g[:full].unflatten(0, (-1, KV8_BLOCK)) - blocks).abs()
        # half a step, the rounding of k and v to bf16, and that of the value read back
        bound = peak / 254 * (1 + 2.0**-6) + (1 + slack) * 2 * BF16_HALF_ULP * blocks.abs()
        assert bool((off <= bound + 2.0**-40).all()), float((off / peak.clamp_min(1e-30)).max())
    off = (g[full:] - w[full:]).abs()
    assert bool((off <= (1 + slack) * BF16_HALF_ULP * w[full:].abs() + slack * 1e-5).all())
    assert bool((got[total:] == 0).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize(
    ("dim", "heads", "kv_heads", "pieces"),
    [
        (64, 4, 2, (1,)),
        (64, 2, 2, (63, 1, 1, 64, 65)),
        (128, 4, 1, (200, 3, 128)),
        (32, 3, 3, (5, 59, 64, 300)),
        (256, 2, 1, (100, 29, 1, 256)),
    ],
)
def test_append_and_gather(dtype, dim, heads, kv_heads, pieces) -> None:  # noqa: ANN001
    batch, room = 3, sum(pieces)
    cache = Kv8Cache.create(slots=batch, max_tokens=room, num_kv_heads=kv_heads, head_dim=dim, device=DEV)
    cache.page_table.copy_(torch.randperm(cache.pages, generator=_gen(1), device=DEV).reshape(batch, -1))
    table = RotaryTable.create(room, dim, DEV)
    q_weight, k_weight = 1 + 0.1 * _randn(dim, seed=1), 1 + 0.1 * _randn(dim, seed=2)
    qkv = _randn(batch, room, (heads + 2 * kv_heads) * dim, seed=dim).to(dtype)
    keys, values, at = [], [], 0
    for n in pieces:
        start = cache.lengths.long()
        part = qkv[:, at : at + n]
        q, marker = sm100_kv8_append(cache, part, heads, q_weight=q_weight, k_weight=k_weight, rope=table)
        assert marker == "sm100_kv8_append"
        q64, k64, v64 = _append64(part, heads, kv_heads, dim, start, q_weight, k_weight, table)
        size = q64.abs().amax(-1, keepdim=True)
        assert bool(((q.double() - q64).abs() <= BF16_HALF_ULP * q64.abs() + 2.0**-20 * size).all())
        keys.append(k64)
        values.append(v64)
        at += n
        # the pending tokens are read with tokens=n, before the lengths move
        k_now, v_now, _ = sm100_kv8_gather(cache, room, tokens=n)
        cache.advance(n)
        k_then, v_then, _ = sm100_kv8_gather(cache, room)
        assert torch.equal(k_now, k_then) and torch.equal(v_now, v_then)
        for b in range(batch):
            _check_quantised(k_then[b], torch.cat(keys, 1)[b], at, 0.01)
            _check_quantised(v_then[b], torch.cat(values, 1)[b], at, 0.0)
    # all at once: the same bits in every full block and in the open one
    whole = Kv8Cache.create(slots=batch, max_tokens=room, num_kv_heads=kv_heads, head_dim=dim, device=DEV)
    whole.page_table.copy_(cache.page_table)
    sm100_kv8_append(whole, qkv, heads, q_weight=q_weight, k_weight=k_weight, rope=table)
    whole.advance(room)
    full = room // KV8_BLOCK
    used = cache.page_table[:, :full].long()
    assert torch.equal(whole.codes[0, used], cache.codes[0, used])
    assert torch.equal(whole.scales[0, used], cache.scales[0, used])
    assert all(torch.equal(a, b) for a, b in zip(sm100_kv8_gather(whole, room)[:2], sm100_kv8_gather(cache, room)[:2]))


def test_append_scales_and_codes_are_the_definition() -> None:
    """No norm, no rotation: scale = max / 127 in fp32, code = rint(x / scale) + 128,
    a block of zeros has scale 0, one that is not finite the scale NaN."""
    cache = Kv8Cache.create(slots=1, max_tokens=192, num_kv_heads=2, head_dim=64, device=DEV)
    qkv = _randn(1, 192, 6 * 64, seed=8).bfloat16()
    x = qkv.view(1, 192, 6, 64)
    x[:, :64, 2] = 0  # keys of kv head 0, block 0
    x[0, 70, 5, 3] = float("inf")  # a value of kv head 1, block 1
    x[0, 130, 3, 0] = float("nan")  # a key of kv head 1, block 2
    sm100_kv8_append(cache, qkv, 2)
    blocks = x[0, :, 2:].float().reshape(3, 64, 2, 2, 64).permute(0, 2, 3, 1, 4)  # block, kv, head, token, dim
    want = blocks.abs().amax((-2, -1)) / 127
    got = cache.scales[0]
    odd = torch.zeros_like(want, dtype=torch.bool)
    odd[1, 1, 1] = odd[2, 0, 1] = True
    assert torch.equal(got.isnan(), odd) and torch.equal(got[~odd], want[~odd]) and float(got[0, 0, 0]) == 0.0
    fine = ~odd & (want > 0)
    code = (blocks[fine].double() / want[fine].double()[:, None, None] + 128)
    assert bool(((cache.codes[0][fine].double() - code).abs() <= 0.5 + 2.0**-15).all())
    assert bool((cache.codes[0, 0, 0, 0] == 128).all())


def test_append_slots_counts_and_bad_indices_leave_the_rest_alone() -> None:
    cache = Kv8Cache.create(slots=5, max_tokens=128, num_kv_heads=1, head_dim=64, device=DEV)
    cache.page_table.add_(0)
    cache.codes.fill_(7)
    cache.lengths.copy_(torch.tensor([0, 60, 10, 128, 0], device=DEV))
    qkv = _randn(4, 70, 3 * 64, seed=2).bfloat16()
    slots = torch.tensor([3, 1, 9, 4], dtype=torch.int32, device=DEV)  # full, held 60, none, empty
    counts = torch.tensor([5, 70, 70, 0], dtype=torch.int32, device=DEV)
    before = cache.codes.clone()
    sm100_kv8_append(cache, qkv, 1, slots=slots, counts=counts)
    changed = (cache.codes != before).flatten(2).any(-1)[0]
    # slot 1 filled its blocks 0 (tokens 60..63) and 1 (64..127); nobody else has a full block
    assert changed.tolist() == [page in (2, 3) for page in range(cache.pages)]
    k, v, _ = sm100_kv8_gather(cache, 130, slots=slots, counts=counts)
    assert bool(k[2].isnan().all()) and bool((k[3] == 0).all())
    assert bool((k[1, 60:, 0].float() - qkv[1, :, 64:128].float()).abs().max() < 0.05)


def test_append_keeps_the_tokens_that_the_caller_accepts() -> None:
    """Drafted tokens: append 9 over a block's end, accept 3, go on."""
    dim, heads = 64, 2
    make = lambda: Kv8Cache.create(slots=1, max_tokens=256, num_kv_heads=heads, head_dim=dim, device=DEV)  # noqa: E731
    drafted, plain = make(), make()
    qkv = _randn(1, 180, 3 * heads * dim, seed=1).bfloat16()
    wrong = _randn(1, 9, 3 * heads * dim, seed=2).bfloat16()
    for cache in (drafted, plain):
        sm100_kv8_append(cache, qkv[:, :58], heads)
        cache.advance(58)
    sm100_kv8_append(drafted, torch.cat((qkv[:, 58:61], wrong[:, 3:]), 1), heads)
    drafted.advance(3)
    sm100_kv8_append(plain, qkv[:, 58:61], heads)
    plain.advance(3)
    for cache in (drafted, plain):
        sm100_kv8_append(cache, qkv[:, 61:180], heads)
        cache.advance(119)
    assert all(torch.equal(a, b) for a, b in zip(sm100_kv8_gather(drafted, 180)[:2], sm100_kv8_gather(plain, 180)[:2]))


# ------------------------------------------------------------------ attention over the cache


def _filled(lengths, kv_heads, dim, seed, room=None):  # noqa: ANN001, ANN202
    """A cache with `lengths` tokens (already advanced) and the values that it holds."""
    room = room or max(max(lengths), 1)
    cache = Kv8Cache.create(slots=len(lengths), max_tokens=room, num_kv_heads=kv_heads, head_dim=dim, device=DEV)
    cache.page_table.copy_(torch.randperm(cache.pages, generator=_gen(seed), device=DEV).reshape(len(lengths), -1))
    most = max(max(lengths), 1)
    qkv = _randn(len(lengths), most, 3 * kv_heads * dim, seed=seed).bfloat16()
    counts = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    sm100_kv8_append(cache, qkv, kv_heads, counts=counts)
    cache.advance(counts)
    k, v, _ = sm100_kv8_gather(cache, most)
    # gather rounds code x scale to bf16; take the exact product instead
    full = cache.page_table.long()
    exact = ((cache.codes[0][full].double() - 128) * cache.scales[0][full].double()[..., None, None])
    exact = exact.permute(0, 2, 1, 4, 3, 5).flatten(2, 3)[:, :, :most]  # slot, kv, token, head, dim
    out = []
    for b, n in enumerate(lengths):
        cut = n // KV8_BLOCK * KV8_BLOCK
        out.append([torch.cat((exact[b, i, :cut], t[b, cut:n].double())) for i, t in enumerate((k, v))])
    return cache, out


def _attention64(q, kv, held, scale):  # noqa: ANN001, ANN202
    """q [T, H, D] at positions held + t over kv = (k, v) [total, Hkv, D]."""
    tokens, heads, _ = q.shape
    k, v = kv
    group = heads // k.shape[1]
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    score = torch.einsum("thd,shd->hts", q.double(), k) * scale
    seen = torch.arange(k.shape[0], device=DEV) <= held + torch.arange(tokens, device=DEV)[:, None]
    weight = torch.softmax(score.masked_fill(~seen, float("-inf")), -1)
    return torch.einsum("hts,shd->thd", weight, v.masked_fill(~seen.any(0)[:, None, None], 0))


def _check_attention(got, want, biggest) -> None:  # noqa: ANN001
    off = (got.double() - want).abs()
    bound = BF16_HALF_ULP * want.abs() + 2.0**-11 * biggest
    assert bool((off <= bound).all()), float((off - bound).max())


CASES = [
    # dim, kv_heads, group, tokens, total lengths
    (64, 1, 1, 1, [1]),
    (64, 2, 1, 1, [1, 2, 15, 16, 17, 31, 63, 64, 65, 127, 128, 129, 200]),
    (128, 2, 4, 1, [1, 64, 500, 63, 1000]),
    (32, 3, 2, 1, [33, 64, 700]),
    (256, 1, 8, 1, [77, 640, 191]),
    (64, 2, 16, 1, [300, 5]),
    (128, 1, 32, 1, [130]),  # two row tiles of one token
    (64, 4, 2, 5, [5, 64, 66, 67, 200]),
    (128, 2, 3, 7, [7, 70, 1000]),
    (128, 1, 1, 16, [16, 80, 4097]),
    (256, 2, 2, 9, [9, 65, 333]),
    (32, 1, 4, 40, [40, 64, 104, 3000]),
    (64, 2, 1, 130, [130, 192, 700]),  # a prompt's worth of rows
    (64, 8, 2, 1, [20000]),  # one sequence over every SM
    (128, 1, 1, 1, [40000]),
]


@pytest.mark.parametrize(("dim", "kv_heads", "group", "tokens", "totals"), CASES)
def test_attention(dim, kv_heads, group, tokens, totals) -> None:  # noqa: ANN001
    cache, kv = _filled(totals, kv_heads, dim, seed=dim + tokens)
    cache.advance(-tokens)  # the last `tokens` are the step at hand
    q = _randn(len(totals), tokens, kv_heads * group, dim, seed=7).bfloat16()
    got, marker = sm100_kv8_attention(cache, q)
    assert marker == "sm100_kv8_attention" and got.shape == (len(totals), tokens, kv_heads * group * dim)
    for b, total in enumerate(totals):
        want = _attention64(q[b], kv[b], total - tokens, dim**-0.5)
        _check_attention(got[b].view(tokens, -1, dim), want, kv[b][1].abs().max())
    assert torch.equal(sm100_kv8_attention(cache, q)[0], got)  # the same bits again


def _widened(cache):  # noqa: ANN001, ANN202
    """The same cache with room for 800000 tokens a slot in the page table, for which
    the kernels of taller row tiles are taken."""
    table = torch.full((cache.slots, 12500), -1, dtype=torch.int32, device=DEV)
    table[:, : cache.max_blocks] = cache.page_table
    return Kv8Cache(cache.codes, cache.scales, cache.tail, table, cache.lengths)


@pytest.mark.parametrize(
    ("dim", "kv_heads", "group", "tokens", "totals"), [case for case in CASES if case[2] * case[3] > 8 and case[0] < 256]
)
def test_attention_tall_row_tiles(dim, kv_heads, group, tokens, totals) -> None:  # noqa: ANN001
    cache, kv = _filled(totals, kv_heads, dim, seed=dim + tokens)
    cache.advance(-tokens)
    wide = _widened(cache)
    q = _randn(len(totals), tokens, kv_heads * group, dim, seed=7).bfloat16()
    got, _ = sm100_kv8_attention(wide, q)
    for b, total in enumerate(totals):
        want = _attention64(q[b], kv[b], total - tokens, dim**-0.5)
        _check_attention(got[b].view(tokens, -1, dim), want, kv[b][1].abs().max())
    assert torch.equal(sm100_kv8_attention(wide, q)[0], got)


@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("tokens", [12, 100])
def test_attention_tall_row_tiles_poisoned(dim, tokens) -> None:  # noqa: ANN001
    """Rows that do not see a block do not see its NaN either; a bad page is NaN."""
    cache, kv = _filled([192, 192], 1, dim, seed=4)
    cache.advance(-tokens)
    cache.scales[0, cache.page_table[0, 2].long()] = float("nan")
    wide = _widened(cache)
    wide.page_table[1, 1] = 10_000  # not a page
    q = _randn(2, tokens, 1, dim, seed=1).bfloat16()
    got = sm100_kv8_attention(wide, q)[0]
    clear = max(0, 128 - (192 - tokens))  # rows that end before the third block
    want = _attention64(q[0], [t.nan_to_num() for t in kv[0]], 192 - tokens, dim**-0.5)
    _check_attention(got[0, :clear].view(clear, 1, dim), want[:clear], kv[0][1].nan_to_num().abs().max())
    assert bool(got[0, clear:].isnan().all())
    assert bool(got[1].isnan().all())


def test_attention_sharp_and_large_scores() -> None:
    """Scores of hundreds: the running maximum moves often; and tiny queries."""
    cache, kv = _filled([1000, 150], 2, 64, seed=3)
    cache.advance(-1)
    for factor in (40.0, 2.0**-30, 2.0**60):
        q = (factor * _randn(2, 1, 4, 64, seed=1)).bfloat16()
        scale = 0.125 if factor < 2.0**50 else 2.0**-63
        got, _ = sm100_kv8_attention(cache, q, scale=scale)
        for b, total in enumerate((1000, 150)):
            want = _attention64(q[b], kv[b], total - 1, scale)
            # scores up to s carry 2^-22 s in fp32: as much relative error in a weight
            spread = float((q[b].double().abs().max() * kv[b][0].abs().max() * 64 * scale))
            bound = BF16_HALF_ULP * want.abs() + (2.0**-11 + 2.0**-21 * spread) * kv[b][1].abs().max()
            assert bool(((got[b].view(1, 4, 64).double() - want).abs() <= bound).all())


def test_attention_counts_slots_strides_and_empty_rows() -> None:
    dim, kv_heads, heads, tokens = 64, 2, 4, 6
    totals = [6, 70, 200, 3, 64]
    cache, kv = _filled(totals, kv_heads, dim, seed=11)
    counts = torch.tensor([6, 2, 0, 3, 5], dtype=torch.int32, device=DEV)
    cache.lengths.sub_(counts)
    order = torch.tensor([4, 2, 0, 3, 1], dtype=torch.int32, device=DEV)
    wide = _randn(5, tokens, 2 * heads * dim, seed=5).bfloat16()
    q = wide[..., heads * dim :].unflatten(2, (heads, dim))  # a slice of longer rows
    got, _ = sm100_kv8_attention(cache, q, slots=order, counts=counts[order.long()].contiguous())
    for b, slot in enumerate(order.tolist()):
        n = int(counts[slot])
        assert bool((got[b, n:] == 0).all())
        if n:
            want = _attention64(q[b, :n], kv[slot], totals[slot] - n, dim**-0.5)
            _check_attention(got[b, :n].view(n, heads, dim), want, kv[slot][1].abs().max())


def test_attention_does_not_read_what_it_must_not() -> None:
    """NaN in unused pages and past the open block's end, infinity in tokens
    that a row must not see yet, blocks poisoned later than a row."""
    dim, totals, tokens = 64, [40, 100, 130, 64 + 3], 4
    cache, kv = _filled(totals, 1, dim, seed=2, room=256)
    cache.advance(-tokens)
    used = torch.zeros(cache.pages, dtype=torch.bool, device=DEV)
    for b, n in enumerate(totals):
        used[cache.page_table[b, : n // 64].long()] = True
        cache.tail[0, b, (n // 64) & 1, :, :, n % 64 :] = float("nan")
        cache.tail[0, b, 1 - (n // 64 & 1)] = float("nan")
    cache.scales[0, ~used] = float("nan")
    q = _randn(4, tokens, 2, dim, seed=6).bfloat16()
    clean, _ = sm100_kv8_attention(cache, q)
    for b, n in enumerate(totals):
        _check_attention(clean[b].view(tokens, 2, dim), _attention64(q[b], kv[b], n - tokens, dim**-0.5), kv[b][1].abs().max())
    # the last token's value is infinite: only the last row may see it
    for b, n in enumerate(totals):
        cache.tail[0, b, (n // 64) & 1, 1, 0, (n - 1) % 64, 5] = float("inf")
        cache.tail[0, b, (n // 64) & 1, 1, 0, (n - 1) % 64, 9] = float("nan")
    got, _ = sm100_kv8_attention(cache, q)
    got, clean = got.view(4, tokens, 2, dim).float(), clean.view(4, tokens, 2, dim).float()
    assert bool(got[:, :3].isfinite().all())
    assert bool(((got[:, :3] - clean[:, :3]).abs() <= 2.0**-8 * clean[:, :3].abs() + 2.0**-9).all())
    assert bool(got[:, 3, :, 5].isinf().all()) and bool(got[:, 3, :, 9].isnan().all())
    assert bool(got[:, 3, :, :5].isfinite().all())


def test_attention_later_block_poisoned() -> None:
    """A chunk over a block's end: rows before a block see nothing of its NaN scale."""
    cache, kv = _filled([192], 1, 64, seed=4)
    cache.advance(-100)  # rows at 92..191; block 2 is tokens 128..191
    cache.scales[0, cache.page_table[0, 2].long()] = float("nan")
    q = _randn(1, 100, 1, 64, seed=1).bfloat16()
    got, _ = sm100_kv8_attention(cache, q)
    want = _attention64(q[0], [t.nan_to_num() for t in kv[0]], 92, 0.125)
    _check_attention(got[0, :36].view(36, 1, 64), want[:36], kv[0][1].nan_to_num().abs().max())
    assert bool(got[0, 36:].isnan().all())


def test_attention_bad_slots_pages_and_lengths_are_nan() -> None:
    cache, _ = _filled([100, 200, 100, 300], 1, 64, seed=4, room=320)
    cache.advance(-1)
    q = _randn(5, 1, 1, 64, seed=1).bfloat16()
    slots = torch.tensor([0, 7, 1, 2, 3], dtype=torch.int32, device=DEV)
    cache.page_table[1, 1] = 10_000  # not a page
    cache.lengths[2] = 100_000  # longer than the table
    got, _ = sm100_kv8_attention(cache, q, slots=slots)
    assert got[:, 0].isnan().all(-1).tolist() == [False, True, True, True, False]
    assert got[:, 0].isfinite().all(-1).tolist() == [True, False, False, False, True]


def test_attention_nonfinite_queries_and_keys() -> None:
    cache, _ = _filled([70], 1, 64, seed=4)
    cache.advance(-1)
    q = _randn(1, 1, 4, 64, seed=1).bfloat16()
    q[0, 0, 1, 3] = float("nan")
    q[0, 0, 2, 3] = float("inf")
    got = sm100_kv8_attention(cache, q)[0].view(4, 64)
    assert got.isnan().all(-1).tolist() == [False, True, True, False]
    cache.tail[0, 0, 1, 0, 0, 2, 0] = float("nan")  # a key in the open block
    assert bool(sm100_kv8_attention(cache, q)[0].isnan().all())


def test_attention_beyond_32_bit_offsets() -> None:
    """More than 4 GB of codes: the pages in use lie at the far end."""
    kv_heads, dim = 8, 256
    page = 2 * kv_heads * KV8_BLOCK * dim
    pages = (1 << 32) // page + 9
    cache = Kv8Cache(
        torch.zeros(pages, 2, kv_heads, KV8_BLOCK, dim, dtype=torch.uint8, device=DEV),
        torch.zeros(pages, 2, kv_heads, device=DEV),
        torch.zeros(1, 2, 2, kv_heads, KV8_BLOCK, dim, dtype=torch.bfloat16, device=DEV),
        torch.tensor([[pages - 1, 3, pages - 4, pages - 2]], dtype=torch.int32, device=DEV),
        torch.zeros(1, dtype=torch.int32, device=DEV),
    )
    qkv = _randn(1, 256, 3 * kv_heads * dim, seed=1).bfloat16()
    sm100_kv8_append(cache, qkv, kv_heads)
    cache.advance(255)
    k, v, _ = sm100_kv8_gather(cache, 256, tokens=1)
    assert float((k[0].float() - qkv.view(256, 3, kv_heads, dim)[:, 1].float()).abs().max()) < 0.05
    q = _randn(1, 1, kv_heads, dim, seed=2).bfloat16()
    got, _ = sm100_kv8_attention(cache, q)
    full = cache.page_table[0].long()
    exact = (cache.codes[0][full].double() - 128) * cache.scales[0][full].double()[..., None, None]
    kv = list(exact.permute(1, 0, 3, 2, 4).flatten(1, 2))
    _check_attention(got.view(1, kv_heads, dim), _attention64(q[0], kv, 255, dim**-0.5), kv[1].abs().max())


def test_streams_and_graphs() -> None:
    """Two streams at once have a workspace each; a captured step replays with
    the lengths that the device holds by then."""
    cache, _ = _filled([5000, 300], 4, 64, seed=9, room=6000)
    cache.advance(-1)
    q = _randn(2, 1, 4, 64, seed=3).bfloat16()
    want, _ = sm100_kv8_attention(cache, q)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = []
    for _ in range(10):
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                outs.append(sm100_kv8_attention(cache, q)[0])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)

    table = RotaryTable.create(6000, 64, DEV)
    qkv = _randn(2, 1, 12 * 64, seed=3).bfloat16()

    def step() -> torch.Tensor:
        queries, _ = sm100_kv8_append(cache, qkv, 4, rope=table)
        context, _ = sm100_kv8_attention(cache, queries)
        cache.advance(1)
        return context

    held = cache.lengths.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    cache.lengths.copy_(held)
    eager = [step().clone() for _ in range(70)]
    cache.lengths.copy_(held)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        context = step()
    for want in eager:
        graph.replay()
        assert torch.equal(context, want)


def test_capture_without_a_call_before() -> None:
    """The first attention of a cache inside a capture takes the spare
    workspace; on a second new stream it is refused."""
    cache, _ = _filled([3000], 2, 64, seed=3)
    cache.advance(-1)
    q = _randn(1, 1, 2, 64, seed=3).bfloat16()
    sm100_kv8_attention(_filled([70], 2, 64, seed=3)[0], q)  # the kernel is set up, the cache is not
    first, second = torch.cuda.Stream(), torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=first):
        got, _ = sm100_kv8_attention(cache, q)
    for _ in range(3):
        got.zero_()
        graph.replay()
        assert torch.equal(got, sm100_kv8_attention(cache, q)[0])
    assert first.cuda_stream in cache._workspaces and second.cuda_stream not in cache._workspaces
    refused = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="before the capture"):
        with torch.cuda.graph(refused, stream=second):
            q.clone()
            sm100_kv8_attention(cache, q)
    assert torch.equal(got, sm100_kv8_attention(cache, q)[0])


# ------------------------------------------------------------------ 4-bit linear


def _check_linear(got, x, weight, bias, gelu) -> None:  # noqa: ANN001
    w = weight.dequantize(torch.float64)
    rows = x.double().reshape(-1, w.shape[1])
    want = rows @ w.t() + (0 if bias is None else bias.double())
    mass = rows.abs() @ w.abs().t() + (0 if bias is None else bias.double().abs())
    steps = w.shape[1] / 16 + w.shape[1] / 32 + 16
    bound = steps * 2.0**-23 * mass
    if gelu:
        want = want * torch.special.ndtr(want)
        bound = 1.13 * bound + 2.0**-21 * want.abs() + 2.0**-23  # |gelu'| < 1.13; erf to a few ulp
    off = (got.double().reshape(want.shape) - want).abs()
    if got.dtype == torch.bfloat16:
        bound = bound + BF16_HALF_ULP * (want.abs() + bound)
    assert bool((off <= bound).all()), float((off / bound).max())


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize(
    ("rows", "inner", "outer"),
    [(1, 8, 1), (1, 1024, 4096), (3, 136, 17), (8, 128, 16), (9, 1000, 333), (16, 4096, 100), (17, 264, 2049),
     (32, 384, 640), (33, 256, 48), (100, 520, 31), (2, 16384, 64)],
)
def test_linear_w4(rows, inner, outer, group, out_dtype) -> None:  # noqa: ANN001
    weight = pack_w4(_randn(outer, inner, seed=outer) * inner**-0.5, group)
    x = _randn(rows, inner, seed=rows).bfloat16()
    bias = _randn(outer, seed=3) if rows % 2 else None
    got, marker = sm100_linear_w4(x, weight, bias, out_dtype=out_dtype)
    assert marker == "sm100_linear_w4" and got.shape == (rows, outer) and got.dtype == out_dtype
    _check_linear(got, x, weight, bias, False)
    got, marker = sm100_linear_w4(x[None], weight, bias, gelu=True, out_dtype=out_dtype)
    assert marker == "sm100_linear_w4_gelu" and got.shape == (1, rows, outer)
    _check_linear(got, x, weight, bias, True)


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize(
    ("rows", "inner", "outer"),
    [(1, 4096, 7117), (8, 4104, 7120), (5, 8192, 4001), (9, 3992, 9001), (16, 4096, 14336), (3, 256, 113900),
     (16, 264, 57003), (1, 65536, 449), (2, 120, 115001)],
)
def test_linear_w4_with_x_in_shared_memory(rows, inner, outer, group, out_dtype) -> None:  # noqa: ANN001
    """Few rows and many columns: tiles within a warp's range, across two and more of
    them, and a last tile that ends past the columns."""
    weight = pack_w4(_randn(outer, inner, seed=outer) * inner**-0.5, group)
    x = _randn(rows, inner, seed=rows).bfloat16()
    bias = _randn(outer, seed=3) if rows % 2 else None
    got, _ = sm100_linear_w4(x, weight, bias, gelu=rows == 8, out_dtype=out_dtype)
    _check_linear(got, x, weight, bias, rows == 8)
    assert torch.equal(sm100_linear_w4(x, weight, bias, gelu=rows == 8, out_dtype=out_dtype)[0], got)
    x[0, inner // 2] = float("nan")
    got, _ = sm100_linear_w4(x, weight, bias, out_dtype=out_dtype)
    assert got.isnan().all(-1).tolist() == [True] + [False] * (rows - 1) and not got[1:].isnan().any()


def test_linear_w4_codes_past_the_end_and_extremes() -> None:
    """Codes beyond K have no say; every code value counts as what it stands for;
    NaN stays in its own row."""
    inner, outer = 72, 40
    weight = pack_w4(_randn(outer, inner, seed=1), 32)
    x = _randn(4, inner, seed=2).bfloat16()
    want, _ = sm100_linear_w4(x, weight)
    wild = pack_w4(torch.cat((weight.dequantize(), 100 * _randn(outer, 56, seed=3)), 1), 32)
    # the same codes and scales up to K, anything past it
    packed = weight.packed.clone()
    code = lambda w: torch.stack((w & 15, w >> 4), -1)  # noqa: E731
    unpack = lambda p: code(p).reshape(outer, 4, 4, 8).transpose(1, 2).flatten(1)  # noqa: E731
    mixed = torch.where(torch.arange(128, device=DEV) < 96, unpack(packed), unpack(wild.packed))
    both = mixed.reshape(outer, 4, 4, 8).transpose(1, 2).reshape(outer, 64, 2)
    weight.packed.copy_(both[..., 0] | (both[..., 1] << 4))
    assert torch.equal(sm100_linear_w4(x, weight)[0], want)
    x[2, 5] = float("nan")
    got, _ = sm100_linear_w4(x, weight)
    assert got.isnan().all(-1).tolist() == [False, False, True, False]


# ------------------------------------------------------------------ refusals


def test_refusals() -> None:
    qkv = torch.zeros(1, 4, 3 * 64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError, match="ineligible"):
        sm100_qk_norm_rope(qkv.half(), 1)
    with pytest.raises(RuntimeError, match="ineligible"):
        sm100_qk_norm_rope(qkv[..., 1:], 1)
    with pytest.raises(RuntimeError, match="ineligible"):
        sm100_qk_norm_rope(qkv, 5)
    with pytest.raises(RuntimeError, match="ineligible"):
        sm100_qk_norm_rope(qkv.cpu(), 1)
    with pytest.raises(ValueError, match="rotary"):
        sm100_qk_norm_rope(qkv, 1, rope=RotaryTable.create(8, 128, DEV))
    with pytest.raises(ValueError, match="rotary"):
        sm100_qk_norm_rope(qkv, 1, rope=RotaryTable.create(8, 12, DEV))
    with pytest.raises(ValueError, match="norm weights"):
        sm100_qk_norm_rope(qkv, 1, q_weight=torch.ones(64, device=DEV, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="positions"):
        sm100_qk_norm_rope(qkv, 1, positions=torch.zeros(5, dtype=torch.int64, device=DEV))
    with pytest.raises(ValueError, match="out must"):
        sm100_qk_norm_rope(qkv, 1, out=qkv[:, :2])

    cache = Kv8Cache.create(slots=2, max_tokens=100, num_kv_heads=1, head_dim=64, device=DEV)
    with pytest.raises(ValueError, match="layer"):
        sm100_kv8_append(cache, qkv, 1, layer=1)
    with pytest.raises(RuntimeError, match="ineligible"):
        sm100_kv8_append(cache, qkv, 2)
    with pytest.raises(ValueError, match="slots"):
        sm100_kv8_append(cache, qkv.expand(3, 4, 192).contiguous(), 1)
    with pytest.raises(ValueError, match="counts"):
        sm100_kv8_append(cache, qkv, 1, counts=torch.ones(1, device=DEV))
    q = torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError, match="ineligible"):
        sm100_kv8_attention(cache, q.float())
    with pytest.raises(RuntimeError, match="ineligible"):
        sm100_kv8_attention(cache, q.transpose(1, 2))
    with pytest.raises(ValueError, match="scale"):
        sm100_kv8_attention(cache, q, scale=float("nan"))
    with pytest.raises(ValueError, match="scale"):
        sm100_kv8_attention(cache, q, scale=-1.0)
    with pytest.raises(ValueError, match="head_dim"):
        Kv8Cache.create(slots=1, max_tokens=64, num_kv_heads=1, head_dim=96, device=DEV)
    with torch.inference_mode(False), torch.enable_grad():
        assert not can_use_sm100_kv8_attention(cache, q)

    weight = pack_w4(torch.randn(16, 64, device=DEV))
    x = torch.zeros(2, 64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError, match="ineligible"):
        sm100_linear_w4(x[:, :56], weight)
    with pytest.raises(RuntimeError, match="ineligible"):
        sm100_linear_w4(x, weight, torch.zeros(15, device=DEV))
    with pytest.raises(ValueError, match="out_dtype"):
        sm100_linear_w4(x, weight, out_dtype=torch.float16)
    with pytest.raises(ValueError, match="group"):
        pack_w4(torch.randn(16, 64, device=DEV), 16)


def test_c_entry_refusals() -> None:
    """Statuses and messages of the C entry points, nothing launched."""
    cache = Kv8Cache.create(slots=1, max_tokens=64, num_kv_heads=2, head_dim=64, device=DEV)
    q = torch.zeros(1, 1, 3, 64, dtype=torch.bfloat16, device=DEV)
    work = cache.workspace(0)
    with pytest.raises(RuntimeError, match="evenly"):
        _native.kv8_attention(cache.reference(0), q, q, None, None, 1.0, work, 0)
    with pytest.raises(RuntimeError, match="workspace of"):
        _native.kv8_attention(cache.reference(0), q[:, :, :2], q, None, None, 1.0, work[:64], 0)
    with pytest.raises(RuntimeError, match="null"):
        _native.kv8_attention(None, q, q, None, None, 1.0, work, 0)
    x = torch.zeros(1, 60, dtype=torch.bfloat16, device=DEV)
    w = pack_w4(torch.randn(16, 64, device=DEV))
    with pytest.raises(RuntimeError, match="bad shape"):
        _native.linear_w4(x, w.packed, w.scales, None, q, 1, 60, 64, 0)
    with pytest.raises(RuntimeError, match="group"):
        _native.linear_w4(x, w.packed, w.scales, None, q, 1, 64, 48, 0)
    assert math.isclose(cache.bytes_per_token, 2 * 2 * (64 + 4 / 64))
