"""Low-rank adapters beside a projection against a plain 64-bit implementation.

Tolerance of a value, from the number formats: products of bf16 numbers are exact in fp32;
sums of K and of R terms are taken by MMAs in steps of 16, and joined over at most 64 warps
and 8 CTAs, each addition off by at most 2^-23 of the magnitudes summed (an MMA may truncate);
the R sums enter the second product as two bf16 terms, 2^-17 of each; then the base, the scale and
the GELU (erf in fp32, 2^-22 of the value at its steepest 1.13) and one rounding of at most half a step of the result."""

from __future__ import annotations

import pytest
import torch

from solution import _native
from solution.kernels import (
    LowRankAdapters,
    can_use_sm100_low_rank_add,
    sm100_linear_w4,
    pack_w4,
    sm100_low_rank_add,
)

gpu = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _inference():
    with torch.inference_mode():
        yield
    if torch.cuda.is_available():
        torch.cuda.synchronize()


def _adapters(count, rank, inner, outer, g, device="cuda"):  # noqa: ANN001, ANN202
    down = (torch.randn(count, rank, inner, generator=g, device=device) * inner**-0.5).bfloat16()
    up = torch.randn(count, outer, rank, generator=g, device=device).bfloat16()
    return LowRankAdapters(down, up, torch.rand(count, generator=g, device=device) + 0.5)


def _expected(x, base, adapters, indices, gelu, out_dtype):  # noqa: ANN001, ANN202
    """The value in 64 bits, and how far an fp32 evaluation may be off."""
    x, base = x.double().flatten(0, -2), base.double().flatten(0, -2)
    index = indices.flatten().repeat_interleave(x.shape[0] // indices.numel())
    y, size = base.clone(), base.abs()
    inner, rank = x.shape[-1], adapters.rank
    steps = inner / 16 + rank / 8 + 72
    off = torch.zeros_like(y)
    for a in range(adapters.count):
        rows = (index == a).nonzero()[:, 0]
        down, up, s = adapters.down[a].double(), adapters.up[a].double(), adapters.scales[a].double()
        y[rows] += (x[rows] @ down.t()) @ up.t() * s
        most = (x[rows].abs() @ down.abs().t()) @ up.abs().t() * s
        off[rows] = most * (steps * 2.0**-23 + 2.0**-17)
        size[rows] += most
    off += size * 2.0**-22
    if gelu:
        y, off = y * torch.special.ndtr(y), 1.13 * off + 2.0**-22 * y.abs()
    off += (y.abs() + off) * torch.finfo(out_dtype).eps / 2
    y[index >= adapters.count] = torch.nan
    return y, off


def _check(x, base, adapters, indices, *, gelu=False, out_dtype=None, in_place=False):  # noqa: ANN001, ANN202
    want, off = _expected(x, base, adapters, indices, gelu, out_dtype or base.dtype)
    got, _ = sm100_low_rank_add(x, base, adapters, indices, gelu=gelu, out_dtype=out_dtype, out=base if in_place else None)
    assert got.dtype == (out_dtype or base.dtype) and (not in_place or got.data_ptr() == base.data_ptr())
    got = got.double().flatten(0, -2)
    bad = want.isnan()
    assert torch.equal(got.isnan(), bad)
    error = torch.where(bad, 0, (got - want).abs() - off)
    assert float(error.max()) <= 0, float(error.max())
    return got


@gpu
@pytest.mark.parametrize(
    ("rows", "inner", "outer", "rank", "count"),
    [
        (1, 8, 1, 8, 1),
        (1, 1024, 4096, 16, 4),
        (2, 40, 63, 24, 2),
        (8, 4096, 1024, 64, 3),
        (5, 520, 264, 128, 2),
        (9, 264, 130, 8, 5),
        (33, 1000, 200, 40, 3),
        (64, 4096, 4096, 16, 16),
        (200, 264, 515, 72, 7),
        (257, 128, 1032, 32, 4),
        (600, 72, 96, 128, 2),
        (1500, 256, 320, 16, 9),
    ],
)
@pytest.mark.parametrize("base_dtype", [torch.bfloat16, torch.float32])
def test_low_rank_add(rows, inner, outer, rank, count, base_dtype) -> None:  # noqa: ANN001
    g = torch.Generator(device="cuda").manual_seed(rows + outer)
    adapters = _adapters(count, rank, inner, outer, g)
    x = torch.randn(rows, inner, generator=g, device="cuda").bfloat16()
    base = torch.randn(rows, outer, generator=g, device="cuda").to(base_dtype)
    indices = torch.randint(-1, count, (rows,), generator=g, device="cuda", dtype=torch.int32)
    for gelu in (False, True):
        for out_dtype in (torch.bfloat16, torch.float32):
            _check(x, base, adapters, indices, gelu=gelu, out_dtype=out_dtype)
    _check(x, base, adapters, indices, gelu=True, in_place=True)
    _check(x, base, adapters, indices, in_place=True)


@gpu
@pytest.mark.parametrize(
    ("batch", "tokens", "inner", "outer", "rank", "count"),
    [
        (4, 300, 264, 1032, 16, 3),
        (2, 700, 1000, 515, 72, 2),
        (16, 64, 72, 200, 8, 5),
        (5, 257, 2056, 384, 128, 3),
        (1, 1024, 8, 130, 64, 1),
        (20, 100, 512, 4096, 40, 4),
        (4, 1100, 264, 1032, 16, 3),
        (32, 64, 136, 200, 64, 3),  # sequences of one adapter with others between them
        (70, 65, 72, 328, 24, 3),  # groups that end anywhere
        (3, 1000, 1000, 8, 72, 2),
        (2, 4096, 8, 136, 8, 2),
        (24, 128, 520, 1160, 112, 30),
        (64, 64, 200, 64, 40, 3),  # several groups for a CTA, in a row and not
    ],
)
@pytest.mark.parametrize("base_dtype", [torch.bfloat16, torch.float32])
def test_prompts(batch, tokens, inner, outer, rank, count, base_dtype) -> None:  # noqa: ANN001
    """Long runs of rows with one adapter each."""
    g = torch.Generator(device="cuda").manual_seed(batch + outer)
    adapters = _adapters(count, rank, inner, outer, g)
    x = torch.randn(batch, tokens, inner, generator=g, device="cuda").bfloat16()
    base = torch.randn(batch, tokens, outer, generator=g, device="cuda").to(base_dtype)
    indices = torch.randint(-1, count + 1, (batch,), generator=g, device="cuda", dtype=torch.int32)
    x[0, 3, 5], x[0, tokens - 1, 0], base[-1, 1, 7] = torch.inf, torch.nan, torch.nan
    keep = torch.ones(batch, tokens, dtype=torch.bool, device="cuda")
    keep[0, 3] = keep[0, -1] = keep[-1, 1] = False
    want = {}
    for gelu in (False, True):
        for out_dtype in (torch.bfloat16, torch.float32):
            value, off = _expected(x, base, adapters, indices, gelu, out_dtype)
            got, _ = sm100_low_rank_add(x, base, adapters, indices, gelu=gelu, out_dtype=out_dtype)
            rows = keep.flatten()
            got = got.double().flatten(0, 1)[rows]
            bad = value[rows].isnan()
            assert torch.equal(got.isnan(), bad)
            assert float(torch.where(bad, 0, (got - value[rows]).abs() - off[rows]).max()) <= 0
            want[gelu, out_dtype] = got
    for gelu in (False, True):  # in place, and the same again
        there = base.clone()
        sm100_low_rank_add(x, there, adapters, indices, gelu=gelu, out=there)
        assert torch.equal(there.double().flatten(0, 1)[keep.flatten()].nan_to_num(5.0), want[gelu, base_dtype].nan_to_num(5.0))


@gpu
@pytest.mark.parametrize("rows", [7, 300, 2500])
def test_indices_of_runs_and_every_mix(rows) -> None:  # noqa: ANN001
    """One index for each sequence; all rows alike; every row another; none at all; indices past the set."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    adapters = _adapters(rows, 16, 64, 192, g)
    x = torch.randn(rows, 64, generator=g, device="cuda").bfloat16()
    base = torch.randn(rows, 192, generator=g, device="cuda")
    order = torch.randperm(rows, generator=g, device="cuda").to(torch.int32)
    for indices in (order, torch.full_like(order, rows - 1), torch.full_like(order, -5), order + rows // 2, -order):
        _check(x, base, adapters, indices, out_dtype=torch.bfloat16)
    _check(x.view(rows, 1, 64), base.view(rows, 1, 192), adapters, order)
    one = torch.tensor([rows - 1], dtype=torch.int32, device="cuda")
    _check(x, base, adapters, one)
    three = torch.tensor([2, -1, 0], dtype=torch.int32, device="cuda")
    _check(torch.randn(3, rows, 64, generator=g, device="cuda").bfloat16(), torch.randn(3, rows, 192, generator=g, device="cuda"),
           adapters, three, gelu=True)


@gpu
def test_rows_are_apart_and_infinities_are_the_formulas() -> None:
    """What a row holds changes no other row's result; an infinity stays one where the formula has it; rows without an adapter
    do not read x."""
    g = torch.Generator(device="cuda").manual_seed(3)
    adapters = _adapters(2, 8, 64, 128, g)  # filled up to 16 ranks: 0 x infinity must not come of that
    x = torch.randn(12, 64, generator=g, device="cuda").bfloat16()
    base = torch.randn(12, 128, generator=g, device="cuda")
    indices = torch.tensor([0, 1, 0, 0, 1, -1, -1, 1, 0, 2, 1, 0], dtype=torch.int32, device="cuda")
    clean, _ = sm100_low_rank_add(x, base, adapters, indices)
    x[2, 5], x[5], x[9, 0], x[10, 63] = torch.inf, torch.nan, torch.inf, torch.nan
    base[3, 7] = -torch.inf
    got, _ = sm100_low_rank_add(x, base, adapters, indices)
    same = [0, 1, 4, 5, 6, 7, 8, 11]
    assert torch.equal(got[same], clean[same])
    h = x[2].double() @ adapters.down[0].double().t()
    want = base[2].double() + (h @ adapters.up[0].double().t()) * adapters.scales[0].double()
    assert torch.equal(got[2].isnan(), want.isnan()) and torch.equal(got[2].isinf(), want.isinf())
    assert bool(got[9].isnan().all()) and bool(got[10].isnan().all())
    assert float(got[3, 7]) == -torch.inf and torch.equal(got[3, :7], clean[3, :7])
    for dtype in (torch.bfloat16, torch.float32):
        wide = torch.tensor([torch.inf, torch.nan, 1e30, -1e30, -50.0, 0.0, -0.0, 3.0] * 16, device="cuda").to(dtype)
        y, _ = sm100_low_rank_add(x[:1], wide[None], adapters, torch.tensor([-1], dtype=torch.int32, device="cuda"), gelu=True)
        assert float(y[0, 0]) == torch.inf and bool(y[0, 1].isnan()) and float(y[0, 2]) > 9e29 and abs(float(y[0, 3])) == 0


@gpu
def test_small_changes_beside_small_bases() -> None:
    """The R sums keep 2^-17 of themselves where the base is 0 and the result is 32 bits wide."""
    g = torch.Generator(device="cuda").manual_seed(8)
    adapters = _adapters(3, 16, 512, 256, g)
    x = torch.randn(40, 512, generator=g, device="cuda").bfloat16() * 2.0**-40
    indices = torch.randint(0, 3, (40,), generator=g, device="cuda", dtype=torch.int32)
    _check(x, torch.zeros(40, 256, device="cuda"), adapters, indices)


@gpu
def test_repeatable_and_the_same_in_a_graph_and_on_another_stream() -> None:
    g = torch.Generator(device="cuda").manual_seed(5)
    adapters = _adapters(6, 64, 1024, 2048, g)
    x = torch.randn(150, 1024, generator=g, device="cuda").bfloat16()
    base = torch.randn(150, 2048, generator=g, device="cuda").bfloat16()
    indices = torch.randint(-1, 6, (150,), generator=g, device="cuda", dtype=torch.int32)
    want, _ = sm100_low_rank_add(x, base, adapters, indices)
    for _ in range(3):
        assert torch.equal(sm100_low_rank_add(x, base, adapters, indices)[0], want)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            held, _ = sm100_low_rank_add(x, base, adapters, indices)
        graph.replay()
        beside, _ = sm100_low_rank_add(x, base, adapters, indices)
    stream.synchronize()
    assert torch.equal(held, want) and torch.equal(beside, want)
    # a replay goes by what the tensors hold by then
    indices.copy_(indices.flip(0))
    adapters.scales.mul_(2)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(held, sm100_low_rank_add(x, base, adapters, indices)[0]) and not torch.equal(held, want)


@gpu
def test_beyond_32_bit_offsets() -> None:
    """The last adapter of a set of more than 2^31 values, and rows past 2^31 values of the result."""
    g = torch.Generator(device="cuda").manual_seed(6)
    count, rank, inner, outer = 70, 128, 8, 260000  # up: 2.3e9 values
    down = torch.randn(count, rank, inner, generator=g, device="cuda").bfloat16()
    up = torch.zeros(count, outer, rank, dtype=torch.bfloat16, device="cuda")
    up[-1] = torch.randn(outer, rank, generator=g, device="cuda").bfloat16()
    adapters = LowRankAdapters(down, up, torch.ones(count, device="cuda"))
    x = torch.randn(3, inner, generator=g, device="cuda").bfloat16()
    base = torch.randn(3, outer, generator=g, device="cuda")
    _check(x, base, adapters, torch.tensor([count - 1, -1, count - 1], dtype=torch.int32, device="cuda"))
    del adapters, up
    adapters = _adapters(2, 8, 8, 40000, g)
    rows = 54000  # 2.16e9 values
    x = torch.randn(rows, 8, generator=g, device="cuda").bfloat16()
    base = torch.ones(rows, 40000, dtype=torch.bfloat16, device="cuda")
    indices = torch.arange(rows, device="cuda").remainder(3).sub(1).to(torch.int32)
    got, _ = sm100_low_rank_add(x, base, adapters, indices, out=base)
    last = slice(rows - 40, rows)
    want, off = _expected(x[last], torch.ones(40, 40000, device="cuda"), adapters, indices[last], False, torch.bfloat16)
    assert bool(((got[last].double() - want).abs() <= off).all())


@gpu
def test_beside_a_packed_projection() -> None:
    """The projection and its adapters as they are used: 4-bit weights, fp32 between the two, GELU after both."""
    g = torch.Generator(device="cuda").manual_seed(9)
    weight = pack_w4(torch.randn(512, 256, generator=g, device="cuda") / 16)
    adapters = _adapters(4, 16, 256, 512, g)
    x = torch.randn(6, 256, generator=g, device="cuda").bfloat16()
    indices = torch.tensor([0, 3, -1, 3, 2, 0], dtype=torch.int32, device="cuda")
    y, _ = sm100_linear_w4(x, weight, None, out_dtype=torch.float32)
    _check(x, y, adapters, indices, gelu=True, out_dtype=torch.bfloat16)


def test_stack_of_ranks() -> None:
    g = torch.Generator().manual_seed(1)
    parts = [(torch.randn(r, 24, generator=g), torch.randn(5, r, generator=g), 0.5 * r) for r in (4, 16, 1)]
    adapters = LowRankAdapters.stack(parts)
    assert (adapters.count, adapters.rank, adapters.in_features, adapters.out_features) == (3, 16, 24, 5)
    for i, (down, up, scale) in enumerate(parts):
        r = down.shape[0]
        assert torch.equal(adapters.down[i, :r], down.bfloat16()) and not adapters.down[i, r:].any()
        assert torch.equal(adapters.up[i, :, :r], up.bfloat16()) and not adapters.up[i, :, r:].any()
        assert float(adapters.scales[i]) == scale
    with pytest.raises(ValueError):
        LowRankAdapters.stack([])
    with pytest.raises(ValueError):
        LowRankAdapters.stack([parts[0], (torch.randn(4, 32), torch.randn(5, 4), 1.0)])
    with pytest.raises(ValueError):
        LowRankAdapters.stack([(torch.randn(129, 24), torch.randn(5, 129), 1.0)])


def test_handle_refusals() -> None:
    good = _adapters(2, 16, 32, 10, torch.Generator().manual_seed(0), device="cpu")
    for down, up, scales in (
        (good.down.float(), good.up, good.scales),
        (good.down[:1], good.up, good.scales),
        (good.down, good.up[..., :8], good.scales),
        (good.down[:, :12], good.up[..., :12], good.scales),
        (good.down[..., :28], good.up, good.scales),
        (good.down, good.up, good.scales.double()),
        (good.down, good.up, good.scales[:1]),
        (good.down.transpose(0, 1).contiguous().transpose(0, 1), good.up, good.scales),
        (good.down[:0], good.up[:0], good.scales[:0]),
    ):
        with pytest.raises(ValueError):
            LowRankAdapters(down, up, scales)
    with pytest.raises(AttributeError):
        good.down = good.down.clone()
    x, base = torch.zeros(3, 32, dtype=torch.bfloat16), torch.zeros(3, 10)
    assert not can_use_sm100_low_rank_add(x, base, good)
    with pytest.raises(RuntimeError):  # no CPU form
        sm100_low_rank_add(x, base, good, torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError):
        sm100_low_rank_add(x, base, good, torch.zeros(3, dtype=torch.int32), out_dtype=torch.float16)


@gpu
def test_results_over_what_the_call_reads_are_refused() -> None:
    adapters = _adapters(8, 8, 8, 8, torch.Generator(device="cuda").manual_seed(5))
    x = torch.zeros(1, 8, dtype=torch.bfloat16, device="cuda")
    base = torch.zeros(1, 8, device="cuda")
    indices = torch.zeros(1, dtype=torch.int32, device="cuda")
    over_indices = torch.zeros(8, device="cuda")
    for its, out in ((indices, adapters.scales.view(1, 8)), (over_indices.view(torch.int32)[5:6], over_indices.view(1, 8))):
        with pytest.raises(ValueError, match="shares memory"):
            sm100_low_rank_add(x, base, adapters, its, out=out)


@gpu
def test_refusals() -> None:
    g = torch.Generator(device="cuda").manual_seed(2)
    adapters = _adapters(2, 16, 64, 48, g)
    x = torch.zeros(6, 64, dtype=torch.bfloat16, device="cuda")
    base = torch.zeros(6, 48, device="cuda")
    indices = torch.zeros(6, dtype=torch.int32, device="cuda")
    assert can_use_sm100_low_rank_add(x, base, adapters)
    for bad_x, bad_base in (
        (x.float(), base),
        (x[:, :32], base),
        (x[:, :56], base),
        (x[:0], base[:0]),
        (x[::2], base[:3]),
        (x, base[:5]),
        (x, base[:, :40]),
        (x, base.half()),
        (x, base.t().contiguous().t()),
        (x.view(2, 3, 64), base),
        (torch.zeros(6 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(6, 64), base),
        (x, torch.zeros(6 * 48 + 1, device="cuda")[1:].view(6, 48)),
    ):
        assert not can_use_sm100_low_rank_add(bad_x, bad_base, adapters)
        with pytest.raises(RuntimeError):
            sm100_low_rank_add(bad_x, bad_base, adapters, indices)
    for bad in (indices.long(), indices[:4], indices[:0], indices.cpu(), torch.zeros(12, dtype=torch.int32, device="cuda")[::2]):
        with pytest.raises(ValueError):
            sm100_low_rank_add(x, base, adapters, bad)
    room = torch.zeros(2 * 6 * 48, device="cuda")
    for out in (
        torch.zeros(6, 48, dtype=torch.bfloat16, device="cuda"),
        torch.zeros(5, 48, device="cuda"),
        torch.zeros(48, 6, device="cuda").t(),
        torch.zeros(6, 48),
    ):
        with pytest.raises(ValueError):
            sm100_low_rank_add(x, base, adapters, indices, out=out)
    with pytest.raises(ValueError):  # part of base
        sm100_low_rank_add(x, room[: 6 * 48].view(6, 48), adapters, indices, out=room[48 : 7 * 48].view(6, 48))
    with pytest.raises(ValueError):  # base's memory in another type
        sm100_low_rank_add(x, base, adapters, indices, out_dtype=torch.bfloat16,
                           out=base.view(torch.bfloat16).view(-1)[: 6 * 48].view(6, 48))
    with pytest.raises(ValueError):  # the adapters' memory
        sm100_low_rank_add(x, base, adapters, indices, out_dtype=torch.bfloat16, out=adapters.up.view(-1)[: 6 * 48].view(6, 48))
    with pytest.raises(ValueError):  # x's memory
        sm100_low_rank_add(x, base, adapters, indices, out_dtype=torch.bfloat16, out=x.view(-1)[: 6 * 48].view(6, 48))
    with torch.inference_mode(False), torch.enable_grad(), pytest.raises(RuntimeError):
        sm100_low_rank_add(x, base, adapters, indices)


def test_c_entry_refusals() -> None:
    lib = _native.load()

    def call(x=16, base=16, base_dtype=0, out=32, out_dtype=0, down=16, up=16, scales=16, indices=16, count=4, m=4, n=8,  # noqa: ANN001, ANN202
             k=8, rank=8, adapters=1, epilogue=0):  # noqa: ANN001
        return lib.b200tx_low_rank_add(x, base, base_dtype, out, out_dtype, down, up, scales, indices, count, m, n, k, rank,
                                       adapters, epilogue, None)

    for bad in (
        {"x": None}, {"base": None}, {"out": None}, {"down": None}, {"up": None}, {"scales": None}, {"indices": None},
        {"x": 8}, {"base": 8}, {"out": 8}, {"down": 8}, {"up": 8}, {"m": 0}, {"n": 0}, {"k": 0}, {"k": 12}, {"rank": 0},
        {"rank": 4}, {"rank": 136}, {"adapters": 0}, {"count": 0}, {"count": 3}, {"base_dtype": 2}, {"out_dtype": 7},
        {"epilogue": 3}, {"m": 1 << 27}, {"base": 32, "base_dtype": 1},
    ):
        assert call(**bad) < 0, bad
