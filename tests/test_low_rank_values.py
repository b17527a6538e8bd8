"""Values of the low-rank adapters where they are hardest: the GELU's tail and infinities, sums that need all terms, and
offsets past 2^31 values in both forms of the kernel.

Tolerance of a GELU whose result has 16 bits: the polynomial, evaluated in fp32, is off by at most 1.05e-7 (in 64 bits over all
fp32 values of a fine grid), the hardware's exponential by 2^-22 of a Q(a) <= 0.17, which is 4.1e-8, together less than
1.5e-7 in absolute terms; then an addition in fp32 (2^-24 of the value) and one rounding of at most half a step of bf16."""

from __future__ import annotations

import pytest
import torch

from solution.kernels import LowRankAdapters, sm100_linear, sm100_low_rank_add

gpu = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def _inference():
    with torch.inference_mode():
        yield
    if torch.cuda.is_available():
        torch.cuda.synchronize()


def _none(rows, inner=64, outer=64, rank=64):  # noqa: ANN001, ANN202
    """Operands whose rows have no adapter: x, adapters, indices (one for all rows)."""
    adapters = LowRankAdapters(
        torch.ones(1, rank, inner, device=DEV).bfloat16(), torch.ones(1, outer, rank, device=DEV).bfloat16(), torch.ones(1, device=DEV)
    )
    return torch.ones(rows, inner, device=DEV).bfloat16(), adapters, torch.tensor([-1], dtype=torch.int32, device=DEV)


@gpu
@pytest.mark.parametrize("rows", [8, 1024])  # groups of 8 rows, and of 128
@pytest.mark.parametrize("base_dtype", [torch.bfloat16, torch.float32])
def test_gelu_of_16_bits_over_its_range(rows, base_dtype) -> None:  # noqa: ANN001
    """Every bf16 value of [-16, 6], and beside them the whole range's largest."""
    bits = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    grid = bits[(bits.float() >= -16) & (bits.float() <= 6)]
    grid = torch.cat((grid, torch.tensor([-3e38, -1e5, -17.0, 7.0, 17.0, 1e5, 3e38]).bfloat16()))
    outer = -(-grid.numel() // 64) * 64
    grid = torch.nn.functional.pad(grid, (0, outer - grid.numel())).to(DEV)
    x, adapters, index = _none(rows, outer=outer)
    got, _ = sm100_low_rank_add(x, grid.to(base_dtype).expand(rows, outer).contiguous(), adapters, index, gelu=True,
                                out_dtype=torch.bfloat16)
    wide = grid.double()
    want = wide * torch.special.ndtr(wide)
    off = 1.5e-7 + want.abs() * 2.0**-24
    off += (want.abs() + off) * torch.finfo(torch.bfloat16).eps / 2
    assert float(((got.double() - want).abs() - off).max()) <= 0
    # down to -6 also 4e-4 of the value itself (3.75e-4 in 64 bits, and 30 x 2^-24 of the exponent in fp32), and the rounding
    tail = (wide <= 0) & (wide >= -6) & (want.abs() > 2.0**-100)
    assert float(((got[0].double() - want)[tail] / want[tail]).abs().max()) <= 4e-4 + 2.0**-8 + 2.0**-20


@gpu
@pytest.mark.parametrize("rows", [3, 1024])
@pytest.mark.parametrize("outer", [64, 67])
@pytest.mark.parametrize("base_dtype", [torch.bfloat16, torch.float32])
def test_gelu_of_infinities(rows, outer, base_dtype) -> None:  # noqa: ANN001
    """As x Phi(x) has them, and the framework's projections: NaN at -infinity, whatever the result's type."""
    x, adapters, index = _none(rows, outer=outer)
    base = torch.zeros(rows, outer, device=DEV, dtype=base_dtype)
    base[:, 5], base[:, 9], base[:, 11], base[:, 60] = -torch.inf, torch.inf, torch.nan, -torch.inf
    bias = torch.zeros(64, device=DEV)
    bias[0] = -torch.inf
    known, _ = sm100_linear(torch.zeros(8, 64, device=DEV).bfloat16(), torch.zeros(64, 64, device=DEV).bfloat16(), bias, gelu=True)
    assert bool(known[0, 0].isnan())
    for adapter in (-1, 0):  # nothing is added, or 64 x 64 ones are
        want = base.double() + (64.0 * 64.0 if adapter == 0 else 0.0)
        want = want * torch.special.ndtr(want)
        for out_dtype in (torch.bfloat16, torch.float32):
            got, _ = sm100_low_rank_add(x, base, adapters, index.fill_(adapter), gelu=True, out_dtype=out_dtype)
            assert torch.equal(got.double().nan_to_num(nan=7.0), want.nan_to_num(nan=7.0)), (adapter, out_dtype)


@gpu
@pytest.mark.parametrize(
    ("rows", "runs", "rank", "outer"),
    [(5, 5, 16, 67), (40, 40, 40, 264), (70, 70, 128, 96), (2048, 2, 64, 264), (1024, 8, 128, 1032), (2000, 2000, 72, 72),
     (2048, 32, 40, 200)],
)
@pytest.mark.parametrize("base_dtype", [torch.bfloat16, torch.float32])
def test_sums_keep_all_their_bits(rows, runs, rank, outer, base_dtype) -> None:  # noqa: ANN001
    """Whole numbers: sums of 20 to 24 bits, exact in fp32, that one rank of up brings to a column each.  A result of 32 bits is the
    sum itself (three bf16 terms; with two, or one of them elsewhere, the last bits are lost)."""
    g = torch.Generator(device=DEV).manual_seed(rank + outer)
    inner, count = 256, 3
    x = torch.randint(1, 256, (rows, inner), generator=g, device=DEV).bfloat16()
    down = torch.randint(1, 256, (count, rank, inner), generator=g, device=DEV).bfloat16()
    of = torch.randint(0, rank, (count, outer), generator=g, device=DEV)
    up = torch.nn.functional.one_hot(of, rank).bfloat16()
    adapters = LowRankAdapters(down, up, torch.ones(count, device=DEV))
    indices = torch.randint(0, count, (runs,), generator=g, device=DEV, dtype=torch.int32)
    base = torch.zeros(rows, outer, device=DEV, dtype=base_dtype)
    got, _ = sm100_low_rank_add(x, base, adapters, indices, out_dtype=torch.float32)
    sums = torch.einsum("mk,ark->mar", x.double(), down.double())  # [rows, count, rank]
    assert 2**20 < float(sums.min()) and float(sums.max()) < 2**24
    index = indices.long().repeat_interleave(rows // runs)
    want = sums[torch.arange(rows, device=DEV), index].gather(1, of[index])
    assert torch.equal(got.double(), want)


@gpu
def test_prompts_past_32_bit_offsets() -> None:
    """Rows past 2^31 values of the result, and an adapter past 2^31 values of up, 128 rows at a time."""
    g = torch.Generator(device=DEV).manual_seed(3)
    rows, outer = 54000, 40000  # 2.16e9 values
    adapters = LowRankAdapters(
        torch.randn(2, 8, 8, generator=g, device=DEV).bfloat16(), torch.randn(2, outer, 8, generator=g, device=DEV).bfloat16(),
        torch.ones(2, device=DEV),
    )
    x = torch.randn(rows, 8, generator=g, device=DEV).bfloat16()
    base = torch.ones(rows, outer, dtype=torch.bfloat16, device=DEV)
    indices = (torch.arange(54, device=DEV) % 3 - 1).flip(0).to(torch.int32)  # the last run has adapter -1, the one before 0
    got, _ = sm100_low_rank_add(x, base, adapters, indices, out=base)
    # the same rows by themselves, warp by warp: their offsets are small
    for run, adapter in ((52, 0), (53, -1), (51, 1)):
        assert int(indices[run]) == adapter
        last = slice((run + 1) * 1000 - 40, (run + 1) * 1000)
        alone, _ = sm100_low_rank_add(x[last], torch.ones(40, outer, dtype=torch.bfloat16, device=DEV), adapters, indices[run : run + 1])
        # both round the same value, which sums in another order may differ in by 2^-20 of the magnitudes
        size = 1 + 64 * x[last].abs().max().double() * adapters.down.abs().max().double() * adapters.up.abs().max().double()
        off = alone.double().abs() * torch.finfo(torch.bfloat16).eps + size * 2.0**-16
        assert bool(((got[last].double() - alone.double()).abs() <= off).all())
    del base, got, adapters
    count, rank, outer = 70, 128, 260000  # up: 2.3e9 values
    up = torch.zeros(count, outer, rank, dtype=torch.bfloat16, device=DEV)
    of = torch.arange(outer, device=DEV) % rank
    up[-1].scatter_(1, of[:, None], 1.0)
    down = torch.zeros(count, rank, 8, dtype=torch.bfloat16, device=DEV)
    down[-1] = torch.randint(-200, 200, (rank, 8), generator=g, device=DEV).bfloat16()
    x = torch.randint(-200, 200, (1024, 8), generator=g, device=DEV).bfloat16()
    adapters = LowRankAdapters(down, up, torch.ones(count, device=DEV))
    got, _ = sm100_low_rank_add(x, torch.zeros(1024, outer, device=DEV), adapters,
                                torch.tensor([count - 1], dtype=torch.int32, device=DEV))
    sums = x.double() @ down[-1].double().t()
    for rows in (slice(0, 8), slice(1016, 1024)):
        assert torch.equal(got[rows].double(), sums[rows][:, of])
