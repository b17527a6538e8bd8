"""4-bit linear layers of many columns whose x does not go to shared memory: the ring
kernels with two column tiles a warp (up to 16 rows) and with 32 rows of x.

Tolerance: the product is summed in fp32, K / 16 tensor-core steps and K / 32 group sums,
each off by at most 2^-23 of the sum of magnitudes; a bf16 result carries 2^-8 more."""

from __future__ import annotations

import pytest
import torch

from solution.kernels import pack_w4, sm100_linear_w4

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _randn(*shape: int, seed: int) -> torch.Tensor:
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV)


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize(
    ("rows", "inner", "outer"),
    [
        (8, 2048, 12288), (3, 1032, 11841), (1, 8, 12001),  # 8 rows, two column tiles
        (16, 8192, 14336), (13, 1000, 12007), (9, 264, 11855),  # 16 rows, two column tiles
        (32, 4096, 14336), (29, 520, 11999), (17, 128, 11841), (71, 776, 12000),  # 32 rows
    ],
)
def test_linear_w4_many_columns(rows: int, inner: int, outer: int, group: int, out_dtype: torch.dtype) -> None:
    with torch.inference_mode():
        weight = pack_w4(_randn(outer, inner, seed=outer) * inner**-0.5, group)
        x = _randn(rows, inner, seed=rows).bfloat16()
        bias = _randn(outer, seed=3) if rows % 2 else None
        got, _ = sm100_linear_w4(x, weight, bias, out_dtype=out_dtype)
        w = weight.dequantize(torch.float64)
        want = x.double() @ w.t() + (0 if bias is None else bias.double())
        mass = x.double().abs() @ w.abs().t() + (0 if bias is None else bias.double().abs())
        bound = (inner / 16 + inner / 32 + 16) * 2.0**-23 * mass
        if out_dtype == torch.bfloat16:
            bound = bound + 2.0**-8 * (want.abs() + bound)
        off = (got.double() - want).abs()
        assert bool((off <= bound).all()), float((off / bound).max())
        assert torch.equal(sm100_linear_w4(x, weight, bias, out_dtype=out_dtype)[0], got)
        x[rows - 1, inner // 2] = float("nan")  # stays in its own row
        got, _ = sm100_linear_w4(x, weight, bias, out_dtype=out_dtype)
        assert got.isnan().all(-1).tolist() == [False] * (rows - 1) + [True] and not got[:-1].isnan().any()


@pytest.mark.parametrize("rows", [65535 * 16, 65535 * 16 + 1, 1 << 20])
def test_linear_w4_as_many_rows_as_there_may_be(rows: int) -> None:
    with torch.inference_mode():
        weight = pack_w4(_randn(3, 16, seed=1), 32)
        x = _randn(rows, 16, seed=2).bfloat16()
        got, _ = sm100_linear_w4(x, weight, out_dtype=torch.float32)
        want = x.double() @ weight.dequantize(torch.float64).t()
        bound = 18 * 2.0**-23 * (x.double().abs() @ weight.dequantize(torch.float64).abs().t())
        assert bool(((got.double() - want).abs() <= bound).all())
