"""Low-rank adapters of many requests beside a shared projection
(csrc/low_rank_kernels.cuh).

The reference runs one set of weights.  A serving batch shares its projections
(``sm100_linear``, ``sm100_linear_w4``), and each request may bring a low-rank
change of its own: ``sm100_low_rank_add`` adds every row's to the projection's
output, with the GELU that would otherwise follow the projection.

    y, _ = sm100_linear_w4(x, weight, bias, out_dtype=torch.float32)
    h, _ = sm100_low_rank_add(x, y, adapters, indices, gelu=True, out_dtype=torch.bfloat16)
"""

from __future__ import annotations

from collections.abc import Sequence

import torch

from ._common import TensorHandle, binding, is_sm100_cuda, library_ready, require

SM100_LOW_RANK_ADD_BACKEND = "sm100_low_rank_add"
SM100_LOW_RANK_ADD_GELU_BACKEND = "sm100_low_rank_add_gelu"
LOW_RANK_MOST = 128

_OUT = (torch.float32, torch.bfloat16)


class LowRankAdapters(TensorHandle):
    """The adapters of one projection, ``scales[a] * up[a] @ down[a]`` each.

    * ``down`` bf16 ``[count, R, K]``, R a multiple of 8 up to 128, K a multiple of 8
    * ``up`` bf16 ``[count, N, R]``
    * ``scales`` float32 ``[count]``

    Their values may be changed in place between calls (an adapter loaded over another).  They are
    finite numbers: with an infinite one of ``up``, NaN may stand where the formula has an infinity.
    """

    def __init__(self, down: torch.Tensor, up: torch.Tensor, scales: torch.Tensor) -> None:
        require(
            down.ndim == 3 and up.ndim == 3 and down.dtype == up.dtype == torch.bfloat16
            and down.shape[0] == up.shape[0] > 0 and down.shape[1] == up.shape[2],
            "down must be a bfloat16 [count, R, K] tensor and up a bfloat16 [count, N, R] one",
        )
        count, rank, inner = down.shape
        require(
            rank % 8 == 0 and 0 < rank <= LOW_RANK_MOST and inner % 8 == 0 and inner > 0 and up.shape[1] > 0,
            f"R must be a multiple of 8 up to {LOW_RANK_MOST}, K a multiple of 8",
        )
        require(scales.dtype == torch.float32 and tuple(scales.shape) == (count,), "scales must be a float32 [count] tensor")
        require(
            all(t.is_contiguous() and t.device == down.device for t in (down, up, scales))
            and down.data_ptr() % 16 == 0 and up.data_ptr() % 16 == 0,
            "the adapters' tensors must be contiguous on one device, down and up 16-byte aligned",
        )
        self.down, self.up, self.scales = down, up, scales
        self.count, self.rank = count, rank
        self.in_features, self.out_features = inner, up.shape[1]
        self.device = down.device

    @classmethod
    def stack(
        cls, adapters: Sequence[tuple[torch.Tensor, torch.Tensor, float]], device: torch.device | str | None = None
    ) -> LowRankAdapters:
        """Adapters ``(down [r, K], up [N, r], scale)`` of any ranks up to 128 as one set,
        each rounded to bf16 and filled up with zeros to the largest rank."""

        require(len(adapters) > 0, "there must be an adapter at least")
        require(all(down.ndim == 2 and up.ndim == 2 for down, up, _ in adapters), "an adapter is (down [r, K], up [N, r], scale)")
        first_down, first_up, _ = adapters[0]
        inner, outer = first_down.shape[1], first_up.shape[0]
        rank = 8 * max(1, max(-(-down.shape[0] // 8) for down, _, _ in adapters))
        require(rank <= LOW_RANK_MOST, f"an adapter's rank is at most {LOW_RANK_MOST}")
        device = first_down.device if device is None else device
        down_all = torch.zeros(len(adapters), rank, inner, dtype=torch.bfloat16, device=device)
        up_all = torch.zeros(len(adapters), outer, rank, dtype=torch.bfloat16, device=device)
        scales = torch.empty(len(adapters), dtype=torch.float32)
        for i, (down, up, scale) in enumerate(adapters):
            require(
                down.shape[1] == inner and up.shape[0] == outer and down.shape[0] == up.shape[1],
                "the adapters of a set must fit one projection",
            )
            down_all[i, : down.shape[0]] = down.detach()
            up_all[i, :, : up.shape[1]] = up.detach()
            scales[i] = float(scale)
        return cls(down_all, up_all, scales.to(device))


def can_use_sm100_low_rank_add(value: torch.Tensor, base: torch.Tensor, adapters: LowRankAdapters) -> bool:
    """Whether the kernel can run on these operands (never raises)."""

    try:
        return (
            library_ready()
            and is_sm100_cuda(value)
            and binding().low_rank_add_ok(value, base, adapters.down, adapters.up)
        )
    except Exception:  # noqa: BLE001 - predicate contract: never raise
        return False


def sm100_low_rank_add(
    value: torch.Tensor,
    base: torch.Tensor,
    adapters: LowRankAdapters,
    indices: torch.Tensor,
    *,
    gelu: bool = False,
    out_dtype: torch.dtype | None = None,
    out: torch.Tensor | None = None,
) -> tuple[torch.Tensor, str]:
    """``base + scale * (value . down^T) . up^T`` with each row's adapter: bf16 ``value``
    ``[..., K]``, ``base`` ``[..., N]`` (float32 or bf16) the projection's output, erf GELU
    after the sum with ``gelu``.  fp32 inside, one rounding to ``out_dtype``
    (default: ``base``'s).  For a bf16 result the row's R sums keep 2^-17 of themselves, and the GELU is
    within 1.5e-7 (4e-4 of the value down to -6) before the rounding.

    ``indices`` int32 holds one adapter for each of the equal runs of rows that it divides
    them into: ``[B]`` for ``[B, T, K]``, or one for each row.  A negative one: no adapter;
    one past the set: the row becomes NaN.  ``out`` may be ``base`` itself, in its dtype.

    Many rows are fastest where an index stands for 64 of them or more and N is a multiple of 8: they
    go by 128 then (8 prompts of 2048 rows, 1024 -> 4096, rank 64: 80 us with 8 indices, 238 with one for each row)."""

    require(out_dtype is None or out_dtype in _OUT, "out_dtype must be float32 or bfloat16")
    result = binding().low_rank_add(
        value, base, adapters.down, adapters.up, adapters.scales, indices, gelu,
        None if out_dtype is None else out_dtype == torch.float32, out,
    )
    return result, SM100_LOW_RANK_ADD_GELU_BACKEND if gelu else SM100_LOW_RANK_ADD_BACKEND


__all__ = [
    "LOW_RANK_MOST",
    "LowRankAdapters",
    "SM100_LOW_RANK_ADD_BACKEND",
    "SM100_LOW_RANK_ADD_GELU_BACKEND",
    "can_use_sm100_low_rank_add",
    "sm100_low_rank_add",
]
