"""Linear layers with 4-bit weights for a few rows (csrc/linear_w4_kernels.cuh).

``sm100_linear`` reads 16-bit weights and pads the rows to a tensor-core tile;
a decoding step has one row per sequence and is bound by the weights' bytes.
Here a weight is ``scale * (code - 8)``, codes in 4 bits, a bf16 scale for each
group of 32, 64 or 128 along K.
"""

from __future__ import annotations

import torch

from ._common import TensorHandle, binding, is_sm100_cuda, library_ready, require

SM100_LINEAR_W4_BACKEND = "sm100_linear_w4"
SM100_LINEAR_W4_GELU_BACKEND = "sm100_linear_w4_gelu"
W4_GROUPS = (32, 64, 128)
_RUN = 128  # weights of a row that are stored together
_ORDER = (0, 2, 4, 6, 1, 3, 5, 7)  # nibble i of a word holds weight _ORDER[i] of its eight

_OUT = (torch.float32, torch.bfloat16)


class W4Weight(TensorHandle):
    """A packed ``[N, K]`` weight.

    * ``packed`` uint8 ``[N, Kp / 2]``, ``Kp`` = K rounded up to 128.  128 weights of a
      row are 16 little-endian words of 8, nibble i of a word holding weight
      ``(0, 2, 4, 6, 1, 3, 5, 7)[i]``; word ``4 a + b`` is stored at ``4 b + a``
    * ``scales`` bf16 ``[Kp / group, N]``
    """

    def __init__(self, packed: torch.Tensor, scales: torch.Tensor, in_features: int) -> None:
        wide = -(-in_features // _RUN) * _RUN
        require(
            in_features > 0 and in_features % 8 == 0 and packed.dtype == torch.uint8 and packed.ndim == 2
            and packed.shape[1] == wide // 2 and packed.shape[0] > 0,
            "packed must be a uint8 [N, Kp / 2] tensor, Kp = K rounded up to 128, K a multiple of 8",
        )
        require(
            scales.dtype == torch.bfloat16 and scales.ndim == 2 and scales.shape[1] == packed.shape[0]
            and scales.shape[0] > 0 and wide % scales.shape[0] == 0 and wide // scales.shape[0] in W4_GROUPS,
            "scales must be a bfloat16 [Kp / group, N] tensor, group 32, 64 or 128",
        )
        require(
            packed.is_contiguous() and scales.is_contiguous() and packed.device == scales.device
            and packed.data_ptr() % 16 == 0,
            "packed and scales must be contiguous on one device, packed 16-byte aligned",
        )
        self.packed = packed
        self.scales = scales
        self.in_features = int(in_features)
        self.out_features = packed.shape[0]
        self.group = wide // scales.shape[0]
        self.device = packed.device

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The ``[N, K]`` weight that the codes stand for."""

        n = self.out_features
        code = torch.stack((self.packed & 15, self.packed >> 4), -1).reshape(n, -1, 4, 4, 8).transpose(2, 3)
        inverse = [_ORDER.index(i) for i in range(8)]
        code = code[..., inverse].reshape(n, -1, self.group).to(torch.float32) - 8
        weight = code * self.scales.t().to(torch.float32)[..., None]
        return weight.reshape(n, -1)[:, : self.in_features].to(dtype)


def pack_w4(weight: torch.Tensor, group: int = 64) -> W4Weight:
    """Quantise a ``[N, K]`` weight, K a multiple of 8: per group
    ``scale = bf16(max |w| / 7)`` and the nearest code (once, when a model is
    loaded; plain torch on the weight's device)."""

    require(weight.ndim == 2 and weight.is_floating_point() and weight.numel() > 0, "weight must be a float [N, K] tensor")
    require(group in W4_GROUPS, f"group {group} is not one of {W4_GROUPS}")
    n, k = weight.shape
    require(k % 8 == 0, "K must be a multiple of 8")
    wide = -(-k // _RUN) * _RUN
    w = torch.nn.functional.pad(weight.detach().float(), (0, wide - k)).reshape(n, wide // group, group)
    scale = (w.abs().amax(-1) / 7).bfloat16()
    step = scale.float()[..., None]
    code = torch.where(step > 0, w / step, torch.zeros_like(w)).round().clamp(-8, 7).add(8).to(torch.uint8)
    code = code.reshape(n, wide // _RUN, 4, 4, 8)[..., list(_ORDER)].transpose(2, 3).reshape(n, wide // 2, 2)
    return W4Weight(code[..., 0] | (code[..., 1] << 4), scale.t().contiguous(), k)


def can_use_sm100_linear_w4(value: torch.Tensor, weight: W4Weight, bias: torch.Tensor | None = None) -> bool:
    """Whether the kernel can run on these operands (never raises)."""

    try:
        return (
            library_ready()
            and is_sm100_cuda(value)
            and binding().linear_w4_ok(value, weight.packed, bias, weight.in_features)
        )
    except Exception:  # noqa: BLE001 - predicate contract: never raise
        return False


def sm100_linear_w4(
    value: torch.Tensor,
    weight: W4Weight,
    bias: torch.Tensor | None = None,
    *,
    gelu: bool = False,
    out_dtype: torch.dtype = torch.bfloat16,
    out: torch.Tensor | None = None,
) -> tuple[torch.Tensor, str]:
    """``[..., K] x [N, K]^T -> [..., N]`` with a packed weight: bf16 ``value``,
    fp32 accumulation, fp32 bias and erf GELU before the cast.  Made for few rows:
    beyond 16 they are taken 16 at a time, or 32 where N is at least 80 for each SM,
    each time reading the weight again.  ``out`` shares no memory with ``value``."""

    require(out_dtype in _OUT, "out_dtype must be float32 or bfloat16")
    result = binding().linear_w4(
        value, weight.packed, weight.scales, bias, weight.in_features, weight.group, gelu,
        out_dtype == torch.float32, out,
    )
    return result, SM100_LINEAR_W4_GELU_BACKEND if gelu else SM100_LINEAR_W4_BACKEND


__all__ = [
    "SM100_LINEAR_W4_BACKEND",
    "SM100_LINEAR_W4_GELU_BACKEND",
    "W4Weight",
    "W4_GROUPS",
    "can_use_sm100_linear_w4",
    "pack_w4",
    "sm100_linear_w4",
]
