"""RMS norm of each query and key head and the rotation by position, in one
pass over the packed projection (csrc/rope_kernels.cuh).

The reference's model has neither (its block applies the projection as it is,
official/torch_transformer_benchmark.py:85-104); models that decode token by
token put both on their queries and keys.  The packed layout is the one the
attention kernels read, ``[B, T, (H + 2 Hkv) * D]`` with query, key and value
heads in this order, so the result goes straight into them; with ``Hkv < H``
groups of query heads share a kv head.
"""

from __future__ import annotations

import ctypes

import torch

from .. import _native
from ._common import TensorHandle, binding, is_sm100_cuda, library_ready, require

SM100_QK_NORM_ROPE_BACKEND = "sm100_qk_norm_rope"
ROPE_HEAD_DIMS = (8, 16, 32, 64, 128, 256)


class RotaryTable(TensorHandle):
    """cos and sin of the angles, fp32 ``[positions, rotary / 2]``.

    The first ``rotary`` dims of a head are turned: pairs ``(i, i + rotary/2)``,
    or ``(2i, 2i + 1)`` with ``interleaved``.  ``rotary`` is a multiple of 8 (of
    16 for head_dim 256).  At a position outside the table the turned dims are NaN.
    """

    def __init__(self, cos: torch.Tensor, sin: torch.Tensor, *, interleaved: bool = False) -> None:
        require(
            cos.ndim == 2 and cos.shape == sin.shape and cos.dtype == sin.dtype == torch.float32
            and cos.is_contiguous() and sin.is_contiguous() and cos.device == sin.device
            and cos.shape[0] > 0 and cos.shape[1] > 0,
            "cos and sin must be contiguous float32 [positions, rotary / 2] tensors on one device",
        )
        self.cos = cos
        self.sin = sin
        self.interleaved = bool(interleaved)
        self.rotary = 2 * cos.shape[1]
        self.device = cos.device
        self._struct = _native.Rope(cos.data_ptr(), sin.data_ptr(), cos.shape[0], self.rotary, int(self.interleaved))
        # what the binding takes: the struct's address, the turned dims and the device
        self.handle = (ctypes.addressof(self._struct), self.rotary, cos.get_device())

    @classmethod
    def create(
        cls, positions: int, rotary: int, device: torch.device | str, *, base: float = 10000.0, interleaved: bool = False
    ) -> RotaryTable:
        """The angles ``position * base ** (-2 i / rotary)``, taken in float64."""

        steps = torch.arange(0, rotary, 2, dtype=torch.float64) / rotary
        angle = torch.arange(positions, dtype=torch.float64)[:, None] * base**-steps
        return cls(angle.cos().float().to(device), angle.sin().float().to(device), interleaved=interleaved)


def can_use_sm100_qk_norm_rope(qkv: torch.Tensor, num_heads: int, num_kv_heads: int | None = None) -> bool:
    """Whether the kernel can read this packed projection (never raises)."""

    try:
        return (
            library_ready()
            and is_sm100_cuda(qkv)
            and binding().qk_norm_rope_ok(qkv, num_heads, num_heads if num_kv_heads is None else num_kv_heads)
        )
    except Exception:  # noqa: BLE001 - predicate contract: never raise
        return False


def sm100_qk_norm_rope(
    qkv: torch.Tensor,
    num_heads: int,
    num_kv_heads: int | None = None,
    *,
    q_weight: torch.Tensor | None = None,
    k_weight: torch.Tensor | None = None,
    eps: float = 1e-6,
    rope: RotaryTable | None = None,
    positions: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
) -> tuple[torch.Tensor, str]:
    """Query and key heads of ``qkv`` ``[B, T, (H + 2 Hkv) * D]`` normed
    (``x / sqrt(mean(x^2) + eps) * weight``; no weight, no norm) and turned by
    their positions (int32 or int64 ``[B, T]`` or ``[T]``; default 0..T-1), value
    heads as they are.  fp32 inside, one rounding to ``qkv``'s dtype.  ``out=qkv``
    works in place and leaves the value heads alone."""

    result = binding().qk_norm_rope(
        qkv, num_heads, num_heads if num_kv_heads is None else num_kv_heads, q_weight, k_weight, eps,
        None if rope is None else rope.handle, positions, out,
    )
    return result, SM100_QK_NORM_ROPE_BACKEND


__all__ = [
    "ROPE_HEAD_DIMS",
    "RotaryTable",
    "SM100_QK_NORM_ROPE_BACKEND",
    "can_use_sm100_qk_norm_rope",
    "sm100_qk_norm_rope",
]
