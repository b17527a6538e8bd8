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
from ._common import is_sm100_cuda, launch, library_ready, require

SM100_QK_NORM_ROPE_BACKEND = "sm100_qk_norm_rope"
ROPE_HEAD_DIMS = (8, 16, 32, 64, 128, 256)

_IO = (torch.float32, torch.bfloat16)


class RotaryTable:
    """cos and sin of the angles, fp32 ``[positions, rotary / 2]``.

    The first ``rotary`` dims of a head are turned: pairs ``(i, i + rotary/2)``,
    or ``(2i, 2i + 1)`` with ``interleaved``.  ``rotary`` is a multiple of 8 (of
    16 for head_dim 256).  A position outside the table gives NaN heads.
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
        self.reference = ctypes.byref(self._struct)

    @classmethod
    def create(
        cls, positions: int, rotary: int, device: torch.device | str, *, base: float = 10000.0, interleaved: bool = False
    ) -> RotaryTable:
        """The angles ``position * base ** (-2 i / rotary)``, taken in float64."""

        steps = torch.arange(0, rotary, 2, dtype=torch.float64) / rotary
        angle = torch.arange(positions, dtype=torch.float64)[:, None] * base**-steps
        return cls(angle.cos().float().to(device), angle.sin().float().to(device), interleaved=interleaved)


def check_norm_weights(
    q_weight: torch.Tensor | None, k_weight: torch.Tensor | None, head_dim: int, device: torch.device
) -> None:
    for weight in (q_weight, k_weight):
        if weight is not None:
            require(
                weight.dtype == torch.float32 and weight.shape == (head_dim,) and weight.is_contiguous()
                and weight.device == device and weight.data_ptr() % 16 == 0,
                "the norm weights must be contiguous, 16-byte aligned float32 [head_dim] tensors on the input's device",
            )


def check_rope(rope: RotaryTable | None, head_dim: int, device: torch.device) -> None:
    if rope is not None:
        require(rope.device == device, "the rotation table must be on the input's device")
        require(
            rope.rotary <= head_dim and rope.rotary % (16 if head_dim == 256 else 8) == 0,
            f"rotary {rope.rotary} must be a multiple of {16 if head_dim == 256 else 8} up to head_dim {head_dim}",
        )


def packed_ok(qkv: torch.Tensor) -> bool:
    """Layout the kernels read: dense heads, any 16-byte aligned token and batch strides."""

    return (
        qkv.ndim == 3
        and qkv.dtype in _IO
        and qkv.stride(2) == 1
        and qkv.stride(0) % 8 == 0
        and qkv.stride(1) % 8 == 0
        and qkv.data_ptr() % 16 == 0
        and qkv.numel() > 0
    )


def can_use_sm100_qk_norm_rope(qkv: torch.Tensor, num_heads: int, num_kv_heads: int | None = None) -> bool:
    """Whether the kernel can read this packed projection (never raises)."""

    try:
        if not library_ready() or torch.is_grad_enabled() or not is_sm100_cuda(qkv) or not packed_ok(qkv):
            return False
        kv_heads = num_heads if num_kv_heads is None else num_kv_heads
        total = num_heads + 2 * kv_heads
        if num_heads <= 0 or kv_heads <= 0 or kv_heads > num_heads or qkv.shape[2] % total:
            return False
        return qkv.shape[2] // total in ROPE_HEAD_DIMS
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

    if not can_use_sm100_qk_norm_rope(qkv, num_heads, num_kv_heads):
        raise RuntimeError("sm100 qk norm + rotation is ineligible for the requested inputs")
    kv_heads = num_heads if num_kv_heads is None else num_kv_heads
    head_dim = qkv.shape[2] // (num_heads + 2 * kv_heads)
    check_norm_weights(q_weight, k_weight, head_dim, qkv.device)
    check_rope(rope, head_dim, qkv.device)
    if positions is not None:
        require(
            positions.dtype in (torch.int32, torch.int64) and positions.device == qkv.device
            and tuple(positions.shape) in ((qkv.shape[0], qkv.shape[1]), (qkv.shape[1],))
            and positions.stride(-1) == 1,
            "positions must be an int32 or int64 [B, T] or [T] tensor on the input's device",
        )
    result = torch.empty(qkv.shape, dtype=qkv.dtype, device=qkv.device) if out is None else out
    if out is not None:
        require(
            out.shape == qkv.shape and out.dtype == qkv.dtype and out.device == qkv.device and packed_ok(out)
            and (out.data_ptr() != qkv.data_ptr() or out.stride() == qkv.stride()),
            "out must have qkv's shape, dtype and device, 16-byte aligned heads, and qkv's strides when it is qkv",
        )
    launch(
        _native.qk_norm_rope, qkv, result, num_heads, kv_heads, head_dim, q_weight, k_weight, float(eps),
        None if rope is None else rope.reference, positions,
    )
    return result, SM100_QK_NORM_ROPE_BACKEND


__all__ = [
    "ROPE_HEAD_DIMS",
    "RotaryTable",
    "SM100_QK_NORM_ROPE_BACKEND",
    "can_use_sm100_qk_norm_rope",
    "check_norm_weights",
    "check_rope",
    "packed_ok",
    "sm100_qk_norm_rope",
]
