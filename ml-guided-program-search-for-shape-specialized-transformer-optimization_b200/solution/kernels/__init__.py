"""Python wrappers over the libb200tx C ABI.

Each wrapper keeps the reference's operator conventions
(solution/shape14/triton_streaming_dh64.py:268-346,
solution/kernels/norm/triton_mixed_residual.py:80-160): ``*_available()``
reports whether the kernel library loads, ``can_use_*`` returns a bool and
never raises, and the op itself returns ``(tensor(s)..., marker)`` where the
marker names the kernel that ran.  Caller-contract violations raise
``ValueError``; ineligible inputs or a failed launch raise ``RuntimeError``.
There is no fallback path.
"""

from .attention import (
    SM100_FLASH_ATTENTION_BACKEND,
    SM100_MMA_ATTENTION_BACKEND,
    can_use_sm100_mma_attention,
    sm100_mma_attention,
    SM100_SIMT_ATTENTION_BACKEND,
    can_use_sm100_simt_attention,
    sm100_simt_attention,
    can_use_sm100_flash_attention,
    sm100_flash_attention,
    sm100_flash_attention_available,
)
from .boundary import (
    SM100_LINEAR_RESIDUAL_NORM_BACKEND,
    SM100_MLP_RESIDUAL_NORM_BACKEND,
    can_use_sm100_linear_residual_norm,
    can_use_sm100_mlp_residual_norm,
    sm100_linear_residual_norm,
    sm100_mlp_residual_norm,
)
from .kv_cache import (
    KV8_BLOCK,
    SM100_KV8_APPEND_BACKEND,
    SM100_KV8_ATTENTION_BACKEND,
    SM100_KV8_GATHER_BACKEND,
    Kv8Cache,
    can_use_sm100_kv8_append,
    can_use_sm100_kv8_attention,
    sm100_kv8_append,
    sm100_kv8_attention,
    sm100_kv8_gather,
)
from .kv_pages import (
    KV8_POOL_ROWS,
    SM100_KV8_COMPACT_BACKEND,
    SM100_KV8_FORK_BACKEND,
    SM100_KV8_RESERVE_BACKEND,
    Kv8Pages,
    sm100_kv8_compact,
    sm100_kv8_fork,
    sm100_kv8_free,
    sm100_kv8_reserve,
)
from .linear_w4 import (
    SM100_LINEAR_W4_BACKEND,
    SM100_LINEAR_W4_GELU_BACKEND,
    W4Weight,
    can_use_sm100_linear_w4,
    pack_w4,
    sm100_linear_w4,
)
from .low_rank import (
    SM100_LOW_RANK_ADD_BACKEND,
    SM100_LOW_RANK_ADD_GELU_BACKEND,
    LowRankAdapters,
    can_use_sm100_low_rank_add,
    sm100_low_rank_add,
)
from .norm import (
    MASK_DROP_UPDATE,
    MASK_ZERO_NORMED,
    MASK_ZERO_RESIDUAL,
    SM100_INITIAL_LAYER_NORM_BACKEND,
    SM100_RESIDUAL_LAYER_NORM_BACKEND,
    can_use_sm100_residual_layer_norm,
    sm100_initial_layer_norm,
    sm100_layer_norm_available,
    sm100_residual_layer_norm,
)
from .projection import (
    SM100_LINEAR_BACKEND,
    SM100_LINEAR_GELU_BACKEND,
    can_use_sm100_linear,
    sm100_linear,
    sm100_linear_available,
)
from .rotary import (
    SM100_QK_NORM_ROPE_BACKEND,
    RotaryTable,
    can_use_sm100_qk_norm_rope,
    sm100_qk_norm_rope,
)
from .verify import (
    SM100_VERIFY_DRAFT_BACKEND,
    can_use_sm100_verify_draft,
    sm100_verify_draft,
)
from . import ops  # noqa: E402 - registers the torch.ops.b200tx.* operators

__all__ = [
    "KV8_POOL_ROWS",
    "Kv8Pages",
    "LowRankAdapters",
    "SM100_KV8_COMPACT_BACKEND",
    "SM100_KV8_FORK_BACKEND",
    "SM100_KV8_RESERVE_BACKEND",
    "SM100_LOW_RANK_ADD_BACKEND",
    "SM100_LOW_RANK_ADD_GELU_BACKEND",
    "SM100_VERIFY_DRAFT_BACKEND",
    "can_use_sm100_low_rank_add",
    "can_use_sm100_verify_draft",
    "sm100_kv8_compact",
    "sm100_kv8_fork",
    "sm100_kv8_free",
    "sm100_kv8_reserve",
    "sm100_low_rank_add",
    "sm100_verify_draft",
    "KV8_BLOCK",
    "Kv8Cache",
    "RotaryTable",
    "SM100_KV8_APPEND_BACKEND",
    "SM100_KV8_ATTENTION_BACKEND",
    "SM100_KV8_GATHER_BACKEND",
    "SM100_LINEAR_W4_BACKEND",
    "SM100_LINEAR_W4_GELU_BACKEND",
    "SM100_QK_NORM_ROPE_BACKEND",
    "W4Weight",
    "can_use_sm100_kv8_append",
    "can_use_sm100_kv8_attention",
    "can_use_sm100_linear_w4",
    "can_use_sm100_qk_norm_rope",
    "pack_w4",
    "sm100_kv8_append",
    "sm100_kv8_attention",
    "sm100_kv8_gather",
    "sm100_linear_w4",
    "sm100_qk_norm_rope",
    "MASK_DROP_UPDATE",
    "MASK_ZERO_NORMED",
    "MASK_ZERO_RESIDUAL",
    "SM100_FLASH_ATTENTION_BACKEND",
    "SM100_MMA_ATTENTION_BACKEND",
    "can_use_sm100_mma_attention",
    "sm100_mma_attention",
    "SM100_SIMT_ATTENTION_BACKEND",
    "can_use_sm100_simt_attention",
    "sm100_simt_attention",
    "SM100_INITIAL_LAYER_NORM_BACKEND",
    "SM100_LINEAR_RESIDUAL_NORM_BACKEND",
    "SM100_MLP_RESIDUAL_NORM_BACKEND",
    "can_use_sm100_linear_residual_norm",
    "can_use_sm100_mlp_residual_norm",
    "sm100_linear_residual_norm",
    "sm100_mlp_residual_norm",
    "SM100_LINEAR_BACKEND",
    "SM100_LINEAR_GELU_BACKEND",
    "SM100_RESIDUAL_LAYER_NORM_BACKEND",
    "can_use_sm100_flash_attention",
    "can_use_sm100_linear",
    "can_use_sm100_residual_layer_norm",
    "sm100_flash_attention",
    "sm100_flash_attention_available",
    "sm100_initial_layer_norm",
    "sm100_layer_norm_available",
    "sm100_linear",
    "sm100_linear_available",
    "sm100_residual_layer_norm",
    "ops",
]
