"""How many drafted tokens count (csrc/verify_kernels.cuh).

A step over drafted tokens (``CachedDecoder.step(x, advance=False)``, or appends
and attention over a ``Kv8Cache`` by hand) gives the target's probabilities for
all of them at once.  ``sm100_verify_draft`` says, from given random numbers, how
many count and which token follows, so that the tokens are distributed as the
target's own; ``cache.advance(accepted + 1)`` (``decoder.advance``) counts them.
"""

from __future__ import annotations

import torch

from ._common import binding, is_sm100_cuda, library_ready

SM100_VERIFY_DRAFT_BACKEND = "sm100_verify_draft"
VERIFY_MOST = 1024  # drafted tokens of a sequence


def can_use_sm100_verify_draft(target: torch.Tensor, drafted: torch.Tensor) -> bool:
    """Whether the kernel can run on these inputs (never raises)."""

    try:
        return library_ready() and is_sm100_cuda(target) and binding().verify_draft_ok(target, drafted)
    except Exception:  # noqa: BLE001 - predicate contract: never raise
        return False


def sm100_verify_draft(
    target: torch.Tensor,
    drafted: torch.Tensor,
    uniform: torch.Tensor,
    *,
    draft: torch.Tensor | None = None,
    counts: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor, str]:
    """Verifies ``drafted`` ``[B, T]`` (int32 or int64, T up to 1024) against the target's probabilities
    ``target`` ``[B, T + 1, V]`` (float32 or bf16) with ``uniform`` float32 ``[B, T + 1]`` in [0, 1).

    Token t counts while ``uniform[t] * draft[t, d] < target[t, d]``; ``draft`` ``[B, T, V]`` are the
    probabilities that the tokens were drawn with (None: 1, as for tokens that were looked up).  The
    token after the last that counts is drawn from ``max(target - draft, 0)`` at the
    first refusal (from the target's row where that leaves nothing), else from the target's last row: the first index whose running sum passes
    ``uniform[T]`` times the whole.  Sequence b has ``counts[b]`` drafted tokens (default T).

    Returns ``tokens`` ``[B, T + 1]`` in ``drafted``'s dtype (those that count, the one after
    them, then -1) and ``accepted`` int32 ``[B]``.  Probabilities need not sum to 1 (a mass that is
    NaN or negative is none; without any mass the token after is -1); a drafted token outside the vocabulary is refused."""

    tokens, accepted = binding().verify_draft(target, drafted, uniform, draft, counts)
    return tokens, accepted, SM100_VERIFY_DRAFT_BACKEND


__all__ = [
    "SM100_VERIFY_DRAFT_BACKEND",
    "VERIFY_MOST",
    "can_use_sm100_verify_draft",
    "sm100_verify_draft",
]
