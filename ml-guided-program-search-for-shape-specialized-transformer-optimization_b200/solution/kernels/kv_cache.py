"""A paged key/value cache in 8 bits and the attention that reads it
(csrc/kv8_cache_kernels.cuh, csrc/kv8_attention_kernels.cuh).

The reference runs whole sequences only (no cache).  Tokens lie in blocks of
64; a full block is held as 8-bit codes with one scale per kv head for keys and
one for values, the open block in bf16, so nothing is quantised twice and a
prompt appended at once leaves the same bits as its tokens one by one.

A step of a model, for each layer: ``sm100_kv8_append`` (norm, rotation, store)
and ``sm100_kv8_attention``; after the last layer ``cache.advance(n)``.
"""

from __future__ import annotations

import ctypes

import torch

from .. import _native
from ._common import TensorHandle, binding, is_sm100_cuda, library_ready, require
from .rotary import RotaryTable

SM100_KV8_APPEND_BACKEND = "sm100_kv8_append"
SM100_KV8_GATHER_BACKEND = "sm100_kv8_gather"
SM100_KV8_ATTENTION_BACKEND = "sm100_kv8_attention"
KV8_BLOCK = _native.KV8_BLOCK
KV8_HEAD_DIMS = (32, 64, 128, 256)
_MOST_STREAMS = 8  # that a cache holds a workspace for; each is 2 to 5 MB


class Kv8Cache(TensorHandle):
    """The tensors of a cache, shared by the layers of a model.

    * ``codes`` uint8 ``[layers, pages, 2, Hkv, 64, D]`` (keys, values): a full
      block of a sequence is one page; a value is ``(code - 128) * scale``
    * ``scales`` float32 ``[layers, pages, 2, Hkv]``
    * ``tail`` bf16 ``[layers, slots, 2, 2, Hkv, 64, D]``: the open blocks, by block parity
    * ``page_table`` int32 ``[slots, max_blocks]``: the page of each block
    * ``lengths`` int32 ``[slots]``: tokens held, before the step at hand

    ``codes``, ``scales`` and ``tail`` may leave out the layers.  The caller
    fills ``page_table`` (``create`` gives each slot pages of its own) and may
    change it and ``lengths`` in place between steps; the kernels check both, store
    nothing out of range and read NaN from there.
    """

    def __init__(
        self,
        codes: torch.Tensor,
        scales: torch.Tensor,
        tail: torch.Tensor,
        page_table: torch.Tensor,
        lengths: torch.Tensor,
    ) -> None:
        if codes.ndim == 5:
            codes, scales, tail = codes[None], scales[None], tail[None]
        require(
            codes.ndim == 6 and codes.dtype == torch.uint8 and codes.shape[2] == 2 and codes.shape[4] == KV8_BLOCK,
            "codes must be a uint8 [layers, pages, 2, kv_heads, 64, head_dim] tensor",
        )
        layers, pages, _, kv_heads, _, dim = codes.shape
        require(dim in KV8_HEAD_DIMS, f"head_dim {dim} is not one of {KV8_HEAD_DIMS}")
        require(
            scales.dtype == torch.float32 and tuple(scales.shape) == (layers, pages, 2, kv_heads),
            "scales must be a float32 [layers, pages, 2, kv_heads] tensor",
        )
        require(
            page_table.dtype == torch.int32 and page_table.ndim == 2
            and lengths.dtype == torch.int32 and tuple(lengths.shape) == (page_table.shape[0],),
            "page_table must be int32 [slots, max_blocks] and lengths int32 [slots]",
        )
        slots, max_blocks = page_table.shape
        require(
            tail.dtype == torch.bfloat16 and tuple(tail.shape) == (layers, slots, 2, 2, kv_heads, KV8_BLOCK, dim),
            "tail must be a bfloat16 [layers, slots, 2, 2, kv_heads, 64, head_dim] tensor",
        )
        require(min(layers, pages, kv_heads, slots, max_blocks) > 0, "the cache must not be empty")
        tensors = (codes, scales, tail, page_table, lengths)
        require(
            all(t.is_contiguous() and t.device == codes.device for t in tensors)
            and codes.data_ptr() % 16 == 0 and tail.data_ptr() % 16 == 0,
            "the cache's tensors must be contiguous on one device, codes and tail 16-byte aligned",
        )
        self.codes, self.scales, self.tail, self.page_table, self.lengths = tensors
        self.layers, self.pages, self.kv_heads, self.head_dim = layers, pages, kv_heads, dim
        self.slots, self.max_blocks = slots, max_blocks
        self.device = codes.device
        self._views = [
            _native.Kv8CacheView(
                codes[i].data_ptr(), scales[i].data_ptr(), tail[i].data_ptr(), page_table.data_ptr(),
                lengths.data_ptr(), pages, slots, max_blocks, kv_heads, dim,
            )
            for i in range(layers)
        ]
        # what the binding takes for a layer: the struct's address and the device
        self._handles = [(ctypes.addressof(view), codes.get_device()) for view in self._views]
        # The attention's workspace (arrival counters that every launch leaves
        # zero, and the parts of split tiles): one for each stream it runs on,
        # and one for each capture, whose graph may be replayed on any stream
        # beside calls on the one that it was captured on.  All are made when
        # they are first asked for; None: the stream has been captured on only.
        self._workspaces: dict[int, torch.Tensor | None] = {}
        self._captured: dict[int, tuple[int, torch.Tensor]] = {}  # stream: capture, workspace; of the last capture
        # Counts and scratch of the pool that the pages are (Kv8Pages); None: nothing but the table says whose they are.
        self._pool: tuple[torch.Tensor, torch.Tensor] | None = None

    @classmethod
    def create(
        cls,
        *,
        slots: int,
        max_tokens: int,
        num_kv_heads: int,
        head_dim: int,
        layers: int = 1,
        pages: int | None = None,
        device: torch.device | str = "cuda",
    ) -> Kv8Cache:
        """An empty cache of ``slots`` sequences of up to ``max_tokens`` tokens: each slot with
        pages of its own, or, with ``pages``, that many pages that no slot holds yet (``Kv8Pages``)."""

        blocks = -(-max_tokens // KV8_BLOCK)
        own = pages is None
        if own:
            pages = slots * blocks
        return cls(
            torch.zeros((layers, pages, 2, num_kv_heads, KV8_BLOCK, head_dim), dtype=torch.uint8, device=device),
            torch.zeros((layers, pages, 2, num_kv_heads), dtype=torch.float32, device=device),
            torch.zeros((layers, slots, 2, 2, num_kv_heads, KV8_BLOCK, head_dim), dtype=torch.bfloat16, device=device),
            torch.arange(pages, dtype=torch.int32, device=device).reshape(slots, blocks)
            if own
            else torch.full((slots, blocks), -1, dtype=torch.int32, device=device),
            torch.zeros(slots, dtype=torch.int32, device=device),
        )

    @property
    def bytes_per_token(self) -> float:
        """Bytes of a full block's token, all layers (codes and scales)."""

        return 2 * self.layers * self.kv_heads * (self.head_dim + 4 / KV8_BLOCK)

    def handle(self, layer: int) -> tuple[int, int]:
        require(0 <= layer < self.layers, f"layer {layer} of a cache of {self.layers}")
        return self._handles[layer]

    def reference(self, layer: int) -> object:
        """The layer's b200tx_kv8_cache, as ctypes passes it."""

        require(0 <= layer < self.layers, f"layer {layer} of a cache of {self.layers}")
        return ctypes.byref(self._views[layer])

    def _new_workspace(self) -> torch.Tensor:
        with torch.cuda.device(self.device):
            made = torch.empty(_native.kv8_workspace_bytes(self.head_dim), dtype=torch.uint8, device=self.device)
            made[: _native.KV8_COUNTER_BYTES].zero_()
        return made

    def workspace(self, stream: int, capture: int | None = None) -> torch.Tensor:
        """What the calls on ``stream`` share, or those of the capture with the
        id ``capture`` on it.  The latter lies in the graph's own memory, and
        its counters are cleared by every replay."""

        if capture is None:
            found = self._workspaces.get(stream)
            if found is None:
                # The oldest goes: it was allocated on the stream that it served, so that
                # the allocator gives its memory out after that stream's launches.
                while len(self._workspaces) >= _MOST_STREAMS:
                    del self._workspaces[next(iter(self._workspaces))]
                found = self._workspaces[stream] = self._new_workspace()
            return found
        if stream not in self._workspaces:
            # a call on the stream comes before its captures; one stream may do without
            if any(held is None for held in self._workspaces.values()):
                raise RuntimeError(
                    "the cache's attention is captured on a second stream that it has not run on: "
                    "call it once on that stream before the capture"
                )
            self._workspaces[stream] = None
        if stream not in self._captured or self._captured[stream][0] != capture:
            self._captured = {s: held for s, held in self._captured.items() if held[0] == capture}
            self._captured[stream] = (capture, self._new_workspace())
        return self._captured[stream][1]

    def advance(self, tokens: int | torch.Tensor, slots: torch.Tensor | None = None) -> None:
        """Count the appended tokens as held (all slots, or ``slots``; as in the
        kernels, a row whose slot is none counts nowhere)."""

        if slots is None:
            self.lengths.add_(tokens)
            return
        inside = slots.clamp(0, self.slots - 1)
        self.lengths.index_add_(0, inside, (inside == slots).to(torch.int32).mul_(tokens))


def can_use_sm100_kv8_append(cache: Kv8Cache, qkv: torch.Tensor, num_heads: int) -> bool:
    """Whether the kernel can append this packed projection (never raises)."""

    try:
        return library_ready() and is_sm100_cuda(qkv) and binding().kv8_append_ok(cache.handle(0), qkv, num_heads)
    except Exception:  # noqa: BLE001 - predicate contract: never raise
        return False


def sm100_kv8_append(
    cache: Kv8Cache,
    qkv: torch.Tensor,
    num_heads: int,
    *,
    layer: int = 0,
    q_weight: torch.Tensor | None = None,
    k_weight: torch.Tensor | None = None,
    eps: float = 1e-6,
    rope: RotaryTable | None = None,
    slots: torch.Tensor | None = None,
    counts: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
) -> tuple[torch.Tensor, str]:
    """Append the keys and values of ``qkv`` ``[B, T, (H + 2 Hkv) * D]`` (float32
    or bf16) to the cache at their sequences' ends, keys normed and rotated on
    the way as ``sm100_qk_norm_rope`` does with position ``lengths + t``; returns
    the queries, normed and rotated, bf16 ``[B, T, H, D]``.

    Row b is slot ``slots[b]`` (default b; a slot once at most) and has ``counts[b]``
    tokens (default T).  ``lengths`` stays as it is until ``cache.advance``: by all the tokens,
    or, for ``T <= 64``, by any number of them (the rest is forgotten)."""

    result = binding().kv8_append(
        cache.handle(layer), qkv, num_heads, q_weight, k_weight, eps, None if rope is None else rope.handle, slots,
        counts, out,
    )
    return result, SM100_KV8_APPEND_BACKEND


def sm100_kv8_gather(
    cache: Kv8Cache,
    max_tokens: int,
    *,
    layer: int = 0,
    batch: int | None = None,
    tokens: int = 0,
    slots: torch.Tensor | None = None,
    counts: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor, str]:
    """The cached keys and values as numbers: two bf16 ``[B, max_tokens, Hkv, D]``
    tensors, zero past each sequence's end.  ``tokens`` (or ``counts``) more than
    ``lengths`` are read: those appended since the last ``advance``."""

    rows = batch if batch is not None else cache.slots if slots is None else slots.shape[0]
    k, v = binding().kv8_gather(cache.handle(layer), cache.codes, rows, max_tokens, tokens, slots, counts)
    return k, v, SM100_KV8_GATHER_BACKEND


def can_use_sm100_kv8_attention(cache: Kv8Cache, q: torch.Tensor) -> bool:
    """Whether the kernel can attend with these queries (never raises)."""

    try:
        return library_ready() and is_sm100_cuda(q) and binding().kv8_attention_ok(cache.handle(0), q)
    except Exception:  # noqa: BLE001 - predicate contract: never raise
        return False


def sm100_kv8_attention(
    cache: Kv8Cache,
    q: torch.Tensor,
    *,
    layer: int = 0,
    scale: float | None = None,
    slots: torch.Tensor | None = None,
    counts: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
) -> tuple[torch.Tensor, str]:
    """``softmax(scale q k^T) v`` of the ``T`` tokens appended last over their
    sequences' keys, causal: ``q`` bf16 ``[B, T, H, D]`` at positions ``lengths + t``.
    Returns the context, bf16 ``[B, T, H * D]``; rows past ``counts[b]`` are zero.
    ``H / Hkv`` query heads share a kv head; ``scale`` defaults to ``D ** -0.5``.
    ``out`` may be a dense ``q``'s own memory."""

    result = binding().kv8_attention(
        cache.handle(layer), q, scale, slots, counts, out, cache._workspaces, cache.workspace
    )
    return result, SM100_KV8_ATTENTION_BACKEND


__all__ = [
    "KV8_BLOCK",
    "KV8_HEAD_DIMS",
    "Kv8Cache",
    "SM100_KV8_APPEND_BACKEND",
    "SM100_KV8_ATTENTION_BACKEND",
    "SM100_KV8_GATHER_BACKEND",
    "can_use_sm100_kv8_append",
    "can_use_sm100_kv8_attention",
    "sm100_kv8_append",
    "sm100_kv8_attention",
    "sm100_kv8_gather",
]
