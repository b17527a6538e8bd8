"""Token-by-token runs of the model over an 8-bit key/value cache.

The reference computes whole sequences (solution/transformer.py:1346-1513);
``CachedDecoder`` goes on from a prompt: ``prompt(x)`` is the forward with the
keys and values kept, ``step(x)`` one or a few tokens of each sequence against
what is kept.  A step's time is the bytes that it reads, so its projections
have 4-bit weights (``weights="w4"``, packed once from the model's) and its
cache 8-bit codes; the prompt runs the bf16 kernels.

    decoder = CachedDecoder(model, slots=8, max_tokens=4096)
    y = decoder.prompt(x)            # [8, T, D], every slot at once
    for _ in range(n):
        y = decoder.step(next_x)     # [8, 1, D]

The model has neither a position rotation nor norms of queries and keys (its
positions come with its inputs); ``rope`` and ``qk_norms`` put them in for
models that do.

The slots may be many requests': each has a low-rank adapter of its own
(``adapters``, ``set_adapters``), takes over another's sequence (``fork``: samples, beams), and keeps as
many of its drafted tokens as are verified (``accept``):

    y = decoder.step(drafts, advance=False)       # [8, 1 + n, D]: the last token and n drafted ones
    tokens, accepted = decoder.accept(probabilities(y), drafted, uniform)

They begin together, with ``prompt``, which takes all slots.  A slot whose request has ended takes another one
in steps of up to 64 tokens that count for it alone (the other slots' rows are anything, and need room to be appended):

    decoder.fork([0, -1, 2, ...])                 # slot 1 is empty
    y = decoder.step(x, advance=False)            # [8, 64, D], its tokens in x[1]
    decoder.advance(counts)                       # int32 [8]: 64 for slot 1, 0 for the others
"""

from __future__ import annotations

from collections.abc import Sequence
from typing import Any

import torch

from ..kernels import (
    Kv8Cache,
    Kv8Pages,
    LowRankAdapters,
    RotaryTable,
    W4Weight,
    pack_w4,
    sm100_flash_attention,
    sm100_initial_layer_norm,
    sm100_kv8_append,
    sm100_kv8_attention,
    sm100_kv8_fork,
    sm100_kv8_reserve,
    sm100_linear,
    sm100_linear_w4,
    sm100_low_rank_add,
    sm100_mma_attention,
    sm100_qk_norm_rope,
    sm100_residual_layer_norm,
    sm100_simt_attention,
    sm100_verify_draft,
)
from ..kernels.kv_cache import KV8_HEAD_DIMS
from ..kernels.kv_pages import KV8_POOL_ROWS
from .cuda_graph import CudaGraphReplay

# Rows of a step up to which its projections go through the 4-bit kernel, which reads the weights
# again for each 16 or 32 rows; above, through the bf16 GEMM with the values that the packed
# weights stand for.  The four layers of 1024 (FFN 4096) at 64 rows: 24 us against 37, at 128 38 against 47, at 256
# 70 against 48; 4096 -> 14336 at 32 rows 28 against 29, at 64 48 against 28.
_W4_ROWS = 64
_REPEATABLE = 64  # tokens that can be appended twice over and leave what once leaves


class CachedDecoder:
    """Prompt and steps of a ``UserOptimizedTransformer`` over a cache of ``slots``
    sequences of up to ``max_tokens`` tokens.  The slots go together: all hold
    the same number of tokens, unless a step's are counted for each slot
    (``accept``, ``advance`` with a tensor).

    * ``weights``: ``"w4"`` packs the projections to 4 bits for the steps (groups
      of ``group``; a step of more than 64 rows takes the same values rounded to
      bf16, which the first such step lays out), ``"bf16"`` runs the steps with the
      model's own, as the prompt always does
    * ``rope``: a ``RotaryTable``; ``qk_norms``: per layer ``(q_weight, k_weight)``,
      fp32 ``[head_dim]`` each
    * ``adapters``: per layer, low-rank adapters of its projections by name (``"qkv"``,
      ``"out"``, ``"ffn_in"``, ``"ffn_out"``; any of them), which ``set_adapters`` gives to the slots
    * ``graph``: replay a step of up to 64 tokens from a CUDA graph, captured once for
      each shape and dtype; ``x`` is copied into the buffer that the graph reads
      (``solution.runtimes.CudaGraphReplay``)

    The model's weights are read when the decoder is made: make a new one
    after loading others.
    """

    def __init__(
        self,
        model: Any,
        *,
        slots: int,
        max_tokens: int,
        weights: str = "w4",
        group: int = 64,
        rope: RotaryTable | None = None,
        qk_norms: list[tuple[torch.Tensor, torch.Tensor]] | None = None,
        qk_norm_eps: float = 1e-6,
        adapters: Sequence[dict[str, LowRankAdapters]] | None = None,
        graph: bool = True,
    ) -> None:
        config = model.config
        self.head_dim = config.d_model // config.num_heads
        if not config.causal:
            raise ValueError("a cache needs a causal model")
        if self.head_dim not in KV8_HEAD_DIMS:
            raise ValueError(f"head_dim {self.head_dim} is not one of {KV8_HEAD_DIMS}")
        if weights not in ("w4", "bf16"):
            raise ValueError(f"weights must be 'w4' or 'bf16', not {weights!r}")
        if qk_norms is not None and len(qk_norms) != config.num_layers:
            raise ValueError("qk_norms must hold one pair of weights per layer")
        if slots < 1 or max_tokens < 1:
            raise ValueError("slots and max_tokens must be positive")
        if adapters is not None:
            if len(adapters) != config.num_layers:
                raise ValueError("adapters must hold one dict per layer")
            for given, layer in zip(adapters, model.layers):
                linears = dict(self._linears(layer))
                for name, adapter in given.items():
                    if name not in linears:
                        raise ValueError(f"adapters are of {tuple(linears)}, not of {name!r}")
                    weight = linears[name].weight
                    if (adapter.out_features, adapter.in_features) != tuple(weight.shape) or adapter.device != weight.device:
                        raise ValueError(f"the adapters of {name!r} do not fit its weight {tuple(weight.shape)} on {weight.device}")
        device = next(model.parameters()).device
        if device.type != "cuda":
            raise RuntimeError("CachedDecoder needs a model on an sm_100 CUDA device; there is no CPU fallback")
        self.model = model
        self.heads = config.num_heads
        self.slots = slots
        self.max_tokens = max_tokens
        self.held = 0  # tokens of each slot, as far as this decoder has counted them; where slots differ, no less than the most
        self.pending = 0  # of those appended last, the ones that may still be counted
        self.rope = rope
        self.qk_norms = qk_norms or [(None, None)] * config.num_layers
        self.qk_norm_eps = float(qk_norm_eps)
        self.graph = bool(graph)
        self.adapters = None if adapters is None else [dict(given) for given in adapters]
        self._differ = False  # whether the slots' tokens have been counted apart
        self._pages: Kv8Pages | None = None  # made by the first fork, or once the cache's pages are a pool by other means
        with torch.inference_mode():
            self.adapter_indices = torch.full((slots,), -1, dtype=torch.int32, device=device)
            model._materialize_shadow_weights()
            self.cache = Kv8Cache.create(
                slots=slots, max_tokens=max_tokens, num_kv_heads=self.heads, head_dim=self.head_dim,
                layers=max(1, config.num_layers), device=device,
            )
            self.step_weights: list[dict[str, W4Weight]] | None = None
            if weights == "w4":
                self.step_weights = [
                    {name: pack_w4(linear.weight, group) for name, linear in self._linears(layer)}
                    for layer in model.layers
                ]
        # what all graphs share, as steps follow one another: memory, and the stream of their captures
        self._capture: tuple[object, torch.cuda.Stream] | None = None
        self._wide_weights: list[dict[str, torch.Tensor]] | None = None  # the packed ones' values in bf16
        self._replays: dict[tuple[object, ...], tuple[torch.Tensor, CudaGraphReplay]] = {}

    @staticmethod
    def _linears(layer: Any) -> tuple[tuple[str, Any], ...]:
        return (
            ("qkv", layer.attention.qkv_proj),
            ("out", layer.attention.out_proj),
            ("ffn_in", layer.ffn_in),
            ("ffn_out", layer.ffn_out),
        )

    # ------------------------------------------------------------ program
    def _program(
        self,
        value: torch.Tensor,
        mask: torch.Tensor | None = None,  # noqa: ARG002 - the graph runtime's program signature
        *,
        out: torch.Tensor | None = None,
        defer_final: bool = False,
        prompt: bool = False,
    ) -> Any:
        """The forward of ``[B, T, D]`` inputs at their sequences' ends; with
        ``defer_final`` the last LayerNorm is handed back as ``finish(out)``."""

        layers = self.model.layers
        final = self.model.final_norm
        batch, tokens, d_model = value.shape
        rows = batch * tokens
        flat = value.reshape(rows, d_model)
        packed = None if prompt else self.step_weights

        def linear(index: int, name: str, module: Any, x: torch.Tensor, *, gelu: bool = False) -> torch.Tensor:
            weight, bias = module.shadow_parameters()
            own = None if self.adapters is None else self.adapters[index].get(name)
            # with adapters the projection stays in 32 bits until theirs are added, and the GELU comes after that
            form = {"gelu": gelu} if own is None else {"out_dtype": torch.float32}
            if packed is not None and rows <= _W4_ROWS:
                y = sm100_linear_w4(x, packed[index][name], bias, **form)[0]
            else:
                if packed is not None:
                    weight = self._wide_weights[index][name]
                y = sm100_linear(x, weight, bias, **form)[0]
            if own is None:
                return y
            return sm100_low_rank_add(x, y, own, self.adapter_indices, gelu=gelu, out_dtype=torch.bfloat16)[0]

        normalized, _ = sm100_initial_layer_norm(flat, (layers[0].norm1 if len(layers) else final).kernel_norm())
        residual = torch.empty((rows, d_model), dtype=torch.float32, device=value.device)
        source = flat
        update = None
        for index, layer in enumerate(layers):
            linears = dict(self._linears(layer))
            q_weight, k_weight = self.qk_norms[index]
            qkv = linear(index, "qkv", linears["qkv"], normalized).view(batch, tokens, 3 * d_model)
            if prompt:
                # The prompt attends to its own bf16 keys; the cache keeps them for the steps.
                if self.rope is not None or q_weight is not None or k_weight is not None:
                    sm100_qk_norm_rope(
                        qkv, self.heads, q_weight=q_weight, k_weight=k_weight, eps=self.qk_norm_eps, rope=self.rope,
                        out=qkv,
                    )
                sm100_kv8_append(self.cache, qkv, self.heads, layer=index)
                attend = (
                    sm100_flash_attention
                    if self.head_dim == 64
                    else sm100_simt_attention
                    if self.head_dim == 256
                    else sm100_mma_attention
                )
                context, _ = attend(qkv, self.heads, causal=True)
            else:
                q, _ = sm100_kv8_append(
                    self.cache, qkv, self.heads, layer=index, q_weight=q_weight, k_weight=k_weight,
                    eps=self.qk_norm_eps, rope=self.rope,
                )
                context, _ = sm100_kv8_attention(self.cache, q, layer=index)
            update = linear(index, "out", linears["out"], context.view(rows, d_model))
            sm100_residual_layer_norm(
                source, update, layer.norm2.kernel_norm(), final_boundary=False, residual_out=residual,
                normalized_out=normalized,
            )
            source = residual
            hidden = linear(index, "ffn_in", linears["ffn_in"], normalized, gelu=True)
            update = linear(index, "ffn_out", linears["ffn_out"], hidden)
            if index + 1 < len(layers):
                sm100_residual_layer_norm(
                    residual, update, layers[index + 1].norm1.kernel_norm(), final_boundary=False,
                    residual_out=residual, normalized_out=normalized,
                )

        def finish(target: torch.Tensor) -> torch.Tensor:
            rows_out = target.view(rows, d_model)
            if update is None:
                sm100_initial_layer_norm(flat, final.kernel_norm(), out_dtype=target.dtype, normalized_out=rows_out)
            else:
                sm100_residual_layer_norm(
                    residual, update, final.kernel_norm(), final_boundary=True, out_dtype=target.dtype,
                    keep_residual=False, normalized_out=rows_out,
                )
            return target

        if defer_final:
            return finish
        return finish(torch.empty_like(value, memory_format=torch.contiguous_format) if out is None else out)

    def _check(self, x: torch.Tensor, held: int) -> None:
        d_model = self.model.config.d_model
        if x.ndim != 3 or x.shape[0] != self.slots or x.shape[1] < 1 or x.shape[2] != d_model:
            raise ValueError(f"x must be [{self.slots}, tokens, {d_model}], not {tuple(x.shape)}")
        if x.device != self.cache.device or not x.is_contiguous():
            raise ValueError("x must be a contiguous tensor on the decoder's device")
        if x.dtype not in (torch.float32, torch.bfloat16):
            raise ValueError("x must be float32 or bfloat16")
        if held and held + x.shape[1] > self.max_tokens and (self._differ or self.cache._pool is not None):
            self.held = held = int(self.cache.lengths.max())  # what the slots really hold: read from the device
        if held + x.shape[1] > self.max_tokens:
            raise ValueError(f"{held} tokens held and {x.shape[1]} more pass the cache's {self.max_tokens}")

    # ------------------------------------------------------------ calls
    def reset(self) -> None:
        """Forget every sequence."""

        with torch.inference_mode():
            self.cache.lengths.zero_()
        self.held = self.pending = 0
        self._differ = False

    def advance(self, tokens: int | torch.Tensor) -> None:
        """Count ``tokens`` of those that the last step appended as held, in every
        slot: any number of them up to 64, else all (a block that a longer call
        fills is only kept as codes, and cannot be open again).  An int32 tensor
        ``[slots]`` counts for each slot its own (of a step of up to 64 tokens; numbers outside
        are taken as none or all); the rest is forgotten."""

        if isinstance(tokens, torch.Tensor):
            if tokens.dtype != torch.int32 or tuple(tokens.shape) != (self.slots,) or tokens.device != self.cache.device:
                raise ValueError(f"tokens must be a number or an int32 [{self.slots}] tensor on the decoder's device")
            if self.pending > _REPEATABLE:
                raise ValueError(f"a step of {self.pending} tokens, more than {_REPEATABLE}, is counted whole")
            with torch.inference_mode():
                self.cache.advance(tokens.clamp(0, self.pending))
            self.held += self.pending
            self.pending = 0
            self._differ = True
            return
        if not 0 <= tokens <= self.pending:
            raise ValueError(f"{tokens} tokens cannot be counted: {self.pending} are not counted yet")
        if tokens != self.pending > _REPEATABLE:
            raise ValueError(f"a step of {self.pending} tokens, more than {_REPEATABLE}, is counted whole")
        with torch.inference_mode():
            self.cache.advance(tokens)
        self.held += tokens
        self.pending -= tokens

    def accept(
        self,
        target: torch.Tensor,
        drafted: torch.Tensor,
        uniform: torch.Tensor,
        *,
        draft: torch.Tensor | None = None,
        counts: torch.Tensor | None = None,
    ) -> tuple[torch.Tensor, torch.Tensor]:
        """Verifies the ``T`` drafted tokens of the last step, ``step(x, advance=False)`` of each slot's last token
        and its drafted ones, and counts those that stand: ``target`` ``[slots, T + 1, V]`` are the probabilities that follow
        from the step's outputs, the rest as in ``solution.kernels.sm100_verify_draft``.  Returns its tokens
        and ``accepted``; each slot holds ``accepted + 1`` tokens more."""

        if drafted.ndim != 2 or drafted.shape[0] != self.slots or drafted.shape[1] + 1 != self.pending or self.pending > _REPEATABLE:
            raise ValueError(
                f"drafted must be [{self.slots}, T] where the last step had T + 1 tokens that are not counted yet, "
                f"{_REPEATABLE} at most; {self.pending} are not"
            )
        with torch.inference_mode():
            tokens, accepted, _ = sm100_verify_draft(target, drafted, uniform, draft=draft, counts=counts)
            self.advance(accepted + 1)
        return tokens, accepted

    def _whole(self, given: Sequence[int] | torch.Tensor, what: str) -> torch.Tensor:
        """A number of each slot, in 64 bits (those that only an unsigned type holds as the largest)."""

        numbers = torch.as_tensor(given)
        if (
            tuple(numbers.shape) != (self.slots,) or numbers.is_floating_point() or numbers.is_complex()
            or numbers.dtype == torch.bool
        ):
            raise ValueError(f"{what} must be {self.slots} whole numbers")
        wide = numbers.long()
        if numbers.dtype == torch.uint64:
            wide = torch.where(wide < 0, torch.iinfo(torch.int64).max, wide)
        return wide

    def set_adapters(self, indices: Sequence[int] | torch.Tensor) -> None:
        """The adapter of each slot from now on, -1: none (for graphs that are captured already, too).
        Numbers on the host are checked; one on the device past a projection's set makes its
        slot's outputs NaN."""

        if self.adapters is None:
            raise ValueError("the decoder was made without adapters")
        given = self._whole(indices, "indices")
        sizes = [own.count for layer in self.adapters for own in layer.values()]
        if given.device.type == "cpu" and sizes and int(given.max()) >= min(sizes):
            raise ValueError(f"adapter {int(given.max())} of {min(sizes)}")
        given = given.clamp(-1, 2**31 - 1)
        with torch.inference_mode():
            self.adapter_indices.copy_(given)

    def fork(self, parents: Sequence[int] | torch.Tensor) -> None:
        """Slot i goes on from slot ``parents[i]``'s sequence, for all slots at once, with its adapter: samples
        of one prompt, or beams in a new order.  Full blocks are shared and not copied.  A number
        below 0 empties the slot, one past the slots leaves it as it is.  Tokens that are not
        counted yet are forgotten."""

        given = self._whole(parents, "parents")
        if self.slots > KV8_POOL_ROWS:
            raise ValueError(f"at most {KV8_POOL_ROWS} slots can be forked")
        if self.pending > _REPEATABLE:
            raise ValueError(f"the last step's {self.pending} tokens cannot be taken back: advance({self.pending}) first")
        with torch.inference_mode():
            pages = self.pages
            source = given.clamp(-1, self.slots).to(device=self.cache.device, dtype=torch.int32).contiguous()
            each = torch.arange(self.slots, dtype=torch.int32, device=self.cache.device)
            sm100_kv8_fork(pages, source, each)
            inside = (source >= 0) & (source < self.slots)
            of = torch.where(inside, source, each).long()
            self.adapter_indices.copy_(torch.where(source < 0, -1, self.adapter_indices[of]))
        self.pending = 0
        self._differ = True

    @property
    def pages(self) -> Kv8Pages:
        """The cache's pages as one pool, to free, fork or compact by hand between steps (any other ``Kv8Pages`` of the
        cache does as well).  From then on the steps reserve the pages that they fill."""

        held = self.cache._pool
        if self._pages is None or held is None or self._pages.refs is not held[0]:
            with torch.inference_mode():
                self._pages = Kv8Pages(self.cache, None if held is None else held[0])
        return self._pages

    def _reserve(self, tokens: int) -> None:
        # There are as many pages as entries of the table, so that none is ever missing.
        if self.cache._pool is None:
            return
        if self.slots <= KV8_POOL_ROWS:
            sm100_kv8_reserve(self.pages, tokens)
            return
        for some in torch.arange(self.slots, dtype=torch.int32, device=self.cache.device).split(KV8_POOL_ROWS):
            sm100_kv8_reserve(self.pages, tokens, slots=some)

    def prompt(self, x: torch.Tensor) -> torch.Tensor:
        """The forward of ``x`` ``[slots, T, D]`` from empty sequences, which it leaves
        in the cache (what the slots held before is forgotten)."""

        self._check(x, 0)
        self.reset()
        with torch.inference_mode():
            self._reserve(x.shape[1])
            y = self._program(x, prompt=True)
        self.pending = x.shape[1]
        self.advance(x.shape[1])
        return y

    def step(self, x: torch.Tensor, *, advance: bool = True) -> torch.Tensor:
        """The forward of the next tokens ``x`` ``[slots, T, D]``.  With
        ``advance=False`` the caller says afterwards how many of them count
        (``decoder.advance(n)``; for up to 64 tokens any number of them, none
        where the next step comes first).  A step of more than 64 tokens that
        fails on its way forgets every sequence."""

        self._check(x, self.held)
        if self.pending > _REPEATABLE:
            raise ValueError(f"the last step's {self.pending} tokens cannot be taken back: advance({self.pending}) first")
        with torch.inference_mode():
            if self.step_weights is not None and self._wide_weights is None and self.slots * x.shape[1] > _W4_ROWS:
                self._wide_weights = [
                    {name: packed.dequantize(torch.bfloat16).contiguous() for name, packed in layer.items()}
                    for layer in self.step_weights
                ]
            self._reserve(x.shape[1])
            # A capture runs the step once before it records it, so that the
            # first call appends the same tokens twice.
            if self.graph and x.shape[1] <= _REPEATABLE:
                key = (tuple(x.shape), x.dtype)
                if key not in self._replays:
                    if self._capture is None:
                        self._capture = (torch.cuda.graph_pool_handle(), torch.cuda.Stream(self.cache.device))
                    pool, stream = self._capture
                    self._replays[key] = (torch.empty_like(x), CudaGraphReplay(pool=pool, stream=stream))
                buffer, replay = self._replays[key]
                y = replay.run(self._program, buffer.copy_(x), None)
            else:
                try:
                    y = self._program(x)
                except BaseException:
                    # the layers that it came to may hold some of it in place of older tokens
                    if x.shape[1] > _REPEATABLE:
                        self.reset()
                    raise
        self.pending = x.shape[1]
        if advance:
            self.advance(x.shape[1])
        return y


__all__ = ["CachedDecoder"]
