"""``out=`` of the decoding operators: in place where a call allows it, beside the
input in a wider buffer, and refused where it shares memory with the input."""

from __future__ import annotations

import pytest
import torch

from solution.kernels import (
    Kv8Cache,
    RotaryTable,
    pack_w4,
    sm100_kv8_append,
    sm100_kv8_attention,
    sm100_linear_w4,
    sm100_qk_norm_rope,
)

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.fixture(autouse=True)
def _inference():
    with torch.inference_mode():
        yield
    torch.cuda.synchronize()


def _randn(*shape: int, seed: int = 1) -> torch.Tensor:
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV)


def test_linear_w4_out() -> None:
    weight = pack_w4(_randn(256, 256))
    store = _randn(12, 256).bfloat16()
    x = store[4:8]
    want, _ = sm100_linear_w4(x, weight)
    for out in (x, store[3:7], store[5:9]):
        with pytest.raises(ValueError, match="shares memory"):
            sm100_linear_w4(x, weight, out=out)
    for out in (store[:4], store[8:]):  # right before and right after
        assert sm100_linear_w4(x, weight, out=out)[0] is out and torch.equal(out, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_norm_rope_out(dtype) -> None:  # noqa: ANN001
    heads, dim, batch, tokens = 2, 64, 3, 7
    width = 3 * heads * dim
    table, weight = RotaryTable.create(64, dim, DEV), 1 + 0.1 * _randn(dim)

    def run(qkv: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
        return sm100_qk_norm_rope(qkv, heads, q_weight=weight, rope=table, out=out)[0]

    wide = _randn(batch, tokens, 2 * width + 64, seed=2).to(dtype)
    left, right = wide[..., :width], wide[..., width + 64 :]
    want = run(left)
    assert torch.equal(run(left, right), want)  # columns beside one another
    flat = torch.empty(batch * tokens * width + 4096, dtype=dtype, device=DEV)
    for shift in (8, 64, width, 2 * width + 8):
        at = flat[: batch * tokens * width].view(batch, tokens, width).copy_(left)
        moved = flat[shift : shift + batch * tokens * width].view(batch, tokens, width)
        with pytest.raises(ValueError, match="shares memory"):
            run(at, moved)
        with pytest.raises(ValueError, match="shares memory"):
            run(moved, at)
    with pytest.raises(ValueError, match="shares memory"):
        run(left, wide[..., 64 : width + 64])  # columns of the same rows that overlap
    with pytest.raises(ValueError, match="shares memory"):
        run(left, torch.empty(1, tokens, width, dtype=dtype, device=DEV).expand(batch, tokens, width))
    same = left[:1].expand(batch, tokens, width)  # one input for every row of the batch: fine to read
    assert torch.equal(run(same), run(left[:1]).expand(batch, tokens, width))
    with pytest.raises(ValueError, match="shares memory"):
        run(same, same)
    flipped = torch.empty(tokens, batch, width, dtype=dtype, device=DEV).transpose(0, 1)
    assert torch.equal(run(left, flipped), want)
    assert torch.equal(run(left, left), want)  # in place, in a wider buffer


def test_append_and_attention_out() -> None:
    cache = Kv8Cache.create(slots=2, max_tokens=6000, num_kv_heads=2, head_dim=64, device=DEV)
    sm100_kv8_append(cache, _randn(2, 5000, 8 * 64).bfloat16(), 4)
    cache.advance(5000)
    qkv = _randn(2, 3, 8 * 64, seed=5).bfloat16()
    store = qkv.flatten()
    for shift in (0, 512, len(store) - 2 * 3 * 256):
        with pytest.raises(ValueError, match="shares memory"):
            sm100_kv8_append(cache, qkv, 4, out=store[shift : shift + 2 * 3 * 256].view(2, 3, 4, 64))
    q, _ = sm100_kv8_append(cache, qkv, 4)
    want, _ = sm100_kv8_attention(cache, q)
    room = torch.zeros(q.numel() + 256, dtype=torch.bfloat16, device=DEV)
    at = room[: q.numel()].view(q.shape).copy_(q)
    with pytest.raises(ValueError, match="shares memory"):
        sm100_kv8_attention(cache, at, out=room[256:].view(2, 3, 256))
    got, _ = sm100_kv8_attention(cache, at, out=at.view(2, 3, 256))  # a dense q's own memory
    assert torch.equal(got, want)
    wide = _randn(2, 3, 2 * 256).bfloat16()[..., :256].unflatten(-1, (4, 64)).copy_(q)
    with pytest.raises(ValueError, match="shares memory"):
        sm100_kv8_attention(cache, wide, out=wide.as_strided((2, 3, 256), (768, 256, 1)))
