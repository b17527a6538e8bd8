"""The 8-bit cache at the ends of the number range: blocks of tiny values, values
that lie halfway between two codes, long tails of small probabilities, and
rows whose scores are all minus infinity."""

from __future__ import annotations

import math

import pytest
import torch

from solution.kernels import KV8_BLOCK, Kv8Cache, sm100_kv8_append, sm100_kv8_attention, sm100_kv8_gather

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


@pytest.fixture(autouse=True)
def _inference():
    with torch.inference_mode():
        yield
    torch.cuda.synchronize()


def _coded(x: torch.Tensor) -> Kv8Cache:
    """A cache of one kv head that holds x, bf16 [tokens, 2, D] (keys, values), appended at once."""
    tokens, _, dim = x.shape
    cache = Kv8Cache.create(slots=1, max_tokens=tokens, num_kv_heads=1, head_dim=dim, device=DEV)
    qkv = torch.cat((torch.zeros_like(x[:, :1]), x), 1).reshape(1, tokens, 3 * dim)
    sm100_kv8_append(cache, qkv.contiguous(), 1)
    cache.advance(tokens)
    return cache


def _definition(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Scales and codes of x in 32 bits, on the CPU: max / 127, rint(x / scale) + 128."""
    blocks = x.float().cpu().unflatten(0, (-1, KV8_BLOCK)).transpose(1, 2)  # block, kv, token, dim
    scale = blocks.abs().amax((-2, -1)) / 127
    code = torch.where(scale[..., None, None] > 0, blocks / scale[..., None, None], torch.zeros_like(blocks))
    return scale, code.round() + 128


@pytest.mark.parametrize("dim", [32, 64, 128, 256])
def test_blocks_of_tiny_values_keep_their_values(dim: int) -> None:
    """Peaks of 2^-60 down to the smallest bf16 number, where the scale and its
    reciprocal leave the normal numbers: every value within half a step."""
    peaks = [-60, -64, -90, -100, -119, -120, -121, -122, -124, -126, -130, -133]
    g = torch.Generator().manual_seed(dim)
    x = (2 * torch.rand(len(peaks), KV8_BLOCK, 2, dim, generator=g) - 1).double()
    x[:, 0, :, 0], x[:, 1, :, 1], x[:, 2, :, 2] = 1.0, -1.0, 0.0
    x = (x * 2.0 ** torch.tensor(peaks, dtype=torch.float64)[:, None, None, None]).flatten(0, 1).to(torch.bfloat16)
    cache = _coded(x.to(DEV))
    scale, code = _definition(x)
    assert torch.equal(cache.scales[0, :, :, 0].cpu(), scale)
    # the definition's quotient is rounded once, the kernel's at most by 2^-22 more: half a step and 2^-15
    want = x.double().unflatten(0, (-1, KV8_BLOCK)).transpose(1, 2) / scale.double()[..., None, None] + 128
    off = (cache.codes[0, :, :, 0].cpu().double() - want).abs()
    assert float(off.max()) <= 0.5 + 2.0**-15, off.amax((1, 2, 3)).tolist()
    k, v, _ = sm100_kv8_gather(cache, len(x))
    got = torch.stack((k, v), 2)[0, :, :, 0].cpu().double()  # token, kv, dim
    step = scale.double().repeat_interleave(KV8_BLOCK, 0)[..., None]
    # half a step and the rounding to bf16 (2^-8, or half the smallest subnormal 2^-133)
    bound = step * (0.5 + 2.0**-15) + 2.0**-8 * x.double().abs() + 2.0**-134
    assert bool(((got - x.double()).abs() <= bound).all())


@pytest.mark.parametrize("dim", [32, 64, 128, 256])
def test_codes_are_the_rounded_quotients(dim: int) -> None:
    """code = rint(x / scale) + 128 with the quotient rounded to 32 bits, bit for bit, halfway
    values (half the block's peak, and other ties) among them."""
    g = torch.Generator().manual_seed(dim)
    blocks = 48
    x = torch.randn(blocks, KV8_BLOCK, 2, dim, generator=g)
    peak = torch.tensor([1 + i / 128 for i in range(blocks)])[:, None, None, None] * 8  # 8 bits: exact in bf16
    x = x.clamp(-7, 7)
    x[:, 0] = peak[:, 0]
    x[:, 1:9] = peak / 2
    x[:, 9:17] = -peak / 2
    x[:, 17:25] = peak * torch.randint(-127, 128, (blocks, 8, 2, dim), generator=g) / 254
    x[1::3] *= 2.0**-30
    x[2::3] *= 2.0**60
    x = x.flatten(0, 1).to(torch.bfloat16)
    cache = _coded(x.to(DEV))
    scale, code = _definition(x)
    assert torch.equal(cache.scales[0, :, :, 0].cpu(), scale)
    assert torch.equal(cache.codes[0, :, :, 0].cpu().float(), code)


def _shared_pages(batch: int, kv_heads: int, dim: int, blocks: int, sinks: int) -> Kv8Cache:
    """Sequences of full blocks that lie in two pages: the first `sinks` blocks in page 0
    (its first key is zero and its value too), all others in page 1."""
    cache = Kv8Cache(
        torch.full((2, 2, kv_heads, KV8_BLOCK, dim), 128, dtype=torch.uint8, device=DEV),
        torch.full((2, 2, kv_heads), 1.0 / 127, device=DEV),
        torch.zeros(batch, 2, 2, kv_heads, KV8_BLOCK, dim, dtype=torch.bfloat16, device=DEV),
        torch.ones(batch, blocks, dtype=torch.int32, device=DEV),
        torch.full((batch,), blocks * KV8_BLOCK - 1, dtype=torch.int32, device=DEV),
    )
    cache.page_table[:, :sinks] = 0
    return cache


def test_a_long_tail_of_small_probabilities_counts() -> None:
    """A token that takes nearly all of the weight before 262144 tokens of 2^-25.05 each. Taken
    together they weigh 2^-7; what probabilities of 16 bits may cost is 2^-11 of the
    largest value.  A warp has some 38000 of the tokens."""
    batch, kv_heads, dim, blocks = 16, 16, 32, 4096
    cache = _shared_pages(batch, kv_heads, dim, blocks, 4)
    codes = cache.codes[0]
    codes[:, 0, :, :, 0] = 128 - 127  # keys (-1, 0, ...): far below the sink's 0
    codes[0, 0, :, 0, 0] = 128  # the first key of page 0
    codes[:, 1] = 255  # values 1, the sink's 0
    codes[0, 1, :, 0] = 128
    low = 25.05 * math.log(2.0)
    q = torch.zeros(batch, 1, kv_heads, dim, device=DEV, dtype=torch.bfloat16)
    q[..., 0] = 1.0
    got, _ = sm100_kv8_attention(cache, q, scale=low)
    tokens = blocks * KV8_BLOCK
    tail = (tokens - 4) * 2.0**-25.05
    want = tail / (4 + tail)
    # scores carry 2^-22 of themselves, 2^-17 in a weight
    bound = 2.0**-8 * want + 2.0**-11 + 2.0**-17 * want
    assert abs(float(got.float().mean()) - want) <= bound and float((got.double() - want).abs().max()) <= bound


@pytest.mark.parametrize("dim", [32, 64, 128, 256])
def test_scores_that_are_all_minus_infinity_give_nan(dim: int) -> None:
    """As softmax does: no weight is defined.  Rows with one finite score are not concerned."""
    cache = Kv8Cache.create(slots=1, max_tokens=64, num_kv_heads=1, head_dim=dim, device=DEV)
    qkv = torch.ones(1, 9, 3 * dim, dtype=torch.bfloat16, device=DEV)
    qkv[0, :3, dim] = float("-inf")  # the first three tokens' keys
    q, _ = sm100_kv8_append(cache, qkv, 1)
    got = sm100_kv8_attention(cache, q)[0][0]
    assert got.isnan().all(-1).tolist() == [True] * 3 + [False] * 6
    assert bool((got[3:] == 1).all())  # all values are 1
