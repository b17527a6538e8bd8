"""The decoding operators without a GPU: packing of 4-bit weights, checks of
handles, registered operators on meta tensors; on the GPU, the registered
operators give the wrappers' bits."""

from __future__ import annotations

import pytest
import torch

from solution import _binding, _native
from solution.kernels import (
    Kv8Cache,
    RotaryTable,
    W4Weight,
    can_use_sm100_kv8_append,
    can_use_sm100_kv8_attention,
    can_use_sm100_linear_w4,
    can_use_sm100_qk_norm_rope,
    ops,
    pack_w4,
    sm100_kv8_append,
    sm100_kv8_attention,
    sm100_linear_w4,
    sm100_qk_norm_rope,
)

B200 = torch.ops.b200tx


def _cache(device: str = "cpu", **kwargs) -> Kv8Cache:  # noqa: ANN003
    return Kv8Cache.create(**{"slots": 2, "max_tokens": 100, "num_kv_heads": 2, "head_dim": 64, "device": device, **kwargs})


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize(("n", "k"), [(1, 8), (5, 128), (17, 136), (3, 1000)])
def test_pack_w4_is_the_nearest_code(n: int, k: int, group: int) -> None:
    weight = torch.randn(n, k, generator=torch.Generator().manual_seed(n + k))
    weight[0] = 0
    packed = pack_w4(weight, group)
    wide = -(-k // 128) * 128
    assert packed.packed.shape == (n, wide // 2) and packed.scales.shape == (wide // group, n) and packed.group == group
    scale = packed.scales.t().float().repeat_interleave(group, 1)[:, :k]
    # the nearest of -8..7 steps; bf16 scales may fall short of max / 7 by 2^-8, so that 7 steps do
    assert bool(((packed.dequantize() - weight).abs() <= scale * (0.5 + 7 * 2.0**-8) + 1e-12).all())
    # a single weight lands where the format says
    one = torch.zeros(2, 256)
    one[1, 128 + 2 * 32 + 3 * 8 + 5] = 7.0  # run 1, word 4 * 2 + 3, weight 5 of its eight
    code = pack_w4(one, 32).packed[1].view(torch.int32).reshape(2, 16)
    stored = code[1, 4 * 3 + 2].item() & 0xFFFFFFFF
    nibble = [0, 2, 4, 6, 1, 3, 5, 7].index(5)
    assert stored == sum((15 if i == nibble else 8) << (4 * i) for i in range(8))


def test_handles_refuse_what_does_not_fit() -> None:
    good = _cache()
    parts = dict(codes=good.codes, scales=good.scales, tail=good.tail, page_table=good.page_table, lengths=good.lengths)
    for name, bad in (
        ("codes", good.codes[:, :, :, :, :32]),
        ("codes", good.codes.to(torch.int16)),
        ("scales", good.scales[:, :1]),
        ("tail", good.tail.float()),
        ("page_table", good.page_table.long()),
        ("lengths", good.lengths[:1]),
    ):
        with pytest.raises(ValueError):
            Kv8Cache(**{**parts, name: bad})
    with pytest.raises(ValueError):
        Kv8Cache(**{**parts, "codes": good.codes.transpose(1, 1)[..., ::2]})
    with pytest.raises(ValueError):
        good.handle(1)
    assert Kv8Cache(*(t[0] for t in (good.codes, good.scales, good.tail)), good.page_table, good.lengths).layers == 1
    with pytest.raises(ValueError):
        RotaryTable(torch.zeros(4, 8), torch.zeros(4, 4))
    with pytest.raises(ValueError):
        RotaryTable(torch.zeros(4, 8).double(), torch.zeros(4, 8).double())
    weight = pack_w4(torch.randn(4, 128))
    with pytest.raises(ValueError):
        W4Weight(weight.packed, weight.scales, 136)
    with pytest.raises(ValueError):
        W4Weight(weight.packed, weight.scales.float(), 128)
    with pytest.raises(ValueError):
        pack_w4(torch.randn(4, 12))


def test_rotary_table_create() -> None:
    table = RotaryTable.create(70000, 16, "cpu")
    angle = 69999 * 10000.0 ** (-2 * 3 / 16)
    want = torch.tensor(angle, dtype=torch.float64)
    assert abs(float(table.cos[69999, 3]) - float(want.cos())) < 1e-7 and abs(float(table.sin[69999, 3]) - float(want.sin())) < 1e-7


def test_cpu_tensors_are_refused() -> None:
    qkv = torch.zeros(1, 2, 6 * 64, dtype=torch.bfloat16)
    cache, weight = _cache(), pack_w4(torch.randn(8, 64))
    with torch.no_grad():
        assert not can_use_sm100_qk_norm_rope(qkv, 2) and not can_use_sm100_kv8_append(cache, qkv, 2)
        assert not can_use_sm100_kv8_attention(cache, qkv.view(1, 2, 6, 64))
        assert not can_use_sm100_linear_w4(qkv[..., :64].contiguous(), weight)
        for call in (
            lambda: sm100_qk_norm_rope(qkv, 2),
            lambda: sm100_kv8_append(cache, qkv, 2),
            lambda: sm100_kv8_attention(cache, qkv.view(1, 2, 6, 64)),
            lambda: sm100_linear_w4(qkv[..., :64].contiguous(), weight),
            lambda: B200.qk_norm_rope(qkv, 2, 2),
            lambda: B200.linear_w4(qkv[..., :64], weight.packed, weight.scales),
        ):
            with pytest.raises(RuntimeError, match="ineligible|no CPU fallback"):
                call()


def test_the_binding_checks_its_arguments() -> None:
    assert _native.BINDING_PATH.exists() and _binding.available()
    module = _binding.load()
    with pytest.raises(TypeError, match="arguments"):
        module.linear_w4(1, 2)
    with pytest.raises(ValueError, match="missing"):
        module.init({})
    with pytest.raises(RuntimeError, match="ineligible"):
        module.linear_w4("x", "w", "s", None, 64, 64, 0, 0, None)
    with pytest.raises(TypeError):
        module.linear_w4("x", "w", "s", None, "k", 64, 0, 0, None)
    with pytest.raises(ValueError, match="Kv8Cache"):
        module.kv8_attention(None, None, None, None, None, None, {}, None)


def test_c_entry_points_check_before_any_device_work() -> None:
    """Status -1 (arguments) or -2 (unsupported) and a message, without a GPU."""
    import ctypes

    lib = _native.load()
    buf = ctypes.create_string_buffer(64)
    at = (ctypes.addressof(buf) + 15) // 16 * 16
    view = _native.Kv8CacheView(at, at, at, at, at, 4, 2, 2, 2, 64)
    ref = ctypes.byref(view)
    rope = ctypes.byref(_native.Rope(at, at, 8, 12, 0))

    def rope_call(q: int = at, dtype: int = 1, dim: int = 64, stride: int = 384, table: object = None) -> int:
        return lib.b200tx_qk_norm_rope(q, at, dtype, 1, 1, 4, 1, dim, stride, stride, stride, stride, None, None, 1e-6,
                                       table, None, 0, 0, None)

    def append(cache: object = ref, q: int = at, heads: int = 4, batch: int = 1) -> int:
        return lib.b200tx_kv8_append(cache, q, 1, at, batch, 1, heads, 512, 512, None, None, None, None, 1e-6, None, None)

    def attend(heads: int = 4, scale: float = 1.0, stride: int = 256) -> int:
        return lib.b200tx_kv8_attention(ref, at, at, 1, 1, heads, stride, stride, None, None, scale, at, 0, None)

    def linear(k: int = 64, group: int = 64, epilogue: int = 0, x: int | None = at) -> int:
        return lib.b200tx_linear_w4(x, k, at, at, None, at, 1, 1, 8, k, group, epilogue, None)

    for call, status, text in (
        (lambda: rope_call(q=at + 2), -1, "16-byte aligned"),
        (lambda: rope_call(dtype=7), -1, "dtype"),
        (lambda: rope_call(dim=96), -2, "head_dim"),
        (lambda: rope_call(stride=12), -1, "multiples of 8"),
        (lambda: rope_call(table=rope), -1, "rotary"),
        (lambda: append(cache=None), -1, "null cache"),
        (lambda: append(q=None), -1, "null tensor"),
        (lambda: append(heads=1), -1, "bad shape"),
        (lambda: append(batch=3), -1, "slots"),
        (lambda: attend(heads=5), -1, "evenly"),
        (lambda: attend(scale=float("inf")), -1, "scale"),
        (lambda: attend(stride=4), -1, "multiples of 8"),
        (lambda: lib.b200tx_kv8_gather(ref, at, at, 1, 0, 0, None, None, None), -1, "bad shape"),
        (lambda: lib.b200tx_kv8_gather(ref, at + 8, at, 1, 1, 0, None, None, None), -1, "aligned"),
        (lambda: linear(k=60), -1, "bad shape"),
        (lambda: linear(group=16), -2, "group"),
        (lambda: linear(epilogue=3), -1, "epilogue"),
        (lambda: linear(x=None), -1, "null"),
    ):
        assert call() == status, text
        assert text in lib.b200tx_last_error().decode(), (text, lib.b200tx_last_error())
    view.head_dim = 96
    assert append() == -2 and "head_dim" in lib.b200tx_last_error().decode()


def _meta(*shape: int, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    return torch.empty(*shape, device="meta", dtype=dtype)


def test_registered_operators_trace_on_meta_tensors() -> None:
    f32, u8, i32 = torch.float32, torch.uint8, torch.int32
    for name in ("qk_norm_rope", "kv8_append", "kv8_attention", "linear_w4"):
        assert name in ops.OPERATORS
    y = B200.qk_norm_rope(_meta(2, 7, 8 * 64), 4, 2, None, None, 1e-6, _meta(9, 32, dtype=f32), _meta(9, 32, dtype=f32))
    assert (tuple(y.shape), y.dtype) == ((2, 7, 512), torch.bfloat16)
    cache = (_meta(6, 2, 2, 64, 64, dtype=u8), _meta(6, 2, 2, dtype=f32), _meta(3, 2, 2, 2, 64, 64),
             _meta(3, 2, dtype=i32), _meta(3, dtype=i32))
    q = B200.kv8_append(*cache, _meta(3, 5, 8 * 64, dtype=f32), 4)
    assert (tuple(q.shape), q.dtype) == ((3, 5, 4, 64), torch.bfloat16)
    assert tuple(B200.kv8_attention(*cache, q).shape) == (3, 5, 256)
    w = pack_w4(torch.randn(24, 200), 32)
    y = B200.linear_w4(_meta(2, 3, 200), w.packed.to("meta"), w.scales.to("meta"), None, True, f32)
    assert (tuple(y.shape), y.dtype) == ((2, 3, 24), f32)
    for call in (
        lambda: B200.qk_norm_rope(_meta(2, 7, 500), 4, 2),
        lambda: B200.qk_norm_rope(_meta(2, 7, 8 * 64), 4, 2, None, None, 1e-6, _meta(9, 32, dtype=f32)),
        lambda: B200.kv8_append(*cache, _meta(3, 5, 8 * 32), 4),
        lambda: B200.kv8_attention(*cache, _meta(3, 5, 3, 64)),
        lambda: B200.kv8_attention(cache[0], cache[1], cache[2][:2], *cache[3:], q),
        lambda: B200.linear_w4(_meta(2, 3, 196), w.packed.to("meta"), w.scales.to("meta")),
    ):
        with pytest.raises(ValueError):
            call()


@pytest.mark.gpu
def test_registered_operators_give_the_wrappers_bits() -> None:
    g = torch.Generator(device="cuda").manual_seed(0)
    randn = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    with torch.inference_mode():
        qkv = randn(2, 70, 6 * 64).bfloat16()
        table = RotaryTable.create(128, 64, "cuda")
        weight = 1 + 0.1 * randn(64)
        want, _ = sm100_qk_norm_rope(qkv, 2, q_weight=weight, k_weight=weight, rope=table)
        got = B200.qk_norm_rope(qkv, 2, 2, weight, weight, 1e-6, table.cos, table.sin)
        assert torch.equal(got, want)
        one, two = _cache("cuda"), _cache("cuda")
        q, _ = sm100_kv8_append(one, qkv, 2, k_weight=weight, rope=table)
        parts = (two.codes[0], two.scales[0], two.tail[0], two.page_table, two.lengths)
        assert torch.equal(B200.kv8_append(*parts, qkv, 2, None, weight, 1e-6, table.cos, table.sin), q)
        assert torch.equal(one.codes, two.codes) and torch.equal(one.tail, two.tail) and torch.equal(one.scales, two.scales)
        assert torch.equal(B200.kv8_attention(*parts, q), sm100_kv8_attention(one, q)[0])
        w = pack_w4(randn(40, 200), 32)
        x = randn(3, 200).bfloat16()
        assert torch.equal(B200.linear_w4(x, w.packed, w.scales, None, True), sm100_linear_w4(x, w, gelu=True)[0])
    torch.library.opcheck(
        B200.linear_w4.default, (x.clone(), w.packed.clone(), w.scales.clone()),
        test_utils=("test_schema", "test_faketensor"),
    )
    fresh = _cache("cuda")
    torch.library.opcheck(
        B200.kv8_append.default,
        (fresh.codes[0], fresh.scales[0], fresh.tail[0], fresh.page_table, fresh.lengths, qkv.clone(), 2),
        test_utils=("test_schema", "test_faketensor"),
    )
