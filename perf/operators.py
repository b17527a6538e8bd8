"""Workloads of the decoding operators: norm and rotation of queries and keys,
the 8-bit key/value cache (append and attention) and 4-bit linear layers.

``run`` computes a case with elementary torch operations in 32 bits, or, where
``own`` is set, with the framework's kernels (``solution.kernels``).
``exact`` computes it from the definition in 64 bits.
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

PACKAGE = "ml-guided-program-search-for-shape-specialized-transformer-optimization_b200"
BLOCK = 64  # tokens that share a scale
WORD_ORDER = (0, 2, 4, 6, 1, 3, 5, 7)  # nibble i of a word holds weight WORD_ORDER[i] of its eight


def _kernels():
    path = os.path.join(os.getcwd(), PACKAGE)
    if path not in sys.path:
        sys.path.insert(0, path)
    import solution.kernels as kernels

    return kernels


# ------------------------------------------------------------------ cases


def listed():
    return [
        # One token of one sequence: what a decoding step asks for before its attention.
        {"name": "rope step", "op": "rope", "batch": 1, "tokens": 1, "heads": 16, "kv_heads": 4, "dim": 64,
         "rotary": 64, "interleaved": False, "norm": True, "type": "bf16"},
        # A ragged prompt in 32 bits, half of each head rotated in adjacent pairs.
        {"name": "rope prompt f32", "op": "rope", "batch": 3, "tokens": 333, "heads": 6, "kv_heads": 2, "dim": 128,
         "rotary": 64, "interleaved": True, "norm": True, "type": "f32"},
        # The benchmark's batch of 8 sequences of 2048 tokens, 16 heads of 64.
        {"name": "rope batch", "op": "rope", "batch": 8, "tokens": 2048, "heads": 16, "kv_heads": 16, "dim": 64,
         "rotary": 64, "interleaved": False, "norm": True, "type": "bf16"},
        # One new token for each of 32 sequences with short histories.
        {"name": "append step", "op": "append", "batch": 32, "tokens": 1, "start": 200, "heads": 16, "kv_heads": 4,
         "dim": 64, "rotary": 64, "interleaved": False, "norm": True},
        # Four prompts of 4000 tokens into empty caches, grouped heads of 128.
        {"name": "append prompt", "op": "append", "batch": 4, "tokens": 4000, "start": 0, "heads": 32, "kv_heads": 8,
         "dim": 128, "rotary": 128, "interleaved": False, "norm": True},
        # One user's step early in a conversation: latency.
        {"name": "attention step", "op": "attention", "batch": 1, "tokens": 1, "context": 1000, "ragged": False,
         "heads": 16, "kv_heads": 16, "dim": 64},
        # A serving batch with histories of very different lengths.
        {"name": "attention batch", "op": "attention", "batch": 64, "tokens": 1, "context": 8192, "ragged": True,
         "heads": 32, "kv_heads": 8, "dim": 128},
        # One step over the longest sequence of the benchmarks.
        {"name": "attention long", "op": "attention", "batch": 1, "tokens": 1, "context": 100000, "ragged": False,
         "heads": 16, "kv_heads": 16, "dim": 64},
        # A run of drafted tokens, checked at once.
        {"name": "attention draft", "op": "attention", "batch": 4, "tokens": 16, "context": 3001, "ragged": True,
         "heads": 8, "kv_heads": 2, "dim": 128},
        # The feed-forward input layer of the benchmark's model for one token.
        {"name": "w4 one token", "op": "w4", "rows": 1, "inner": 1024, "outer": 4096, "group": 64, "gelu": True,
         "bias": True, "type": "bf16"},
        # A wide layer for a handful of tokens.
        {"name": "w4 few tokens", "op": "w4", "rows": 8, "inner": 8192, "outer": 28672, "group": 128, "gelu": False,
         "bias": False, "type": "bf16"},
        # Odd widths, the finest groups and a 32-bit result.
        {"name": "w4 odd", "op": "w4", "rows": 29, "inner": 4744, "outer": 5003, "group": 32, "gelu": False,
         "bias": True, "type": "f32"},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("rope", "append", "attention", "attention", "w4", "w4"))
    if op == "w4":
        case = {"op": op, "rows": _log(rng, 1, 32), "inner": 8 * _log(rng, 16, 2048), "outer": _log(rng, 64, 32768),
                "group": rng.choice((32, 64, 128)), "gelu": rng.random() < 0.5, "bias": rng.random() < 0.5,
                "type": rng.choice(("bf16", "f32"))}
        case["outer"] = min(case["outer"], 8192 * 28672 // case["inner"])
        return case
    dim = rng.choice((32, 64, 128, 256))
    kv_heads = rng.choice((1, 2, 3, 4, 8, 16))
    heads = kv_heads * rng.choice((1, 2, 3, 4, 8) if op == "attention" else (1, 2, 4))
    if op == "attention":
        tokens = 1 if rng.random() < 0.7 else _log(rng, 2, 32)
        context = tokens + _log(rng, 1, 65536)
        batch = _log(rng, 1, 128)
        batch = max(1, min(batch, 64 * 8192 * 8 * 128 // (context * heads * dim)))
        return {"op": op, "batch": batch, "tokens": tokens, "context": context, "ragged": rng.random() < 0.5,
                "heads": heads, "kv_heads": kv_heads, "dim": dim}
    rotary = rng.choice((dim, dim // 2))
    shape = {"heads": heads, "kv_heads": kv_heads, "dim": dim, "rotary": rotary,
             "interleaved": rng.random() < 0.3, "norm": rng.random() < 0.8}
    most = 4 * 4000 * 48 * 128 // ((heads + 2 * kv_heads) * dim)
    if op == "rope":
        tokens = _log(rng, 1, 8192)
        batch = max(1, min(_log(rng, 1, 64), most // tokens))
        return {"op": op, "batch": batch, "tokens": tokens, **shape, "type": rng.choice(("bf16", "f32"))}
    kind = rng.choice(("step", "draft", "prompt"))
    tokens = {"step": 1, "draft": _log(rng, 2, 64), "prompt": _log(rng, 65, 4000)}[kind]
    # a step or a draft starts anywhere in a block, a prompt at the start of one
    start = 64 * rng.randint(0, 4) if kind == "prompt" else rng.randint(0, 500)
    batch = max(1, min(_log(rng, 1, 64), most // (tokens + start)))
    return {"op": op, "batch": batch, "tokens": tokens, "start": start, **shape}


# ------------------------------------------------------------------ inputs


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rope_table(positions, rotary):
    """cos and sin of position * 10000^(-2i/rotary), [positions, rotary/2]."""
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * torch.pow(
        10000.0, -torch.arange(0, rotary, 2, dtype=torch.float64, device="cuda") / rotary)
    return angle.cos().float(), angle.sin().float()


def _norm_weights(case, g):
    if not case["norm"]:
        return None, None
    return tuple(1 + 0.1 * torch.randn(case["dim"], generator=g, device="cuda") for _ in range(2))


def _packed(case, g, dtype):
    """The packed projection [batch, tokens, q heads then k heads then v heads]."""
    width = (case["heads"] + 2 * case["kv_heads"]) * case["dim"]
    return torch.randn(case["batch"], case["tokens"], width, generator=g, device="cuda").to(dtype)


def _cache(batch, held, room, kv_heads, dim, g):
    """A paged cache that holds held[b] tokens of each sequence: full blocks as
    codes with a scale, the open block in 16 bits; pages in a shuffled order."""
    max_blocks = -(-room // BLOCK)
    pages = batch * max_blocks
    table = torch.randperm(pages, generator=g, device="cuda").to(torch.int32).reshape(batch, max_blocks)
    # keys have a few strong channels, as they do in practice
    channel = 1 + 3 * (torch.rand(2, kv_heads, 1, dim, generator=g, device="cuda") < 0.05)
    codes = torch.empty(pages, 2, kv_heads, BLOCK, dim, dtype=torch.uint8, device="cuda")
    scales = torch.empty(pages, 2, kv_heads, device="cuda")
    some = max(1, (1 << 28) // (2 * kv_heads * BLOCK * dim))
    for at in range(0, pages, some):
        x = torch.randn(min(some, pages - at), 2, kv_heads, BLOCK, dim, generator=g, device="cuda").mul_(channel)
        s = x.abs().amax(dim=(-2, -1)) / 127
        scales[at:at + some] = s
        codes[at:at + some] = x.div_(s[..., None, None]).round_().add_(128).to(torch.uint8)
    tail = torch.randn(batch, 2, 2, kv_heads, BLOCK, dim, generator=g, device="cuda").mul_(channel).bfloat16()
    return {"codes": codes, "scales": scales, "tail": tail, "page_table": table,
            "lengths": torch.tensor(held, dtype=torch.int32, device="cuda")}


def _ragged(total, least, batch, g):
    """Lengths spread evenly over the logarithm, the longest one among them."""
    u = torch.rand(batch, generator=g, device="cuda").tolist()
    u[0] = 1.0
    return [max(least, min(total, int(round(least * (total / least) ** x)))) for x in u]


def prepare(case, seed):
    g = _generator(seed)
    state = {"case": dict(case)}
    op = case["op"]
    if op == "rope":
        state["qkv"] = _packed(case, g, torch.bfloat16 if case["type"] == "bf16" else torch.float32)
        state["q_weight"], state["k_weight"] = _norm_weights(case, g)
        state["cos"], state["sin"] = _rope_table(case["tokens"] + 64, case["rotary"])
        first = torch.randint(0, 64, (case["batch"], 1), generator=g, device="cuda")
        state["positions"] = (first + torch.arange(case["tokens"], device="cuda")).to(torch.int32)
        if own:
            kernels = _kernels()
            state["rope"] = kernels.RotaryTable(state["cos"], state["sin"], interleaved=case["interleaved"])
    elif op == "append":
        state["qkv"] = _packed(case, g, torch.bfloat16)
        state["q_weight"], state["k_weight"] = _norm_weights(case, g)
        spread = 1 if case["start"] % BLOCK == 0 else min(case["start"], 100)
        back = torch.randint(0, spread, (case["batch"],), generator=g, device="cuda").tolist()
        held = [case["start"] - b for b in back]
        room = case["start"] + case["tokens"]
        state["cache"] = _cache(case["batch"], held, room, case["kv_heads"], case["dim"], g)
        state["cos"], state["sin"] = _rope_table(room, case["rotary"])
        state["room"] = room
        if own:
            kernels = _kernels()
            state["rope"] = kernels.RotaryTable(state["cos"], state["sin"], interleaved=case["interleaved"])
            state["handle"] = kernels.Kv8Cache(**state["cache"])
    elif op == "attention":
        total = case["context"]
        least = case["tokens"]
        lens = _ragged(total, least, case["batch"], g) if case["ragged"] else [total] * case["batch"]
        held = [n - case["tokens"] for n in lens]
        state["cache"] = _cache(case["batch"], held, total, case["kv_heads"], case["dim"], g)
        state["q"] = torch.randn(case["batch"], case["tokens"], case["heads"], case["dim"], generator=g,
                                 device="cuda").bfloat16()
        if own:
            state["handle"] = _kernels().Kv8Cache(**state["cache"])
    else:
        n, k, group = case["outer"], case["inner"], case["group"]
        wide = -(-k // 128) * 128
        weight = torch.randn(n, k, generator=g, device="cuda") * k ** -0.5
        weight = torch.nn.functional.pad(weight, (0, wide - k)).reshape(n, wide // group, group)
        scale = (weight.abs().amax(-1) / 7).bfloat16()
        code = torch.where(scale[..., None] > 0, weight / scale[..., None].float(), 0).round_().clamp_(-8, 7).add_(8)
        code = code.to(torch.uint8).reshape(n, wide // 128, 4, 4, 8)[..., WORD_ORDER]
        # 128 weights of a row are 16 words of 8: word (a, b) of the 4 x 4 is stored at (b, a)
        code = code.transpose(2, 3).reshape(n, wide // 2, 2)
        state["packed"] = code[..., 0] | (code[..., 1] << 4)
        state["scales"] = scale.t().contiguous()  # [wide / group, n]
        state["x"] = torch.randn(case["rows"], k, generator=g, device="cuda").bfloat16()
        state["bias"] = 0.1 * torch.randn(n, generator=g, device="cuda") if case["bias"] else None
        if own:
            state["handle"] = _kernels().W4Weight(state["packed"], state["scales"], k)
    return state


# ------------------------------------------------------------------ plain forms


def _rms(x, weight, eps=1e-6):
    return x if weight is None else x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * weight


def _rotate(x, cos, sin, interleaved):
    """x [batch, tokens, heads, dim]; cos, sin [batch, tokens, 1, rotary/2]."""
    half = cos.shape[-1]
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, x[..., 2 * half:]), -1)


def _norm_rope(state, positions):
    """q [.., heads, dim], k and v [.., kv_heads, dim] in 32 bits."""
    case = state["case"]
    x = state["qkv"].float().unflatten(-1, (-1, case["dim"]))
    q, k, v = x.split((case["heads"], case["kv_heads"], case["kv_heads"]), 2)
    cos, sin = state["cos"][positions][:, :, None], state["sin"][positions][:, :, None]
    q = _rotate(_rms(q, state["q_weight"]), cos, sin, case["interleaved"])
    k = _rotate(_rms(k, state["k_weight"]), cos, sin, case["interleaved"])
    return q, k, v


def _stored(cache, total, dtype):
    """[batch, 2, kv_heads, tokens, dim]: what the cache holds of sequences of
    total[b] tokens (the open block read from its 16-bit slot)."""
    table = cache["page_table"].long()
    batch, blocks = table.shape
    x = (cache["codes"][table].to(dtype) - 128) * cache["scales"][table].to(dtype)[..., None, None]
    block = torch.arange(blocks, device="cuda")
    open_block = total.long() // BLOCK
    tail = cache["tail"][torch.arange(batch, device="cuda"), open_block % 2].to(dtype)
    x = torch.where((block == open_block[:, None])[:, :, None, None, None, None], tail[:, None], x)
    return x.permute(0, 2, 3, 1, 4, 5).flatten(3, 4)


def _append_plain(state):
    case, cache = state["case"], state["cache"]
    batch, tokens, start = case["batch"], case["tokens"], cache["lengths"].long()
    positions = start[:, None] + torch.arange(tokens, device="cuda")
    q, k, v = _norm_rope(state, positions)
    new = torch.stack((k, v), 1).bfloat16().float().transpose(2, 3)  # [batch, 2, kv_heads, tokens, dim]
    held = _stored(cache, start, torch.float32)
    room = held.shape[3]
    at = torch.arange(room, device="cuda") - start[:, None]  # [batch, room]
    index = at.clamp(0, tokens - 1)[:, None, None, :, None].expand(*held.shape[:3], room, case["dim"])
    fresh = (at >= 0)[:, None, None, :, None]
    x = torch.where(fresh, new.gather(3, index), held).unflatten(3, (-1, BLOCK))
    # blocks that fill in this call get their scale and codes now
    scale = x.abs().amax((-2, -1), keepdim=True) / 127
    coded = torch.where(scale > 0, x / scale, 0).round() * scale
    block = torch.arange(room // BLOCK, device="cuda")
    filled = (block >= start[:, None] // BLOCK) & (block < (start[:, None] + tokens) // BLOCK)
    x = torch.where(filled[:, None, None, :, None, None], coded, x).flatten(3, 4)
    x = torch.where((at < tokens)[:, None, None, :, None], x, 0)[:, :, :, :state["room"]]
    x = x.transpose(2, 3).bfloat16()
    return q.bfloat16(), x[:, 0], x[:, 1]


def _attention_plain(state):
    case, cache, q = state["case"], state["cache"], state["q"]
    batch, tokens, heads, dim = q.shape
    total = cache["lengths"] + tokens
    x = _stored(cache, total, torch.float32)
    kv_heads = x.shape[2]
    rows = q.float().reshape(batch, tokens, kv_heads, heads // kv_heads, dim).permute(0, 2, 1, 3, 4).flatten(2, 3)
    score = rows @ x[:, 0].transpose(-1, -2) * dim ** -0.5
    last = cache["lengths"][:, None] + torch.arange(tokens, device="cuda")
    seen = torch.arange(x.shape[3], device="cuda") <= last.repeat_interleave(heads // kv_heads, 1)[..., None]
    score = score.masked_fill(~seen[:, None], float("-inf"))
    p = (score - score.amax(-1, keepdim=True)).exp()
    p = p / p.sum(-1, keepdim=True)
    # what lies past a sequence's end is no value of its own
    value = x[:, 1].masked_fill((torch.arange(x.shape[3], device="cuda") >= total[:, None])[:, None, :, None], 0)
    out = (p @ value).unflatten(2, (tokens, -1)).permute(0, 2, 1, 3, 4)
    return out.reshape(batch, tokens, heads * dim).bfloat16()


def _unpacked(state, dtype):
    packed, scales = state["packed"], state["scales"]
    n, group = packed.shape[0], packed.shape[1] * 2 // scales.shape[0]
    code = torch.stack((packed & 15, packed >> 4), -1).reshape(n, -1, 4, 4, 8).transpose(2, 3)
    order = torch.empty(8, dtype=torch.long, device="cuda")
    order[list(WORD_ORDER)] = torch.arange(8, device="cuda")
    code = code[..., order].reshape(n, -1, group).to(dtype) - 8
    return (code * scales.t().to(dtype)[..., None]).reshape(n, -1)[:, :state["case"]["inner"]]


def _w4_plain(state):
    case = state["case"]
    y = state["x"].float() @ _unpacked(state, torch.float32).t()
    if state["bias"] is not None:
        y = y + state["bias"]
    if case["gelu"]:
        y = 0.5 * y * (1 + torch.erf(y * 2 ** -0.5))
    return y if case["type"] == "f32" else y.bfloat16()


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        kernels = _kernels()
        with torch.no_grad():
            if op == "rope":
                return kernels.sm100_qk_norm_rope(
                    state["qkv"], case["heads"], case["kv_heads"], q_weight=state["q_weight"],
                    k_weight=state["k_weight"], rope=state["rope"], positions=state["positions"])[0]
            if op == "append":
                q, _ = kernels.sm100_kv8_append(
                    state["handle"], state["qkv"], case["heads"], q_weight=state["q_weight"],
                    k_weight=state["k_weight"], rope=state["rope"])
                k, v, _ = kernels.sm100_kv8_gather(state["handle"], state["room"], tokens=case["tokens"])
                return q, k, v
            if op == "attention":
                return kernels.sm100_kv8_attention(state["handle"], state["q"])[0]
            return kernels.sm100_linear_w4(
                state["x"], state["handle"], state["bias"], gelu=case["gelu"],
                out_dtype=torch.float32 if case["type"] == "f32" else torch.bfloat16)[0]
    if op == "rope":
        parts = _norm_rope(state, state["positions"].long())
        return torch.cat(parts, 2).flatten(2).to(state["qkv"].dtype)
    if op == "append":
        return _append_plain(state)
    if op == "attention":
        return _attention_plain(state)
    return _w4_plain(state)


# ------------------------------------------------------------------ floor and 64-bit values


def work(case):
    op = case["op"]
    if op == "w4":
        m, n, k = case["rows"], case["outer"], case["inner"]
        bytes_ = n * k / 2 + 2 * n * k / case["group"] + 2 * m * k + m * n * (4 if case["type"] == "f32" else 2)
        return {"bytes": bytes_ + (4 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    width = (case["heads"] + 2 * case["kv_heads"]) * case["dim"]
    if op == "rope":
        values = case["batch"] * case["tokens"] * width
        return {"bytes": 2 * values * (2 if case["type"] == "bf16" else 4), "flops": 6 * values}
    if op == "append":
        new = case["batch"] * case["tokens"]
        kv = 2 * case["kv_heads"] * case["dim"]
        held = case["batch"] * (case["start"] + case["tokens"])
        # the projection in, the queries out, the new tokens' codes written, all values read back and given out
        bytes_ = 2 * new * width + 2 * new * case["heads"] * case["dim"] + new * kv + 3 * held * kv
        return {"bytes": bytes_, "flops": 6 * new * width}
    # ragged lengths are spread evenly over the logarithm between the new tokens and the longest context
    low, high = case["tokens"], case["context"]
    mean = (high - low) / math.log(high / low) if case["ragged"] and high > low else high
    mean = (high + (case["batch"] - 1) * mean) / case["batch"]
    keys = case["batch"] * mean
    q = case["batch"] * case["tokens"] * case["heads"] * case["dim"]
    return {"bytes": 2 * keys * case["kv_heads"] * case["dim"] + 4 * q,
            "flops": 4 * keys * case["tokens"] * case["heads"] * case["dim"]}


def _exact_heads(state, positions):
    """Norm and rotation in 64 bits, the rotation as a product of complex numbers."""
    case = state["case"]
    x = state["qkv"].double().unflatten(-1, (-1, case["dim"]))
    turn = torch.complex(state["cos"].double(), state["sin"].double())[positions][:, :, None]
    out = []
    q, k, v = x.split((case["heads"], case["kv_heads"], case["kv_heads"]), 2)
    for part, weight in ((q, state["q_weight"]), (k, state["k_weight"])):
        if weight is not None:
            part = part / (part.square().mean(-1, keepdim=True) + 1e-6).sqrt() * weight.double()
        head, rest = part[..., :case["rotary"]], part[..., case["rotary"]:]
        pairs = head.unflatten(-1, (-1, 2) if case["interleaved"] else (2, -1))
        if not case["interleaved"]:
            pairs = pairs.transpose(-1, -2)
        pairs = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        if not case["interleaved"]:
            pairs = pairs.transpose(-1, -2)
        out.append(torch.cat((pairs.flatten(-2), rest), -1))
    return (*out, v)


def _exact_sequence(cache, b, total):
    """[2, kv_heads, total, dim] of one sequence in 64 bits, block by block."""
    full = total // BLOCK
    pages = cache["page_table"][b, :full].long()
    x = (cache["codes"][pages].double() - 128) * cache["scales"][pages].double()[..., None, None]
    x = x.permute(1, 2, 0, 3, 4).flatten(2, 3)
    return torch.cat((x, cache["tail"][b, full % 2][:, :, :total - full * BLOCK].double()), 2)


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "rope":
        return torch.cat(_exact_heads(state, state["positions"].long()), 2).flatten(2)
    if op == "w4":
        y = state["x"].double() @ _unpacked(state, torch.float64).t()
        y = y if state["bias"] is None else y + state["bias"].double()
        return y * torch.special.ndtr(y) if case["gelu"] else y
    cache, lengths = state["cache"], state["cache"]["lengths"].tolist()
    if op == "append":
        positions = torch.tensor(lengths, device="cuda")[:, None] + torch.arange(case["tokens"], device="cuda")
        q, k, v = _exact_heads(state, positions)
        out = torch.zeros(2, case["batch"], state["room"], case["kv_heads"], case["dim"], dtype=torch.float64,
                          device="cuda")
        for b, start in enumerate(lengths):
            new = torch.stack((k[b], v[b])).bfloat16().double().transpose(1, 2)
            x = torch.cat((_exact_sequence(cache, b, start), new), 2)
            total = start + case["tokens"]
            low, high = start // BLOCK * BLOCK, total // BLOCK * BLOCK
            if high > low:  # the blocks that fill now
                y = x[:, :, low:high].unflatten(2, (-1, BLOCK))
                s = y.abs().amax((-2, -1), keepdim=True) / 127
                x[:, :, low:high] = (torch.where(s > 0, y / s, 0).round() * s).flatten(2, 3)
            out[:, b, :total] = x.transpose(1, 2)
        return q, out[0], out[1]
    if 16 * 4 * case["batch"] * case["context"] * case["heads"] * case["dim"] * case["tokens"] > 1e14:
        return None
    rows = []
    for b, held in enumerate(lengths):
        x = _exact_sequence(cache, b, held + case["tokens"])
        group = case["heads"] // case["kv_heads"]
        q = state["q"][b].double().unflatten(1, (-1, group)).permute(1, 2, 0, 3)  # kv head, group, token, dim
        score = q @ x[0][:, None].transpose(-1, -2) / math.sqrt(case["dim"])
        late = torch.ones(case["tokens"], x.shape[2], dtype=torch.bool, device="cuda").triu(held + 1)
        weight = torch.softmax(score.masked_fill(late, float("-inf")), -1)
        rows.append((weight @ x[1][:, None]).permute(2, 0, 1, 3).reshape(case["tokens"], -1))
    return torch.stack(rows)
