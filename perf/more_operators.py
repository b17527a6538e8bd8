"""Workloads of the operators for many requests over one cached decoder: low-rank
adapters beside a shared projection, forking, turnover and compaction of the
8-bit cache's pages, and verification of drafted tokens.

``run`` computes a case with elementary torch operations, or, where ``own`` is
set, with the framework's kernels (``solution.kernels``).  ``exact`` computes it
from the definition in 64 bits.
"""

from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

PACKAGE = "ml-guided-program-search-for-shape-specialized-transformer-optimization_b200"
BLOCK = 64  # tokens of a page


def _kernels():
    path = os.path.join(os.getcwd(), PACKAGE)
    if path not in sys.path:
        sys.path.insert(0, path)
    import solution.kernels as kernels

    return kernels


# ------------------------------------------------------------------ cases


def listed():
    return [
        # The feed-forward input layer of the benchmark's model for one token of one request.
        {"name": "adapters one token", "op": "adapters", "batch": 1, "tokens": 1, "inner": 1024, "outer": 4096, "rank": 16,
         "count": 8, "gelu": True, "base": "f32", "type": "bf16", "spread": "sequences"},
        # A serving batch: 64 requests, a token each, over 32 adapters (some requests without one).
        {"name": "adapters batch", "op": "adapters", "batch": 64, "tokens": 1, "inner": 4096, "outer": 14336, "rank": 16,
         "count": 32, "gelu": False, "base": "bf16", "type": "bf16", "spread": "sequences"},
        # Odd widths and a 32-bit result, rows in no order.
        {"name": "adapters odd", "op": "adapters", "batch": 29, "tokens": 7, "inner": 4744, "outer": 5003, "rank": 24,
         "count": 5, "gelu": False, "base": "f32", "type": "f32", "spread": "rows"},
        # Eight prompts of 2048 tokens, an adapter each, in the benchmark's widths.
        {"name": "adapters prompt", "op": "adapters", "batch": 8, "tokens": 2048, "inner": 1024, "outer": 4096, "rank": 64,
         "count": 16, "gelu": True, "base": "bf16", "type": "bf16", "spread": "sequences"},
        # Beams of one user: four kept, four replaced by copies of kept ones.
        {"name": "fork beams", "op": "fork", "slots": 8, "kept": 4, "context": 1000, "layers": 4, "kv_heads": 16, "dim": 64},
        # Sixteen samples of each of eight prompts that have just been read.
        {"name": "fork samples", "op": "fork", "slots": 136, "kept": 8, "context": 4000, "layers": 4, "kv_heads": 8,
         "dim": 128},
        # Two of a batch's requests end, and the pages of two new prompts are taken.
        {"name": "turnover step", "op": "turnover", "slots": 32, "ended": 2, "context": 2048, "spare": 1.25},
        # Half of a large pool's requests change, with prompts up to the longest sequence of the benchmarks.
        {"name": "turnover pool", "op": "turnover", "slots": 128, "ended": 64, "context": 100000, "spare": 1.0},
        # A small pool, a third of whose pages are free, before it is saved.
        {"name": "compact small", "op": "compact", "slots": 6, "context": 1000, "free": 0.33, "layers": 2, "kv_heads": 4,
         "dim": 64},
        # A pool of a serving process, half of it free.
        {"name": "compact pool", "op": "compact", "slots": 64, "context": 2048, "free": 0.5, "layers": 4, "kv_heads": 16,
         "dim": 64},
        # One user's four drafted tokens, taken from a lookup (no draft probabilities).
        {"name": "verify lookup", "op": "verify", "batch": 1, "tokens": 4, "vocab": 32000, "draft": False, "ragged": False},
        # A batch's drafts of a small model, of differing numbers.
        {"name": "verify batch", "op": "verify", "batch": 64, "tokens": 8, "vocab": 128000, "draft": True, "ragged": True},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("adapters", "adapters", "fork", "turnover", "compact", "verify"))
    if op == "adapters":
        inner, outer = 8 * _log(rng, 16, 1024), _log(rng, 64, 16384)
        tokens = 1 if rng.random() < 0.5 else _log(rng, 2, 2048)
        batch = max(1, min(_log(rng, 1, 256), 8 * 2048 * (1024 + 2 * 4096) // (tokens * (inner + 2 * outer))))
        return {"op": op, "batch": batch, "tokens": tokens, "inner": inner, "outer": outer,
                "rank": rng.choice((8, 16, 24, 32, 64, 72, 128)), "count": _log(rng, 1, 64), "gelu": rng.random() < 0.5,
                "base": rng.choice(("bf16", "f32")), "type": rng.choice(("bf16", "f32")),
                "spread": rng.choice(("sequences", "rows"))}
    heads = {"kv_heads": rng.choice((1, 2, 3, 4, 8, 16)), "dim": rng.choice((32, 64, 128, 256))}
    if op == "fork":
        layers = rng.randint(1, 8)
        most = 136 * 4 * 8 * 128 // (layers * heads["kv_heads"] * heads["dim"])  # slots whose tails are those of the largest
        slots = max(2, min(_log(rng, 2, 256), most))
        # the cache takes 5 GB at most
        room = int(5e9) // (slots * layers * heads["kv_heads"] * heads["dim"] * 2)
        return {"op": op, "slots": slots, "kept": rng.randint(1, slots - 1), "context": min(_log(rng, 10, 32000), room),
                "layers": layers, **heads}
    if op == "turnover":
        slots = _log(rng, 1, 256)
        context = min(_log(rng, 64, 100000), 128 * 100000 // slots)
        return {"op": op, "slots": slots, "ended": rng.randint(1, max(1, slots // 2)), "context": context,
                "spare": rng.choice((0.7, 1.0, 1.25, 2.0))}
    if op == "compact":
        layers, free = rng.randint(1, 8), rng.uniform(0.02, 0.8)
        pages = int(64 * 32 * 4 * 16 * 64 * (1 - free)) // (layers * heads["kv_heads"] * heads["dim"])
        context = min(_log(rng, 64, 32000), pages * BLOCK)
        slots = max(1, min(_log(rng, 1, 128), pages * BLOCK // context))
        return {"op": op, "slots": slots, "context": context, "free": free, "layers": layers, **heads}
    vocab, tokens = _log(rng, 500, 256000), rng.randint(1, 16)
    batch = max(1, min(_log(rng, 1, 256), 64 * 128000 // vocab))
    batch = max(1, min(batch, 2 * 64 * 9 * 128000 // (vocab * (tokens + 1))))
    return {"op": op, "batch": batch, "tokens": tokens, "vocab": vocab, "draft": rng.random() < 0.6,
            "ragged": rng.random() < 0.5}


# ------------------------------------------------------------------ inputs


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _rand(g, *shape):
    return torch.rand(*shape, generator=g, device="cuda")


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _lengths(g, count, context):
    """Lengths between a quarter of the context and all of it, the longest among them."""
    held = (context * (0.25 + 0.75 * _rand(g, count))).to(torch.int32).clamp_(1, context)
    held[0] = context
    return held


def _tables(g, lengths, max_blocks, pages):
    """Pages in a shuffled order for the full blocks of each slot; -1 past them."""
    full = (lengths // BLOCK).long()
    used = torch.arange(max_blocks, device="cuda") < full[:, None]
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    at = used.flatten().long().cumsum(0).view(used.shape) - 1
    return torch.where(used, order[at.clamp(0, pages - 1)], -1).to(torch.int32)


def _counted(table, pages):
    flat = table.flatten().long()
    held = flat >= 0
    return torch.zeros(pages, dtype=torch.int32, device="cuda").index_add_(0, flat.clamp_min(0), held.to(torch.int32))


def _prepare_adapters(case, state, g):
    rows, k, n, r, count = case["batch"] * case["tokens"], case["inner"], case["outer"], case["rank"], case["count"]
    state["x"] = _randn(g, case["batch"], case["tokens"], k).bfloat16()
    state["base"] = _randn(g, case["batch"], case["tokens"], n).to(TYPES[case["base"]])
    # trained adapters: the product is a fraction of the projection's output
    state["down"] = (_randn(g, count, r, k) * k ** -0.5).bfloat16()
    state["up"] = (_randn(g, count, n, r) * r ** -0.5).bfloat16()
    state["scales"] = 0.25 + _rand(g, count)
    many = rows if case["spread"] == "rows" else case["batch"]
    # one in eight without an adapter
    index = torch.randint(0, count, (many,), generator=g, device="cuda")
    none = _rand(g, many) < 0.125
    none[0] = False
    state["indices"] = torch.where(none, -1, index).to(torch.int32)
    if own:
        state["handle"] = _kernels().LowRankAdapters(state["down"], state["up"], state["scales"])


def _prepare_pages(case, state, g):
    op = case["op"]
    slots, layers = case["slots"], case.get("layers", 1)
    heads, dim = case.get("kv_heads", 1), case.get("dim", 32)
    max_blocks = -(-case["context"] // BLOCK) + 1
    if op == "turnover":
        # a page for every block of every slot, times what is spare
        pages = max(1, int(slots * max_blocks * case["spare"]))
        lengths = _lengths(g, slots, min(case["context"], int(case["spare"] * case["context"])))
        least = max(1, pages // slots) * BLOCK
        lengths = lengths.clamp_max(least)
        # of the pages' contents nothing is read here: the smallest heads stand for any
        codes = torch.zeros(layers, pages, 2, heads, BLOCK, dim, dtype=torch.uint8, device="cuda")
    elif op == "fork":
        lengths = _lengths(g, slots, case["context"])
        pages = slots * max_blocks
        # shared pages are neither read nor written
        codes = torch.empty(layers, pages, 2, heads, BLOCK, dim, dtype=torch.uint8, device="cuda")
    else:
        # of the pages, the lengths fill all but the free ones' share on average
        pages = max(slots, math.ceil(0.625 * slots * case["context"] / BLOCK / (1 - case["free"])))
        lengths = _lengths(g, slots, case["context"]).clamp_max(pages // slots * BLOCK + BLOCK - 1)
        codes = torch.randint(0, 256, (layers, pages, 2, heads, BLOCK, dim), generator=g, device="cuda", dtype=torch.uint8)
    cache = {
        "codes": codes,
        "scales": _rand(g, layers, pages, 2, heads) if op == "compact" else torch.zeros(layers, pages, 2, heads, device="cuda"),
        "tail": _randn(g, layers, slots, 2, 2, heads, BLOCK, dim).bfloat16() if op == "fork"
        else torch.zeros(layers, slots, 2, 2, heads, BLOCK, dim, dtype=torch.bfloat16, device="cuda"),
        "page_table": _tables(g, lengths, max_blocks, pages),
        "lengths": lengths,
    }
    # what is put back before each compaction lies together
    ints = torch.cat((_counted(cache["page_table"], pages), cache["page_table"].flatten()))
    state["ints"], state["saved"] = ints, ints.clone()
    state["refs"], cache["page_table"] = ints[:pages], ints[pages:].view(slots, max_blocks)
    state["cache"] = cache
    order = torch.randperm(slots, generator=g, device="cuda").to(torch.int32)
    if op == "fork":
        kept = order[:case["kept"]]
        state["target"] = order[case["kept"]:].contiguous()
        state["source"] = kept[torch.randint(0, case["kept"], (slots - case["kept"],), generator=g, device="cuda")]
    elif op == "turnover":
        state["slots"] = order[:case["ended"]].contiguous()
        state["counts"] = _lengths(g, case["ended"], case["context"])
    if own:
        kernels = _kernels()
        state["handle"] = kernels.Kv8Pages(kernels.Kv8Cache(**cache), state["refs"])


def _prepare_verify(case, state, g):
    batch, tokens, vocab = case["batch"], case["tokens"], case["vocab"]
    state["target"] = torch.empty(batch, tokens + 1, vocab, device="cuda")
    draft = torch.empty(batch, tokens, vocab, device="cuda")
    drafted = torch.empty(batch, tokens, dtype=torch.int64, device="cuda")
    for b in range(batch):  # a draft model's logits are near the target's
        logits = 2.5 * _randn(g, tokens + 1, vocab)
        state["target"][b] = torch.softmax(logits, -1)
        draft[b] = torch.softmax(logits[:-1] + 0.7 * _randn(g, tokens, vocab), -1)
        sums = draft[b].cumsum(-1)
        drafted[b] = (sums < _rand(g, tokens, 1) * sums[:, -1:]).sum(-1).clamp_max(vocab - 1)
    if not case["draft"]:  # a lookup is right most of the time: put its tokens where the target's mass is
        state["target"] *= 0.3
        state["target"][:, :-1].scatter_add_(2, drafted[..., None], torch.full((batch, tokens, 1), 0.7, device="cuda"))
    state["draft"] = draft if case["draft"] else None
    state["drafted"] = drafted
    state["uniform"] = _rand(g, batch, tokens + 1)
    state["counts"] = None
    if case["ragged"]:
        state["counts"] = torch.randint(0, tokens + 1, (batch,), generator=g, device="cuda", dtype=torch.int32)


def prepare(case, seed):
    g = _generator(seed)
    state = {"case": dict(case)}
    if case["op"] == "adapters":
        _prepare_adapters(case, state, g)
    elif case["op"] == "verify":
        _prepare_verify(case, state, g)
    else:
        _prepare_pages(case, state, g)
    return state


# ------------------------------------------------------------------ plain forms


def _adapters_plain(state):
    case = state["case"]
    x, base = state["x"].float().flatten(0, 1), state["base"].float().flatten(0, 1)
    count, rank, _ = state["down"].shape
    index = state["indices"]
    index = index.repeat_interleave(x.shape[0] // index.shape[0])
    mine = (index[:, None] == torch.arange(count, device="cuda")).float() * state["scales"]
    # every row against all adapters, of which the mask leaves its own
    h = x @ state["down"].float().flatten(0, 1).t()
    h = (h.view(-1, count, rank) * mine[..., None]).flatten(1)
    y = base + h @ state["up"].float().transpose(1, 2).flatten(0, 1)
    if case["gelu"]:
        y = 0.5 * y * (1 + torch.erf(y * 2 ** -0.5))
    return y.to(TYPES[case["type"]]).view(*state["base"].shape)


def _drop(refs, entries, sign):
    flat = entries.flatten().long()
    refs.index_add_(0, flat.clamp_min(0), (flat >= 0).to(torch.int32) * sign)


def _fork_plain(state):
    cache, refs = state["cache"], state["refs"]
    table, lengths, tail = cache["page_table"], cache["lengths"], cache["tail"]
    source, target = state["source"].long(), state["target"].long()
    held = lengths[source]
    full = held // BLOCK
    rows = torch.where(torch.arange(table.shape[1], device="cuda") < full[:, None], table[source], -1)
    _drop(refs, table[target], -1)
    _drop(refs, rows, 1)
    table[target] = rows
    open_rows = torch.arange(BLOCK, device="cuda") < (held % BLOCK)[:, None]
    parity = (full % 2).long()
    tail[:, target, parity] = torch.where(open_rows[:, None, None, :, None], tail[:, source, parity], tail[:, target, parity])
    lengths[target] = held
    return table, lengths, refs, tail


def _turnover_plain(state):
    cache, refs = state["cache"], state["refs"]
    table, lengths, slots = cache["page_table"], cache["lengths"], state["slots"].long()
    _drop(refs, table[slots], -1)
    table[slots] = -1
    lengths[slots] = 0
    block = torch.arange(table.shape[1], device="cuda")
    wanted = block < (state["counts"] // BLOCK)[:, None]
    free = refs == 0
    pages = torch.argsort((~free).to(torch.uint8), stable=True)  # the free ones in front, the lowest first
    at = wanted.flatten().long().cumsum(0).view(wanted.shape) - 1
    given = wanted & (at < free.sum())
    rows = torch.where(given, pages[at.clamp(0, pages.shape[0] - 1)].to(torch.int32), -1)
    table[slots] = rows
    _drop(refs, rows, 1)
    return table, lengths, refs, (wanted & ~given).sum(1).to(torch.int32)


def _compact_plain(state):
    cache, refs = state["cache"], state["refs"]
    used = refs > 0
    count = used.sum()
    low = torch.arange(refs.shape[0], device="cuda") < count
    to, of = (~used & low).nonzero()[:, 0], (used & ~low).nonzero()[:, 0]
    cache["codes"][:, to] = cache["codes"][:, of]
    cache["scales"][:, to] = cache["scales"][:, of]
    where = torch.arange(refs.shape[0], device="cuda", dtype=torch.int32)
    where[of] = to.to(torch.int32)
    table = cache["page_table"]
    table.copy_(torch.where(table >= 0, where[table.clamp_min(0).long()], -1))
    refs[to] = refs[of]
    refs[of] = 0
    return table, refs, count.to(torch.int32).view(1), cache["codes"], cache["scales"]


def _verify_plain(state):
    target, draft, drafted, uniform = state["target"], state["draft"], state["drafted"], state["uniform"].double()
    batch, tokens = drafted.shape
    counts = state["counts"] if state["counts"] is not None else torch.full((batch,), tokens, device="cuda", dtype=torch.int32)
    p = target[:, :-1].gather(2, drafted[..., None])[..., 0].double()
    q = draft.gather(2, drafted[..., None])[..., 0].double() if draft is not None else 1.0
    position = torch.arange(tokens, device="cuda")
    good = (uniform[:, :-1] * q < p) & (position < counts[:, None])
    accepted = good.long().cumprod(1).sum(1)
    rows = torch.arange(batch, device="cuda")
    mass = target[rows, accepted].double()
    refused = accepted < counts
    last = accepted.clamp_max(tokens - 1)
    if draft is not None:
        other = draft[rows, last].double()
    else:
        other = torch.zeros_like(mass).scatter_(1, drafted[rows, last][:, None], torch.inf)
    rest = torch.where(refused[:, None], (mass - other).clamp_min(0), mass)
    rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, mass)
    sums = rest.cumsum(-1)
    sampled = (sums > uniform[:, -1:] * sums[:, -1:]).to(torch.uint8).argmax(-1)
    place = torch.arange(tokens + 1, device="cuda")
    padded = torch.nn.functional.pad(drafted, (0, 1))
    out = torch.where(place < accepted[:, None], padded, -1)
    return torch.where(place == accepted[:, None], sampled[:, None], out), accepted.to(torch.int32)


def _run_own(state):
    case, kernels = state["case"], _kernels()
    op = case["op"]
    if op == "adapters":
        return kernels.sm100_low_rank_add(state["x"], state["base"], state["handle"], state["indices"], gelu=case["gelu"],
                                          out_dtype=TYPES[case["type"]])[0]
    if op == "verify":
        return kernels.sm100_verify_draft(state["target"], state["drafted"], state["uniform"], draft=state["draft"],
                                          counts=state["counts"])[:2]
    pages, cache = state["handle"], state["cache"]
    if op == "fork":
        kernels.sm100_kv8_fork(pages, state["source"], state["target"])
        return cache["page_table"], cache["lengths"], state["refs"], cache["tail"]
    if op == "turnover":
        kernels.sm100_kv8_free(pages, state["slots"])
        missing, _ = kernels.sm100_kv8_reserve(pages, case["context"], slots=state["slots"], counts=state["counts"])
        return cache["page_table"], cache["lengths"], state["refs"], missing
    state["ints"].copy_(state["saved"])
    used, _ = kernels.sm100_kv8_compact(pages)
    return cache["page_table"], state["refs"], used, cache["codes"], cache["scales"]


def run(state):
    with torch.no_grad():
        if own:
            return _run_own(state)
        op = state["case"]["op"]
        if op == "compact":
            state["ints"].copy_(state["saved"])
        return {"adapters": _adapters_plain, "fork": _fork_plain, "turnover": _turnover_plain, "compact": _compact_plain,
                "verify": _verify_plain}[op](state)


# ------------------------------------------------------------------ floor and 64-bit values


def work(case):
    op = case["op"]
    if op == "adapters":
        rows, k, n, r = case["batch"] * case["tokens"], case["inner"], case["outer"], case["rank"]
        # of `many` independent choices, one in eight none
        many = rows if case["spread"] == "rows" else case["batch"]
        used = case["count"] * (1 - (1 - 0.875 / case["count"]) ** many)
        size = {"bf16": 2, "f32": 4}
        bytes_ = 2 * rows * k + rows * n * (size[case["base"]] + size[case["type"]]) + 2 * used * r * (k + n)
        return {"bytes": bytes_, "flops": 2 * 0.875 * rows * r * (k + n)}
    if op == "verify":
        rows = case["batch"] * (1.6 if case["draft"] else 1)  # one of the target's, and of the draft's unless all count
        return {"bytes": 4 * rows * case["vocab"] + 24 * case["batch"] * case["tokens"], "flops": 2 * rows * case["vocab"]}
    blocks = 0.625 * case["context"] / BLOCK  # full blocks of a slot, on average
    if op == "fork":
        copies = case["slots"] - case["kept"]
        token = 4 * case["layers"] * case["kv_heads"] * case["dim"]
        return {"bytes": copies * (2 * 31.5 * token + 4 * 6 * blocks), "flops": 0}
    if op == "turnover":
        pages = case["slots"] * (case["context"] / BLOCK + 1) * case["spare"]
        return {"bytes": 4 * pages + case["ended"] * blocks * 4 * 6, "flops": 0}
    page = 2 * case["layers"] * case["kv_heads"] * (BLOCK * case["dim"] + 4)
    used = case["slots"] * blocks
    # each used page lies above the used ones' number with the free ones' share
    return {"bytes": 2 * used * case["free"] * page + 4 * used / (1 - case["free"]) + 8 * case["slots"] * blocks, "flops": 0}


def _exact_adapters(case, state):
    x, base = state["x"].double().flatten(0, 1), state["base"].double().flatten(0, 1)
    each = x.shape[0] // state["indices"].shape[0]
    y = base.clone()
    index = [i for i in state["indices"].tolist() for _ in range(each)]
    for a in sorted(set(index) - {-1}):
        rows = torch.tensor([r for r, i in enumerate(index) if i == a], device="cuda")
        delta = (x[rows] @ state["down"][a].double().t()) @ state["up"][a].double().t()
        y[rows] += delta * state["scales"][a].double()
    if case["gelu"]:
        y = y * torch.special.ndtr(y)
    return y.view(*state["base"].shape)


def _recount(table, pages):
    return np.bincount(table[table >= 0], minlength=pages).astype(np.int32)


def _exact_pages(case, state):
    cache = {k: v.clone() for k, v in state["cache"].items()}
    table, lengths = cache["page_table"].cpu().numpy(), cache["lengths"].cpu().numpy()
    pages = cache["codes"].shape[1]
    if case["op"] == "fork":
        before = cache["tail"].clone()
        for s, t in zip(state["source"].tolist(), state["target"].tolist()):
            full, rest = divmod(int(lengths[s]), BLOCK)
            table[t] = -1
            table[t, :full] = table[s, :full]
            lengths[t] = lengths[s]
            cache["tail"][:, t, full % 2, :, :, :rest] = before[:, s, full % 2, :, :, :rest]
        return table, lengths, _recount(table, pages), cache["tail"]
    if case["op"] == "turnover":
        slots, counts = state["slots"].tolist(), state["counts"].tolist()
        table[slots] = -1
        lengths[slots] = 0
        free = [int(p) for p in np.flatnonzero(_recount(table, pages) == 0)][::-1]
        missing = []
        for slot, n in zip(slots, counts):
            lacks = 0
            for block in range(n // BLOCK):
                if free:
                    table[slot, block] = free.pop()
                else:
                    lacks += 1
            missing.append(lacks)
        return table, lengths, _recount(table, pages), np.array(missing, dtype=np.int32)
    refs = _recount(table, pages)
    used = int((refs > 0).sum())
    low = 0
    for page in range(used, pages):
        if refs[page] == 0:
            continue
        while refs[low] != 0:
            low += 1
        cache["codes"][:, low] = cache["codes"][:, page]
        cache["scales"][:, low] = cache["scales"][:, page]
        table[table == page] = low
        refs[low], refs[page] = refs[page], 0
    return table, refs, np.array([used], dtype=np.int32), cache["codes"], cache["scales"]


def _exact_verify(case, state):
    drafted, uniform = state["drafted"].cpu().numpy(), state["uniform"].double().cpu().numpy()
    counts = [case["tokens"]] * case["batch"] if state["counts"] is None else state["counts"].tolist()
    out = np.full((case["batch"], case["tokens"] + 1), -1, dtype=np.int64)
    accepted = np.zeros(case["batch"], dtype=np.int32)
    for b, n in enumerate(counts):
        t = 0
        while t < n:
            token = drafted[b, t]
            q = 1.0 if state["draft"] is None else float(state["draft"][b, t, token])
            if not uniform[b, t] * q < float(state["target"][b, t, token]):
                break
            out[b, t] = token
            t += 1
        mass = state["target"][b, t].double().cpu().numpy()
        if t < n:
            rest = mass.copy()
            if state["draft"] is None:
                rest[drafted[b, t]] = 0
            else:
                rest = np.maximum(mass - state["draft"][b, t].double().cpu().numpy(), 0)
            mass = rest if rest.sum() > 0 else mass
        sums = np.cumsum(mass)
        out[b, t] = np.searchsorted(sums, uniform[b, -1] * sums[-1], side="right")
        accepted[b] = t
    return out, accepted


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "adapters":
        return _exact_adapters(case, state)
    if case["op"] == "verify":
        return _exact_verify(case, state)
    return _exact_pages(case, state)
