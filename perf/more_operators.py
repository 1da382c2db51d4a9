"""The operators of a decode step that verifies drafted tokens, as cases that can be timed: rotation and append of several new
tokens per sequence with the per-head norms of queries and keys, attention of a tree of drafted tokens over the paged cache, and
sampling of the next tokens from given random numbers.

``own`` False computes an operator's plain form in elementary torch operations, ``own`` True makes the calls a serving
loop makes: programs of a ``ChipWorker``, registered once, on device-resident tensors.  ``listed()`` holds named cases over
the range in use, ``draw(rng)`` gives further ones, ``exact`` restates the definitions in 64 bits.
"""

from __future__ import annotations

import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "e4m3": torch.float8_e4m3fn}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4, "e4m3": 1}
_EPS = 1e-6
_TOP = 448.0  # the largest e4m3 value
_LEAST = 2.0 ** -25  # a random number below it counts as it

# What a serving process keeps: one worker, and each program registered once.
_worker = None
_handles: dict = {}


def _call(program: str, *args) -> None:
    global _worker
    from pypto_amd import runtime

    if _worker is None:
        _worker = runtime.ChipWorker(runtime.RunConfig(platform="mi355x", device_id=0))
    if program not in _handles:
        _handles[program] = _worker.register(getattr(runtime, program))
    _handles[program](*args, stream=torch.cuda.current_stream().cuda_stream)


def listed() -> list[dict]:
    return [
        # one user, no drafts: one new token's heads are normed, rotated and appended
        {"name": "append_one_token", "kind": "append", "batch": 1, "n_lo": 1, "n_hi": 1, "ctx_lo": 4096, "ctx_hi": 4096, "hq": 32, "hkv": 8, "d": 128,
         "block": 128, "qkv": "bf16", "cache": "bf16", "norm": True},
        # a serving batch, a few drafted tokens for each sequence, fp32 sums of the projection in front
        {"name": "append_tree_batch_16", "kind": "append", "batch": 16, "n_lo": 3, "n_hi": 48, "ctx_lo": 512, "ctx_hi": 4096, "hq": 32, "hkv": 8, "d": 128,
         "block": 128, "qkv": "fp32", "cache": "bf16", "norm": True},
        # the same over e4m3 caches: blocks whose scale grows are coded again
        {"name": "append_tree_fp8_32", "kind": "append", "batch": 32, "n_lo": 1, "n_hi": 24, "ctx_lo": 64, "ctx_hi": 2048, "hq": 64, "hkv": 8, "d": 128,
         "block": 64, "qkv": "bf16", "cache": "e4m3", "norm": True},
        # prompts of several users, appended at once, without the norms
        {"name": "append_prompts_4", "kind": "append", "batch": 4, "n_lo": 1500, "n_hi": 4500, "ctx_lo": 0, "ctx_hi": 700, "hq": 40, "hkv": 8, "d": 128,
         "block": 128, "qkv": "fp16", "cache": "fp16", "norm": False},
        # one user with sixteen drafts
        {"name": "tree_one_sequence", "kind": "tree", "batch": 1, "n_lo": 16, "n_hi": 16, "ctx_lo": 4096, "ctx_hi": 4096, "hq": 32, "hkv": 8, "d": 128,
         "block": 128, "q": "bf16", "cache": "bf16"},
        # a ragged serving batch: some sequences without drafts, some with many
        {"name": "tree_batch_16", "kind": "tree", "batch": 16, "n_lo": 1, "n_hi": 40, "ctx_lo": 512, "ctx_hi": 4096, "hq": 32, "hkv": 8, "d": 128,
         "block": 128, "q": "bf16", "cache": "bf16"},
        # e4m3 caches of many users with a short chain of drafts each
        {"name": "tree_fp8_batch_32", "kind": "tree", "batch": 32, "n_lo": 4, "n_hi": 8, "ctx_lo": 2000, "ctx_hi": 16000, "hq": 64, "hkv": 8, "d": 128,
         "block": 64, "q": "fp16", "cache": "e4m3"},
        # wide heads and large trees over long contexts: the products bound it
        {"name": "tree_long_64_drafts", "kind": "tree", "batch": 4, "n_lo": 64, "n_hi": 64, "ctx_lo": 20000, "ctx_hi": 32000, "hq": 64, "hkv": 8, "d": 128,
         "block": 64, "q": "fp16", "cache": "fp16"},
        # one user's next token
        {"name": "sample_one_token", "kind": "sample", "rows": 1, "vocab": 151936, "dtype": "bf16", "mode": "top_p"},
        # a serving batch in which every request has filters of its own
        {"name": "sample_batch_64", "kind": "sample", "rows": 64, "vocab": 151936, "dtype": "fp32", "mode": "mixed"},
        # a token for every node of the batch's trees, from the whole distribution
        {"name": "sample_tree_nodes_320", "kind": "sample", "rows": 320, "vocab": 32000, "dtype": "fp16", "mode": "plain"},
        # the same for large trees and a large vocabulary
        {"name": "sample_tree_nodes_500", "kind": "sample", "rows": 500, "vocab": 128000, "dtype": "fp32", "mode": "mixed"},
    ]


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    """Spread over the logarithm of [lo, hi]."""
    return min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))


def draw(rng: random.Random) -> dict:
    most = max(_cost(c) for c in listed())
    while True:
        kind = rng.choice(("append", "tree", "sample"))
        half = rng.choice(("bf16", "fp16"))
        hkv = rng.choice((1, 2, 4, 8, 8, 10))
        hq = hkv * rng.choice((1, 2, 4, 5, 8))
        n_hi = _log_int(rng, 1, 64)
        case = {"kind": kind, "batch": _log_int(rng, 1, 64), "n_lo": rng.randint(1, n_hi), "n_hi": n_hi}
        case["ctx_lo"] = rng.choice((0, 1, _log_int(rng, 1, 4000)))
        case["ctx_hi"] = case["ctx_lo"] + _log_int(rng, 1, 12000)
        case |= {"hq": hq, "hkv": hkv, "d": rng.choice((64, 128, 128, 128, 256)), "block": rng.choice((16, 32, 64, 128))}
        if kind == "append":
            if rng.random() < 0.3:  # prompts
                case |= {"batch": rng.randint(1, 6), "n_lo": _log_int(rng, 64, 2000), "n_hi": _log_int(rng, 2000, 5000)}
            case |= {"qkv": rng.choice((half, half, "fp32")), "cache": rng.choice((half, half, "e4m3")), "norm": rng.random() < 0.7}
        elif kind == "tree":
            case |= {"q": half, "cache": rng.choice((half, half, "e4m3"))}
            if case["cache"] == "e4m3" and case["block"] < 32:
                continue
        else:
            case = {"kind": kind, "rows": _log_int(rng, 1, 512), "vocab": _log_int(rng, 1000, 200000), "dtype": rng.choice((half, half, "fp32")),
                    "mode": rng.choice(("greedy", "plain", "top_k", "top_p", "min_p", "mixed", "mixed"))}
        if _cost(case) <= most and (kind == "sample" or _pool(case) * hkv * case["block"] * case["d"] <= 3e8):
            return case


def _cost(case: dict) -> float:
    w = work(case)
    return max(w["bytes"] / 4e12, w["flops"] / 1e15)


def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """Tokens in the cache and new tokens of every sequence: spread evenly over their ranges, long contexts with any number of new tokens."""
    batch = case["batch"]
    spread = lambda lo, hi: [lo + (hi - lo) * b // max(1, batch - 1) for b in range(batch)] if batch > 1 else [hi]
    ctx, new = spread(case["ctx_lo"], case["ctx_hi"]), spread(case["n_lo"], case["n_hi"])
    random.Random(batch).shuffle(new)
    return ctx, new


def _pool(case: dict) -> int:
    """Blocks of the cache: what the sequences hold, and a few that nobody has."""
    return sum(-(-(c + n) // case["block"]) for c, n in zip(*_lengths(case))) + 3


def work(case: dict) -> dict:
    """Bytes and arithmetic of one pass: every input read once, every output written once."""
    kind = case["kind"]
    if kind == "sample":
        rows, vocab = case["rows"], case["vocab"]
        return {"bytes": rows * (vocab * _SIZE[case["dtype"]] + 28), "flops": 12 * rows * vocab}
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    ctx, new = _lengths(case)
    t = sum(new)
    if kind == "append":
        moved = (hq + 2 * hkv) * d * _SIZE[case["qkv"]] + hq * d * 2 + 2 * hkv * d * _SIZE[case["cache"]] + 4 * d
        return {"bytes": t * moved + 8 * case["batch"], "flops": t * (hq + 2 * hkv) * d * 8}
    keys = sum(c + n for c, n in zip(ctx, new))
    pairs = sum(n * c + n * (n + 1) // 2 for c, n in zip(ctx, new))
    return {"bytes": 2 * keys * hkv * d * _SIZE[case["cache"]] + t * hq * d * 4, "flops": 4 * pairs * hq * d}


# ---- inputs ------------------------------------------------------------------------------------------


def _drafts(new: list[int], rng: random.Random) -> tuple[list[int], list[list[int]]]:
    """A random tree for every sequence: the depth of each of its nodes, and the nodes that it sees (its ancestors and itself) as bits."""
    depths, masks, words = [], [], -(-max(new) // 32)
    for n in new:
        depth, sees = [0], [1]
        for i in range(1, n):
            parent = max(0, i - 1 - int(rng.expovariate(0.5)))
            depth.append(depth[parent] + 1)
            sees.append(sees[parent] | 1 << i)
        depths += depth
        masks += [[(m >> 32 * w & 0xFFFFFFFF) - (m >> 32 * w + 31 & 1) * (1 << 32) for w in range(words)] for m in sees]
    return depths, masks


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    normal = lambda *shape: torch.randn(shape, device="cuda", generator=g)
    uniform = lambda *shape: torch.rand(shape, device="cuda", generator=g)
    empty = lambda shape, dtype: torch.empty(shape, dtype=dtype, device="cuda")
    ints = lambda values: torch.tensor(values, dtype=torch.int32, device="cuda")
    kind, s = case["kind"], {"case": case}
    if kind == "sample":
        rows, vocab, mode = case["rows"], case["vocab"], case["mode"]
        # most of the mass on some tens of tokens, the rest in a long tail; some rows are flatter than others
        logits = normal(rows, vocab) * (1.5 + uniform(rows, 1))
        hot = torch.randint(0, vocab, (rows, 40), device="cuda", generator=g)
        logits.scatter_add_(1, hot, 6 + 4 * uniform(rows, 40))
        s["logits"] = logits.to(_DTYPES[case["dtype"]])
        which = torch.arange(rows, device="cuda") % 4 if mode == "mixed" else None
        some = lambda name, i: mode == name or (which == i if mode == "mixed" else torch.zeros(rows, dtype=torch.bool, device="cuda"))
        pick = lambda at, value, off: torch.where(torch.as_tensor(at, device="cuda").expand(rows), value, off)
        temperature = 0.6 + 0.7 * uniform(rows)
        s["temperature"] = torch.zeros_like(temperature) if mode == "greedy" else temperature
        if mode == "mixed" and rows > 8:
            s["temperature"][5] = 0.0
        k = torch.randint(1, 200, (rows,), device="cuda", generator=g, dtype=torch.int32)
        s["top_k"] = pick(some("top_k", 0), k, torch.zeros_like(k))
        s["top_p"] = pick(some("top_p", 1), 0.5 + 0.49 * uniform(rows), torch.ones(rows, device="cuda"))
        s["min_p"] = pick(some("min_p", 2), 0.01 + 0.1 * uniform(rows), torch.zeros(rows, device="cuda"))
        s["uniform"] = uniform(rows)
        s["tokens"], s["probs"] = empty((rows,), torch.int32), empty((rows,), torch.float32)
        return s
    hq, hkv, d, block = case["hq"], case["hkv"], case["d"], case["block"]
    ctx, new = _lengths(case)
    order = list(range(case["batch"]))
    rng.shuffle(order)
    ctx, new = [ctx[b] for b in order], [new[b] for b in order]
    t, pool = sum(new), _pool(case)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    s["starts"], s["ctx"] = ints(starts), ints(ctx)
    free = list(range(pool))
    rng.shuffle(free)
    width = max(-(-(c + n) // block) for c, n in zip(ctx, new)) + 1
    table = []
    for c, n in zip(ctx, new):
        used = -(-(c + n) // block)
        table.append(free[:used] + [-1] * (width - used))
        free = free[used:]
    s["table"] = ints(table)
    cache = _DTYPES[case["cache"]]
    rows = pool * hkv * block
    if cache == torch.float8_e4m3fn:
        for name in ("key", "value"):
            s[name] = (normal(rows, d) * 100).clamp(-_TOP, _TOP).to(cache)
            s[name[0] + "_scale"] = (0.006 + 0.004 * uniform(pool, hkv)).contiguous()
    else:
        s["key"], s["value"] = normal(rows, d).to(cache), normal(rows, d).to(cache)
    prompts = max(new) > 256
    depths, masks = ([i for n in new for i in range(n)], None) if prompts else _drafts(new, rng)
    if kind == "append":
        half = case["cache"] if case["cache"] != "e4m3" else case["qkv"] if case["qkv"] != "fp32" else "bf16"
        s["positions"] = ints([c + depths[starts[b] + i] for b, (c, n) in enumerate(zip(ctx, new)) for i in range(n)])
        angle = torch.arange(max(c + n for c, n in zip(ctx, new)) + 1, dtype=torch.float64, device="cuda")[:, None] \
            * 1e6 ** (-torch.arange(d // 2, dtype=torch.float64, device="cuda") * 2 / d)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        if case["norm"]:
            s["gamma_q"], s["gamma_k"] = 1 + 0.2 * normal(d), 1 + 0.2 * normal(d)
        s["qkv"] = normal(t, (hq + 2 * hkv) * d).to(_DTYPES[case["qkv"]])
        s["q_out"] = empty((t * hq, d), _DTYPES[half])
    else:
        s["mask"] = ints(masks)
        s["q"] = (1.5 * normal(t * hq, d)).to(_DTYPES[case["q"]])
        s["out"] = empty((t * hq, d), _DTYPES[case["q"]])
    return s


# ---- one pass ----------------------------------------------------------------------------------------


def run(s: dict):
    return {"append": _append, "tree": _tree, "sample": _sample}[s["case"]["kind"]](s)


def _places(s: dict) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """Of every new token: its sequence, its number in that, its block and its place in the block."""
    starts = s["starts"].long()
    token = torch.arange(len(s["positions"]) if "positions" in s else len(s["mask"]), device="cuda")
    seq = torch.searchsorted(starts, token, right=True) - 1
    number = token - starts[seq]
    index = s["ctx"].long()[seq] + number
    block = s["case"]["block"]
    return seq, number, s["table"].long()[seq, index // block], index % block


def _append(s: dict):
    case = s["case"]
    hq, hkv, d, block = case["hq"], case["hkv"], case["d"], case["block"]
    fp8 = case["cache"] == "e4m3"
    out = {"q": s["q_out"], "key": s["key"], "value": s["value"]} | ({"k_scale": s["k_scale"], "v_scale": s["v_scale"]} if fp8 else {})
    if own:
        _call("rope_append_tokens" + ("_fp8" if fp8 else "") + ("_normed" if case["norm"] else ""), s["qkv"], s["positions"], s["starts"], s["ctx"],
              s["cos"], s["sin"], *((s["gamma_q"], s["gamma_k"]) if case["norm"] else ()), s["table"], s["key"], s["value"],
              *((s["k_scale"], s["v_scale"]) if fp8 else ()), s["q_out"], hq, hkv, d, block, *((_EPS,) if case["norm"] else ()))
        return out
    x = s["qkv"].float().view(-1, hq + 2 * hkv, d)
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    if case["norm"]:
        q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + _EPS) * s["gamma_q"]
        k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + _EPS) * s["gamma_k"]
    cos, sin = s["cos"][s["positions"].long()][:, None], s["sin"][s["positions"].long()][:, None]
    turned = lambda y: torch.cat((y[..., :d // 2] * cos - y[..., d // 2:] * sin, y[..., d // 2:] * cos + y[..., :d // 2] * sin), -1)
    s["q_out"].copy_(turned(q).reshape(-1, d).to(s["q_out"].dtype))
    _, number, blk, place = _places(s)
    heads = torch.arange(hkv, device="cuda")
    first = torch.full((len(s["key"]) // (hkv * block),), block, device="cuda").scatter_reduce(0, blk, place, "amin")  # of each block's new rows
    for name, y in (("key", turned(k)), ("value", v)):
        rows = s[name].view(-1, hkv, block, d)
        if fp8:
            scale = s[name[0] + "_scale"]
            most = torch.zeros_like(scale).scatter_reduce(0, blk[:, None].expand(-1, hkv), y.abs().amax(-1), "amax") / _TOP
            fresh = torch.where(most > 0, most, 1.0)
            touched, begun = (first < block)[:, None], (first > 0)[:, None]
            after = torch.where(touched, torch.where(begun, torch.maximum(scale, most), fresh), scale)
            again = torch.unique(blk)  # its rows of before in the new scale
            old = rows[again].float() * scale[again][:, :, None, None] / after[again][:, :, None, None]
            keep = (after[again] == scale[again])[:, :, None, None] | (torch.arange(block, device="cuda") >= first[again][:, None])[:, None, :, None]
            rows[again] = torch.where(keep, rows[again].float(), old.clamp(-_TOP, _TOP)).to(rows.dtype)
            scale.copy_(after)
            y = (y / scale[blk][:, :, None]).clamp(-_TOP, _TOP)
        rows[blk[:, None], heads, place[:, None]] = y.to(rows.dtype)
    return out


def _tree(s: dict):
    case = s["case"]
    hq, hkv, d, block = case["hq"], case["hkv"], case["d"], case["block"]
    fp8 = case["cache"] == "e4m3"
    if own:
        _call("tree_attention", s["q"], s["key"], s["value"], s["table"], s["ctx"], s["starts"], s["mask"], s["out"],
              *((s["k_scale"], s["v_scale"]) if fp8 else ()), hq, hkv, d, block, d ** -0.5)
        return s["out"]
    # every sequence's rows and keys side by side, as many for each as the largest one has
    batch, group = case["batch"], hq // hkv
    seq, number, _, _ = _places(s)
    new = s["starts"][1:] - s["starts"][:-1]
    longest, most = s["table"].shape[1] * block, s["mask"].shape[1] * 32
    at = torch.arange(longest, device="cuda")
    blk = s["table"].long()[:, at // block].clamp(min=0)
    gather = lambda c: c.view(-1, hkv, block, d)[blk, :, at % block].float()
    keys, values = gather(s["key"]), gather(s["value"])
    if fp8:
        keys, values = keys * s["k_scale"][blk][..., None], values * s["v_scale"][blk][..., None]
    there = at < (s["ctx"] + new)[:, None]
    values = torch.where(there[:, :, None, None], values, 0.0)
    queries = torch.zeros((batch, most, hkv, group, d), device="cuda")
    queries[seq, number] = s["q"].float().view(-1, hkv, group, d)
    queries = queries.permute(0, 2, 1, 3, 4).reshape(batch, hkv, most * group, d)
    bits = (s["mask"][:, :, None] >> torch.arange(32, dtype=torch.int32, device="cuda") & 1).flatten(1).bool()
    node = at - s["ctx"][:, None]
    sees = torch.zeros((batch, most, most), dtype=torch.bool, device="cuda")
    sees[seq, number] = bits
    in_tree = ((node >= 0) & (node < new[:, None]))[:, None] & sees.gather(2, node.clamp(0, most - 1).long()[:, None].expand(-1, most, -1))
    sees = (node < 0)[:, None] | in_tree
    scores = (queries @ keys.permute(0, 2, 3, 1).contiguous()).mul_(d ** -0.5).view(batch, hkv, most, group, longest)
    scores.masked_fill_(~sees[:, None, :, None], -torch.inf)
    top = scores.amax(-1, keepdim=True)
    power = scores.sub_(torch.where(top == -torch.inf, 0.0, top)).exp_()
    total = power.sum(-1, keepdim=True)
    y = power.view(batch, hkv, -1, longest) @ values.permute(0, 2, 1, 3).contiguous()
    y = y.view(batch, hkv, most, group, d) / torch.where(total > 0, total, 1.0)
    return y.permute(0, 2, 1, 3, 4)[seq, number].reshape(-1, d).to(s["out"].dtype)


def _sample(s: dict):
    if own:
        _call("sample_tokens", s["logits"], s["temperature"], s["top_k"], s["top_p"], s["min_p"], s["uniform"], s["tokens"], s["probs"])
        return {"tokens": s["tokens"], "probs": s["probs"]}
    # in 64 bits: a random number or a filter's border may lie next to the sum of any of the tokens in front
    logits = s["logits"].double()
    greedy = ~(s["temperature"] > 0)
    power = ((logits - logits.amax(-1, keepdim=True)) / torch.where(greedy, 1.0, s["temperature"])[:, None].double()).exp()
    order = logits.sort(dim=-1, descending=True, stable=True).indices
    rank = torch.arange(logits.shape[1], device="cuda")
    k = torch.where(s["top_k"] > 0, s["top_k"], logits.shape[1])
    by_rank = power.gather(1, order)
    by_rank = torch.where(rank < torch.where(greedy, 1, k)[:, None], by_rank, 0.0)
    in_front = by_rank.cumsum(-1)
    kept = (in_front - by_rank < s["top_p"].double()[:, None] * in_front[:, -1:]) | (s["top_p"] >= 1)[:, None]
    by_rank = torch.where(kept & (by_rank >= s["min_p"].double().clamp(max=1.0)[:, None]), by_rank, 0.0)
    weight = torch.zeros_like(power).scatter_(1, order, by_rank)
    sums = weight.cumsum(-1)
    token = (sums > s["uniform"].double().clamp(min=_LEAST)[:, None] * sums[:, -1:]).int().argmax(-1)
    probs = weight.gather(1, token[:, None]).squeeze(1) / weight.sum(-1)
    return {"tokens": token.to(torch.int32), "probs": probs.float()}


# ---- the definitions in 64 bits ------------------------------------------------------------------------


def _e4m3(v: torch.Tensor) -> torch.Tensor:
    """The e4m3 value nearest to each 64-bit value, ties to even: three bits behind the leading one, steps of 2^-9 below 2^-6."""
    exponent = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(exponent - 3)
    return (torch.round(v / step) * step).clamp(-_TOP, _TOP)


def _exact_append(case: dict, s: dict) -> dict:
    hq, hkv, d, block = case["hq"], case["hkv"], case["d"], case["block"]
    x = s["qkv"].double().reshape(-1, hq + 2 * hkv, d)
    if case["norm"]:
        size = torch.sqrt(x.square().sum(-1, keepdim=True) / d + _EPS)
        x = torch.cat((x[:, :hq] / size[:, :hq] * s["gamma_q"].double(), x[:, hq:-hkv] / size[:, hq:-hkv] * s["gamma_k"].double(), x[:, -hkv:]), 1)
    at = s["positions"].long()
    turn = torch.complex(s["cos"][at].double(), s["sin"][at].double())[:, None]
    y = torch.complex(x[..., :d // 2], x[..., d // 2:])[:, :-hkv] * turn
    y = torch.cat((y.real, y.imag), -1)
    out = {"q": y[:, :hq].reshape(-1, d)}
    starts, ctx, table = s["starts"].tolist(), s["ctx"].tolist(), s["table"].tolist()
    for name, rows in (("key", y[:, hq:]), ("value", x[:, -hkv:])):
        held = s[name].double().view(-1, hkv, block, d)
        scales = s[name[0] + "_scale"].double() if case["cache"] == "e4m3" else None
        for b, c in enumerate(ctx):
            first, last = c, c + starts[b + 1] - starts[b]
            while first < last:  # the new rows of one block
                stop = min(last, (first // block + 1) * block)
                blk, place = table[b][first // block], first % block
                fresh = rows[starts[b] + first - c:starts[b] + stop - c].transpose(0, 1)
                if scales is not None:
                    need = fresh.abs().amax((1, 2)) / _TOP
                    scale = torch.where(need > 0, need, 1.0) if place == 0 else torch.maximum(scales[blk], need)
                    if place:
                        again = _e4m3(held[blk, :, :place] * (scales[blk] / scale)[:, None, None])
                        held[blk, :, :place] = torch.where((scale > scales[blk])[:, None, None], again, held[blk, :, :place])
                    scales[blk] = scale
                    fresh = _e4m3(fresh / scale[:, None, None])
                held[blk, :, place:place + stop - first] = fresh
                first = stop
        out[name] = held.view(-1, d)
        if scales is not None:
            out[name[0] + "_scale"] = scales
    return out


def _exact_tree(case: dict, s: dict):
    hq, hkv, d, block = case["hq"], case["hkv"], case["d"], case["block"]
    group = hq // hkv
    starts, ctx, table = s["starts"].tolist(), s["ctx"].tolist(), s["table"].tolist()
    q = s["q"].view(-1, hkv, group, d)
    out = torch.zeros((len(q), hkv, group, d), dtype=torch.float64, device="cuda")
    for b, c in enumerate(ctx):
        n = starts[b + 1] - starts[b]
        words = s["mask"][starts[b]:starts[b + 1]].tolist()
        hidden = torch.zeros((n, c + n), dtype=torch.bool, device="cuda")
        hidden[:, c:] = torch.tensor([[not words[i][j // 32] >> j % 32 & 1 for j in range(n)] for i in range(n)], device="cuda")
        blocks = table[b][:-(-(c + n) // block)]
        for h in range(hkv):
            k, v = (s[name].view(-1, hkv, block, d)[blocks, h].double() for name in ("key", "value"))
            if case["cache"] == "e4m3":
                k, v = k * s["k_scale"][blocks, h].double()[:, None, None], v * s["v_scale"][blocks, h].double()[:, None, None]
            k, v = k.reshape(-1, d)[:c + n], v.reshape(-1, d)[:c + n]
            score = q[starts[b]:starts[b + 1], h].double().reshape(n * group, d) @ k.t() / d ** 0.5
            score = score.masked_fill(torch.repeat_interleave(hidden, group, 0), -torch.inf)
            out[starts[b]:starts[b + 1], h] = (torch.softmax(score, -1) @ v).view(n, group, d)
    return out.view(-1, d)


def _exact_sample(case: dict, s: dict) -> dict:
    tokens, probs = [], []
    rows = zip(s["logits"], *(s[name].tolist() for name in ("temperature", "top_k", "top_p", "min_p", "uniform")))
    for logits, temperature, k, p, least, u in rows:
        logits = logits.double()
        # tokens from the best on; of equal ones the first
        order = torch.argsort(logits, descending=True, stable=True)
        if temperature <= 0:
            tokens.append(order[0])
            probs.append(torch.ones((), dtype=torch.float64, device="cuda"))
            continue
        order = order[:k] if k > 0 else order
        share = torch.softmax(logits[order] / temperature, 0)
        if p < 1:  # the fewest whose sum reaches p
            order = order[:int((share.cumsum(0) < p).sum()) + 1]
        share = share[:len(order)]
        order = order[share / share[0] >= least]
        order = order.sort().values
        share = torch.softmax(logits[order] / temperature, 0)
        sums = share.cumsum(0)
        at = int((sums <= max(u, _LEAST) * sums[-1]).sum())
        tokens.append(order[at])
        probs.append(share[at])
    return {"tokens": torch.stack(tokens).to(torch.int32), "probs": torch.stack(probs)}


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    return {"append": _exact_append, "tree": _exact_tree, "sample": _exact_sample}[case["kind"]](case, s)
