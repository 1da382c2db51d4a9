"""The operators of a feed-forward layer of experts on block-scaled e4m3 operands, as cases that can be timed: RMSNorm with
the residual's addition and e4m3 output, the block-scaled matrix product, the router and the experts' FFN.

``own`` False computes an operator's plain form in elementary torch operations, ``own`` True makes the calls a serving
loop makes: programs of a ``ChipWorker``, registered once, on device-resident tensors.  ``listed()`` holds named cases over
the range in use, ``draw(rng)`` gives further ones, ``exact`` restates the definitions in 64 bits.
"""

from __future__ import annotations

import random

import torch
import torch.nn.functional as F

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_F8 = torch.float8_e4m3fn
_BLOCK = 128  # elements of a row that share a scale; a weight's scale covers as many of its rows
_EPS = 1e-6

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
        # one user waiting for the next token: the launch and one row's round trips are all of it
        {"name": "norm_one_token", "kind": "norm", "rows": 1, "cols": 4096, "dtype": "bf16", "residual": True, "normed": True},
        # the rest of a chunked prompt riding with a decode batch, in front of a dense projection (no 16-bit output wanted)
        {"name": "norm_mixed_batch_333", "kind": "norm", "rows": 333, "cols": 5120, "dtype": "fp16", "residual": True, "normed": False},
        # prefill of long prompts in a wide model, in front of router and experts
        {"name": "norm_prefill_4096", "kind": "norm", "rows": 4096, "cols": 8192, "dtype": "bf16", "residual": True, "normed": True},
        # q, k and v of one new token
        {"name": "product_one_token", "kind": "product", "m": 1, "k": 4096, "n": 6144, "out": "fp32"},
        # a serving batch, one token each: bound by reading the weights
        {"name": "product_batch_48", "kind": "product", "m": 48, "k": 4096, "n": 14336, "out": "fp16"},
        # some hundred tokens against an output width that is no multiple of anything
        {"name": "product_mixed_333", "kind": "product", "m": 333, "k": 5120, "n": 5003, "out": "bf16"},
        # prefill of a prompt (the FFN benchmark's widths)
        {"name": "product_prefill_2048", "kind": "product", "m": 2048, "k": 4096, "n": 11008, "out": "bf16"},
        # the router of one new token
        {"name": "route_one_token", "kind": "route", "tokens": 1, "experts": 64, "top_k": 6, "groups": 1, "kept": 1, "score": "softmax",
         "bias": False, "renormalize": True, "dtype": "fp32"},
        # the router of a prompt, many experts in groups, balanced by a bias
        {"name": "route_prefill_4096", "kind": "route", "tokens": 4096, "experts": 256, "top_k": 8, "groups": 8, "kept": 4, "score": "sigmoid",
         "bias": True, "renormalize": True, "dtype": "fp32"},
        # the experts of one new token
        {"name": "experts_one_token", "kind": "experts", "tokens": 1, "hidden": 4096, "inter": 1408, "experts": 64, "top_k": 8, "out": "bf16"},
        # a serving batch that reaches most experts with a few rows each
        {"name": "experts_batch_40", "kind": "experts", "tokens": 40, "hidden": 2048, "inter": 1024, "experts": 60, "top_k": 4, "out": "fp16"},
        # prefill of a prompt
        {"name": "experts_prefill_2048", "kind": "experts", "tokens": 2048, "hidden": 4096, "inter": 1408, "experts": 64, "top_k": 8, "out": "bf16"},
    ]


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    """Spread over the logarithm of [lo, hi]."""
    return min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))


def draw(rng: random.Random) -> dict:
    most = max(_cost(c) for c in listed())
    while True:
        kind = rng.choice(("norm", "product", "route", "experts"))
        half = rng.choice(("bf16", "fp16"))
        if kind == "norm":
            case = {"kind": kind, "rows": _log_int(rng, 1, 8192), "cols": _log_int(rng, 512, 16384) // 8 * 8, "dtype": half,
                    "residual": rng.random() < 0.75, "normed": rng.random() < 0.5}
        elif kind == "product":
            case = {"kind": kind, "m": _log_int(rng, 1, 4096), "k": _log_int(rng, 4, 128) * _BLOCK, "n": _log_int(rng, 64, 20000),
                    "out": rng.choice((half, half, "fp32"))}
        elif kind == "route":
            groups, size = rng.choice(((1, 8), (1, 60), (1, 128), (1, 384), (4, 16), (8, 20), (8, 32)))
            kept = rng.randint(max(1, groups // 4), groups)
            case = {"kind": kind, "tokens": _log_int(rng, 1, 16384), "experts": groups * size, "top_k": rng.randint(1, min(8, kept * size)),
                    "groups": groups, "kept": kept, "score": rng.choice(("softmax", "sigmoid")), "bias": rng.random() < 0.5,
                    "renormalize": rng.random() < 0.75, "dtype": rng.choice(("fp32", "fp32", "bf16", "fp16"))}
        else:
            experts = rng.choice((8, 16, 32, 60, 64, 128))
            case = {"kind": kind, "tokens": _log_int(rng, 1, 4096), "hidden": _log_int(rng, 4, 40) * _BLOCK, "inter": _log_int(rng, 2, 32) * _BLOCK,
                    "experts": experts, "top_k": rng.randint(1, 8), "out": half}
            if experts * case["hidden"] * case["inter"] > 64 * 4096 * 1408:
                continue
        if _cost(case) <= most:
            return case


def _cost(case: dict) -> float:
    w = work(case)
    return max(w["bytes"] / 4e12, w["flops"] / 1e15)


def work(case: dict) -> dict:
    """Bytes and arithmetic of one pass: every input read once (of the experts those that a token uses), every output written once."""
    kind = case["kind"]
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    if kind == "norm":
        rows, cols = case["rows"], case["cols"]
        sixteen = 1 + 2 * case["residual"] + case["normed"]  # x; residual and sum; normed
        return {"bytes": rows * (cols * (2 * sixteen + 1) + 4 * -(-cols // _BLOCK)) + 4 * cols, "flops": 8 * rows * cols}
    if kind == "product":
        m, k, n = case["m"], case["k"], case["n"]
        scales = 4 * (k // _BLOCK) * (m + -(-n // _BLOCK))
        return {"bytes": (m + n) * k + scales + m * n * size[case["out"]], "flops": 2 * m * k * n}
    if kind == "route":
        t, e = case["tokens"], case["experts"]
        return {"bytes": t * (e * size[case["dtype"]] + case["top_k"] * 8) + 4 * e * case["bias"], "flops": 10 * t * e}
    t, h, i, e, top = case["tokens"], case["hidden"], case["inter"], case["experts"], case["top_k"]
    used = e * (1 - (1 - top / e) ** t)
    return {"bytes": int(used * 3 * h * i * (1 + 4 / _BLOCK ** 2)) + t * (h * (1 + 4 / _BLOCK + size[case["out"]]) + top * 8),
            "flops": 6 * t * top * h * i}


# ---- inputs ------------------------------------------------------------------------------------------


def _groups(v: torch.Tensor) -> torch.Tensor:
    """The last dimension cut into groups of 128, the last one filled up with zeros."""
    return F.pad(v, (0, -v.shape[-1] % _BLOCK)).unflatten(-1, (-1, _BLOCK))


def _quantise(v: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """e4m3 codes of fp32 rows and one fp32 scale per 128 columns (1 for a group of zeros)."""
    groups = _groups(v)
    amax = groups.abs().amax(-1)
    scale = torch.where(amax > 0, (amax / 448).clamp(min=2.0 ** -126), 1.0)
    codes = (groups / scale.unsqueeze(-1)).clamp(-448, 448).to(_F8)
    return codes.flatten(-2)[..., :v.shape[-1]].contiguous(), scale


def _weights(count: int, n: int, k: int, g: torch.Generator) -> tuple[torch.Tensor, torch.Tensor]:
    """``count`` matrices [n, k] of unit gain as e4m3 codes with a scale for each block of 128 x 128."""
    codes = torch.empty((count, n, k), dtype=_F8, device="cuda")
    rows = -(-n // _BLOCK) * _BLOCK
    scale = torch.empty((count, rows // _BLOCK, k // _BLOCK), device="cuda")
    for c in range(count):
        blocks = torch.randn((rows, k), device="cuda", generator=g).mul_(k ** -0.5).view(rows // _BLOCK, _BLOCK, k // _BLOCK, _BLOCK)
        scale[c] = blocks.abs().amax((1, 3)) / 448
        codes[c] = (blocks / scale[c][:, None, :, None]).view(rows, k)[:n].clamp(-448, 448).to(_F8)
    return codes, scale


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, device="cuda", generator=g)
    empty = lambda shape, dtype: torch.empty(shape, dtype=dtype, device="cuda")
    kind, s = case["kind"], {"case": case}
    if kind == "norm":
        rows, cols, dtype = case["rows"], case["cols"], _DTYPES[case["dtype"]]
        # a few channels far larger than the rest, as a residual stream has
        channel = torch.where(torch.rand(cols, device="cuda", generator=g) < 0.01, 12.0, 1.0)
        s["x"] = normal(rows, cols).to(dtype)
        s["gamma"] = 1 + 0.2 * normal(cols)
        if case["residual"]:
            s["residual"] = (normal(rows, cols) * 2 * channel).to(dtype)
            s["sum"] = empty((rows, cols), dtype)
        if case["normed"]:
            s["normed_out"] = empty((rows, cols), dtype)
        s["codes"], s["scale"] = empty((rows, cols), _F8), empty((rows, -(-cols // _BLOCK)), torch.float32)
    elif kind == "product":
        m, k, n = case["m"], case["k"], case["n"]
        s["a"], s["a_scale"] = _quantise(normal(m, k) * torch.rand(m, 1, device="cuda", generator=g).add(0.5))
        w, ws = _weights(1, n, k, g)
        s["w"], s["w_scale"] = w[0], ws[0]
        s["out"] = empty((m, n), _DTYPES[case["out"]])
    elif kind == "route":
        t, e = case["tokens"], case["experts"]
        s["logits"] = (normal(t, e) * 1.5 + 0.5 * normal(e)).to(_DTYPES[case["dtype"]])
        if case["bias"]:
            s["bias"] = 0.1 * normal(e)
        s["ids"], s["weights"] = empty((t, case["top_k"]), torch.int32), empty((t, case["top_k"]), torch.float32)
    else:
        t, h, i, e, top = case["tokens"], case["hidden"], case["inter"], case["experts"], case["top_k"]
        s["x"], s["x_scale"] = _quantise(normal(t, h))
        # some experts are asked for more often than others
        weights, ids = (normal(t, e) + 0.3 * normal(e)).softmax(-1).topk(top, -1)
        s["ids"], s["weights"] = ids.to(torch.int32), weights / weights.sum(-1, keepdim=True)
        s["gate"], s["gate_scale"] = _weights(e, i, h, g)
        s["up"], s["up_scale"] = _weights(e, i, h, g)
        s["down"], s["down_scale"] = _weights(e, h, i, g)
        s["out"] = empty((t, h), _DTYPES[case["out"]])
    return s


# ---- one pass ----------------------------------------------------------------------------------------


def run(s: dict):
    return {"norm": _norm, "product": _product, "route": _route, "experts": _experts}[s["case"]["kind"]](s)


def _norm(s: dict):
    case = s["case"]
    residual, normed = case["residual"], case["normed"]
    if own:
        _call(("add_" if residual else "") + "rms_norm_fp8_block" + ("_normed" if normed else ""), s["x"],
              *((s["residual"],) if residual else ()), s["gamma"], *((s["sum"],) if residual else ()),
              *((s["normed_out"],) if normed else ()), s["codes"], s["scale"], _EPS)
        out = {"codes": s["codes"], "scale": s["scale"]}
        return out | ({"sum": s["sum"]} if residual else {}) | ({"normed": s["normed_out"]} if normed else {})
    v = s["x"].float()
    if residual:
        v = v + s["residual"].float()
    n = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + _EPS) * s["gamma"]
    codes, scale = _quantise(n)
    out = {"codes": codes, "scale": scale}
    return out | ({"sum": v.to(s["x"].dtype)} if residual else {}) | ({"normed": n.to(s["x"].dtype)} if normed else {})


def _dequantised(codes: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """fp32 values of rows with a scale per 128 columns."""
    return (_groups(codes.float()) * scale.unsqueeze(-1)).flatten(-2)[..., :codes.shape[-1]]


def _matrix(codes: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """fp32 values of matrices [.., n, k] with a scale for each block of 128 x 128."""
    return _dequantised(codes, scale.repeat_interleave(_BLOCK, -2)[..., :codes.shape[-2], :])


def _product(s: dict):
    if own:
        _call("projection_fp8_block", s["a"], s["a_scale"], s["w"], s["w_scale"], s["out"])
        return s["out"]
    return (_dequantised(s["a"], s["a_scale"]) @ _matrix(s["w"], s["w_scale"]).t()).to(s["out"].dtype)


def _route(s: dict):
    case = s["case"]
    if own:
        _call("route_experts_biased" if case["bias"] else "route_experts", s["logits"], *((s["bias"],) if case["bias"] else ()), s["ids"],
              s["weights"], case["groups"], case["kept"], int(case["score"] == "sigmoid"), int(case["renormalize"]), 1.0)
        return {"ids": s["ids"], "weights": s["weights"]}
    logits = s["logits"].double()  # two experts' keys may differ in the last bits only
    score = torch.sigmoid(logits) if case["score"] == "sigmoid" else torch.softmax(logits, -1)
    key = score + s["bias"].double() if case["bias"] else logits
    groups = key.unflatten(-1, (case["groups"], -1))
    best = groups.sort(dim=-1, descending=True).values[..., :2 if case["bias"] else 1].sum(-1)
    left_out = best.sort(dim=-1, descending=True, stable=True).indices[:, case["kept"]:]
    key = groups.scatter(1, left_out.unsqueeze(-1).expand(-1, -1, groups.shape[-1]), -torch.inf).flatten(1)
    ids = key.sort(dim=-1, descending=True, stable=True).indices[:, :case["top_k"]]
    weights = score.gather(1, ids)
    if case["renormalize"]:
        weights = weights / weights.sum(-1, keepdim=True)
    return {"ids": ids.to(torch.int32), "weights": weights.float()}


def _experts(s: dict):
    if own:
        _call("experts_ffn_fp8_block", s["x"], s["x_scale"], s["ids"], s["weights"], s["gate"], s["gate_scale"], s["up"], s["up_scale"],
              s["down"], s["down_scale"], s["out"])
        return s["out"]
    # The rows of every expert in use side by side, as many for each as the busiest one has
    tokens, top = s["ids"].shape
    used, expert = torch.unique(s["ids"], return_inverse=True)
    expert = expert.flatten()
    order = torch.argsort(expert, stable=True)
    counts = torch.bincount(expert, minlength=len(used))
    place = torch.empty_like(expert)
    place[order] = torch.arange(len(expert), device="cuda") - (counts.cumsum(0) - counts)[expert[order]]
    rows = torch.zeros((len(used), int(counts.max()), s["x"].shape[1]), device="cuda")
    rows[expert, place] = _dequantised(s["x"], s["x_scale"]).repeat_interleave(top, 0)
    rows = rows.transpose(1, 2).contiguous()
    used = used.long()
    gate = _matrix(s["gate"][used], s["gate_scale"][used]) @ rows
    up = _matrix(s["up"][used], s["up_scale"][used]) @ rows
    h = _dequantised(*_quantise((F.silu(gate) * up).transpose(1, 2).contiguous())).transpose(1, 2).contiguous()
    y = (_matrix(s["down"][used], s["down_scale"][used]) @ h).transpose(1, 2)[expert, place]
    return (y.view(tokens, top, -1) * s["weights"].unsqueeze(-1)).sum(1).to(s["out"].dtype)


# ---- the definitions in 64 bits ------------------------------------------------------------------------


def _e4m3(v: torch.Tensor) -> torch.Tensor:
    """The e4m3 value nearest to each 64-bit value, ties to even: three bits behind the leading one, steps of 2^-9 below 2^-6."""
    exponent = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(exponent - 3)
    return (torch.round(v / step) * step).clamp(-448, 448)


def _coded(v: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows whose length is a multiple of 128: e4m3 values and scales of each group."""
    by_group = v.reshape(*v.shape[:-1], -1, 128)
    top = by_group.abs().max(-1, keepdim=True).values
    scale = torch.where(top > 0, (top / 448).clamp(min=2.0 ** -126), torch.ones_like(top))
    return _e4m3(by_group / scale).reshape(v.shape), scale.squeeze(-1)


def _spread(scale: torch.Tensor, n: int, k: int) -> torch.Tensor:
    """One 64-bit scale per element of an [n, k] matrix, from one per block."""
    return torch.kron(scale.double(), torch.ones((128, 128), dtype=torch.float64, device=scale.device))[:n, :k]


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "norm":
        total = s["x"].double()
        if case["residual"]:
            total = total + s["residual"].double()
        n = total / torch.sqrt((total ** 2).sum(-1, keepdim=True) / case["cols"] + _EPS) * s["gamma"].double()
        whole = torch.zeros((case["rows"], s["scale"].shape[1] * 128), dtype=torch.float64, device="cuda")
        whole[:, :case["cols"]] = n
        codes, scale = _coded(whole)
        out = {"codes": codes[:, :case["cols"]], "scale": scale}
        if case["residual"]:
            out["sum"] = total
        if case["normed"]:
            out["normed"] = n
        return out
    if kind == "product":
        a = s["a"].double() * torch.repeat_interleave(s["a_scale"].double(), 128, 1)
        return a @ (s["w"].double() * _spread(s["w_scale"], case["n"], case["k"])).t()
    if kind == "route":
        raw = s["logits"].double()
        if case["score"] == "sigmoid":
            score = 1 / (1 + torch.exp(-raw))
        else:
            power = torch.exp(raw - raw.max(-1, keepdim=True).values)
            score = power / power.sum(-1, keepdim=True)
        key = score + s["bias"].double() if case["bias"] else raw.clone()
        size = case["experts"] // case["groups"]
        worth = torch.stack([sum(torch.topk(key[:, i:i + size], min(2 if case["bias"] else 1, size)).values.unbind(1))
                             for i in range(0, case["experts"], size)], 1)
        # a group stays if fewer than `kept` are ahead of it: larger, or as large with a lower index
        index = torch.arange(case["groups"], device="cuda")
        ahead = (worth[:, None, :] > worth[:, :, None]) | ((worth[:, None, :] == worth[:, :, None]) & (index[None, :] < index[:, None]))
        key[(ahead.sum(-1) >= case["kept"]).repeat_interleave(size, 1)] = -torch.inf
        ids = []
        for _ in range(case["top_k"]):
            top = key.max(-1, keepdim=True).values
            place = torch.arange(case["experts"], device="cuda").expand_as(key).masked_fill(key != top, case["experts"]).min(-1, keepdim=True).values
            ids.append(place)
            key.scatter_(1, place, -torch.inf)
        ids = torch.cat(ids, 1)
        weights = torch.take_along_dim(score, ids, 1)
        return {"ids": ids.to(torch.int32), "weights": weights / weights.sum(-1, keepdim=True) if case["renormalize"] else weights}
    h, i = case["hidden"], case["inter"]
    x = s["x"].double() * torch.repeat_interleave(s["x_scale"].double(), 128, 1)
    out = torch.zeros((case["tokens"], h), dtype=torch.float64, device="cuda")
    for e in range(case["experts"]):
        token, slot = (s["ids"] == e).nonzero(as_tuple=True)
        if len(token) == 0:
            continue
        gate, up = (x[token] @ (s[w][e].double() * _spread(s[w + "_scale"][e], i, h)).t() for w in ("gate", "up"))
        codes, scale = _coded(gate / (1 + torch.exp(-gate)) * up)
        y = (codes * torch.repeat_interleave(scale, 128, 1)) @ (s["down"][e].double() * _spread(s["down_scale"][e], h, i)).t()
        out.index_add_(0, token, y * s["weights"][token, slot].double()[:, None])
    return out
