"""Plain restatements in 64 bits of the operators of a step that verifies drafted tokens (no counterpart in the reference beyond their forms
for one token per sequence, examples/models/qwen3_jit/kernels/attention.py:39-102 and examples/models/04_paged_attention.py:272-365): written
token by token and row by row, on the CPU."""

from __future__ import annotations

import numpy as np
import torch

TOP = 448.0


def e4m3(v: torch.Tensor) -> torch.Tensor:
    """The e4m3 value nearest to each 64-bit value, ties to even; beyond the largest, that."""
    exponent = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(exponent - 3)
    return (torch.round(v / step) * step).clamp(-TOP, TOP)


def owners(starts, tokens: int) -> list[tuple[int, int] | None]:
    """For each token its sequence and its number there, None where it belongs to nobody."""
    starts = [int(x) for x in starts]
    out: list = [None] * tokens
    for b in range(len(starts) - 1):
        for t in range(max(0, starts[b]), min(tokens, starts[b + 1])):
            out[t] = (b, t - starts[b])
    return out


def turn(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """rope of rows x[.., D] by one position's factors (R/2 of them, or D), and the size |x_i cos| + |x_j sin| of what each element is made of."""
    d, w = x.shape[-1], cos.shape[-1]
    half = d // 2 if w == d else w
    lo, hi = (slice(0, half), slice(half, d)) if w == d else (slice(0, half), slice(0, half))
    a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
    y = torch.cat((a * cos[lo] - b * sin[lo], b * cos[hi] + a * sin[hi], rest), -1)
    size = torch.cat(((a * cos[lo]).abs() + (b * sin[lo]).abs(), (b * cos[hi]).abs() + (a * sin[hi]).abs(), rest.abs()), -1)
    return y, size


def rope_append(qkv, positions, starts, ctx_lens, cos, sin, gamma_q, gamma_k, table, key, value, k_scale, v_scale, hq, hkv, d, bs, eps):
    """-> dict: q [T, Hq, D] (None rows: NaN), key and value [pool, Hkv, bs, D] as values, the sizes of what they are made of, scales, owned [T]."""
    qkv, cos, sin = (x.detach().cpu().double() for x in (qkv, cos, sin))
    tokens, pool = len(qkv), key.numel() // (hkv * bs * d)
    x = qkv.view(tokens, hq + 2 * hkv, d)
    out = {"q": torch.full((tokens, hq, d), float("nan"), dtype=torch.float64), "q_size": torch.zeros((tokens, hq, d), dtype=torch.float64),
           "owned": torch.zeros(tokens, dtype=torch.bool), "bad": False}
    held = {n: c.detach().cpu().double().view(pool, hkv, bs, d).clone() for n, c in (("key", key), ("value", value))}
    sizes = {n: torch.zeros_like(c) for n, c in held.items()}
    fresh = {n: torch.zeros((pool, bs), dtype=torch.bool) for n in held}
    scales = {"key": k_scale, "value": v_scale}
    rows: dict = {}  # block -> its new rows: place -> (keys, values)
    max_blocks = table.shape[1]
    for t, who in enumerate(owners(starts.tolist(), tokens)):
        if who is None:
            continue
        b, i = who
        n, pos = int(ctx_lens[b]) + i, int(positions[t])
        blk = int(table[b, n // bs]) if 0 <= n < max_blocks * bs else -1
        if not 0 <= pos < len(cos) or not 0 <= blk < pool:
            out["bad"] = True
            continue
        heads = x[t].clone()
        if gamma_q is not None:
            r = 1 / torch.sqrt((heads ** 2).mean(-1, keepdim=True) + eps)
            heads[:hq] = heads[:hq] * r[:hq] * gamma_q.cpu().double()
            heads[hq:hq + hkv] = heads[hq:hq + hkv] * r[hq:hq + hkv] * gamma_k.cpu().double()
        y, size = turn(heads[:hq + hkv], cos[pos], sin[pos])
        out["q"][t], out["q_size"][t], out["owned"][t] = y[:hq], size[:hq], True
        rows.setdefault(blk, {})[n % bs] = {"key": (y[hq:], size[hq:]), "value": (heads[hq + hkv:], heads[hq + hkv:].abs())}
    for blk, new in rows.items():
        for name in held:
            if scales[name] is not None:
                before = float(1.0) if scales[name] is None else scales[name][blk].cpu().double()
                most = torch.stack([r[name][0].abs().nan_to_num(0, 0, 0).amax(-1) for r in new.values()]).amax(0) / TOP
                place = min(new)
                after = torch.where(most > 0, most, 1.0) if place == 0 else torch.maximum(before, most)
                out.setdefault(name + "_scale", {})[blk] = after
                if place:
                    grown = (after > before)[:, None, None]
                    old = held[name][blk][:, :place] * before[:, None, None]
                    held[name][blk][:, :place] = torch.where(grown, e4m3(old / after[:, None, None]), held[name][blk][:, :place])
            for place, r in new.items():
                y, size = r[name]
                if scales[name] is not None:
                    after = out[name + "_scale"][blk][:, None]
                    size = size / after
                    y = y / after  # before its rounding
                held[name][blk][:, place], sizes[name][blk][:, place], fresh[name][blk, place] = y, size, True
    for name in held:
        out[name], out[name + "_size"], out[name + "_fresh"] = held[name], sizes[name], fresh[name]
    return out


def tree_attention(query, key, value, table, ctx_lens, starts, mask, hq, hkv, d, bs, scale, k_scale=None, v_scale=None):
    """-> out [T, Hq, D] (NaN rows: nobody's), and for each row the sum of p |v| over that of p, and the largest scale * sum |q k|."""
    tokens, group = mask.shape[0], hq // hkv
    q = query.detach().cpu().double().view(tokens, hkv, group, d)
    pool = key.numel() // (hkv * bs * d)
    keys, values = (x.detach().cpu().view(pool, hkv, bs, d) for x in (key, value))
    out = torch.full((tokens, hkv, group, d), float("nan"), dtype=torch.float64)
    mass, reach = torch.zeros_like(out), torch.zeros((tokens, hkv, group, 1), dtype=torch.float64)
    words = mask.cpu().tolist()
    table, ctx_lens = table.cpu(), ctx_lens.tolist()
    for t, who in enumerate(owners(starts.tolist(), tokens)):
        if who is None:
            continue
        b, _ = who
        ctx, count = ctx_lens[b], int(starts[b + 1]) - int(starts[b])
        seen = list(range(ctx)) + [ctx + j for j in range(min(count, 32 * len(words[t]))) if words[t][j // 32] >> (j % 32) & 1]
        if not seen:
            out[t] = 0
            continue
        n = torch.tensor(seen)
        blk = table[b, n // bs].long()
        for h in range(hkv):
            k, v = keys[blk, h, n % bs].double(), values[blk, h, n % bs].double()
            if k_scale is not None:
                k, v = k * k_scale.cpu()[blk, h].double()[:, None], v * v_scale.cpu()[blk, h].double()[:, None]
            p = torch.softmax(q[t, h] @ k.t() * scale, -1)
            out[t, h], mass[t, h] = p @ v, p @ v.abs()
            reach[t, h] = (q[t, h].abs() @ k.abs().t() * abs(scale)).amax(-1, keepdim=True)
    return out.view(tokens, hq, d), mass.view(tokens, hq, d), reach.view(tokens, hq, 1)


def sample(logits, temperature, top_k, top_p, min_p, uniform) -> tuple[int, float]:
    """Token and probability of one row; None or neutral values leave a filter out.  Weights are 64-bit values, their running sums have 64 bits of mantissa: of ten thousand
    weights that differ by 1e-13, sums in 64-bit values are off by more than the differences make."""
    l = np.asarray(logits, dtype=np.float64).copy()
    l[np.isnan(l)] = -np.inf
    best = l.max()
    if best == -np.inf:
        return -1, 0.0
    if not temperature > 0:
        return int(np.argmax(l)), 1.0
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        x = np.where(l == best, 0.0, (l - best) / np.float64(temperature))
    w = np.where(l == -np.inf, 0.0, np.exp(np.where(np.isnan(x), -np.inf, x)))
    order = np.argsort(-l, kind="stable")
    order = order[l[order] > -np.inf]
    if top_k is not None and top_k > 0:
        order = order[:top_k]
    if top_p is not None and top_p < 1:
        sums = np.cumsum(w[order].astype(np.longdouble))
        need = max(float(top_p), 0.0) * sums[-1]
        order = order[:int(np.sum(sums < need)) + 1]
    if min_p is not None and min_p > 0:
        order = order[w[order] >= min(float(min_p), 1.0)]
    order = np.sort(order)
    sums = np.cumsum(w[order].astype(np.longdouble))
    u = min(max(float(uniform), 2.0 ** -25), 1 - 2.0 ** -24)
    at = int(np.sum(sums <= u * sums[-1]))
    return int(order[at]), float(w[order[at]] / sums[-1])
