"""CPU oracle: e4m3 operands with a scale for each block of 128 - the norm that makes them, their products, a router
and the experts' FFN - in 64 bits.

TEST INFRASTRUCTURE ONLY - see ``oracle/__init__.py``.  The reference has none of these operators: PARITY UNPINNED against
it; they are pinned by mathematics (tests/test_oracle_fp8_block.py).  Every function works on the device of its inputs.
"""

from __future__ import annotations

import torch

BLOCK = 128
E4M3_MAX = 448.0


def round_e4m3(v: torch.Tensor) -> torch.Tensor:
    """The nearest e4m3 value, ties to even, of 64-bit values within +-464 (beyond, +-448)."""
    exponent = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(exponent - 3)
    return (torch.round(v / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def quantize_rows(v: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """e4m3 values [.., cols] and scales [.., ceil(cols / 128)]: amax / 448, 1 for a group of zeros, not below 2^-126."""
    cols = v.shape[-1]
    groups = torch.nn.functional.pad(v.double(), (0, -cols % BLOCK)).unflatten(-1, (-1, BLOCK))
    amax = groups.abs().amax(-1)
    scale = torch.where(amax > 0, (amax / E4M3_MAX).clamp(min=2.0 ** -126), torch.ones_like(amax))
    return round_e4m3(groups / scale.unsqueeze(-1)).flatten(-2)[..., :cols], scale


def dequantize_rows(values: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    return values.double() * scale.double().repeat_interleave(BLOCK, -1)[..., :values.shape[-1]]


def quantize_matrix(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes (float8_e4m3fn) [.., n, k] and fp32 scales [.., ceil(n / 128), ceil(k / 128)], one per block of 128 x 128."""
    n, k = w.shape[-2:]
    blocks = torch.nn.functional.pad(w.float(), (0, -k % BLOCK, 0, -n % BLOCK))
    blocks = blocks.unflatten(-1, (-1, BLOCK)).unflatten(-3, (-1, BLOCK))  # [.., n / 128, 128, k / 128, 128]
    amax = blocks.abs().amax((-1, -3))
    scale = torch.where(amax > 0, (amax / E4M3_MAX).clamp(min=2.0 ** -126), torch.ones_like(amax))
    codes = (blocks / scale[..., :, None, :, None]).flatten(-4, -3).flatten(-2)[..., :n, :k]
    return codes.clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).contiguous(), scale


def dequantize_matrix(codes: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    n, k = codes.shape[-2:]
    spread = scale.double().repeat_interleave(BLOCK, -2).repeat_interleave(BLOCK, -1)
    return codes.double() * spread[..., :n, :k]


def rms_norm(x: torch.Tensor, residual: torch.Tensor | None, gamma: torch.Tensor | None, eps: float):
    """(x + residual, its norm), 64 bits."""
    s = x.double() if residual is None else x.double() + residual.double()
    n = s * torch.rsqrt((s * s).mean(-1, keepdim=True) + eps)
    return s, n if gamma is None else n * gamma.double()


def projection(a: torch.Tensor, a_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor) -> torch.Tensor:
    return dequantize_rows(a, a_scale) @ dequantize_matrix(w, w_scale).transpose(-1, -2)


def route(logits: torch.Tensor, bias: torch.Tensor | None, top_k: int, n_groups: int = 1, topk_groups: int = 1, sigmoid: bool = False,
          renormalize: bool = True, scale: float = 1.0):
    """(ids int32 [T, top_k], weights [T, top_k] in 64 bits), one comparison at a time."""
    raw = logits.double()
    raw = torch.where(raw.isnan(), -torch.inf, raw)
    if sigmoid:
        score = 1 / (1 + torch.exp(-raw))
    else:
        top = raw.max(-1, keepdim=True).values
        power = torch.where(raw == top, 1.0, torch.exp(raw - top))
        score = power / power.sum(-1, keepdim=True)
    key = raw if bias is None else score + bias.double()
    key = torch.where(key.isnan(), -torch.inf, key)
    tokens, experts = raw.shape
    size = experts // n_groups
    ids = torch.zeros((tokens, top_k), dtype=torch.int32)
    weights = torch.zeros((tokens, top_k), dtype=torch.float64)
    for t in range(tokens):
        k = key[t].tolist()
        worth = [sum(sorted(k[g * size:(g + 1) * size], reverse=True)[:1 if bias is None else 2]) for g in range(n_groups)]
        worth = [-float("inf") if w != w else w for w in worth]
        kept = sorted(range(n_groups), key=lambda g: (-worth[g], g))[:topk_groups]
        able = [e for e in range(experts) if e // size in kept]
        chosen = sorted(able, key=lambda e: (-k[e], e))[:top_k]
        ids[t] = torch.tensor(chosen, dtype=torch.int32)
        w = score[t][chosen].cpu()
        if renormalize:
            w = w / w.sum() if w.sum() > 0 else torch.zeros_like(w)
        weights[t] = w * scale
    return ids, weights


def experts_ffn(x, x_scale, ids, weights, gate, gate_scale, up, up_scale, down, down_scale):
    """(out [T, H] in 64 bits, how far an fp32 evaluation may be off, element by element).

    A sum of k products in 32 bits is off by at most (132 + k / 128) * 2^-24 of the sum of magnitudes: 128 roundings inside a block, one
    per block, and four of the scales.  Through SwiGLU, whose derivative by g is at most 1.1 |u| and by u |SiLU(g)|, and with 2^-17 for
    exponential and reciprocal, that bounds the error of h, and with it that of a group's scale.  A code of h moves by a step where
    h / scale lies that near to a border between two codes: the second result takes the codes at both ends of h's range.
    """
    tokens, hidden = x.shape
    out = torch.zeros((tokens, hidden), dtype=torch.float64, device=x.device)
    slack = torch.zeros_like(out)
    xs = dequantize_rows(x, x_scale)
    roundings = lambda k: (132 + k // BLOCK) * 2.0 ** -24
    for e in range(gate.shape[0]):
        token, slot = (ids == e).nonzero(as_tuple=True)
        if len(token) == 0:
            continue
        wg, wu, d = (dequantize_matrix(w[e], s[e]).t() for w, s in ((gate, gate_scale), (up, up_scale), (down, down_scale)))
        g, u = xs[token] @ wg, xs[token] @ wu
        off_g, off_u = (xs[token].abs() @ w.abs() * roundings(hidden) for w in (wg, wu))
        silu = g / (1 + torch.exp(-g))
        h = silu * u
        off = 1.1 * off_g * (u.abs() + off_u) + silu.abs() * off_u + 2.0 ** -17 * h.abs()
        q, s = quantize_rows(h)
        off_s = off.unflatten(-1, (-1, BLOCK)).amax(-1) / (s * E4M3_MAX) + 2.0 ** -22  # relative
        wide, off_wide = s.repeat_interleave(BLOCK, -1), off_s.repeat_interleave(BLOCK, -1)
        reach = off / wide + (h / wide).abs() * off_wide
        moved = round_e4m3(h / wide + reach) - round_e4m3(h / wide - reach)
        w = weights[token, slot].double()[:, None]
        out.index_add_(0, token, w * ((q * wide) @ d))
        # ... of the second product, and of the sum over a token's slots
        rest = off_wide + roundings(gate.shape[1]) + ids.shape[1] * 2.0 ** -24
        slack.index_add_(0, token, w.abs() * ((moved * wide * (1 + rest) + rest * (q * wide).abs()) @ d.abs()))
    return out, slack
