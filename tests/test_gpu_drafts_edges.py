"""Append, attention of drafted trees and sampling at the ends of what their documentation allows: borders a unit wide, batches that do not fit, sizes at the limits of a
form, scores and scales that are no ordinary numbers, masked rows."""

import random

import numpy as np
import pytest
import torch

from oracle import drafts as od
from pypto_amd import runtime
from test_gpu_drafts import BF, F32, F8, FP, HALF_STEP, Batch, _append, _attend, _check_append, _check_sample, _check_tree, _gen, _ints, _randn, _sample, _tree_masks

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,cache", [(128, BF), (256, FP), (128, F8), (80, BF)])
@pytest.mark.parametrize("contexts", [(40, 70), (3000, 5000)])  # one part of the keys a workgroup, and several that are joined
def test_tree_of_sequences_that_pass_the_batch_has_the_tokens_that_are_there(worker, d, cache, contexts):
    """token_starts that end past T, or begin in front of row 0: the rows that there are belong to their sequences, which are as much shorter, and the call is reported."""
    for starts, there in (([0, 6, 15], [0, 6, 11]), ([0, 6, 2 ** 31 - 1], [0, 6, 11]), ([-3, 4, 11], [0, 4, 11]), ([0, 11, 20], [0, 11, 11])):
        b = Batch(d, [(c, 20) for c in contexts], 2, d, 32, cache)
        b.tokens, b.starts = 11, _ints(starts)
        dtype = BF if cache == F8 else cache
        mask = torch.full((11, 1), -1, dtype=torch.int32, device="cuda")
        dirty = Batch(1, [(c, 20) for c in contexts], 2, d, 32, cache)  # a call of another plan leaves its own in the scratch
        _attend(worker, dirty, 8, dtype, torch.full((40, 1), -1, dtype=torch.int32, device="cuda"), 0.1)
        worker.sync()
        q, out = _attend(worker, b, 8, dtype, mask, d ** -0.5)
        with pytest.raises(ValueError, match="tree_attention"):
            worker.sync()
        worker.sync()
        b.starts = _ints(there)
        _check_tree(b, 8, dtype, mask, d ** -0.5, q, out)


@pytest.mark.parametrize("d,cache", [(128, BF), (128, F8), (20, FP)])
def test_append_of_sequences_that_pass_the_batch_has_the_tokens_that_are_there(worker, d, cache, monkeypatch):
    oracle = od.rope_append
    for starts, there in (([0, 6, 15], [0, 6, 11]), ([-3, 4, 11], [0, 4, 11]), ([0, 11, 20], [0, 11, 11])):
        b = Batch(d, [(5, 20), (16, 20)], 2, d, 8, cache)
        b.tokens, b.starts = 11, _ints(starts)
        out = BF if cache == F8 else cache
        monkeypatch.setattr(od, "rope_append", lambda qkv, pos, _, *rest: oracle(qkv, pos, _ints(there), *rest))
        got, want = _append(worker, b, 4, BF, out)
        with pytest.raises(ValueError, match="rope_append_tokens"):
            worker.sync()
        worker.sync()
        _check_append(b, got, want, out)


@pytest.mark.parametrize("step", [1, 2])
def test_sample_counts_weights_of_one_unit(worker, step):
    """Weights are whole numbers of 2^-44 of the largest, rounded: one of 0.93 units counts as one, also where the border of top_k lies behind it.  The smallest random number asks for
    a running sum of more than 2^19 units: the first token has a thousand fewer, 1500 tokens of one unit follow (a step apart), the largest logit comes last."""
    vocab, best, ln2 = 20000, 19000, float(np.log(2.0))
    logits = torch.full((1, vocab), -45.5 * ln2)  # a third of a unit: nothing
    logits[0, 0] = float(np.log(2.0 ** 19 - 1000)) - 44 * ln2
    small = torch.arange(1, 1 + 1500 * step, step)
    logits[0, small] = -44.1 * ln2
    logits[0, 5000:5010] = -44.8 * ln2  # the border's, more than half a unit
    logits[0, best] = 0.0
    units = np.exp(logits[0].double().numpy()) * 2.0 ** 44
    assert abs(units[0] - round(units[0])) < 0.49 and (units[small] > 0.6).all() and (units[small] < 1.4).all()
    need = 2 ** 19 - round(units[0]) + 1  # so many of them pass 2^19
    assert 900 < need < 1100
    tokens, probs, _ = _sample(worker, logits.cuda(), 1.0, 2 + 1500 + 5, 1.0, 0.0, 0.0)
    assert tokens == [int(small[need - 1])]
    total = 2 ** 44 + round(units[0]) + 1500 + 5
    assert probs[0] == pytest.approx(units[small[0]] / total, rel=2.0 ** -22)


def test_tree_keeps_scratch_for_what_is_cut(worker):
    """Partial results are of sequences whose keys are cut: 2^15 tokens of 64 heads of 128 in long prompts, 1.07 GB of them in 32 bits, take no such scratch."""
    n, seqs, hq, d, bs = 512, 64, 64, 128, 128
    tokens = n * seqs
    pool = seqs * (n // bs)
    g = _gen(1)
    key, value = (_randn(g, pool * 8 * bs, d).to(BF) for _ in range(2))
    table = torch.arange(pool, dtype=torch.int32, device="cuda").view(seqs, -1)
    starts = torch.arange(0, tokens + 1, n, dtype=torch.int32, device="cuda")
    ctx = torch.zeros(seqs, dtype=torch.int32, device="cuda")
    chain = [(1 << (i + 1)) - 1 for i in range(n)]
    words = [[m >> 32 * w & 0xFFFFFFFF for w in range(n // 32)] for m in chain]
    mask = torch.tensor([[w - (1 << 32) if w >> 31 else w for w in r] for r in words], dtype=torch.int64).to(torch.int32).cuda().repeat(seqs, 1)
    q = torch.randn((tokens * hq, d), dtype=BF, device="cuda", generator=g)
    out = torch.empty_like(q)
    worker.sync()
    torch.cuda.synchronize()
    before = torch.cuda.mem_get_info()[0]
    worker.run(runtime.tree_attention, q, key, value, table, ctx, starts, mask, out, hq, 8, d, bs, d ** -0.5)
    worker.sync()
    assert before - torch.cuda.mem_get_info()[0] < 600 << 20
    # of three sequences' first, middle and last rows what the oracle says
    for s in (0, 31, 63):
        for i in (0, 255, 511):
            t = s * n + i
            want, mass, reach = od.tree_attention(q.view(tokens, -1)[t].view(hq, d), key, value, table[s:s + 1], _ints([i]), _ints([0, 1]), _ints([[1]]), hq, 8, d, bs,
                                                  d ** -0.5)
            got = out.view(tokens, hq, d)[t].double().cpu()
            off = HALF_STEP[BF] + 2 * reach * (d + 12) * 2.0 ** -24 + 2.0 ** -19
            assert ((got - want[0]).abs() <= (off * (mass + want.abs()) + HALF_STEP[BF] * want.abs())[0]).all()


@pytest.mark.parametrize("batch,hkv", [(1 << 12, 8), ((1 << 15) + 1, 8), (1 << 19, 8), (1 << 15, 256)])
def test_tree_of_very_many_sequences(worker, batch, hkv):
    """Single tokens without a context that see themselves alone: their values."""
    d, bs, pool = 64, 16, 64
    g = _gen(batch)
    key, value = (_randn(g, pool * hkv * bs, d).to(BF) for _ in range(2))
    table = torch.randint(0, pool, (batch, 1), device="cuda", generator=g, dtype=torch.int32)
    ctx = torch.randint(0, bs, (batch,), device="cuda", generator=g, dtype=torch.int32)
    ctx[: batch // 2] = 0
    starts = torch.arange(batch + 1, dtype=torch.int32, device="cuda")
    mask = torch.ones((batch, 1), dtype=torch.int32, device="cuda")
    q = torch.randn((batch * hkv, d), dtype=BF, device="cuda", generator=g)
    out = torch.empty_like(q)
    worker.run(runtime.tree_attention, q, key, value, table, ctx, starts, mask, out, hkv, hkv, d, bs, d ** -0.5)
    worker.sync()
    rows = value.view(pool, hkv, bs, d)
    got = out.view(batch, hkv, d)
    half = batch // 2
    assert torch.equal(got[:half], rows[table[:half, 0].long(), :, 0])
    at = list(range(half, batch, max(1, half * hkv // 400))) + [batch - 1]
    want, mass, reach = od.tree_attention(q.view(batch, -1)[at].reshape(-1, d), key, value, table[at], ctx[at], torch.arange(len(at) + 1), mask[at], hkv, hkv, d, bs, d ** -0.5)
    off = HALF_STEP[BF] + 2 * reach * (d + 12) * 2.0 ** -24 + 2.0 ** -19
    assert ((got[at].double().cpu() - want).abs() <= off * (mass + want.abs()) + HALF_STEP[BF] * want.abs()).all()


@pytest.mark.parametrize("d", [64, 128, 256, 80])
def test_tree_scores_that_are_no_ordinary_numbers(worker, d):
    """By either form: a score below -6.9e29 weighs nothing, among others or alone; infinite ones are NaN, as their softmax is; one of -1e29 counts."""
    b = Batch(d, [(64, 4), (3, 2), (5, 1), (2, 1), (33, 1)], 2, d, 32, BF)
    hq = 4
    key = b.key.view(b.pool, 2, 32, d)

    def put(seq, n, v):
        key[b.table[seq][n // 32], :, n % 32] = v

    big = 1.0e15
    q = torch.full((b.tokens * hq, d), big, device="cuda").to(BF)
    unit = float(torch.tensor(big).to(BF)) * d  # a key of v all over scores v * unit
    for n in range(68):
        put(0, n, -2.0e30 / unit)          # weighs nothing ...
    put(0, 50, -1.0e29 / unit)             # ... this alone counts
    for n in range(5):
        put(1, n, -1.0e31 / unit)          # nothing that counts: zeros
    for n in range(6):
        put(2, n, -5.0e29 / unit)          # every one as much as the others
    put(3, 0, float("inf"))
    put(3, 1, 1.0 / unit)
    for n in range(34):
        put(4, n, -float("inf"))
    put(4, 33, 1.0 / unit)                 # the token itself
    mask = torch.full((b.tokens, 1), -1, dtype=torch.int32, device="cuda")
    q, out = _attend(worker, b, hq, BF, mask, 1.0, q=q)
    worker.sync()
    got = out.view(b.tokens, 2, 2, d).double().cpu()
    value = b.value.view(b.pool, 2, 32, d).double().cpu()
    at = lambda seq, n: value[b.table[seq][n // 32], :, n % 32]
    assert torch.equal(got[:4], at(0, 50)[None, :, None].expand(4, 2, 2, d))
    assert (got[4:6] == 0).all()
    rows = torch.stack([at(2, n) for n in range(6)])
    assert ((got[6] - rows.mean(0)[:, None]).abs() <= 2.0 ** -7 * rows.abs().mean(0)[:, None]).all()
    assert got[7].isnan().all()
    assert torch.equal(got[8], at(4, 33)[:, None].expand(2, 2, d))


@pytest.mark.parametrize("d,cache", [(64, BF), (128, FP), (256, BF), (128, F8), (80, FP)])
def test_tree_equal_scores_weigh_the_same_however_large(worker, d, cache):
    """A thousand equal keys: the mean of their values, by scores of 10 to 10^10 that the scale rounds."""
    b = Batch(d, [(1000, 24)], 2, d, 32, cache)
    b.key.copy_((torch.sign(_randn(b.g, d)) * (256 if cache == F8 else 40000)).to(cache)[None].expand_as(b.key).clone())
    if cache == F8:
        b.k_scale.fill_(150.0)
    sign = torch.sign(b.key[0].float())
    dtype = BF if cache == F8 else cache
    size = torch.logspace(-6.5, 3.0, 24, device="cuda")  # of the scores too, times 40000 d
    size[1::2] *= -1
    q = (size[:, None, None] * sign).expand(24, 4, d).reshape(-1, d).to(dtype)
    mask = torch.full((24, 1), -1, dtype=torch.int32, device="cuda")
    scale = 1.1
    q, out = _attend(worker, b, 4, dtype, mask, scale, q=q)
    worker.sync()
    value = b.value.view(b.pool, 2, 32, d).double().cpu() * (b.v_scale.double().cpu()[:, :, None, None] if cache == F8 else 1)
    rows = torch.stack([value[b.table[0][n // 32], :, n % 32] for n in range(1024)])
    want, mass = rows.mean(0)[None, :, None], rows.abs().mean(0)[None, :, None]
    got = out.view(24, 2, 2, d).double().cpu()
    # weights of 1 to 2^-13 either way, sums in 32 bits, a rounding
    assert ((got - want).abs() <= (2.0 ** -12 + 2.0 ** -13) * mass + HALF_STEP[dtype] * want.abs()).all()


@pytest.mark.parametrize("d", [64, 128, 256, 80])
@pytest.mark.parametrize("which", ["k_scale", "v_scale"])
def test_tree_rows_are_not_reached_by_scales_of_blocks_that_they_do_not_see(worker, d, which):
    """A block of drafts whose scale is infinite or NaN, between others: what sees none of its tokens is as ever, what does is nothing finite."""
    for bad in (float("inf"), float("nan")):
        b = Batch(d, [(32, 100), (70, 20)], 2, d, 32, F8)
        inside = range(32, 64)  # drafts of the middle block
        mask = _tree_masks(random.Random(d), b.lens, b.tokens, 0, "any")
        mask[::2, 1] = 0  # half of the rows see nothing of it
        q = _randn(b.g, b.tokens * 4, d).to(BF)
        scales = getattr(b, which).clone()
        getattr(b, which)[b.table[0][2]] = bad
        _, out = _attend(worker, b, 4, BF, mask, d ** -0.5, q=q)
        worker.sync()
        setattr(b, which, scales)
        want, mass, reach = od.tree_attention(q, b.key, b.value, b.blocks, b.ctx, b.starts, mask, 4, 2, d, 32, d ** -0.5, b.k_scale, b.v_scale)
        got = out.view(b.tokens, 4, d).double().cpu()
        sees = mask[:, 1].cpu() != 0
        sees[100:] = False
        assert sees.sum() > 40 and (~sees[:100]).sum() == 50 and len(inside) == 32
        off = HALF_STEP[BF] + 2 * reach * (d + 12) * 2.0 ** -24 + 2.0 ** -19
        assert ((got - want).abs() <= off * (mass + want.abs()) + HALF_STEP[BF] * want.abs())[~sees].all()
        if which == "v_scale" or bad != bad:
            assert not got[sees].isfinite().any()


def test_tree_a_bad_scale_in_front_of_a_tiny_one(worker):
    """Rows that do not see the first block, whose value scale is NaN, over one of the smallest numbers."""
    b = Batch(3, [(0, 40)], 2, 128, 32, F8)
    mask = torch.zeros((40, 2), dtype=torch.int32, device="cuda")
    mask[:, 1] = 0xFF
    mask[::3, 0] = 1
    q = _randn(b.g, 40 * 4, 128).to(BF)
    for tiny in (1e-40, 2.0 ** -149, 0.0, 1.0, 1e30):
        b.v_scale[b.table[0][0]], b.v_scale[b.table[0][1]] = 0.5, tiny
        want, mass, _ = od.tree_attention(q, b.key, b.value, b.blocks, b.ctx, b.starts, mask, 4, 2, 128, 32, 0.1, b.k_scale, b.v_scale)
        b.v_scale[b.table[0][0]] = float("nan")
        _, out = _attend(worker, b, 4, BF, mask, 0.1, q=q)
        worker.sync()
        got = out.view(40, 4, 128).double().cpu()
        sees = torch.arange(40) % 3 == 0
        assert ((got - want).abs() <= 2.0 ** -6 * mass + 2.0 ** -134 + 448 * 2.0 ** -149)[~sees].all()
        assert not got[sees].isfinite().any()


def _fastest(worker, logits, *args):
    """Microseconds a call, the best of several dozens in a row."""
    r = logits.shape[0]
    f = lambda v, t=F32: torch.full((r,), v, dtype=t, device="cuda")
    t, k, p, m, u = args
    given = (f(t), f(k, torch.int32), f(p), f(m), f(u))
    tokens, probs = f(0, torch.int32), f(0.0)
    times = []
    for _ in range(4):
        a, z = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        for _ in range(10):
            worker.run(runtime.sample_tokens, logits, *given, tokens, probs)
        z.record()
        z.synchronize()
        times.append(a.elapsed_time(z) * 100)
    worker.sync()
    return min(times)


@pytest.mark.parametrize("dtype,masked", [(F32, -float("inf")), (F32, torch.finfo(F32).min), (BF, torch.finfo(BF).min), (FP, torch.finfo(FP).min), (F32, -1e4)])
def test_sample_of_masked_rows_is_like_that_of_others(worker, dtype, masked):
    """Logits that weigh nothing - masked ones, by infinity, the type's lowest value or any far one - take nothing from the intervals of the others: a high temperature
    over 151936 logits is 61 us for 64 rows, and was eleven times that with one masked logit."""
    g = _gen(9)
    logits = _randn(g, 64, 151936).to(dtype)
    plain = _fastest(worker, logits, 30.0, 0, 0.9, 0.0, 0.4)
    for where in (slice(1000, 1001), slice(0, 3000), slice(151000, None), slice(None, None, 3)):
        rows = logits.clone()
        rows[:, where] = masked
        args = (30.0, torch.tensor([0, 60000] * 3), torch.tensor([0.9, 0.5, 1.0] * 2), 0.0, torch.rand(6, device="cuda", generator=g))
        _check_sample(worker, rows[:6].contiguous(), *args)
        assert _fastest(worker, rows, 30.0, 0, 0.9, 0.0, 0.4) < 3 * plain


@pytest.mark.parametrize("dtype", [F32, BF])
def test_sample_by_a_large_top_k_and_top_p(worker, dtype):
    """Far apart, the two borders' intervals are collected by themselves and nothing of what lies between: 64 rows of 151936 ordinary logits, of which top_k leaves thousands."""
    g = _gen(12)
    logits = (2 * _randn(g, 64, 151936)).to(dtype)
    logits[:, 17:57] += 6
    alone = _fastest(worker, logits, 1.0, 0, 0.9, 0.0, 0.4)
    for k in (5000, 20000, 50000):
        ks = torch.tensor([k, k + 1, k - 7, k] * 2)
        _check_sample(worker, logits[:8].contiguous(), 1.0, ks, torch.tensor([0.9, 0.5, 0.99, 0.999, 0.9999, 0.95, 0.0, 0.3]), torch.tensor([0.0] * 7 + [1e-4]),
                      torch.rand(8, device="cuda", generator=g))
        assert _fastest(worker, logits, 1.0, k, 0.9, 0.0, 0.4) < 3 * alone


@pytest.mark.parametrize("d,cache", [(64, BF), (128, F8), (256, FP), (80, BF), (96, F8)])
@pytest.mark.parametrize("scale", [-0.3, 0.0])
def test_tree_of_negative_scales_and_of_none(worker, d, cache, scale):
    """Signs of the queries turned, and every key of the same weight; rows that see nothing of a chunk among them."""
    lens = [(0, 7), (5, 0), (31, 1), (33, 40), (600, 3), (0, 70)]
    for kind in ("tree", "any", "none"):
        b = Batch(d, lens, 2, d, 32, cache, pad=1, first=1)
        dtype = FP if cache == F8 else cache
        mask = _tree_masks(random.Random(d), lens, b.tokens, 1, kind)
        q, out = _attend(worker, b, 8, dtype, mask, scale)
        worker.sync()
        _check_tree(b, 8, dtype, mask, scale, q, out)
