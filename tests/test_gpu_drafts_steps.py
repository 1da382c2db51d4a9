"""Append, attention and sampling as a step that verifies drafted tokens makes them: one behind the other, captured, on other streams, at their limits."""

import random

import numpy as np
import pytest
import torch

from oracle import drafts as od
from pypto_amd import runtime
from test_gpu_drafts import BF, F32, F8, FP, HALF_STEP, TINY, Batch, _append, _attend, _check_append, _check_tree, _gen, _ints, _randn, _sample, _tree_masks

pytestmark = pytest.mark.gpu


# ---- the operators by themselves, further out ----------------------------------------------------------------


@pytest.mark.parametrize("lens", [[(i * 7 % 90, 1 + i % 3) for i in range(70)], [(i % 40, i % 4) for i in range(131)], [(3, 1)] * 64 + [(700, 40)]])
@pytest.mark.parametrize("group", [1, 12, 40])
def test_tree_attention_of_more_sequences_than_lanes(worker, lens, group):
    for d, cache in ((64, BF), (128, F8)):
        b = Batch(group, lens, 2, d, 32, cache, pad=1, first=1)
        dtype = FP if cache == F8 else cache
        mask = _tree_masks(random.Random(group), lens, b.tokens, 1, "tree")
        q, out = _attend(worker, b, 2 * group, dtype, mask, d ** -0.5)
        worker.sync()
        _check_tree(b, 2 * group, dtype, mask, d ** -0.5, q, out)


@pytest.mark.parametrize("d", [64, 128, 256, 80])
def test_tree_attention_over_blocks_of_very_different_scales(worker, d):
    """Zeros among them.  A value scale below 2^-60 of another's counts as that: what it is off by is 448 * 2^-60 of the largest scale."""
    lens = [(32 * 9 + 5, 6), (32 * 4, 3), (40, 40)]
    b = Batch(d, lens, 2, d, 32, F8)
    for seq, scales in ((0, (1.0, 0.0, 2.0 ** -126, 2.0 ** -100, 0.01, 0.0, 100.0, 2.0 ** -126, 3.0, 0.5)), (1, (0.0, 0.0, 2.0 ** -126, 0.0, 0.0)),
                        (2, (2.0 ** -126, 1.0, 0.0))):
        for i, v in enumerate(scales):
            b.v_scale[b.table[seq][i]] = v
    b.k_scale[b.table[0][2]] = 0.0
    mask = _tree_masks(random.Random(d), lens, b.tokens, 0, "chain")
    for dtype in (BF, FP):
        q, out = _attend(worker, b, 8, dtype, mask, d ** -0.5)
        worker.sync()
        want, mass, reach = od.tree_attention(q, b.key, b.value, b.blocks, b.ctx, b.starts, mask, 8, 2, d, 32, d ** -0.5, b.k_scale, b.v_scale)
        got = out.view(b.tokens, 8, d).cpu().double()
        off = HALF_STEP[dtype] + 2 * reach * (d + 12) * 2.0 ** -24 + 2.0 ** -19
        assert ((got - want).abs() <= off * (mass + want.abs()) + HALF_STEP[dtype] * want.abs() + TINY[dtype] + 448 * 2.0 ** -60 * 100).all()


def test_append_of_many_tokens(worker):
    """So many that a workgroup takes four groups of heads, the last of them not whole."""
    for cache, qdtype, norm in ((BF, F32, True), (FP, FP, False), (F8, BF, True)):
        b = Batch(5, [(30, 500), (0, 1), (700, 333), (0, 600)], 8, 128, 64, cache, pad=3, first=1)
        out = BF if cache == F8 else cache
        got, want = _append(worker, b, 40, qdtype, out, norm=norm)
        worker.sync()
        _check_append(b, got, want, out)


@pytest.mark.parametrize("rows,vocab,dtype", [(1100, 300, BF), (2049, 33, F32), (3, 1 << 19, BF), (2, (1 << 19) - 1, F32), (40, 20481, FP)])
def test_sample_of_many_rows_and_of_the_longest(worker, rows, vocab, dtype):
    g, rng = _gen(vocab), random.Random(rows)
    logits = (2 * _randn(g, rows, vocab)).to(dtype)
    t = [rng.choice((0.0, 0.7, 1.0, 2.0)) for _ in range(rows)]
    k = [rng.choice((0, 0, 7, 200)) for _ in range(rows)]
    p = [rng.choice((1.0, 0.4, 0.95)) for _ in range(rows)]
    m = [rng.choice((0.0, 0.0, 0.02)) for _ in range(rows)]
    tokens, probs, given = _sample(worker, logits, torch.tensor(t), torch.tensor(k), torch.tensor(p), torch.tensor(m),
                                   torch.rand(rows, device="cuda", generator=g))
    for r in range(0, rows, max(1, rows // 60)):
        token, prob = od.sample(logits[r].double().cpu().numpy(), *(x[r] for x in given))
        assert tokens[r] == token
        assert probs[r] == pytest.approx(prob, rel=2.0 ** -22, abs=1e-30)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_sample_of_rows_that_are_nearly_flat(worker, dtype):
    """High temperatures and logits close together: the whole row within a few powers of two, or within one of them."""
    g = _gen(13)
    vocab = 60000
    logits = (_randn(g, 16, vocab) * torch.tensor([2.0, 0.1, 1e-4, 0.0], device="cuda").repeat_interleave(4)[:, None]).to(dtype)
    logits[3] += 1000
    logits[7, 100:200] = -float("inf")
    logits[9, 5] = float("nan")
    t = torch.tensor([1.0, 30.0, 1e4, 1e9] * 4)
    for k, p, m in ((0, 0.9, 0.0), (30000, 1.0, 0.0), (20000, 0.5, 0.0), (0, 0.99, 0.97), (59999, 1.0, 0.5)):
        tokens, probs, given = _sample(worker, logits, t, k, p, m, torch.rand(16, device="cuda", generator=g))
        for r, row in enumerate(logits.double().cpu().numpy()):
            token, prob = od.sample(row, *(x[r] for x in given))
            assert tokens[r] == token
            assert probs[r] == pytest.approx(prob, rel=2.0 ** -22, abs=1e-30)


def test_sample_of_tiny_temperatures_and_logits(worker):
    """Differences and temperatures near the smallest numbers: 64 log2(e) / T is more than 32 bits hold."""
    g = _gen(3)
    logits = _randn(g, 12, 3000) * torch.tensor([1e-36, 1e-38, 1e-40, 1e-44], device="cuda").repeat_interleave(3)[:, None]
    t = torch.tensor([1e-38, 3e-41, 1e-45] * 4)
    for k, p in ((0, 1.0), (20, 1.0), (0, 0.7), (50, 0.9)):
        tokens, probs, given = _sample(worker, logits, t, k, p, 0.0, torch.rand(12, device="cuda", generator=g))
        rows = logits.double().cpu().numpy()
        assert tokens == [od.sample(rows[r], *(x[r] for x in given))[0] for r in range(12)]


def test_offsets_past_32_bits(worker):
    """Blocks at the end of caches of more than 2^32 bytes give what they give at the start of small ones; rows of logits likewise."""
    hkv, d, bs, hq, per = 8, 128, 64, 16, 6
    pool = (1 << 32) // (hkv * bs * d * 2) + 40
    lens = [(200, 9), (64, 1), (0, 30)]
    for cache in (BF, F8):
        small = Batch(8, lens, hkv, d, bs, cache, spare=0)
        n = small.pool
        grow = pool * (2 if cache == F8 else 1)
        rows = grow * hkv * bs
        big_k, big_v = (torch.zeros((rows, d), dtype=torch.uint8 if cache == F8 else cache, device="cuda").view(cache) for _ in range(2))
        shift = grow - n
        for big, c in ((big_k, small.key), (big_v, small.value)):
            big[shift * hkv * bs:].view(torch.uint8).copy_(c.view(torch.uint8))
        big_table = torch.where(small.blocks < n, small.blocks + shift, small.blocks)
        scales, big_scales = (), ()
        if cache == F8:
            scales = (small.k_scale.clone(), small.v_scale.clone())
            big_scales = tuple(torch.cat((torch.ones((shift, hkv), device="cuda"), s)) for s in scales)
        qkv = _randn(small.g, small.tokens, (hq + 2 * hkv) * d).to(BF)
        pos = torch.arange(small.tokens, dtype=torch.int32, device="cuda")
        angle = torch.rand((64, d // 2), device="cuda", generator=small.g)
        mask = _tree_masks(random.Random(1), lens, small.tokens, 0, "tree")
        program = runtime.rope_append_tokens_fp8 if cache == F8 else runtime.rope_append_tokens
        outs = []
        for key, value, table, sc in ((small.key, small.value, small.blocks, scales), (big_k, big_v, big_table, big_scales)):
            q = torch.empty((small.tokens * hq, d), dtype=BF, device="cuda")
            out = torch.empty_like(q)
            worker.run(program, qkv, pos, small.starts, small.ctx, angle.cos(), angle.sin(), table, key, value, *sc, q, hq, hkv, d, bs)
            worker.run(runtime.tree_attention, q, key, value, table, small.ctx, small.starts, mask, out, *sc, hq, hkv, d, bs, d ** -0.5)
            worker.sync()
            outs.append((q, out, key[-n * hkv * bs:].view(torch.uint8).clone(), value[-n * hkv * bs:].view(torch.uint8).clone()))
        assert all(torch.equal(a, b) for a, b in zip(*outs))
        assert not big_k[:64].view(torch.uint8).any()
        del big_k, big_v, outs, key, value
    vocab, rows = 1 << 19, (1 << 32) // (1 << 20) + 5
    logits = torch.empty((rows, vocab), dtype=FP, device="cuda")
    last = _randn(_gen(4), 5, vocab).to(FP)
    logits[:-5] = last[0]
    logits[-5:] = last
    u = torch.full((rows,), 0.37, device="cuda")
    k = torch.where(torch.arange(rows, device="cuda") % 2 == rows % 2, 0, 100).int()
    tokens = _sample(worker, logits, 1.0, k, 0.9, 0.0, u)[0]
    alone = _sample(worker, last, 1.0, k[-5:], 0.9, 0.0, u[-5:])[0]
    assert tokens[-5:] == alone


# ---- a step ----------------------------------------------------------------------------------------------------


class Step:
    """What a verifying step keeps: a batch's caches, its table, its drafts and buffers of fixed sizes, padded."""

    HQ, HKV, D, BS, VOCAB, EPS = 8, 2, 128, 32, 2000, 1e-6
    MASK_WORDS = 2

    def __init__(self, seed, batch, tokens, cache=BF, blocks=12):
        self.g, self.rng, self.batch, self.tokens, self.cache = _gen(seed), random.Random(seed), batch, tokens, cache
        hq, hkv, d = self.HQ, self.HKV, self.D
        self.pool = batch * blocks
        order = list(range(self.pool))
        self.rng.shuffle(order)
        self.table = _ints([order[b * blocks:(b + 1) * blocks] for b in range(batch)])
        rows = self.pool * hkv * self.BS
        if cache == F8:
            self.caches = [torch.zeros((rows, d), dtype=torch.uint8, device="cuda").view(F8) for _ in range(2)]
            self.scales = [torch.ones((self.pool, hkv), device="cuda") for _ in range(2)]
        else:
            self.caches = [torch.zeros((rows, d), dtype=cache, device="cuda") for _ in range(2)]
            self.scales = []
        self.dtype = BF if cache == F8 else cache
        angle = torch.outer(torch.arange(400, device="cuda").float(), 10000.0 ** (-torch.arange(d // 2, device="cuda") / (d // 2)))
        self.cos, self.sin = angle.cos(), angle.sin()
        self.gammas = [1 + 0.2 * _randn(self.g, d) for _ in range(2)]
        self.embedding = _randn(self.g, self.VOCAB, (hq + 2 * hkv) * d)
        self.w_out = (0.05 * _randn(self.g, hq * d, self.VOCAB)).to(self.dtype)
        self.ctx = torch.zeros(batch, dtype=torch.int32, device="cuda")
        self.starts = torch.zeros(batch + 1, dtype=torch.int32, device="cuda")
        self.drafted = torch.zeros(tokens, dtype=torch.int32, device="cuda")
        self.positions = torch.zeros(tokens, dtype=torch.int32, device="cuda")
        self.mask = torch.zeros((tokens, self.MASK_WORDS), dtype=torch.int32, device="cuda")
        self.uniform = torch.zeros(tokens, device="cuda")
        self.temperature = torch.full((tokens,), 0.8, device="cuda")
        self.top_k = torch.full((tokens,), 40, dtype=torch.int32, device="cuda")
        self.top_p = torch.full((tokens,), 0.9, device="cuda")
        self.min_p = torch.zeros(tokens, device="cuda")
        self.qkv = torch.zeros((tokens, (hq + 2 * hkv) * d), dtype=self.dtype, device="cuda")
        self.q = torch.zeros((tokens * hq, d), dtype=self.dtype, device="cuda")
        self.out = torch.zeros_like(self.q)
        self.logits = torch.zeros((tokens, self.VOCAB), device="cuda")
        self.chosen = torch.zeros(tokens, dtype=torch.int32, device="cuda")
        self.probs = torch.zeros(tokens, device="cuda")

    def plan(self, counts, contexts=None):
        """Trees of `counts` nodes, the first of each its root: random tokens, positions by depth, what each node sees."""
        starts, token, pos, mask, self.parents = [0], [], [], [], []
        ctx = self.ctx.tolist() if contexts is None else contexts
        for n, c in zip(counts, ctx):
            sees, depth, parents = [], [], []
            for i in range(n):
                parent = self.rng.randrange(i) if i else -1
                parents.append(parent)
                depth.append(depth[parent] + 1 if i else 0)
                sees.append((sees[parent] if i else 0) | 1 << i)
            pos += [c + x for x in depth]
            mask += sees
            token += [self.rng.randrange(self.VOCAB) for _ in range(n)]
            self.parents.append(parents)
            starts.append(starts[-1] + n)
        pad = self.tokens - len(token)
        assert pad >= 0
        self.starts.copy_(_ints(starts))
        self.ctx.copy_(_ints(ctx))
        self.drafted.copy_(_ints(token + [0] * pad))
        self.positions.copy_(_ints(pos + [2 ** 31 - 1] * pad))  # nobody's tokens are not looked at
        words = [[m >> 32 * w & 0xFFFFFFFF for w in range(self.MASK_WORDS)] for m in mask] + [[0xFFFFFFFF] * self.MASK_WORDS] * pad
        self.mask.copy_(torch.tensor([[w - (1 << 32) if w >> 31 else w for w in r] for r in words], dtype=torch.int64).to(torch.int32))
        self.uniform.copy_(torch.rand(self.tokens, device="cuda", generator=self.g))
        return starts

    def run(self, worker, stream=0):
        hq, hkv, d, bs = self.HQ, self.HKV, self.D, self.BS
        self.qkv.copy_(self.embedding[self.drafted.long()])
        append = runtime.rope_append_tokens_fp8_normed if self.cache == F8 else runtime.rope_append_tokens_normed
        worker.run(append, self.qkv, self.positions, self.starts, self.ctx, self.cos, self.sin, *self.gammas, self.table, *self.caches, *self.scales, self.q,
                   hq, hkv, d, bs, self.EPS, stream=stream)
        worker.run(runtime.tree_attention, self.q, *self.caches, self.table, self.ctx, self.starts, self.mask, self.out, *self.scales, hq, hkv, d, bs,
                   d ** -0.5, stream=stream)
        worker.run(runtime.projection, self.out.view(self.tokens, hq * d), self.w_out, self.logits, stream=stream)
        worker.run(runtime.sample_tokens, self.logits, self.temperature, self.top_k, self.top_p, self.min_p, self.uniform, self.chosen, self.probs, stream=stream)

    def results(self):
        return [x.clone() for x in (*(c.view(torch.uint8) for c in self.caches), *self.scales, self.q, self.out, self.logits, self.chosen, self.probs)]

    def copy(self):
        other = object.__new__(Step)
        other.__dict__ = {k: v.clone() if isinstance(v, torch.Tensor) else [x.clone() for x in v] if k in ("caches", "scales", "gammas") else v
                          for k, v in self.__dict__.items()}
        return other

    def follow(self, other):
        for k, v in self.__dict__.items():
            if isinstance(v, torch.Tensor):
                v.copy_(other.__dict__[k])
        for k in ("caches", "scales"):
            for a, b in zip(self.__dict__[k], other.__dict__[k]):
                a.view(torch.uint8).copy_(b.view(torch.uint8))


@pytest.mark.parametrize("cache", [BF, FP, F8])
def test_steps_that_verify_drafts(worker, cache):
    """Prompts, then trees of drafts: each operator's part of each step against the oracle, what is accepted moved to the front of the cache, and on."""
    s = Step(1, 5, 150, cache)
    hq, hkv, d, bs = s.HQ, s.HKV, s.D, s.BS
    generated = 0
    for step, counts in enumerate(([31, 1, 64, 17, 9], [5, 9, 1, 12, 4], [1, 1, 1, 1, 1], [16, 16, 33, 3, 0])):
        starts = s.plan(counts)
        used = starts[-1]
        if step == 0:  # prompts are chains
            for b, n in enumerate(counts):
                for i in range(n):
                    s.positions[starts[b] + i] = i
                    m = (1 << (i + 1)) - 1
                    s.mask[starts[b] + i] = torch.tensor([w - (1 << 32) if w >> 31 else w for w in (m & 0xFFFFFFFF, m >> 32)]).int()
        before = s.copy()
        s.run(worker)
        worker.sync()
        # the rows appended, by the oracle from the caches as they were
        want = od.rope_append(s.qkv, s.positions, s.starts, s.ctx, s.cos, s.sin, *s.gammas, s.table, *before.caches, *(before.scales or (None, None)), hq, hkv, d,
                              bs, s.EPS)
        assert not want["bad"]
        b = object.__new__(Batch)
        b.__dict__ = dict(pool=s.pool, hkv=hkv, bs=bs, d=d, cache=cache, key=before.caches[0], value=before.caches[1],
                          k_scale=before.scales[0] if s.scales else None, v_scale=before.scales[1] if s.scales else None)
        got = {"q": s.q.view(s.tokens, hq, d).cpu().double(), "key": s.caches[0], "value": s.caches[1]}
        if s.scales:
            got |= {"key_scale": s.scales[0], "value_scale": s.scales[1]}
        got["q"][~want["owned"]] = 7  # what no call wrote
        _check_append(b, got, want, s.dtype)
        # the attention over what the append left
        b.__dict__ |= dict(key=s.caches[0], value=s.caches[1], tokens=s.tokens, blocks=s.table, ctx=s.ctx, starts=s.starts)
        if s.scales:
            b.k_scale, b.v_scale = s.scales
        out = s.out.clone()
        out.view(s.tokens, -1)[used:] = 7
        _check_tree(b, hq, s.dtype, s.mask, d ** -0.5, s.q, out)
        # the tokens chosen from the logits
        rows, chosen = s.logits.double().cpu().numpy(), s.chosen.tolist()
        for t in range(used):
            token, prob = od.sample(rows[t], s.temperature[t].item(), 40, s.top_p[t].item(), 0.0, s.uniform[t].item())
            assert chosen[t] == token and s.probs[t].item() == pytest.approx(prob, rel=2.0 ** -22)
        # walk every tree from its root along nodes whose token was chosen, and keep the path's rows only
        ctx = s.ctx.tolist()
        for q, n in enumerate(counts):
            path = list(range(n)) if step == 0 else [0][:n]
            while step and n:
                nxt = [i for i in range(n) if s.parents[q][i] == path[-1] and (s.drafted[starts[q] + i] == chosen[starts[q] + path[-1]] or s.rng.random() < 0.4)]
                if not nxt:
                    break
                path.append(nxt[0])
            places = lambda at: [(s.table[q, i // bs].item(), i % bs) for i in at]
            src, dst = places([ctx[q] + i for i in path]), places(range(ctx[q], ctx[q] + len(path)))
            if cache != F8:  # rows of e4m3 blocks of different scales are not moved like this: the drafts' order is kept there
                for c in s.caches:
                    view = c.view(s.pool, hkv, bs, d)
                    moved = torch.stack([view[blk, :, i].clone() for blk, i in src]) if src else None
                    for r, (blk, i) in enumerate(dst):
                        view[blk, :, i] = moved[r]
            ctx[q] += len(path)
            generated += len(path)
        s.ctx.copy_(_ints(ctx))
    assert generated > 130


@pytest.mark.parametrize("cache", [BF, F8])
def test_captured_steps_follow_lengths_and_contents(worker, cache):
    """One recorded step serves other lengths, tokens and tables; two recorded steps of different sizes share the scratch; eager calls go between."""
    stream = torch.cuda.Stream()
    steps = [Step(3, 4, 60, cache), Step(4, 9, 200, cache)]
    twins = [s.copy() for s in steps]
    graphs = []
    for s in steps:
        s.plan([3] * s.batch)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            s.run(worker, stream.cuda_stream)
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                s.run(worker, stream.cuda_stream)
        graphs.append(graph)
    rng = random.Random(9)
    for replay in range(5):
        for s, twin, graph in zip(steps, twins, graphs):
            counts = [rng.choice((0, 1, 2, 5, 11, 16)) if s.batch == 4 else rng.randrange(0, 23) for _ in range(s.batch)]
            s.plan(counts, [rng.randrange(0, 300) for _ in range(s.batch)])
            s.table.copy_(s.table.flip(0))
            twin.follow(s)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            twin.run(worker)
            worker.sync()
            assert all(torch.equal(a, b) for a, b in zip(s.results(), twin.results())), (replay, counts)
    # both at once in one stream's order
    torch.cuda.synchronize()
    for graph in graphs * 2:
        graph.replay()
    for twin in twins * 2:
        twin.run(worker)
    worker.sync()
    torch.cuda.synchronize()
    for s, twin in zip(steps, twins):
        assert all(torch.equal(a, b) for a, b in zip(s.results(), twin.results()))


def test_steps_on_a_stream_of_the_callers(worker):
    """Inputs made on a stream, the step on it, results read on it: nothing waits for, or runs on, another."""
    s, stream = Step(6, 4, 60), torch.cuda.Stream()
    s.plan([7, 1, 20, 3], [100, 0, 31, 64])
    twin = s.copy()
    twin.run(worker)
    worker.sync()
    want = twin.results()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        slow = torch.zeros(1 << 28, device="cuda")
        good = s.drafted.clone()
        s.drafted.zero_()
        for _ in range(20):
            slow.add_(1.0)
        s.drafted.copy_(good)
        s.run(worker, stream.cuda_stream)
        got = s.results()
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_calls_on_host_tensors(worker):
    """Tensors in host memory are copied in and, where a call writes them, back."""
    g = torch.Generator().manual_seed(1)
    logits = torch.randn((3, 500), generator=g)
    f = lambda v: torch.full((3,), v)
    tokens, probs = torch.zeros(3, dtype=torch.int32), torch.zeros(3)
    worker.run(runtime.sample_tokens, logits, f(1.0), torch.zeros(3, dtype=torch.int32), f(0.8), f(0.0), f(0.4), tokens, probs)
    assert tokens.tolist() == [od.sample(logits[r].double().numpy(), 1.0, 0, 0.8, 0.0, 0.4)[0] for r in range(3)]
    b = Batch(2, [(9, 3), (0, 2)], 2, 64, 16, BF)
    mask = _tree_masks(random.Random(2), b.lens, 5, 0, "tree")
    q, out = _attend(worker, b, 4, BF, mask, 0.125)
    worker.sync()
    host = torch.zeros((20, 64), dtype=BF)
    worker.run(runtime.tree_attention, q.cpu(), b.key.cpu(), b.value.cpu(), b.blocks.cpu(), b.ctx.cpu(), b.starts.cpu(), mask.cpu(), host, 4, 2, 64, 16, 0.125)
    assert torch.equal(host, out.cpu())


@pytest.mark.parametrize("cache", [BF, F8])
def test_rows_of_nobody_stay_as_they_were_in_host_memory_too(worker, cache):
    b = Batch(3, [(9, 3), (30, 2)], 2, 64, 32, cache, pad=4, first=2)
    mask = _tree_masks(random.Random(2), b.lens, b.tokens, 2, "tree")
    scales = [x.cpu() for x in b.scales()]
    caches = [b.key.cpu(), b.value.cpu()]
    table = torch.ones((40, 32))
    q, out = (torch.full((b.tokens * 4, 64), 7.0, dtype=BF) for _ in range(2))
    program = runtime.rope_append_tokens_fp8 if cache == F8 else runtime.rope_append_tokens
    qkv = _randn(b.g, b.tokens, 8 * 64).to(BF).cpu()
    worker.run(program, qkv, torch.arange(b.tokens, dtype=torch.int32), b.starts.cpu(), b.ctx.cpu(), table, table * 0, b.blocks.cpu(), *caches, *scales, q, 4, 2, 64, 32)
    worker.run(runtime.tree_attention, q, *caches, b.blocks.cpu(), b.ctx.cpu(), b.starts.cpu(), mask.cpu(), out, *scales, 4, 2, 64, 32, 0.125)
    nobody = torch.ones(b.tokens, dtype=torch.bool)
    nobody[2:7] = False
    for x in (q, out):
        rows = x.view(b.tokens, -1).float()
        assert (rows[nobody] == 7).all() and (rows[~nobody] != 7).any(1).all()
    assert torch.equal(q.view(b.tokens, -1)[2:7], qkv[2:7, :256])  # turned by nothing
