"""Append with norms and rotation, attention of drafted trees and sampling on the GPU against the 64-bit oracle."""

import ctypes as C
import random

import numpy as np
import pytest
import torch

from oracle import drafts as od
from pypto_amd import _lib, runtime

pytestmark = pytest.mark.gpu
F8, BF, FP, F32 = torch.float8_e4m3fn, torch.bfloat16, torch.float16, torch.float32
HALF_STEP = {BF: 2.0 ** -8, FP: 2.0 ** -11, F32: 2.0 ** -24}  # relative, of a rounding to the type
TINY = {BF: 2.0 ** -134, FP: 2.0 ** -25, F32: 2.0 ** -150}    # half a step among the smallest values
CODE = {BF: 0x40, FP: 0x33, F32: 0x34, F8: 0x31}
# fp32 evaluation: a row's squares are added 8 to a lane and over at most 6 joins, then a division, a root, a division and three products: 20 roundings
# of 2^-24; a rotated element is two such products and their sum
NORM = 2.0 ** -19


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(shape, device="cuda", generator=g)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Batch:
    """A ragged batch over a paged cache of random contents: lens of (context, new tokens)."""

    def __init__(self, seed, lens, hkv, d, bs, cache, *, pad=0, spare=2, first=0):
        self.g, rng = _gen(seed), random.Random(seed)
        self.lens, self.hkv, self.d, self.bs, self.cache = lens, hkv, d, bs, cache
        used = [-(-(c + n) // bs) for c, n in lens]
        self.pool = sum(used) + spare
        free = list(range(self.pool))
        rng.shuffle(free)
        width = max(used + [1]) + 1
        self.table = [[free.pop() for _ in range(u)] + [2 ** 31 - 1 - i for i in range(width - u)] for u in used]  # what is not used is no block
        starts = [first]
        for _, n in lens:
            starts.append(starts[-1] + n)
        self.tokens = starts[-1] + pad
        self.starts, self.ctx, self.blocks = _ints(starts), _ints([c for c, _ in lens]), _ints(self.table)
        shape = (self.pool * hkv * bs, d)
        if cache == F8:
            self.key, self.value = ((_randn(self.g, *shape) * 100).clamp(-448, 448).to(F8) for _ in range(2))
            self.k_scale, self.v_scale = (0.004 + 0.006 * torch.rand((self.pool, hkv), device="cuda", generator=self.g) for _ in range(2))
        else:
            self.key, self.value = _randn(self.g, *shape).to(cache), _randn(self.g, *shape).to(cache)
            self.k_scale = self.v_scale = None

    def scales(self):
        return (self.k_scale, self.v_scale) if self.cache == F8 else ()


# ---- rope_append_tokens --------------------------------------------------------------------------------


def _append(worker, b, hq, qdtype, out, *, norm=True, width=None, eps=1e-5, max_pos=None, positions=None, scale=1.0):
    g, d, hkv = b.g, b.d, b.hkv
    width = d // 2 if width is None else width
    top = max([c + n for c, n in b.lens] + [1]) if max_pos is None else max_pos
    qkv = (scale * _randn(g, b.tokens, (hq + 2 * hkv) * d)).to(qdtype)
    pos = positions if positions is not None else torch.randint(0, top, (b.tokens,), device="cuda", generator=g, dtype=torch.int32)
    angle = torch.rand((top, width), device="cuda", generator=g) * 6.3
    cos, sin = angle.cos(), angle.sin()
    gammas = (1 + 0.3 * _randn(g, d), 1 + 0.3 * _randn(g, d)) if norm else ()
    q_out = torch.full((b.tokens * hq, d), 7.0, dtype=out, device="cuda")
    fp8 = b.cache == F8
    key, value, ks, vs = (x.clone() if x is not None else None for x in (b.key, b.value, b.k_scale, b.v_scale))
    program = {(0, 0): runtime.rope_append_tokens, (0, 1): runtime.rope_append_tokens_normed, (1, 0): runtime.rope_append_tokens_fp8,
               (1, 1): runtime.rope_append_tokens_fp8_normed}[fp8, norm]
    worker.run(program, qkv, pos, b.starts, b.ctx, cos, sin, *gammas, b.blocks, key, value, *((ks, vs) if fp8 else ()), q_out, hq, hkv, d, b.bs,
               *((eps,) if norm else ()))
    want = od.rope_append(qkv, pos, b.starts, b.ctx, cos, sin, *(gammas or (None, None)), b.blocks, b.key, b.value, b.k_scale, b.v_scale, hq, hkv, d,
                          b.bs, eps)
    return {"q": q_out.view(b.tokens, hq, d).cpu().double(), "key": key, "value": value, "key_scale": ks, "value_scale": vs}, want


def _near(got, want, size, dtype):
    assert ((got - want).abs() <= want.abs() * HALF_STEP[dtype] + 2 * size * NORM + TINY[dtype]).all()


def _check_append(b, got, want, out):
    owned = want["owned"]
    _near(got["q"][owned], want["q"][owned], want["q_size"][owned], out)
    assert (got["q"][~owned] == 7).all()
    for name, before in (("key", b.key), ("value", b.value)):
        now, was = (c.view(b.pool, b.hkv, b.bs, b.d).cpu() for c in (got[name], before))
        fresh = want[name + "_fresh"][:, None].expand(-1, b.hkv, -1)
        if b.cache != F8:
            assert torch.equal(now[~fresh].view(torch.int16), was[~fresh].view(torch.int16))
            if name == "value":  # rounded from what it is
                assert torch.equal(now[fresh], want[name][fresh].to(b.cache))
            else:
                _near(now[fresh].double(), want[name][fresh], want[name + "_size"][fresh], b.cache)
            continue
        scales = (b.k_scale if name == "key" else b.v_scale).cpu().double().clone()
        for blk, s in want.get(name + "_scale", {}).items():
            scales[blk] = s
        have = got[name + "_scale"].cpu().double()
        assert ((have - scales).abs() <= scales * (4 * NORM + 2.0 ** -23)).all()
        now, was = now.double(), was.double()
        y, size = want[name][fresh], want[name + "_size"][fresh]
        half = torch.maximum(y.abs() * 2.0 ** -4, torch.full_like(y, 2.0 ** -10))
        assert ((now[fresh] - y).abs() <= half * (1 + 2.0 ** -20) + 8 * size * NORM).all()
        # rows in front: as they were, or coded again within half a step
        rest = ~fresh
        changed = (scales > (b.k_scale if name == "key" else b.v_scale).cpu().double())[:, :, None].expand(-1, -1, b.bs)
        assert torch.equal(now[rest & ~changed], was[rest & ~changed])
        again = rest & changed
        ratio = ((b.k_scale if name == "key" else b.v_scale).cpu().double() / scales)[:, :, None, None].expand_as(was)
        y = (was * ratio)[again]
        half = torch.maximum(y.abs() * 2.0 ** -4, torch.full_like(y, 2.0 ** -10))
        # rows behind the new ones are nobody's and may be either
        in_front = torch.zeros_like(fresh)
        first = torch.where(want[name + "_fresh"].any(1), want[name + "_fresh"].int().argmax(1), 0)
        in_front |= (torch.arange(b.bs)[None, None] < first[:, None, None])
        ok = ((now[again] - y).abs() <= half * (1 + 2.0 ** -10)).all(-1)
        assert ok[in_front[again]].all()


# batch, query heads, KV heads, head_dim, block, table columns (None: D / 2)
APPEND = [
    ([(0, 1)], 1, 1, 128, 16, None),
    ([(4095, 1)], 32, 8, 128, 128, None),
    ([(0, 5), (7, 0), (15, 1), (16, 33), (100, 17), (0, 0)], 8, 2, 128, 16, None),
    ([(3, 70), (61, 3)], 5, 5, 64, 64, None),
    ([(9, 9), (0, 2)], 6, 3, 256, 32, None),
    ([(9, 9), (0, 2)], 3, 1, 512, 32, 256),
    ([(2, 11), (5, 3)], 4, 2, 80, 16, 16),      # half of the lanes that a power of two takes, 32 elements turned
    ([(2, 11), (5, 3)], 4, 4, 96, 24, 48),
    ([(1, 6)], 2, 2, 128, 16, 128),             # the reference's tables
    ([(1, 6)], 3, 1, 128, 16, 8),
    ([(i % 23, i % 4) for i in range(131)], 4, 1, 64, 16, None),   # more sequences than a wavefront has lanes
    ([(i % 5, 1 + (i == 77)) for i in range(4200)], 1, 1, 64, 8, None),
]


@pytest.mark.parametrize("lens,hq,hkv,d,bs,width", APPEND)
@pytest.mark.parametrize("cache", [BF, FP, F8])
@pytest.mark.parametrize("norm", [True, False])
def test_append(worker, lens, hq, hkv, d, bs, width, cache, norm):
    for i, qdtype in enumerate((BF, FP, F32)):
        b = Batch(len(lens) * d + i, lens, hkv, d, bs, cache, pad=i, first=i % 2)
        out = cache if cache != F8 else (BF, FP, BF)[i]
        got, want = _append(worker, b, hq, qdtype, out, norm=norm, width=width)
        worker.sync()
        _check_append(b, got, want, out)


@pytest.mark.parametrize("d,width,dtype", [(20, None, BF), (130, 65, FP), (520, 260, BF), (128, 12, FP), (34, 34, BF), (2, 1, FP)])
def test_append_of_other_widths(worker, d, width, dtype):
    """Rows that do not come in eights: one wavefront a head."""
    for norm in (True, False):
        b = Batch(d, [(3, 4), (0, 9)], 2, d, 8, dtype, pad=1)
        got, want = _append(worker, b, 4, F32, dtype, norm=norm, width=width)
        worker.sync()
        _check_append(b, got, want, dtype)


@pytest.mark.parametrize("cache", [BF, F8])
def test_append_leaves_out_what_has_no_place_and_says_so(worker, cache):
    """A position outside the tables, an index outside the table, a block outside the cache: the other tokens are as ever."""
    for case in ("position", "negative", "table", "pool", "length"):
        b = Batch(11, [(5, 6), (14, 9), (0, 3)], 2, 64, 8, cache, pad=2)
        pos = torch.arange(b.tokens, dtype=torch.int32, device="cuda")
        if case == "position":
            pos[7] = 40
        elif case == "negative":
            pos[0] = -1
        elif case == "table":
            b.ctx[1] = b.blocks.shape[1] * 8 - 2
            b.blocks[1] = _ints([x % b.pool for x in range(b.blocks.shape[1])])
        elif case == "pool":
            b.blocks[2, 0] = b.pool
        else:
            b.ctx[0] = -3
        got, want = _append(worker, b, 4, BF, BF, max_pos=40, positions=pos)
        assert want["bad"]
        with pytest.raises(ValueError, match="rope_append_tokens"):
            worker.sync()
        worker.sync()  # reported once
        if case != "table":  # where two sequences share blocks the e4m3 rows have no oracle
            if cache == F8 and case in ("position", "negative"):
                assert torch.equal(got["q"][want["owned"]].isnan(), torch.zeros_like(got["q"][want["owned"]], dtype=torch.bool))
                _near(got["q"][want["owned"]], want["q"][want["owned"]], want["q_size"][want["owned"]], BF)
            else:
                _check_append(b, got, want, BF)


def test_append_fp8_infinities_nan_and_zeros(worker):
    b = Batch(3, [(0, 4)], 1, 64, 8, F8)
    qkv = torch.ones((4, 3 * 64), dtype=BF, device="cuda")
    qkv[0, 128:] = torch.tensor([float("inf"), -float("inf"), float("nan"), 2.0] + [1.0] * 60, device="cuda")
    qkv[:, 64:128] = 0
    key, value, ks, vs = b.key.clone(), b.value.clone(), b.k_scale.clone(), b.v_scale.clone()
    one = torch.ones((8, 32), device="cuda")
    q = torch.zeros((4, 64), dtype=BF, device="cuda")
    worker.run(runtime.rope_append_tokens_fp8, qkv, _ints([0, 1, 2, 3]), b.starts, b.ctx, one, one * 0, b.blocks, key, value, ks, vs, q, 1, 1, 64, 8)
    worker.sync()
    blk = b.table[0][0]
    assert vs[blk, 0] == np.float32(2.0) / np.float32(448) and ks[blk, 0] == 1
    row = value.view(b.pool, 8, 64)[blk, 0].float()
    assert row[0] == 448 and row[1] == -448 and row[2].isnan() and row[3] == 448 and (row[4:] == 224).all()
    assert (key.view(b.pool, 8, 64)[blk, :4].float() == 0).all()


def test_append_twice_equals_one_call(worker):
    """16-bit rows do not depend on how the tokens are split over calls, nor on where a call's tensors start."""
    b = Batch(21, [(3, 40)], 2, 128, 16, BF)
    g, hq = b.g, 4
    qkv, pos = _randn(g, 40, 8 * 128).to(BF), torch.arange(3, 43, dtype=torch.int32, device="cuda")
    angle = torch.rand((64, 64), device="cuda", generator=g)
    gam = (1 + _randn(g, 128), 1 + _randn(g, 128))

    def call(lo, hi, ctx, key, value, shift):
        buf = torch.empty(qkv[lo:hi].numel() + shift, dtype=BF, device="cuda")
        src = buf[shift:].view(hi - lo, -1)
        src.copy_(qkv[lo:hi])
        out = torch.empty(((hi - lo) * hq, 128), dtype=BF, device="cuda")
        worker.run(runtime.rope_append_tokens_normed, src, pos[lo:hi].clone(), _ints([0, hi - lo]), _ints([ctx]), angle.cos(), angle.sin(), *gam, b.blocks,
                   key, value, out, hq, 2, 128, 16, 1e-6)
        return out

    k0, v0, k1, v1 = b.key.clone(), b.value.clone(), b.key.clone(), b.value.clone()
    whole = call(0, 40, 3, k0, v0, 0)
    parts = torch.cat((call(0, 17, 3, k1, v1, 0), call(17, 40, 20, k1, v1, 8)))
    worker.sync()
    assert torch.equal(whole, parts) and torch.equal(k0, k1) and torch.equal(v0, v1)
    off = call(0, 40, 3, k1, v1, 3)  # not at a multiple of 16 bytes: the other form, the same values to a rounding or two
    worker.sync()
    assert ((off.float() - whole.float()).abs() <= 2.0 ** -7 * whole.float().abs() + 2.0 ** -10).all()


# ---- tree_attention --------------------------------------------------------------------------------------


def _tree_masks(rng, lens, tokens, first, kind):
    words = max(1, -(-max(n for _, n in lens) // 32))
    rows = [[rng.getrandbits(32) for _ in range(words)] for _ in range(tokens)]  # nobody's rows and bits of nobody hold anything
    t = first
    for _, n in lens:
        sees = []
        for i in range(n):
            if kind == "chain":
                m = (1 << (i + 1)) - 1
            elif kind == "any":
                m = rng.getrandbits(32 * words)
            elif kind == "none":
                m = 0
            else:
                parent = rng.randrange(-1, i) if i else -1
                m = (sees[parent] if parent >= 0 else 0) | 1 << i
            sees.append(m)
            noise = rng.getrandbits(32 * words) >> n << n  # tokens that the sequence does not have
            rows[t + i] = [((m | noise) >> 32 * w) & 0xFFFFFFFF for w in range(words)]
        t += n
    return torch.tensor([[w - (1 << 32) if w >> 31 else w for w in r] for r in rows], dtype=torch.int64).to(torch.int32).cuda()


def _attend(worker, b, hq, dtype, mask, scale, q=None, out=None):
    q = _randn(b.g, b.tokens * hq, b.d).to(dtype) if q is None else q
    out = torch.full((b.tokens * hq, b.d), 7.0, dtype=dtype, device="cuda") if out is None else out
    worker.run(runtime.tree_attention, q, b.key, b.value, b.blocks, b.ctx, b.starts, mask, out, *b.scales(), hq, b.hkv, b.d, b.bs, scale)
    return q, out


def _check_tree(b, hq, dtype, mask, scale, q, out):
    """Every probability is off by half a step of the type and by its score's error: 2^-24 for each of D products and a dozen roundings more, of the sum of
    the products' sizes; the result is a mean weighted by them, and is rounded once."""
    want, mass, reach = od.tree_attention(q, b.key, b.value, b.blocks, b.ctx, b.starts, mask, hq, b.hkv, b.d, b.bs, scale, b.k_scale, b.v_scale)
    got = out.view(b.tokens, hq, b.d).cpu().double()
    nobody = want.isnan().all(-1).all(-1)
    assert (got[nobody] == 7).all()
    got, want, mass, reach = (x[~nobody] for x in (got, want, mass, reach))
    off = HALF_STEP[dtype] + 2 * reach * (b.d + 12) * 2.0 ** -24 + 2.0 ** -19
    assert ((got - want).abs() <= off * (mass + want.abs()) + HALF_STEP[dtype] * want.abs() + TINY[dtype]).all()


TREES = [
    ([(0, 1)], 1, 1, 16),
    ([(1, 1)], 4, 1, 16),
    ([(0, 7), (5, 0), (31, 1), (32, 33), (33, 16), (100, 3), (0, 0)], 8, 2, 16),
    ([(500, 16)], 32, 8, 128),
    ([(300, 64), (17, 40), (1000, 1)], 16, 2, 64),
    ([(40, 70)], 8, 1, 32),         # three words of mask
    ([(0, 130)], 4, 4, 32),
    ([(2500, 5), (63, 9)], 40, 8, 32),
]


@pytest.mark.parametrize("lens,hq,hkv,bs", TREES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("cache", [BF, FP, F8])
def test_tree_attention(worker, lens, hq, hkv, bs, d, cache):
    for i, kind in enumerate(("tree", "any", "chain")):
        b = Batch(d + i, lens, hkv, d, bs if cache != F8 else max(bs, 32), cache, pad=i, first=i % 2)
        dtype = cache if cache != F8 else (BF, FP, BF)[i]
        mask = _tree_masks(random.Random(i), lens, b.tokens, i % 2, kind)
        q, out = _attend(worker, b, hq, dtype, mask, d ** -0.5)
        worker.sync()
        _check_tree(b, hq, dtype, mask, d ** -0.5, q, out)


@pytest.mark.parametrize("d,bs,cache", [(80, 16, BF), (20, 7, FP), (128, 24, BF), (256, 5, FP), (96, 32, F8), (128, 16, F8), (1, 3, BF), (33, 16, F8)])
def test_tree_attention_of_other_shapes(worker, d, bs, cache):
    lens = [(50, 9), (0, 3), (7, 34), (3, 0)]
    b = Batch(d, lens, 2, d, bs, cache, pad=1)
    dtype = cache if cache != F8 else FP
    mask = _tree_masks(random.Random(d), lens, b.tokens, 0, "tree")
    q, out = _attend(worker, b, 6, dtype, mask, 0.2)
    worker.sync()
    _check_tree(b, 6, dtype, mask, 0.2, q, out)


@pytest.mark.parametrize("d", [64, 128, 80])
@pytest.mark.parametrize("cache", [BF, F8])
def test_tree_rows_that_see_nothing_are_zeros(worker, d, cache):
    lens = [(0, 5), (3, 2), (0, 40)]
    b = Batch(1, lens, 2, d, 32, cache)
    mask = _tree_masks(random.Random(5), lens, b.tokens, 0, "none")
    mask[3, 0] = 1 << 2  # one of them sees one other
    dtype = BF if cache == F8 else cache
    q, out = _attend(worker, b, 4, dtype, mask, 1.0)
    worker.sync()
    _check_tree(b, 4, dtype, mask, 1.0, q, out)
    assert (out.view(b.tokens, -1)[[0, 1, 2, 4]] == 0).all() and (out.view(b.tokens, -1)[7:] == 0).all()


@pytest.mark.parametrize("d", [64, 128, 256, 80])
@pytest.mark.parametrize("cache", [BF, FP, F8])
def test_tree_what_a_row_does_not_see_has_no_part_in_it(worker, d, cache):
    """Infinities and NaN in keys and values that some rows of a tile see and others do not, and in what lies behind a sequence's last token."""
    lens = [(37, 6), (0, 20), (70, 1)]
    b = Batch(d, lens, 2, d, 32, cache)
    dtype = FP if cache == F8 else cache
    rng = random.Random(8)
    mask = _tree_masks(rng, lens, b.tokens, 0, "chain")
    nan, inf = float("nan"), float("inf") if cache != F8 else float("nan")
    clean_k, clean_v = b.key.clone(), b.value.clone()

    def put(cache_t, seq, n, value, what):
        c = cache_t.view(b.pool, 2, 32, d)
        c[b.table[seq][n // 32], :, n % 32, what] = torch.tensor(value, device="cuda").to(cache_t.dtype)

    put(b.value, 0, 37 + 3, inf, 0)
    put(b.value, 0, 37 + 4, nan, d - 1)
    put(b.key, 0, 37 + 5, nan, slice(None))
    put(b.value, 1, 17, nan, slice(None))
    put(b.value, 1, 18, -inf, 3)
    for seq, n in ((0, 43), (1, 20), (2, 71), (2, 95)):  # behind the last token
        put(b.key, seq, n, nan, slice(None))
        put(b.value, seq, n, nan, slice(None))
    q, out = _attend(worker, b, 4, dtype, mask, d ** -0.5)
    worker.sync()
    got = out.view(b.tokens, 4, d).double().cpu()
    b.key, b.value = clean_k, clean_v
    want, mass, reach = od.tree_attention(q, b.key, b.value, b.blocks, b.ctx, b.starts, mask, 4, 2, d, 32, d ** -0.5, b.k_scale, b.v_scale)
    ok = torch.ones((b.tokens, d), dtype=torch.bool)  # elements that no such value reaches
    ok[3:6, 0] = False
    ok[4:6, d - 1] = False
    ok[5] = False
    ok[6 + 17:26] = False
    off = (2 * HALF_STEP[dtype] + 2 * reach * (d + 12) * 2.0 ** -24 + 2.0 ** -19) * (mass + want.abs()) + TINY[dtype]
    assert ((got - want).abs() <= off)[ok[:, None].expand(-1, 4, -1)].all()
    assert (got[3:6, :, 0].isnan() | got[3:6, :, 0].isinf()).all() and got[4:6, :, d - 1].isnan().all() and got[5].isnan().all()
    assert got[6 + 17:26].isnan().all()


def test_tree_reports_lengths_and_blocks_that_do_not_fit(worker):
    for d in (128, 80):
        for case in ("bits", "table", "pool", "length"):
            lens = [(10, 40 if case == "bits" else 4), (20, 3)]
            b = Batch(4, lens, 1, d, 32, BF)
            mask = torch.full((b.tokens, 1), -1, dtype=torch.int32, device="cuda")
            if case == "table":
                b.ctx[0] = b.blocks.shape[1] * 32 - 2
                b.blocks[0] = _ints([x % b.pool for x in range(b.blocks.shape[1])])
            elif case == "pool":
                b.blocks[0, 0] = -1
            elif case == "length":
                b.ctx[0] = -1
            q, out = _attend(worker, b, 2, BF, mask, 0.1)
            with pytest.raises(ValueError, match="tree_attention"):
                worker.sync()
            worker.sync()
            # the other sequence is as ever
            n0 = lens[0][1]
            want, mass, _ = od.tree_attention(q, b.key, b.value, b.blocks, _ints([0, 20]), _ints([n0, n0, n0 + 3]), mask, 2, 1, d, 32, 0.1)
            got = out.view(b.tokens, 2, d)[n0:].double().cpu()
            assert ((got - want[n0:]).abs() <= 2.0 ** -6 * (mass[n0:] + want[n0:].abs())).all()


def test_tree_of_one_token_is_paged_attention(worker):
    """One new token per sequence that sees itself: what paged_attention gives for contexts one longer.  Both round every probability once, to half a step
    of bfloat16 on either side of its value, and their row sums are of the rounded ones: each is off by at most 2^-8 of sum p |v| + |out|, besides this one's
    rounding of the result."""
    lens = [(0, 1), (77, 1), (1000, 1), (2047, 1)]
    b = Batch(9, lens, 8, 128, 128, BF)
    q = _randn(b.g, 4 * 32, 128).to(BF)
    mask = torch.ones((4, 1), dtype=torch.int32, device="cuda")
    _, out = _attend(worker, b, 32, BF, mask, 128 ** -0.5, q=q)
    want = torch.empty((4 * 32, 128), device="cuda")
    width = b.blocks.shape[1]
    cfg = torch.tensor([4, 32, 8, 128, 128, width, int(np.float32(128 ** -0.5).view(np.uint32))], dtype=torch.int64)
    worker.run(runtime.paged_attention, q, b.key, b.value, b.blocks.flatten(), b.ctx + 1, want, cfg)
    worker.sync()
    exact, mass, reach = od.tree_attention(q, b.key, b.value, b.blocks, b.ctx, b.starts, mask, 32, 8, 128, 128, 128 ** -0.5)
    off = 2 * (2.0 ** -8 + 2 * reach * 140 * 2.0 ** -24 + 2.0 ** -19) * (mass + exact.abs()) + 2.0 ** -8 * exact.abs()
    assert ((out.double() - want.double()).abs().cpu().view(4, 32, 128) <= off).all()


# ---- sample_tokens ---------------------------------------------------------------------------------------


def _sample(worker, logits, temperature, top_k, top_p, min_p, uniform):
    r = logits.shape[0]
    f = lambda v: torch.as_tensor(v, dtype=F32, device="cuda").expand(r).contiguous()
    args = (f(temperature), torch.as_tensor(top_k, dtype=torch.int32, device="cuda").expand(r).contiguous(), f(top_p), f(min_p), f(uniform))
    tokens, probs = torch.full((r,), -7, dtype=torch.int32, device="cuda"), torch.full((r,), -7.0, device="cuda")
    worker.run(runtime.sample_tokens, logits, *args, tokens, probs)
    worker.sync()
    return tokens.tolist(), probs.tolist(), [a.tolist() for a in args]


def _check_sample(worker, logits, *args):
    tokens, probs, given = _sample(worker, logits, *args)
    rows = logits.double().cpu().numpy()
    for r in range(len(rows)):
        t, k, p, m, u = (g[r] for g in given)
        token, prob = od.sample(rows[r], t, k, p, m, u)
        assert tokens[r] == token, (r, t, k, p, m, u)
        assert probs[r] == pytest.approx(prob, rel=2.0 ** -22, abs=1e-30)  # two roundings to 32 bits and sums off by 2^-45 a token


@pytest.mark.parametrize("vocab", [1, 2, 63, 64, 65, 1000, 1024, 1025, 4097, 32000, 50001, 151936])
@pytest.mark.parametrize("dtype", [BF, FP, F32])
def test_sample(worker, vocab, dtype):
    g = _gen(vocab)
    rows = 24
    logits = (_randn(g, rows, vocab) * (0.5 + 3 * torch.rand((rows, 1), device="cuda", generator=g))).to(dtype)
    rng = random.Random(vocab)
    t = [rng.choice((0.0, 0.3, 0.7, 1.0, 1.0, 1.7, 30.0)) for _ in range(rows)]
    k = [rng.choice((0, 0, 1, 2, 5, 50, 300, 3000, vocab - 1, vocab, -1)) for _ in range(rows)]
    p = [rng.choice((1.0, 1.0, 0.1, 0.5, 0.9, 0.99, 0.9999, 0.0)) for _ in range(rows)]
    m = [rng.choice((0.0, 0.0, 0.0, 1e-4, 0.05, 0.5, 1.0, 2.0)) for _ in range(rows)]
    _check_sample(worker, logits, torch.tensor(t), torch.tensor(k), torch.tensor(p), torch.tensor(m), torch.rand(rows, device="cuda", generator=g))


@pytest.mark.parametrize("dtype", [BF, FP, F32])
def test_sample_of_few_different_values(worker, dtype):
    """Thousands of equal logits at every border: which of them stay goes by their index."""
    g = _gen(6)
    for levels, vocab in ((1, 5000), (2, 40000), (3, 9000), (7, 100000)):
        logits = torch.randint(0, levels, (16, vocab), device="cuda", generator=g).to(dtype) * 0.5
        k = torch.randint(0, vocab, (16,), device="cuda", generator=g, dtype=torch.int32)
        p = torch.where(torch.arange(16, device="cuda") % 2 == 0, 1.0, 0.1 + 0.8 * torch.rand(16, device="cuda", generator=g))
        k[8:12] = 0
        _check_sample(worker, logits, 1.0, k, p, 0.0, torch.rand(16, device="cuda", generator=g))


def test_sample_of_peaked_and_of_very_wide_rows(worker):
    g = _gen(7)
    scale = torch.tensor([1e-30, 1e-3, 1.0, 50.0, 1e4, 1e20, 1e37, 3.0], device="cuda").repeat_interleave(4)[:, None]
    logits = _randn(g, 32, 20000).clamp(-3, 3) * scale
    t = torch.tensor([1.0, 1e-20, 1e20, float("inf")] * 8)
    _check_sample(worker, logits, t, torch.tensor([0, 40] * 16), torch.tensor([1.0, 1.0, 0.6, 0.9] * 8), 0.0, torch.rand(32, device="cuda", generator=g))


def test_sample_of_infinities_nan_and_parameters_that_say_nothing(worker):
    inf, nan = float("inf"), float("nan")
    logits = torch.full((12, 3000), -inf, device="cuda")
    logits[1, 7] = nan
    logits[2, [5, 2999]] = torch.tensor([inf, inf], device="cuda")
    logits[3, 100:200] = 1.0
    logits[4] = nan
    logits[5, 2998] = -3e38
    logits[6:, 10:20] = torch.arange(10, device="cuda").float()
    logits[6:, 15] = nan
    t = torch.tensor([1.0, 0.0, 1.0, 1.0, 1.0, 1.0, nan, -1.0, 1.0, 1.0, 1.0, 1.0])
    k = torch.tensor([0, 3, 0, 2000, 5, 1, 0, 0, -5, 3, 0, 2 ** 31 - 1])
    p = torch.tensor([1.0, 0.5, 1.0, 0.5, 0.5, 0.5, 1.0, 1.0, nan, 2.0, -1.0, 1.0])
    m = torch.tensor([0.0, 0.0, 0.0, 0.0, 0.5, 1.0, 0.0, 0.0, nan, -1.0, 0.0, inf])
    u = torch.tensor([0.5, 0.5, 0.75, 0.5, 0.5, 0.0, 0.5, 0.5, 0.3, 0.999999, 0.5, 0.5])
    _check_sample(worker, logits, t, k, p, m, u)
    # random numbers outside of [0, 1) are moved into it
    tokens, _, _ = _sample(worker, torch.zeros((4, 100), device="cuda"), 1.0, 0, 1.0, 0.0, torch.tensor([-1.0, nan, 1.0, inf]))
    assert tokens == [0, 0, 99, 99]


def test_sample_frequencies(worker):
    """Evenly spaced random numbers give every token as often as its share says, to one."""
    logits = torch.randn(50, device="cuda", generator=_gen(1)).expand(20000, 50).contiguous()
    u = (torch.arange(20000, device="cuda") + 0.5) / 20000
    tokens, _, _ = _sample(worker, logits, 0.8, 0, 1.0, 0.0, u)
    share = torch.softmax(logits[0].double() / 0.8, 0).cpu() * 20000
    count = torch.bincount(torch.tensor(tokens), minlength=50)
    assert ((count - share).abs() <= 1.01).all()


def test_sample_rows_of_any_alignment_and_of_optional_filters(worker):
    lib, g = _lib.load(), _gen(2)
    for dtype, shift in ((BF, 1), (FP, 3), (F32, 1), (F32, 2)):
        buf = _randn(g, 7 * 2049 + shift).to(dtype)
        logits = buf[shift:].view(7, 2049)
        t, u = torch.full((7,), 0.9, device="cuda"), torch.rand(7, device="cuda", generator=g)
        tokens = torch.full((7,), -7, dtype=torch.int32, device="cuda")
        _lib.check(lib.pto_hip_sample_tokens(logits.data_ptr(), t.data_ptr(), None, None, None, u.data_ptr(), tokens.data_ptr(), None, 7, 2049,
                                             CODE[dtype], None))
        worker.sync()
        assert tokens.tolist() == [od.sample(logits[r].double().cpu().numpy(), t[r].item(), None, None, None, u[r].item())[0] for r in range(7)]


# ---- refusals --------------------------------------------------------------------------------------------


def test_refusals(worker):
    b = Batch(1, [(3, 2)], 2, 64, 16, BF)
    qkv, pos, table = _randn(b.g, 2, 8 * 64).to(BF), _ints([0, 1]), torch.ones((8, 32), device="cuda")
    q = torch.empty((8, 64), dtype=BF, device="cuda")
    good = [qkv, pos, b.starts, b.ctx, table, table, b.blocks, b.key, b.value, q, 4, 2, 64, 16]

    def bad(program, args, match, **at):
        args = list(args)
        for i, v in at.items():
            args[int(i[1:])] = v
        with pytest.raises((ValueError, RuntimeError), match=match):
            worker.run(program, *args)

    app = runtime.rope_append_tokens
    worker.run(app, *good)
    worker.sync()
    bad(app, good, "qkv must be", _0=qkv[:, :-64].contiguous())
    bad(app, good, "qkv dtype", _0=torch.zeros((2, 8 * 64), dtype=torch.int8, device="cuda"))
    bad(app, good, "positions", _1=_ints([0]))
    bad(app, good, "positions", _1=torch.zeros(2, device="cuda"))
    bad(app, good, "token_starts", _2=_ints([0, 1, 2]))
    bad(app, good, "rope_cos", _4=table[:4].contiguous())
    bad(app, good, "rope tables", _4=torch.ones((8, 40), device="cuda"), _5=torch.ones((8, 40), device="cuda"))
    bad(app, good, "block_table", _6=b.blocks.flatten())
    bad(app, good, "caches of", _7=b.key.to(FP), _8=b.value.to(FP))
    bad(app, good, "key/value cache", _8=b.value[:-16].contiguous())
    bad(app, good, "q_out", _9=q.float())
    bad(app, good, "scalar", _12=0)
    bad(app, good, "overlaps an input", _9=qkv.view(-1)[:512].view(8, 64))
    bad(app, good, "two outputs overlap", _8=b.key)
    bad(app, good[:-1], "takes 10")
    fp8 = Batch(1, [(3, 2)], 2, 64, 16, F8)
    good8 = [qkv, pos, b.starts, b.ctx, table, table, fp8.blocks, fp8.key, fp8.value, fp8.k_scale, fp8.v_scale, q, 4, 2, 64, 16]
    bad(runtime.rope_append_tokens_fp8, good8, "scale must be", _9=fp8.k_scale[1:].contiguous())
    bad(runtime.rope_append_tokens_fp8, good8, "FP8E4M3FN", _7=b.key, _8=b.value)
    bad(runtime.rope_append_tokens_fp8, good8, "multiple of 8", _4=table[:, :31].contiguous(), _5=table[:, :31].contiguous())

    mask, out = _ints([[1], [3]]), torch.empty_like(q)
    good = [q, b.key, b.value, b.blocks, b.ctx, b.starts, mask, out, 4, 2, 64, 16, 0.1]
    tree = runtime.tree_attention
    worker.run(tree, *good)
    worker.sync()
    bad(tree, good, "divide over", _8=8, _9=3, _1=b.key.view(-1, 64)[:96].contiguous(), _2=b.value[:96].contiguous(), _0=torch.cat((q, q)), _7=torch.cat((q, q)))
    bad(tree, good, "one dtype", _7=out.float())
    bad(tree, good, "tree_mask", _6=mask.float())
    bad(tree, good, "tree_mask", _6=_ints([[1]]))
    bad(tree, good, "caches of", _1=fp8.key, _2=fp8.value)
    bad(tree, good, "overlaps", _7=q)
    bad(tree, good, "finite", _12=float("inf"))
    bad(tree, good, "mask words", _6=torch.zeros((2, 33), dtype=torch.int32, device="cuda"))
    bad(tree, good + [], "query dtype", _0=q.float(), _7=out.float(), _1=b.key.float(), _2=b.value.float())
    wide = Batch(1, [(3, 2)], 2, 512, 16, BF)
    q512 = torch.empty((8, 512), dtype=BF, device="cuda")
    bad(tree, [q512, wide.key, wide.value, wide.blocks, wide.ctx, wide.starts, mask, torch.empty_like(q512), 4, 2, 512, 16, 0.1], "head_dim at most 256")

    r, v = 3, 100
    f = torch.ones(r, device="cuda")
    i = torch.ones(r, dtype=torch.int32, device="cuda")
    good = [torch.zeros((r, v), device="cuda"), f, i, f, f, f, i.clone(), f.clone()]
    worker.run(runtime.sample_tokens, *good)
    worker.sync()
    bad(runtime.sample_tokens, good, "dtype", _0=torch.zeros((r, v), dtype=torch.int32, device="cuda"))
    bad(runtime.sample_tokens, good, "temperature", _1=f[:2].contiguous())
    bad(runtime.sample_tokens, good, "top_k", _2=f)
    bad(runtime.sample_tokens, good, "overlap", _7=f)
    bad(runtime.sample_tokens, good, "dims", _0=torch.zeros(r, device="cuda"))
    bad(runtime.sample_tokens, good, "at most", _0=torch.zeros((r, (1 << 19) + 1), dtype=BF, device="cuda"))


def test_empty_batches(worker):
    b = Batch(1, [(0, 0)], 1, 64, 16, BF)
    q = torch.empty((0, 64), dtype=BF, device="cuda")
    table = torch.ones((8, 32), device="cuda")
    worker.run(runtime.rope_append_tokens, torch.empty((0, 3 * 64), dtype=BF, device="cuda"), _ints([]), b.starts, b.ctx, table, table, b.blocks, b.key,
               b.value, q, 1, 1, 64, 16)
    worker.run(runtime.tree_attention, q, b.key, b.value, b.blocks, b.ctx, b.starts, torch.empty((0, 1), dtype=torch.int32, device="cuda"),
               torch.empty_like(q), 1, 1, 64, 16, 1.0)
    z = torch.empty(0, device="cuda")
    worker.run(runtime.sample_tokens, torch.empty((0, 50), device="cuda"), z, _ints([]), z, z, z, _ints([]), z.clone())
    worker.sync()
