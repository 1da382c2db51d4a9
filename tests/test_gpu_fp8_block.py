"""Block-scaled e4m3 operators on the GPU - norm and quantiser, product, router, experts - against the 64-bit oracle."""

import pytest
import torch

from oracle import fp8_block as ob
from pypto_amd import _lib, runtime

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}  # relative, of a rounding to the type
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}    # half a step among the smallest values
GUARD = 256


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(shape, device="cuda", generator=g)


class _Fenced:
    """A tensor with a fence of known bytes on either side of it, checked by intact()."""

    def __init__(self, shape, dtype, fill=0x5B, inside=None):
        n = torch.Size(shape).numel() * torch.empty(0, dtype=dtype).element_size()
        self.buf = torch.full((2 * GUARD + (n + 15) // 16 * 16,), fill, dtype=torch.uint8, device="cuda")
        self.n, self.fill = n, fill
        self.t = self.buf[GUARD:GUARD + n].view(dtype).view(shape)
        if inside is not None:
            self.t.copy_(inside)

    def intact(self):
        return bool((self.buf[:GUARD] == self.fill).all() and (self.buf[GUARD + self.n:] == self.fill).all())


def _codes_of(values):
    """Codes between fences of NaN codes."""
    return _Fenced(values.shape, F8, fill=0x7F, inside=values.to(F8)).t


# ---- norm and quantiser --------------------------------------------------------------------------------

NORM_SHAPES = [(2100, 8200), (1, 8), (3, 120), (2, 128), (5, 136), (7, 1000), (4, 2048), (3, 2056), (2, 4104), (33, 5120), (3, 8200), (2, 16384)]


def _check_codes(codes, scale, n, slack):
    """Codes and scales against the exact rows n: every value within half a step of its group's scale, `slack` relative aside."""
    cols = n.shape[-1]
    wide = scale.double().repeat_interleave(128, -1)[:, :cols]
    _, want = ob.quantize_rows(n)
    assert ((scale.double() - want).abs() <= want * (slack + 2.0 ** -23)).all()
    got = codes.double() * wide
    half = torch.maximum(n.abs() * 2.0 ** -4, wide * 2.0 ** -10)
    assert ((got - n).abs() <= half * (1 + 2.0 ** -20) + slack * n.abs()).all()


@pytest.mark.parametrize("rows,cols", NORM_SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("normed", [False, True])
def test_norm(worker, rows, cols, dtype, residual, normed):
    """The sum's rounding is exact; the norm's fp32 evaluation is off by at most 2^-17: 64 squares in a row and 8 + log2(256) joins are 80
    half-ulps of 2^-24, halved by the root, and half a dozen roundings behind it."""
    g = _gen(rows * cols)
    x, r = (_randn(g, rows, cols) * 3).to(dtype), (_randn(g, rows, cols) * torch.where(torch.rand(cols, device="cuda", generator=g) < 0.05, 30.0, 1.0)).to(dtype)
    if rows > 1:
        x[1], r[1] = 0, 0  # a row of zeros: every group's scale is 1
    gamma = 1 + 0.2 * _randn(g, cols)
    codes, scale = _Fenced((rows, cols), F8), _Fenced((rows, -(-cols // 128)), torch.float32)
    sums, out = _Fenced((rows, cols), dtype), _Fenced((rows, cols), dtype)
    program = {(0, 0): runtime.rms_norm_fp8_block, (0, 1): runtime.rms_norm_fp8_block_normed, (1, 0): runtime.add_rms_norm_fp8_block,
               (1, 1): runtime.add_rms_norm_fp8_block_normed}[residual, normed]
    worker.run(program, x, *((r,) if residual else ()), gamma, *((sums.t,) if residual else ()), *((out.t,) if normed else ()), codes.t, scale.t, 1e-6)
    worker.sync()
    s, n = ob.rms_norm(x, r if residual else None, gamma, 1e-6)
    slack = 2.0 ** -17
    _check_codes(codes.t, scale.t, n, slack)
    if rows > 1:
        assert (scale.t[1] == 1).all() and (codes.t[1].float() == 0).all()
    if residual:
        assert torch.equal(sums.t, (x.float() + r.float()).to(dtype))
    if normed:
        assert ((out.t.double() - n).abs() <= n.abs() * (HALF_STEP[dtype] + slack) + TINY[dtype]).all()
    assert all(f.intact() for f in (codes, scale, sums, out))


def test_norm_in_place_and_without_a_weight(worker):
    """sum_out may be x or residual, normed_out x: the calls have the bits of the one with buffers of their own."""
    lib, g = _lib.load(), _gen(5)
    x, r = _randn(g, 9, 4104).bfloat16(), _randn(g, 9, 4104).bfloat16()

    def call(x, r, s, n):
        codes, scale = torch.zeros((9, 4104), dtype=torch.uint8, device="cuda"), torch.zeros((9, 33), device="cuda")
        _lib.check(lib.pto_hip_rms_norm_fp8_block(x.data_ptr(), r.data_ptr(), None, s.data_ptr(), n.data_ptr(), codes.data_ptr(), scale.data_ptr(),
                                                  9, 4104, 1e-5, 0x40, None))
        worker.sync()
        return s.clone(), n.clone(), codes, scale

    want = call(x, r, torch.empty_like(x), torch.empty_like(x))
    _check_codes(want[2].view(F8), want[3], ob.rms_norm(x, r, None, 1e-5)[1], 2.0 ** -17)
    for which in ("x", "r"):
        a, b = x.clone(), r.clone()
        got = call(a, b, a if which == "x" else b, b if which == "x" else a)
        assert all(torch.equal(p, q) for p, q in zip(got, want))
    assert lib.pto_hip_rms_norm_fp8_block(x.data_ptr(), r.data_ptr(), None, x.data_ptr(), x.data_ptr(), want[2].data_ptr(), want[3].data_ptr(), 9,
                                          4104, 1e-5, 0x40, None) == _lib.ERR_INVALID_VALUE


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,cols", [(1, 8), (5, 200), (3, 4096), (2, 16384)])
def test_quantiser_is_exact(worker, dtype, rows, cols):
    """Without a norm nothing is computed but the scale's division and the quotients: the codes are the oracle's to the bit."""
    g = _gen(cols)
    x = (_randn(g, rows, cols) * torch.exp2(torch.randint(-14, 8, (rows, 1), device="cuda", generator=g).float())).to(dtype)
    x[0, :8] = 0
    codes, scale = _Fenced((rows, cols), F8), _Fenced((rows, -(-cols // 128)), torch.float32)
    worker.run(runtime.quantize_fp8_block, x, codes.t, scale.t)
    worker.sync()
    # on the CPU: torch multiplies by 1 / 448 on the GPU, which is not the division
    x = x.cpu().float()
    amax = torch.nn.functional.pad(x, (0, -cols % 128)).unflatten(-1, (-1, 128)).abs().amax(-1)
    want = torch.where(amax > 0, (amax / 448).clamp(min=2.0 ** -126), 1.0)
    assert torch.equal(scale.t.cpu(), want)
    wide = want.repeat_interleave(128, -1)[:, :cols]
    assert torch.equal(codes.t.cpu().view(torch.uint8), (x / wide).to(F8).view(torch.uint8))
    assert codes.intact() and scale.intact()


def test_quantiser_on_infinities_nan_and_the_smallest_values(worker):
    x = torch.zeros((6, 256), dtype=torch.bfloat16, device="cuda")
    x[0, 3], x[0, 200] = float("inf"), 5.0
    x[1, 7], x[1, 8] = float("nan"), 2.0
    x[2, 0], x[2, 1] = 2.0 ** -133, -2.0 ** -130  # subnormal: the scale stays a normal number
    x[3, 0] = -0.0
    x[4, 5], x[4, 6] = 3e38, 1e30
    x[5, 100] = -float("inf")
    codes, scale = torch.zeros((6, 256), dtype=F8, device="cuda"), torch.zeros((6, 2), device="cuda")
    worker.run(runtime.quantize_fp8_block, x, codes, scale)
    worker.sync()
    c, s = codes.float().cpu(), scale.cpu()
    assert s[0, 0] == float("inf") and c[0, 3].isnan() and (c[0, 4:128] == 0).all() and c[0, 200] == 448
    assert c[1, 7].isnan() and c[1, 8] == 448 and s[1, 0] == torch.tensor(2.0) / 448
    assert s[2, 0] == 2.0 ** -126 and c[2, 0] == 2.0 ** -7 and c[2, 1] == -2.0 ** -4
    assert codes.view(torch.uint8)[3, 0].item() == 0x80 and s[3, 0] == 1
    assert c[4, 5] == 448 and c[4, 6] == 0
    assert c[5, 100].isnan() and s[5, 1] == 1


# ---- product -------------------------------------------------------------------------------------------

# rows and channels at, below and above every tile's; one block of k to many, with and without an odd one behind
PRODUCT_SHAPES = [(1, 128, 1), (1, 4096, 130), (3, 256, 5), (15, 384, 100), (16, 512, 128), (17, 640, 129), (33, 1024, 257), (64, 1152, 384), (65, 2816, 100),
                  (127, 896, 511), (128, 128, 256), (130, 4224, 48), (255, 1664, 260), (257, 512, 1003), (300, 2048, 640), (513, 768, 321)]


def _product(worker, a, sa, w, sw, dtype):
    out = _Fenced((a.shape[0], w.shape[0]), dtype)
    worker.run(runtime.projection_fp8_block, a, sa, w, sw, out.t)
    worker.sync()
    assert out.intact()
    return out.t


@pytest.fixture(params=[0, 16, 64, 128, 256])
def rows(request, worker):
    """Every height of a product's tiles, the library's own choice first."""
    worker.set_option("block_gemm_rows", request.param)
    yield request.param
    worker.set_option("block_gemm_rows", 0)


# ... and, of a projection's, every width and several ranges of k
@pytest.fixture(params=[(0, 0, 0), (16, 0, 0), (64, 64, 0), (64, 128, 0), (64, 256, 0), (128, 0, 0), (256, 0, 0), (64, 64, 3), (64, 128, 2), (64, 256, 4),
                        (128, 0, 3), (256, 0, 2)], ids=str)
def tile(request, worker):
    for name, value in zip(("block_gemm_rows", "block_gemm_cols", "gemm_splits"), request.param):
        worker.set_option(name, value)
    yield request.param
    for name in ("block_gemm_rows", "block_gemm_cols", "gemm_splits"):
        worker.set_option(name, 0)


@pytest.mark.parametrize("m,k,n", PRODUCT_SHAPES)
def test_product_is_exact_on_whole_numbers_and_stays_inside(worker, tile, m, k, n):
    """Whole numbers up to 8 and scales of 2^-8 and 2^-7: every sum is a multiple of 2^-16 below 64 * 4224 * 2^-14, which
    fp32 holds exactly in any order.  Past the operands' ends lie NaN codes."""
    g = torch.Generator().manual_seed(m + k + n)
    num = lambda count: torch.randint(-8, 9, (count, k), generator=g).float()
    scale = lambda count: torch.exp2(-7.0 - torch.randint(0, 2, (count, k // 128), generator=g).float())
    a, w, sa, sw = num(m), num(n), scale(m), scale(-(-n // 128))
    want = ob.projection(a.cuda(), sa.cuda(), w.cuda(), sw.cuda())
    fenced = lambda t: _Fenced(t.shape, torch.float32, fill=0xFF, inside=t).t  # all ones: a NaN
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        got = _product(worker, _codes_of(a), fenced(sa), _codes_of(w), fenced(sw), dtype)
        assert torch.equal(got, want.float().to(dtype)), dtype


@pytest.mark.parametrize("tile", [(0, 0, 0), (16, 0, 0)], ids=str, indirect=True)
@pytest.mark.parametrize("m,k,n", [(1, 256, 4200), (16, 1152, 4097), (3, 3968, 5003), (5, 640, 8192), (1, 128, 8193), (16, 1408, 8300), (9, 4096, 9000), (40, 512, 8200)])
def test_product_of_few_rows_and_many_channels(worker, tile, m, k, n):
    """16 or 32 channels a workgroup, four or eight wavefronts: their steps end unevenly."""
    a, sa, w, sw = _operands(_gen(k + n), m, k, n)
    for dtype in (torch.float32, torch.float16):
        got = _product(worker, a, sa, w, sw, dtype).double()
        want = ob.projection(a, sa, w, sw)
        bound = (ob.dequantize_rows(a, sa).abs() @ ob.dequantize_matrix(w, sw).abs().t()) * (132 + k // 128) * 2.0 ** -24
        assert ((got - want).abs() <= bound + (want.abs() + bound) * HALF_STEP[dtype] + TINY[dtype]).all()


def _operands(g, m, k, n):
    a, sa = ob.quantize_rows(_randn(g, m, k))
    w, sw = ob.quantize_matrix(_randn(g, n, k) * k ** -0.5)
    return a.to(F8), sa.float(), w, sw


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k,n", [(1, 4096, 515), (24, 2816, 96), (130, 4096, 256), (300, 11008, 300), (600, 1024, 900)])
def test_product_on_quantised_values(worker, tile, m, k, n, dtype):
    """fp32 sums of k products in any order: at most (128 + k / 128 + 4) roundings in a row, each of the sum of magnitudes."""
    a, sa, w, sw = _operands(_gen(k + n), m, k, n)
    got = _product(worker, a, sa, w, sw, dtype).double()
    want = ob.projection(a, sa, w, sw)
    sizes = ob.dequantize_rows(a, sa).abs() @ ob.dequantize_matrix(w, sw).abs().t()
    bound = sizes * (132 + k // 128) * 2.0 ** -24
    assert ((got - want).abs() <= bound + (want.abs() + bound) * HALF_STEP[dtype] + TINY[dtype]).all()


def test_product_rows_do_not_depend_on_their_batch(worker, tile):
    """A row's scales and codes are its own: NaN in one row stays in that row."""
    a, sa, w, sw = _operands(_gen(9), 70, 1024, 260)
    want = _product(worker, a, sa, w, sw, torch.float32)
    bad = a.clone()
    bad.view(torch.uint8)[33, 5] = 0x7F
    got = _product(worker, bad, sa, w, sw, torch.float32)
    assert got[33].isnan().all()
    keep = torch.arange(70, device="cuda") != 33
    assert torch.equal(got[keep], want[keep])


def test_product_refusals(worker):
    a, sa, w, sw = _operands(_gen(1), 4, 256, 200)
    out = torch.zeros((4, 200), dtype=torch.bfloat16, device="cuda")
    run = lambda *args: worker.run(runtime.projection_fp8_block, *args)
    with pytest.raises(ValueError, match="a8 must be FP8E4M3FN"):
        run(a.float(), sa, w, sw, out)
    with pytest.raises(ValueError, match=r"scales of a8 must be FP32 \[4, 2\]"):
        run(a, sa[:, :1].contiguous(), w, sw, out)
    with pytest.raises(ValueError, match="w8 must be"):
        run(a, sa, w[:, :128].contiguous(), sw, out)
    with pytest.raises(ValueError, match=r"w_scale must be FP32 \[2, 2\]"):
        run(a, sa, w, sw[:1].contiguous(), out)
    with pytest.raises(ValueError, match=r"out must be \[M, N\]"):
        run(a, sa, w, sw, out[:, :100].contiguous())
    with pytest.raises(ValueError, match="contiguous"):
        run(a, sa, w, sw, out.t())
    with pytest.raises(ValueError, match="multiple of 16"):
        run(torch.zeros(4 * 256 + 8, dtype=torch.uint8, device="cuda")[8:].view(F8).view(4, 256), sa, w, sw, out)
    run(a[:0], sa[:0], w, sw, out[:0])  # no rows: nothing happens
    worker.sync()


# ---- router --------------------------------------------------------------------------------------------


def _route(worker, logits, bias, top_k, n_groups=1, topk_groups=1, sigmoid=False, renormalize=True, scale=1.0):
    t = logits.shape[0]
    ids, weights = _Fenced((t, top_k), torch.int32), _Fenced((t, top_k), torch.float32)
    worker.run(runtime.route_experts if bias is None else runtime.route_experts_biased, logits, *(() if bias is None else (bias,)), ids.t,
               weights.t, n_groups, topk_groups, int(sigmoid), int(renormalize), scale)
    worker.sync()
    assert ids.intact() and weights.intact()
    return ids.t, weights.t


def _check_route(worker, logits, bias, *args, **kw):
    ids, weights = _route(worker, logits, bias, *args, **kw)
    want, w = ob.route(logits.cpu(), None if bias is None else bias.cpu(), *args, **kw)
    assert torch.equal(ids.cpu(), want)
    # one rounding at the end and, in 32 bits, a few of an exponential and a sum of up to 1024
    assert ((weights.cpu().double() - w).abs() <= w.abs() * 2.0 ** -20 + 2.0 ** -140).all()


@pytest.mark.parametrize("experts,top_k,groups,kept", [(1, 1, 1, 1), (8, 2, 1, 1), (60, 4, 1, 1), (64, 6, 8, 3), (65, 65 - 1, 1, 1), (128, 8, 4, 4), (160, 6, 8, 3),
                                                       (256, 8, 8, 4), (320, 10, 64, 7), (512, 8, 16, 2), (1000, 3, 50, 20), (1024, 64, 64, 64)])
@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("biased", [False, True])
def test_router(worker, experts, top_k, groups, kept, sigmoid, biased):
    g = _gen(experts + top_k)
    bias = 0.1 * _randn(g, experts) if biased else None
    for tokens, dtype in ((1, torch.float32), (37, torch.float32), (30, torch.bfloat16), (9, torch.float16)):
        logits = (_randn(g, tokens, experts) * 2).to(dtype)
        _check_route(worker, logits, bias, top_k, groups, kept, sigmoid=sigmoid, renormalize=tokens != 9, scale=2.5)


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("biased", [False, True])
def test_router_ties_go_to_the_lowest_index(worker, sigmoid, biased):
    """Few distinct logits, so that most choices are ties; with a bias of zeros as well as without."""
    g = _gen(3)
    for experts, groups, kept in ((64, 1, 1), (256, 8, 3), (130, 5, 2)):
        logits = torch.randint(-2, 3, (25, experts), device="cuda", generator=g).float()
        _check_route(worker, logits, torch.zeros(experts, device="cuda") if biased else None, 7, groups, kept, sigmoid=sigmoid)
        _check_route(worker, torch.zeros_like(logits), torch.zeros(experts, device="cuda") if biased else None, 7, groups, kept, sigmoid=sigmoid)


def test_router_keys_that_differ_past_32_bits(worker):
    """Two experts whose keys differ by less than an ulp of 32 bits, either way round."""
    logits = torch.full((2, 96), -4.0, device="cuda")
    logits[:, 10], logits[:, 70] = 0.0, 0.0
    bias = torch.zeros(96, device="cuda")
    bias[10], bias[70] = 1.0, 1.0
    logits[0, 70], logits[1, 10] = 1e-9, 1e-9
    ids, _ = _route(worker, logits, bias, 2, sigmoid=True)
    assert ids.tolist() == [[70, 10], [10, 70]]
    _check_route(worker, logits, bias, 2, sigmoid=True)


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("groups,kept", [(1, 1), (4, 2)])
def test_router_on_rows_that_leave_little(worker, sigmoid, biased, groups, kept):
    inf, nan, low = float("inf"), float("nan"), torch.finfo(torch.float32).min
    logits = _randn(_gen(4), 9, 72)
    logits[0] = -inf
    logits[1] = low
    logits[2, 3:] = -inf
    logits[3, ::2] = nan
    logits[4] = nan
    logits[5, 5] = inf
    logits[6, 5], logits[6, 60], logits[6, 61] = inf, inf, nan
    logits[7] = inf
    logits[8, :70] = low
    bias = None
    if biased:
        bias = 0.1 * _randn(_gen(5), 72)
        bias[2], bias[40] = -inf, nan
    _check_route(worker, logits, bias, 5, groups, kept, sigmoid=sigmoid)


def test_router_refusals(worker):
    logits = torch.zeros((4, 64), device="cuda")
    ids, w = torch.zeros((4, 6), dtype=torch.int32, device="cuda"), torch.zeros((4, 6), device="cuda")
    run = lambda *a: worker.run(runtime.route_experts, *a)
    with pytest.raises(ValueError, match="logits dtype INT32"):
        run(logits.int(), ids, w, 1, 1, 0, 1, 1.0)
    with pytest.raises(ValueError, match="expert_ids must be INT32"):
        run(logits, ids.long(), w, 1, 1, 0, 1, 1.0)
    with pytest.raises(ValueError, match="expert_weights must be FP32"):
        run(logits, ids, w[:, :5].contiguous(), 1, 1, 0, 1, 1.0)
    with pytest.raises(ValueError, match="bias must be FP32 with 64"):
        worker.run(runtime.route_experts_biased, logits, torch.zeros(63, device="cuda"), ids, w, 1, 1, 0, 1, 1.0)
    with pytest.raises(ValueError, match="neither softmax"):
        run(logits, ids, w, 1, 1, -1, 1, 1.0)
    with pytest.raises(ValueError, match="do not divide"):
        run(logits, ids, w, 5, 1, 0, 1, 1.0)
    run(logits[:0], ids[:0], w[:0], 1, 1, 0, 1, 1.0)
    worker.sync()


# ---- experts -------------------------------------------------------------------------------------------


def _experts_case(seed, tokens, hidden, inter, experts, top_k):
    g = _gen(seed)
    x, xs = ob.quantize_rows(_randn(g, tokens, hidden))
    ids = torch.rand((tokens, experts), device="cuda", generator=g).argsort(-1)[:, :top_k]
    if ids.shape[1] < top_k:
        ids = torch.randint(0, experts, (tokens, top_k), device="cuda", generator=g)
    w = torch.rand((tokens, top_k), device="cuda", generator=g) + 0.1
    mats = []
    for n, k in ((inter, hidden), (inter, hidden), (hidden, inter)):
        mats += list(ob.quantize_matrix(_randn(g, experts, n, k) * (2.0 * k ** -0.5)))
    return [x.to(F8), xs.float(), ids.int().contiguous(), w] + mats


def _check_experts(worker, args, dtype):
    out = _Fenced(args[0].shape, dtype)
    worker.run(runtime.experts_ffn_fp8_block, *args, out.t)
    worker.sync()
    want, slack = ob.experts_ffn(*args)
    # slack: codes of h next to a border, and fp32 sums on both sides of the codes
    bad = ((out.t.double() - want).abs() > slack * (1 + HALF_STEP[dtype]) + want.abs() * HALF_STEP[dtype] + TINY[dtype]).sum().item()
    assert bad == 0 and out.intact(), bad
    return out.t


EXPERT_SHAPES = [(1, 256, 128, 4, 2), (1, 1024, 1408, 16, 8), (2, 128, 256, 8, 1), (3, 512, 384, 8, 8), (7, 640, 256, 60, 4), (16, 256, 128, 1, 1), (40, 512, 512, 60, 4),
                 (33, 384, 128, 2, 2), (100, 1024, 256, 16, 2), (130, 256, 640, 8, 3), (300, 512, 256, 8, 2), (515, 1152, 384, 4, 2), (700, 256, 256, 64, 8)]


@pytest.mark.parametrize("tokens,hidden,inter,experts,top_k", EXPERT_SHAPES)
def test_experts(worker, rows, tokens, hidden, inter, experts, top_k):
    args = _experts_case(tokens + hidden, tokens, hidden, inter, experts, top_k)
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        _check_experts(worker, args, dtype)


@pytest.mark.parametrize("tokens", [1, 5, 90, 600])
def test_experts_on_uneven_routes(worker, rows, tokens):
    """Slots without an expert, tokens without any, one expert for all, the same expert twice in a row."""
    args = _experts_case(tokens, tokens, 384, 256, 12, 4)
    ids = args[2]
    ids[::3, 1] = -1
    ids[::2, 3] = -(2 ** 31)
    ids[-1] = -1
    out = _check_experts(worker, args, torch.bfloat16)
    assert (out[-1] == 0).all()
    ids[:] = 7
    _check_experts(worker, args, torch.bfloat16)
    ids[:] = -1
    assert (_check_experts(worker, args, torch.float32) == 0).all()


def test_an_expert_that_there_is_not_is_left_out_and_reported(worker):
    args = _experts_case(2, 6, 256, 128, 4, 2)
    args[2][3, 0] = 4
    args[2][5, 1] = 2 ** 31 - 1
    out = torch.empty((6, 256), dtype=torch.float32, device="cuda")
    worker.run(runtime.experts_ffn_fp8_block, *args, out)
    with pytest.raises(ValueError, match="an expert that there is not"):
        worker.sync()
    worker.sync()  # reported once
    want, slack = ob.experts_ffn(*args)
    assert ((out.double() - want).abs() <= slack + want.abs() * 2.0 ** -24).all()


def test_a_token_s_result_does_not_depend_on_its_batch(worker, rows):
    """NaN and infinities of one token, and weights that nobody asked for, reach no other token."""
    args = _experts_case(8, 50, 512, 256, 16, 3)
    args[2].clamp_(max=14)
    want = _check_experts(worker, args, torch.float32)
    for i in (4, 6, 8):
        args[i].view(torch.uint8)[15] = 0x7F
    x = args[0].clone()
    x.view(torch.uint8)[20] = 0x7F
    args[1][20] = float("inf")
    out = torch.empty_like(want)
    worker.run(runtime.experts_ffn_fp8_block, x, *args[1:], out)
    worker.sync()
    keep = torch.arange(50, device="cuda") != 20
    assert out[20].isnan().all() and torch.equal(out[keep], want[keep])


def test_experts_refusals(worker):
    args = _experts_case(3, 4, 256, 128, 4, 2)
    out = torch.zeros((4, 256), dtype=torch.bfloat16, device="cuda")

    def run(i, t, out=out):
        worker.run(runtime.experts_ffn_fp8_block, *args[:i], t, *args[i + 1:], out)

    with pytest.raises(ValueError, match="x8 must be FP8E4M3FN"):
        run(0, args[0].float())
    with pytest.raises(ValueError, match="scales of x8"):
        run(1, args[1][:, :1].contiguous())
    with pytest.raises(ValueError, match="expert_ids must be INT32"):
        run(2, args[2].long())
    with pytest.raises(ValueError, match="expert_weights must be FP32"):
        run(3, args[3].bfloat16())
    with pytest.raises(ValueError, match="w_up8 must be"):
        run(6, args[6][:3].contiguous())
    with pytest.raises(ValueError, match="w_down_scale must be FP32"):
        run(9, args[9][:, :1].contiguous())
    with pytest.raises(ValueError, match=r"out must be \[T, H\]"):
        run(0, args[0], out[:2])
    worker.run(runtime.experts_ffn_fp8_block, args[0][:0], args[1][:0], args[2][:0], args[3][:0], *args[4:], out[:0])
    worker.sync()


# ---- together ------------------------------------------------------------------------------------------


class _Layer:
    """The feed-forward half of a mixture layer as a serving loop calls it, on buffers of its own."""

    def __init__(self, worker, tokens, hidden, inter, experts, top_k, seed):
        g = _gen(seed)
        self.w = worker
        self.h = {p: worker.register(getattr(runtime, p)) for p in ("add_rms_norm_fp8_block_normed", "projection", "route_experts_biased", "experts_ffn_fp8_block")}
        new = lambda shape, dtype: torch.empty(shape, dtype=dtype, device="cuda")
        self.x, self.res = _randn(g, tokens, hidden).bfloat16(), (2 * _randn(g, tokens, hidden)).bfloat16()
        self.gamma, self.router = 1 + 0.1 * _randn(g, hidden), (_randn(g, hidden, experts) * hidden ** -0.5).bfloat16()
        self.bias = 0.1 * _randn(g, experts)
        self.mats = _experts_case(seed, 1, hidden, inter, experts, 1)[4:]
        self.sum, self.normed, self.out = new((tokens, hidden), torch.bfloat16), new((tokens, hidden), torch.bfloat16), new((tokens, hidden), torch.bfloat16)
        self.codes, self.scale = new((tokens, hidden), F8), new((tokens, hidden // 128), torch.float32)
        self.logits, self.ids, self.weights = new((tokens, experts), torch.float32), new((tokens, top_k), torch.int32), new((tokens, top_k), torch.float32)
        self.top_k = top_k

    def step(self, stream=0):
        call = lambda p, *a: self.h[p](*a, stream=stream)
        call("add_rms_norm_fp8_block_normed", self.x, self.res, self.gamma, self.sum, self.normed, self.codes, self.scale, 1e-6)
        call("projection", self.normed, self.router, self.logits)
        call("route_experts_biased", self.logits, self.bias, self.ids, self.weights, 4, 2, 1, 1, 2.0)
        call("experts_ffn_fp8_block", self.codes, self.scale, self.ids, self.weights, *self.mats, self.out)

    def check(self):
        s, n = ob.rms_norm(self.x, self.res, self.gamma, 1e-6)
        _check_codes(self.codes, self.scale, n, 2.0 ** -17)
        want, w = ob.route(self.logits.cpu(), self.bias.cpu(), self.top_k, 4, 2, sigmoid=True, scale=2.0)
        assert torch.equal(self.ids.cpu(), want) and torch.allclose(self.weights.cpu().double(), w, rtol=2.0 ** -20, atol=0)
        logits = self.normed.double() @ self.router.double()
        sizes = self.normed.double().abs() @ self.router.double().abs()
        assert ((self.logits.double() - logits).abs() <= sizes * self.x.shape[1] * 2.0 ** -24).all()
        out, slack = ob.experts_ffn(self.codes, self.scale, self.ids, self.weights, *self.mats)
        assert ((self.out.double() - out).abs() <= slack * (1 + 2.0 ** -8) + out.abs() * 2.0 ** -8 + 2.0 ** -134).all()

    def results(self):
        return [t.clone() for t in (self.sum, self.normed, self.codes.view(torch.uint8), self.scale, self.logits, self.ids, self.weights, self.out)]


@pytest.mark.parametrize("tokens", [1, 3, 50, 400])
def test_the_operators_of_a_layer_together(worker, tokens):
    layer = _Layer(worker, tokens, 512, 256, 16, 4, seed=tokens)
    layer.step()
    worker.sync()
    layer.check()


@pytest.mark.parametrize("tokens", [1, 3, 50, 400])
def test_a_captured_layer_on_another_stream(worker, tokens):
    """Recorded once, replayed with other inputs and with eager calls of another size between the replays; every replay has the
    bits of an eager call on its inputs."""
    layer, other = _Layer(worker, tokens, 512, 256, 16, 4, seed=tokens), _Layer(worker, 7, 512, 256, 16, 4, seed=99)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        layer.step(stream.cuda_stream)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        layer.step(torch.cuda.current_stream().cuda_stream)
    for i in range(4):
        layer.x.copy_(_randn(_gen(i), *layer.x.shape))
        torch.cuda.synchronize()
        layer.step()
        worker.sync()
        want = layer.results()
        for t in (layer.sum, layer.normed, layer.scale, layer.logits, layer.weights, layer.out):
            t.fill_(float("nan"))
        layer.ids.fill_(-1)
        other.step()
        worker.sync()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(layer.results(), want)), i
    worker.sync()


# ---- the ends of what is allowed -----------------------------------------------------------------------


def test_norm_of_more_rows_than_a_launch_holds(worker):
    """The last rows have the bits of a call on them alone."""
    rows, cols, last = (1 << 23) + 5, 8, 9
    g = _gen(1)
    x, r, gamma = _randn(g, rows, cols).bfloat16(), _randn(g, rows, cols).bfloat16(), 1 + 0.1 * _randn(g, cols)

    def call(x, r):
        n = len(x)
        outs = [torch.empty((n, cols), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        outs += [torch.empty((n, cols), dtype=F8, device="cuda"), torch.empty((n, 1), device="cuda")]
        worker.run(runtime.add_rms_norm_fp8_block_normed, x, r, gamma, *outs, 1e-6)
        worker.sync()
        outs[2] = outs[2].view(torch.uint8)
        return outs

    for got, want in zip(call(x, r), call(x[-last:].contiguous(), r[-last:].contiguous())):
        assert torch.equal(got[-last:], want)


def test_router_of_more_tokens_than_a_launch_holds(worker):
    tokens, last = (1 << 25) + 3, 7
    logits = torch.randint(-100, 100, (tokens, 3), dtype=torch.int8, device="cuda", generator=_gen(2)).bfloat16()
    bias = torch.tensor([0.0, 0.1, -0.1], device="cuda")

    def call(logits):
        ids, weights = torch.empty((len(logits), 2), dtype=torch.int32, device="cuda"), torch.empty((len(logits), 2), device="cuda")
        worker.run(runtime.route_experts_biased, logits, bias, ids, weights, 1, 1, 1, 1, 1.0)
        worker.sync()
        return ids, weights

    for got, want in zip(call(logits), call(logits[-last:].contiguous())):
        assert torch.equal(got[-last:], want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m", [3, 16, 70])
def test_product_of_the_longest_rows(worker, tile, m, dtype):
    a, sa, w, sw = _operands(_gen(m), m, 65536, 130)
    got = _product(worker, a, sa, w, sw, dtype).double()
    want = ob.projection(a, sa, w, sw)
    sizes = ob.dequantize_rows(a, sa).abs() @ ob.dequantize_matrix(w, sw).abs().t()
    bound = sizes * (132 + 512) * 2.0 ** -24
    assert ((got - want).abs() <= bound + (want.abs() + bound) * HALF_STEP[dtype] + TINY[dtype]).all()


@pytest.mark.parametrize("m,k,n", [(5, 384, 100), (130, 640, 256), (300, 1024, 512)])
def test_product_on_scales_and_results_aligned_to_their_elements(worker, tile, m, k, n):
    """One element behind a 16-byte boundary: the bits of the call on aligned ones."""
    a, sa, w, sw = _operands(_gen(k), m, k, n)
    shifted = lambda t: torch.cat([t.new_zeros(1), t.flatten()])[1:].view(t.shape)
    want = _product(worker, a, sa, w, sw, torch.float32)
    out = _Fenced((m * n + 1,), torch.float32)
    worker.run(runtime.projection_fp8_block, a, shifted(sa), w, shifted(sw), out.t[1:].view(m, n))
    worker.sync()
    assert torch.equal(out.t[1:].view(m, n), want) and out.intact()


@pytest.mark.parametrize("tile", [(0, 0, 0), (64, 64, 0), (64, 128, 0), (64, 256, 0), (128, 0, 0), (256, 0, 0)], ids=str, indirect=True)
def test_product_past_32_bits(worker, tile):
    """Rows that lie beyond the first 4 GB of codes, and results beyond the first 4 GB."""
    m, k, n, last = (1 << 18) + 33, 16512, 8320, 40
    a = torch.empty((m, k), dtype=torch.uint8, device="cuda")
    sa = torch.empty((m, k // 128), device="cuda")
    tail, scales, w, sw = _operands(_gen(3), last, k, n)
    a[:], sa[:] = 0, 1
    a[-last:], sa[-last:] = tail.view(torch.uint8), scales
    out = torch.empty((m, n), dtype=torch.bfloat16, device="cuda")
    worker.run(runtime.projection_fp8_block, a.view(F8), sa, w, sw, out)
    worker.sync()
    want = ob.projection(tail, scales, w, sw)
    bound = (ob.dequantize_rows(tail, scales).abs() @ ob.dequantize_matrix(w, sw).abs().t()) * (132 + k // 128) * 2.0 ** -24
    assert ((out[-last:].double() - want).abs() <= bound + (want.abs() + bound) * 2.0 ** -8 + 2.0 ** -134).all()
    assert (out[:-last].view(torch.int16) == 0).all()


@pytest.mark.parametrize("tokens,hidden,inter,experts,top_k", [(4200, 256, 128, 16, 8), (2, 128, 128, 1024, 64), (40, 128, 256, 1024, 64), (520, 128, 128, 1024, 64),
                                                               (2, 65536, 128, 2, 2), (70, 65536, 128, 2, 1), (2, 128, 65536, 2, 1), (70, 128, 65536, 2, 1)])
def test_experts_at_the_ends(worker, tokens, hidden, inter, experts, top_k):
    """Several passes, the most experts and slots of a token, the longest rows; recorded and replayed with the bits of the eager call."""
    args = _experts_case(tokens + hidden, tokens, hidden, inter, experts, top_k)
    run = worker.register(runtime.experts_ffn_fp8_block)
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        want = _check_experts(worker, args, dtype)
        out, graph = torch.empty_like(want), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run(*args, out, stream=torch.cuda.current_stream().cuda_stream)
        for _ in range(3):
            out.fill_(float("nan"))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
    worker.sync()


@pytest.mark.parametrize("tokens", [2, 100])
def test_experts_past_32_bits(worker, tokens):
    """The last of 66 experts, whose matrices lie beyond the first 4 GB: the bits of a call that has it alone."""
    experts, hidden, inter = 66, 8192, 8320
    alone = _experts_case(4, tokens, hidden, inter, 1, 1)
    args = list(alone)
    for i in range(4, 10):
        args[i] = torch.empty((experts, *alone[i].shape[1:]), dtype=alone[i].dtype, device="cuda")
        args[i][-1].view(torch.uint8 if i % 2 == 0 else torch.float32).copy_(alone[i][0].view(torch.uint8 if i % 2 == 0 else torch.float32))
    args[2] = torch.full_like(alone[2], experts - 1)
    outs = []
    worker.set_option("block_gemm_rows", 16 if tokens < 16 else 64)
    try:
        for case in (args, alone):
            outs.append(torch.empty((tokens, hidden), dtype=torch.float32, device="cuda"))
            worker.run(runtime.experts_ffn_fp8_block, *case, outs[-1])
            worker.sync()
    finally:
        worker.set_option("block_gemm_rows", 0)
    assert outs[1].isfinite().all() and outs[1].abs().max() > 0 and torch.equal(*outs)


def test_two_threads_on_one_stream(worker):
    """Calls of two threads are issued one after the other: each has the results of its own call."""
    import threading

    cases = [_experts_case(i, 300 + 40 * i, 512, 256, 16, 4) for i in range(2)]
    want = [_check_experts(worker, c, torch.bfloat16) for c in cases]
    outs = [[torch.empty_like(w) for _ in range(20)] for w in want]
    run, errors = worker.register(runtime.experts_ffn_fp8_block), []

    def work(i):
        try:
            for out in outs[i]:
                run(*cases[i], out)
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    worker.sync()
    assert not errors
    assert all(torch.equal(out, w) for outs_i, w in zip(outs, want) for out in outs_i)


@pytest.mark.parametrize("experts,top_k,groups,kept", [(256, 8, 8, 4), (64, 6, 1, 1), (512, 10, 32, 5)])
@pytest.mark.parametrize("sigmoid", [False, True])
def test_router_of_many_tokens(worker, experts, top_k, groups, kept, sigmoid):
    """Enough of them that some choices fall between keys, and groups, that 32 bits do not tell apart."""
    g = _gen(experts)
    logits = _randn(g, 5000, experts).bfloat16()
    _check_route(worker, logits, 0.01 * _randn(g, experts), top_k, groups, kept, sigmoid=sigmoid)


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("big", [1e6, 3e38, float("inf"), float("-inf")])
def test_router_on_biases_that_swallow_the_scores(worker, sigmoid, big):
    g = _gen(6)
    logits = _randn(g, 40, 96)
    bias = torch.zeros(96, device="cuda")
    bias[[3, 17, 50, 51, 52, 80]] = big
    bias[48:60] = -abs(big)
    for groups, kept in ((1, 1), (8, 3), (8, 5)):
        _check_route(worker, logits, bias, 7, groups, kept, sigmoid=sigmoid)


def test_two_graphs_that_share_scratch(worker):
    """Recorded one behind the other, replayed in turn on one stream: each has the bits of its eager call, whichever ran before."""
    stream = torch.cuda.Stream()
    cases = [_experts_case(20 + i, t, 512, 384, 16, 4) for i, t in enumerate((5, 90, 700))]
    a, sa, w, sw = _operands(_gen(30), 40, 8192, 512)  # few tiles, a long k: ranges in slabs
    run, product = worker.register(runtime.experts_ffn_fp8_block), worker.register(runtime.projection_fp8_block)
    outs = [torch.empty((len(c[0]), 512), dtype=torch.bfloat16, device="cuda") for c in cases] + [torch.empty((40, 512), dtype=torch.float16, device="cuda")]

    def call(i, st):
        if i < 3:
            run(*cases[i], outs[i], stream=st)
        else:
            product(a, sa, w, sw, outs[i], stream=st)

    want, graphs = [], []
    for i in range(4):
        call(i, 0)
        worker.sync()
        want.append(outs[i].clone())
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=stream):
            call(i, torch.cuda.current_stream().cuda_stream)
    for order in ((0, 1, 2, 3), (3, 1, 0, 2), (2, 0, 3, 1)):
        for out in outs:
            out.fill_(float("nan"))
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            for i in order:
                graphs[i].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, w) for out, w in zip(outs, want)), order
    worker.sync()


def test_results_over_operands_are_refused(worker):
    raw = lambda n: torch.zeros(n, dtype=torch.uint8, device="cuda")
    buf = raw(1 << 16)
    part = lambda at, dtype, *shape: buf[at:at + torch.Size(shape).numel() * torch.empty(0, dtype=dtype).element_size()].view(dtype).view(shape)
    # product: out from the last byte of the codes on, and over the scales
    a, sa, w, sw = part(0, F8, 4, 256), part(2048, torch.float32, 4, 2), part(4096, F8, 16, 256), part(16384, torch.float32, 1, 2)
    for at in (1008, 2064, 4096 + 4080, 16384):
        with pytest.raises(ValueError, match="out overlaps an operand"):
            worker.run(runtime.projection_fp8_block, a, sa, w, sw, part(at, torch.float32, 4, 16))
    worker.run(runtime.projection_fp8_block, a, sa, w, sw, part(1024, torch.float32, 4, 16))  # right behind the codes
    # router
    logits, ids = part(0, torch.float32, 4, 8), part(1024, torch.int32, 4, 2)
    with pytest.raises(ValueError, match="overlap"):
        worker.run(runtime.route_experts, logits, ids, part(112, torch.float32, 4, 2), 1, 1, 0, 1, 1.0)
    with pytest.raises(ValueError, match="overlap"):
        worker.run(runtime.route_experts, logits, ids, part(1028, torch.float32, 4, 2), 1, 1, 0, 1, 1.0)
    # norm: a shifted sum, codes over the rows, two outputs in one place
    x, gamma, codes, scale = part(0, torch.bfloat16, 4, 128), part(2048, torch.float32, 128), part(4096, F8, 4, 128), part(8192, torch.float32, 4, 1)
    other, free = part(16384, torch.bfloat16, 4, 128), part(20480, torch.bfloat16, 4, 128)
    run = lambda *args: worker.run(runtime.add_rms_norm_fp8_block_normed, *args, 1e-6)
    for args in ((x, other, gamma, part(256, torch.bfloat16, 4, 128), free, codes, scale), (x, other, gamma, free, other, part(512, F8, 4, 128), scale),
                 (x, other, gamma, free, x, codes, part(2048, torch.float32, 4, 1))):
        with pytest.raises(ValueError, match="overlaps an input"):
            run(*args)
    for args in ((x, other, gamma, free, free, codes, scale), (x, other, gamma, x, x, codes, scale), (x, other, gamma, free, x, codes, part(4608 - 16, torch.float32, 4, 1))):
        with pytest.raises(ValueError, match="two outputs overlap"):
            run(*args)
    run(x, other, gamma, other, x, codes, scale)
    # experts
    args = _experts_case(1, 2, 128, 128, 2, 1)
    with pytest.raises(ValueError, match="out overlaps an operand"):
        worker.run(runtime.experts_ffn_fp8_block, *args, args[4].view(torch.uint8).flatten()[:512].view(torch.bfloat16).view(2, 128))
    worker.sync()


@pytest.mark.parametrize("rows,cols", [(700, 4096), (300, 8200), (900, 752), (64, 16384)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_norm_codes_are_those_of_the_exact_rows(worker, rows, cols, dtype):
    """n / scale is decided on 64 bits wherever 32 might pass a border between two codes: every code that is not subnormal is the exact one."""
    g = _gen(rows + cols)
    x = _randn(g, rows, cols) * torch.where(torch.rand(cols, device="cuda", generator=g) < 0.02, 20.0, 1.0)
    big, small = (1e15, 1e-36) if dtype == torch.bfloat16 else (100.0, 1e-5)
    x[0:3] *= big
    x[3:6] *= small
    if dtype == torch.bfloat16:
        x[6:9] *= 1e-39
    x = x.to(dtype)
    gamma = 1 + 0.3 * _randn(g, cols)
    gamma[5], gamma[7] = 0.0, -2.0
    codes, scale = torch.empty((rows, cols), dtype=F8, device="cuda"), torch.empty((rows, -(-cols // 128)), device="cuda")
    worker.run(runtime.rms_norm_fp8_block, x, gamma, codes, scale, 1e-6)
    worker.sync()
    n = ob.rms_norm(x, None, gamma, 1e-6)[1]
    want, exact_scale = ob.quantize_rows(n)
    ratio = n / exact_scale.repeat_interleave(128, -1)[:, :cols]
    regular = (ratio.abs() >= 2.0 ** -6) & (exact_scale.repeat_interleave(128, -1)[:, :cols] > 2.0 ** -125)
    assert torch.equal(codes.double()[regular], want[regular])
    _check_codes(codes, scale, n, 2.0 ** -17)


@pytest.mark.parametrize("cols", [128, 1000, 4104])
def test_norm_of_rows_that_are_not_finite(worker, cols):
    """A NaN makes its row NaN; an infinity leaves a NaN of itself and zeros; neither reaches another row, and every scale is 1."""
    inf, nan = float("inf"), float("nan")
    x = _randn(_gen(cols), 6, cols).bfloat16()
    clean = x.clone()
    x[1, 3], x[2, cols - 1], x[3, 0], x[4, 5], x[4, 6] = nan, inf, -inf, inf, nan
    gamma = 1 + 0.1 * _randn(_gen(1), cols)

    def call(x):
        outs = [torch.empty((6, cols), dtype=torch.bfloat16, device="cuda"), torch.empty((6, cols), dtype=F8, device="cuda"), torch.empty((6, -(-cols // 128)), device="cuda")]
        worker.run(runtime.rms_norm_fp8_block_normed, x, gamma, *outs, 1e-6)
        worker.sync()
        return outs[0].float(), outs[1].float(), outs[2]

    normed, codes, scale = call(x)
    want = call(clean)
    for got, w in zip((normed, codes, scale), want):
        assert torch.equal(got[[0, 5]], w[[0, 5]])
    assert (scale[1:5] == 1).all()
    for values in (normed, codes):
        assert values[1].isnan().all() and values[4].isnan().all()
        for row, at in ((2, cols - 1), (3, 0)):
            rest = torch.arange(cols, device="cuda") != at
            assert values[row, at].isnan() and (values[row, rest] == 0).all()
    # no eps, no values: 0 / 0
    zeros = torch.zeros((6, cols), dtype=torch.bfloat16, device="cuda")
    out, codes, scale = torch.empty_like(zeros), torch.empty((6, cols), dtype=F8, device="cuda"), torch.empty((6, -(-cols // 128)), device="cuda")
    worker.run(runtime.rms_norm_fp8_block_normed, zeros, gamma, out, codes, scale, 0.0)
    worker.sync()
    assert out.isnan().all() and codes.float().isnan().all() and (scale == 1).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_infinite_results_of_an_expert_stay_in_their_channels(worker, rows, dtype):
    """One block of an expert's down scales is infinite: 128 channels of its tokens are lost, everything else keeps its bits."""
    args = _experts_case(12, 90, 384, 256, 6, 2)
    want = _check_experts(worker, args, dtype)
    args[9][3, 1, 0] = float("inf")  # expert 3, channels 128 to 255
    out = torch.empty_like(want)
    worker.run(runtime.experts_ffn_fp8_block, *args, out)
    worker.sync()
    hit = (args[2] == 3).any(-1)
    assert hit.any() and not hit.all()
    assert not out[hit, 128:256].isfinite().any()
    keep = torch.ones_like(out, dtype=torch.bool)
    keep[hit, 128:256] = False
    assert torch.equal(out[keep], want[keep])


@pytest.mark.parametrize("rows", [64, 256], indirect=True)
@pytest.mark.parametrize("tokens,experts", [(128, 256), (128, 257), (129, 256), (1, 256), (1025, 40), (2050, 1000)])
def test_experts_at_the_borders_of_the_plan_s_forms(worker, rows, tokens, experts):
    _check_experts(worker, _experts_case(tokens + experts, tokens, 128, 128, experts, 8), torch.bfloat16)


@pytest.mark.parametrize("sigmoid,big", [(True, 32.0), (True, 64.0), (True, 1024.0), (False, 1024.0), (True, 1e6), (False, 1e6)])
@pytest.mark.parametrize("size", [2, 4, 32])
def test_router_on_groups_whose_two_best_keys_cancel(worker, sigmoid, big, size):
    """A group's best key is biased up and its second down: their sum is small, the roundings of 32-bit keys are those of the summands.  The
    groups' logits differ by about as much, so that the order of the sums falls between them."""
    g = _gen(size)
    bias = torch.full((2, size), -2.0 * big, device="cuda")
    bias[:, 0], bias[:, 1] = big, -big
    logits = _randn(g, 6000, 1, size).expand(-1, 2, -1) + big * 2.0 ** -24 * _randn(g, 6000, 2, size)
    _check_route(worker, logits.flatten(1).contiguous(), bias.flatten(), 2, 2, 1, sigmoid=sigmoid)


def test_router_on_biases_of_both_signs(worker):
    """Ordinary logits; in every group some experts are pushed up and the others down."""
    g = _gen(7)
    bias = torch.where(torch.rand(256, device="cuda", generator=g) < 0.03, 1024.0, -1024.0)
    bias.view(8, 32)[:, 5] = 1024.0
    _check_route(worker, _randn(g, 20000, 256), bias, 8, 8, 4, sigmoid=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cols", [512, 4104])
def test_norm_codes_on_ties(worker, dtype, cols):
    """x is 3/4 of its group's largest value, or 3/32: 448 times which is 21/16 of a power of two, a tie that goes to 20/16.  The groups' weights
    leave it one, whatever their own last bits and the statistic's are."""
    g = _gen(cols)
    rows, groups = 300, -(-cols // 128)
    whole = torch.randint(32, 64, (rows, groups, 1), device="cuda", generator=g).float()  # six bits: 3/4 of it has eight
    which = torch.rand((rows, groups, 128), device="cuda", generator=g)
    which[..., 0] = 1
    ratio = torch.where(which < 0.5, 0.75, torch.where(which < 0.75, -0.75 / 8, 1.0))
    x = (whole * ratio).flatten(1)[:, :cols].to(dtype).contiguous()
    gamma = (1 + torch.rand((groups, 1), device="cuda", generator=g)).expand(-1, 128).flatten()[:cols].contiguous()
    codes, scale = torch.empty((rows, cols), dtype=F8, device="cuda"), torch.empty((rows, groups), device="cuda")
    worker.run(runtime.rms_norm_fp8_block, x, gamma, codes, scale, 1e-6)
    worker.sync()
    want = torch.where(ratio == 0.75, 320.0, torch.where(ratio < 0, -40.0, 448.0)).flatten(1)[:, :cols]
    assert torch.equal(codes.float(), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("residual", [False, True])
def test_norm_codes_below_the_smallest_normal_code(worker, dtype, residual):
    """Groups of one large value and many whose codes are subnormal, steps of 2^-9: random ones, and 2^-16 of the large one, which is
    448 * 2^-16 = 3.5 steps, a tie that goes to the fourth, whatever row, weight and statistic are."""
    g = _gen(11)
    rows, cols = 600, 4096
    x = _randn(g, rows, cols // 128, 128) * 2.0 ** -16
    top = 1 + torch.rand((rows, cols // 128), device="cuda", generator=g)
    x[..., 0] = top
    x = (x * 256).to(dtype)
    x[..., 64:] = x[..., :1] * 2.0 ** -16
    gamma = 1 + 0.3 * torch.rand((cols // 128, 128), device="cuda", generator=g)
    gamma[:, 64:] = gamma[:, :1]
    x, gamma = x.flatten(1).contiguous(), gamma.flatten()
    codes, scale = torch.empty((rows, cols), dtype=F8, device="cuda"), torch.empty((rows, cols // 128), device="cuda")
    r, sums = torch.zeros_like(x), torch.empty_like(x)
    if residual:
        worker.run(runtime.add_rms_norm_fp8_block, x, r, gamma, sums, codes, scale, 1e-6)
    else:
        worker.run(runtime.rms_norm_fp8_block, x, gamma, codes, scale, 1e-6)
    worker.sync()
    want, _ = ob.quantize_rows(ob.rms_norm(x, None, gamma, 1e-6)[1])
    assert (want.unflatten(-1, (-1, 128))[..., 64:] == 4 * 2.0 ** -9).all()
    assert torch.equal(codes.double(), want)


@pytest.mark.parametrize("cols", [256, 1000, 8200])
def test_norm_where_the_weighted_sum_leaves_fp32_and_its_norm_does_not(worker, cols):
    """s * gamma overflows, or is too small for 24 bits, while s * rsqrt(..) * gamma is an ordinary number."""
    g = _gen(cols)
    out, codes, scale = torch.empty((4, cols), dtype=torch.bfloat16, device="cuda"), torch.empty((4, cols), dtype=F8, device="cuda"), torch.empty(
        (4, -(-cols // 128)), device="cuda")

    def check(x, gamma):
        worker.run(runtime.rms_norm_fp8_block_normed, x, gamma, out, codes, scale, 0.0)
        worker.sync()
        n = ob.rms_norm(x, None, gamma, 0.0)[1]
        _check_codes(codes, scale, n, 2.0 ** -17)
        assert ((out.double() - n).abs() <= n.abs() * (HALF_STEP[torch.bfloat16] + 2.0 ** -17) + TINY[torch.bfloat16]).all()

    x = _randn(g, 4, cols)
    check((x * 1e16).bfloat16(), 1e24 * (1 + 0.2 * _randn(g, cols)))
    check((x * 1e-16).bfloat16(), 1e-26 * (1 + 0.2 * _randn(g, cols)))
    # a row whose sum of squares passes fp32 is normalised to zeros, in 16 bits as in codes
    gamma = 2 + 0.1 * torch.rand(cols, device="cuda", generator=g)
    worker.run(runtime.rms_norm_fp8_block_normed, (x.sign() * 3e38).bfloat16(), gamma, out, codes, scale, 1e-6)
    worker.sync()
    assert (out == 0).all() and (codes.float() == 0).all() and (scale == 1).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cols", [512, 2048, 4104, 16384])
def test_norm_codes_are_those_of_the_exact_sums(worker, dtype, cols):
    """x is 3/4 of its group's largest value or an eighth of that, 448 times which is a tie between two codes; the residual, too small for the
    fp32 sum to show it, decides."""
    g = _gen(cols)
    rows = 300
    whole = torch.randint(32, 64, (rows, -(-cols // 128), 1), device="cuda", generator=g).float()  # six bits: 3/4 of it has eight
    which = torch.rand((rows, -(-cols // 128), 128), device="cuda", generator=g)
    x = torch.where(which < 0.5, whole * 0.75, torch.where(which < 0.75, whole * 0.75 / 8, whole))
    x[..., 0] = whole[..., 0]
    small = 2.0 ** -26 if dtype == torch.bfloat16 else 2.0 ** -20  # of up to 64: below the last of its 24 bits
    r = torch.where(torch.rand(x.shape, device="cuda", generator=g) < 0.5, -small, small)
    r = torch.where(x == whole, 0.0, r)
    x, r = (t.flatten(1)[:, :cols].to(dtype).contiguous() for t in (x, r))
    gamma = torch.full((cols,), 0.5, device="cuda")
    codes, scale = torch.empty((rows, cols), dtype=F8, device="cuda"), torch.empty((rows, -(-cols // 128)), device="cuda")
    sums = torch.empty_like(x)
    worker.run(runtime.add_rms_norm_fp8_block, x, r, gamma, sums, codes, scale, 1e-6)
    worker.sync()
    s, n = ob.rms_norm(x, r, gamma, 1e-6)
    want, _ = ob.quantize_rows(n)
    assert torch.equal(sums, s.to(dtype)) and not torch.equal(want, ob.quantize_rows(ob.rms_norm(x, None, gamma, 1e-6)[1])[0])
    assert torch.equal(codes.double(), want)
    # the sum over the residual and the norm over x, as a loop that keeps its buffers calls it
    got, again, normed = torch.empty_like(codes), torch.empty_like(scale), x.clone()
    worker.run(runtime.add_rms_norm_fp8_block_normed, normed, r, gamma, r, normed, got, again, 1e-6)
    worker.sync()
    assert torch.equal(got.double(), want) and torch.equal(again, scale) and torch.equal(r, sums)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_norm_codes_around_the_smallest_normal_code(worker, dtype):
    """2^-12 of a largest value of 7 is a code of 2^-6 itself, whichever side of it 32 bits see; ties next to it send the group to 64 bits."""
    g = _gen(21)
    rows, groups = 64, 64
    x = torch.full((rows, groups, 128), 7.0, device="cuda")
    x[..., 1:50] = 2.0 ** -12
    x[..., 50:90] = -15 / 16 * 2.0 ** -12  # 7.5 of the steps of 2^-9 that 2^-6 has eight of
    x[..., 90:100] = 5.25
    x = x.flatten(1).to(dtype)
    gamma = (1 + torch.rand((groups, 1), device="cuda", generator=g)).expand(-1, 128).flatten().contiguous()
    codes, scale = torch.empty(x.shape, dtype=F8, device="cuda"), torch.empty((rows, groups), device="cuda")
    worker.run(runtime.rms_norm_fp8_block, x, gamma, codes, scale, 1e-6)
    worker.sync()
    want = torch.full((128,), 448.0, device="cuda")
    want[1:50], want[50:90], want[90:100] = 2.0 ** -6, -(2.0 ** -6), 320.0
    assert (codes.float().unflatten(-1, (-1, 128)) == want).all()


def test_experts_whose_rows_would_not_fit_the_scratch_at_once(worker):
    """500 tokens of 64 slots of 65536 channels, whose rows would be 8 GB in fp32: several passes.  Tokens of the first, the second and the last have the bits of a
    call of theirs alone, and the library's scratch has not grown by those rows."""
    args = _experts_case(5, 500, 65536, 128, 2, 64)
    some = [0, 1, 130, 498, 499]
    few = [t[some].contiguous() for t in args[:4]] + args[4:]
    out, want = torch.empty((500, 65536), device="cuda"), torch.empty((5, 65536), device="cuda")
    worker.set_option("block_gemm_rows", 64)
    try:
        worker.run(runtime.experts_ffn_fp8_block, *few, want)
        worker.sync()
        free = torch.cuda.mem_get_info()[0]
        worker.run(runtime.experts_ffn_fp8_block, *args, out)
        worker.sync()
        assert free - torch.cuda.mem_get_info()[0] < 6e9
    finally:
        worker.set_option("block_gemm_rows", 0)
    assert torch.equal(out[some], want) and want.isfinite().all() and want.abs().amax() > 0
