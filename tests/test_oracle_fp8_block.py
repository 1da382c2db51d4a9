"""The oracle of the block-scaled e4m3 operators, and what the library refuses before it looks for a device (CPU)."""

import pytest
import torch

from oracle import fp8_block as ob
from pypto_amd import _lib

F8 = torch.float8_e4m3fn


def test_rounding_is_the_format_s_own():
    """Every e4m3 value is a fixed point, a midpoint goes to the even code, and torch's cast agrees on random values."""
    table = torch.arange(256, dtype=torch.uint8).view(F8).double()
    finite = table[~table.isnan()]
    assert torch.equal(ob.round_e4m3(finite), finite)
    pos = torch.unique(finite[finite >= 0])
    mid = (pos[:-1] + pos[1:]) / 2
    even = torch.where(torch.arange(len(mid)) % 2 == 0, pos[:-1], pos[1:])  # code numbers ascend with the values
    assert torch.equal(ob.round_e4m3(mid), even) and torch.equal(ob.round_e4m3(-mid), -even)
    v = torch.randn(20000, generator=torch.Generator().manual_seed(1)) * 40
    assert torch.equal(ob.round_e4m3(v.double()), v.clamp(-448, 448).to(F8).double())


def test_row_groups_and_matrix_blocks():
    g = torch.Generator().manual_seed(2)
    x = torch.randn((5, 300), generator=g) * torch.tensor([1e-4, 1.0, 1.0, 50.0, 1e4])[:, None]
    x[1, 128:256] = 0
    q, s = ob.quantize_rows(x)
    assert q.shape == (5, 300) and s.shape == (5, 3) and s[1, 1] == 1 and (q[1, 128:256] == 0).all()
    assert (q.reshape(-1).abs().max() == 448) and torch.allclose(s[0, 2], x[0, 256:].abs().max().double() / 448)
    back = ob.dequantize_rows(q, s)
    wide = s.repeat_interleave(128, -1)[:, :300]
    assert ((back - x).abs() <= torch.maximum(x.abs() * 2.0 ** -4, wide * 2.0 ** -10) * (1 + 1e-9)).all()
    assert torch.equal(ob.quantize_rows(back)[0], q)
    w = torch.randn((2, 200, 256), generator=g)
    codes, scale = ob.quantize_matrix(w)
    assert codes.shape == w.shape and scale.shape == (2, 2, 2)
    assert torch.allclose(scale[1, 1, 0], w[1, 128:, :128].abs().max() / 448)
    wide = scale.repeat_interleave(128, -2).repeat_interleave(128, -1)[:, :200]
    assert ((ob.dequantize_matrix(codes, scale) - w).abs() <= torch.maximum(w.abs() * 2.0 ** -4, wide * 2.0 ** -10) * (1 + 1e-6)).all()


def test_router_closed_cases():
    ids, w = ob.route(torch.zeros(2, 8), None, 3)
    assert ids.tolist() == [[0, 1, 2]] * 2 and torch.allclose(w, torch.full((2, 3), 1 / 3, dtype=torch.float64))
    logits = torch.tensor([[0.0, 3.0, 2.0, 1.0, 5.0, -9.0, 0.0, 0.0]])
    ids, w = ob.route(logits, None, 2, renormalize=False)
    assert ids.tolist() == [[4, 1]] and torch.allclose(w, torch.softmax(logits.double(), -1)[:, [4, 1]])
    # two groups, one stays: without a bias the one with the best expert, with one the one with the best pair
    assert ob.route(logits, None, 2, 2, 1)[0].tolist() == [[4, 6]]
    assert ob.route(logits, torch.zeros(8), 2, 2, 1, sigmoid=True)[0].tolist() == [[1, 2]]
    # a bias moves the choice and not the weights
    bias = torch.tensor([9.0, 0, 0, 0, 0, 0, 0, 0])
    ids, w = ob.route(logits, bias, 1, sigmoid=True, renormalize=False, scale=2.5)
    assert ids.tolist() == [[0]] and torch.allclose(w, torch.tensor([[1.25]], dtype=torch.float64))
    nan, inf = float("nan"), float("inf")
    ids, w = ob.route(torch.tensor([[nan, -inf, 1.0, -inf]]), None, 4)
    assert ids.tolist() == [[2, 0, 1, 3]] and w.tolist() == [[1.0, 0, 0, 0]]
    assert ob.route(torch.tensor([[inf, 0.0, inf]]), None, 2)[1].tolist() == [[0.5, 0.5]]


def test_experts_on_values_that_every_step_holds():
    """Gate weights that make the gate large, so that SiLU is the identity there: h = g * u is a product of small whole numbers."""
    t, h, i, e = 3, 128, 128, 4
    x = torch.zeros((t, h))
    x[:, 0] = torch.tensor([1.0, 2.0, 4.0])
    gate, up, down = torch.zeros((e, i, h)), torch.zeros((e, i, h)), torch.zeros((e, h, i))
    gate[:, :, 0], up[:, 0, 0] = 256.0, torch.arange(1.0, e + 1)
    down[:, 5, 0] = 1.0
    ones = lambda *s: torch.ones(s)
    ids = torch.tensor([[0, 3], [-1, 2], [-1, -1]], dtype=torch.int32)
    w = torch.tensor([[0.5, 0.25], [9.0, 1.0], [1.0, 1.0]])
    out, slack = ob.experts_ffn(x.to(F8), ones(t, 1), ids, w, gate.to(F8), ones(e, 1, 1), up.to(F8), ones(e, 1, 1), down.to(F8), ones(e, 1, 1))
    want = torch.zeros((t, h), dtype=torch.float64)
    want[0, 5] = 0.5 * 256 * 1 + 0.25 * 256 * 4
    want[1, 5] = 512 * 2 * 3
    assert torch.allclose(out, want, rtol=1e-12) and (slack[2] == 0).all() and (slack[0, 5] > 0)


def _refused(rc, status, text):
    assert rc == status
    assert text in _lib.load().pto_hip_last_error(), _lib.load().pto_hip_last_error()


BF16, FP16, FP32, I32 = 0x40, 0x33, 0x34, 0x13
INVALID, UNSUPPORTED = _lib.ERR_INVALID_VALUE, _lib.ERR_UNSUPPORTED
P = 1 << 20  # an address that no refused call looks behind


def test_refusals_of_the_norm():
    fn = _lib.load().pto_hip_rms_norm_fp8_block
    call = lambda rows=4, cols=256, dtype=BF16, x=P, res=None, gamma=P, sums=None, normed=None, codes=P, scale=P: fn(
        x, res, gamma, sums, normed, codes, scale, rows, cols, 1e-6, dtype, None)
    _refused(call(rows=-1), INVALID, b"bad shape")
    _refused(call(cols=0), INVALID, b"bad shape")
    _refused(call(rows=1 << 31), INVALID, b"bad shape")
    _refused(call(dtype=FP32), INVALID, b"dtype FP32")
    _refused(call(cols=252), UNSUPPORTED, b"multiple of 8")
    _refused(call(cols=16392), UNSUPPORTED, b"at most 16384")


def test_refusals_of_the_product():
    fn = _lib.load().pto_hip_projection_fp8_block
    call = lambda m=4, k=256, n=8, dtype=BF16: fn(P, P, P, P, P, m, k, n, dtype, None)
    _refused(call(m=-1), INVALID, b"bad shape")
    _refused(call(n=0), INVALID, b"bad shape")
    _refused(call(k=0), INVALID, b"bad shape")
    _refused(call(dtype=I32), INVALID, b"output dtype INT32")
    _refused(call(k=192), UNSUPPORTED, b"multiple of 128")
    _refused(call(k=65664), UNSUPPORTED, b"at most 65536")


def test_refusals_of_the_router():
    fn = _lib.load().pto_hip_route_experts
    call = lambda t=4, e=64, k=4, groups=1, kept=1, score=0, renorm=1, dtype=FP32: fn(P, None, P, P, t, e, k, groups, kept, score, renorm, 1.0,
                                                                                   dtype, None)
    _refused(call(t=-1), INVALID, b"bad shape")
    _refused(call(k=0), INVALID, b"bad shape")
    _refused(call(dtype=I32), INVALID, b"logits dtype")
    _refused(call(score=2), INVALID, b"neither softmax (0) nor sigmoid (1)")
    _refused(call(renorm=2), INVALID, b"renormalize")
    _refused(call(groups=3), INVALID, b"do not divide")
    _refused(call(groups=0), INVALID, b"do not divide")
    _refused(call(groups=4, kept=5), INVALID, b"topk_groups 5")
    _refused(call(groups=4, kept=0), INVALID, b"topk_groups 0")
    _refused(call(groups=8, kept=1, k=9), INVALID, b"top_k 9 of the 8")
    _refused(call(e=1025), UNSUPPORTED, b"at most 1024 experts")
    _refused(call(e=256, k=65), UNSUPPORTED, b"top_k 64")
    _refused(call(e=130, groups=65, kept=65), UNSUPPORTED, b"64 groups")


def test_refusals_of_the_experts():
    fn = _lib.load().pto_hip_experts_ffn_fp8_block
    call = lambda t=4, h=256, i=128, e=8, k=2, dtype=BF16: fn(*[P] * 11, t, h, i, e, k, dtype, None)
    _refused(call(t=-1), INVALID, b"bad shape")
    _refused(call(e=0), INVALID, b"bad shape")
    _refused(call(k=0), INVALID, b"bad shape")
    _refused(call(dtype=I32), INVALID, b"output dtype")
    _refused(call(h=200), UNSUPPORTED, b"multiples of 128")
    _refused(call(i=64), UNSUPPORTED, b"multiples of 128")
    _refused(call(i=65664), UNSUPPORTED, b"at most 65536")
    _refused(call(e=1025), UNSUPPORTED, b"at most 1024 experts")
    _refused(call(k=65), UNSUPPORTED, b"top_k 64")


@pytest.mark.skipif(torch.cuda.device_count() > 0, reason="another test may have bound a device")
def test_good_arguments_before_init_fail_loudly():
    lib = _lib.load()
    assert lib.pto_hip_rms_norm_fp8_block(P, None, P, None, None, P, P, 4, 256, 1e-6, BF16, None) == _lib.ERR_NOT_INITIALIZED
    assert lib.pto_hip_quantize_fp8_block(P, P, P, 4, 256, BF16, None) == _lib.ERR_NOT_INITIALIZED
    assert lib.pto_hip_projection_fp8_block(P, P, P, P, P, 4, 256, 8, BF16, None) == _lib.ERR_NOT_INITIALIZED
    assert lib.pto_hip_route_experts(P, None, P, P, 4, 64, 4, 1, 1, 0, 1, 1.0, FP32, None) == _lib.ERR_NOT_INITIALIZED
    assert lib.pto_hip_experts_ffn_fp8_block(*[P] * 11, 4, 256, 128, 8, 2, BF16, None) == _lib.ERR_NOT_INITIALIZED
