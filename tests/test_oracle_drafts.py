"""The oracle of the drafted-token operators against known answers, and the entry points' refusals that need no device."""

import ctypes as C

import numpy as np
import pytest
import torch

from oracle import drafts as od
from pypto_amd import _lib


def test_owners_leave_out_what_lies_outside_the_sequences():
    assert od.owners([1, 3, 3, 4], 6) == [None, (0, 0), (0, 1), (2, 0), None, None]


def test_turn_by_a_quarter_and_by_reference_tables():
    x = torch.tensor([[1.0, 2.0, 3.0, 4.0, 5.0]], dtype=torch.float64)
    y, size = od.turn(x, torch.zeros(2, dtype=torch.float64), torch.ones(2, dtype=torch.float64))  # R = 4: the fifth stays
    assert y.tolist() == [[-3.0, -4.0, 1.0, 2.0, 5.0]] and size.tolist() == [[3.0, 4.0, 1.0, 2.0, 5.0]]
    x = torch.tensor([[1.0, 2.0]], dtype=torch.float64)
    y, _ = od.turn(x, torch.tensor([2.0, 3.0], dtype=torch.float64), torch.tensor([5.0, 7.0], dtype=torch.float64))
    assert y.tolist() == [[1 * 2 - 2 * 5, 2 * 3 + 1 * 7]]


def test_e4m3_rounds_to_even_and_keeps_to_its_range():
    v = torch.tensor([0.0, 17.0, 18.0, 19.0, 500.0, -500.0, 2.0 ** -10, 3 * 2.0 ** -10], dtype=torch.float64)
    assert od.e4m3(v).tolist() == [0.0, 16.0, 18.0, 20.0, 448.0, -448.0, 0.0, 2 * 2.0 ** -9]


def test_append_takes_a_blocks_new_rows_together():
    """Two rows into a block that holds one: the scale grows to the larger of both, the row in front is coded again."""
    one = torch.ones((4, 1))
    key = torch.zeros((1, 1, 4, 2), dtype=torch.float64)
    key[0, 0, 0] = 100.0
    scale = torch.tensor([[0.5]])
    qkv = torch.tensor([[1.0, 1.0, 448.0, 0.0, 1.0, 1.0], [1.0, 1.0, 896.0, 0.0, 1.0, 1.0]])
    got = od.rope_append(qkv, torch.tensor([0, 1]), torch.tensor([0, 2]), torch.tensor([1]), one, 0 * one, None, None, torch.tensor([[0]]), key, key,
                         scale, scale, 1, 1, 2, 4, 0.0)
    assert got["key_scale"][0].tolist() == [2.0] and got["key"][0, 0, :3].tolist() == [[24.0, 24.0], [224.0, 0.0], [448.0, 0.0]]  # 25 is a tie
    assert got["value_scale"][0].tolist() == [0.5] and got["value"][0, 0, 0].tolist() == [100.0, 100.0]


def test_tree_attention_of_a_fork():
    """Two children of one root see the root and themselves, not each other; a row that sees nothing is zeros."""
    key = torch.zeros((1, 1, 4, 1))
    value = torch.tensor([1.0, 2.0, 4.0, 8.0]).view(1, 1, 4, 1)
    out, _, _ = od.tree_attention(torch.zeros((4, 1)), key, value, torch.tensor([[0]]), torch.tensor([0]), torch.tensor([0, 4]),
                                  torch.tensor([[1], [3], [5], [0]]), 1, 1, 1, 4, 1.0)
    assert out.flatten().tolist() == [1.0, 1.5, 2.5, 0.0]


@pytest.mark.parametrize("args,want", [
    (dict(temperature=0.0), (1, 1.0)),
    (dict(temperature=1.0, uniform=0.0), (0, 1 / 7)),
    (dict(temperature=1.0, uniform=0.15), (1, 4 / 7)),
    (dict(temperature=1.0, uniform=0.9), (3, 1 / 7)),
    (dict(temperature=1.0, top_k=2, uniform=0.9), (1, 4 / 5)),  # of equal ones the first: index 0
    (dict(temperature=1.0, top_p=0.57, uniform=0.999), (1, 1.0)),
    (dict(temperature=1.0, top_p=0.58, uniform=0.0), (0, 1 / 5)),
    (dict(temperature=1.0, top_p=0.0, uniform=0.7), (1, 1.0)),
    (dict(temperature=1.0, min_p=0.26, uniform=0.7), (1, 1.0)),
    (dict(temperature=0.5, uniform=0.05), (0, 1 / 19)),
])
def test_sample_of_one_row(args, want):
    logits = np.log(np.array([1.0, 4.0, 1.0, 1.0]))
    full = dict(temperature=1.0, top_k=None, top_p=None, min_p=None, uniform=0.5) | args
    token, prob = od.sample(logits, **full)
    assert token == want[0] and prob == pytest.approx(want[1], rel=1e-12)


def test_sample_of_infinities_and_nan():
    none = dict(top_k=None, top_p=None, min_p=None)
    inf, nan = float("inf"), float("nan")
    assert od.sample([-inf, nan, -inf], 1.0, uniform=0.5, **none) == (-1, 0.0)
    assert od.sample([1.0, inf, nan, inf], 1.0, uniform=0.5, **none) == (3, 0.5)
    assert od.sample([1.0, nan, 1.0], 0.0, uniform=0.5, **none) == (0, 1.0)


def test_entry_points_refuse_before_init():
    lib = _lib.load()
    assert lib.pto_hip_rope_append_tokens(None, None) == _lib.ERR_NOT_INITIALIZED
    assert lib.pto_hip_tree_attention(None, None) == _lib.ERR_NOT_INITIALIZED
    assert lib.pto_hip_sample_tokens(*[None] * 8, 1, 8, 0x34, None) == _lib.ERR_NOT_INITIALIZED
    assert C.sizeof(_lib.RopeAppendArgs) == 14 * 8 + 9 * 8 + 5 * 4 + 4
    assert C.sizeof(_lib.TreeAttentionArgs) == 10 * 8 + 9 * 8 + 3 * 4 + 4
