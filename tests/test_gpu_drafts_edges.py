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
