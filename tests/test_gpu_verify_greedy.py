"""Greedy verification of drafted tokens over rows that have no largest number, on the GPU."""

from __future__ import annotations

import math

import pytest
import torch

from gemma4_posttrain_jax_amd import kernels

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V", [1, 5, 4097, 40000])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_greedy_over_rows_of_minus_infinity(V, dtype, device):
    """Where nothing but -inf is left the first of it is the largest logit, NaN before it passed over."""

    inf = math.inf
    logits = torch.zeros((5, 3, V), dtype=dtype)
    logits[:, 2, V // 2] = 1.0
    logits[:3, :2] = -inf
    logits[3, 0, :V - 1], logits[3, 0, V - 1] = math.nan, -inf
    logits[4, 0] = -inf
    drafts = torch.tensor([[0, 0], [0, V - 1], [V - 1, 0], [V - 1, 0], [0, 0]], dtype=torch.int32)
    tokens, count, logp = [t.cpu() for t in kernels.verify_draft(logits.to(device), drafts.to(device), None, None,
                                                                 temperature=0.0)]
    want = [[0, 0, V // 2], [0, 0, V // 2 if V == 1 else -1], [0, 0 if V == 1 else -1, V // 2 if V == 1 else -1],
            [V - 1, 0, V // 2], [0, 0, V // 2]]
    assert tokens.tolist() == want
    assert count.tolist() == [sum(t >= 0 for t in row) - 1 for row in want]
    for b in range(5):  # log_softmax over nothing but -inf is no number
        assert bool(logp[b, :int(count[b]) + 1].isnan()[0]) and (b < 4 or bool(logp[b, 1:].isfinite().all()))


@pytest.mark.parametrize("V", [3, 5000])
def test_greedy_over_rows_of_no_numbers(V, device):
    """Nothing is accepted there, no id outside the vocabulary either, and the token is 0."""

    logits = torch.zeros((4, 2, V))
    logits[:, 0] = math.nan
    drafts = torch.tensor([[2 ** 31 - 1], [0], [-1], [V]], dtype=torch.int32)
    tokens, count, _ = kernels.verify_draft(logits.to(device), drafts.to(device), None, None, temperature=0.0)
    assert count.tolist() == [0] * 4 and tokens.tolist() == [[0, -1]] * 4
