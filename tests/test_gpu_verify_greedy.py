"""Greedy verification of drafted tokens over rows that have no largest number, on the GPU."""

from __future__ import annotations

import math

import pytest
import torch

from gemma4_posttrain_jax_amd import kernels

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V", [3, 5000])
def test_greedy_over_rows_of_no_numbers(V, device):
    """Nothing is accepted there, no id outside the vocabulary either, and the token is 0."""

    logits = torch.zeros((4, 2, V))
    logits[:, 0] = math.nan
    drafts = torch.tensor([[2 ** 31 - 1], [0], [-1], [V]], dtype=torch.int32)
    tokens, count, _ = kernels.verify_draft(logits.to(device), drafts.to(device), None, None, temperature=0.0)
    assert count.tolist() == [0] * 4 and tokens.tolist() == [[0, -1]] * 4
