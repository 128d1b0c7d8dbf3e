"""Single elements of a paged cache that are no numbers: what they reach and what they do not."""

from __future__ import annotations

import math

import pytest
import torch

import paged_util as P
from gemma4_posttrain_jax_amd import kernels

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("D,ps,pages", [(64, 32, 3), (128, 64, 14), (256, 32, 40), (512, 64, 3), (512, 64, 20)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_a_value_that_is_no_number_reaches_its_dim_alone(device, e4m3, D, ps, pages, bad):
    """One element of one attended value, not its vector's largest (so that an e4m3 vector keeps its scale): the other
    dims keep their bits, in its row and in the others, in whole rows and in cut ones."""

    g = torch.Generator().manual_seed(D + pages)
    B, R, dim = 3, 4, 5
    randn = lambda *s: torch.randn(s, generator=g).to(BF16)  # noqa: E731
    k, v, q = randn(B * pages, 1, ps, D), randn(B * pages, 1, ps, D), (0.2 * randn(B, 1, R, D)).to(BF16)
    table = torch.randperm(B * pages, generator=g).view(B, pages).to(torch.int32)
    lengths = [pages * ps, pages * ps - 9, ps + 1]
    page = int(table[1, pages - 2])
    v[page, 0, 11, dim], v[page, 0, 11, 0] = 0.25, 4.0
    call = lambda v: kernels.paged_decode_attention(  # noqa: E731
        P.filled(B * pages, 1, D, ps, e4m3, k, v, device), q.to(device), page_table=table.to(device),
        lengths=torch.tensor(lengths, dtype=torch.int32, device=device))
    want = call(v)
    v[page, 0, 11, dim] = bad
    got = call(v)
    assert want.isfinite().all()
    others = torch.arange(D, device=device) != dim
    assert torch.equal(got[..., others], want[..., others])
    assert torch.equal(got[[0, 2]], want[[0, 2]])
    # an infinity stays one in bf16 and becomes a NaN in e4m3; its probability is above 0
    assert (got[1, ..., dim].isnan() if e4m3 or math.isnan(bad) else got[1, ..., dim] == math.inf).all()
