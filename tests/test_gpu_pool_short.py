"""A pool with too few pages: what the entries that get none hold, on the GPU against plain lists."""

from __future__ import annotations

import pytest
import torch

import pool_util as plain
from gemma4_posttrain_jax_amd import kernels
from gemma4_posttrain_jax_amd.kvcache import new_paged_layer

pytestmark = pytest.mark.gpu


def _i32(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


@pytest.mark.parametrize("rows", [3, 32, 33, 400])
@pytest.mark.parametrize("spare", [0, 1, 5])
def test_reserve_leaves_entries_without_a_page_as_they_were(rows, spare, device):
    """Entries of -1, of the pool's size, far beyond it and below -1 hold no page; with the pages used up they stay."""

    P = 2 * rows + spare
    refs = [1] * (2 * rows) + [0] * spare
    table = [[2 * b, (-1, P, 2 ** 31 - 1, -7)[b % 4], 2 * b + 1, (P + 1, -1, -2 ** 31, P)[b % 4]] for b in range(rows)]
    r, t = _i32(refs, device), _i32(table, device)
    short = kernels.paged_reserve(r, t, _i32([128] * rows, device), page_size=32)
    before = [list(row) for row in table]
    assert short.tolist() == [plain.reserve(refs, table, [128] * rows, 32)] == [2 * rows - spare]
    assert t.tolist() == table and r.tolist() == refs
    got = [(a, b) for x, y in zip(before, t.tolist()) for a, b in zip(x, y) if not 0 <= a < P]
    assert [b for _, b in got[:spare]] == list(range(2 * rows, P)) and all(a == b for a, b in got[spare:])


@pytest.mark.parametrize("rows", [4, 40])
def test_fork_writes_minus_one_where_there_is_no_page(rows, device):
    layer = new_paged_layer(3, 1, 64, 32, device=device)
    refs, table = [1, 1, 0], [[0, 1]]
    r, out = _i32(refs, device), torch.full((rows, 2), 77, dtype=torch.int32, device=device)
    _, short = kernels.paged_fork([layer], r, _i32(table, device), _i32([0] * rows, device), _i32([40], device), out=out)
    assert short.tolist() == [rows - 1] and r.tolist() == [1 + rows, 1, 1]
    assert out.tolist() == [[0, 2]] + [[0, -1]] * (rows - 1)
