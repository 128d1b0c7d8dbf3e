"""Which paged attention calls need a workspace: those whose table or window reaches past what one workgroup takes.
The lengths are on the device and have no part in it."""

from __future__ import annotations

import ctypes

import pytest

from gemma4_posttrain_jax_amd import _lib
from test_paged_refusals import _decode


def _need(**kw) -> int:
    return _lib.lib().g4_paged_decode_workspace_size(ctypes.byref(_decode(**kw)))


@pytest.mark.parametrize("batch,border", [(1, 640), (32, 640), (33, 1024), (600, 1024)])  # two heads: up to 64 pairs, more
def test_the_border_between_whole_and_cut_rows(batch, border):
    """In 32-position chunks that a row can touch: a window's first may begin before it, so it counts 31 positions more."""

    def table(n):
        return dict(batch=batch, max_pages=n, table_stride=n)

    wide, pages = table(1000), border // 64
    assert _need(**table(pages)) == 0 < _need(**table(pages + 1))
    assert _need(**wide, window=border - 31) == 0 < _need(**wide, window=border - 30)
    # a window as long as the table or longer changes nothing
    for window in (border, border + 64, 1 << 30):
        assert _need(**table(pages), window=window) == 0
    assert _need(**table(pages + 1), window=1 << 30) == _need(**table(pages + 1)) > 0


def test_large_batches_need_a_plan():
    """Beyond 512 rows 8 bytes per (row, head) and 8 per row and one more."""

    wide = dict(max_pages=1000, table_stride=1000)
    need = lambda batch: _need(batch=batch, **wide)  # noqa: E731
    assert need(512) - need(511) == 2 * 8
    assert need(513) - need(512) == 2 * 8 + 514 * 8
    assert need(5000) - need(4999) == 3 * 8
