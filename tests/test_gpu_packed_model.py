"""Packed prompts in the model: what a prefill keeps of its description, and the steps that follow it."""

from __future__ import annotations

import pytest
import torch

from gemma4_posttrain_jax_amd import config as C
from gemma4_posttrain_jax_amd import kernels
from gemma4_posttrain_jax_amd import model as M
from gemma4_posttrain_jax_amd.kvcache import PagedSpec, init_paged_kv_cache
from test_gpu_paged_run import CFG, _params

pytestmark = pytest.mark.gpu


def _packed(lens, tail, device):
    """The description of prompts of ``lens`` tokens with ``tail`` tokens of no prompt behind them, ids and places."""

    T = sum(lens) + tail
    cu = torch.tensor([0, *lens], dtype=torch.int32, device=device).cumsum(0, dtype=torch.int32)
    starts = kernels.packed_starts(cu, T)
    rows = torch.tensor([b for b, n in enumerate(lens) for _ in range(n)] + [0] * tail, dtype=torch.int32, device=device)
    ids = (torch.arange(T, device=device) * 37 % 500)[None]
    places = (torch.arange(T, dtype=torch.int32, device=device) - starts)[None]
    return M.PackedPrompts(starts, rows, cu.diff(), max(lens)), ids, places


def test_steps_leave_the_prompts_description(device):
    """A captured step's append adds to the cache's ``held`` in place: the description of the prompts is another tensor, and a
    second prefill by it stores what the first stored."""

    cfg = C.config_from_hf(CFG)
    params = _params(cfg, device)
    lens = [60, 7, 33]
    packed, ids, places = _packed(lens, 5, device)

    def prefill():
        empty = init_paged_kv_cache(cfg, len(lens), 128, PagedSpec(32), device)
        return M.forward_gemma4_text(params, ids, places, config=cfg, kv_cache=empty, packed=packed)[1]

    first, cache = prefill(), prefill()
    for step in range(45):  # past the window of 40
        tok = torch.full((3, 1), step, dtype=torch.int32, device=device)
        slot = torch.full((3,), int(cache.length), dtype=torch.int32, device=device)
        _, cache = M.forward_gemma4_text(params, tok, cache.held[:, None].clone(), config=cfg, kv_cache=cache, cache_mode="append",
                                         write_pos=slot)
    assert cache.held.tolist() == [n + 45 for n in lens]
    assert packed.lengths.tolist() == lens
    again = prefill()
    assert first.held.tolist() == again.held.tolist() == lens
    for x, y in zip(first.layers, again.layers):
        if x is not None:
            assert torch.equal(x.key, y.key) and torch.equal(x.value, y.value)
