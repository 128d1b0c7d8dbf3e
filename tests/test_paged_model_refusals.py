"""What a model's forward refuses to do with a paged cache, on the CPU: it refuses before any kernel runs."""

from __future__ import annotations

import pytest
import torch

from gemma4_posttrain_jax_amd import config as C
from gemma4_posttrain_jax_amd import kernels
from gemma4_posttrain_jax_amd import model as M
from gemma4_posttrain_jax_amd import sampler as SMP
from gemma4_posttrain_jax_amd.kvcache import PagedSpec, init_paged_kv_cache
from test_gpu_paged_run import CFG, _params, _prompts


class Launched(Exception):
    pass


@pytest.fixture
def run(monkeypatch):
    """(config, params, prompt ids, mask, forward): a forward that gets past its checks raises Launched."""

    def launch(*args, **kw):
        raise Launched

    for name in ("rms_norm", "decode_prologue"):
        monkeypatch.setattr(kernels, name, launch)
    cfg = C.config_from_hf(CFG)
    params = _params(cfg, "cpu")
    ids, mask = _prompts(cfg, [0, 3], 20, "cpu")

    def forward(ids, mask, cache, mode="prefill", **kw):
        return M.forward_gemma4_lm(params, ids, torch.zeros_like(ids), config=cfg, attention_mask=mask, kv_cache=cache,
                                   cache_mode=mode, **kw)

    return cfg, params, ids, mask, forward


def _cache(cfg, capacity=40):
    return init_paged_kv_cache(cfg, 2, capacity, PagedSpec(32), "cpu")


@pytest.mark.parametrize("b,s", [(0, 5), (1, 3), (1, 19), (0, 19), (1, 10)])
def test_prefill_refuses_masks_with_zeros_behind_ones(run, b, s):
    cfg, params, ids, mask, forward = run
    with pytest.raises(Launched):
        forward(ids, mask, _cache(cfg))
    mask = mask.clone()
    mask[b, s] = False
    left_padded = (b, s) == (1, 3)  # one pad more
    error = dict(expected_exception=Launched) if left_padded else dict(expected_exception=ValueError, match="left-padded")
    with pytest.raises(**error):
        forward(ids, mask, _cache(cfg))
    with pytest.raises(**error):
        SMP.prefill(params, cfg, ids, mask, max_new_tokens=4, paged=PagedSpec(32))


def test_prefill_takes_rows_of_pads_alone(run):
    cfg, _, ids, mask, forward = run
    for m in (torch.zeros_like(mask), torch.ones_like(mask), mask[:1]):  # one mask for all rows too
        with pytest.raises(Launched):
            forward(ids, m, _cache(cfg))


@pytest.mark.parametrize("graphed", [False, True])
def test_step_refuses_a_mask_of_more_columns(run, graphed):
    """Not the step's column, but the mask of all positions: its first column says nothing about the step."""

    cfg, _, ids, mask, forward = run
    cache = _cache(cfg)._replace(length=20, held=torch.tensor([20, 17], dtype=torch.int32))
    kw = dict(write_pos=torch.tensor([20, 20], dtype=torch.int32)) if graphed else {}
    with pytest.raises(Launched):
        forward(ids[:, :1], mask[:, -1:], cache, "append", **kw)
    with pytest.raises(ValueError, match="attention_mask"):
        forward(ids[:, :1], mask, cache, "append", **kw)
    with pytest.raises(ValueError, match="attention_mask"):
        forward(ids, mask[:, 1:], _cache(cfg))


@pytest.mark.parametrize("graphed", [False, True])
@pytest.mark.parametrize("held", [None, [20, 17]])
@pytest.mark.parametrize("pad", [0, 3])
def test_step_refuses_a_full_cache(run, graphed, held, pad):
    """A token behind the last page would be dropped, and its row's attention would go on without it."""

    cfg, _, ids, mask, forward = run
    kw = dict(write_pos=torch.tensor([63, 63], dtype=torch.int32)) if graphed else {}
    cache = _cache(cfg)._replace(held=None if held is None else torch.tensor(held, dtype=torch.int32), pad=pad)
    assert cache.capacity == 64
    with pytest.raises(Launched):
        forward(ids[:, :1], mask[:, -1:], cache._replace(length=63 + pad), "append", **kw)
    for length in (64, 65, 1000):
        with pytest.raises(ValueError, match="no place"):
            forward(ids[:, :1], mask[:, -1:], cache._replace(length=length + pad), "append", **kw)
