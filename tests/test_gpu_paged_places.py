"""Where a model's tokens stand in a paged cache: in the order in which a row's real tokens came, whatever their
position ids, as in the dense cache."""

from __future__ import annotations

import pytest
import torch

import paged_util as P
from gemma4_posttrain_jax_amd import config as C
from gemma4_posttrain_jax_amd import kernels
from gemma4_posttrain_jax_amd import model as M
from gemma4_posttrain_jax_amd import sampler as SMP
from gemma4_posttrain_jax_amd.kvcache import PagedSpec, init_kv_cache, init_paged_kv_cache
from test_gpu_paged_run import CFG, _params, _prompts

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
# a position id per number of real tokens before the token
POSITIONS = {"count": lambda n: n, "gaps": lambda n: 3 * n + 50, "stalls": lambda n: n // 2}


@pytest.mark.parametrize("graphed", [False, True])
@pytest.mark.parametrize("positions", POSITIONS)
def test_places_are_the_dense_caches(device, positions, graphed):
    """A padded prompt and steps, one row of which pauses, with positions that count, leave gaps or repeat: every
    step's attention is over the row's tokens so far, and layer 0 (whose input is the embedding alone) holds the keys
    of the dense cache's real slots one after the other."""

    cfg = C.config_from_hf(dict(CFG, sliding_window=200))  # a dense ring that drops nothing
    params = _params(cfg, device)
    pads, S, steps = [0, 11, 59], 60, 8
    ids, mask = _prompts(cfg, pads, S, device)
    position = POSITIONS[positions]
    pos = position((mask.cumsum(-1) - 1).clamp(min=0)).to(torch.int32)
    run = dict(config=cfg, attention_mask=mask, cache_mode="prefill", logits_to_keep=1)
    dense = M.forward_gemma4_lm(params, ids, pos, kv_cache=init_kv_cache(cfg, 3, S + steps, BF16, device), **run)
    paged = M.forward_gemma4_lm(params, ids, pos, kv_cache=init_paged_kv_cache(cfg, 3, S + steps, PagedSpec(32), device), **run)
    assert torch.equal(dense.logits, paged.logits)
    dense, paged = dense.kv_cache, paged.kv_cache
    step = SMP.GraphedDecodeStep(params, cfg, paged) if graphed else None
    counts = mask.sum(-1).to(torch.int32)
    seen, attend = [], kernels.paged_decode_attention
    real = [mask]
    g = torch.Generator().manual_seed(5)
    for i in range(steps):
        tok = torch.randint(0, cfg.vocab_size, (3,), generator=g).to(torch.int32).to(device)
        on = torch.tensor([True, i not in (1, 2), True], device=device)
        real.append(on[:, None])
        dense = SMP.decode_step(params, cfg, tok, position(counts).int(), dense, attention_mask=on).kv_cache
        if graphed:
            step.step(tok, position(counts).int(), on)
        else:
            with pytest.MonkeyPatch.context() as patch:
                patch.setattr(kernels, "paged_decode_attention",
                              lambda *a, lengths, **kw: (seen.append(lengths.tolist()), attend(*a, lengths=lengths, **kw))[1])
                paged = SMP.decode_step(params, cfg, tok, position(counts).int(), paged, attention_mask=on).kv_cache
            want = [int(n) + 1 if o else 0 for n, o in zip(counts, on)]
            assert seen == [want] * cfg.num_hidden_layers, i
            seen.clear()
        counts += on
    cache = step.kv_cache if graphed else paged
    assert cache.length == S + steps
    k_dense, _ = dense.layers[0].reference_layout()
    k_paged, _ = kernels.paged_read(cache.layers[0], page_table=cache.window_table, lengths=counts, start=0, count=S + steps)
    real = torch.cat(real, dim=1)
    for b in range(3):
        want = k_dense[b, : S + steps][real[b]].double()
        # the dense cache rounds after the norm, the rotation's factors and the result, the pages once: 4 half steps, each
        # of at most the size of the rotated pair; the f32 steps between are less than one more
        size = want.abs() + want.abs().roll(want.shape[-1] // 2, -1)
        n = int(counts[b])
        assert want.shape[0] == n
        assert ((k_paged[b, :n].double() - want).abs() <= 5 * P.U_BF16 * size).all(), b
        assert (k_paged[b, n:] == 0).all()
    assert torch.equal(cache.held, counts)


def test_an_older_cache_object_goes_on_from_its_own_tokens(device):
    """Two steps from one cache object, and captured steps made from it: each goes on from the tokens that the object
    held, and a captured step's snapshot keeps its count."""

    cfg = C.config_from_hf(CFG)
    params = _params(cfg, device)
    ids, mask = _prompts(cfg, [0, 7], 30, device)
    tok = lambda i: torch.tensor([5 + i, 90 + i], dtype=torch.int32, device=device)  # noqa: E731
    n = mask.sum(-1).to(torch.int32)
    fresh = lambda: SMP.prefill(params, cfg, ids, mask, max_new_tokens=8, paged=PagedSpec(32)).kv_cache  # noqa: E731
    step = lambda i, at, cache: SMP.decode_step(params, cfg, tok(i), n + at, cache)  # noqa: E731
    want = step(1, 0, fresh()).logits
    cache = fresh()
    first = step(0, 0, cache)
    assert torch.equal(step(1, 0, cache).logits, want)
    assert torch.equal(cache.held, n) and torch.equal(first.kv_cache.held, n + 1)
    gs = SMP.GraphedDecodeStep(params, cfg, cache)
    on = torch.ones(2, dtype=torch.bool, device=device)
    assert torch.equal(gs.step(tok(1), n, on), want[:, -1].float())
    snapshot = gs.kv_cache
    after = gs.step(tok(2), n + 1, on).clone()
    assert torch.equal(cache.held, n) and torch.equal(snapshot.held, n + 1) and torch.equal(gs.kv_cache.held, n + 2)
    assert torch.equal(step(2, 1, snapshot).logits[:, -1].float(), after)


@pytest.mark.parametrize("graphed", [False, True])
def test_places_of_a_cache_without_counts_are_the_positions(device, graphed):
    """Pages that the caller fills itself, rows of any length: a step's token goes to its position id."""

    cfg = C.config_from_hf(CFG)
    params = _params(cfg, device)
    ids, mask = _prompts(cfg, [0, 7], 30, device)
    n = mask.sum(-1).to(torch.int32)
    tok, on = torch.tensor([5, 90], dtype=torch.int32, device=device), torch.ones(2, dtype=torch.bool, device=device)
    logits = []
    for counted in (True, False):
        cache = SMP.prefill(params, cfg, ids, mask, max_new_tokens=8, paged=PagedSpec(32)).kv_cache
        if not counted:
            cache = cache._replace(held=None)
        if graphed:
            gs = SMP.GraphedDecodeStep(params, cfg, cache)
            logits.append([gs.step(tok + i, n + i, on).clone() for i in range(3)])
            cache = gs.kv_cache
        else:
            logits.append([])
            for i in range(3):
                out = SMP.decode_step(params, cfg, tok + i, n + i, cache)
                logits[-1].append(out.logits.clone())
                cache = out.kv_cache
        assert (cache.held is None) == (not counted) and cache.length == 33
    assert all(torch.equal(a, b) for a, b in zip(*logits))


@pytest.mark.parametrize("graphed", [False, True])
def test_steps_up_to_a_full_cache(device, graphed):
    """Rows may fill their last page, pads that all of them have not counted; the step behind it is refused. Up to
    there the logits are those of a wider table."""

    cfg = C.config_from_hf(CFG)
    params = _params(cfg, device)
    ids, mask = _prompts(cfg, [4, 9], 24, device)
    n = mask.sum(-1).to(torch.int32)
    tok, on = torch.tensor([5, 90], dtype=torch.int32, device=device), torch.ones(2, dtype=torch.bool, device=device)
    logits = []
    for more in (8, 40):  # one page or two
        cache = SMP.prefill(params, cfg, ids, mask, max_new_tokens=more, paged=PagedSpec(32)).kv_cache
        assert cache.capacity == (32 if more == 8 else 64) and cache.pad == 4
        gs = SMP.GraphedDecodeStep(params, cfg, cache) if graphed else None
        logits.append([])
        for i in range(12):  # the longest row holds 20 tokens of the prompt
            if graphed:
                logits[-1].append(gs.step(tok + i, n + i, on).clone())
            else:
                out = SMP.decode_step(params, cfg, tok + i, n + i, cache)
                logits[-1].append(out.logits.clone())
                cache = out.kv_cache
        if more == 8:
            with pytest.raises(ValueError, match="no place"):
                gs.step(tok, n + 12, on) if graphed else SMP.decode_step(params, cfg, tok, n + 12, cache)
            if graphed:
                with pytest.raises(ValueError, match="no place"):
                    gs.replay_logits()
                assert gs.length == 36 and gs.kv_cache.held.tolist() == [32, 27]
    assert all(torch.equal(a, b) for a, b in zip(*logits))


def test_a_drawing_step_refuses_a_full_cache(device):
    cfg = C.config_from_hf(CFG)
    params = _params(cfg, device)
    ids, mask = _prompts(cfg, [0, 9], 31, device)
    cache = SMP.prefill(params, cfg, ids, mask, max_new_tokens=1, paged=PagedSpec(32)).kv_cache
    gs = SMP.GraphedDecodeStep(params, cfg, cache, temperature=0.0)
    n, on = mask.sum(-1).to(torch.int32), torch.ones(2, dtype=torch.bool, device=device)
    gs.step_sample(n, n, on)
    with pytest.raises(ValueError, match="no place"):
        gs.step_sample(n, n + 1, on)
    with pytest.raises(ValueError, match="no place"):
        gs.replay_sample()
    with pytest.raises(ValueError, match="no place"):
        SMP.GraphedDecodeStep(params, cfg, gs.kv_cache)
