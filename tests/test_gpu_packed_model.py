"""Packed prompts in the model: what a prefill keeps of its description, and the steps that follow it."""

from __future__ import annotations

import pytest
import torch

from gemma4_posttrain_jax_amd import config as C
from gemma4_posttrain_jax_amd import kernels
from gemma4_posttrain_jax_amd import model as M
from gemma4_posttrain_jax_amd import sampler as SMP
from gemma4_posttrain_jax_amd.kvcache import PagedSpec, init_paged_kv_cache
from test_gpu_paged_run import CFG, CFG512, _params, _prompts

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


@pytest.mark.parametrize("lens,tail,capacity", [([300, 1, 64], 7, 320), ([2500], 0, 4096)])
def test_a_prompts_tokens_share_its_table(lens, tail, capacity, device, monkeypatch):
    """The tables that go into the pages' appends hold an entry per token, however long the rows may become; what a row
    holds is read back through its own table, and a prefill of padded rows stores the same places."""

    cfg = C.config_from_hf(CFG)
    params = _params(cfg, device)
    packed, ids, places = _packed(lens, tail, device)
    append, entries = kernels.paged_append, []

    def spy(layer, k, v, *, page_table, **kw):
        entries.append(page_table.numel())
        return append(layer, k, v, page_table=page_table, **kw)

    monkeypatch.setattr(kernels, "paged_append", spy)
    empty = init_paged_kv_cache(cfg, len(lens), capacity, PagedSpec(32), device)
    _, cache = M.forward_gemma4_text(params, ids, places, config=cfg, kv_cache=empty, packed=packed)
    assert entries and max(entries) <= ids.shape[1]
    monkeypatch.undo()
    S = max(lens)
    padded, at = torch.zeros((len(lens), S), dtype=ids.dtype, device=device), 0
    for b, n in enumerate(lens):
        padded[b, S - n:] = ids[0, at:at + n]
        at += n
    mask = torch.arange(S, device=device)[None] >= S - cache.held[:, None]
    pos = (mask.cumsum(dim=1) - 1).clamp(min=0).to(torch.int32)
    other = init_paged_kv_cache(cfg, len(lens), capacity, PagedSpec(32), device)
    _, dense = M.forward_gemma4_text(params, padded, pos, config=cfg, attention_mask=mask, kv_cache=other)
    for i, (x, y) in enumerate(zip(cache.layers, dense.layers)):
        if x is None:
            continue
        table = cache.window_table if cfg.layer_types[i] == C.SLIDING else cache.page_table
        for b, n in enumerate(lens):
            first = max(0, n - cfg.sliding_window) if cfg.layer_types[i] == C.SLIDING else 0
            read = [kernels.paged_read(z, page_table=table[b:b + 1].contiguous(), lengths=cache.held[b:b + 1].contiguous(),
                                       start=first, count=n - first) for z in (x, y)]
            for got, want in zip(*read):
                got, want = got.float(), want.float()
                # places: a token's neighbour is some 1.4 of its size away; the roundings of a few bf16 layers, a few hundredths
                assert bool(((got - want).norm(dim=-1) <= 0.2 * want.norm(dim=-1) + 1e-3).all()), (i, b)
        used = (y.key != 0).flatten(1).any(dim=1)
        assert torch.equal((x.key != 0).flatten(1).any(dim=1), used) and int(used.sum()) >= len(lens)


@pytest.mark.parametrize("other", [-1, 2, 2 ** 31 - 1])
def test_the_rows_of_tokens_of_no_prompt_may_be_any(other, device):
    cfg = C.config_from_hf(CFG)
    params = _params(cfg, device)
    packed, ids, places = _packed([33, 4], 9, device)
    rows = packed.rows.clone()
    rows[37:] = other
    caches = []
    for p in (packed, packed._replace(rows=rows)):
        empty = init_paged_kv_cache(cfg, 2, 64, PagedSpec(32), device)
        caches.append(M.forward_gemma4_text(params, ids, places, config=cfg, kv_cache=empty, packed=p)[1])
    for x, y in zip(*(c.layers for c in caches)):
        if x is not None:
            assert torch.equal(x.key, y.key) and torch.equal(x.value, y.value)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("kwargs,G,pads,S,steps", [(CFG, 3, [0, 11, 59], 60, 50), (CFG512, 2, [5, 0, 64], 70, 40),
                                                   (CFG, 1, [0, 3], 33, 34)])
def test_steps_after_a_group_are_those_of_rows_of_their_own(kwargs, G, pads, S, steps, e4m3, device):
    """Decode steps over shared, forked and copied pages give the bits that they give over a cache in which every row has pages of
    its own with the same contents; each row takes other tokens. Beside them the steps after a prefill of the repeated rows."""

    cfg = C.config_from_hf(kwargs)
    params = _params(cfg, device)
    ids, mask = _prompts(cfg, pads, S, device)
    spec = PagedSpec(32, e4m3)
    cache = SMP.prefill_group(params, cfg, ids, mask, completions=G, max_new_tokens=steps, paged=spec).kv_cache
    B, held = len(pads) * G, cache.held.tolist()
    own = init_paged_kv_cache(cfg, B, cache.capacity, spec, device)
    assert own.capacity == cache.capacity
    for i, (x, y) in enumerate(zip(cache.layers, own.layers)):
        if x is None:
            continue
        sliding = cfg.layer_types[i] == C.SLIDING
        src, dst = (cache.window_table, own.window_table) if sliding else (cache.page_table, own.page_table)
        for b, n in enumerate(held):
            first = max(0, n - cfg.sliding_window) // 32 if sliding else 0
            for e in range(first, -(-n // 32)):
                for t, u in zip(x, y):
                    if t is not None:
                        u[int(dst[b, e])] = t[int(src[b, e])]
    own = own._replace(length=cache.length, held=cache.held.clone())
    G_rows = lambda t: t.repeat_interleave(G, dim=0)  # noqa: E731
    dense = SMP.prefill(params, cfg, G_rows(ids), G_rows(mask), max_new_tokens=steps, paged=spec).kv_cache
    for s in range(steps):
        tok = (torch.arange(B, dtype=torch.int32, device=device) * 13 + 7 * s) % cfg.vocab_size
        got, want, near = [SMP.decode_step(params, cfg, tok, c.held.clone(), c) for c in (cache, own, dense)]
        cache, own, dense = got.kv_cache, want.kv_cache, near.kv_cache
        assert torch.equal(got.logits, want.logits), s
        assert got.kv_cache.held.tolist() == [n + s + 1 for n in held]
        if not e4m3:  # other GEMM shapes and attention roundings of the prompt: a bf16 model's last bits, amplified by a few layers
            far = (got.logits.float() - near.logits.float()).abs().max()
            assert float(far) <= 2e-2 * max(1.0, float(near.logits.float().abs().max())), s


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("kwargs", [CFG, CFG512])
def test_rows_that_ended_are_freed_and_the_pool_compacted(kwargs, e4m3, device):
    """By the counts that the cache carries; the rows that go on give the bits that they give without."""

    cfg = C.config_from_hf(kwargs)
    params = _params(cfg, device)
    ids, mask = _prompts(cfg, [0, 20, 65], 70, device)
    G, steps = 3, 30
    caches = [SMP.prefill_group(params, cfg, ids, mask, completions=G, max_new_tokens=steps, paged=PagedSpec(32, e4m3)).kv_cache
              for _ in range(2)]
    count = lambda c: torch.bincount(c.page_table[c.page_table >= 0].long(), minlength=c.refs.numel()).to(torch.int32)  # noqa: E731
    full = [x for i, x in enumerate(caches[0].layers) if x is not None and cfg.layer_types[i] != C.SLIDING]
    assert torch.equal(caches[0].refs, count(caches[0])) and int(caches[0].refs.max()) == G
    ended = [0, 3, 4, 5, 8]
    going = [b for b in range(9) if b not in ended]
    for s in range(steps):
        tok = (torch.arange(9, dtype=torch.int32, device=device) * 11 + s) % cfg.vocab_size
        got, want = [SMP.decode_step(params, cfg, tok, c.held.clone(), c) for c in caches]
        caches = [got.kv_cache, want.kv_cache]
        assert torch.equal(got.logits[going], want.logits[going]), s
        if s == 10:
            c = caches[0]
            keep = torch.full((9,), c.capacity, dtype=torch.int32, device=device)
            keep[ended] = 0
            kernels.paged_free(c.refs, c.page_table, keep, page_size=32)
            live = int(kernels.paged_compact(full, c.refs, c.page_table))
            assert torch.equal(c.refs, count(c)) and bool((c.refs[:live] > 0).all()) and bool((c.refs[live:] == 0).all())
            assert live < int((caches[1].refs > 0).sum()) and bool((c.page_table[ended] == -1).all())
