"""Several completions per prompt: the packed prefill, the fork of its pages and the rings' copies in the model, then
decode steps and generate; and the pool's operators with drafted tokens, as a serving loop uses them together."""

from __future__ import annotations

import pytest
import torch

import paged_util as P
import pool_util as plain
from gemma4_posttrain_jax_amd import config as C
from gemma4_posttrain_jax_amd import kernels
from gemma4_posttrain_jax_amd import model as M
from gemma4_posttrain_jax_amd import sampler as SMP
from gemma4_posttrain_jax_amd.kvcache import PagedSpec, init_paged_kv_cache, new_layer_cache, new_paged_layer
from packed_util import packed_reference
from test_gpu_paged_run import CFG, CFG512, _params, _prompts

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _slots(layer, table, length, window):
    """The bits of a row's keys and values, position by position, of those that its attention reads."""

    first = max(0, length - window) if window else 0
    count = length - first
    k, v = kernels.paged_read(layer, page_table=table, start=first, count=max(count, 1),
                              lengths=torch.full((table.shape[0],), length, dtype=torch.int32, device=table.device))
    return torch.stack([k, v])[:, :, :count]


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("kwargs,G,pads,S,steps", [(CFG, 3, [0, 11, 59], 60, 40), (CFG512, 1, [5, 0], 70, 3),
                                                   (CFG, 4, [0], 1, 2), (CFG, 2, [63, 32, 0, 31, 1], 64, 34)])
def test_the_rows_hold_their_prompt(kwargs, G, pads, S, steps, e4m3, device, monkeypatch):
    """Packed attention in the model is that of 64 bits over what it is given; what it stores is the prepared k / v
    of each prompt's tokens, bit for bit the same in all its rows; and each step writes pages of its row alone."""

    cfg = C.config_from_hf(kwargs)
    params = _params(cfg, device)
    ids, mask = _prompts(cfg, pads, S, device)
    lens = [S - p for p in pads]
    attend, calls = kernels.packed_prefill_attention, []

    def checked(q, k, vt, starts, *, window, longest):
        assert longest == max(lens)
        out = attend(q, k, vt, starts, window=window, longest=longest)
        T = q.shape[0]
        layer = new_layer_cache(1, q.shape[1], q.shape[3], T, False, BF16, device)._replace(key=k, value_t=vt)
        kk, vv = (t[0].cpu() for t in layer.reference_layout())
        want, bound = packed_reference(q.cpu(), kk, vv, lens, window)
        assert bool(((out.cpu().double() - want).abs() <= bound).all())
        calls.append(window)
        return out

    monkeypatch.setattr(kernels, "packed_prefill_attention", checked)
    out = SMP.prefill_group(params, cfg, ids, mask, completions=G, max_new_tokens=steps, paged=PagedSpec(32, e4m3))
    assert calls == [cfg.sliding_window if t == C.SLIDING else 0 for t in cfg.layer_types]
    cache, N = out.kv_cache, len(pads)
    assert out.logits.shape[0] == N * G and cache.batch == N * G and cache.held.tolist() == [n for n in lens for _ in range(G)]
    dense = SMP.prefill(params, cfg, ids, mask, max_new_tokens=steps, paged=PagedSpec(32, e4m3))
    # other GEMM shapes and attention roundings: a bf16 model's last bits, amplified by a few layers
    assert float((out.logits[::G].float() - dense.logits.float()).abs().max()) <= 2e-2 * max(1.0, float(dense.logits.float().abs().max()))

    def check_rows(cache, host):
        for i, layer in enumerate(cache.layers):
            if layer is None:
                continue
            window = cfg.sliding_window if cfg.layer_types[i] == C.SLIDING else 0
            table = cache.window_table if window else cache.page_table
            for p in range(N):
                rows = _slots(layer, table[p * G:(p + 1) * G].contiguous(), host[p], window)
                assert torch.equal(rows.view(torch.int16), rows[:, :1].expand_as(rows).contiguous().view(torch.int16)), (i, p)

    check_rows(cache, lens)
    # the first layer's keys and values are the prepared ones (later layers': through the checked attention)
    table = cache.window_table if cfg.layer_types[0] == C.SLIDING else cache.page_table
    for p, n in enumerate(lens):
        want = _slots(dense.kv_cache.layers[0], dense.kv_cache.window_table[p:p + 1].contiguous(), n, cfg.sliding_window).double()
        got = _slots(cache.layers[0], table[p * G:p * G + 1].contiguous(), n, cfg.sliding_window).double()
        step = 2.0 ** -3 if e4m3 else 2.0 ** -7  # a stored value next to a border may round the other way: one step
        assert bool(((got - want).abs() <= step * want.abs() + 2.0 ** -9 * want.abs().amax()).all())
    # all rows take the same tokens: they stay equal, in pages of their own
    for s in range(steps):
        tok = torch.arange(N, dtype=torch.int32, device=device).repeat_interleave(G) * 7 + s
        d = SMP.decode_step(params, cfg, tok, cache.held, cache)
        cache = d.kv_cache
        x = d.logits.view(N, G, -1)
        assert torch.equal(x, x[:, :1].expand_as(x))
    check_rows(cache, [n + steps for n in lens])
    for i, layer in enumerate(cache.layers):  # the page of the newest token is a row's own
        if layer is not None:
            table = cache.window_table if cfg.layer_types[i] == C.SLIDING else cache.page_table
            own = [table[b, (n - 1) // 32].item() for b, n in enumerate(cache.held.tolist())]
            assert len(set(own)) == N * G


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("top_k,temperature", [(0, 0.0), (0, 1.0), (8, 0.7), (0, 25.0)])
def test_generate_several_completions(e4m3, top_k, temperature, device):
    """Greedy: the completions of a prompt are one. Hot (this model repeats its last token at the others): other noise per
    row. The same call gives the same batch."""

    cfg = C.config_from_hf(CFG)
    params = _params(cfg, device)
    ids, mask = _prompts(cfg, [0, 9, 30], 40, device)
    sc = SMP.SamplerConfig(max_prompt_len=40, max_new_tokens=50, temperature=temperature, top_k=top_k, seed=3)
    run = SMP.NativeRollout(params, cfg, sc, paged=PagedSpec(32, e4m3), completions=4)
    batch = run.generate(ids, mask)
    assert batch.completion_ids.shape == (12, 50) and batch.prompt_ids.shape == (12, 40)
    assert torch.equal(batch.prompt_ids, ids.repeat_interleave(4, dim=0))
    rows = batch.completion_ids.view(3, 4, 50)
    if temperature == 0:
        assert torch.equal(rows, rows[:, :1].expand_as(rows))
    elif temperature > 20:
        assert not torch.equal(rows[:, 0], rows[:, 1])
    again = run.generate(ids, mask)
    assert torch.equal(again.completion_ids, batch.completion_ids) and torch.equal(again.rollout_logps, batch.rollout_logps)


def test_generate_ends_at_eos_and_leaves_other_rows(device):
    cfg = C.config_from_hf(CFG)
    params = _params(cfg, device)
    ids, mask = _prompts(cfg, [0, 5], 33, device)
    sc = SMP.SamplerConfig(max_prompt_len=33, max_new_tokens=40, temperature=1.0, seed=1, eos_ids=tuple(range(0, 512, 16)))
    batch = SMP.generate(params, cfg, ids, mask, sampler_config=sc, paged=PagedSpec(64), completions=5)
    free = SMP.generate(params, cfg, ids, mask, sampler_config=sc._replace(eos_ids=()), paged=PagedSpec(64), completions=5)
    for b in range(10):
        n = int(batch.lengths[b])
        assert torch.equal(batch.completion_ids[b, :n], free.completion_ids[b, :n])
        assert n == 40 or int(batch.completion_ids[b, n - 1]) % 16 == 0


def test_group_refusals(device):
    cfg = C.config_from_hf(CFG)
    params = _params(cfg, device)
    ids, mask = _prompts(cfg, [0, 9], 20, device)
    sc = SMP.SamplerConfig(max_prompt_len=20, max_new_tokens=5)
    with pytest.raises(ValueError, match="PagedSpec"):
        SMP.generate(params, cfg, ids, mask, sampler_config=sc, completions=2)
    with pytest.raises(ValueError, match="needs a token"):
        SMP.prefill_group(params, cfg, ids, mask & (torch.arange(2, device=device) > 0)[:, None], completions=2, max_new_tokens=5)
    with pytest.raises(ValueError, match="completions 0"):
        SMP.prefill_group(params, cfg, ids, mask, completions=0, max_new_tokens=5)
    with pytest.raises(ValueError, match="page_size"):
        SMP.prefill_group(params, cfg, ids, mask, completions=2, max_new_tokens=5, paged=PagedSpec(48))
    out = SMP.prefill_group(params, cfg, ids, mask, completions=2, max_new_tokens=1, paged=PagedSpec(32))
    cache = out.kv_cache
    for _ in range(12):  # 20 + 12 positions fill the one page
        tok = torch.zeros(4, dtype=torch.int32, device=device)
        cache = SMP.decode_step(params, cfg, tok, cache.held, cache).kv_cache
    with pytest.raises(ValueError, match="no place"):
        SMP.decode_step(params, cfg, tok, cache.held, cache)


def test_short_rows_have_place_as_long_as_the_longest(device):
    """100 and 10 tokens, five more asked for, pages of 32: every row has a page for each token up to the 28th, which fills the
    longest row's last page; the 29th is refused."""

    cfg = C.config_from_hf(CFG)
    params = _params(cfg, device)
    ids, mask = _prompts(cfg, [0, 90], 100, device)
    cache = SMP.prefill_group(params, cfg, ids, mask, completions=2, max_new_tokens=5, paged=PagedSpec(32)).kv_cache
    tok = torch.zeros(4, dtype=torch.int32, device=device)
    for _ in range(28):
        cache = SMP.decode_step(params, cfg, tok, cache.held, cache).kv_cache
    last = ((cache.held - 1) // 32).long()
    assert cache.held.tolist() == [128, 128, 38, 38]
    assert bool((cache.page_table.gather(1, last[:, None]) >= 0).all())
    full = next(i for i, t in enumerate(cfg.layer_types) if t != C.SLIDING and cache.layers[i] is not None)
    k, _ = kernels.paged_read(cache.layers[full], page_table=cache.page_table, lengths=cache.held, start=0, count=128)
    assert all(bool((k[b, :n].float().abs().amax(dim=(1, 2)) > 0).all()) for b, n in enumerate(cache.held.tolist()))
    with pytest.raises(ValueError, match="no place"):
        SMP.decode_step(params, cfg, tok, cache.held, cache)


def test_packed_tokens_of_no_prompt_are_not_stored(device):
    cfg = C.config_from_hf(CFG)
    params = _params(cfg, device)
    lens, T = [20, 7], 40
    ids = torch.arange(T, device=device)[None] * 3 % 500
    cu = torch.tensor([0, 20, 27], dtype=torch.int32, device=device)
    starts = kernels.packed_starts(cu, T)
    rows = torch.tensor([0] * 20 + [1] * 7 + [0] * 13, dtype=torch.int32, device=device)
    places = (torch.arange(T, dtype=torch.int32, device=device) - starts)[None]
    packed = M.PackedPrompts(starts, rows, cu.diff(), 20)
    empty = init_paged_kv_cache(cfg, 2, 64, PagedSpec(32), device)
    _, cache = M.forward_gemma4_text(params, ids, places, config=cfg, kv_cache=empty, packed=packed)
    assert cache.held.tolist() == lens
    for i, layer in enumerate(cache.layers):
        if layer is None:
            continue
        table = cache.window_table if cfg.layer_types[i] == C.SLIDING else cache.page_table
        k, v = kernels.paged_read(layer, page_table=table, lengths=torch.full_like(cache.held, 32), start=0, count=32)
        for b, n in enumerate(lens):
            assert bool((k[b, n:] == 0).all()) and bool((v[b, n:] == 0).all()) and bool((k[b, n - 1] != 0).any())
    with pytest.raises(ValueError, match="attention_mask"):
        M.forward_gemma4_text(params, ids, places, config=cfg, kv_cache=empty, packed=packed,
                              attention_mask=torch.ones(1, T, device=device))


@pytest.mark.parametrize("e4m3", [False, True])
def test_a_serving_loop(e4m3, device):
    """Prompts packed, stored and forked; then drafted tokens appended, attended to, verified and, where rejected, their
    pages given back; rows that end are freed and the pool compacted. Every attention is that of 64 bits over the
    tokens that plain lists say each row holds, every table and count the lists' own."""

    H, R, D, ps, N, G, K, V = 2, 4, 128, 32, 3, 3, 5, 64
    g = torch.Generator().manual_seed(21)
    lens = [70, 33, 64]
    T = sum(lens)
    P_pages, M = 90, 8
    layers = [new_paged_layer(P_pages, H, D, ps, e4m3=e4m3, device=device) for _ in range(2)]
    refs, table = [0] * P_pages, [[-1] * M for _ in range(N)]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    d_refs, d_table = i32(refs), i32(table)
    assert kernels.paged_reserve(d_refs, d_table, i32(lens), page_size=ps).tolist() == [plain.reserve(refs, table, lens, ps)]

    # the prompts: attention over their own chunk, k / v into the pages
    rnd = lambda *s: torch.randn(s, generator=g).to(BF16)  # noqa: E731
    q, k, v = rnd(T, H, R, D), rnd(T, H, D), rnd(T, H, D)
    q = (q.float() * 2 / D ** 0.5).to(BF16)
    chunk = new_layer_cache(1, H, D, T, False, BF16, device)
    kernels.kv_append(chunk, k.to(device)[None], v.to(device)[None], write_pos=0)
    cu = i32([0] + list(torch.tensor(lens).cumsum(0)))
    starts = kernels.packed_starts(cu, T)
    out = kernels.packed_prefill_attention(q.to(device), chunk.key, chunk.value_t, starts)
    want, bound = packed_reference(q, k, v, lens, 0)
    assert bool(((out.cpu().double() - want).abs() <= bound).all())
    row = torch.repeat_interleave(torch.arange(N), torch.tensor(lens))
    place = torch.arange(T) - torch.tensor([0] + lens).cumsum(0)[row]
    for layer in layers:
        kernels.paged_append(layer, k.to(device)[:, None], v.to(device)[:, None], write_pos=place.to(torch.int32).to(device),
                             page_table=d_table[row.to(device)].contiguous())
    text = [[(k[t], v[t]) for t in range(T) if row[t] == p] for p in range(N)]  # what each row holds, as lists

    # to G completions each
    parents = [p for p in range(N) for _ in range(G)]
    d_rows, short = kernels.paged_fork(layers, d_refs, d_table, i32(parents), i32(lens))
    rows, _, lacking = plain.fork(refs, table, parents, lens, ps, M)
    kernels.paged_free(d_refs, d_table, i32([0] * N), page_size=ps)
    plain.free(refs, table, [0] * N, ps)
    assert short.tolist() == [lacking] == [0] and d_rows.tolist() == rows and d_refs.tolist() == refs
    text = [list(text[p]) for p in parents]
    held, alive = [lens[p] for p in parents], [True] * (N * G)

    for step in range(8):
        B = N * G
        # a step of K + 1 tokens per row: the last one and K drafts
        want_len = [(n + K + 1) if a else 0 for n, a in zip(held, alive)]
        kernels.paged_reserve(d_refs, d_rows, i32(want_len), page_size=ps)
        plain.reserve(refs, rows, want_len, ps)
        assert d_rows.tolist() == rows and d_refs.tolist() == refs
        kk, vv, qq = rnd(B, K + 1, H, D), rnd(B, K + 1, H, D), (rnd(B, K + 1, H, R, D).float() * 2 / D ** 0.5).to(BF16)
        for layer in layers:
            kernels.paged_append(layer, kk.to(device), vv.to(device), page_table=d_rows,
                                 write_pos=i32([n if a else -(K + 1) for n, a in zip(held, alive)]))
        for b in range(B):
            if alive[b]:
                text[b] = text[b][:held[b]] + [(kk[b, s], vv[b, s]) for s in range(K + 1)]
        lengths = i32([n + s + 1 if a else 0 for n, a in zip(held, alive) for s in range(K + 1)])
        att = kernels.paged_decode_attention(layers[step % 2], qq.to(device).view(B * (K + 1), H, R, D), lengths=lengths,
                                             page_table=d_rows.repeat_interleave(K + 1, dim=0))
        for b in range(B):
            if not alive[b]:
                continue
            ks, vs = (torch.stack(x)[None].transpose(1, 2) for x in zip(*text[b]))  # [1, H, n, D]
            if e4m3:
                ks, vs = P.dequantised(ks), P.dequantised(vs)
            n = ks.shape[2]
            pad = -n % ps
            ks, vs = (torch.nn.functional.pad(x.double(), (0, 0, 0, pad)) for x in (ks, vs))
            one = torch.zeros((K + 1, 1), dtype=torch.int32)
            want, bound = P.attention(ks, vs, one.expand(K + 1, 1), [held[b] + s + 1 for s in range(K + 1)], qq[b], 0) \
                if n <= ps else P.attention(
                    torch.cat(ks.split(ps, dim=2)), torch.cat(vs.split(ps, dim=2)),
                    torch.arange((n + pad) // ps, dtype=torch.int32).expand(K + 1, -1), [held[b] + s + 1 for s in range(K + 1)],
                    qq[b], 0)
            got = att.view(B, K + 1, H, R, D)[b].cpu().double()
            assert bool(((got - want).abs() <= bound).all()), (step, b)
        # verified
        logits = torch.randn(B, K + 1, V, generator=g)
        near = logits[:, :K] + 0.3 * torch.randn(B, K, V, generator=g)
        drafts = (near - torch.log(-torch.log(torch.rand(B, K, V, generator=g).clamp(min=1e-7)))).argmax(-1).to(torch.int32)
        tokens, count, _ = kernels.verify_draft(
            logits.to(device), drafts.to(device), torch.rand(B, K, generator=g).to(device),
            torch.rand(B, V, generator=g).to(device), temperature=1.0, draft_logits=near.to(device),
            draft_lengths=i32([K if a else 0 for a in alive]))
        kept = count.tolist()
        assert all(tokens[b, :kept[b]].tolist() == drafts[b, :kept[b]].tolist() for b in range(B))
        held = [n + 1 + c if a else 0 for n, a, c in zip(held, alive, kept)]
        # a row ends now and then; rejected positions' pages go back
        for b in range(B):
            if alive[b] and (step * 5 + b) % 11 == 0:
                alive[b], held[b], text[b] = False, 0, []
        kernels.paged_free(d_refs, d_rows, i32(held), page_size=ps)
        plain.free(refs, rows, held, ps)
        assert d_rows.tolist() == rows and d_refs.tolist() == refs
        if step % 3 == 2:
            live = kernels.paged_compact(layers, d_refs, d_rows)
            n, _ = plain.compact(refs, rows)
            assert live.tolist() == [n] and d_rows.tolist() == rows and d_refs.tolist() == refs
    assert sum(alive) not in (0, N * G)
