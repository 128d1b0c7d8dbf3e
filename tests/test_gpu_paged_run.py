"""The paged cache's operators together, as a rollout uses them: prompt and step appends with the attention
that reads them, the model's prefill and decode steps, generate, graphs and streams."""

from __future__ import annotations

import math

import pytest
import torch

import paged_util as P
from gemma4_posttrain_jax_amd import config as C
from gemma4_posttrain_jax_amd import kernels
from gemma4_posttrain_jax_amd import model as M
from gemma4_posttrain_jax_amd import sampler as SMP
from gemma4_posttrain_jax_amd.kvcache import PagedSpec, init_paged_kv_cache, new_paged_layer

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
CFG = dict(
    vocab_size=512, hidden_size=128, intermediate_size=256, num_hidden_layers=5, num_attention_heads=8,
    num_key_value_heads=2, head_dim=64, global_head_dim=64,
    layer_types=["sliding_attention", "sliding_attention", "full_attention", "sliding_attention", "full_attention"],
    sliding_window=40, num_kv_shared_layers=2, hidden_size_per_layer_input=0, final_logit_softcapping=30.0,
)
CFG512 = dict(CFG, global_head_dim=512, sliding_window=33, num_kv_shared_layers=0)


def _params(cfg, device):
    g = torch.Generator().manual_seed(3)
    w = lambda *s, scale=0.05: (torch.randn(s, generator=g) * scale).to(BF16).to(device)  # noqa: E731
    norm = lambda n: M.RMSNormParams((1 + 0.1 * torch.randn(n, generator=g)).to(BF16).to(device))  # noqa: E731
    layers = []
    for i in range(cfg.num_hidden_layers):
        own = not C.is_kv_shared(cfg, i)
        D, H = C.layer_head_dim(cfg, i), C.layer_kv_heads(cfg, i)
        R = cfg.num_attention_heads // H
        m, F = cfg.hidden_size, C.layer_intermediate_size(cfg, i)
        qk = lambda: M.RMSNormParams((0.3 * (1 + 0.1 * torch.randn(D, generator=g))).to(BF16).to(device))  # noqa: E731
        att = M.AttentionParams(w(m, R, H, D), w(m, H, D) if own else None, w(m, H, D) if own else None, w(R, H, D, m), qk(),
                                qk() if own else None)
        layers.append(M.DecoderLayerParams(norm(m), att, norm(m), norm(m), M.MLPParams(w(m, F), w(m, F), w(F, m)), norm(m),
                                           None, torch.ones((), dtype=BF16, device=device)))
    return M.Gemma4TextParams(w(cfg.vocab_size, cfg.hidden_size, scale=0.5), None, None, None, tuple(layers),
                              norm(cfg.hidden_size))


def _prompts(cfg, pads, S, device):
    g = torch.Generator().manual_seed(4)
    ids = torch.randint(0, cfg.vocab_size, (len(pads), S), generator=g).to(torch.int32).to(device)
    mask = torch.arange(S)[None, :] >= torch.tensor(pads)[:, None]
    return ids, mask.to(device)


@pytest.mark.parametrize("e4m3,D,H,R,ps,window,pads,S,steps", [
    (True, 64, 2, 3, 32, 40, [0, 17, 69], 70, 70), (False, 128, 1, 8, 32, 0, [5, 0], 33, 40),
    (True, 256, 2, 4, 64, 100, [0, 90], 91, 45), (True, 512, 1, 8, 32, 0, [30, 2, 0], 31, 36),
])
def test_prompt_and_steps(device, e4m3, D, H, R, ps, window, pads, S, steps):
    """A prompt chunk, then one token a step: what the pages hold is checked against the prepared k / v, each
    step's attention against 64 bits over what the pages hold. Sliding: a cyclic table of the fewest pages."""

    B, eps, total = len(pads), 1e-6, S + steps
    g = torch.Generator().manual_seed(7)
    M_ = (total + ps - 1) // ps
    cycle = min(M_, (window + ps - 2) // ps + 1) if window else M_
    order = torch.randperm(B * cycle, generator=g).view(B, cycle).to(torch.int32)
    table = order[:, torch.arange(M_) % cycle].contiguous()
    layer = new_paged_layer(B * cycle, H, D, ps, e4m3=e4m3, device=device)
    qw, kw = ((0.3 + 0.1 * torch.rand(D, generator=g)).to(BF16) for _ in range(2))
    rows = torch.randn((B, total, (R + 2) * H * D), generator=g).to(BF16)
    angle = torch.rand((B, total, D // 2), generator=g) * 30
    cos, sin = (torch.cat([f(angle)] * 2, dim=-1) for f in (torch.cos, torch.sin))
    q_all = rows[..., : H * R * D].view(B, total, H, R, D)
    k_all, v_all = rows[..., H * R * D: H * (R + 1) * D].view(B, total, H, D), rows[..., H * (R + 1) * D:].view(B, total, H, D)
    k_want, k_err = P.prepared(k_all, kw, True, (cos[:, :, None], sin[:, :, None]), eps)
    v_want, v_err = P.prepared(v_all, None, True, None, eps)
    dev_table, common = table.to(device), dict(flags=P.ALL_FLAGS, eps=eps, q_norm_weight=qw.to(device),
                                               k_norm_weight=kw.to(device))
    for s0, n in [(0, S)] + [(S + i, 1) for i in range(steps)]:
        part = rows[:, s0: s0 + n].contiguous().to(device)
        q = part[..., : H * R * D].view(B, n, H, R, D)
        q_out = torch.empty((B, n, H, R, D), dtype=BF16, device=device)
        pos = torch.tensor([s0 - p for p in pads], dtype=torch.int32, device=device)
        kernels.paged_append(layer, part[..., H * R * D: H * (R + 1) * D].view(B, n, H, D),
                             part[..., H * (R + 1) * D:].view(B, n, H, D), page_table=dev_table, write_pos=pos,
                             keep=window, q=q, q_out=q_out, rope_cos=cos[:, s0: s0 + n].contiguous().to(device),
                             rope_sin=sin[:, s0: s0 + n].contiguous().to(device), **common)
        lengths = [s0 + n - p for p in pads]
        out = kernels.paged_decode_attention(layer, q_out[:, -1].contiguous(), page_table=dev_table,
                                             lengths=torch.tensor(lengths, dtype=torch.int32, device=device), window=window)
        if n > 1 or s0 % 7 == 0 or s0 == total - 1:
            k, v = P.slots_of(layer)
            want, bound = P.attention(k, v, table, lengths, q_out[:, -1], window)
            assert ((out.cpu().double() - want).abs() <= bound).all(), s0
            for b, length in enumerate(lengths):
                for p in range(max(0, length - window) if window else 0, length):
                    s = p + pads[b]
                    for got, y, err in ((k, k_want, k_err), (v, v_want, v_err)):
                        y, err, x = y[b, s], err[b, s], got[int(table[b, p // ps]), :, p % ps]
                        u = P.U_E4M3 if e4m3 else P.U_BF16
                        floor = 2.0 ** -10 * 2 * y.abs().amax(dim=-1, keepdim=True) / 448 if e4m3 else 0.0
                        assert ((x - y).abs() <= u * y.abs() + floor + (1 + u) * err).all(), (s0, b, p)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("kwargs", [CFG, CFG512])
def test_model_steps_in_pages(device, kwargs, e4m3, monkeypatch):
    """The prefill is the dense path's, bit by bit. Every decode step's attention, with the q, table, lengths and
    window that the model gives it, is that of 64 bits over what the pages hold, and the pages hold the prepared
    k / v of every step, past the sliding layers' window and cycle of pages."""

    cfg = C.config_from_hf(kwargs)
    params = _params(cfg, device)
    pads, S, steps = [0, 11, 59], 60, 50
    ids, mask = _prompts(cfg, pads, S, device)
    dense = SMP.prefill(params, cfg, ids, mask, max_new_tokens=steps)
    paged = SMP.prefill(params, cfg, ids, mask, max_new_tokens=steps, paged=PagedSpec(32, e4m3))
    assert torch.equal(dense.logits, paged.logits)
    cache = paged.kv_cache
    calls, appends = [], []
    attend, append = kernels.paged_decode_attention, kernels.paged_append

    def checked_attend(layer, q, *, page_table, lengths, window):
        out = attend(layer, q, page_table=page_table, lengths=lengths, window=window)
        calls.append((layer, page_table, lengths.tolist(), window))
        if step % 9 == 0 or step == steps - 1:
            want, bound = P.attention(*P.slots_of(layer), page_table.cpu(), lengths.tolist(), q, window)
            assert ((out.cpu().double() - want).abs() <= bound).all(), step
        return out

    def checked_append(layer, k, v, **kw):
        append(layer, k, v, **kw)
        appends.append(layer)
        got = P.slots_of(layer)
        rope = (kw["rope_cos"].cpu()[:, 0, None], kw["rope_sin"].cpu()[:, 0, None])
        for g, x, w, r in zip(got, (k, v), (kw["k_norm_weight"].cpu(), None), (rope, None)):
            want, err = P.prepared(x[:, 0].cpu(), w, True, r, kw["eps"])
            for b, p in enumerate(kw["write_pos"].tolist()):
                y = g[int(kw["page_table"][b, p // 32]), :, p % 32]
                u = P.U_E4M3 if e4m3 else P.U_BF16
                floor = 2.0 ** -10 * 2 * want[b].abs().amax(dim=-1, keepdim=True) / 448 if e4m3 else 0.0
                assert ((y - want[b]).abs() <= u * want[b].abs() + floor + (1 + u) * err[b]).all(), (step, b)

    monkeypatch.setattr(kernels, "paged_decode_attention", checked_attend)
    monkeypatch.setattr(kernels, "paged_append", checked_append)
    g = torch.Generator().manual_seed(5)
    n = mask.sum(-1).to(torch.int32)
    own = [i for i, layer in enumerate(cache.layers) if layer is not None]
    for step in range(steps):
        calls.clear(), appends.clear()
        tok = torch.randint(0, cfg.vocab_size, (3,), generator=g).to(torch.int32).to(device)
        out = SMP.decode_step(params, cfg, tok, n + step, cache)
        cache = out.kv_cache
        assert out.logits.isfinite().all()
        assert [a is cache.layers[i] for a, i in zip(appends, own)] == [True] * len(own)
        assert len(calls) == cfg.num_hidden_layers
        for i, (layer, table, lengths, window) in enumerate(calls):
            sliding = cfg.layer_types[i] == C.SLIDING
            assert layer is cache.layers[C.kv_source_layers(cfg)[i]]
            assert table is (cache.window_table if sliding else cache.page_table)
            assert lengths == (n + step + 1).tolist() and window == (cfg.sliding_window if sliding else 0)
    assert cache.length == S + steps


def test_model_prefill_quantises_what_the_dense_cache_holds(device):
    cfg = C.config_from_hf(CFG)
    params = _params(cfg, device)
    pads, S = [0, 11, 59], 60
    ids, mask = _prompts(cfg, pads, S, device)
    # a window as long as the prompt keeps every key in the dense ring
    cfg_all = cfg._replace(sliding_window=64)
    dense = SMP.prefill(params, cfg_all, ids, mask, max_new_tokens=4).kv_cache
    paged = SMP.prefill(params, cfg_all, ids, mask, max_new_tokens=4, paged=PagedSpec(32, e4m3=True)).kv_cache
    n = torch.tensor([S - p for p in pads], dtype=torch.int32, device=device)
    for i, (d, p) in enumerate(zip(dense.layers, paged.layers)):
        assert (d is None) == (p is None)
        if d is None:
            continue
        table = paged.window_table if cfg.layer_types[i] == C.SLIDING else paged.page_table
        got = kernels.paged_read(p, page_table=table, lengths=n, start=0, count=S)
        for x, ref in zip(got, d.reference_layout()):
            for b, pad in enumerate(pads):
                y = ref[b, pad:S].double()
                # the dense cache rounds to bf16 after the norm, the rotation's factors and the result: 4 half steps of
                # the larger of the two terms; then half a step of e4m3, or of the scale's smallest
                size = y.abs() + y.abs().roll(y.shape[-1] // 2, -1)
                bound = P.U_E4M3 * y.abs() + 2.0 ** -10 * y.abs().amax(-1, keepdim=True) / 224 + 5 * P.U_BF16 * size
                assert ((x[b, : S - pad].double() - y).abs() <= bound).all(), (i, b)
                assert (x[b, S - pad:] == 0).all()


@pytest.mark.parametrize("e4m3", [False, True])
def test_inactive_rows_store_nothing(device, e4m3):
    cfg = C.config_from_hf(CFG)
    params = _params(cfg, device)
    ids, mask = _prompts(cfg, [0, 3], 20, device)
    cache = SMP.prefill(params, cfg, ids, mask, max_new_tokens=8, paged=PagedSpec(32, e4m3)).kv_cache
    raw = lambda: [x.view(torch.uint8).clone() for l in cache.layers if l is not None for x in l if x is not None]  # noqa: E731
    before = raw()
    tok, pos = torch.tensor([5, 6], device=device), torch.tensor([20, 17], device=device)
    out = SMP.decode_step(params, cfg, tok, pos, cache, attention_mask=torch.zeros(2, dtype=torch.bool, device=device))
    assert all(torch.equal(a, b) for a, b in zip(before, raw()))
    assert out.logits.isfinite().all()
    SMP.decode_step(params, cfg, tok, pos, cache, attention_mask=torch.tensor([False, True], device=device))
    for layer, table in ((cache.layers[0], cache.window_table), (cache.layers[2], cache.page_table)):
        k, _ = kernels.paged_read(layer, page_table=table, lengths=torch.tensor([30, 30], dtype=torch.int32, device=device),
                                  start=16, count=5)
        assert (k[0, 4] == 0).all() and (k[1, 1] != 0).any() and (k[1, 2:] == 0).all()


@pytest.mark.parametrize("e4m3", [False, True])
def test_graphed_steps_equal_eager_ones(device, e4m3):
    """Two captured steps over caches of their own, replayed in turn with eager work between, against eager
    steps on third caches: the same logits, bit by bit."""

    cfg = C.config_from_hf(CFG)
    params = _params(cfg, device)
    prompts = [_prompts(cfg, pads, 45, device) for pads in ([0, 44, 7], [20, 0, 1])]
    steps = 12
    fresh = lambda i: SMP.prefill(params, cfg, *prompts[i], max_new_tokens=steps, paged=PagedSpec(32, e4m3)).kv_cache  # noqa: E731
    graphs, eager = [SMP.GraphedDecodeStep(params, cfg, fresh(i)) for i in range(2)], [fresh(i) for i in range(2)]
    g = torch.Generator().manual_seed(6)
    for step in range(steps):
        for i in range(2):
            tok = torch.randint(0, cfg.vocab_size, (3,), generator=g).to(torch.int32).to(device)
            pos = (prompts[i][1].sum(-1) + step).to(torch.int32)
            active = torch.tensor([True, step < 5, True], device=device)
            got = graphs[i].step(tok, pos, active).clone()
            out = SMP.decode_step(params, cfg, tok, pos, eager[i], attention_mask=active)
            eager[i] = out.kv_cache
            rows = active.cpu()
            assert torch.equal(got.cpu()[rows], out.logits[:, -1].float().cpu()[rows]), (step, i)
    again = [fresh(i) for i in range(2)]
    for i in range(2):  # a replayed step is deterministic
        runs = []
        for cache in (again[i], fresh(i)):
            gs = SMP.GraphedDecodeStep(params, cfg, cache)
            pos = prompts[i][1].sum(-1).to(torch.int32)
            outs = []
            for step in range(4):
                outs.append(gs.step(torch.full((3,), 9 + step, dtype=torch.int32, device=device), pos + step,
                                    torch.ones(3, dtype=torch.bool, device=device)).clone())
                torch.cuda.synchronize()
            runs.append(outs)
        assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_one_row_steps(device):
    """A single sequence: one token's rows have no stride to follow."""

    cfg = C.config_from_hf(CFG)
    params = _params(cfg, device)
    ids, mask = _prompts(cfg, [3], 20, device)
    out = SMP.prefill(params, cfg, ids, mask, max_new_tokens=6, paged=PagedSpec(32, True))
    step = SMP.GraphedDecodeStep(params, cfg, out.kv_cache)
    eager = SMP.prefill(params, cfg, ids, mask, max_new_tokens=6, paged=PagedSpec(32, True)).kv_cache
    for i in range(6):
        tok, pos = torch.tensor([7 + i], dtype=torch.int32, device=device), torch.tensor([17 + i], dtype=torch.int32, device=device)
        got = step.step(tok, pos, torch.ones(1, dtype=torch.bool, device=device)).clone()
        ref = SMP.decode_step(params, cfg, tok, pos, eager)
        eager = ref.kv_cache
        assert torch.equal(got, ref.logits[:, -1].float())


@pytest.mark.parametrize("e4m3", [False, True])
def test_captured_operators_replay_like_eager(device, e4m3):
    """Append, split attention (its workspace the graph's own) and read in one graph, replayed with new inputs and
    eager work between; two graphs in turn."""

    B, H, R, D, ps, M_ = 2, 1, 4, 128, 64, 80
    g = torch.Generator().manual_seed(8)
    table = torch.randperm(B * M_, generator=g).view(B, M_).to(torch.int32).to(device)

    def fresh():
        layer = new_paged_layer(B * M_, H, D, ps, e4m3=e4m3, device=device)
        x = torch.randn((B, 5000, 2 * H * D), generator=torch.Generator().manual_seed(9)).to(BF16).to(device)
        kernels.paged_append(layer, x[..., : H * D].view(B, 5000, H, D), x[..., H * D:].view(B, 5000, H, D), page_table=table,
                             write_pos=torch.tensor([0, -1234], dtype=torch.int32, device=device))
        return layer

    def run(layer, s):
        kernels.paged_append(layer, s["k"], s["v"], page_table=table, write_pos=s["pos"])
        out = kernels.paged_decode_attention(layer, s["q"], page_table=table, lengths=s["len"])
        return [out, *kernels.paged_read(layer, page_table=table, lengths=s["len"], start=4990, count=12)]

    def inputs(i):
        gg = torch.Generator().manual_seed(100 + i)
        r = lambda *s: (torch.randn(s, generator=gg)).to(BF16).to(device)  # noqa: E731
        pos = [5000 + i, 3766 + i] if i % 3 else [17, -1]
        return dict(k=r(B, 1, H, D), v=r(B, 1, H, D), q=0.2 * r(B, H, R, D),
                    pos=torch.tensor(pos, dtype=torch.int32, device=device),
                    len=torch.tensor([p + 1 for p in pos], dtype=torch.int32, device=device))

    static = [inputs(0), inputs(0)]
    layers, ref = [fresh(), fresh()], fresh()
    graphs, results = [], []
    for i in range(2):
        run(layers[i], static[i])
        torch.cuda.synchronize()
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
            results.append(run(layers[i], static[i]))
        torch.cuda.current_stream().wait_stream(side)
        graphs.append(graph)
    run(ref, inputs(0))
    for i in range(1, 9):
        new = inputs(i)
        want = run(ref, new)
        for j in range(2):
            for name, t in new.items():
                static[j][name].copy_(t)
            graphs[j].replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(results[j], want)), (i, j)


def test_calls_on_two_streams(device):
    """Split calls on two streams at once, each with its own workspace, equal the same calls in turn."""

    H, R, D, ps = 1, 8, 256, 64
    cases = []
    for i in range(2):
        n = [9000 + 100 * i, 30]
        M_ = (max(n) + ps - 1) // ps
        layer = new_paged_layer(2 * M_, H, D, ps, e4m3=True, device=device)
        x = torch.randn((2, max(n), 2 * H * D), generator=torch.Generator().manual_seed(i)).to(BF16).to(device)
        table = torch.arange(2 * M_, dtype=torch.int32, device=device).view(2, M_)
        kernels.paged_append(layer, x[..., : H * D].view(2, -1, H, D), x[..., H * D:].view(2, -1, H, D), page_table=table,
                             write_pos=torch.zeros(2, dtype=torch.int32, device=device))
        q = (0.1 * torch.randn((2, H, R, D), generator=torch.Generator().manual_seed(10 + i))).to(BF16).to(device)
        cases.append((layer, q, table, torch.tensor(n, dtype=torch.int32, device=device)))
    call = lambda c: kernels.paged_decode_attention(c[0], c[1], page_table=c[2], lengths=c[3])  # noqa: E731
    want = [call(c).clone() for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for _ in range(10):
        for st, c, o in zip(streams, cases, outs):
            with torch.cuda.stream(st):
                o.append(call(c))
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for got, w in zip(outs, want) for o in got)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("top_k,temperature", [(0, 0.0), (0, 1.0), (8, 0.7)])
def test_generate_in_pages(device, e4m3, top_k, temperature):
    """A rollout in pages: rows stop at their EOS, the same key draws the same tokens, and the draws and
    log-probabilities are those of the steps' logits when the drawn tokens are fed to a step that returns them."""

    cfg = C.config_from_hf(CFG)
    params = _params(cfg, device)
    ids, mask = _prompts(cfg, [0, 30, 13, 5], 32, device)
    N = 24
    sc = SMP.SamplerConfig(max_prompt_len=32, max_new_tokens=N, temperature=temperature, top_k=top_k, seed=3,
                           eos_ids=tuple(range(0, 512, 64)))
    roll = SMP.NativeRollout(params, cfg, sc, paged=PagedSpec(32, e4m3))
    got, again = roll.generate(ids, mask), roll.generate(ids, mask)
    assert torch.equal(got.completion_ids, again.completion_ids) and torch.equal(got.rollout_logps, again.rollout_logps)
    done = torch.zeros(4, dtype=torch.bool, device=device)
    for t in range(N):
        assert torch.equal(got.completion_mask[:, t], ~done)
        done |= (got.completion_ids[:, t] % 64 == 0) & ~done
    assert (got.rollout_logps[~got.completion_mask] == 0).all()
    out = SMP.prefill(params, cfg, ids, mask, max_new_tokens=N, paged=PagedSpec(32, e4m3))
    step = SMP.GraphedDecodeStep(params, cfg, out.kv_cache)
    logits, n = out.logits[:, -1].float(), mask.sum(-1).to(torch.int32)
    for t in range(N):
        on = got.completion_mask[:, t]
        tok = got.completion_ids[:, t]
        logp = torch.log_softmax(logits.double(), dim=-1).gather(-1, tok[:, None].long())[:, 0]
        # f32 log-softmax of 512 soft-capped logits (|x| <= 30): each exp's argument is off by 60 u and its result by 2 u,
        # their sum by 512 u more, the logarithm and two differences by less than 40 u: 614 u
        assert ((logp - got.rollout_logps[:, t].double()).abs()[on] <= 614 * P.U32).all(), t
        if temperature <= 0:
            assert torch.equal(logits.argmax(-1)[on].int(), tok[on].int())
        if top_k:
            least = logits.topk(top_k, dim=-1).values[:, -1]
            assert (logits.gather(-1, tok[:, None].long())[:, 0] >= least)[on].all()
        logits = step.step(tok, n + t, on).clone()


def test_paged_model_refusals(device):
    cfg = C.config_from_hf(CFG)
    params = _params(cfg, device)
    ids, mask = _prompts(cfg, [0, 3], 20, device)
    holes = mask.clone()
    holes[0, 5] = False
    with pytest.raises(ValueError, match="left-padded"):
        SMP.prefill(params, cfg, ids, holes, max_new_tokens=2, paged=PagedSpec())
    with pytest.raises(ValueError, match="cache_dtype"):
        SMP.prefill(params, cfg, ids, mask, max_new_tokens=2, paged=PagedSpec(), cache_dtype=BF16)
    with pytest.raises(ValueError, match="page_size"):
        SMP.prefill(params, cfg, ids, mask, max_new_tokens=2, paged=PagedSpec(48))
    cache = SMP.prefill(params, cfg, ids, mask, max_new_tokens=2, paged=PagedSpec()).kv_cache
    with pytest.raises(ValueError, match="empty cache"):
        M.forward_gemma4_text(params, ids, ids, config=cfg, attention_mask=mask, kv_cache=cache, cache_mode="prefill")
    with pytest.raises(ValueError, match="do not fit"):
        M.forward_gemma4_text(params, torch.cat([ids] * 4, 1), torch.cat([ids] * 4, 1), config=cfg,
                              kv_cache=init_paged_kv_cache(cfg, 2, 20, PagedSpec(), device))
    f32 = params._replace(embed_tokens=params.embed_tokens.float())
    with pytest.raises(ValueError, match="bfloat16 model"):
        M.forward_gemma4_text(f32, ids, ids, config=cfg, attention_mask=mask,
                              kv_cache=init_paged_kv_cache(cfg, 2, 20, PagedSpec(), device))


@pytest.mark.parametrize("B", [1, 3])
def test_a_step_leaves_the_callers_mask(device, B):
    """A step without host-side values whose mask is a column of a wider tensor: that tensor stays, and the result
    is that of a mask of its own."""

    cfg = C.config_from_hf(CFG)
    params = _params(cfg, device)
    ids, mask = _prompts(cfg, [3, 0, 9][:B], 20, device)
    tok = torch.tensor([5, 6, 7][:B], dtype=torch.int32, device=device)[:, None]
    pos = mask.sum(-1, keepdim=True).to(torch.int32)
    wide = torch.zeros((B + 1, 64), dtype=torch.bool, device=device)  # a row behind the last
    wide[:B, 40] = torch.tensor([True, False, True][:B], device=device)
    before = wide.clone()
    outs = []
    for m in (wide[:B, 40:41], wide[:B, 40:41].clone(memory_format=torch.contiguous_format)):
        cache = SMP.prefill(params, cfg, ids, mask, max_new_tokens=4, paged=PagedSpec(32)).kv_cache
        outs.append(M.forward_gemma4_lm(params, tok, pos, config=cfg, attention_mask=m, kv_cache=cache, cache_mode="append",
                                      write_pos=pos[:, 0].clone()).logits)
        assert torch.equal(wide, before)
    assert torch.equal(*outs)
