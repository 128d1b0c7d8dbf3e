"""A model's decode step over pages, layer by layer, against the model's definition in 64 bits: the projections of
the layer's input, q / k / v with the layer's own norms and its type's rotation, and the attention over the pages."""

from __future__ import annotations

import math

import pytest
import torch

import paged_util as P
from gemma4_posttrain_jax_amd import config as C
from gemma4_posttrain_jax_amd import kernels
from gemma4_posttrain_jax_amd import model as M
from gemma4_posttrain_jax_amd import sampler as SMP
from gemma4_posttrain_jax_amd.kvcache import PagedSpec
from oracle import g4_oracle as O
from test_gpu_paged_run import CFG, CFG512, _params, _prompts

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _rotation(inv_freq, positions):
    """cos, sin and their errors ``[B, D]``: f32 frequencies off by 4 u (a power and a division), their product with the
    position by one more, and the functions by 4 u."""

    angle = positions.double()[:, None] * torch.from_numpy(inv_freq).double()[None]
    angle = torch.cat([angle, angle], dim=-1)
    return angle.cos(), angle.sin(), 4 * P.U32 + 5 * P.U32 * angle


def _turned(x, weight, rotation, eps):
    """``x [B, ..., D]`` normed by ``weight`` (None: not) and turned (None: not), the f32 error before a rounding, and
    the size of the rotation's terms."""

    rope, off = None, 0.0
    if rotation is not None:
        shape = (x.shape[0],) + (1,) * (x.dim() - 2) + (x.shape[-1],)
        rope, off = [t.view(shape) for t in rotation[:2]], rotation[2].view(shape)
    want, err = P.prepared(x, weight, weight is not None, rope, eps)
    flat = P.prepared(x, weight, weight is not None, None, eps)[0].abs()
    pair = flat + flat.roll(flat.shape[-1] // 2, -1)
    terms = flat if rope is None else flat * rope[0].abs() + flat.roll(flat.shape[-1] // 2, -1) * rope[1].abs()
    return want, err + off * pair, terms


def _off(got, want, bound):
    return ((got.cpu().double() - want).abs() / bound.clamp(min=1e-30)).max().item()


@pytest.mark.parametrize("kwargs", [CFG, CFG512])
def test_every_layer_of_a_step(device, kwargs, monkeypatch):
    cfg, ocfg = C.config_from_hf(kwargs), O.config_from_hf(kwargs)
    params = _params(cfg, device)
    pads, S, steps = [0, 11, 59], 60, 4
    ids, mask = _prompts(cfg, pads, S, device)
    cache = SMP.prefill(params, cfg, ids, mask, max_new_tokens=steps, paged=PagedSpec(32)).kv_cache
    raw, ready, attended = [], [], []
    append, prepare, attend = kernels.paged_append, kernels.prepare_q, kernels.paged_decode_attention

    def record_append(layer, k, v, *, q, q_out, **kw):
        append(layer, k, v, q=q, q_out=q_out, **kw)
        raw.append([t[:, 0].cpu() for t in (q, k, v)])
        ready.append(q_out[:, 0].cpu())

    def record_prepare(q, q_out, **kw):
        prepare(q, q_out, **kw)
        raw.append([q[:, 0].cpu(), None, None])
        ready.append(q_out[:, 0].cpu())

    def record_attend(layer, q, **kw):
        attended.append(attend(layer, q, **kw))
        return attended[-1]

    monkeypatch.setattr(kernels, "paged_append", record_append)
    monkeypatch.setattr(kernels, "prepare_q", record_prepare)
    monkeypatch.setattr(kernels, "paged_decode_attention", record_attend)
    inv, eps = O.rope_inv_freq(ocfg), cfg.rms_norm_eps
    n = mask.sum(-1).cpu()
    g = torch.Generator().manual_seed(5)
    caught = set()
    for step in range(steps):
        tok = torch.randint(0, cfg.vocab_size, (3, 1), generator=g).to(torch.int32)
        for seen in (raw, ready, attended):
            seen.clear()
        outs = []
        _, cache = M.forward_gemma4_text(params, tok.to(device), (n + step)[:, None].int().to(device), config=cfg,
                                         kv_cache=cache, cache_mode="append", layer_outputs=outs)
        assert len(raw) == len(ready) == len(attended) == len(outs) == cfg.num_hidden_layers
        embedded = (params.embed_tokens.cpu()[tok[:, 0].long()].float() * torch.tensor(math.sqrt(cfg.hidden_size)).to(BF16).float())
        inputs = [embedded.to(BF16)] + [x[:, 0].cpu() for x in outs[:-1]]
        for i, lp in enumerate(params.layers):
            at, shared = lp.attention, C.is_kv_shared(cfg, i)
            kind = cfg.layer_types[i]
            sliding = kind == C.SLIDING
            # the projections: a half step of the normed input, f32 sums, and a half step of the result
            h, h_err = P.prepared(inputs[i], lp.input_norm.weight.cpu(), True, None, eps)
            h_err = P.U_BF16 * h.abs() + (1 + P.U_BF16) * h_err
            for x, w in zip(raw[i], (at.q_proj, at.k_proj, at.v_proj)):
                if x is None:
                    continue
                w = w.cpu().double()
                w = w.transpose(1, 2) if w.dim() == 4 else w  # [M, H, R, D] or [M, H, D]
                want = torch.tensordot(h, w, 1)
                err = torch.tensordot(h_err + (cfg.hidden_size + 2) * P.U32 * (h.abs() + h_err), w.abs(), 1)
                assert _off(x, want, P.U_BF16 * want.abs() + (1 + P.U_BF16) * err) <= 1, (step, i)
            # q: rounded once, but by a kv-shared layer after the norm, in its factors and in the sum: 4 half steps of the terms
            rotation = _rotation(inv[O.SLIDING if sliding else O.FULL], n + step)
            steps_off = 4 if shared else 1

            def q_off(weight, rotation):
                want, err, terms = _turned(raw[i][0], weight, rotation, eps)
                # (1 + u)^4 - 1 <= 4.02 u
                bound = P.U_BF16 * want.abs() + (steps_off - 1) * 1.02 * P.U_BF16 * terms + (1 + 4 * P.U_BF16) * err
                return _off(ready[i], want, bound)

            weight = at.q_norm.weight.cpu()
            assert q_off(weight, rotation) <= 1, (step, i)
            # what the bound would not let pass
            other = _rotation(inv[O.FULL if sliding else O.SLIDING], n + step)
            for name, wrong in (("no norm", (None, rotation)), ("no rotation", (weight, None)),
                                ("a plain norm", (torch.ones_like(weight), rotation)),
                                ("the next position", (weight, _rotation(inv[O.SLIDING if sliding else O.FULL], n + step + 1))),
                                ("the other type's", (weight, other) if other[0].shape == rotation[0].shape else (weight, None))):
                if q_off(*wrong) > 1:
                    caught.add((i, name))
            # k / v in their places, the attention over them
            src = C.kv_source_layers(cfg)[i]
            table = (cache.window_table if sliding else cache.page_table).cpu()
            pages = P.slots_of(cache.layers[src])
            if not shared:
                for got, x, w, rope in zip(pages, raw[i][1:], (at.k_norm.weight.cpu(), torch.ones_like(weight)), (rotation, None)):
                    want, err, _ = _turned(x, w, rope, eps)
                    for b, place in enumerate((n + step).tolist()):
                        at_place = got[int(table[b, place // 32]), :, place % 32]
                        assert _off(at_place, want[b], P.U_BF16 * want[b].abs() + (1 + P.U_BF16) * err[b]) <= 1, (step, i, b)
            want, bound = P.attention(*pages, table, (n + step + 1).tolist(), ready[i], cfg.sliding_window if sliding else 0)
            assert _off(attended[i], want, bound) <= 1, (step, i)
    names = {"no norm", "no rotation", "a plain norm", "the next position", "the other type's"}
    assert caught == {(i, name) for i in range(cfg.num_hidden_layers) for name in names}
