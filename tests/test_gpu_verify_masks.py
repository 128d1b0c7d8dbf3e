"""Verification of drafted tokens over logits that are masked with finite values or lie far from zero, on the GPU against 64
bits."""

from __future__ import annotations

import math

import pytest
import torch

from gemma4_posttrain_jax_amd import kernels
from test_gpu_verify import _inputs

pytestmark = pytest.mark.gpu

LOWEST = torch.finfo(torch.float32).min


def decided(logits, drafts, uniforms, noise, temperature, draft_logits=None):
    """The operator in 64 bits, row by row, also where p - q leaves no weight: the token is then drawn from p."""

    B, K1, V = logits.shape
    tokens, counts = torch.full((B, K1), -1, dtype=torch.int32), []
    logp = torch.zeros((B, K1), dtype=torch.float64)
    first = lambda hit: int(torch.nonzero(hit)[0, 0])  # noqa: E731
    for b in range(B):
        x, i = logits[b].double(), 0
        policy = torch.log_softmax(x, dim=-1)
        if temperature <= 0:
            while i < K1 - 1 and int(drafts[b, i]) == first(x[i] == x[i].max()):
                i += 1
            token = first(x[i] == x[i].max())
        else:
            p = torch.softmax(x / temperature, dim=-1)
            q = None if draft_logits is None else torch.softmax(draft_logits[b].double() / temperature, dim=-1)
            while i < K1 - 1:
                d = int(drafts[b, i])
                if not float(uniforms[b, i]) * (1.0 if q is None else float(q[i, d])) < float(p[i, d]):
                    break
                i += 1
            w = p[i].clone()
            if i < K1 - 1 and q is None:
                w[int(drafts[b, i])] = 0.0
            elif i < K1 - 1:
                w = torch.clamp(w - q[i], min=0.0)
            pace = torch.where(noise[b] > 0, 1 / -torch.log(noise[b].double()), torch.zeros(()).double())
            race = (w if bool((w * pace > 0).any()) else p[i]) * pace
            token = first(race == race.max())
        tokens[b, :i], tokens[b, i] = drafts[b, :i], token
        for s in range(i + 1):
            logp[b, s] = policy[s, int(tokens[b, s])]
        counts.append(i)
    return tokens, torch.tensor(counts, dtype=torch.int32), logp


def _check(device, logits, drafts, u, noise, temperature, q=None):
    put = lambda t: None if t is None else t.to(device)  # noqa: E731
    got = [t.cpu() for t in kernels.verify_draft(put(logits), put(drafts), put(u), put(noise), temperature=temperature,
                                                 draft_logits=put(q))]
    wt, wc, wl = decided(logits, drafts, u, noise, temperature, q)
    assert torch.equal(got[1], wc), (got[1].tolist(), wc.tolist())
    assert torch.equal(got[0], wt), (got[0].tolist(), wt.tolist())
    # a log-probability is x - max less the logarithm of a sum: one rounding of each, of their difference and of the result,
    # and of the sum (at most 100 levels), whose exponentials are within 4 u and the rounding of their argument, u |x - max| with a
    # weighted mean below 16; a masked column has weight 0
    assert torch.equal(got[2].isfinite(), wl.isfinite())
    there = wl.isfinite()
    bound = 2.0 ** -24 * (2 * wl.abs() + 140)
    assert bool(((got[2].double() - wl).abs() <= bound)[there].all())
    return wc


@pytest.mark.parametrize("low", [-1e4, -65504.0, -1e9, -1e10, -1e20, LOWEST, -math.inf])
@pytest.mark.parametrize("temperature", [0.0, 1e-6, 1e-5, 0.7, 1.0])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("draft", [False, True])
def test_masked_stretches(low, temperature, dtype, draft, device):
    """Thousands of masked columns in a row, so that threads see nothing else; of the last row all but a few columns."""

    B, K, V = 4, 2, 12001
    logits, drafts, u, noise, q = _inputs(B, K, V, dtype, 61, True)
    low = max(low, float(torch.finfo(dtype).min)) if math.isfinite(low) else low
    logits[:, :, 2000:9000] = low
    logits[3, :, 30:] = low
    q[1:3, :, 3000:11000] = low
    q[3, :, 10:] = low
    if temperature < 0.1:  # what a drafter says at such temperatures
        drafts = q.float().argmax(dim=-1).to(torch.int32)
    _check(device, logits, drafts, u, noise, temperature, q if draft else None)


@pytest.mark.parametrize("level", [3e4, -1e6, 1e7, -1e10, 1e10, -1e20, 1e20])
@pytest.mark.parametrize("temperature", [0.0, 1e-6, 1e-3, 0.7, 1.0])
@pytest.mark.parametrize("draft", [False, True])
def test_rows_far_from_zero(level, temperature, draft, device):
    """All logits around a level, whose quotient by the temperature has no place for the differences in f32."""

    B, K, V = 5, 2, 9001
    logits, drafts, u, noise, q = _inputs(B, K, V, torch.float32, 62, True)
    logits, q = logits + level, q + level
    if temperature < 0.1:
        drafts = q.argmax(dim=-1).to(torch.int32)
    _check(device, logits, drafts, u, noise, temperature, q if draft else None)


@pytest.mark.parametrize("level", [0.0, -1e10, 1e20])
@pytest.mark.parametrize("temperature", [0.5, 1.0])
def test_the_residual_of_level_rows(level, temperature, device):
    """p is 1 / V everywhere, q twice that on the first half: a draft is accepted by u < 1/2, else the token is one of the other half;
    a looked-up draft has p = 1 / V, and the token is another."""

    B, K, V = 6, 1, 8192
    noise = torch.rand(B, V, generator=torch.Generator().manual_seed(63))
    logits = torch.full((B, K + 1, V), level)
    q = torch.full((B, K, V), level)
    q[:, :, V // 2:] = LOWEST
    u = torch.tensor([0.1, 0.3, 0.49, 0.51, 0.75, 0.99])[:, None]
    drafts = noise[:, :V // 2].argmax(dim=-1, keepdim=True).to(torch.int32)
    assert _check(device, logits, drafts, u, noise, temperature, q).tolist() == [1, 1, 1, 0, 0, 0]
    drafts = noise.argmax(dim=-1, keepdim=True).to(torch.int32)
    assert _check(device, logits, drafts, u, noise, temperature).tolist() == [0] * B


@pytest.mark.parametrize("temperature", [0.0, 1.0])
@pytest.mark.parametrize("low", [-1e10, -65504.0 * 64])
def test_many_masked_logits(low, temperature, device):
    """As many as are taken in two steps per thread, whole stretches of a workgroup masked."""

    B, K, V = 8, 1, (1 << 21) + 1
    assert B * (K + 1) * V >= 1 << 25
    g = torch.Generator().manual_seed(64)
    logits = (torch.randn(B, K + 1, V, generator=g) * 2).to(torch.bfloat16)
    logits[:, :, :500000] = low
    logits[::2, :, 900000:2000000] = low
    drafts = logits[:, :K].float().argmax(dim=-1).to(torch.int32)
    drafts[1::3] -= 1
    _check(device, logits, drafts, torch.rand(B, K, generator=g) * 1e-5, torch.rand(B, V, generator=g), temperature)
