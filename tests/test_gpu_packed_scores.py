"""Packed attention of scores far from zero, on the GPU against 64 bits."""

from __future__ import annotations

import math

import pytest
import torch

from gemma4_posttrain_jax_amd import kernels
from gemma4_posttrain_jax_amd.kvcache import new_layer_cache

pytestmark = pytest.mark.gpu

U32, U_BF16 = 2.0 ** -24, torch.finfo(torch.bfloat16).eps / 2
FORMS = {"pieces": ([3000], 1, 2), "small": ([500, 300, 700], 2, 4), "large": ([3000], 3, 8)}  # sequences, kv heads, rows per head


def _inputs(form, D, level, seed, device):
    """Scores level + x_j that f32 sums exactly in any order: q . k_j = a b + 1 x_j, x a few steps of f32 at the level."""

    lens, H, R = FORMS[form]
    T = sum(lens)
    g = torch.Generator().manual_seed(seed)
    step = max(0.125, 2.0 ** (math.floor(math.log2(abs(level))) - 23) if level else 0.0)
    x = (torch.randint(-8, 9, (T, H), generator=g) * step).double()
    root = 2.0 ** (math.floor(math.log2(abs(level))) // 2) if level else 1.0
    q, k = torch.zeros(T, H, R, D), torch.zeros(T, H, D)
    q[..., 3], k[..., 3] = root, level / root
    q[..., D - 5], k[..., D - 5] = 1.0, x.float()
    v = torch.randn(T, H, D, generator=g).to(torch.bfloat16)
    assert torch.equal(k.to(torch.bfloat16).float(), k) and torch.equal(q.to(torch.bfloat16).float(), q)
    chunk = new_layer_cache(1, H, D, T, False, torch.bfloat16, device)
    kernels.kv_append(chunk, k.to(torch.bfloat16).to(device)[None], v.to(device)[None], write_pos=0)
    cu = torch.tensor([0, *lens], dtype=torch.int32, device=device).cumsum(0, dtype=torch.int32)
    return lens, x, v, q.to(torch.bfloat16).to(device), chunk, kernels.packed_starts(cu, T)


def _check(got, lens, x, v, level, window, skip=()):
    a = 0
    for b, n in enumerate(lens):
        i = torch.arange(n)
        hidden = i[None, :] > i[:, None]
        if window:
            hidden |= i[None, :] <= i[:, None] - window
        for h in range(0 if b in skip else x.shape[1]):
            s = x[a:a + n, h][None, :].expand(n, n).masked_fill(hidden, -math.inf)
            w = torch.softmax(s, dim=-1)
            vh = v[a:a + n, h].double()
            want, mass = w @ vh, w @ vh.abs()
            # the scores are exact. Exponents (s - m) log2(e) are within 2 u of themselves, of 24 where weights count; below a maximum
            # of 1024 they are formed with m log2(e), off by u 1024 log2(e), which may differ from one maximum to the next;
            # exp2 2 u, sums (n + 16) u, each for the numerator and the denominator; weights and result once to bf16
            rel = 2 * (2 * 24 + 2 + min(abs(level), 1024.0) * 1.45 + n + 16) * U32
            bound = (U_BF16 + rel) * mass * (1 + U_BF16) + U_BF16 * want.abs() + 1e-30
            err = (got[a:a + n, h, 0] - want).abs()
            assert bool((err <= bound).all()), (b, h, float((err - bound).max()))
        a += n


@pytest.mark.parametrize("level", [0.0, 2.0 ** 9, 3 * 2.0 ** 12, -2.0 ** 16, 2.0 ** 20, -5 * 2.0 ** 20, 2.0 ** 26, -2.0 ** 33, 2.0 ** 33,
                                   5 * 2.0 ** 40])
@pytest.mark.parametrize("D", [64, 256, 512])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("window", [0, 200])
def test_scores_around_a_level(level, D, form, window, device):
    lens, x, v, q, chunk, starts = _inputs(form, D, level, D + 1, device)
    got = kernels.packed_prefill_attention(q, chunk.key, chunk.value_t, starts, window=window, longest=max(lens)).cpu().double()
    assert torch.equal(got, got[:, :, :1].expand_as(got))  # equal rows of a head
    _check(got, lens, x, v, level, window)


@pytest.mark.parametrize("level", [0.0, 2.0 ** 20, -2.0 ** 33])
@pytest.mark.parametrize("D", [64, 256, 512])
def test_scores_around_a_level_beside_no_numbers(level, D, device):
    """A sequence between two others whose keys and values are no numbers: rows of both share workgroups."""

    lens, x, v, q, chunk, starts = _inputs("small", D, level, D + 2, device)
    a, b = lens[0], lens[0] + lens[1]
    keys, values = (t[0].clone() for t in chunk.reference_layout())
    keys[a:b:2], values[a:b:3], values[a + 1:b:3] = math.nan, math.nan, math.inf
    other = new_layer_cache(1, x.shape[1], D, sum(lens), False, torch.bfloat16, device)
    kernels.kv_append(other, keys[None].contiguous(), values[None].contiguous(), write_pos=0)
    got = kernels.packed_prefill_attention(q, other.key, other.value_t, starts, longest=max(lens)).cpu().double()
    _check(got, lens, x, v, level, 0, skip=(1,))
    assert not bool(got[a:b].isfinite().any())


def test_levels_that_rise_and_fall(device):
    """Each stretch of 100 keys at another level, up and down by more than f32 holds beside them: rows see the highest so far."""

    D, n = 128, 1000
    levels = [0.0, -2.0 ** 30, 2.0 ** 12, 2.0 ** 11, 2.0 ** 20, 2.0 ** 20 + 2048, 0.0, 2.0 ** 34, -2.0 ** 34, 2.0 ** 34]
    g = torch.Generator().manual_seed(5)
    s = torch.tensor(levels).repeat_interleave(100).double()
    q, k = torch.zeros(n, 1, 2, D), torch.zeros(n, 1, D)
    q[..., 0], q[..., 1] = 2.0 ** 17, 2.0 ** 11
    first = (s / 2.0 ** 17).to(torch.bfloat16).double()
    k[:, 0, 0], k[:, 0, 1] = first.float(), ((s - first * 2.0 ** 17) / 2.0 ** 11).float()
    assert torch.equal(k.to(torch.bfloat16).float(), k)
    v = torch.randn(n, 1, D, generator=g).to(torch.bfloat16)
    chunk = new_layer_cache(1, 1, D, n, False, torch.bfloat16, device)
    kernels.kv_append(chunk, k.to(torch.bfloat16).to(device)[None], v.to(device)[None], write_pos=0)
    starts = torch.zeros(n, dtype=torch.int32, device=device)
    for longest in (100, n):  # whole, in pieces
        got = kernels.packed_prefill_attention(q.to(torch.bfloat16).to(device), chunk.key, chunk.value_t, starts,
                                               longest=longest).cpu().double()
        _check(got, [n], s[:, None], v, 1024.0, 0)
