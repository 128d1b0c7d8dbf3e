"""Attention of packed prompts on the GPU against 64 bits: sequences of every length about the tiles' edges, windows,
groups, tokens of no sequence, and values that a row must not see."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from gemma4_posttrain_jax_amd import _lib, kernels
from gemma4_posttrain_jax_amd.kvcache import group_keys, group_values, key_shape, slot_stride_for
from packed_util import packed_reference

pytestmark = pytest.mark.gpu


def _inputs(lens, tail, H, R, D, seed, device, scale=2.0):
    g = torch.Generator().manual_seed(seed)
    T = sum(lens) + tail
    q = (torch.randn(T, H, R, D, generator=g) * scale / math.sqrt(D)).to(torch.bfloat16)
    k = torch.randn(T, H, D, generator=g).to(torch.bfloat16)
    v = torch.randn(T, H, D, generator=g).to(torch.bfloat16)
    return q, k, v


def _laid_out(k, v, device, fill=0.0):
    T, H, D = k.shape
    Sp = slot_stride_for(T)
    kk = torch.full((1, H, Sp, D), fill, dtype=torch.bfloat16)
    vv = torch.full((1, H, Sp, D), fill, dtype=torch.bfloat16)
    kk[0, :, :T], vv[0, :, :T] = k.transpose(0, 1), v.transpose(0, 1)
    return group_keys(kk).to(device), group_values(vv).to(device)


def _run(q, k, v, lens, window, device, fill=0.0, **kw):
    cu = torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32, device=device)
    starts = kernels.packed_starts(cu, q.shape[0])
    kk, vv = _laid_out(k, v, device, fill)
    return kernels.packed_prefill_attention(q.to(device), kk, vv, starts, window=window, **kw)


def _check(got, q, k, v, lens, window):
    want, bound = packed_reference(q, k, v, lens, window)
    err = (got.cpu().double() - want).abs()
    assert bool((err <= bound).all()), f"off by {float((err - bound).max())} at {int((err - bound).argmax())}"


@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("lens,tail", [([1], 0), ([33, 0, 1, 65, 2], 3), ([130, 31, 32, 97], 0)])
def test_lengths_and_windows(D, window, lens, tail, device):
    q, k, v = _inputs(lens, tail, 2, 4, D, 1, device)
    _check(_run(q, k, v, lens, window, device), q, k, v, lens, window)


@pytest.mark.parametrize("R", [1, 2, 3, 5, 8, 16, 17])
def test_groups(R, device):
    lens = [70, 3, 41]
    q, k, v = _inputs(lens, 0, 1, R, 128, 2, device)
    _check(_run(q, k, v, lens, 0, device), q, k, v, lens, 0)


@pytest.mark.parametrize("D,window", [(256, 0), (256, 512), (128, 0), (512, 0), (64, 100)])
def test_long_prompts(D, window, device):
    lens = [1, 1500, 700]
    q, k, v = _inputs(lens, 11, 1, 2, D, 3, device)
    _check(_run(q, k, v, lens, window, device), q, k, v, lens, window)


@pytest.mark.parametrize("D", [64, 256, 512])
def test_many_short_prompts(D, device):
    g = torch.Generator().manual_seed(4)
    lens = torch.randint(0, 9, (300,), generator=g).tolist()
    q, k, v = _inputs(lens, 0, 2, 4, D, 5, device)
    _check(_run(q, k, v, lens, 0, device), q, k, v, lens, 0)


@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_what_a_row_does_not_see_does_not_reach_it(D, device):
    """NaN and infinities behind the last token, in another prompt, before the window and behind a token."""

    lens, window, tail = [37, 90, 50], 32, 4
    q, k, v = _inputs(lens, tail, 2, 4, D, 6, device)
    clean_k, clean_v = k.clone(), v.clone()
    for t, x in ((5, math.nan), (60, math.inf), (100, -math.inf), (36, math.nan), (178, math.nan)):
        v[t, :, ::3] = x
        k[t, :, ::5] = x if t != 60 else math.nan
    got = _run(q, k, v, lens, window, device, fill=math.nan).cpu()
    want, bound = packed_reference(q, clean_k, clean_v, lens, window)
    start = 0
    for n in lens:
        for t in range(start, start + n):
            seen = range(max(start, t - window + 1), t + 1)
            if not any(j in seen for j in (5, 60, 100, 36, 178)):
                assert bool(((got[t].double() - want[t]).abs() <= bound[t]).all()), t
            elif 5 in seen or 36 in seen:
                assert bool(got[t].isnan().all()), t  # the scores are NaN
        start += n
    assert bool((got[start:] == 0).all())


@pytest.mark.parametrize("D", [64, 256, 512])
def test_a_seen_infinity_and_its_neighbours(D, device):
    """An infinite value reaches the rows that see it, in its dims, and no other."""

    lens = [45, 45]
    q, k, v = _inputs(lens, 0, 1, 2, D, 7, device)
    v[20, 0, 3] = math.inf
    got = _run(q, k, v, lens, 0, device).cpu().double()
    v[20, 0, 3] = 0.0
    want, bound = packed_reference(q, k, v, lens, 0)
    hit = torch.zeros_like(want, dtype=torch.bool)
    hit[20:45, :, :, 3] = True
    assert bool((got[hit] == math.inf).all())
    assert bool(((got - want).abs() <= bound)[~hit].all())


def test_scores_far_apart(device):
    """Maxima that rise along a row by more than the slack, and scores beyond e^88 of each other."""

    lens = [300]
    q, k, v = _inputs(lens, 0, 1, 4, 128, 8, device, scale=40.0)
    k = (k.float() * torch.linspace(0.1, 3.0, 300)[:, None, None]).to(torch.bfloat16)
    _check(_run(q, k, v, lens, 0, device), q, k, v, lens, 0)


def test_the_same_call_gives_the_same_bits_and_takes_an_out(device):
    lens = [100, 200, 3]
    q, k, v = _inputs(lens, 0, 2, 4, 256, 9, device)
    first = _run(q, k, v, lens, 0, device)
    out = torch.full_like(first, math.nan)
    assert _run(q, k, v, lens, 0, device, out=out) is out
    assert torch.equal(out.view(torch.int16), first.view(torch.int16))


@pytest.mark.parametrize("bounds,tokens,want", [
    ([0, 3, 3, 5], 7, [0, 0, 0, 3, 3, -1, -1]),
    ([0, 0, 0], 2, [-1, -1]),
    ([0, 4], 2, [0, 0]),
    ([2, 4], 5, [-1, -1, 2, 2, -1]),
])
def test_starts(bounds, tokens, want, device):
    cu = torch.tensor(bounds, dtype=torch.int32, device=device)
    assert kernels.packed_starts(cu, tokens).tolist() == want


def test_starts_that_are_none(device):
    """A start behind its token or below 0 is no sequence: zeros, whatever the other rows are."""

    q, k, v = _inputs([64], 0, 1, 1, 128, 10, device)
    starts = torch.zeros(64, dtype=torch.int32, device=device)
    starts[10], starts[20], starts[63] = 11, -2 ** 31, 2 ** 31 - 1
    kk, vv = _laid_out(k, v, device)
    got = kernels.packed_prefill_attention(q.to(device), kk, vv, starts).cpu().double()
    want, bound = packed_reference(q, k, v, [64], 0)
    none = torch.zeros(64, dtype=torch.bool)
    none[[10, 20, 63]] = True
    assert bool((got[none] == 0).all())
    assert bool(((got - want).abs() <= bound)[~none].all())


# --- few rows with many keys: pieces of the keys, joined --------------------------------------------------------------


def _pieces(q, window=0, longest=0):
    T, H, R, D = q.shape
    a = _lib.G4PackedPrefillArgs(tokens=T, kv_heads=H, group=R, head_dim=D, window=window, longest=longest)
    return _lib.lib().g4_packed_prefill_workspace_size(ctypes.byref(a))


@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("lens,tail,R,longest", [([1100], 0, 2, 0), ([900], 5, 8, 900), ([1, 800, 0, 31, 400, 33], 2, 3, 800),
                                                 ([2500], 0, 1, 2500)])
def test_keys_in_pieces(D, lens, tail, R, longest, device):
    q, k, v = _inputs(lens, tail, 1, R, D, 11, device)
    assert _pieces(q, 0, longest) > 0
    got = _run(q, k, v, lens, 0, device, fill=math.nan, longest=longest)
    _check(got, q, k, v, lens, 0)
    again = _run(q, k, v, lens, 0, device, fill=math.nan, longest=longest)
    assert torch.equal(got, again)


@pytest.mark.parametrize("longest", [0, 1, 100, 770, 1000, 5000])
def test_a_wrong_longest_costs_time_only(longest, device):
    lens = [30, 1500, 7]
    q, k, v = _inputs(lens, 3, 2, 2, 64, 12, device)
    _check(_run(q, k, v, lens, 0, device, longest=longest), q, k, v, lens, 0)
    _check(_run(q, k, v, lens, 900, device, longest=longest), q, k, v, lens, 900)


@pytest.mark.parametrize("D,R", [(64, 2), (512, 1)])
def test_pieces_of_many_sizes_of_score(D, R, device):
    """Scores that rise or fall by hundreds along the keys: a piece's maximum is far below or above the others'."""

    T = 1200
    for sign in (1, -1):
        q, k, v = _inputs([T], 0, 1, R, D, 13, device)
        q[..., 0] = 1.0
        k[..., 0] = (sign * torch.arange(T) / 4).to(torch.bfloat16)[:, None]
        assert _pieces(q) > 0
        _check(_run(q, k, v, [T], 0, device), q, k, v, [T], 0)


def test_pieces_with_values_that_are_not_finite(device):
    """A NaN or infinite value reaches the tokens behind it and no other; scores of -inf in whole pieces are as none."""

    T, D = 1300, 64
    q, k, v = _inputs([T], 0, 1, 2, D, 14, device)
    assert _pieces(q) > 0
    want, bound = packed_reference(q, k, v, [T], 0)
    v[700, 0, 5], v[900, 0, 6] = math.nan, math.inf
    got = _run(q, k, v, [T], 0, device).cpu().double()
    assert bool(got[700:, ..., 5].isnan().all()) and bool((got[900:, ..., 6] == math.inf).all())
    want[700:, ..., 5], want[900:, ..., 6] = 0, 0
    got[700:, ..., 5], got[900:, ..., 6] = 0, 0
    assert bool(((got - want).abs() <= bound).all())
    q, k, v = _inputs([T], 0, 1, 2, D, 14, device)
    q[..., 0] = 1.0
    k[:800, :, 0] = -math.inf
    got = _run(q, k, v, [T], 0, device)
    assert bool((got[:800] == 0).all())
    want, bound = packed_reference(q[800:], k[800:], v[800:], [T - 800], 0)
    assert bool(((got[800:].cpu().double() - want).abs() <= bound).all())


def test_pieces_in_a_graph_with_eager_calls_between(device):
    lens = [1000, 300]
    (q, k, v), (q2, k2, v2) = (_inputs(lens, 0, 1, 4, 256, s, device) for s in (15, 16))
    a, b = _run(q, k, v, lens, 0, device), _run(q2, k2, v2, lens, 0, device)
    starts = kernels.packed_starts(torch.tensor([0, 1000, 1300], dtype=torch.int32, device=device), 1300)
    qd, (kk, vv) = q.to(device), _laid_out(k, v, device)
    assert _pieces(q) > 0
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        kernels.packed_prefill_attention(qd, kk, vv, starts)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kernels.packed_prefill_attention(qd, kk, vv, starts)
    new = (q2.to(device), *_laid_out(k2, v2, device))
    old = (q.to(device), *_laid_out(k, v, device))
    for replay in range(4):
        for to, x in zip((qd, kk, vv), new if replay % 2 else old):
            to.copy_(x)
        graph.replay()
        assert torch.equal(_run(q, k, v, lens, 0, device), a)
        torch.cuda.synchronize()
        assert torch.equal(out, b if replay % 2 else a)


# --- many rows: blocks of 128 -----------------------------------------------------------------------------


MANY = [33, 0, 1, 130, 65, 2, 250, 31, 45]  # 557 tokens of 8 x 16 heads: 560 workgroups of 128 rows


@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("window", [0, 40])
def test_many_rows(D, window, device):
    q, k, v = _inputs(MANY, 3, 8, 16, D, 21, device)
    got = _run(q, k, v, MANY, window, device, fill=math.nan)
    _check(got, q, k, v, MANY, window)


@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_many_rows_with_values_that_are_not_finite(D, device):
    q, k, v = _inputs(MANY, 3, 8, 16, D, 22, device)
    want, bound = packed_reference(q, k, v, MANY, 0)
    v[180, 3, 5], v[400, 2, 6] = math.nan, math.inf  # in the 130 and the 250 tokens
    got = _run(q, k, v, MANY, 0, device).cpu().double()
    ends = [sum(MANY[:i + 1]) for i in range(len(MANY))]
    for at, h, d in ((180, 3, 5), (400, 2, 6)):
        end = next(e for e in ends if e > at)
        assert not bool(got[at:end, h, :, d].isfinite().any())
        got[at:end, h, :, d] = want[at:end, h, :, d] = 0
    assert bool(((got - want).abs() <= bound).all())


@pytest.mark.parametrize("tokens,window,longest", [(511, 0, 0), (512, 0, 0), (513, 0, 0), (255, 40, 0), (256, 40, 0), (257, 40, 0),
                                                   (257, 0, 50)])
def test_about_the_change_of_blocks(tokens, window, longest, device):
    """8 heads of 16: as many workgroups of two blocks per wave as tokens. One block per wave up to 512, up to 256 where a window or
    the sequences' length make them alike."""

    lens = [50] * 5 + [tokens - 250] if longest else [tokens - 200, 200]
    q, k, v = _inputs(lens, 0, 8, 16, 64, 23, device)
    _check(_run(q, k, v, lens, window, device, longest=longest), q, k, v, lens, window)


# --- far offsets, other streams ----------------------------------------------------------------------------------------


def test_heads_past_4_gib(device):
    """Keys and values of 2 GiB a head: the fourth head's lie past 2^32 bytes, as does what the call must not reach."""

    H, D, T, Sp = 4, 512, 150, 1 << 21
    lens = [40, 110]
    q, k, v = _inputs(lens, 0, H, 2, D, 41, device)
    kk = torch.empty(key_shape(1, H, Sp, D), dtype=torch.bfloat16, device=device)
    vv = torch.empty((1, H, Sp // 8, D, 8), dtype=torch.bfloat16, device=device)
    ks, vs = _laid_out(k, v, device, math.nan)
    kk[:, :, :ks.shape[2]], vv[:, :, :vs.shape[2]] = ks, vs
    starts = kernels.packed_starts(torch.tensor([0, 40, 150], dtype=torch.int32, device=device), T)
    _check(kernels.packed_prefill_attention(q.to(device), kk, vv, starts), q, k, v, lens, 0)


def test_rows_past_4_gib(device):
    """66000 tokens of 2 x 64 heads of 256: queries and results of 4.3 GB; the last sequences against 64 bits."""

    H, R, D, T = 2, 64, 256, 66000
    lens = [600] * 109 + [500, 90, 10]
    assert sum(lens) == T
    g = torch.Generator(device=device).manual_seed(42)
    q = torch.empty((T, H, R, D), dtype=torch.bfloat16, device=device).normal_(0, 0.1, generator=g)
    k, v = (torch.empty((T, H, D), dtype=torch.bfloat16, device=device).normal_(0, 1, generator=g) for _ in range(2))
    kk, vv = _laid_out(k.cpu(), v.cpu(), device)
    cu = torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32, device=device)
    out = kernels.packed_prefill_attention(q, kk, vv, kernels.packed_starts(cu, T), window=64)
    for a, n in ((0, 600), (T - 100, 90), (T - 10, 10)):
        _check(out[a:a + n], q[a:a + n].cpu(), k[a:a + n].cpu(), v[a:a + n].cpu(), [n], 64)


def test_calls_on_two_streams(device):
    """Calls in pieces that overlap on two streams have workspaces of their own."""

    lens = [1200]
    calls = []
    for seed in (43, 44):
        q, k, v = _inputs(lens, 0, 1, 4, 128, seed, device)
        calls.append((q.to(device), *_laid_out(k, v, device)))
    starts = kernels.packed_starts(torch.tensor([0, 1200], dtype=torch.int32, device=device), 1200)
    assert _pieces(calls[0][0]) > 0
    want = [kernels.packed_prefill_attention(*c, starts) for c in calls]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(kernels.packed_prefill_attention(*calls[i], starts))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])


# --- more blocks than are at work at once: in the order of their keys ----------------------------------------------------


@pytest.mark.parametrize("D,H,R", [(64, 2, 16), (256, 8, 4), (512, 3, 8), (512, 4, 8)])
@pytest.mark.parametrize("lens,tail", [([700, 1, 0, 400, 33, 64, 1000, 3], 45), ([2201], 0)])
def test_sorted_blocks(D, H, R, lens, tail, device):
    """Runs of blocks across the sequences' borders and the tokens of none, a short run at the end."""

    q, k, v = _inputs(lens, tail, H, R, D, 61, device)
    assert 0 < _pieces(q) < 4096 and _pieces(q, 0, 200) == 0
    got = _run(q, k, v, lens, 0, device, fill=math.nan)
    _check(got, q, k, v, lens, 0)
    for longest in (1, 300, 2201):  # whatever the order, the same bits
        assert torch.equal(_run(q, k, v, lens, 0, device, fill=math.nan, longest=longest), got)


def test_sorted_blocks_with_any_starts(device):
    """starts that no sequences give: tokens of none in the middle, a start behind its token, one far back."""

    T, H, R, D = 1500, 4, 16, 128
    q, k, v = _inputs([T], 0, H, R, D, 62, device)
    starts = (torch.arange(T, dtype=torch.int32) // 300) * 300
    starts[100:230], starts[500], starts[700:705], starts[1400] = -1, 501, 2 ** 31 - 1, 3
    assert 0 < _pieces(q) < 4096
    kk, vv = _laid_out(k, v, device)
    got = kernels.packed_prefill_attention(q.to(device), kk, vv, starts.to(device)).cpu().double()
    for t in (0, 99, 100, 229, 230, 499, 500, 501, 702, 705, 1399, 1400, 1499):
        a = int(starts[t])
        if not 0 <= a <= t:
            assert bool((got[t] == 0).all())
            continue
        want, bound = packed_reference(q[a:t + 1], k[a:t + 1], v[a:t + 1], [t + 1 - a], 0)
        assert bool(((got[t] - want[-1]).abs() <= bound[-1]).all()), t


def test_sorted_blocks_of_long_sequences(device):
    """Blocks of more than 1024 chunks, which share bins; sampled tokens against 64 bits."""

    lens, R, D = [7777, 36000, 1], 4, 64
    q, k, v = _inputs(lens, 0, 1, R, D, 63, device)
    assert 0 < _pieces(q) < 4096
    got = _run(q, k, v, lens, 0, device).cpu().double()
    for t in list(range(0, 43778, 1999)) + [7776, 7777, 43776, 43777]:
        a = 0 if t < 7777 else 7777 if t < 43777 else 43777
        x, kk, vv = q[t, 0].double(), k[a:t + 1, 0].double(), v[a:t + 1, 0].double()
        s = x @ kk.T
        top = s.amax(dim=-1, keepdim=True)
        w = torch.softmax(s, dim=-1)
        # packed_reference's bound for one token
        ds = (D + 2) * 2.0 ** -24 * (x.abs() @ kk.abs().T) + 4 * 2.0 ** -24 * (1 + s.abs() + top.abs())
        rel = 2 * ds.amax(dim=-1, keepdim=True) + (2 * len(kk) + 16) * 2.0 ** -24
        mass = w @ vv.abs()
        bound = (2.0 ** -8 + rel) * mass * (1 + 2.0 ** -8) + 2.0 ** -8 * (w @ vv).abs() + 1e-37
        assert bool(((got[t, 0] - w @ vv).abs() <= bound).all()), t


def test_sorted_blocks_in_a_graph_and_on_streams(device):
    """Replays with other sequences and calls on two streams, each with an order of its own."""

    T, H, R, D = 2201, 2, 16, 64
    sets = []
    for i, lens in enumerate(([2201], [300, 1901], [1100, 1, 1100])):
        q, k, v = _inputs(lens, 0, H, R, D, 70 + i, device)
        cu = torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32, device=device)
        sets.append((q.to(device), *_laid_out(k, v, device), kernels.packed_starts(cu, T)))
    assert 0 < _pieces(sets[0][0]) < 4096
    want = [kernels.packed_prefill_attention(*s) for s in sets]
    static = [t.clone() for t in sets[0]]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        kernels.packed_prefill_attention(*static)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kernels.packed_prefill_attention(*static)
    for i in (1, 2, 0, 1):
        for to, x in zip(static, sets[i]):
            to.copy_(x)
        graph.replay()
        assert torch.equal(kernels.packed_prefill_attention(*sets[2 - i]), want[2 - i])
        torch.cuda.synchronize()
        assert torch.equal(out, want[i])
    streams, got = [torch.cuda.Stream() for _ in sets], [[] for _ in sets]
    for _ in range(4):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(kernels.packed_prefill_attention(*sets[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(x, w) for g, w in zip(got, want) for x in g)


def test_many_heads_of_few_blocks(device):
    """More workgroups than are at work at once, but one or two blocks a head: no order to find."""

    T, H, R, D = 300, 260, 1, 64
    q, k, v = _inputs([T], 0, H, R, D, 75, device)
    assert _pieces(q) == 0
    got = _run(q, k, v, [T], 0, device)
    _check(got[:, ::37], q[:, ::37], k[:, ::37], v[:, ::37], [T], 0)
