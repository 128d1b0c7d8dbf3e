"""Verification of drafted tokens on the GPU against 64 bits: acceptance, the race, greedy, log-probabilities, and the
distribution of what comes out."""

from __future__ import annotations

import math

import pytest
import torch

from gemma4_posttrain_jax_amd import kernels

pytestmark = pytest.mark.gpu


def verified(logits, drafts, uniforms, noise, temperature, draft_logits=None, lengths=None):
    """The operator in 64 bits on the CPU, row by row."""

    B, K1, V = logits.shape
    tokens = torch.full((B, K1), -1, dtype=torch.int32)
    logp = torch.zeros((B, K1), dtype=torch.float64)
    counts = []
    for b in range(B):
        x = logits[b].double()
        n = K1 - 1 if lengths is None else min(max(int(lengths[b]), 0), K1 - 1)
        policy = torch.log_softmax(x, dim=-1)
        i = 0
        if temperature <= 0:
            best = [int(torch.nonzero(r == r.max())[0, 0]) for r in x]
            while i < n and int(drafts[b, i]) == best[i]:
                i += 1
            token = best[i]
        else:
            p = torch.softmax(x / temperature, dim=-1)
            q = None if draft_logits is None else torch.softmax(draft_logits[b].double() / temperature, dim=-1)
            while i < n:
                d = int(drafts[b, i])
                if not 0 <= d < V or not float(uniforms[b, i]) * (1.0 if q is None else float(q[i, d])) < float(p[i, d]):
                    break
                i += 1
            w = p[i].clone()
            if i < n:
                if q is not None:
                    w = torch.clamp(w - q[i], min=0.0)
                elif 0 <= int(drafts[b, i]) < V:
                    w[int(drafts[b, i])] = 0.0
            race = torch.where(noise[b] > 0, w / -torch.log(noise[b].double()), torch.zeros(()).double())
            token = int(torch.nonzero(race == race.max())[0, 0])
        tokens[b, :i] = drafts[b, :i]
        tokens[b, i] = token
        for s in range(i + 1):
            logp[b, s] = policy[s, int(tokens[b, s])]
        counts.append(i)
    return tokens, torch.tensor(counts, dtype=torch.int32), logp


def _inputs(B, K, V, dtype, seed, draft, near=0.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, K + 1, V, generator=g) * 2
    top = torch.randint(0, V, (B, K + 1, min(V, 4)), generator=g)
    x.scatter_(2, top, 6 + 4 * torch.rand(top.shape, generator=g))
    logits = x.to(dtype)
    y = x[:, :K] + near * torch.randn(B, K, V, generator=g)
    q = y.to(dtype) if draft else None
    pick = (y if draft else x[:, :K]) - torch.log(-torch.log(torch.rand(B, K, V, generator=g).clamp(min=1e-7)))
    drafts = pick.argmax(dim=-1).to(torch.int32)
    return logits, drafts, torch.rand(B, K, generator=g), torch.rand(B, V, generator=g), q


def _check(got, want):
    (tokens, count, logp), (wt, wc, wl) = [t.cpu() for t in got], want
    assert torch.equal(count, wc)
    assert torch.equal(tokens, wt)
    # x - max and the logarithm of an f32 sum of f32 exponentials of up to 2^18 terms, each within 4 u plus the rounding of
    # its argument, 2 u |x - max|, whose weighted mean is below 16 here; the sums in at most 64 + 8 + 8 + 4 levels
    bound = 2.0 ** -24 * (2 * wl.abs() + 4 + 32 + 84)
    assert bool(((logp.double() - wl).abs() <= bound).all())


@pytest.mark.parametrize("V", [1, 2, 7, 8, 9, 1000, 2049, 4097, 32003])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("temperature", [0.0, 0.7, 1.0])
@pytest.mark.parametrize("draft", [False, True])
def test_against_64_bits(V, dtype, temperature, draft, device):
    B, K = 5, 3
    logits, drafts, u, noise, q = _inputs(B, K, V, dtype, V + 17, draft)
    got = kernels.verify_draft(logits.to(device), drafts.to(device), u.to(device), noise.to(device), temperature=temperature,
                               draft_logits=None if q is None else q.to(device))
    _check(got, verified(logits, drafts, u, noise, temperature, q))


@pytest.mark.parametrize("B,K,V", [(1, 1, 262144), (1, 63, 500), (3, 8, 131071), (40, 7, 40000), (300, 2, 33)])
@pytest.mark.parametrize("temperature", [0.0, 1.0, 1.3])
def test_sizes_and_ragged_drafts(B, K, V, temperature, device):
    logits, drafts, u, noise, q = _inputs(B, K, V, torch.bfloat16, 5, True, near=0.2)
    lengths = (torch.arange(B, dtype=torch.int32) * 5 % (K + 3)) - 1  # clamped: -1, and beyond K
    got = kernels.verify_draft(logits.to(device), drafts.to(device), u.to(device), noise.to(device), temperature=temperature,
                               draft_logits=q.to(device), draft_lengths=lengths.to(device))
    _check(got, verified(logits, drafts, u, noise, temperature, q, lengths))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_at_any_element(dtype, device):
    """Views: odd offsets, rows and batches apart, noise rows apart."""

    B, K, V = 3, 2, 1021
    logits, drafts, u, noise, q = _inputs(B, K, V, dtype, 6, True)
    big = torch.full((B, K + 2, V + 6), math.nan, dtype=dtype, device=device)
    big[:, 1:, 3:V + 3] = logits.to(device)
    qbig = torch.full((B + 1, K, V + 3), math.nan, dtype=dtype, device=device)
    qbig[1:, :, 1:V + 1] = q.to(device)
    nbig = torch.full((B, V + 5), math.nan, device=device)
    nbig[:, 1:V + 1] = noise.to(device)
    got = kernels.verify_draft(big[:, 1:, 3:V + 3], drafts.to(device), u.to(device), nbig[:, 1:V + 1], temperature=1.0,
                               draft_logits=qbig[1:, :, 1:V + 1])
    _check(got, verified(logits, drafts, u, noise, 1.0, q))


def test_masked_logits(device):
    """-inf and the type's lowest value in most columns, drafts among them; a row with one column left."""

    B, K, V = 6, 3, 777
    logits, drafts, u, noise, q = _inputs(B, K, V, torch.float32, 7, True)
    low = torch.finfo(torch.float32).min
    logits[:3, :, 100:] = -math.inf
    logits[3:, :, 100:] = low
    q[1:4, :, 50:] = low
    logits[5, :, 1:] = -math.inf
    for T in (0.0, 0.7, 1.0):
        got = kernels.verify_draft(logits.to(device), drafts.to(device), u.to(device), noise.to(device), temperature=T,
                                   draft_logits=q.to(device))
        wt, wc, wl = verified(logits, drafts, u, noise, T, q)
        assert torch.equal(got[0].cpu(), wt) and torch.equal(got[1].cpu(), wc)
        assert bool((got[2].cpu().double() - wl).abs().nan_to_num(0.0).max() < 1e-4)


def test_ids_outside_the_vocabulary_are_not_accepted(device):
    B, K, V = 4, 2, 50
    logits, drafts, u, noise, q = _inputs(B, K, V, torch.bfloat16, 8, True)
    drafts[0, 0], drafts[1, 1], drafts[2, 0], drafts[3, 0] = -1, V, 2 ** 31 - 1, -2 ** 31
    u.zero_()
    for T, ql in ((0.0, None), (1.0, None), (1.0, q)):
        got = kernels.verify_draft(logits.to(device), drafts.to(device), u.to(device), noise.to(device), temperature=T,
                                   draft_logits=None if ql is None else ql.to(device))
        _check(got, verified(logits, drafts, u, noise, T, ql))


def test_greedy_takes_the_first_of_equal_logits(device):
    logits = torch.zeros(2, 3, 9000, dtype=torch.bfloat16)
    logits[:, :, 8191] = logits[:, :, 4100] = logits[:, :, 4099] = 3.0
    drafts = torch.tensor([[4099, 4100], [4099, 4099]], dtype=torch.int32)
    tokens, count, _ = kernels.verify_draft(logits.to(device), drafts.to(device), None, None, temperature=0.0)
    assert tokens.tolist() == [[4099, 4099, -1], [4099, 4099, 4099]] and count.tolist() == [1, 2]


def test_noise_at_its_ends(device):
    """A column of noise 0 is never drawn, one next to 1 wins, equal scores go to the lowest id."""

    logits = torch.zeros(3, 2, 300)
    drafts = torch.full((3, 1), 7, dtype=torch.int32)
    u = torch.ones(3, 1)  # 1 * q < p is false: rejected, the residual is p without 7
    noise = torch.full((3, 300), 0.5)
    noise[0, 200] = 1 - 2.0 ** -24
    noise[1, :] = 0.0
    noise[1, 299] = 0.25
    tokens, count, _ = kernels.verify_draft(logits.to(device), drafts.to(device), u.to(device), noise.to(device), temperature=1.0)
    assert tokens[:, 0].tolist() == [200, 299, 0] and count.tolist() == [0, 0, 0]


def test_where_no_weight_is_left_the_token_is_drawn_from_p(device):
    """p = q everywhere and a draft of probability 0: rejected with an empty residual."""

    logits = torch.zeros(1, 2, 64)
    logits[..., 10] = -math.inf
    noise = torch.rand(1, 64, generator=torch.Generator().manual_seed(9))
    tokens, count, _ = kernels.verify_draft(logits.to(device), torch.tensor([[10]], dtype=torch.int32, device=device),
                                            torch.full((1, 1), 0.5, device=device), noise.to(device), temperature=1.0,
                                            draft_logits=logits[:, :1].to(device).contiguous())
    noise[0, 10] = 0
    assert count.tolist() == [0] and tokens[0, 0].item() == int(noise.argmax())


def test_rows_of_no_numbers(device):
    """NaN in a row: nothing accepted there, a token inside the vocabulary; other rows as they are."""

    B, K, V = 4, 2, 600
    logits, drafts, u, noise, q = _inputs(B, K, V, torch.bfloat16, 10, True)
    want = verified(logits, drafts, u, noise, 1.0, q)
    logits[1, 0, 5] = math.nan
    logits[2] = -math.inf
    got = [t.cpu() for t in kernels.verify_draft(logits.to(device), drafts.to(device), u.to(device), noise.to(device),
                                                 temperature=1.0, draft_logits=q.to(device))]
    for b in (0, 3):
        assert torch.equal(got[0][b], want[0][b]) and got[1][b] == want[1][b]
    for b in (1, 2):
        assert got[1][b] == 0 and got[0][b].tolist() == [0, -1, -1]


@pytest.mark.parametrize("draft", [False, True])
def test_the_first_token_has_the_targets_distribution(draft, device):
    """Whatever the drafter says, the first token is drawn from p: 400000 rows, counts within 5 deviations."""

    B, V = 400000, 11
    g = torch.Generator(device=device).manual_seed(11)
    p = torch.softmax(torch.linspace(-2, 2, V, device=device), dim=0)
    q = torch.softmax(torch.cos(torch.arange(V, device=device) * 1.7) * 1.5, dim=0)
    drafts = torch.multinomial(q, B, replacement=True, generator=g).to(torch.int32)[:, None].contiguous()
    logits = p.log().expand(B, 2, V).contiguous()
    tokens, count, logp = kernels.verify_draft(
        logits, drafts, torch.rand((B, 1), generator=g, device=device), torch.rand((B, V), generator=g, device=device),
        temperature=1.0, draft_logits=q.log().expand(B, 1, V).contiguous() if draft else None)
    seen = torch.bincount(tokens[:, 0], minlength=V).double()
    assert bool(((seen - B * p.double()).abs() <= 5 * (B * p.double() * (1 - p.double())).sqrt()).all())
    rate = float(torch.minimum(p, q).sum()) if draft else float((p * q).sum())
    assert abs(float(count.double().mean()) - rate) <= 5 * math.sqrt(rate * (1 - rate) / B)


def test_the_same_call_gives_the_same_bits(device):
    logits, drafts, u, noise, q = _inputs(4, 3, 70000, torch.bfloat16, 12, True)
    args = [t.to(device) for t in (logits, drafts, u, noise)]
    first = kernels.verify_draft(*args, temperature=0.9, draft_logits=q.to(device))
    again = kernels.verify_draft(*args, temperature=0.9, draft_logits=q.to(device))
    assert all(torch.equal(x, y) for x, y in zip(first, again))


# --- many logits: two steps per thread -------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("temperature", [0.0, 0.05, 1.0, 1.3])
def test_many_logits(dtype, temperature, device):
    """2^25 logits and more; the levels of a row's stretches of 2048 columns rise and fall, by less and by more than what a running
    maximum may lag, and some stretches are masked."""

    B, K, V = 58, 7, 40001
    logits, drafts, u, noise, q = _inputs(B, K, V, dtype, 31, True)
    assert logits.numel() + q.numel() >= 2 ** 25
    level = torch.tensor([0, 3, 6, 9, -4, 40, 7, 60, -math.inf, 0, 2, 61, 5, -30, -math.inf, 4, 62, 1, 66, 0.5])
    for b in range(0, B, 3):
        shift = level.roll(b).repeat_interleave(2048)[:V]
        logits[b] += shift.to(dtype)
        q[b] += shift.to(dtype)
    logits[1, :, :20000] = -math.inf
    got = kernels.verify_draft(logits.to(device), drafts.to(device), u.to(device), noise.to(device), temperature=temperature,
                               draft_logits=q.to(device))
    want = verified(logits, drafts, u, noise, temperature, q)
    if temperature == 0.05:
        _near_ties(got[0].cpu(), want, logits, q, noise, temperature)
    _check(got, want)


def _near_ties(tokens, want, logits, q, noise, temperature):
    """Where the next token differs, takes the operator's into ``want`` if the race is a tie for f32 probabilities. Each is off by
    eps = u (120 + 2 |x - max| / T) of itself: a sum of up to 100 levels, exp and the product within 2 u each, and the
    exponent's rounding. The drafts here are not drawn at this temperature, so that rows are rejected whose p and q both
    are one token's but for 2^-24: all that p - q has is below its error eps (p + q)."""

    wt, wc, wl = want
    for b in (tokens != wt).any(dim=-1).nonzero()[:, 0].tolist():
        i = int(wc[b])
        got = int(tokens[b, i])
        x, y = logits[b, i].double(), q[b, min(i, q.shape[1] - 1)].double()
        p = torch.softmax(x / temperature, dim=-1)
        z = torch.softmax(y / temperature, dim=-1) if i < q.shape[1] else torch.zeros_like(p)
        eps = [2.0 ** -24 * (120 + 2 * (t.max() - t).clamp(max=1e4) / temperature) for t in (x, y)]
        pace = torch.where(noise[b] > 0, 1 / -torch.log(noise[b].double()), torch.zeros(()).double()) * (1 + 2.0 ** -20)
        w, error = torch.clamp(p - z, min=0.0), eps[0] * p + eps[1] * z
        assert float((w + error)[got] * pace[got]) >= float(((w - error) * pace).max())
        wt[b, i], wl[b, i] = got, torch.log_softmax(x, dim=-1)[got]


def test_unlikely_drafts(device):
    """Drafts whose probabilities are far below f32's range are accepted by their ratio."""

    B, K, V = 4, 1, 300
    logits, q = torch.zeros(B, K + 1, V), torch.zeros(B, K, V)
    logits[:, 0, 7], q[:, 0, 7] = 40.0, 40.0
    logits[:, 0, 9], q[:, 0, 9] = torch.tensor([-80.0, -81.0, -80.0, -80.0]), torch.tensor([-80.25, -80.0, -79.875, -80.0])
    drafts, u = torch.full((B, K), 9, dtype=torch.int32), torch.tensor([[0.9], [0.9], [0.25], [0.4]])
    noise = torch.rand(B, V, generator=torch.Generator().manual_seed(3))
    got = kernels.verify_draft(logits.to(device), drafts.to(device), u.to(device), noise.to(device), temperature=0.5,
                               draft_logits=q.to(device))
    assert got[1].tolist() == [1, 0, 1, 1]  # p / q = e^.5, e^-2, e^-.25, 1


def test_many_logits_replayed_in_a_graph(device):
    """Replays with new inputs between eager calls of other sizes give what eager calls give."""

    B, K, V = 4, 3, 5000
    sets = [[None if t is None else t.to(device) for t in _inputs(B, K, V, torch.bfloat16, s, True)] for s in (41, 42, 43)]
    other = [t.to(device) for t in _inputs(9, 5, 3001, torch.bfloat16, 44, True)]

    def run(logits, drafts, u, noise, q):
        return kernels.verify_draft(logits, drafts, u, noise, temperature=0.9, draft_logits=q)

    want = [[t.clone() for t in run(*s)] for s in sets]
    theirs = [t.clone() for t in run(*other)]
    static = [t.clone() for t in sets[0]]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run(*static)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(*static)
    for i in (1, 2, 0, 1):
        for to, x in zip(static, sets[i]):
            to.copy_(x)
        graph.replay()
        assert all(torch.equal(x, y) for x, y in zip(run(*other), theirs))
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, want[i]))


def test_two_streams_at_once(device):
    """Calls that overlap on two streams have workspaces of their own."""

    sets = [[t.to(device) for t in _inputs(6, 3, 20000, torch.bfloat16, s, True)] for s in (45, 46)]
    run = lambda s: kernels.verify_draft(s[0], s[1], s[2], s[3], temperature=0.8, draft_logits=s[4])  # noqa: E731
    want = [[t.clone() for t in run(s)] for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(run(sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for out in got[i]:
            assert all(torch.equal(x, y) for x, y in zip(out, want[i]))


def test_rows_past_4_gib(device):
    """Logits and the drafter's of more than 2^32 bytes each: their last rows give what they give alone."""

    B, K, V = 260, 33, 262144
    logits = torch.empty((B, K + 1, V), dtype=torch.bfloat16, device=device).normal_()
    q = torch.empty((B, K, V), dtype=torch.bfloat16, device=device).normal_()
    assert min(logits.numel(), q.numel()) * 2 > 2 ** 32
    g = torch.Generator(device=device).manual_seed(5)
    drafts = torch.randint(0, V, (B, K), generator=g, device=device, dtype=torch.int32)
    drafts[:, 2:] = q[:, 2:].argmax(dim=-1).to(torch.int32)
    u = torch.rand(B, K, generator=g, device=device) * 0.5
    noise = torch.rand(B, V, generator=g, device=device)
    got = kernels.verify_draft(logits, drafts, u, noise, temperature=1.0, draft_logits=q)
    for rows in (slice(0, 3), slice(B - 3, B)):
        want = kernels.verify_draft(logits[rows], drafts[rows], u[rows], noise[rows], temperature=1.0, draft_logits=q[rows])
        assert torch.equal(got[0][rows], want[0]) and torch.equal(got[1][rows], want[1])
        # another split of the sums: 84 levels' roundings, and those of the logarithm and the difference
        bound = 2.0 ** -23 * (2 * want[2].abs() + 120)
        assert bool(((got[2][rows] - want[2]).abs() <= bound).all())


@pytest.mark.parametrize("B,V", [(1024, 500), (1025, 500), (205, 20000), (205, 20481)])  # 1024, 1025, 1025, 1230 chunks of 4096
@pytest.mark.parametrize("temperature,draft", [(0.7, True), (1.0, False)])
def test_about_the_change_of_who_decides(B, V, temperature, draft, device):
    K = 3
    logits, drafts, u, noise, q = _inputs(B, K, V, torch.bfloat16, 51, draft)
    lengths = (torch.arange(B, dtype=torch.int32) * 7 % (K + 1))
    got = kernels.verify_draft(logits.to(device), drafts.to(device), u.to(device), noise.to(device), temperature=temperature,
                               draft_logits=None if q is None else q.to(device), draft_lengths=lengths.to(device))
    _check(got, verified(logits, drafts, u, noise, temperature, q, lengths))
