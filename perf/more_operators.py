"""Operators of rollouts with several completions per prompt, case by case: what a program that serves Gemma 4
rollouts has this framework do between the prompts and the first steps of their completions.

Kinds of case:
- ``packed``: causal attention of prompts of different lengths that stand one behind the other, without pads
  (``kernels.packed_prefill_attention``);
- ``fork``: the completions of a batch of prompts take over the prompts' pages: whole pages shared, the last one
  copied (``kernels.paged_fork``), the prompts' own rows let go (``kernels.paged_free``) and pages for the new tokens
  taken (``kernels.paged_reserve``);
- ``copy``: pages copied to other pages in all layers at once (``kernels.paged_copy``);
- ``compact``: the pages in use moved to the front of the pool (``kernels.paged_compact``);
- ``verify``: drafted tokens accepted or replaced by the target's probabilities (``kernels.verify_draft``).

Packed keys and values are one row of the framework's dense layouts, ``key [1, H, S / 32, D / 32, 2, 16, 32]`` and
``value [1, H, S / 8, D, 8]`` (slot 8 a + 4 b + c of a 32-slot chunk is half b, lane 4 a + c of a key run; values in
groups of 8 slots). Pages hold the same per page, ``key [P, H, page / 32, D / KR, 2, 16, KR]``, ``value [P, H, page / 8,
D, 8]`` and in e4m3 ``key_scale`` / ``value_scale [P, H, page]``; here the layers of a cache are stacked in front.
``refs [P]`` counts the table entries that hold a page, 0 for a free one; fresh pages are the lowest free ones in
the order of the rows that take them.

The plain forms are elementary torch operations; ``exact`` restates each operator in 64 bits, row by row.
"""

from __future__ import annotations

import importlib
import importlib.util
import math
import sys
from pathlib import Path

import torch

own = False

DEV = "cuda"
BF16, F8, E8 = torch.bfloat16, torch.float8_e4m3fn, torch.float8_e8m0fnu


def listed() -> list[dict]:
    return [
        # one short interactive prompt, a sliding layer: the launch's latency
        dict(name="packed_single", kind="packed", seqs=1, lo=23, hi=23, tail=0, heads=2, group=4, dim=256, window=512),
        # a sliding layer of the benchmark's prompts, of 32 to 480 tokens instead of 256 each
        dict(name="packed_rollout", kind="packed", seqs=256, lo=32, hi=480, tail=0, heads=2, group=4, dim=256,
             window=512),
        # a global layer over a few long prompts
        dict(name="packed_long", kind="packed", seqs=3, lo=2047, hi=8191, tail=5, heads=2, group=4, dim=256, window=0),
        # a stock configuration's global layer (head dim 512) over ragged prompts, tokens of no prompt behind them
        dict(name="packed_wide", kind="packed", seqs=13, lo=1, hi=2001, tail=37, heads=1, group=8, dim=512, window=0),
        # one prompt to four completions on one layer: the launches' latency
        dict(name="fork_single", kind="fork", prompts=1, share=4, lo=701, hi=701, new=64, layers=1, heads=2, dim=256,
             page=64, e4m3=False, busy=40, spare=9),
        # 16 prompts to 16 completions each over the global layers of the benchmark's model
        dict(name="fork_rollout", kind="fork", prompts=16, share=16, lo=200, hi=767, new=128, layers=2, heads=2, dim=256,
             page=64, e4m3=False, busy=200, spare=100),
        # the rings of 16 prompts to those of 64 completions: a window of 512 on sliding layers, e4m3
        dict(name="copy_rings", kind="copy", parents=16, share=4, ring=9, layers=8, heads=2, dim=256, page=64,
             e4m3=True, spare=11),
        # a pool after half of its rows have ended, small pages
        dict(name="compact_rows", kind="compact", rows=64, lo=1, hi=2047, ended=0.5, layers=2, heads=2, dim=256, page=32,
             e4m3=False, spare=100),
        # a large pool of few layers in e4m3, of which little moves: the search through the pool
        dict(name="compact_large", kind="compact", rows=256, lo=2048, hi=8191, ended=0.05, layers=1, heads=1, dim=128,
             page=32, e4m3=True, spare=1000),
        # one row's drafts at the benchmark's vocabulary
        dict(name="verify_single", kind="verify", rows=1, drafts=4, vocab=262144, bf16=True, draft_logits=True,
             ragged=False, temperature=1.0),
        # a rollout batch's, with the drafter's own logits
        dict(name="verify_rollout", kind="verify", rows=64, drafts=4, vocab=262144, bf16=True, draft_logits=True,
             ragged=False, temperature=0.7),
        # drafts looked up in the prompt (no drafter's logits), of different numbers, an odd vocabulary, f32 logits
        dict(name="verify_lookup", kind="verify", rows=33, drafts=7, vocab=32003, bf16=False, draft_logits=False,
             ragged=True, temperature=1.0),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def draw(rng) -> dict:
    kind = rng.choices(["packed", "fork", "copy", "compact", "verify"], [5, 3, 1, 2, 4])[0]
    heads, dim, page, e4m3 = rng.choice([1, 2, 3, 4]), rng.choice([64, 128, 256, 512]), rng.choice([32, 64, 128, 256]), \
        rng.random() < 0.5
    if kind == "packed":
        group = rng.choice([1, 2, 3, 4, 8, 16])
        hi = _log_int(rng, 1, min(8192, math.isqrt(2 * 10 ** 11 // (heads * group * dim))))
        most = min(2 * 10 ** 11 // (hi * hi * heads * group * dim), 10 ** 9 // (hi * hi * heads * group),
                   25 * 10 ** 7 // (hi * heads * group * dim))
        return dict(kind=kind, seqs=_log_int(rng, 1, max(1, min(512, most))), lo=rng.randint(0, hi), hi=hi,
                    tail=rng.choice([0, 0, rng.randint(1, 100)]), heads=heads, group=group, dim=dim,
                    window=rng.choice([0, 0, 512, rng.randint(1, 1024)]))
    # pages of all layers that fit what the largest listed cache takes
    layers = rng.choice([1, 2, 4, 8])
    size = layers * heads * dim * page * (2 if e4m3 else 4)
    most = max(12, (380 << 20) // size)
    if kind == "fork":
        hi = rng.randint(1, max(1, min(2048, most // 4 * page)))
        new = _log_int(rng, 1, max(1, min(512, most // 4 * page)))
        prompts = _log_int(rng, 1, max(1, min(64, most // 4 // (hi // page + 1))))
        share = _log_int(rng, 1, max(1, min(64, most // 2 // (prompts * (new // page + 2)))))
        return dict(kind=kind, prompts=prompts, share=share, lo=rng.randint(0, hi), hi=hi, new=new, layers=layers,
                    heads=heads, dim=dim, page=page, e4m3=e4m3, busy=rng.randint(0, min(500, most // 8)),
                    spare=rng.randint(0, min(100, most // 8)))
    if kind == "copy":
        ring = rng.randint(1, min(9, most // 4))
        share = _log_int(rng, 1, max(1, min(16, most // (3 * ring))))
        return dict(kind=kind, parents=_log_int(rng, 1, max(1, min(64, most // (ring * (share + 1))))), share=share,
                    ring=ring, layers=layers, heads=heads, dim=dim, page=page, e4m3=e4m3,
                    spare=rng.randint(0, min(50, most // 8)))
    if kind == "compact":
        hi = _log_int(rng, 1, max(1, min(8192, most // 2 * page)))
        return dict(kind=kind, rows=_log_int(rng, 1, max(1, min(512, most // (hi // page + 1)))), lo=rng.randint(1, hi),
                    hi=hi, ended=rng.choice([0.0, 0.1, 0.5, 0.9, 1.0]), layers=layers, heads=heads, dim=dim, page=page,
                    e4m3=e4m3, spare=rng.randint(0, min(500, most // 8)))
    vocab = _log_int(rng, 2, 262144)
    drafts = rng.choice([1, 2, 3, 4, 5, 7, 8])
    bf16 = rng.random() < 0.6
    most = (64 * 11 * 262144) // (vocab * (2 * drafts + 3) * (1 if bf16 else 2))
    return dict(kind=kind, rows=_log_int(rng, 1, max(1, min(256, most))), drafts=drafts, vocab=vocab, bf16=bf16,
                draft_logits=rng.random() < 0.6, ragged=rng.random() < 0.4, temperature=rng.choice([0.0, 0.7, 1.0, 1.0, 1.3]))


# --- what a program has in hand ------------------------------------------------------------------------


def _spread(lo: int, hi: int, n: int) -> list[int]:
    """n lengths, spread evenly over [lo, hi], the longest first."""

    return [hi - (hi - lo) * i // max(1, n - 1) for i in range(n)]


def _shuffled(values: list[int], g: torch.Generator) -> torch.Tensor:
    t = torch.tensor(values, dtype=torch.int32, device=DEV)
    return t[torch.randperm(len(values), generator=g, device=DEV)]


def _normal(shape, g: torch.Generator, std: float = 1.0) -> torch.Tensor:
    return torch.empty(shape, dtype=BF16, device=DEV).normal_(0.0, std, generator=g)


def _cache(case: dict, pages: int, g: torch.Generator) -> dict:
    """The stacked layers of a cache; what the pages hold stands for stored keys and values."""

    L, H, D, ps, e4m3 = case["layers"], case["heads"], case["dim"], case["page"], case["e4m3"]
    kr = 64 if e4m3 else 32
    s = {"key": _normal((L, pages, H, ps // 32, D // kr, 2, 16, kr), g), "value": _normal((L, pages, H, ps // 8, D, 8), g)}
    if e4m3:
        s = {n: x.to(F8) for n, x in s.items()}
        for n in ("key_scale", "value_scale"):
            s[n] = torch.randint(118, 122, (L, pages, H, ps), dtype=torch.uint8, generator=g, device=DEV).view(E8)
    return s


def _table(counts: list[int], width: int, order: torch.Tensor) -> torch.Tensor:
    """Rows of ``counts[b]`` pages each, in the order in which ``order`` has them; -1 beyond."""

    at = torch.arange(width, device=DEV)[None, :]
    n = torch.tensor(counts, device=DEV)[:, None]
    ids = (n.cumsum(0) - n + at).clamp(max=order.numel() - 1)
    return torch.where(at < n, order[ids], torch.full((), -1, device=DEV)).to(torch.int32)


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEV).manual_seed(seed)
    return {"case": case, **{"packed": _prepare_packed, "fork": _prepare_fork, "copy": _prepare_copy,
                             "compact": _prepare_compact, "verify": _prepare_verify}[case["kind"]](case, g)}


def _prepare_packed(case: dict, g: torch.Generator) -> dict:
    H, R, D = case["heads"], case["group"], case["dim"]
    lens = _shuffled(_spread(case["lo"], case["hi"], case["seqs"]), g)
    cu = torch.cat([torch.zeros(1, dtype=torch.int32, device=DEV), lens.cumsum(0).to(torch.int32)])
    T = max(1, int(cu[-1]) + case["tail"])
    slots = (T + 63) // 64 * 64
    t = torch.arange(T, dtype=torch.int32, device=DEV)
    seq = torch.searchsorted(cu, t, right=True, out_int32=True) - 1
    # scores with a deviation of about 2, as trained norms of q and k give; starts: the first token of each token's
    # prompt, -1 for a token of none
    return dict(cu=cu, starts=torch.where(seq < case["seqs"], cu[seq.long()], torch.full_like(t, -1)),
                longest=case["hi"], q=_normal((T, H, R, D), g, 2.0 / math.sqrt(D)),
                key=_normal((1, H, slots // 32, D // 32, 2, 16, 32), g), value=_normal((1, H, slots // 8, D, 8), g))


def _prepare_fork(case: dict, g: torch.Generator) -> dict:
    ps, new, share = case["page"], case["new"], case["share"]
    lens = _shuffled(_spread(case["lo"], case["hi"], case["prompts"]), g)
    host = lens.tolist()
    held = [(n + ps - 1) // ps for n in host]
    fresh = sum((n + new + ps - 1) // ps - n // ps for n in host)
    used = sum(held) + case["busy"]
    pages = used + share * fresh + case["spare"]
    order = torch.randperm(pages, generator=g, device=DEV)
    refs = torch.zeros(pages, dtype=torch.int32, device=DEV)
    refs[order[:used]] = 1  # the prompts' pages and those of rows that run along
    parents = torch.arange(case["prompts"], dtype=torch.int32, device=DEV).repeat_interleave(share)
    width = (case["hi"] + new + ps - 1) // ps
    return dict(lengths=lens, parents=parents, refs=refs, table=_table(held, width, order),
                target=lens[parents.long()] + new, none=torch.zeros_like(lens), **_cache(case, pages, g))


def _prepare_copy(case: dict, g: torch.Generator) -> dict:
    n, ring = case["parents"], case["ring"]
    pages = n * ring * (1 + case["share"]) + case["spare"]
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    src = order[:n * ring].view(n, 1, ring).expand(n, case["share"], ring).reshape(-1).contiguous()
    return dict(src=src, dst=order[n * ring: n * ring * (1 + case["share"])].contiguous(), **_cache(case, pages, g))


def _prepare_compact(case: dict, g: torch.Generator) -> dict:
    ps, B = case["page"], case["rows"]
    lens = _shuffled(_spread(case["lo"], case["hi"], B), g).tolist()
    held = [(n + ps - 1) // ps for n in lens]
    pages = sum(held) + case["spare"]
    table = _table(held, max(held), torch.randperm(pages, generator=g, device=DEV))
    ended = torch.rand(B, generator=g, device=DEV) < case["ended"]
    table = torch.where(ended[:, None], torch.full_like(table, -1), table)
    if B > 2:  # rows in pairs share their first page
        table[1::2, 0] = torch.where(ended[1::2] | ended[0:B // 2 * 2:2], table[1::2, 0], table[0:B // 2 * 2:2, 0])
    refs = torch.bincount(table[table >= 0].long(), minlength=pages).to(torch.int32)
    return dict(refs=refs, table=table, **_cache(case, pages, g))


def _prepare_verify(case: dict, g: torch.Generator) -> dict:
    B, K, V = case["rows"], case["drafts"], case["vocab"]
    # capped logits of a trained head: a broad background and a few likely tokens; the drafter's are near them
    x = torch.empty((B, K + 1, V), device=DEV).normal_(0.0, 2.0, generator=g)
    likely = torch.randint(0, V, (B, K + 1, 8), generator=g, device=DEV)
    x.scatter_(2, likely, 8.0 + 8.0 * torch.rand((B, K + 1, 8), generator=g, device=DEV))
    x = 30.0 * torch.tanh(x / 30.0)
    s = {"logits": x.to(BF16 if case["bf16"] else torch.float32)}
    near = x[:, :K]
    if case["draft_logits"]:
        near = near + torch.empty((B, K, V), device=DEV).normal_(0.0, 0.5, generator=g)
        s["draft_logits"] = near = near.to(s["logits"].dtype)
    noise = torch.rand((B, K, V), generator=g, device=DEV).clamp_(min=1e-7)
    heat = case["temperature"] or 1.0
    s["drafts"] = (near.float() / heat - torch.log(-torch.log(noise))).argmax(dim=-1).to(torch.int32)
    if not case["draft_logits"]:  # half of a prompt's continuations are not what the model says
        other = torch.randint(0, V, (B, K), dtype=torch.int32, generator=g, device=DEV)
        s["drafts"] = torch.where(torch.rand((B, K), generator=g, device=DEV) < 0.4, other, s["drafts"])
    if case["ragged"]:
        s["number"] = torch.randint(0, K + 1, (B,), dtype=torch.int32, generator=g, device=DEV)
    s["uniforms"] = torch.rand((B, K), generator=g, device=DEV)
    s["noise"] = torch.rand((B, V), generator=g, device=DEV)
    return s


# --- one pass --------------------------------------------------------------------------------------------


def _tokens(s: dict) -> tuple[torch.Tensor, torch.Tensor]:
    """The f32 keys and values ``[S, H, D]`` of packed prompts."""

    _, H, C, N, _, _, kr = s["key"].shape
    k = s["key"].view(H, C, N, 2, 4, 4, kr).permute(1, 4, 3, 5, 0, 2, 6).reshape(C * 32, H, N * kr)
    return k.float(), s["value"][0].permute(1, 3, 0, 2).reshape(C * 32, H, -1).float()


def _packed(s: dict) -> torch.Tensor:
    T, H, R, D = s["q"].shape
    k, v = _tokens(s)
    L, n = max(1, s["longest"]), s["cu"][1:] - s["cu"][:-1]
    at = torch.arange(L, device=DEV)
    there = at[None, :] < n[:, None]  # [N, L]: the prompts side by side, padded
    tok = torch.where(there, s["cu"][:-1, None] + at, torch.zeros_like(at)).long()
    q = s["q"].float()[tok].permute(0, 2, 3, 1, 4)  # [N, H, R, L, D]
    scores = torch.matmul(q, k[tok].permute(0, 2, 3, 1)[:, :, None])
    seen = at[None, :] <= at[:, None]
    if s["case"]["window"]:
        seen = seen & (at[None, :] > at[:, None] - s["case"]["window"])
    scores.masked_fill_(~seen, -math.inf)
    p = scores.sub_(scores.amax(dim=-1, keepdim=True)).exp_()
    rows = torch.matmul(p, v[tok].permute(0, 2, 1, 3)[:, :, None]).div_(p.sum(dim=-1, keepdim=True))
    out = torch.zeros((T + 1, H, R, D), device=DEV)
    out[torch.where(there, tok, torch.full_like(tok, T))] = rows.permute(0, 3, 1, 2, 4)
    return out[:T].to(BF16)


def _raw(t: torch.Tensor) -> torch.Tensor:
    return t if t.dtype == BF16 else t.view(torch.uint8)


_ARRAYS = ("key", "value", "key_scale", "value_scale")


def _pages(s: dict) -> dict:
    return {n: s[n] for n in _ARRAYS if n in s}


def _move(t: torch.Tensor, src: torch.Tensor, dst: torch.Tensor, slots: torch.Tensor | None) -> None:
    """Pages ``src`` of a stacked array to ``dst``; with ``slots`` the 32-slot chunks of each that hold them."""

    x = _raw(t)
    x = x.view(*x.shape[:3], _slots(t) // 32, -1)
    if slots is None:
        x[:, dst] = x[:, src]
        return
    live = (torch.arange(x.shape[3], device=DEV) * 32 < slots[:, None])[None, :, None, :, None]
    x[:, dst] = torch.where(live, x[:, src], x[:, dst])


def _slots(t: torch.Tensor) -> int:
    """Positions per page of a stacked array: keys have 7 dims behind the layers, values 5, scales 3."""

    return {8: lambda: t.shape[3] * 32, 6: lambda: t.shape[3] * 8, 4: lambda: t.shape[3]}[t.dim()]()


def _take(refs: torch.Tensor, wanted: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The lowest free pages for the true entries of ``wanted``, in their order: (their indexes, the pages, how
    many got none)."""

    at = torch.nonzero(wanted.reshape(-1))[:, 0]
    free = torch.nonzero(refs <= 0)[:, 0]
    n = min(at.numel(), free.numel())
    refs[free[:n]] = 1
    return at[:n], free[:n], torch.full((1,), at.numel() - n, dtype=torch.int32, device=DEV)


def _fork(s: dict) -> dict:
    ps, refs, prompts = s["case"]["page"], s["refs"].clone(), s["table"].clone()
    P, M = refs.numel(), prompts.shape[1]
    parent = s["parents"].long()
    n = s["lengths"][parent].clamp(0, M * ps)
    whole, at = n // ps, torch.arange(M, device=DEV)
    rows = prompts[parent]
    held = (rows >= 0) & (rows < P)
    shared = held & (at < whole[:, None])
    table = torch.where(shared, rows, torch.full_like(rows, -1))
    refs.index_add_(0, rows[shared].long(), torch.ones_like(rows[shared]))
    ids, fresh, short = _take(refs, held & (at == whole[:, None]) & (n % ps > 0)[:, None])
    table.view(-1)[ids] = fresh.to(torch.int32)
    for t in _pages(s).values():
        _move(t, rows.view(-1)[ids].long(), fresh, (n % ps)[ids // M])
    # the prompts' rows let go
    held = (prompts >= 0) & (prompts < P)
    refs.index_add_(0, prompts[held].long(), torch.full_like(prompts[held], -1))
    prompts.fill_(-1)
    # pages for the new tokens
    want = (s["target"].clamp(min=0) + ps - 1) // ps
    ids, fresh, lacking = _take(refs, (at < want[:, None]) & ((table < 0) | (table >= P)))
    table.view(-1)[ids] = fresh.to(torch.int32)
    return dict(table=table, prompts=prompts, refs=refs, short=short, lacking=lacking, **_pages(s))


def _copy(s: dict) -> dict:
    for t in _pages(s).values():
        _move(t, s["src"].long(), s["dst"].long(), None)
    return _pages(s)


def _compact(s: dict) -> dict:
    refs, table = s["refs"].clone(), s["table"].clone()
    P = refs.numel()
    live = refs > 0
    n = live.sum()
    page = torch.arange(P, device=DEV)
    src, dst = torch.nonzero(live & (page >= n))[:, 0], torch.nonzero(~live & (page < n))[:, 0]
    page[src] = dst
    refs[dst] = refs[src]
    refs[src] = 0
    table = torch.where((table >= 0) & (table < P), page[table.clamp(0, P - 1).long()].to(torch.int32), table)
    for t in _pages(s).values():
        _move(t, src, dst, None)
    return dict(table=table, refs=refs, live=n.to(torch.int32).view(1), **_pages(s))


def _first(hit: torch.Tensor) -> torch.Tensor:
    """The lowest true column of each row."""

    col = torch.arange(hit.shape[-1], device=DEV)
    return torch.where(hit, col, torch.full_like(col, hit.shape[-1])).amin(dim=-1)


def _probs(x: torch.Tensor, heat: float) -> torch.Tensor:
    """Softmax over the last axis of x / heat, the sums in 64 bits."""

    e = torch.exp((x - x.amax(dim=-1, keepdim=True)) / heat)
    return e / e.sum(dim=-1, keepdim=True, dtype=torch.float64)


def _verify(s: dict) -> dict:
    heat, x = s["case"]["temperature"], s["logits"].float()
    B, K1, V = x.shape
    K, drafts, row = K1 - 1, s["drafts"].long(), torch.arange(B, device=DEV)
    step = torch.arange(K, device=DEV)
    number = s.get("number", torch.full((B,), K, dtype=torch.int32, device=DEV)).clamp(0, K)
    if heat > 0:
        p = _probs(x, heat)
        chance = p[:, :K].gather(2, drafts[..., None])[..., 0]
        q = _probs(s["draft_logits"].float(), heat) if "draft_logits" in s else None
        said = 1.0 if q is None else q.gather(2, drafts[..., None])[..., 0]
        good = s["uniforms"].double() * said < chance
    else:
        best = _first(x == x.amax(dim=-1, keepdim=True))
        good = drafts == best[:, :K]
    good = good & (step < number[:, None])
    count = good.long().cumprod(dim=-1).sum(dim=-1)
    if heat > 0:
        last = p[row, count]
        rejected = count < number
        at = count.clamp(max=K - 1)
        if q is None:
            away = torch.zeros_like(last).scatter_(1, drafts[row, at][:, None], 1.0)
            left = last * (1.0 - away)
        else:
            left = (last - q[row, at]).clamp(min=0.0)
        last = torch.where(rejected[:, None], left, last)
        race = last / -torch.log(s["noise"].double())
        drawn = _first(race == race.amax(dim=-1, keepdim=True))
    else:
        drawn = best[row, count]
    slot = torch.arange(K1, device=DEV)
    tokens = torch.cat([drafts, drawn[:, None]], dim=1)
    tokens = torch.where(slot == count[:, None], drawn[:, None], tokens)
    there = slot <= count[:, None]
    logp = x.gather(2, tokens[..., None])[..., 0] - x.amax(dim=-1)
    logp = logp - torch.exp(x - x.amax(dim=-1, keepdim=True)).sum(dim=-1, dtype=torch.float64).log()
    return dict(tokens=torch.where(there, tokens, torch.full_like(tokens, -1)).to(torch.int32), count=count.to(torch.int32),
                logp=torch.where(there, logp, torch.zeros_like(logp)).float())


def _framework():
    """The framework's ``kernels`` and ``kvcache`` modules (its directory's name is no identifier)."""

    name = "gemma4_posttrain_jax_amd"
    if name not in sys.modules:
        where = Path(__file__).resolve().parent.parent / "gemma4-posttrain-jax_amd"
        spec = importlib.util.spec_from_file_location(name, where / "__init__.py", submodule_search_locations=[str(where)])
        module = importlib.util.module_from_spec(spec)
        sys.modules[name] = module
        spec.loader.exec_module(module)
    return [sys.modules.get(f"{name}.{m}") or importlib.import_module(f"{name}.{m}") for m in ("kernels", "kvcache")]


def _call(s: dict):
    kernels, kvcache = _framework()
    case = s["case"]
    if case["kind"] == "packed":
        return kernels.packed_prefill_attention(s["q"], s["key"], s["value"], s["starts"], window=case["window"])
    if case["kind"] == "verify":
        tokens, count, logp = kernels.verify_draft(s["logits"], s["drafts"], s["uniforms"], s["noise"],
                                                   temperature=case["temperature"], draft_logits=s.get("draft_logits"),
                                                   draft_lengths=s.get("number"))
        return dict(tokens=tokens, count=count, logp=logp)
    layers = [kvcache.PagedLayerCache(*x) for x in zip(*(s[n].unbind(0) if n in s else [None] * case["layers"]
                                                         for n in _ARRAYS))]
    if case["kind"] == "copy":
        kernels.paged_copy(layers, s["src"], s["dst"])
        return _pages(s)
    refs, table = s["refs"].clone(), s["table"].clone()
    if case["kind"] == "compact":
        live = kernels.paged_compact(layers, refs, table)
        return dict(table=table, refs=refs, live=live, **_pages(s))
    forked, short = kernels.paged_fork(layers, refs, table, s["parents"], s["lengths"])
    kernels.paged_free(refs, table, s["none"], page_size=case["page"])
    lacking = kernels.paged_reserve(refs, forked, s["target"], page_size=case["page"])
    return dict(table=forked, prompts=table, refs=refs, short=short, lacking=lacking, **_pages(s))


def run(state: dict):
    if own:
        return _call(state)
    return {"packed": _packed, "fork": _fork, "copy": _copy, "compact": _compact, "verify": _verify}[state["case"]["kind"]](state)


def _seen(n: int, window: int) -> int:
    """(query, key) pairs of a causal prompt of n tokens."""

    w = min(n, window) if window else n
    return w * (w + 1) // 2 + (n - w) * w


def work(case: dict) -> dict:
    """Bytes that have to be read and written once, and the operations; a page that several rows copy is read
    once, and of a verification's rows that no draft reaches none are read."""

    if case["kind"] == "packed":
        H, R, D = case["heads"], case["group"], case["dim"]
        lens = _spread(case["lo"], case["hi"], case["seqs"])
        T = max(1, sum(lens) + case["tail"])
        return {"bytes": T * H * D * (4 * R + 4) + 4 * T,
                "flops": 4.0 * sum(_seen(n, case["window"]) for n in lens) * H * R * D}
    if case["kind"] == "verify":
        B, K, V = case["rows"], case["drafts"], case["vocab"]
        size, steps = 2 if case["bf16"] else 4, (case["drafts"] / 2 if case["ragged"] else case["drafts"])
        draw = case["temperature"] > 0
        rows = steps + 1 + (steps if case["draft_logits"] and draw else 0)
        return {"bytes": int(B * V * (rows * size + (4 if draw else 0))), "flops": 3.0 * B * V * rows}
    H, D, ps = case["heads"], case["dim"], case["page"]
    slot = case["layers"] * H * (2 * D * (1 if case["e4m3"] else 2) + (2 if case["e4m3"] else 0))
    if case["kind"] == "copy":
        n = case["parents"] * case["ring"]
        return {"bytes": n * (1 + case["share"]) * ps * slot, "flops": 0}
    if case["kind"] == "fork":
        lens, new, share = _spread(case["lo"], case["hi"], case["prompts"]), case["new"], case["share"]
        width = (case["hi"] + new + ps - 1) // ps
        fresh = sum((n + new + ps - 1) // ps - n // ps for n in lens)
        pages = sum((n + ps - 1) // ps for n in lens) + case["busy"] + share * fresh + case["spare"]
        tables = 4 * width * case["prompts"] * (1 + share)
        return {"bytes": sum(n % ps for n in lens) * (1 + share) * slot + 4 * pages + tables, "flops": 0}
    lens = _spread(case["lo"], case["hi"], case["rows"])
    held = sum((n + ps - 1) // ps for n in lens)
    live, pages = held * (1 - case["ended"]), held + case["spare"]
    moved = live * (pages - live) / pages
    return {"bytes": int(2 * moved * ps * slot + 4 * pages + 4 * case["rows"] * ((case["hi"] + ps - 1) // ps)), "flops": 0}


# --- the operators' definitions in 64 bits -----------------------------------------------------------------


def _exact_packed(case: dict, s: dict):
    T, H, R, D = s["q"].shape
    t, d = torch.arange(T, device=DEV)[:, None], torch.arange(D, device=DEV)[None, :]
    lane = t % 32 // 8 * 4 + t % 4
    key_at = (((t // 32 * (D // 32) + d // 32) * 2 + t % 8 // 4) * 16 + lane) * 32 + d % 32
    value_at = (t // 8 * D + d) * 8 + t % 8
    out = torch.zeros((T, H, R, D), dtype=torch.float64, device=DEV)
    bounds = s["cu"].tolist()
    for h in range(H):
        k = s["key"][0, h].reshape(-1)[key_at].double()
        v = s["value"][0, h].reshape(-1)[value_at].double()
        for a, b in zip(bounds[:-1], bounds[1:]):
            i = torch.arange(b - a, device=DEV)
            hidden = i[None, :] > i[:, None]
            if case["window"]:
                hidden |= i[None, :] <= i[:, None] - case["window"]
            for r in range(R):
                if b > a:
                    w = (s["q"][a:b, h, r].double() @ k[a:b].T).masked_fill_(hidden, -math.inf)
                    out[a:b, h, r] = torch.softmax(w, dim=-1) @ v[a:b]
    return out


def _exact_moves(s: dict, moves: list[tuple[int, int, int]], page: int) -> dict:
    """The arrays in 64 bits after (source, target, slots) of ``moves``, the sources as they were before."""

    out = {}
    for n, t in _pages(s).items():
        out[n] = t.double()
        per = t[0, 0, 0].numel() // page  # elements of a slot and head
        before, after = out[n].clone().view(t.shape[0], t.shape[1], t.shape[2], -1), out[n].view(t.shape[0], t.shape[1], t.shape[2], -1)
        for a, b, slots in moves:
            m = (slots + 31) // 32 * 32 * per
            after[:, b, :, :m] = before[:, a, :, :m]
    return out


def _exact_fork(case: dict, s: dict) -> dict:
    ps, refs, prompts = case["page"], s["refs"].tolist(), s["table"].tolist()
    free = iter([p for p, n in enumerate(refs) if n <= 0])
    children, moves, short, lacking = [], [], 0, 0
    lens = s["lengths"].tolist()
    for a in s["parents"].tolist():
        row, n = prompts[a], lens[a]
        child = [-1] * len(row)
        for e in range(n // ps):
            child[e] = row[e]
            refs[row[e]] += 1
        if n % ps:
            p = next(free, None)
            short += p is None
            if p is not None:
                child[n // ps], refs[p] = p, 1
                moves.append((row[n // ps], p, n % ps))
        children.append(child)
    for row in prompts:
        for p in row:
            if p >= 0:
                refs[p] -= 1
    free = iter([p for p, n in enumerate(refs) if n <= 0])
    for child, n in zip(children, s["target"].tolist()):
        for e in range((n + ps - 1) // ps):
            if child[e] < 0:
                p = next(free, None)
                lacking += p is None
                if p is not None:
                    child[e], refs[p] = p, 1
    whole = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    return dict(table=whole(children), prompts=whole([[-1] * len(r) for r in prompts]), refs=whole(refs),
                short=whole([short]), lacking=whole([lacking]), **_exact_moves(s, moves, ps))


def _exact_compact(case: dict, s: dict) -> dict:
    refs, table = s["refs"].tolist(), s["table"].tolist()
    n = sum(x > 0 for x in refs)
    holes = [p for p in range(n) if refs[p] <= 0]
    moves = list(zip([p for p in range(n, len(refs)) if refs[p] > 0], holes))
    to = dict(moves)
    for a, b in moves:
        refs[a], refs[b] = refs[b], refs[a]
    whole = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    return dict(table=whole([[to.get(p, p) for p in row] for row in table]), refs=whole(refs), live=whole([n]),
                **_exact_moves(s, [(a, b, case["page"]) for a, b in moves], case["page"]))


def _exact_verify(case: dict, s: dict) -> dict:
    B, K, V, heat = case["rows"], case["drafts"], case["vocab"], case["temperature"]
    tokens = torch.full((B, K + 1), -1, dtype=torch.int32, device=DEV)
    logp = torch.zeros((B, K + 1), dtype=torch.float64, device=DEV)
    counts = []
    number = s["number"].tolist() if case["ragged"] else [K] * B
    drafts, u = s["drafts"].tolist(), s["uniforms"].tolist()
    for b in range(B):
        x = s["logits"][b].double()
        policy = torch.log_softmax(x, dim=-1)
        p = torch.softmax(x / heat, dim=-1) if heat > 0 else None
        q = torch.softmax(s["draft_logits"][b].double() / heat, dim=-1) if case["draft_logits"] and heat > 0 else None
        top = [int(torch.nonzero(row == row.max())[0, 0]) for row in x] if p is None else None
        i, token = 0, None
        while i < number[b]:
            d = drafts[b][i]
            if p is None:
                taken = d == top[i]
            else:
                taken = u[b][i] * (1.0 if q is None else float(q[i, d])) < float(p[i, d])
            if not taken:
                break
            tokens[b, i], logp[b, i] = d, policy[i, d]
            i += 1
        if p is None:
            token = top[i]
        else:
            w = p[i].clone()
            if i < number[b]:
                if q is None:
                    w[drafts[b][i]] = 0.0
                else:
                    w = torch.clamp(w - q[i], min=0.0)
            race = w / -torch.log(s["noise"][b].double())
            token = int(torch.nonzero(race == race.max())[0, 0])
        tokens[b, i], logp[b, i] = token, policy[i, token]
        counts.append(i)
    return dict(tokens=tokens, count=torch.tensor(counts, dtype=torch.int32, device=DEV), logp=logp)


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["kind"] == "copy":
        moves = [(a, b, case["page"]) for a, b in zip(s["src"].tolist(), s["dst"].tolist())]
        return _exact_moves(s, moves, case["page"])
    return {"packed": _exact_packed, "fork": _exact_fork, "compact": _exact_compact,
            "verify": _exact_verify}[case["kind"]](case, s)
