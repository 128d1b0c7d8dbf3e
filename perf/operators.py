"""The paged KV cache's operators, case by case: what a program that serves Gemma 4 rollouts from pages
has this framework do.

Kinds of case:
- ``attend``: one new token per row over its pages (``kernels.paged_decode_attention``);
- ``append``: the norms and rotation of a step's or a prompt chunk's q / k / v and the write of k / v into
  the pages, quantised where the pages hold e4m3 (``kernels.paged_append``);
- ``read``: the pages back as token-major bf16 rows (``kernels.paged_read``).

The cache of one layer: ``key [P, H, page / 32, D / KR, 2, 16, KR]`` and ``value [P, H, page / 8, D, 8]``, the
operand order of the framework's attention kernels (slot 8 a + 4 b + c of a 32-slot chunk is half b, lane
4 a + c of a key run of KR dims, KR = min(D, 32) in bf16 and 64 in e4m3; values in groups of 8 slots). e4m3
pages have a power-of-two scale per slot and head, ``key_scale`` / ``value_scale [P, H, page]`` (e8m0).
Position p of row b is slot p % page of page ``page_table[b, p / page]``.

The plain forms are elementary torch operations in 32 bits; ``exact`` restates each operator in 64 bits,
row by row, with the places in a page computed by the layout's formula.
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
EPS = 1e-6
MIN_EXP, MAX_EXP = -100, 120  # the range of a scale's exponent


def listed() -> list[dict]:
    return [
        # one interactive sequence, a sliding layer: the launches' latency
        dict(name="attend_single", kind="attend", batch=1, heads=2, group=4, dim=256, page=64, e4m3=False, window=512,
             lo=701, hi=701, share=1, prompt=0),
        # the benchmark's sliding-window decode batch: 64 rows past their window
        dict(name="attend_window", kind="attend", batch=64, heads=2, group=4, dim=256, page=64, e4m3=True, window=512,
             lo=1536, hi=2047, share=1, prompt=0),
        # a global layer of the rollout batch, prompts of 200 and more and their completions, small pages
        dict(name="attend_rollout", kind="attend", batch=256, heads=2, group=4, dim=256, page=32, e4m3=False, window=0,
             lo=200, hi=767, share=1, prompt=0),
        # 8 prompts with 8 completions each, which share their prompt's pages
        dict(name="attend_group", kind="attend", batch=64, heads=2, group=4, dim=256, page=64, e4m3=True, window=0,
             lo=4100, hi=4611, share=8, prompt=4096),
        # the benchmark's long-context decode: ragged rows of up to 32768 positions, in bf16 and in e4m3
        dict(name="attend_long", kind="attend", batch=16, heads=2, group=4, dim=256, page=128, e4m3=False, window=0,
             lo=1024, hi=32768, share=1, prompt=0),
        dict(name="attend_long_e4m3", kind="attend", batch=16, heads=2, group=4, dim=256, page=128, e4m3=True,
             window=0, lo=1024, hi=32768, share=1, prompt=0),
        # a stock configuration's global layer (head dim 512), an odd batch, lengths from one token on
        dict(name="attend_wide", kind="attend", batch=7, heads=1, group=8, dim=512, page=64, e4m3=True, window=0, lo=1,
             hi=5001, share=1, prompt=0),
        # the new tokens of a step of the rollout batch
        dict(name="append_step", kind="append", batch=256, seq=1, heads=2, group=4, dim=256, page=64, e4m3=True,
             start=512, pad=256, keep=0),
        # the rollout batch's left-padded prompts, one layer
        dict(name="append_prompt", kind="append", batch=256, seq=256, heads=2, group=4, dim=256, page=64, e4m3=True,
             start=0, pad=192, keep=0),
        # long prompts into a sliding layer's pages, which keep the window only; odd sizes, bf16
        dict(name="append_window", kind="append", batch=11, seq=1999, heads=1, group=8, dim=128, page=32, e4m3=False,
             start=0, pad=1500, keep=512),
        # the pages of a few long prompts, read back for another consumer
        dict(name="read_prompt", kind="read", batch=16, heads=2, dim=256, page=64, e4m3=True, lo=2048, hi=8191, start=0,
             count=8191),
        # a short stretch out of the middle of a few rows
        dict(name="read_stretch", kind="read", batch=5, heads=2, dim=512, page=32, e4m3=False, lo=90, hi=500, start=37,
             count=100),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def draw(rng) -> dict:
    kind = rng.choices(["attend", "append", "read"], [5, 3, 2])[0]
    heads, dim, page, e4m3 = rng.choice([1, 2, 3, 4]), rng.choice([64, 128, 256, 512]), rng.choice([32, 64, 128, 256]), \
        rng.random() < 0.6
    if kind == "attend":
        hi = _log_int(rng, 1, 32768)
        most = (16 * 32768 * 2 * 256) // (max(hi, 64) * heads * dim)  # values in the keys of one layer
        batch = _log_int(rng, 1, max(1, min(512, most)))
        share = rng.choice([1, 1, 2, 5])
        lo = rng.randint(0, hi)
        return dict(kind=kind, batch=batch, heads=heads, group=rng.choice([1, 2, 3, 4, 8, 16]), dim=dim, page=page,
                    e4m3=e4m3, window=rng.choice([0, 0, 512, rng.randint(1, 2048)]), lo=lo, hi=hi, share=share,
                    prompt=lo // page * page if share > 1 else 0)
    if kind == "append":
        seq = rng.choice([1, 1, _log_int(rng, 2, 4096), _log_int(rng, 2, 4096)])
        group = rng.choice([1, 2, 3, 4, 8])
        start = rng.choice([0, rng.randint(1, 4096)])
        most = min((256 * 256 * 2 * 6 * 256) // (seq * heads * (group + 2) * dim),
                   (16 * 16384 * 2 * 256) // ((start + seq) * heads * dim))
        keep = rng.choice([0, 0, 512, 100]) if seq > 1 else 0
        return dict(kind=kind, batch=_log_int(rng, 1, max(1, min(512, most))), seq=seq, heads=heads, group=group,
                    dim=dim, page=page, e4m3=e4m3, start=start,
                    pad=rng.choice([0, seq // 2, seq]) if seq > 1 else rng.choice([0, 64]), keep=keep)
    count = _log_int(rng, 1, 8192)
    most = (16 * 8191 * 2 * 256) // (count * heads * dim)
    start = rng.choice([0, rng.randint(0, 2 * count)])
    hi = start + rng.randint(1, 2 * count)
    return dict(kind=kind, batch=_log_int(rng, 1, max(1, min(256, most // 2))), heads=heads, dim=dim, page=page, e4m3=e4m3,
                lo=rng.randint(0, hi), hi=hi, start=start, count=count)


# --- what a program has in hand ------------------------------------------------------------------------


def _lengths(case: dict) -> list[int]:
    """The rows' lengths: spread evenly over [lo, hi], the longest first."""

    n = case["batch"]
    return [case["hi"] - (case["hi"] - case["lo"]) * i // max(1, n - 1) for i in range(n)]


def _pads(case: dict) -> list[int]:
    n = case["batch"]
    return [case["pad"] * i // max(1, n - 1) for i in range(n)]


def _key_run(dim: int, e4m3: bool) -> int:
    return min(dim, 64 if e4m3 else 32)


def _pages(rows: list[int], width: int, share: int, shared: int, g: torch.Generator) -> tuple[int, torch.Tensor]:
    """The number of pages and a table ``[B, width]``: row b has ``rows[b]`` pages of its own in any order, the
    first ``shared`` of them in common with the other rows of its group of ``share``; -1 beyond."""

    ids, used = [], 0
    for b, n in enumerate(rows):
        head = ids[b - 1][:shared] if b % share else list(range(used, used + min(n, shared)))
        used += 0 if b % share else len(head)
        head = head[:n]
        ids.append(head + list(range(used, used + n - len(head))))
        used += n - len(head)
    table = torch.full((len(rows), width), -1, dtype=torch.int64)
    for b, row in enumerate(ids):
        table[b, :len(row)] = torch.tensor(row, dtype=torch.int64)
    pages = used + 3  # a few that no row has
    order = torch.randperm(pages, generator=g, device=DEV)
    table = table.to(DEV)
    return pages, torch.where(table >= 0, order[table.clamp(min=0)], table).to(torch.int32)


def _quantise(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """f32 vectors ``[..., D]`` to e4m3 and the power of two that each is divided by first: the least with
    max |x| / 2^e <= 448."""

    frac, exp = torch.frexp(x.abs().amax(dim=-1))
    e = torch.where(frac <= 0.875, exp - 9, exp - 8).clamp(MIN_EXP, MAX_EXP)
    return torch.ldexp(x, -e[..., None]).to(F8), (e + 127).to(torch.uint8).view(E8)


def _cache(case: dict, pages: int, g: torch.Generator, empty: bool = False) -> dict:
    H, D, ps, e4m3 = case["heads"], case["dim"], case["page"], case["e4m3"]
    kr = _key_run(D, e4m3)
    key, value = (pages, H, ps // 32, D // kr, 2, 16, kr), (pages, H, ps // 8, D, 8)
    if empty:
        if not e4m3:
            return dict(key=torch.zeros(key, dtype=BF16, device=DEV), value=torch.zeros(value, dtype=BF16, device=DEV))
        byte = lambda shape: torch.zeros(shape, dtype=torch.uint8, device=DEV)  # noqa: E731
        return dict(key=byte(key).view(F8), value=byte(value).view(F8),
                    key_scale=byte((pages, H, ps)).view(E8), value_scale=byte((pages, H, ps)).view(E8))
    # keys as normed and rotated rows have them, values of order 1; a token's size varies
    s = {}
    for name, shape in (("key", key), ("value", value)):
        x = torch.empty((pages, H, ps, D), dtype=BF16, device=DEV).normal_(0.0, 1.0, generator=g)
        x *= torch.empty((pages, H, ps, 1), dtype=BF16, device=DEV).uniform_(0.7, 1.4, generator=g)
        if e4m3:
            q, scale = _quantise(x.float())
            x = q.view(torch.uint8)
            s[name + "_scale"] = scale
        if name == "key":
            x = x.view(pages, H, ps // 32, 4, 2, 4, D // kr, kr).permute(0, 1, 2, 6, 4, 3, 5, 7)
        else:
            x = x.view(pages, H, ps // 8, 8, D).transpose(3, 4)
        x = x.reshape(shape).contiguous()
        s[name] = x.view(F8) if e4m3 else x
    return s


def _shuffled(values: list[int], g: torch.Generator) -> torch.Tensor:
    t = torch.tensor(values, dtype=torch.int32, device=DEV)
    return t[torch.randperm(len(values), generator=g, device=DEV)]


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEV).manual_seed(seed)
    B, H, D, ps = case["batch"], case["heads"], case["dim"], case["page"]
    s = {"case": case}
    if case["kind"] in ("attend", "read"):
        s["lengths"] = _shuffled(_lengths(case), g)
        shared = case.get("prompt", 0) // ps
        rows = [(n + ps - 1) // ps for n in s["lengths"].tolist()]
        pages, s["table"] = _pages(rows, max(1, max(rows)), case.get("share", 1), shared, g)
        s.update(_cache(case, pages, g))
        if case["kind"] == "attend":
            # scores with a deviation of about 2, as trained norms of q and k give
            s["q"] = torch.empty((B, H, case["group"], D), dtype=BF16, device=DEV).normal_(0.0, 2.0 / math.sqrt(D), generator=g)
        return s
    S, R = case["seq"], case["group"]
    pads = _shuffled(_pads(case), g)
    s["write_pos"] = case["start"] - pads  # position of each row's token 0; a pad's is below 0
    top = case["start"] + S
    width = (top + ps - 1) // ps
    if case["keep"]:  # a sliding layer's pages, taken in turn
        own_pages = (case["keep"] + ps - 1) // ps + 1
        pages, table = _pages([own_pages] * B, own_pages, 1, 0, g)
        s["table"] = table[:, torch.arange(width, device=DEV) % own_pages].contiguous()
    else:
        pages, s["table"] = _pages([width] * B, width, 1, 0, g)
    s.update(_cache(case, pages, g, empty=True))
    rows = torch.empty((B, S, (R + 2) * H * D), dtype=BF16, device=DEV).normal_(generator=g)  # the projections' output
    s["q"], s["k"], s["v"] = rows[..., : H * R * D].view(B, S, H, R, D), \
        rows[..., H * R * D: H * (R + 1) * D].view(B, S, H, D), rows[..., H * (R + 1) * D:].view(B, S, H, D)
    weight = lambda: (D ** -0.25 * torch.empty(D, device=DEV).normal_(1.0, 0.1, generator=g)).to(BF16)  # noqa: E731
    s["qw"], s["kw"] = weight(), weight()
    pos = (s["write_pos"][:, None] + torch.arange(S, device=DEV)).clamp(min=0).double()
    angle = pos[..., None] * 1e4 ** (-torch.arange(0, D, 2, dtype=torch.float64, device=DEV) / D)
    s["cos"], s["sin"] = (torch.cat([f(angle)] * 2, dim=-1).float() for f in (torch.cos, torch.sin))
    return s


# --- one pass --------------------------------------------------------------------------------------------


def _key_tokens(key: torch.Tensor) -> torch.Tensor:
    """A view of ``key [P, H, C, N, 2, 16, KR]`` by page, chunk, slot (a, b, c), head and dims (N, KR)."""

    P, H, C, N, _, _, kr = key.shape
    return key.view(P, H, C, N, 2, 4, 4, kr).permute(0, 2, 5, 4, 6, 1, 3, 7)


def _f32(payload: torch.Tensor, scale: torch.Tensor | None) -> torch.Tensor:
    return payload.float() if scale is None else payload.view(F8).float() * scale.view(E8).float()[..., None]


def _bytes(t: torch.Tensor) -> torch.Tensor:
    return t if t.dtype == BF16 else t.view(torch.uint8)


def _gather(s: dict, pages: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The f32 keys and values ``[B, n * page, H, D]`` of ``pages [B, n]``."""

    B, n = pages.shape
    H, D, ps = s["key"].shape[1], s["value"].shape[3], s["value"].shape[2] * 8
    k = _key_tokens(_bytes(s["key"]))[pages].reshape(B, n * ps, H, D)
    v = _bytes(s["value"])[pages].permute(0, 1, 3, 5, 2, 4).reshape(B, n * ps, H, D)
    if "key_scale" not in s:
        return k.float(), v.float()
    ks, vs = (_bytes(s[x])[pages].transpose(2, 3).reshape(B, n * ps, H) for x in ("key_scale", "value_scale"))
    return _f32(k, ks), _f32(v, vs)


def _attend(s: dict) -> torch.Tensor:
    ps, window, table, n = s["case"]["page"], s["case"]["window"], s["table"], s["lengths"][:, None]
    first, width = torch.zeros_like(n), table.shape[1]
    if window:  # the pages that the window of each row touches
        first = (n - window).clamp(min=0) // ps
        width = min(width, (window + ps - 1) // ps + 1)
    at = (first + torch.arange(width, device=table.device)).clamp(max=table.shape[1] - 1).long()
    k, v = _gather(s, table.gather(1, at).clamp(min=0).long())
    pos = first * ps + torch.arange(width * ps, device=table.device)
    valid = pos < n
    if window:
        valid &= pos >= n - window
    scores = torch.matmul(s["q"].float(), k.permute(0, 2, 3, 1))  # [B, H, R, L]
    scores = torch.where(valid[:, None, None, :], scores, torch.full_like(scores, -math.inf))
    p = torch.exp(scores - scores.amax(dim=-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min))
    total = p.sum(dim=-1, keepdim=True)
    out = torch.matmul(p, v.permute(0, 2, 1, 3)) / torch.where(total > 0, total, torch.ones_like(total))
    return out.to(BF16)


def _rms(x: torch.Tensor, w: torch.Tensor | None) -> torch.Tensor:
    x = x.float()
    y = x * torch.rsqrt(x.square().mean(dim=-1, keepdim=True) + EPS)
    return y if w is None else y * w.float()


def _rotate(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    half = x.shape[-1] // 2
    return x * cos + torch.cat([-x[..., half:], x[..., :half]], dim=-1) * sin


def _append(s: dict) -> dict:
    S, ps, keep = s["case"]["seq"], s["case"]["page"], s["case"]["keep"]
    cos, sin = s["cos"][:, :, None], s["sin"][:, :, None]
    q = _rotate(_rms(s["q"], s["qw"]), cos[..., None, :], sin[..., None, :]).to(BF16)
    k, v = _rotate(_rms(s["k"], s["kw"]), cos, sin), _rms(s["v"], None)
    i = torch.arange(S, device=k.device)
    pos = s["write_pos"][:, None].long() + i
    stored = (pos >= 0) & (i >= S - (keep or S))
    row, tok = torch.nonzero(stored, as_tuple=True)
    p = pos[row, tok]
    page, slot = s["table"][row, p // ps].long(), p % ps
    out = {"q": q, "key": s["key"], "value": s["value"]}
    kt, vt = k[row, tok], v[row, tok]  # [n, H, D]
    if s["case"]["e4m3"]:
        (kt, ks), (vt, vs) = _quantise(kt), _quantise(vt)
        kt, vt = kt.view(torch.uint8), vt.view(torch.uint8)
        _bytes(s["key_scale"]).transpose(1, 2)[page, slot] = ks.view(torch.uint8)
        _bytes(s["value_scale"]).transpose(1, 2)[page, slot] = vs.view(torch.uint8)
        out.update(key_scale=s["key_scale"], value_scale=s["value_scale"])
    rows = _key_tokens(_bytes(s["key"]))
    r = slot % 32
    rows[page, slot // 32, r // 8, r // 4 % 2, r % 4] = kt.to(rows.dtype).view(-1, rows.shape[5], rows.shape[6], rows.shape[7])
    cols = _bytes(s["value"]).permute(0, 2, 4, 1, 3)
    cols[page, slot // 8, slot % 8] = vt.to(cols.dtype)
    return out


def _read(s: dict) -> list[torch.Tensor]:
    ps, start, count = s["case"]["page"], s["case"]["start"], s["case"]["count"]
    pos = start + torch.arange(count, device=DEV)
    first, last = start // ps, (start + count - 1) // ps
    width = s["table"].shape[1]
    pages = s["table"][:, torch.arange(first, last + 1, device=DEV).clamp(max=width - 1)].clamp(min=0).long()
    there = (pos[None, :] < s["lengths"][:, None])[:, :, None, None]
    at = start - first * ps
    return [torch.where(there, x[:, at: at + count], torch.zeros((), device=DEV)).to(BF16) for x in _gather(s, pages)]


def _framework():
    """The framework's ``kernels``, ``kvcache`` and ``_lib`` modules (its directory's name is no identifier)."""

    name = "gemma4_posttrain_jax_amd"
    if name not in sys.modules:
        where = Path(__file__).resolve().parent.parent / "gemma4-posttrain-jax_amd"
        spec = importlib.util.spec_from_file_location(name, where / "__init__.py", submodule_search_locations=[str(where)])
        module = importlib.util.module_from_spec(spec)
        sys.modules[name] = module
        spec.loader.exec_module(module)
    return [sys.modules.get(f"{name}.{m}") or importlib.import_module(f"{name}.{m}") for m in ("kernels", "kvcache", "_lib")]


def _call(s: dict):
    kernels, kvcache, lib = _framework()
    case = s["case"]
    layer = kvcache.PagedLayerCache(s["key"], s["value"], s.get("key_scale"), s.get("value_scale"))
    if case["kind"] == "attend":
        return kernels.paged_decode_attention(layer, s["q"], page_table=s["table"], lengths=s["lengths"],
                                              window=case["window"])
    if case["kind"] == "read":
        return list(kernels.paged_read(layer, page_table=s["table"], lengths=s["lengths"], start=case["start"],
                                       count=case["count"]))
    flags = (lib.G4_APPEND_NORM_Q | lib.G4_APPEND_ROPE_Q | lib.G4_APPEND_NORM_K | lib.G4_APPEND_ROPE_K
             | lib.G4_APPEND_NORM_V)
    q = torch.empty(s["q"].shape, dtype=BF16, device=DEV)
    kernels.paged_append(layer, s["k"], s["v"], page_table=s["table"], write_pos=s["write_pos"], keep=case["keep"],
                         flags=flags, eps=EPS, q=s["q"], q_out=q, q_norm_weight=s["qw"], k_norm_weight=s["kw"],
                         rope_cos=s["cos"], rope_sin=s["sin"])
    out = {"q": q, "key": layer.key, "value": layer.value}
    if case["e4m3"]:
        out.update(key_scale=layer.key_scale, value_scale=layer.value_scale)
    return out


def run(state: dict):
    if own:
        return _call(state)
    return {"attend": _attend, "append": _append, "read": _read}[state["case"]["kind"]](state)


def work(case: dict) -> dict:
    """Bytes that have to be read and written once, and the operations; pages that rows share are read once."""

    B, H, D, ps = case["batch"], case["heads"], case["dim"], case["page"]
    size = H * (2 * D * (1 if case["e4m3"] else 2) + (2 if case["e4m3"] else 0))  # one position's K and V
    if case["kind"] == "attend":
        keys = [min(n, case["window"] or n) for n in _lengths(case)]
        R, rows = case["group"], B * H * case["group"] * D
        alone = sum(keys)
        if case["share"] > 1 and not case["window"]:  # the shared pages count for the first row of a group
            alone -= sum(min(n, case["prompt"] // ps * ps) for i, n in enumerate(keys) if i % case["share"])
        return {"bytes": alone * size + 4 * rows, "flops": 4.0 * sum(keys) * H * R * D}
    if case["kind"] == "read":
        there = sum(max(0, min(n - case["start"], case["count"])) for n in _lengths(case))
        return {"bytes": there * size + B * case["count"] * H * D * 4, "flops": 0}
    S, R = case["seq"], case["group"]
    kept = 0
    for pad in _pads(case):
        first = max(0, S - case["keep"] if case["keep"] else 0, pad - case["start"])
        kept += max(0, S - first)
    return {"bytes": B * S * (H * R * D * 4 + D * 8) + kept * (H * D * 4 + size),
            "flops": 8.0 * (B * S * H * R + 2 * kept * H) * D}


# --- the operators' definitions in 64 bits -----------------------------------------------------------------


def _places(case: dict, table: torch.Tensor, b: int, pos: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Offsets of the keys, values ``[n, H, D]`` and scales ``[n, H]`` of row b's positions in the cache's arrays."""

    H, D, ps = case["heads"], case["dim"], case["page"]
    kr = _key_run(D, case["e4m3"])
    h, d = torch.arange(H, device=DEV)[None, :, None], torch.arange(D, device=DEV)[None, None, :]
    slot = (pos % ps)[:, None, None]
    head = table[b].long()[pos // ps][:, None, None] * H + h
    lane = slot % 32 // 8 * 4 + slot % 4
    key = (((slot // 32 * (D // kr) + d // kr) * 2 + slot % 8 // 4) * 16 + lane) * kr + d % kr
    value = (slot // 8 * D + d) * 8 + slot % 8
    return head * (ps * D) + key, head * (ps * D) + value, (head * ps + slot)[..., 0]


def _values(s: dict, name: str, at: torch.Tensor, scale_at: torch.Tensor) -> torch.Tensor:
    if not s["case"]["e4m3"]:
        return s[name].view(-1)[at].double()
    exps = s[name + "_scale"].view(torch.uint8).view(-1)[scale_at].double() - 127
    return s[name].view(torch.uint8).view(-1)[at].view(F8).double() * torch.exp2(exps)[..., None]


def _to_e4m3(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The values of ``x [n, H, D]`` (f64) in e4m3 after division by each vector's scale, and the scales."""

    top = x.abs().amax(dim=-1)
    e = torch.ceil(torch.log2(top / 448)).clamp(MIN_EXP, MAX_EXP)
    e = torch.where(top > 0, e, torch.full_like(e, MIN_EXP))
    y = x / torch.exp2(e)[..., None]
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step, torch.exp2(e)


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    B, H, D, ps = case["batch"], case["heads"], case["dim"], case["page"]
    if case["kind"] == "append":
        S, R = case["seq"], case["group"]
        half = D // 2
        out = {"q": torch.empty((B, S, H, R, D), dtype=torch.float64, device=DEV),
               "key": s["key"].double(), "value": s["value"].double()}
        if case["e4m3"]:
            out.update({n: s[n].double() for n in ("key_scale", "value_scale")})
        for b in range(B):
            c, n = s["cos"][b].double(), s["sin"][b].double()

            def turn(x, b=b, c=c, n=n):  # [S, heads, D], pairs (d, d + D / 2)
                x1, x2 = x[..., :half], x[..., half:]
                c1, c2, n1, n2 = c[:, None, :half], c[:, None, half:], n[:, None, :half], n[:, None, half:]
                return torch.cat([x1 * c1 - x2 * n1, x2 * c2 + x1 * n2], dim=-1)

            norm = lambda x: x / (x.square().sum(dim=-1, keepdim=True) / D + EPS).sqrt()  # noqa: E731
            out["q"][b] = turn(norm(s["q"][b].double().reshape(S, H * R, D)) * s["qw"].double()).view(S, H, R, D)
            k, v = turn(norm(s["k"][b].double()) * s["kw"].double()), norm(s["v"][b].double())
            p0 = int(s["write_pos"][b])
            first = max(0, -p0, S - case["keep"] if case["keep"] else 0)
            if first >= S:
                continue
            ka, va, sa = _places(case, s["table"], b, p0 + torch.arange(first, S, device=DEV))
            for name, x, at in (("key", k[first:], ka), ("value", v[first:], va)):
                if case["e4m3"]:
                    x, scale = _to_e4m3(x)
                    out[name + "_scale"].view(-1)[sa] = scale
                out[name].view(-1)[at] = x
        return out
    if case["kind"] == "read":
        outs = [torch.zeros((B, case["count"], H, D), dtype=torch.float64, device=DEV) for _ in range(2)]
        for b, n in enumerate(s["lengths"].tolist()):
            pos = case["start"] + torch.arange(max(0, min(n - case["start"], case["count"])), device=DEV)
            if len(pos):
                ka, va, sa = _places(case, s["table"], b, pos)
                for x, name, at in zip(outs, ("key", "value"), (ka, va)):
                    x[b, : len(pos)] = _values(s, name, at, sa)
        return outs
    out = torch.zeros((B, H, case["group"], D), dtype=torch.float64, device=DEV)
    for b, n in enumerate(s["lengths"].tolist()):
        first = max(0, n - case["window"]) if case["window"] else 0
        if n == 0:
            continue
        ka, va, sa = _places(case, s["table"], b, torch.arange(first, n, device=DEV))
        k, v = _values(s, "key", ka, sa), _values(s, "value", va, sa)
        for h in range(H):
            p = torch.softmax(s["q"][b, h].double() @ k[:, h].T.contiguous(), dim=-1)
            out[b, h] = p @ v[:, h].contiguous()
    return out
