"""The paged KV cache on the GPU: append, one-token attention and read-back against plain 64-bit
restatements, with bounds that count the roundings."""

from __future__ import annotations

import math

import pytest
import torch

import paged_util as P
from gemma4_posttrain_jax_amd import kernels
from gemma4_posttrain_jax_amd._lib import G4Error
from gemma4_posttrain_jax_amd.kvcache import new_paged_layer

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _randn(seed: int, *shape, scale: float = 1.0) -> torch.Tensor:
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(BF16)


def _i32(values, device) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device=device)


def _same(a: torch.Tensor, b: torch.Tensor) -> None:
    torch.testing.assert_close(a.cpu().double(), b.cpu().double(), rtol=0, atol=0, equal_nan=True)


# --- append -------------------------------------------------------------------------------------------------


def _stored(B, S, write_pos, table, ps, pages, keep):
    """(row, token, page, slot) of every token that an append stores."""

    for b in range(B):
        for s in range(S):
            p = write_pos[b] + s
            if p < 0 or p >= table.shape[1] * ps or (keep and s < S - keep):
                continue
            page = int(table[b, p // ps])
            if 0 <= page < pages:
                yield b, s, page, p % ps


APPENDS = [  # e4m3, D, H, page, S, write_pos, keep
    (False, 64, 1, 32, 1, [0], 0),
    (True, 64, 3, 32, 1, [31, -1, 64], 0),
    (True, 256, 2, 64, 1, [63, 64, 200, 7], 0),
    (False, 512, 1, 128, 1, [5, 127], 0),
    (True, 512, 1, 32, 2, [31, -1], 0),
    (False, 128, 2, 32, 7, [0, 29], 0),
    (True, 128, 2, 32, 8, [8, -3], 0),
    (True, 256, 1, 64, 37, [-36, -37, -40, 0, 91], 0),
    (False, 256, 2, 64, 65, [3, -8], 0),
    (True, 64, 2, 256, 300, [0, -111], 0),
    (True, 128, 1, 32, 90, [0, 17], 40),
    (False, 512, 1, 32, 41, [-5, 64], 33),
    (True, 512, 2, 32, 33, [2147483600, -2147483648], 0),
]


@pytest.mark.parametrize("e4m3,D,H,ps,S,write_pos,keep", APPENDS)
def test_append_moves_and_quantises_exactly(device, e4m3, D, H, ps, S, write_pos, keep):
    """Without preparation the append only moves (bf16) or quantises (e4m3): equal to the reference bit by
    bit, and every other slot as it was."""

    B = len(write_pos)
    M = max(2, (min(max(write_pos), 1000) + S + ps - 1) // ps)
    pages = B * M + 2
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(1))[: B * M].view(B, M).to(torch.int32)
    table[0, 1] = -1
    table[-1, M - 1] = pages  # one past the last
    rows = _randn(2, B, S, 2 * H * D + 8, scale=3.0)  # a row stride of its own
    k, v = rows[..., : H * D].view(B, S, H, D), rows[..., H * D: 2 * H * D].view(B, S, H, D)
    before_k, before_v = _randn(3, pages, H, ps, D), _randn(4, pages, H, ps, D)
    layer = P.filled(pages, H, D, ps, e4m3, before_k, before_v, device)
    want_k, want_v = P.slots_of(layer)
    for b, s, page, slot in _stored(B, S, write_pos, table, ps, pages, keep):
        want_k[page, :, slot] = P.dequantised(k[b, s]) if e4m3 else k[b, s].double()
        want_v[page, :, slot] = P.dequantised(v[b, s]) if e4m3 else v[b, s].double()
    dev = rows.to(device)
    kernels.paged_append(layer, dev[..., : H * D].view(B, S, H, D), dev[..., H * D: 2 * H * D].view(B, S, H, D),
                         page_table=table.to(device), write_pos=_i32(write_pos, device), keep=keep)
    got_k, got_v = P.slots_of(layer)
    _same(got_k, want_k)
    _same(got_v, want_v)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("D,S", [(64, 1), (128, 9), (256, 17), (512, 3), (512, 8)])
def test_append_of_rows_at_any_offset(device, e4m3, D, S):
    """Rows, weights and table rows that start anywhere: an odd row stride, an odd first element, a table cut out of a
    wider one; the same bits as aligned copies."""

    H, R, B, ps = 3, 2, 2, 32
    wide = _randn(2, B, S, (R + 2) * H * D + 5).to(device)[..., 1:-2]
    wide = wide.as_strided((B, S, (R + 2) * H * D), wide.stride(), wide.storage_offset())
    weights = _randn(3, 2 * D + 3).to(device)
    angle = torch.rand((B, S, D), generator=torch.Generator().manual_seed(4)).to(device)
    tables = torch.arange(2 * 8, dtype=torch.int32, device=device).view(2, 8)

    def run(rows, qw, kw, table):
        layer = new_paged_layer(16, H, D, ps, e4m3=e4m3, device=device)
        q_out = torch.empty((B, S, H, R, D), dtype=BF16, device=device)
        kernels.paged_append(layer, rows[..., H * R * D: H * (R + 1) * D].unflatten(-1, (H, D)),
                             rows[..., H * (R + 1) * D: H * (R + 2) * D].unflatten(-1, (H, D)), page_table=table,
                             write_pos=_i32([3, 30], device), flags=P.ALL_FLAGS,
                             q=rows[..., : H * R * D].unflatten(-1, (H, R, D)), q_out=q_out, q_norm_weight=qw,
                             k_norm_weight=kw, rope_cos=angle.cos(), rope_sin=angle.sin())
        return [q_out] + [x.view(torch.uint8) for x in layer if x is not None]

    got = run(wide, weights[1: D + 1], weights[D + 3:], tables[:, 2:5])
    want = run(wide.contiguous(), weights[1: D + 1].clone(), weights[D + 3:].clone(), tables[:, 2:5].contiguous())
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    n = _i32([3 + S, 30 + S], device)
    layer = new_paged_layer(16, H, D, ps, e4m3=e4m3, device=device)
    with pytest.raises(G4Error, match="aligned"):
        q = torch.empty(B * H * R * D + 1, dtype=BF16, device=device)[1:].view(B, H, R, D)
        kernels.paged_decode_attention(layer, q, page_table=tables[:, 2:5], lengths=n)


def test_append_quantises_every_bf16_value(device):
    """All 65536 bf16 bit patterns, infinities and NaN among them, beside small and large neighbours."""

    D, S = 64, 1024
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(BF16)
    k = bits.view(1, S, 1, D)  # neighbours in one vector: equal sign and exponent
    v = bits[torch.randperm(65536, generator=torch.Generator().manual_seed(0))].view(1, S, 1, D)  # any exponents
    layer = new_paged_layer(S // 32, 1, D, 32, e4m3=True, device=device)
    table = torch.arange(S // 32, dtype=torch.int32, device=device)[None]
    kernels.paged_append(layer, k.to(device), v.to(device), page_table=table, write_pos=_i32([0], device))
    got = P.slots_of(layer)
    for x, g, name in ((k, got[0], "key"), (v, got[1], "value")):
        y, e = P.to_e4m3(x[0, :, 0])
        scale = getattr(layer, name + "_scale").cpu().view(torch.uint8).view(S).long()
        assert torch.equal(scale, e.long() + 127)
        _same(g.reshape(S, D), y * torch.exp2(e.double())[:, None])


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("D,H,R,S,pads", [(64, 1, 1, 1, [0]), (128, 2, 3, 5, [0, 2]), (256, 2, 4, 1, [0, 0, 1]),
                                          (256, 2, 4, 19, [0, 18, 19]), (512, 1, 16, 33, [7, 0]), (64, 4, 8, 40, [1, 0])])
def test_append_prepares_q_k_v(device, e4m3, D, H, R, S, pads):
    B, ps, eps = len(pads), 32, 1e-6
    M = (S + ps - 1) // ps
    rows = _randn(5, B, S, (R + 2) * H * D, scale=2.0)
    qw, kw = _randn(6, D).abs() + 0.5, _randn(7, D).abs() + 0.5
    angle = torch.rand((B, S, D // 2), generator=torch.Generator().manual_seed(8)) * 50
    cos, sin = (torch.cat([f(angle)] * 2, dim=-1) for f in (torch.cos, torch.sin))
    table = torch.arange(B * M, dtype=torch.int32).view(B, M)
    layer = new_paged_layer(B * M, H, D, ps, e4m3=e4m3, device=device)
    dev = rows.to(device)

    def views(t):
        return (t[..., : H * R * D].view(B, S, H, R, D), t[..., H * R * D: H * (R + 1) * D].view(B, S, H, D),
                t[..., H * (R + 1) * D:].view(B, S, H, D))

    q, k, v = views(dev)
    q_out = torch.full((B, S, H, R, D), math.nan, dtype=BF16, device=device)
    kernels.paged_append(layer, k, v, page_table=table.to(device), write_pos=_i32([-p for p in pads], device),
                         flags=P.ALL_FLAGS, eps=eps, q=q, q_out=q_out, q_norm_weight=qw.to(device),
                         k_norm_weight=kw.to(device), rope_cos=cos.to(device), rope_sin=sin.to(device))
    q, k, v = views(rows)
    want, err = P.prepared(q, qw, True, (cos[:, :, None, None], sin[:, :, None, None]), eps)
    off = (q_out.cpu().double() - want).abs()
    assert (off <= P.U_BF16 * want.abs() + (1 + P.U_BF16) * err).all()
    got_k, got_v = P.slots_of(layer)
    for x, w, rope, got in ((k, kw, (cos[:, :, None], sin[:, :, None]), got_k), (v, None, None, got_v)):
        want, err = P.prepared(x, w, True, rope, eps)
        seen = torch.zeros(got.shape[0], got.shape[2], dtype=torch.bool)
        for b, s, page, slot in _stored(B, S, [-p for p in pads], table, ps, B * M, 0):
            seen[page, slot] = True
            y, dy = want[b, s], err[b, s]
            off = (got[page, :, slot] - y).abs()
            if e4m3:
                # half a step relative to the value, or of the smallest step 2^-9 of the scale; the scale is at most
                # 2 max |x| / 448 (it goes to the next power of two)
                floor = 2.0 ** -10 * 2 * y.abs().amax(dim=-1, keepdim=True) / 448
                assert (off <= P.U_E4M3 * y.abs() + floor + (1 + P.U_E4M3) * dy).all()
            else:
                assert (off <= P.U_BF16 * y.abs() + (1 + P.U_BF16) * dy).all()
        assert (got.permute(0, 2, 1, 3)[~seen] == 0).all()  # pads and slots beyond the prompt untouched


# --- attention ----------------------------------------------------------------------------------------------


def _cache(device, e4m3, H, D, ps, lengths, seed=0, shuffle=True, scale=1.0):
    M = max(1, max((n + ps - 1) // ps for n in lengths))
    B = len(lengths)
    pages = B * M + 1
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(pages, generator=g) if shuffle else torch.arange(pages)
    table = order[: B * M].view(B, M).to(torch.int32)
    for b, n in enumerate(lengths):
        table[b, (n + ps - 1) // ps:] = -1
    k = _randn(seed + 1, pages, H, ps, D, scale=scale)
    v = _randn(seed + 2, pages, H, ps, D)
    return P.filled(pages, H, D, ps, e4m3, k, v, device), table


def _check(layer, table, lengths, q, window, device):
    got = kernels.paged_decode_attention(layer, q.to(device), page_table=table.to(device), lengths=_i32(lengths, device),
                                         window=window)
    k, v = P.slots_of(layer)
    want, bound = P.attention(k, v, table, lengths, q, window)
    off = (got.cpu().double() - want).abs()
    worst = (off / bound.clamp(min=1e-30)).max()
    assert (off <= bound).all(), f"{worst:.2f} of the bound"
    return got


ATTENDS = [  # D, H, R, page, lengths, window
    (64, 1, 1, 32, [1], 0),
    (64, 2, 16, 32, [31, 32, 33, 0], 0),
    (128, 2, 3, 32, [257, 1, 64, 700], 0),
    (128, 3, 8, 256, [5, 1000], 100),
    (256, 2, 4, 64, [701], 512),
    (256, 2, 4, 64, [0, 1, 63, 64, 65, 511, 512, 513, 1025], 512),
    (256, 1, 16, 128, [300, 129, 2], 1),
    (256, 4, 1, 32, [2049, 40], 0),
    (512, 1, 8, 64, [1, 5001, 77], 0),
    (512, 2, 16, 32, [90, 333], 45),
    (512, 1, 2, 1024, [1030, 3], 0),
    (512, 1, 16, 64, [4000], 0),
    (64, 1, 4, 256, [20000], 0),
    (128, 1, 2, 64, [9000, 3, 0, 9001, 0, 64], 5000),
]


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("D,H,R,ps,lengths,window", ATTENDS)
def test_attention_matches_64_bits(device, e4m3, D, H, R, ps, lengths, window):
    layer, table = _cache(device, e4m3, H, D, ps, lengths)
    q = _randn(9, len(lengths), H, R, D, scale=2.0 / math.sqrt(D))
    got = _check(layer, table, lengths, q, window, device)
    for b, n in enumerate(lengths):
        if n == 0:
            assert (got[b] == 0).all()


@pytest.mark.parametrize("e4m3", [False, True])
def test_attention_many_rows(device, e4m3):
    """More rows than compute units, ragged, the longest and the empty ones anywhere."""

    lengths = [(37 * i * i) % 203 for i in range(300)]
    lengths[150] = 900
    layer, table = _cache(device, e4m3, 1, 64, 32, lengths)
    _check(layer, table, lengths, _randn(9, len(lengths), 1, 5, 64, scale=0.25), 0, device)


@pytest.mark.parametrize("e4m3,D,H,R,B,M,window", [
    (True, 64, 1, 2, 700, 40, 0), (False, 64, 1, 1, 257, 64, 0), (True, 128, 3, 3, 300, 36, 1100),
    (False, 256, 1, 4, 90, 50, 0), (True, 256, 2, 1, 40, 300, 0), (True, 512, 2, 2, 200, 34, 0),
    (False, 512, 1, 16, 3, 200, 0), (True, 64, 2, 4, 1100, 33, 0),
])
def test_attention_of_cut_rows(device, e4m3, D, H, R, B, M, window):
    """Tables so long that rows are cut into pieces: more rows than a wave looks at once, more (row, head)s than
    workgroups are resident, long rows among empty and one-token ones. The tables' pages are drawn at random, so rows
    share them."""

    g = torch.Generator().manual_seed(B)
    ps, pages = 32, 64
    table = torch.randint(-1, pages, (B, M), generator=g).to(torch.int32)
    lengths = torch.randint(0, 70, (B,), generator=g)
    lengths[torch.randperm(B, generator=g)[: max(2, B // 40)]] = torch.randint(M * ps // 2, M * ps + 50, (max(2, B // 40),), generator=g)
    lengths[0], lengths[B - 1] = 0, M * ps
    layer = P.filled(pages, H, D, ps, e4m3, _randn(1, pages, H, ps, D), _randn(2, pages, H, ps, D), device)
    got = _check(layer, table, lengths.tolist(), _randn(9, B, H, R, D, scale=2.0 / math.sqrt(D)), window, device)
    assert (got[0] == 0).all()


SHARED = [  # D, H, R, page, rows, common pages, pages of a row, window
    (256, 2, 4, 64, 8, 12, 16, 0),
    (256, 1, 4, 32, 7, 25, 40, 0),
    (256, 2, 2, 128, 9, 6, 7, 500),
    (128, 2, 1, 32, 19, 30, 41, 0),
    (128, 1, 3, 64, 5, 40, 40, 0),  # all pages
    (64, 3, 8, 32, 4, 21, 90, 0),
    (64, 1, 5, 1024, 6, 2, 4, 1100),
    (64, 2, 4, 32, 130, 20, 25, 0),  # more rows than a wave looks at once
    (512, 1, 4, 64, 4, 12, 20, 0),
    (128, 1, 16, 64, 4, 12, 20, 0),
]


def _shared_table(D, B, common, M):
    """Rows that begin with the same pages and go on with pages of their own; one page of the pool is in no row."""

    pages = common + B * (M - common) + 1
    table = torch.empty(B, M, dtype=torch.int32)
    g = torch.Generator().manual_seed(D)
    ids = torch.randperm(pages, generator=g).to(torch.int32)
    for b in range(B):
        table[b, :common] = ids[:common]
        table[b, common:] = ids[common + b * (M - common): common + (b + 1) * (M - common)]
    return table, pages, ids


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("spoil", ["none", "page", "hole", "first", "short", "empty"])
@pytest.mark.parametrize("D,H,R,ps,B,common,M,window", SHARED)
def test_attention_of_rows_that_share_pages(device, e4m3, spoil, D, H, R, ps, B, common, M, window):
    """Rows with the same pages at their beginning and ragged ends; then with one row of them that has another page or
    none in the middle of it or at its start, ends in it, or is empty."""

    table, pages, ids = _shared_table(D, B, common, M)
    lengths = [common * ps + (37 * b * b + 5 * b) % ((M - common) * ps + 1) - (b % 3 == 2) * (ps // 2) for b in range(B)]
    odd = 2 if B > 2 else 1
    if spoil == "page":
        table[odd, common // 2] = ids[-1]
    elif spoil == "hole":
        table[odd, common // 2] = -1
        table[0, common - 1] = 2 ** 31 - 1
    elif spoil == "first":
        table[odd, 0] = ids[-1]
        table[B - 1, common - 1] = -5
    elif spoil == "short":
        lengths[odd] = common // 2 * ps + 7
    elif spoil == "empty":
        lengths[odd] = 0
    layer = P.filled(pages, H, D, ps, e4m3, _randn(1, pages, H, ps, D), _randn(2, pages, H, ps, D), device)
    _check(layer, table, lengths, _randn(9, B, H, R, D, scale=2.0 / math.sqrt(D)), window, device)


@pytest.mark.parametrize("e4m3", [False, True])
def test_nan_of_one_row_stays_there(device, e4m3):
    """Rows that share pages: a NaN in one row's own page, or in its query, reaches no other row."""

    D, ps, B, common, M = 128, 64, 4, 12, 14
    table, pages, _ = _shared_table(D, B, common, M)
    lengths = [common * ps + 70, common * ps + 3, common * ps, common * ps + 128]
    k, v, q = _randn(1, pages, 1, ps, D), _randn(2, pages, 1, ps, D), _randn(9, B, 1, 4, D, scale=0.2)
    layer = P.filled(pages, 1, D, ps, e4m3, k, v, device)
    want = _check(layer, table, lengths, q, 0, device)
    k[int(table[1, common]), 0, 1, 5] = math.nan
    v[int(table[3, common]), 0, 9, 5] = math.nan
    q[2, 0, 1, 3] = math.nan
    layer = P.filled(pages, 1, D, ps, e4m3, k, v, device)
    got = kernels.paged_decode_attention(layer, q.to(device), page_table=table.to(device), lengths=_i32(lengths, device))
    assert torch.equal(got[0], want[0]) and torch.equal(got[2, 0, [0, 2, 3]], want[2, 0, [0, 2, 3]])
    assert got[1].isnan().all() and got[2, 0, 1].isnan().all() and got[3, :, :, 5].isnan().all()
    assert torch.equal(got[3, :, :, 6:], want[3, :, :, 6:]) or e4m3  # an e4m3 vector's NaN may change its scale


def test_attention_more_rows_than_fit_a_workgroup_row(device):
    lengths = [(7 * i) % 40 for i in range(4500)]
    layer, table = _cache(device, True, 1, 64, 32, lengths)
    _check(layer, table, lengths, _randn(9, len(lengths), 1, 1, 64, scale=0.25), 0, device)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("scale", [0.02, 30.0])
def test_attention_flat_and_peaked_scores(device, e4m3, scale):
    lengths = [400, 65]
    layer, table = _cache(device, e4m3, 2, 128, 64, lengths)
    _check(layer, table, lengths, _randn(9, 2, 2, 4, 128, scale=scale / math.sqrt(128)), 0, device)


@pytest.mark.parametrize("e4m3", [False, True])
def test_attention_ignores_what_unattended_slots_hold(device, e4m3):
    """NaN and infinities in the slots behind a row, before its window and in pages of no row."""

    lengths, window, D, ps = [70, 33, 130, 0], 40, 128, 32
    layer, table = _cache(device, e4m3, 2, D, ps, lengths)
    q = _randn(9, 4, 2, 4, D, scale=0.2)
    want = _check(layer, table, lengths, q, window, device).clone()
    for t in (layer.key, layer.value):
        raw = t.view(torch.uint8) if e4m3 else t
        on = torch.zeros((layer.num_pages, ps), dtype=torch.bool)
        for b, n in enumerate(lengths):
            for p in range(max(0, n - window), n):
                on[int(table[b, p // ps]), p % ps] = True
        if t is layer.key:
            off = (~on).view(-1, 1, ps // 32, 1, 4, 2, 4, 1).permute(0, 1, 2, 3, 5, 4, 6, 7).reshape(-1, 1, ps // 32, 1, 2, 16, 1)
        else:
            off = (~on).view(-1, 1, ps // 8, 1, 8)
        bad = torch.tensor(0x7F, dtype=torch.uint8) if e4m3 else torch.tensor(math.nan, dtype=BF16)
        raw.copy_(torch.where(off.expand(t.shape), bad, raw.cpu()))
        if e4m3:
            sc = (layer.key_scale if t is layer.key else layer.value_scale).view(torch.uint8)
            sc.copy_(torch.where(~on[:, None, :], torch.tensor(255, dtype=torch.uint8), sc.cpu()))
    got = kernels.paged_decode_attention(layer, q.to(device), page_table=table.to(device), lengths=_i32(lengths, device),
                                         window=window)
    assert torch.equal(got, want)


def test_attention_with_missing_and_repeated_pages(device):
    """Entries outside the pages are left out of the softmax, one row's table repeats a page, two rows share."""

    D, ps = 64, 32
    layer, _ = _cache(device, True, 1, D, ps, [200, 200])
    table = torch.tensor([[0, -1, 1, 2, 1000000, 3], [0, 0, 0, 1, -7, -1], [-1, -1, -1, -1, -1, -1], [4, 5, 6, 7, 8, 9]],
                         dtype=torch.int32)
    lengths = [180, 128, 192, 100000]  # the last longer than its table
    got = _check(layer, table, lengths, _randn(9, 4, 1, 4, D, scale=0.3), 0, device)
    assert (got[2] == 0).all()


def test_attention_of_infinite_scores(device):
    """A key of -inf against a positive query is a probability of 0; keys of -inf alone give zeros, as documented;
    NaN and +inf scores give NaN."""

    D, ps = 64, 32
    k, v = torch.zeros(4, 1, ps, D, dtype=BF16), _randn(3, 4, 1, ps, D)
    k[0, 0, :5, 0] = -math.inf
    k[1, 0, :, 0] = -math.inf
    k[2, 0, 3, 0] = math.inf
    k[3, 0, 4, 0] = math.nan
    layer = P.filled(4, 1, D, ps, False, k, v, device)
    q = torch.zeros(4, 1, 2, D, dtype=BF16)
    q[..., 0] = 1.0
    got = kernels.paged_decode_attention(layer, q.to(device), page_table=_i32([[0], [1], [2], [3]], device),
                                         lengths=_i32([12, 32, 9, 9], device)).cpu()
    want = v[0, 0, 5:12].double().mean(dim=0)
    assert ((got[0].double() - want).abs() <= 2 * P.U_BF16 * v[0, 0, 5:12].double().abs().mean(dim=0) + 1e-6).all()
    assert (got[1] == 0).all()
    assert got[2].isnan().all() and got[3].isnan().all()


@pytest.mark.parametrize("D", [64, 512])
def test_e4m3_pages_of_infinities_and_nan(device, D):
    """An element that is no number is NaN in e4m3 and takes nothing from its neighbours: a key's makes the row's
    result NaN where it is attended, a value's its own dim only; reading gives NaN for the element alone."""

    ps, n = 32, 9
    k, v = _randn(1, 3, n, 1, D), _randn(2, 3, n, 1, D)
    k[0, 3, 0, 5] = math.inf
    v[1, 2, 0, 7], v[1, 4, 0, 60] = -math.inf, math.nan
    layer = new_paged_layer(3, 1, D, ps, e4m3=True, device=device)
    table = _i32([[0], [1], [2]], device)
    kernels.paged_append(layer, k.to(device), v.to(device), page_table=table, write_pos=_i32([0, 0, 0], device))
    q = _randn(3, 3, 1, 2, D, scale=0.1).to(device)
    call = lambda lengths: kernels.paged_decode_attention(layer, q, page_table=table, lengths=_i32(lengths, device)).cpu()  # noqa: E731
    out = call([n, n, n])
    assert out[0].isnan().all() and out[2].isfinite().all()
    bad = torch.zeros(D, dtype=torch.bool)
    bad[[7, 60]] = True
    assert out[1][..., bad].isnan().all() and out[1][..., ~bad].isfinite().all()
    assert call([3, 2, n])[:2].isfinite().all()  # none of them attended
    rk, rv = kernels.paged_read(layer, page_table=table, lengths=_i32([n] * 3, device), start=0, count=n)
    for got, x in ((rk, k), (rv, v)):
        _same(got, P.dequantised(x))


def test_attention_beyond_32_bit_offsets(device):
    """Pages whose places in the pool pass 2^32 bytes and elements."""

    H, D, ps = 2, 512, 1024
    pages = 4200  # 4200 * 2 * 1024 * 512 elements = 2^32 + 109 M, 2 bytes each
    layer = new_paged_layer(pages, H, D, ps, device=device)
    use = [pages - 1, 4097, 2100]
    k, v = _randn(1, 3, H, ps, D, scale=1.0), _randn(2, 3, H, ps, D)
    small = P.filled(3, H, D, ps, False, k, v, device)
    for i, p in enumerate(use):
        layer.key[p].copy_(small.key[i])
        layer.value[p].copy_(small.value[i])
    lengths = [2500, 1025]
    table, other = _i32([use, use], device), _i32([[0, 1, 2]] * 2, device)
    q = _randn(9, 2, H, 4, D, scale=2.0 / math.sqrt(D)).to(device)
    n = _i32(lengths, device)
    assert torch.equal(kernels.paged_decode_attention(layer, q, page_table=table, lengths=n),
                       kernels.paged_decode_attention(small, q, page_table=other, lengths=n))
    got, want = (kernels.paged_read(c, page_table=t, lengths=n, start=1000, count=50)
                 for c, t in ((layer, table), (small, other)))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    new = _randn(4, 2, 1, H, D).to(device)
    for c, t in ((layer, table), (small, other)):
        kernels.paged_append(c, new, new, page_table=t[:1].expand(2, 3).contiguous(), write_pos=_i32([7, 1040], device))
    assert all(torch.equal(layer.key[p], small.key[i]) and torch.equal(layer.value[p], small.value[i])
               for i, p in enumerate(use))
    del layer
    torch.cuda.empty_cache()


# --- read back ----------------------------------------------------------------------------------------------


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("D,H,ps,lengths,start,count", [
    (64, 1, 32, [1], 0, 1), (64, 3, 32, [0, 31, 100], 5, 70), (128, 2, 64, [65, 300], 64, 1),
    (256, 2, 64, [700, 1, 64, 65], 0, 701), (512, 1, 256, [300, 20], 37, 400), (256, 1, 32, [90], 1000, 33),
])
def test_read_back(device, e4m3, D, H, ps, lengths, start, count):
    layer, table = _cache(device, e4m3, H, D, ps, lengths)
    if len(lengths) > 1 and table.shape[1] > 1:
        table[1, 0] = -1
    k, v = P.slots_of(layer)
    got = kernels.paged_read(layer, page_table=table.to(device), lengths=_i32(lengths, device), start=start, count=count)
    for g, x in zip(got, (k, v)):
        want = torch.zeros((len(lengths), count, H, D), dtype=torch.float64)
        for b, n in enumerate(lengths):
            for i in range(count):
                p = start + i
                if p < min(n, table.shape[1] * ps) and 0 <= int(table[b, p // ps]) < layer.num_pages:
                    want[b, i] = x[int(table[b, p // ps]), :, p % ps]
        _same(g, want)
