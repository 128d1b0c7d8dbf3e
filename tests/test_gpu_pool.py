"""The page pool on the GPU against plain lists, bit for bit: fresh pages, forks, copies, frees and compaction."""

from __future__ import annotations

import pytest
import torch

import pool_util as plain
from gemma4_posttrain_jax_amd import kernels
from gemma4_posttrain_jax_amd.kvcache import new_paged_layer

pytestmark = pytest.mark.gpu


def _i32(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


def _layer(P, H, D, ps, e4m3, seed, device):
    layer = new_paged_layer(P, H, D, ps, e4m3=e4m3, device=device)
    g = torch.Generator().manual_seed(seed)
    for t in layer:
        if t is not None:
            raw = t.view(torch.int16) if t.dtype == torch.bfloat16 else t.view(torch.uint8)
            raw.copy_(torch.randint(0, 256, raw.shape, generator=g).to(raw.dtype))  # any bytes: copies look at none
    return layer


def _bytes(layer):
    return [None if t is None else t.cpu().view(torch.int16 if t.dtype == torch.bfloat16 else torch.uint8) for t in layer]


def _same(layer, want):
    for got, w in zip(_bytes(layer), want):
        assert (got is None) == (w is None)
        assert got is None or torch.equal(got, w)


def _pool(P, rows, width, used, seed):
    """refs and a table of rows of up to ``width`` of ``used`` pages in any order, some of them with holes."""

    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(P, generator=g)[:used].tolist()
    refs, table = [0] * P, []
    for b in range(rows):
        n = int(torch.randint(0, width + 1, (1,), generator=g))
        row = [order.pop() if order else -1 for _ in range(n)] + [-1] * (width - n)
        if n > 2 and b % 3 == 0:
            row[1] = -1 if b % 2 else P + 5
        table.append(row)
        for p in row:
            if 0 <= p < P:
                refs[p] += 1
    return refs, table


@pytest.mark.parametrize("P,rows,width", [(1, 1, 1), (63, 5, 9), (64, 3, 4), (257, 40, 5), (1024, 9, 70), (5000, 300, 20),
                                          (70000, 1100, 60)])
def test_reserve(P, rows, width, device):
    refs, table = _pool(P, rows, width, P // 3, 1)
    g = torch.Generator().manual_seed(2)
    lengths = torch.randint(-40, 32 * width + 100, (rows,), generator=g).tolist()
    r, t = _i32(refs, device), _i32(table, device)
    short = kernels.paged_reserve(r, t, _i32(lengths, device), page_size=32)
    want = plain.reserve(refs, table, lengths, 32)
    assert short.tolist() == [want] and r.tolist() == refs and t.tolist() == table


def test_reserve_in_a_pool_past_the_spans(device):
    """Over a million pages, where one count in LDS stands for several groups; refs below 0 are free."""

    P = (1 << 20) + 12345
    refs = torch.ones(P, dtype=torch.int32, device=device)
    free = torch.randperm(P, generator=torch.Generator().manual_seed(3))[:5000].sort().values
    refs[free.to(device)] = -3
    table = torch.full((100, 49), -1, dtype=torch.int32, device=device)
    short = kernels.paged_reserve(refs, table, torch.full((100,), 49 * 64, dtype=torch.int32, device=device), page_size=64)
    assert short.tolist() == [0]
    assert torch.equal(table.flatten().cpu(), free[:4900].to(torch.int32))
    assert int((refs <= 0).sum()) == 100


def test_reserve_over_a_wider_tables_columns(device):
    refs, table = _pool(100, 6, 8, 20, 4)
    t = _i32(table, device)
    lengths = [300] * 6
    r = _i32(refs, device)
    kernels.paged_reserve(r, t[:, :5], _i32(lengths, device), page_size=64)
    narrow = [row[:5] for row in table]
    plain.reserve(refs, narrow, lengths, 64)
    assert t.tolist() == [a + row[5:] for a, row in zip(narrow, table)] and r.tolist() == refs


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("H,D,ps", [(1, 64, 32), (2, 256, 64), (3, 512, 128), (1, 128, 1024)])
def test_fork(H, D, ps, e4m3, device):
    P = 40 if ps == 1024 else 300
    refs, table = _pool(P, 7, 5, P // 3, 5)
    g = torch.Generator().manual_seed(6)
    lengths = [min(n, 5 * ps) for n in (0, 1, ps, ps + 1, 3 * ps - 1, 5 * ps, 7 * ps)]
    lengths[0] = -4
    parents = [6, 5, 4, 4, 4, 3, 2, 1, 0, -1, 7, 2 ** 31 - 1, 4]
    layers = [_layer(P, H, D, ps, e4m3, 7, device), _layer(P, 1, 128, ps, not e4m3, 8, device)]
    before = [type(x)(*(None if t is None else t.clone() for t in x)) for x in layers]
    r = _i32(refs, device)
    t = _i32(table, device)
    children, short = kernels.paged_fork(layers, r, t, _i32(parents, device), _i32(lengths, device))
    want, moves, lacking = plain.fork(refs, table, parents, lengths, ps, 5)
    assert children.tolist() == want and short.tolist() == [lacking] and r.tolist() == refs and t.tolist() == table
    for x, old in zip(layers, before):
        _same(x, plain.moved(old, moves, ps))


@pytest.mark.parametrize("width", [1, 3, 9])
def test_fork_into_a_table_of_another_width(width, device):
    refs, table = _pool(200, 6, 5, 60, 9)
    lengths, parents = [160, 150, 33, 32, 31, 97], [0, 1, 2, 3, 4, 5, 5, 1]
    layer = _layer(200, 2, 64, 32, False, 10, device)
    old = type(layer)(*(None if t is None else t.clone() for t in layer))
    wide = torch.full((8, 20), 77, dtype=torch.int32, device=device)
    r = _i32(refs, device)
    out, short = kernels.paged_fork([layer], r, _i32(table, device), _i32(parents, device), _i32(lengths, device),
                                    out=wide[:, 2:2 + width])
    want, moves, lacking = plain.fork(refs, table, parents, lengths, 32, width)
    assert out.tolist() == want and short.tolist() == [lacking] and r.tolist() == refs
    assert bool((wide[:, :2] == 77).all()) and bool((wide[:, 2 + width:] == 77).all())
    _same(layer, plain.moved(old, moves, 32))


def test_fork_with_too_few_pages(device):
    refs, table = [1, 1, 1, 0, 1, 0, 1], [[0, 1], [2, 4]]
    layer = _layer(7, 1, 64, 32, True, 11, device)
    old = type(layer)(*(t.clone() for t in layer))
    r = _i32(refs, device)
    out, short = kernels.paged_fork([layer], r, _i32(table, device), _i32([0, 1, 0, 1], device), _i32([40, 50], device))
    want, moves, lacking = plain.fork(refs, table, [0, 1, 0, 1], [40, 50], 32, 2)
    assert lacking == 2 and short.tolist() == [2] and out.tolist() == want and r.tolist() == refs
    _same(layer, plain.moved(old, moves, 32))


@pytest.mark.parametrize("n", [1, 300, 5000])
def test_fork_of_many_children(n, device):
    P = 6000
    refs, table = _pool(P, 16, 8, 100, 12)
    lengths = [37 * b % 250 for b in range(16)]
    parents = [i * 7 % 16 for i in range(n)]
    layer = _layer(P, 1, 64, 32, True, 13, device)
    old = type(layer)(*(t.clone() for t in layer))
    r = _i32(refs, device)
    out, short = kernels.paged_fork([layer], r, _i32(table, device), _i32(parents, device), _i32(lengths, device))
    want, moves, lacking = plain.fork(refs, table, parents, lengths, 32, 8)
    assert out.tolist() == want and short.tolist() == [lacking] and r.tolist() == refs
    _same(layer, plain.moved(old, moves, 32))


@pytest.mark.parametrize("rows,width", [(1, 1), (7, 5), (513, 33)])
def test_free(rows, width, device):
    refs, table = _pool(4000, rows, width, 3000, 14)
    g = torch.Generator().manual_seed(15)
    keep = torch.randint(-10, 64 * width + 70, (rows,), generator=g).tolist()
    keep[0] = 2 ** 31 - 1 if rows > 1 else 0
    r, t = _i32(refs, device), _i32(table, device)
    kernels.paged_free(r, t, _i32(keep, device), page_size=64)
    plain.free(refs, table, keep, 64)
    assert r.tolist() == refs and t.tolist() == table


def test_a_page_held_by_several_entries_is_counted_once_per_entry(device):
    refs, table = [0, 3, 2, 0], [[1, 2], [1, 2], [1, -1]]
    r, t = _i32(refs, device), _i32(table, device)
    kernels.paged_free(r, t, _i32([0, 32, 0], device), page_size=32)
    assert r.tolist() == [0, 1, 0, 0] and t.tolist() == [[-1, -1], [1, -1], [-1, -1]]


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("P,rows,width,used", [(1, 1, 1, 1), (64, 4, 5, 20), (300, 40, 7, 200), (300, 40, 7, 0),
                                               (5000, 100, 30, 2500)])
def test_compact(P, rows, width, used, e4m3, device):
    refs, table = _pool(P, rows, width, used, 16)
    if rows > 2:  # shared pages
        for b in range(1, rows, 5):
            table[b] = list(table[b - 1])
        refs = [0] * P
        for row in table:
            for p in row:
                if 0 <= p < P:
                    refs[p] += 1
    layers = [_layer(P, 1, 64, 32, e4m3, 17, device), _layer(P, 2, 64, 32, False, 18, device)]
    before = [type(x)(*(None if t is None else t.clone() for t in x)) for x in layers]
    r, t = _i32(refs, device), _i32(table, device)
    live = kernels.paged_compact(layers, r, t)
    n, moves = plain.compact(refs, table)
    assert live.tolist() == [n] and r.tolist() == refs and t.tolist() == table
    for x, old in zip(layers, before):
        _same(x, plain.moved(old, [(a, b, 32) for a, b in moves], 32))
    assert kernels.paged_compact(layers, r, t).tolist() == [n] and r.tolist() == refs  # nothing left to move


def test_copy_over_many_layers(device):
    """More layers than one launch takes, of different heads, dims and formats; pairs outside the pool left out."""

    P, ps = 30, 64
    layers = [_layer(P, 1 + i % 3, (64, 128, 256, 512)[i % 4], ps, i % 2 == 0, 20 + i, device) for i in range(37)]
    before = [type(x)(*(None if t is None else t.clone() for t in x)) for x in layers]
    src, dst = [3, 3, 29, -1, 5, 30, 7, 8], [0, 10, 11, 12, -1, 13, 7, 2 ** 31 - 1]
    kernels.paged_copy(layers, _i32(src, device), _i32(dst, device))
    for x, old in zip(layers, before):
        _same(x, plain.moved(old, [(3, 0, ps), (3, 10, ps), (29, 11, ps)], ps))


def test_copy_past_4_gib(device):
    """Pages whose bytes lie past 2^32 from the start of the array."""

    P, H, D, ps = 2100, 2, 512, 1024  # 2 MiB of keys a page
    layer = new_paged_layer(P, H, D, ps, device=device)
    layer.key[3].fill_(1.5)
    layer.value[2098].fill_(2.5)
    kernels.paged_copy([layer], _i32([3, 2098], device), _i32([2099, 1], device))
    assert bool((layer.key[2099] == 1.5).all()) and bool((layer.value[1] == 2.5).all())
    assert bool((layer.key[1] == 0).all()) and bool((layer.value[2099] == 0).all())


@pytest.mark.parametrize("rows", [1, 31, 32, 33])
@pytest.mark.parametrize("P", [1, 255, 16384, 16385])
def test_about_the_change_to_one_launch(P, rows, device):
    """Up to 32 rows of up to 16384 pages go by one launch."""

    refs, table = _pool(P, rows, 7, P // 2, 20 + rows)
    lengths = [(37 * b) % 300 for b in range(rows)]
    r, t = _i32(refs, device), _i32(table, device)
    short = kernels.paged_reserve(r, t, _i32(lengths, device), page_size=32)
    assert short.tolist() == [plain.reserve(refs, table, lengths, 32)] and r.tolist() == refs and t.tolist() == table
    layer = _layer(P, 1, 64, 32, True, 21, device)
    old = type(layer)(*(None if x is None else x.clone() for x in layer))
    parents = [(5 * b) % (rows + 1) for b in range(rows)]  # one of them outside, several of one row
    children, short = kernels.paged_fork([layer], r, t, _i32(parents, device), _i32(lengths, device))
    want, moves, lacking = plain.fork(refs, table, parents, lengths, 32, 7)
    assert children.tolist() == want and short.tolist() == [lacking] and r.tolist() == refs
    _same(layer, plain.moved(old, moves, 32))


def _step(layers, refs, table, parents, lengths, none, target):
    """A serving step: children in place of their parents, pages for what they will hold, the pool compacted."""

    children, short = kernels.paged_fork(layers, refs, table, parents, lengths)
    kernels.paged_free(refs, table, none, page_size=32)
    lacking = kernels.paged_reserve(refs, children, target, page_size=32)
    live = kernels.paged_compact(layers, refs, children)
    return children, short, lacking, live


@pytest.mark.parametrize("rows,P", [(6, 120), (50, 700)])
def test_replays_between_eager_calls(rows, P, device):
    """The five calls captured into a graph, replayed on new tables with eager calls of another pool between."""

    width, layers = 6, [_layer(P, 1, 64, 32, False, 30, device), _layer(P, 2, 128, 32, True, 31, device)]
    other = [_layer(90, 1, 64, 32, False, 32, device)]
    first = [[None if t is None else t.clone() for t in x] for x in layers + other]

    def restore(xs, was):
        for x, old in zip(xs, was):
            for t, o in zip(x, old):
                if t is not None:
                    t.copy_(o)

    def inputs(seed, P, rows):
        refs, table = _pool(P, rows, width, P // 2, seed)
        g = torch.Generator().manual_seed(seed)
        parents = torch.randint(0, rows, (rows,), generator=g).tolist()
        lengths = torch.randint(0, 32 * width, (rows,), generator=g).tolist()
        return [_i32(x, device) for x in (refs, table, parents, lengths, [0] * rows, [n + 20 for n in lengths])]

    def outcome(xs, args, out):
        return [t.clone() for t in (*args[:2], *out)] + [b for x in xs for b in _bytes(x) if b is not None]

    def eager(xs, was, args):
        restore(xs, was)
        args = [t.clone() for t in args]
        return outcome(xs, args, _step(xs, *args))

    sets = [inputs(s, P, rows) for s in (41, 42, 43)]
    want = [eager(layers, first[:2], s) for s in sets]
    theirs = inputs(44, 90, 9)
    want_theirs = eager(other, first[2:], theirs)
    static = [t.clone() for t in sets[0]]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        _step(layers, *[t.clone() for t in static])
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _step(layers, *static)
    for i in (1, 2, 0, 1):
        restore(layers, first[:2])
        for to, x in zip(static, sets[i]):
            to.copy_(x)
        graph.replay()
        assert all(torch.equal(x, y) for x, y in zip(eager(other, first[2:], theirs), want_theirs))
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(outcome(layers, static, out), want[i]))


def test_pools_on_two_streams(device):
    """Calls of two pools that overlap on two streams."""

    pools = []
    for seed in (51, 52):
        refs, table = _pool(3000, 200, 9, 1500, seed)
        pools.append((_layer(3000, 1, 64, 32, False, seed, device), refs, table))
    torch.cuda.synchronize()
    lengths, parents = [(31 * b) % 280 for b in range(200)], [(7 * b) % 200 for b in range(200)]
    args = [_i32(x, device) for x in (parents, lengths)]
    got, streams = [], [torch.cuda.Stream(), torch.cuda.Stream()]
    ready = [(_i32(refs, device), _i32(table, device)) for _, refs, table in pools]
    torch.cuda.synchronize()
    for (layer, _, _), (r, t), stream in zip(pools, ready, streams):
        with torch.cuda.stream(stream):
            got.append((r, *kernels.paged_fork([layer], r, t, *args)))
    torch.cuda.synchronize()
    for (_, refs, table), (r, children, short) in zip(pools, got):
        want, _, lacking = plain.fork(refs, table, parents, lengths, 32, 9)
        assert children.tolist() == want and short.tolist() == [lacking] and r.tolist() == refs


def test_the_same_layer_twice_and_one_page(device):
    """A layer that is named twice is copied alike; a pool of one page."""

    layer = _layer(1, 1, 64, 32, True, 60, device)
    r, t = _i32([1], device), _i32([[0]], device)
    children, short = kernels.paged_fork([layer, layer], r, t, _i32([0, 0], device), _i32([32], device))
    assert children.tolist() == [[0], [0]] and r.tolist() == [3] and short.tolist() == [0]
    children, short = kernels.paged_fork([layer], r, t, _i32([0, 0], device), _i32([31], device))
    assert children.tolist() == [[-1], [-1]] and r.tolist() == [3] and short.tolist() == [2]
    assert kernels.paged_compact([layer], r, t).tolist() == [1] and t.tolist() == [[0]]
    kernels.paged_free(r, t, _i32([0], device), page_size=32)
    assert r.tolist() == [2] and t.tolist() == [[-1]]


@pytest.mark.parametrize("P", [2559, 2560, 2561])
def test_compact_about_the_change_to_one_launch(P, device):
    refs, table = _pool(P, 100, 30, P // 2, 71)
    layer = _layer(P, 1, 64, 32, True, 72, device)
    old = type(layer)(*(None if x is None else x.clone() for x in layer))
    r, t = _i32(refs, device), _i32(table, device)
    live = kernels.paged_compact([layer], r, t)
    n, moves = plain.compact(refs, table)
    assert live.tolist() == [n] and r.tolist() == refs and t.tolist() == table
    _same(layer, plain.moved(old, [(a, b, 32) for a, b in moves], 32))
