"""Paged attention of cut rows in large batches: more rows than one wave looks at, whose pieces a launch of its own
lays out."""

from __future__ import annotations

import math

import pytest
import torch

import paged_util as P
from gemma4_posttrain_jax_amd import kernels

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _randn(seed, *shape, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(BF16)


def _case(device, B, H, D, M, R=2, ps=32, pages=64, e4m3=True):
    g = torch.Generator().manual_seed(B + D)
    table = torch.randint(-1, pages, (B, M), generator=g).to(torch.int32)
    layer = P.filled(pages, H, D, ps, e4m3, _randn(1, pages, H, ps, D), _randn(2, pages, H, ps, D), device)
    return table, layer, _randn(9, B, H, R, D, scale=2.0 / math.sqrt(D))


# Where the lookup takes one, two or three steps of 64, and at the border below it
@pytest.mark.parametrize("B,H,D,e4m3", [(256, 1, 64, True), (257, 1, 64, True), (258, 3, 64, False), (512, 2, 64, True), (513, 2, 64, False),
                                        (1024, 2, 64, True),
                                        (1025, 1, 512, True), (4095, 1, 64, True), (4097, 1, 64, False), (4200, 2, 128, True)])
@pytest.mark.parametrize("rows", ["one", "mixed", "equal", "empty"])
def test_rows_of_large_batches(device, B, H, D, e4m3, rows):
    """One long row among empty and short ones, a few, all rows at the border to two pieces, or no row at all; every
    row against 64 bits that can hold more than a few positions, and every 37th of the others."""

    M = 36
    table, layer, q = _case(device, B, H, D, M, e4m3=e4m3)
    g = torch.Generator().manual_seed(B)
    lengths = torch.randint(0, 12, (B,), generator=g)
    if rows == "one":
        lengths[(3 * B) // 7] = M * 32
    elif rows == "mixed":
        lengths[torch.randperm(B, generator=g)[:20]] = torch.randint(1, M * 32 + 40, (20,), generator=g)
        lengths[0], lengths[B - 1] = M * 32 - 1, M * 32
    elif rows == "equal":
        lengths[:] = 33
    else:
        lengths[:] = 0
    n = lengths.to(torch.int32).to(device)
    q_dev, t_dev = q.to(device), table.to(device)
    got = kernels.paged_decode_attention(layer, q_dev, page_table=t_dev, lengths=n)
    again = kernels.paged_decode_attention(layer, q_dev, page_table=t_dev, lengths=n)
    assert torch.equal(got, again)
    got = got.cpu().double()
    assert (got[lengths == 0] == 0).all()
    check = sorted(set(torch.nonzero(lengths > 40)[:, 0].tolist()) | set(range(0, B, 37)) | {1, B - 2, B - 1})
    k, v = P.slots_of(layer)
    want, bound = P.attention(k, v, table[check], lengths[check].tolist(), q[check], 0)
    assert ((got[check] - want).abs() <= bound).all()


def test_windows_of_a_large_batch_in_a_graph(device):
    """A window, the pieces laid out again at every replay for new lengths, eager calls of other sizes between."""

    B, H, D, M, window = 600, 1, 64, 60, 1200
    table, layer, q = _case(device, B, H, D, M)
    t_dev, q_dev = table.to(device), q.to(device)
    lengths = torch.zeros(B, dtype=torch.int32, device=device)
    call = lambda n: kernels.paged_decode_attention(layer, q_dev, page_table=t_dev, lengths=n, window=window)  # noqa: E731
    call(lengths)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        out = call(lengths)
    torch.cuda.current_stream().wait_stream(side)
    for i in range(5):
        new = torch.randint(0, 60, (B,), generator=torch.Generator().manual_seed(i)).to(torch.int32)
        new[i::101] = M * 32 - 7 * i
        want = call(new.to(device)).clone()
        lengths.copy_(new)
        graph.replay()
        kernels.paged_decode_attention(layer, q_dev[:300], page_table=t_dev[:300], lengths=lengths[:300])
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
        some = list(range(i, B, 101)) + [0, B - 1]
        k, v = P.slots_of(layer)
        ref, bound = P.attention(k, v, table[some], new[some].tolist(), q[some], window)
        assert ((out.cpu().double()[some] - ref).abs() <= bound).all(), i


def test_time_goes_with_the_rows(device):
    """Short rows in a wide table: four times the rows take about four times as long (sixteen times where every
    workgroup reads every length)."""

    times = []
    for B in (8192, 32768):
        table, layer, q = _case(device, B, 1, 64, 36)
        t_dev, q_dev = table.to(device), q.to(device)
        n = torch.randint(1, 40, (B,), generator=torch.Generator().manual_seed(0)).to(torch.int32).to(device)
        call = lambda: kernels.paged_decode_attention(layer, q_dev, page_table=t_dev, lengths=n)  # noqa: E731
        call()
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        best = math.inf
        for _ in range(5):
            torch.cuda.synchronize()
            start.record()
            call()
            end.record()
            end.synchronize()
            best = min(best, start.elapsed_time(end))
        times.append(best)
    assert times[1] <= 8 * times[0], times
