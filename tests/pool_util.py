"""The page pool restated plainly (Python lists) for its tests: which fresh page goes where, what is shared, copied,
given back and moved."""

from __future__ import annotations


def _fresh(refs):
    return iter([p for p, n in enumerate(refs) if n <= 0])


def _held(p, refs):
    return 0 <= p < len(refs)


def reserve(refs, table, lengths, ps):
    """In place; returns the shortage."""

    fresh, short = _fresh(refs), 0
    for row, n in zip(table, lengths):
        for e in range(min(-(-max(n, 0) // ps), len(row))):
            if not _held(row[e], refs):
                p = next(fresh, None)
                if p is None:
                    short += 1
                else:
                    row[e], refs[p] = p, 1
    return short


def fork(refs, table, parents, lengths, ps, width):
    """``refs`` in place; returns (children, [(source, target, slots)], shortage)."""

    fresh, short, children, moves = _fresh(refs), 0, [], []
    for a in parents:
        child = [-1] * width
        children.append(child)
        if not 0 <= a < len(table):
            continue
        n = min(max(lengths[a], 0), min(len(table[a]), width) * ps)
        for e in range(n // ps):
            if _held(table[a][e], refs):
                child[e] = table[a][e]
        e = n // ps
        if n % ps and _held(table[a][e], refs):
            p = next(fresh, None)
            if p is None:
                short += 1
            else:
                child[e] = p
                moves.append((table[a][e], p, n % ps))
    for child in children:
        for p in child:
            if p >= 0:
                refs[p] += 1
    for _, p, _ in moves:
        refs[p] = 1
    return children, moves, short


def free(refs, table, keep, ps):
    for row, n in zip(table, keep):
        for e in range(-(-max(n, 0) // ps), len(row)):
            if _held(row[e], refs):
                refs[row[e]] -= 1
            row[e] = -1


def compact(refs, table):
    """In place; returns (pages in use, [(source, target)])."""

    n = sum(x > 0 for x in refs)
    moves = list(zip([p for p in range(n, len(refs)) if refs[p] > 0], [p for p in range(n) if refs[p] <= 0]))
    to = dict(moves)
    for a, b in moves:
        refs[b], refs[a] = refs[a], 0
    for row in table:
        row[:] = [to.get(p, p) for p in row]
    return n, moves


def moved(layer, moves, ps):
    """What a layer's arrays (on the CPU, as bytes or bf16) hold after (source, target, slots) of ``moves``, the sources
    as they were before: the 32-slot chunks that hold the slots."""

    import torch

    out = []
    for t in layer:
        if t is None:
            out.append(None)
            continue
        x = t.cpu().view(torch.int16 if t.dtype == torch.bfloat16 else torch.uint8)
        before, after = x.reshape(x.shape[0], x.shape[1], -1), x.clone().view(x.shape[0], x.shape[1], -1)
        per = before.shape[2] // ps
        for a, b, slots in moves:
            m = -(-slots // 32) * 32 * per
            after[b, :, :m] = before[a, :, :m]
        out.append(after.view(x.shape))
    return out
