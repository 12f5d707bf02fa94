"""Which pages of a batch are read once for several token rows, as work for the kernels of
``ops.attention_shared``.

Pure host code.  The rows' page lists form a tree: rows whose lists begin alike share a node,
with the pages that all of them see whole (so that nothing in them is hidden from any row); below
it they part, and what a row has alone, its partly filled last page among it, is its tail.  Every
node's queries, (row, head of a kv head's group), are cut into tiles, its pages into chunks, so
that the CTAs fill the device; see ``attention_shared.cuh`` for a unit's eight numbers.
"""
from __future__ import annotations

from typing import List, Sequence, Tuple

import numpy as np

PAGE = 64


def _alike(a: Sequence[int], b: Sequence[int], low: int, high: int) -> int:
    """The first index in ``low .. high`` at which the lists differ (``high`` if at none)."""
    if a is b or a[low:high] == b[low:high]:
        return high
    good, bad = low, high  # alike below ``good``, not alike below ``bad``
    while bad - good > 1:
        mid = (good + bad) // 2
        if a[good:mid] == b[good:mid]:
            good = mid
        else:
            bad = mid
    return good


def shared_nodes(tables: Sequence[Sequence[int]], seqs: Sequence[int], positions: Sequence[int],
                 ahead: int = 0) -> Tuple[List[tuple], List[tuple]]:
    """(nodes, tails): nodes (rows, first page, end page) that several rows share, parents before children;
    tails (row, first page, end page), ``ahead`` pages longer than they are (rows that will grow)."""
    nodes: List[tuple] = []
    tails: List[tuple] = []

    def tail(row: int, depth: int) -> None:
        end = positions[row] // PAGE + 1 + ahead
        if end > depth:
            tails.append((row, depth, end))

    # (a padding row has a tail of no pages: the unit that writes its zeros)
    tails += [(r, 0, 0) for r in range(len(seqs)) if positions[r] < 0]
    work = [([r for r in range(len(seqs)) if positions[r] >= 0], 0)]
    while work:
        rows, depth = work.pop()
        if not rows:
            continue
        if len(rows) == 1:
            tail(rows[0], depth)
            continue
        whole = [(positions[r] + 1) // PAGE for r in rows]
        first, end = tables[seqs[rows[0]]], min(whole)
        if end > depth:
            for r in rows[1:]:
                end = _alike(first, tables[seqs[r]], depth, end)
                if end == depth:
                    break
        if end > depth:
            nodes.append((rows, depth, end))
        classes = {}
        for r, n in zip(rows, whole):
            if n > end:
                classes.setdefault(tables[seqs[r]][end], []).append(r)
            else:
                tail(r, end)
        if end == depth and len(classes) == 1 and len(next(iter(classes.values()))) == len(rows):
            raise ValueError("page lists that neither share a page nor part")  # (cannot be)
        work.extend((c, end) for c in classes.values())
    return nodes, tails


def shared_units(nodes: Sequence[tuple], tails: Sequence[tuple], seqs: Sequence[int], group: int, kv_heads: int,
                 kinds: Sequence[tuple], ending: int):
    """(units of every kind [*, 8], members, record offsets [rows + 1]).

    ``kinds``: (most entries of a unit, CTAs of the kind that the device holds at once, or warps of a kind that goes warp by warp,
    fewest and most pages of a chunk, whether each of those takes several units in turn), entries ascending, 0 where the kernel
    has no such kind; ``ending``: the last kind that takes units whose rows end inside them."""
    pieces = []  # (rows, first, end, ends, kind)
    total = [0] * len(kinds)
    for rows, a, b, ends in [(*n, 0) for n in nodes] + [([r], a, b, 1 + r) for r, a, b in tails]:
        entries = len(rows) * group
        may = [i for i, k in enumerate(kinds) if k[0] and (not ends or i <= ending)]
        kind = next((i for i in may if entries <= kinds[i][0]), may[-1])
        pieces.append((rows, a, b, ends, kind))
        total[kind] += -(-entries // kinds[kind][0]) * (b - a) * kv_heads
    # pages of a chunk: as few as leave no more CTAs of the kind than it has at once (a few more would run by themselves), or,
    # of units dealt in turn, an even share of all pages
    share = [1] * len(kinds)
    for i, (tile, ctas, least, most, dealt) in enumerate(kinds):
        mine = [(b - a, -(-len(rows) * group // tile) * kv_heads) for rows, a, b, _, kind in pieces if kind == i]
        if mine:
            share[i] = min(most, max(least, -(-total[i] // ctas)))
            while not dealt and share[i] < min(most, max(n for n, _ in mine)) and \
                    sum(-(-n // share[i]) * tiles for n, tiles in mine) > ctas:
                share[i] += 1 + share[i] // 16
            share[i] = min(share[i], most)
    units: List[List[tuple]] = [[] for _ in kinds]
    members: List[int] = []
    slots = [0] * len(seqs)
    for rows, a, b, ends, kind in pieces:
        entries, tile = len(rows) * group, kinds[kind][0]
        chunks = max(1, -(-(b - a) // share[kind]))
        per = max(1, -(-(b - a) // chunks))
        at, slot = len(members), slots[rows[0]]
        members.extend(rows)
        for c in range(a, b, per) if b > a else (a,):
            for e in range(0, entries, tile):
                units[kind].append((at, e, min(tile, entries - e), c, min(b, c + per), slot, seqs[rows[0]], ends))
            slot += 1
        for r in rows:
            slots[r] = slot
    for kind in units:  # the units that take longest first: the last to start are short
        kind.sort(key=lambda u: u[3] - u[4])
    record = np.zeros(len(seqs) + 1, dtype=np.int32)
    np.cumsum(slots, out=record[1:])
    return ([np.asarray(kind, dtype=np.int32).reshape(-1, 8) for kind in units], np.asarray(members, dtype=np.int32), record)
