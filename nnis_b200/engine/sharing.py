"""Which steps read shared pages once for several rows, and the plans they do it by.

Rows share pages where their sequences were forked from one another (``CacheManager.fork``) and, with
several tokens of a sequence in one step, where those see the same pages.  A step's context asks for
the plan (``ops.SharedPlan``) of a cache group and a head layout: ``SharedRows`` makes it then, for a step
that is launched kernel by kernel; ``KeptPlans`` holds plans of a captured step at addresses that stay.
"""
from __future__ import annotations

from typing import Dict, Optional, Sequence, Tuple

import torch

from ..cache import PAGE_SIZE
from ..csrc import ops

# Bytes of keys and values that sharing has to take off what the rows of a layer read one by one: it costs a launch or two more
# and a merge.  us a layer of a decode step, one by one -> shared, bytes saved: bfloat16, 9 heads over 3 of 64, 8 rows behind 64
# pages (22 MB) 7.2 -> 9.6, 4 behind 256 (38 MB) 14.5 -> 12.4, 16 behind 64 (47 MB) 12.9 -> 10.0, 64 behind 256 137 -> 19; 32 over 32 of
# 64, 8 behind 4 (15 MB) 5.2 -> 7.6, 4 behind 16 (25 MB) 10.2 -> 7.8, 2 behind 64 (34 MB) 15.5 -> 11; 32 over 8 of 128, 8 behind 16
# (29 MB) 10.9 -> 13.4, 16 behind 16 (63 MB) 14.9 -> 10.8.  Of 270 such batches (heads 9/3 to 20/1) the 87 of more bytes are at most 8 %
# slower (64 rows behind 8 pages, 39 MB, 11.2 -> 12.1).
LEAST_BYTES = 32 << 20
# The kernels of float32, and of head sizes other than 64 and 128, take a page of a unit for so and so many (query head, page) of the kernels
# that read row by row, by (dtype, whether 64 or 128): shared only where what the rows see alike outweighs that.  us a layer, one by one ->
# shared: float32, 32 heads over 32 of 64, 2 rows behind 64 pages 41 -> 48, 4 behind 21 35 -> 24, 64 behind 1 26 -> 55; 9 over 3, 2
# behind 341 76 -> 34; 12 over 12 of 96, 2 behind 114 48 -> 88, 8 behind 16 40 -> 21, 64 behind 2 34 -> 51.  bfloat16, 12 over 12 of 96, 2 behind
# 512 107 -> 345, 4 behind 303 120 -> 205, 16 behind 15 32 -> 26, 16 behind 61 100 -> 61; 16 over 4 of 96, 2 behind 341 74 -> 97, 4
# behind 228 98 -> 75, 64 behind 43 231 -> 94; 8 over 2 of 256, 8 behind 73 90 -> 102, 16 behind 34 89 -> 74.  Of 537 such batches 84 are
# slower by the rule of bytes alone, up to 3.2 times; by both rules 4, up to 1.55 times (64 rows of 4 heads over 4 of 250).
PAGE_COST = {(torch.float32, True): 3, (torch.float32, False): 5, (torch.bfloat16, False): 8}
AHEAD = 8  # pages that the plan of a step which is looked at every time lets its sequences grow by

PlanKey = Tuple[int, int, int, int]  # cache group, heads, key/value heads, head size


def shared_tree(cache, group: int, slots: Sequence[int], seqs: Sequence[int], positions: Sequence[int], least_bytes: int,
                ahead: int = 0):
    """(nodes, tails) of the rows' pages (``ops.shared_nodes``), or None where sharing takes off too few bytes to pay."""
    g = cache.groups[group]
    if g.window > 0:
        return None
    nodes, tails = ops.shared_nodes([cache.page_table(group, s) for s in slots], seqs, positions, ahead)
    saved = sum((len(rows) - 1) * (b - a) for rows, a, b in nodes)
    return (nodes, tails) if saved * PAGE_SIZE * g.kv_heads * (g.head_dim + g.value_dim) * g.k.element_size() >= least_bytes else None


def heads_share(tree, positions: Sequence[int], key: PlanKey, dtype: torch.dtype, ahead: int = 0) -> bool:
    """Whether the kernels of this head layout and type gain by reading such a tree's pages once (``PAGE_COST``)."""
    _, heads, kv_heads, head_dim = key
    cost = PAGE_COST.get((dtype, head_dim in (64, 128)), 0)
    if not cost:
        return True
    group = heads // kv_heads
    # (a unit of up to 64 entries takes twice as long as one of up to 16)
    tiles = lambda rows: 1 if rows * group <= 16 else 2 * -(-rows * group // 64)
    nodes, tails = tree
    units = sum(tiles(len(rows)) * (b - a) for rows, a, b in nodes) + tiles(1) * sum(max(0, b - a - ahead) for _, a, b in tails)
    return cost * units < group * sum(p // PAGE_SIZE + 1 for p in positions if p >= 0)


class SharedRows:
    """The plans of one step: the sequence (a place in ``slots``) and the position of every row.  ``drafted``: a sequence brings
    several tokens, for which the kernels of prompts would walk its pages with a tile hardly filled: any sharing pays."""

    def __init__(self, engine, slots: Sequence[int], seqs: Sequence[int], positions: Sequence[int], drafted: bool):
        self.engine, self.slots, self.seqs, self.positions = engine, slots, seqs, positions
        self._least = 0 if drafted else LEAST_BYTES
        self._trees: Dict[int, Optional[tuple]] = {}
        self._plans: Dict[PlanKey, Optional[ops.SharedPlan]] = {}

    def plan(self, *key) -> Optional[ops.SharedPlan]:
        if key not in self._plans:
            group, e = key[0], self.engine
            if group not in self._trees:
                self._trees[group] = shared_tree(e.cache, group, self.slots, self.seqs, self.positions, self._least)
            tree = self._trees[group]
            pays = tree is not None and (self._least == 0 or heads_share(tree, self.positions, key, e.dtype))
            self._plans[key] = ops.attention_shared_plan_of(
                *tree, self.seqs, self.positions, *key[1:], e.dtype, e.device) if pays else None
        return self._plans[key]


class KeptPlans:
    """The plans of a captured step of ``rows`` rows: each as large as ``rooms`` says, its contents replaced by ``fill``."""

    def __init__(self, engine, rows: int, cols: int, rooms: Sequence[Tuple[PlanKey, tuple]]):
        self.plans = {key: ops.SharedPlan.with_room(rows, *key[1:], engine.dtype, engine.device, room, cols) for key, room in rooms}
        self._filled = None

    def plan(self, *key) -> Optional[ops.SharedPlan]:
        return self.plans.get(key)

    def fill(self, units: Dict[PlanKey, tuple]) -> None:
        if units is not self._filled:
            for key, plan in self.plans.items():
                plan.fill(*units[key])
            self._filled = units


class BatchUnits:
    """What a batch of single tokens shares, for captured steps: made anew when its sequences or what they share have
    changed, or when they grow beyond what it reaches.  ``drafted``: the rows are tokens of one sequence, which share whatever they see alike."""

    def __init__(self, engine, drafted: bool = False):
        self.engine, self.drafted = engine, drafted
        self._made_for = self._positions = self._units = None
        self._until = 0

    def units(self, slots: Sequence[int], positions: Sequence[int], rows: int, ahead: Optional[int] = None) -> Optional[Dict[PlanKey, tuple]]:
        """Per attention of the model that gains by it, its units, members and record offsets, for ``rows`` rows of which
        the first are the sequences; None where none gains.  ``ahead``: they cover as many pages beyond these positions, for a
        caller that does not ask again while its sequences grow; None: these positions, for one that asks at every step."""
        cache = self.engine.cache
        if not self.drafted and (len(slots) < 2 or not cache.shares_pages()):
            return None
        made_for = (tuple(slots), None if self.drafted else cache.share_epoch, rows)  # (a plan names columns of a table, not pages)
        reach = (ahead or 0) * PAGE_SIZE
        if made_for == self._made_for and all(0 <= now - then <= self._until - reach for now, then in zip(positions, self._positions)):
            return self._units
        ahead = AHEAD if ahead is None else ahead
        seqs, padding = list(range(len(slots))), rows - len(slots)
        trees: Dict[int, Optional[tuple]] = {}
        units = {}
        for key in self.engine.model.shared_keys():
            if key[0] not in trees:
                trees[key[0]] = shared_tree(cache, key[0], slots, seqs + [0] * padding, list(positions) + [-1] * padding,
                                              0 if self.drafted else LEAST_BYTES, ahead)
            if trees[key[0]] is not None and (self.drafted or heads_share(trees[key[0]], positions, key, self.engine.dtype, ahead)):
                units[key] = ops.attention_shared_units(*trees[key[0]], seqs + [0] * padding, *key[1:], self.engine.dtype,
                                                        self.engine.device)
        self._made_for, self._positions, self._until = made_for, list(positions), ahead * PAGE_SIZE
        self._units = units or None
        return self._units


def rooms_of(units: Optional[Dict[PlanKey, tuple]]) -> Optional[tuple]:
    """The sizes, in powers of two, of plans that hold these units: part of a captured step's key."""
    if units is None:
        return None
    up = lambda n: 0 if n == 0 else 1 << (n - 1).bit_length()
    return tuple(sorted((key, (*(up(len(k)) for k in kinds), up(max(1, len(members))), up(max(1, int(record[-1])))))
                        for key, (kinds, members, record) in units.items()))
