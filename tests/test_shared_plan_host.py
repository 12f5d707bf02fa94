"""The plans of attention over shared pages: every key that a row sees is in one unit, once, read by the row's own page id
(no GPU)."""
import random

import pytest

from nnis_b200.csrc.shared_plan import PAGE, shared_nodes, shared_units

NONE = (0, 0, 0, 0, False)
# (most entries, CTAs at once, fewest and most pages of a chunk, from a queue) per kind
KINDS = [((16, 600, 1, 16, True), (32, 400, 4, 16, False), (128, 300, 2, 1 << 20, False)),
         (NONE, (32, 8, 2, 16, False), (128, 8, 2, 100, False)),
         ((16, 8, 1, 3, True), (64, 600, 2, 16, False), NONE), ((16, 1, 4, 16, False), (64, 1, 4, 16, False), NONE)]


def batch(seed):
    rng = random.Random(seed)
    tables, nxt = [], 0
    for _ in range(rng.randrange(1, 12)):
        begin = rng.choice(tables) if tables and rng.random() < 0.7 else []
        t = list(begin[:rng.randrange(0, len(begin) + 1)])
        for _ in range(rng.randrange(0 if t else 1, 6)):
            t.append(nxt)
            nxt += 1
        tables.append(t)
    seqs, positions = [], []
    for i, t in enumerate(tables):
        top = rng.randrange(0, len(t) * PAGE)
        for j in range(rng.choice((1, 1, 2, 5))):
            seqs.append(i)
            positions.append(max(0, top - j) if rng.random() < 0.9 else -1)
    return rng, tables, seqs, positions


@pytest.mark.parametrize("ahead", [0, 3])
@pytest.mark.parametrize("kinds", KINDS)
def test_every_visible_key_is_in_one_unit(kinds, ahead):
    for seed in range(60):
        rng, tables, seqs, positions = batch(seed)
        group = rng.choice((1, 3, 5, 20, 40))
        nodes, tails = shared_nodes(tables, seqs, positions, ahead)
        units, members, record = shared_units(nodes, tails, seqs, group, rng.choice((1, 3, 32)), kinds, 1)
        keys, slots = {}, set()
        for kind, (most, *_) in zip(units, kinds):
            for at, first, count, begin, end, slot, seq, ends in kind.tolist():
                assert 0 < count <= most and (end > begin or (begin, end) == (0, 0) and ends)
                for e in range(first, first + count):
                    row, head = int(members[at + e // group]), e % group
                    assert not ends or ends == 1 + row
                    assert record[row] + slot < record[row + 1] and (row, head, slot) not in slots
                    slots.add((row, head, slot))
                    for page in range(begin, end):
                        seen = positions[row] + 1 - page * PAGE
                        if ends and seen <= 0:
                            continue  # (room to grow)
                        assert tables[seq][page] == tables[seqs[row]][page] and (row, head, page) not in keys
                        assert ends or seen >= PAGE  # (nothing is hidden in pages that rows share)
                        keys[row, head, page] = min(PAGE, seen)
        for row, pos in enumerate(positions):
            assert record[row + 1] > record[row]
            for head in range(group):
                assert sum(keys.get((row, head, p), 0) for p in range(len(tables[seqs[row]]))) == pos + 1
                assert sum((row, head, s) in slots for s in range(record[row + 1] - record[row])) == record[row + 1] - record[row]


def test_what_is_shared_and_what_is_not():
    shared = list(range(10))
    tables = [shared + [20], shared + [21, 22], shared[:4] + [30], [40, 41]]
    nodes, tails = shared_nodes(tables, [0, 1, 2, 3], [650, 700, 300, 100])
    assert nodes == [([0, 1, 2], 0, 4), ([0, 1], 4, 10)]
    assert sorted(tails) == [(0, 10, 11), (1, 10, 11), (2, 4, 5), (3, 0, 2)]
    # several tokens of a sequence see its whole pages alike; a page that ends inside them is each one's own
    nodes, tails = shared_nodes([[5, 6, 7]], [0, 0, 0], [126, 127, 128])
    assert nodes == [([0, 1, 2], 0, 1), ([1, 2], 1, 2)] and sorted(tails) == [(0, 1, 2), (2, 2, 3)]


def test_chunks_fit_the_device_where_they_can():
    """A kind's CTAs are no more than it has at once unless its pieces alone are."""
    tables = [list(range(62)) + [100 + r] for r in range(24)]
    nodes, tails = shared_nodes(tables, range(24), [62 * PAGE + 9] * 24)
    units, _, _ = shared_units(nodes, tails, range(24), 1, 32, ((16, 1776, 1, 16, True), (32, 444, 4, 16, False),
                                                                          (128, 296, 2, 1 << 20, False)), 1)
    assert len(units[1]) * 32 <= 444 and sum(u[4] - u[3] for u in units[1].tolist()) == 62
    assert len(units[0]) == 24


def test_entry_points_refuse_empty_records():
    """Argument errors are found before anything is launched; numbers that no field holds are the caller's error."""
    from nnis_b200.csrc import ops
    for name, fields in ops._ENTRY_FIELDS.items():
        call = ops._entry(name)
        zeros = [0.0 if c == "f" else 0 for c in fields]
        assert call(*zeros) == -1
        for i, c in enumerate(fields):
            with pytest.raises(ops.KernelError):
                call(*zeros[:i], {"p": 1 << 64, "i": 1 << 31, "f": "one"}[c], *zeros[i + 1:])
