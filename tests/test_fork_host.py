"""Sequences that share pages: who holds what, when a page is copied, and that nothing a sequence holds is written by
another (no GPU: the store is host memory, and what a step would write is written by the test)."""
import random

import pytest
import torch

from nnis_b200.cache import PAGE_SIZE, CacheFull, CacheManager, KVRequest, SlotError, StateRequest

D = 2


def make(requests=None, max_tokens=64 * 12, max_slots=6, max_positions=10_000):
    requests = requests if requests is not None else [KVRequest(1, D), KVRequest(1, D)]
    return CacheManager(requests, torch.float32, torch.device("cpu"), max_tokens, max_slots, max_positions)


class Writer:
    """Writes a mark per (sequence's history, position) into every layer's k and v, as a step does, and checks them."""

    def __init__(self, cache):
        self.cache, self.marks, self.next = cache, {}, 1.0

    def acquire(self):
        slot = self.cache.acquire()
        self.marks[slot] = []
        return slot

    def fork(self, slot, length=None):
        new = self.cache.fork(slot, length)
        self.marks[new] = list(self.marks[slot][:self.cache.length(new)])
        return new

    def step(self, counts):
        slots = list(counts)
        lengths = [self.cache.length(s) + n for s, n in counts.items()]
        self.cache.reserve(slots, lengths)
        for s, n in counts.items():
            for _ in range(n):
                at = len(self.marks[s])
                for g in self.cache.groups:
                    page = g.tables[s][at // PAGE_SIZE]
                    for t in (g.k, g.v):
                        if t is not None:
                            t[:, page, :, at % PAGE_SIZE] = self.next
                self.marks[s].append(self.next)
                self.next += 1.0
        self.cache.commit(slots, lengths)

    def truncate(self, slot, length):
        self.cache.truncate(slot, length)
        del self.marks[slot][length:]

    def release(self, slot):
        self.cache.release(slot)
        del self.marks[slot]

    def check(self):
        self.cache.check()
        for s, marks in self.marks.items():
            assert self.cache.length(s) == len(marks)
            for g in self.cache.groups:
                first = g.first_needed_page(len(marks)) * PAGE_SIZE
                for at in range(first, len(marks)):
                    page = g.tables[s][at // PAGE_SIZE]
                    assert page >= 0 and float(g.k[0, page, 0, at % PAGE_SIZE, 0]) == marks[at]
                    assert g.v is None or float(g.v[-1, page, -1, at % PAGE_SIZE, -1]) == marks[at]


def test_a_fork_shares_pages_until_it_writes():
    w = Writer(make())
    a = w.acquire()
    w.step({a: PAGE_SIZE + 5})
    b = w.fork(a)
    c = w.fork(a)
    cache = w.cache
    assert cache.usage()["pages_held"] == [2] and cache.usage()["pages_shared"] == [2]
    assert cache.page_table(0, a) == cache.page_table(0, b) == cache.page_table(0, c)
    version = cache.versions[b]
    w.step({b: 1, c: 1})  # the page is a's, too: both get copies
    assert cache.page_table(0, a)[0] == cache.page_table(0, b)[0] and cache.usage()["pages_held"] == [4]
    assert len({cache.page_table(0, s)[1] for s in (a, b, c)}) == 3 and cache.versions[b] > version
    w.step({a: 1})        # the last holder writes in place
    assert cache.usage()["pages_held"] == [4]
    w.check()
    w.release(a)
    w.check()
    w.release(b)
    w.release(c)
    assert cache.usage()["pages_held"] == [0] and not cache.shares_pages()


def test_all_holders_write_in_one_step():
    """Of n holders of a page n - 1 get copies, the last keeps it."""
    w = Writer(make())
    a = w.acquire()
    w.step({a: 7})
    others = [w.fork(a) for _ in range(3)]
    w.step({s: 2 for s in [a, *others]})
    assert w.cache.usage()["pages_held"] == [4] and not w.cache.shares_pages()
    w.check()


def test_forks_at_an_earlier_length_and_truncated_ones():
    w = Writer(make())
    a = w.acquire()
    w.step({a: 3 * PAGE_SIZE})
    b = w.fork(a, PAGE_SIZE)          # a page end: nothing to copy when it goes on
    w.step({b: 3})
    assert w.cache.page_table(0, b)[0] == w.cache.page_table(0, a)[0] and w.cache.usage()["pages_held"] == [4]
    c = w.fork(a, PAGE_SIZE + 1)
    w.truncate(c, 10)                 # now inside a page that a and b hold
    w.step({c: 1})
    w.step({a: 1, b: 70})
    w.check()
    empty = w.fork(a, 0)
    w.step({empty: 1})
    w.check()
    w.truncate(a, 5)                  # a's own first page is b's as well
    w.step({a: 2})
    w.check()


def test_a_fork_that_does_not_fit_changes_nothing():
    w = Writer(make(max_tokens=PAGE_SIZE * 2, max_slots=2))
    a = w.acquire()
    w.step({a: 70})
    b = w.fork(a)
    with pytest.raises(CacheFull):
        w.fork(a)
    before = (list(w.cache.page_table(0, a)), list(w.cache.page_table(0, b)), w.cache.versions[:], w.cache.epoch)
    with pytest.raises(CacheFull):
        w.cache.reserve([b], [71])    # its copy has no page
    with pytest.raises(CacheFull):
        w.cache.reserve([a, b], [71, 71])
    assert before == (list(w.cache.page_table(0, a)), list(w.cache.page_table(0, b)), w.cache.versions[:], w.cache.epoch)
    w.check()
    w.release(a)
    w.step({b: 1})
    w.check()


def test_refusals():
    w = Writer(make())
    a = w.acquire()
    w.step({a: 10})
    for bad in (11, -1):
        with pytest.raises(SlotError):
            w.cache.fork(a, bad)
    with pytest.raises(SlotError):
        w.cache.fork(5)
    w.check()


def test_states_are_copied_and_fork_where_they_are():
    c = make([KVRequest(1, D), StateRequest((3,), torch.float32, (((2, 2), torch.float32),))])
    a = c.acquire()
    c.reserve([a], [9])
    c.commit([a], [9])
    view = c.view(1)
    view.state[a] = 5.0
    view.extra[0][a] = 6.0
    b = c.fork(a)
    assert bool((view.state[b] == 5.0).all()) and bool((view.extra[0][b] == 6.0).all())
    view.state[b] = 1.0
    assert bool((view.state[a] == 5.0).all())
    with pytest.raises(SlotError):
        c.fork(a, 3)
    c.check()


def test_windowed_groups_give_shared_pages_back_once():
    w = Writer(make([KVRequest(1, D, 40), KVRequest(1, D), KVRequest(1, D, 40, keep_first=3)], max_tokens=64 * 30))
    a = w.acquire()
    w.step({a: 50})
    b = w.fork(a)
    w.step({a: 200})
    w.check()
    w.step({b: 30})
    w.step({b: 130})
    w.check()
    c = w.fork(b)
    with pytest.raises(SlotError):
        w.cache.fork(b, 60)  # the window's pages before it are gone
    w.step({c: 1, b: 100, a: 64})
    w.check()
    for s in (a, b, c):
        w.release(s)
    assert w.cache.usage()["pages_held"] == [0, 0, 0]
    w.cache.check()


def test_compact_moves_held_pages_to_the_lowest_places():
    w = Writer(make([KVRequest(1, D), KVRequest(2, D, values=False)], max_tokens=64 * 12))
    slots = [w.acquire() for _ in range(4)]
    for s in slots:
        w.step({s: 2 * PAGE_SIZE + 3})
    f = w.fork(slots[3])
    w.release(slots[0])
    w.release(slots[2])
    versions = w.cache.versions[:]
    assert w.cache.compact() == [3, 3]
    for g in w.cache.groups:
        assert sorted({p for t in g.tables.values() for p in t}) == list(range(g.pool.held)) == list(range(6))
    assert w.cache.page_table(0, f) == w.cache.page_table(0, slots[3]) and w.cache.versions[f] > versions[f]
    w.check()
    assert w.cache.compact() == [0, 0]
    w.step({f: 1, slots[1]: 64, slots[3]: 1})
    w.check()


def test_snapshots_of_forked_sequences():
    w = Writer(make())
    a = w.acquire()
    w.step({a: 20})
    snap = w.cache.snapshot(a)
    b = w.fork(a)
    w.step({a: 60})
    w.cache.restore(snap)
    del w.marks[a][20:]
    w.check()
    w.step({a: 1, b: 1})
    w.check()


@pytest.mark.parametrize("seed", range(25))
def test_any_order_of_forks_steps_truncations_releases_and_moves(seed):
    rng = random.Random(seed)
    w = Writer(make([KVRequest(1, D), KVRequest(1, D, values=False)], max_tokens=64 * 24, max_slots=7))
    for _ in range(120):
        held = list(w.marks)
        kind = rng.choice(("new", "fork", "fork", "step", "step", "step", "truncate", "release", "compact"))
        try:
            if kind == "new":
                w.acquire()
            elif kind == "fork" and held:
                s = rng.choice(held)
                w.fork(s, rng.choice((None, rng.randrange(0, w.cache.length(s) + 1))))
            elif kind == "step" and held:
                some = rng.sample(held, rng.randrange(1, len(held) + 1))
                w.step({s: rng.choice((1, 1, 5, 64, 90)) for s in some})
            elif kind == "truncate" and held:
                s = rng.choice(held)
                w.truncate(s, rng.randrange(0, w.cache.length(s) + 1))
            elif kind == "release" and held:
                w.release(rng.choice(held))
            elif kind == "compact":
                w.cache.compact()
        except CacheFull:
            pass
        w.check()
    for s in list(w.marks):
        w.release(s)
    assert w.cache.usage()["pages_held"] == [0, 0] and not w.cache.shares_pages()


# ---- the generation loop above it ------------------------------------------------------------------
def test_prompts_that_begin_alike_run_that_once():
    from nnis_b200.engine.generate import GenerationConfig, GenerationRequest, pages_needed, plan_batches, prefix_groups
    from test_generation_host import ScriptedBackend, expected, gen

    class Forking(ScriptedBackend):
        def fork_slot(self, slot):
            new = self.acquire_slot()
            self.held[new] = list(self.held[slot])
            return new

    long = [(i * 7) % 50 for i in range(70)]
    prompts = [long + [1, 2], [3], long + [1], long + [1, 2], [5] * 70, long[:PAGE_SIZE]]
    reqs = [GenerationRequest(p, GenerationConfig(4)) for p in prompts]
    assert prefix_groups(reqs, range(6)) == [([0, 2, 3], 70)]
    assert prefix_groups(reqs, [0, 3]) == [([0, 3], 71)]  # (each keeps a token of its own)
    b = Forking()
    res = gen(b, max_batch=8).generate(reqs, share_prefix=True)
    assert [r.token_ids for r in res] == [expected(p, 4) for p in prompts] and not b.held
    assert [n for _, n in b.steps[0]] == [70] and sorted(n for _, n in b.steps[1]) == [1, 1, 2, 2, 64, 70]
    plain = ScriptedBackend()
    assert [r.token_ids for r in gen(plain, max_batch=8).generate(reqs)] == [r.token_ids for r in res]
    assert len(plain.steps[0]) == 6

    pages = [pages_needed(r) for r in reqs]
    assert pages == [2, 1, 2, 2, 2, 2]
    assert plan_batches(reqs, [True] * 6, 8, 5) == [[0, 1, 2], [3, 4], [5]]
    assert plan_batches(reqs, [True] * 6, 8, 5, True) == [[0, 1, 2, 3], [4, 5]]  # 2 + 1 + 1 + 1
    # a batch whose shared prompt fails is run request by request, without sharing
    b = Forking(fail_on_step=1)
    res = gen(b).generate(reqs[:3], share_prefix=True)
    assert [r.token_ids for r in res] == [expected(p, 4) for p in prompts[:3]] and not b.held


def test_drafts_looked_up_in_the_text():
    from nnis_b200 import LookupDrafter
    d = LookupDrafter(2)
    assert d.propose([1, 2, 3, 4, 1, 2], 3, 0.0) == ([3, 4, 1], None)
    assert d.propose([1, 2, 3, 4, 1, 2, 3], 2, 0.0) == ([4, 1], None)
    assert d.propose([1, 2, 3, 4, 1, 2, 3, 9], 2, 0.0) == ([], None)
    assert d.propose([7, 7], 5, 0.0) == ([7], None)  # another sequence
    d.begin()
    assert d.propose([5], 2, 0.0) == ([], None)
    with pytest.raises(ValueError):
        LookupDrafter(0)


def test_the_command_line_shares_prefixes_of_batches_only():
    from nnis_b200.cli.main import UsageError, parse_args
    batch = ["generate-batch", "--model", "m", "--prompt-ids", "1,2", "--prompt-ids", "1,3", "--seed", "1", "--seed", "2"]
    assert not parse_args(batch).share_prefix and parse_args([*batch, "--share-prefix"]).share_prefix
    with pytest.raises(UsageError):
        parse_args(["generate", "--model", "m", "--prompt-ids", "1,2", "--share-prefix"])
