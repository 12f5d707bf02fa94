"""Kept plans of shared pages reach as far as the generation that runs by them (no GPU: what a captured step would do is
recorded, and the plan that it would do it by looked at)."""
from types import SimpleNamespace

import pytest
import torch

from nnis_b200.cache import PAGE_SIZE, CacheManager, KVRequest, SlotError
from nnis_b200.csrc import ops
from nnis_b200.engine import sharing
from nnis_b200.engine.api import EngineBackend
from nnis_b200.engine.generate import GenerationConfig, GenerationRequest, Generator

HEADS, KV_HEADS, DIM, VOCAB = 4, 2, 2, 50


def last_keys(units, rows):
    """Per row, the end of the pages that its units cover."""
    (kinds, members, _), = units.values()
    group, ends = HEADS // KV_HEADS, [0] * rows
    for kind in kinds:
        for at, first, count, begin, end, *_ in kind.tolist():
            for e in range(first, first + count):
                row = int(members[at + e // group])
                ends[row] = max(ends[row], end)
    return [e * PAGE_SIZE for e in ends]


class Recorder:
    """A captured step: which rows it runs, and the units it runs them by."""

    def __init__(self, rows):
        self.rows, self.positions, self.tokens, self.reach, self.launches = rows, {}, {}, None, 0
        self.picked, self.logits, self.plans = torch.zeros(rows, dtype=torch.int32), None, self

    def fill(self, units):
        self.reach = last_keys(units, self.rows)

    def upload(self, tokens, positions, slots):
        self.positions = dict(enumerate(positions))
        return 0

    def set_row(self, row, slot, token, position):
        self.positions[row] = position

    def clear_row(self, row):
        self.positions.pop(row, None)

    def sync_pages(self, row, slot):
        pass

    def launch(self):
        self.launches += 1
        for row, position in self.positions.items():
            assert position < self.reach[row], f"row {row}: keys end at {self.reach[row]}, its own lies at {position}"
            self.positions[row] = position + 1
            self.picked[row] = (7 * position + row) % VOCAB

    def picks_to_host(self, into):
        into.copy_(self.picked)
        return SimpleNamespace(synchronize=lambda: None)


class Backend(EngineBackend):
    def __init__(self, engine):
        super().__init__(engine)
        self._pinned, self.recorders = torch.empty((2, 64), dtype=torch.int32), {}

    def _decoder(self, rows, max_context, want_logits=False, rooms=None):
        assert rooms is not None
        return self.recorders.setdefault((rows, rooms), Recorder(self._decoder_key(rows, max_context, want_logits)[0]))

    def greedy(self, logits):
        return (self._picked if self._picked is not None else logits.argmax(1)).tolist()


def make_engine(max_tokens=1 << 15):
    cache = CacheManager([KVRequest(KV_HEADS, DIM)], torch.float32, torch.device("cpu"), max_tokens, 16, 1 << 14)

    def step(batch, most):
        slots = [s.slot for s in batch]
        lengths = [cache.length(s.slot) + len(s.tokens) for s in batch]
        cache.reserve(slots, lengths)
        cache.commit(slots, lengths)
        return torch.zeros((sum(len(s.want) for s in batch), VOCAB))

    return SimpleNamespace(
        cache=cache, model=SimpleNamespace(blocks=[], shared_keys=lambda: [(0, HEADS, KV_HEADS, DIM)], all_share=True),
        spec=SimpleNamespace(vocab_size=VOCAB, max_positions=1 << 14), device=torch.device("cpu"), dtype=torch.float32,
        step_in_portions=step, acquire_slot=cache.acquire, release_slot=cache.release, fork=cache.fork)


@pytest.fixture(autouse=True)
def share_whatever_can_be(monkeypatch):
    monkeypatch.setattr(sharing, "LEAST_BYTES", 1)
    monkeypatch.setattr(sharing, "PAGE_COST", {})
    monkeypatch.setattr(ops, "sm_count", lambda device: 148)


@pytest.mark.parametrize("last", [1, 5])
@pytest.mark.parametrize("new", [1, 40, 575, 1000])
def test_greedy_generation_behind_a_shared_prompt_sees_its_newest_keys(new, last):
    """Prompts that have one token (or five) of their own behind what they share, far beyond the room of a step's plan."""
    engine = make_engine()
    backend = Backend(engine)
    prompt = [i % VOCAB for i in range(1001)]
    requests = [GenerationRequest(prompt + [i] * last, GenerationConfig(new)) for i in range(8)]
    results = Generator(backend, VOCAB, 1 << 14, 8, 1 << 15).generate(requests, share_prefix=True)
    assert [r.error for r in results] == [None] * 8 and [len(r.token_ids) for r in results] == [new] * 8
    assert sum(r.launches for r in backend.recorders.values()) == new - (1 if last > 1 else 0)
    assert engine.cache.usage()["pages_held"] == [0]


def test_units_that_are_kept_reach_as_far_as_they_are_asked_to():
    engine = make_engine()
    cache = engine.cache
    a = cache.acquire()
    cache.reserve([a], [641])
    cache.commit([a], [641])
    slots, kept = [a, cache.fork(a)], sharing.BatchUnits(engine)

    def reach(at, *ahead):
        units = kept.units(slots, [at, at], 2, *ahead)
        return units, min(last_keys(units, 2))

    first, end = reach(640)
    assert end >= 641
    for at in (650, 700, 640 + sharing.AHEAD * PAGE_SIZE):  # (made anew only where they end)
        assert reach(at)[0] is first and reach(at)[1] > at
    again, end = reach(660, 16)
    assert again is not first and end >= 660 + 16 * PAGE_SIZE
    assert reach(660, 16)[0] is again and reach(900)[0] is again and reach(660, 3)[0] is again
    further, end = reach(700, 16)
    assert further is not again and end >= 700 + 16 * PAGE_SIZE


@pytest.mark.parametrize("fails", ["buffers", "capture"])
def test_drafted_steps_that_cannot_be_captured_are_launched_kernel_by_kernel(monkeypatch, fails):
    """No memory for a captured step's buffers, or for its graph: a warning, the step by the engine, and no second try."""
    from nnis_b200.engine import api
    engine = make_engine()
    tries, steps = [], []

    class Fails:
        graph = None

        def __init__(self, *a, **k):
            tries.append(1)
            if fails == "buffers":
                raise torch.cuda.OutOfMemoryError("out of memory")
            self.plans = SimpleNamespace(fill=lambda units: None)

        def upload(self, *a):
            return 0

        def capture(self):
            raise RuntimeError("out of memory")

        launch = capture

    def step(batch, drafted=False):
        assert drafted
        steps.append([(s.slot, list(s.tokens), list(s.want)) for s in batch])
        engine.step_in_portions(batch, 100)
        return "logits"

    monkeypatch.setattr(api, "GraphDecoder", Fails)
    engine.step = step
    backend = EngineBackend(engine)
    slot = engine.acquire_slot()
    engine.cache.reserve([slot], [100])
    engine.cache.commit([slot], [100])
    with pytest.warns(RuntimeWarning, match="could not be captured"):
        assert backend.drafted_logits(slot, [1, 2, 3], True) == "logits"
    assert backend.drafted_logits(slot, [4, 5, 6], True) == "logits"
    assert steps == [[(slot, [1, 2, 3], [0, 1, 2])], [(slot, [4, 5, 6], [0, 1, 2])]]
    assert len(tries) == 1 and not backend._decoders and engine.cache.length(slot) == 106
    engine.cache.check()


@pytest.mark.parametrize("share", [True, False])
def test_pages_stay_where_they_are_while_a_generation_shares_them(share):
    """A callback that compacts the cache after the sequence has ended by whose table the others read what they share: refused, with
    nothing moved; without shared pages, and afterwards, they move."""
    engine = make_engine()
    cache = engine.cache

    class Plain(Recorder):
        def launch(self):
            self.reach = {r: 1 << 20 for r in range(self.rows)}
            super().launch()

    class AnyBackend(Backend):
        def _decoder(self, rows, max_context, want_logits=False, rooms=None):
            made = (Recorder if rooms else Plain)(self._decoder_key(rows, max_context, want_logits)[0])
            if not rooms:
                made.plans = None
            return made

    first = cache.acquire()  # (its pages lie in front of the generation's, and are given back in the middle of it)
    cache.reserve([first], [300])
    cache.commit([first], [300])
    seen, refused, moved = [0] * 4, [], []

    def on_token(i, token):
        seen[i] += 1
        if i == 1 and seen[i] == 20:
            cache.release(first)
            before = [list(t) for t in cache.groups[0].tables.values()]
            try:
                moved.append(cache.compact())
            except SlotError:
                refused.append(before == [list(t) for t in cache.groups[0].tables.values()])

    prompt = [i % VOCAB for i in range(1001)]
    requests = [GenerationRequest(prompt + [i], GenerationConfig(5 if i == 0 else 40)) for i in range(4)]
    results = Generator(AnyBackend(engine), VOCAB, 1 << 14, 8, 1 << 15).generate(requests, on_token, share_prefix=share)
    assert [r.error for r in results] == [None] * 4
    assert (refused, len(moved)) == (([True], 0) if share else ([], 1))
    slot = cache.acquire()
    assert cache.compact() == [0] and cache.usage()["pages_held"] == [0]
    cache.release(slot)
    cache.check()


@pytest.mark.parametrize("tokens,most", [(2, 1), (5, 1), (64, 1), (64, 4), (100, 100)])
def test_drafted_steps_are_captured_whatever_the_batch(monkeypatch, tokens, most):
    """A model for one sequence (``max_batch=1``), or for many, takes a token and its drafts by a captured step."""
    from nnis_b200.engine import api
    engine = make_engine()
    monkeypatch.setattr(api, "GraphDecoder", lambda engine, rows, context, want_logits, rooms: made.append(rows) or Drafted(rows))
    made, launched = [], []

    class Drafted(Recorder):
        graph, capture = None, lambda self: None

        def launch(self):
            launched.append(dict(self.positions))
            self.logits = torch.zeros((self.rows, VOCAB))

    backend = EngineBackend(engine, most)
    slot = engine.acquire_slot()
    engine.cache.reserve([slot], [100])
    engine.cache.commit([slot], [100])
    assert backend.drafted_logits(slot, [3] * tokens, True).shape == (tokens, VOCAB)
    assert launched == [{r: 100 + r for r in range(tokens)}] and made[0] >= tokens
