"""Drafted generation's random numbers and drafters, without a GPU."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from nnis_b200 import SessionDrafter
from nnis_b200.sampling import SplitMix64


def drafter_of(seed):
    """A session drafter of a model that is not there."""
    engine = SimpleNamespace(device=torch.device("cpu"), cache=SimpleNamespace(fixed_history=lambda: False))
    return SessionDrafter(SimpleNamespace(engine=engine, new_session=lambda: None), seed=seed)


def draw(weights, u):
    running = np.cumsum(weights)
    return int(min(np.searchsorted(running, u * running[-1], side="right"), len(weights) - 1))


@pytest.mark.parametrize("offset", [0, 1, -1 << 62])
def test_a_drafter_of_the_policys_seed_draws_numbers_of_its_own(offset):
    """Three tokens of a target p by a drafter q with the policy's own seed (or one beside it), 20,000 seeds: as often as p
    says.  A frequency is within 4.5 standard deviations of its mean, sqrt(p (1 - p) / n) each, for all twelve but once in 12,000
    such tests (normal tails)."""
    p, n, drafts = np.array([0.1, 0.2, 0.3, 0.4]), 20000, 4
    q = p[::-1].copy()
    left = np.maximum(p - q, 0.0)
    counts = np.zeros((3, 4))
    for seed in range(n):
        policy = SplitMix64(seed)
        own = SplitMix64(int(drafter_of(seed + offset)._rng.item()))
        tokens = [draw(p, policy.next_unit_f64())]
        while len(tokens) < 3:
            proposed = [draw(q, own.next_unit_f64()) for _ in range(drafts)]
            numbers = [policy.next_unit_f64() for _ in range(drafts + 1)]  # an accept draw a draft, then the pick's
            kept = next((i for i, d in enumerate(proposed) if not numbers[i] * q[d] < p[d]), drafts)
            tokens += proposed[:kept] + [draw(p if kept == drafts else left, numbers[drafts])]
        for place in range(3):
            counts[place, tokens[place]] += 1
    assert (np.abs(counts / n - p) <= 4.5 * np.sqrt(p * (1 - p) / n)).all(), counts / n


class FakeSession:
    """``InferenceSession.generate_drafted`` over a model that continues every token by the next number."""

    def __init__(self, monkeypatch, vocab=50):
        from nnis_b200.engine import api
        self.length, self.seen = 0, []
        row = lambda tokens: torch.nn.functional.one_hot(torch.tensor([(t + 1) % vocab for t in tokens]), vocab).float()

        def step(batch):
            s, = batch
            self.length += len(s.tokens)
            return row([s.tokens[w] for w in s.want]) if s.want else None

        def drafted(slot, tokens, again):
            self.length += len(tokens)
            return row(tokens)

        def verify(verifier, logits, drafts, draft_logits):
            self.seen.append((len(drafts), None if draft_logits is None else tuple(draft_logits.shape)))
            picks = logits.argmax(1).tolist()
            kept = next((i for i, d in enumerate(drafts) if d != picks[i]), len(drafts))
            return kept, picks[kept]

        engine = SimpleNamespace(cache=SimpleNamespace(fixed_history=lambda: False, length=lambda slot: self.length),
                                 spec=SimpleNamespace(vocab_size=vocab, max_positions=1000), device=torch.device("cpu"), workspace=None,
                                 acquire_slot=lambda: 0, release_slot=lambda slot: setattr(self, "length", 0), step=step,
                                 truncate=lambda slot, n: setattr(self, "length", n))
        backend = SimpleNamespace(drafted_logits=drafted, decode_logits=lambda slot, token, again: drafted(slot, [token], again)[0])
        monkeypatch.setattr(api.device_sampling.DraftVerifier, "verify", verify)
        self.session = api.InferenceSession(SimpleNamespace(engine=engine, backend=backend,
                                                            _generator=SimpleNamespace(refusal=lambda request: None)))


@pytest.mark.parametrize("surplus", [0, 3])
@pytest.mark.parametrize("wrong", [False, True])
def test_drafts_beyond_the_room_are_dropped_with_their_logits(monkeypatch, surplus, wrong):
    """A drafter that gives more tokens than it was asked for, each with its logits, or none but logits all the same."""
    from nnis_b200 import GenerationConfig

    class Drafter:
        begin = lambda self: None

        def propose(self, tokens, count, temperature):
            n = count + surplus if len(tokens) % 3 else 0
            drafts = [(tokens[-1] + 1 + i + (i == 1 and wrong)) % 50 for i in range(n)]
            return drafts, torch.zeros((count + surplus, 50))

    fake = FakeSession(monkeypatch)
    got = fake.session.generate_drafted([5], GenerationConfig(17), Drafter(), drafts=4)
    assert got == list(range(6, 23)) and fake.length == 18
    assert any(n for n, _ in fake.seen) and all(n <= 4 and shape == ((n, 50) if n else None) for n, shape in fake.seen)


def test_a_drafting_model_on_another_device_is_refused(monkeypatch):
    """Its kernels would be launched on this one's: the current device is the model's that runs."""
    from nnis_b200 import GenerationConfig
    fake = FakeSession(monkeypatch)
    fake.session.engine.device = torch.device("cuda:0")
    monkeypatch.setattr("nnis_b200.engine.api.device_sampling.DraftVerifier.__init__", lambda self, *a: setattr(self, "temperature", 0.0))
    drafter = drafter_of(0)
    drafter.llm.spec = SimpleNamespace(vocab_size=50)
    drafter.llm.engine.device = torch.device("cuda:1")
    with pytest.raises(ValueError, match="cuda:1"):
        fake.session.generate_drafted([5], GenerationConfig(4), drafter)
    assert fake.length == 0 and not fake.seen
    drafter.begin, drafter.propose = lambda: None, lambda tokens, count, temperature: ([], None)
    for first in (torch.device("cuda"), "cuda:0", "cuda"):  # (however it is named)
        drafter.llm.engine.device = first
        assert fake.session.generate_drafted([5], GenerationConfig(4), drafter) == [6, 7, 8, 9]
