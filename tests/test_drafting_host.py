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
