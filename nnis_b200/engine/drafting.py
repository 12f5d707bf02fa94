"""Where drafted tokens come from, for ``InferenceSession.generate_drafted``.

A drafter proposes the next few tokens of a sequence; the session runs them in one step with the token
before them, keeps those that the target model keeps (``sampling.device.verify_drafts``), takes one more
from the target's own distribution and forgets the rest.  The tokens are distributed as the target's
alone, whatever the drafter proposes; a good one makes several of them a step.
"""
from __future__ import annotations

from typing import Dict, List, Optional, Sequence, Tuple

import torch

from ..sampling import SplitMix64
from ..sampling import device as device_sampling


CAPTURED = 16  # most tokens that a drafting model takes by a captured step


class LookupDrafter:
    """Drafts what followed the last time that the sequence's last ``ngram`` tokens (or fewer, down to one) came up in it."""

    def __init__(self, ngram: int = 3):
        if ngram < 1:
            raise ValueError(f"ngram must be positive; got {ngram}")
        self.ngram = ngram
        self.begin()

    def begin(self) -> None:
        """A new sequence."""
        self._after: Dict[Tuple[int, ...], int] = {}  # tokens -> the place behind their last occurrence
        self._seen: List[int] = []

    def propose(self, tokens: Sequence[int], count: int, temperature: float) -> Tuple[List[int], Optional[torch.Tensor]]:
        """At most ``count`` tokens to follow ``tokens``, and the logits that they were drawn from (None: drawn from none)."""
        tokens = list(tokens)
        if tokens[:len(self._seen)] != self._seen:
            self.begin()
        # (the last token is followed by nothing yet: runs that end with it are entered when it is)
        for end in range(max(1, len(self._seen)), len(tokens)):
            for n in range(1, min(self.ngram, end) + 1):
                self._after[tuple(tokens[end - n:end])] = end
        self._seen = tokens
        for n in range(min(self.ngram, len(tokens)), 0, -1):
            at = self._after.get(tuple(tokens[-n:]))
            if at is not None:
                return tokens[at:at + count], None
        return [], None


class SessionDrafter:
    """Drafts with a second, smaller model of the same vocabulary on the same device: an ``LLM`` of its own, a session of which
    follows the sequence.  With a temperature its tokens are drawn at that temperature, from a generator of the drafter's own
    (``seed``, of a stream that no policy's seed gives), and come with their logits; greedy drafts are its likeliest tokens."""

    STREAM = 0x6472616674657273  # told apart from policies' seeds by it

    def __init__(self, llm, seed: int = 0):
        if llm.engine.cache.fixed_history():
            raise ValueError("a drafting model goes back over refused tokens: it keeps no state of fixed size and no window")
        self.llm = llm
        self.session = llm.new_session()
        # The verification draws from SplitMix64 of the policy's seed.  With that state here the numbers that drew the drafts would
        # decide about them, too, and what is kept would no longer be distributed as the target's: the state is one mixed from the seed.
        self._rng = device_sampling.seed_states([SplitMix64(seed ^ self.STREAM).next_u64()], llm.engine.device)
        self._held: List[int] = []  # the tokens that the session has executed

    def begin(self) -> None:
        self.session.reset()
        self._held = []

    def close(self) -> None:
        self.session.close()

    def propose(self, tokens: Sequence[int], count: int, temperature: float) -> Tuple[List[int], Optional[torch.Tensor]]:
        from .engine import SequenceStep
        tokens, engine = list(tokens), self.llm.engine
        count = min(count, engine.spec.max_positions - len(tokens))
        if count <= 0:
            return [], None
        same = next((i for i, (a, b) in enumerate(zip(self._held, tokens)) if a != b), min(len(self._held), len(tokens)))
        same = min(same, len(tokens) - 1)  # (the last token's logits are wanted)
        self.session.truncate(same)
        fresh, backend, slot = tokens[same:], self.llm.backend, self.session.slot
        if len(fresh) == 1:
            logits = backend.decode_logits(slot, fresh[0], True)
        elif len(fresh) <= CAPTURED:
            logits = backend.drafted_logits(slot, fresh, True)[-1]
        else:
            logits = engine.step([SequenceStep(slot, fresh, [len(fresh) - 1])])
        vocab, drafts = engine.spec.vocab_size, []
        kept = torch.empty((count, vocab), dtype=torch.float32, device=engine.device) if temperature > 0 else None
        picked = torch.empty(1, dtype=torch.int32, device=engine.device)
        at = torch.full((1,), temperature, dtype=torch.float32, device=engine.device)
        for i in range(count):
            if kept is not None:
                kept[i].copy_(logits.reshape(-1))
                device_sampling.temperature(kept[i:i + 1], at, self._rng, picked)
            else:
                device_sampling.greedy(logits.reshape(1, -1), picked)
            drafts.append(int(picked.item()))
            if i + 1 < count:
                logits = backend.decode_logits(slot, drafts[-1], True)
        self._held = tokens + drafts[:-1]
        return drafts, kept
