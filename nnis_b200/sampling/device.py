"""Picking tokens on the device: greedy argmax for any batch, and seeded
temperature sampling whose generator state lives beside the batch on the GPU.
The kernels are in ``csrc/sampling.cu``."""
from __future__ import annotations

from typing import Optional

import torch

from ..csrc import ops
from .config import SamplingConfig, SamplingError
from .host import SplitMix64


def greedy(logits: torch.Tensor, out: torch.Tensor) -> torch.Tensor:
    """int32 ids of the largest logit per row; ties go to the lower id."""
    ops.argmax(logits, out)
    return out


def seed_states(seeds, device) -> torch.Tensor:
    """SplitMix64 states (the seeds themselves) as an int64 device tensor."""
    signed = [s - (1 << 64) if s >= (1 << 63) else s for s in seeds]
    return torch.tensor(signed, dtype=torch.int64, device=device)


def temperature(logits: torch.Tensor, temperatures: torch.Tensor, rng_state: torch.Tensor,
                out: torch.Tensor) -> torch.Tensor:
    ops.sample_temperature(logits, temperatures, rng_state, out)
    return out


def verify_drafts(logits: torch.Tensor, drafts: torch.Tensor, first_row: torch.Tensor, temperatures: torch.Tensor,
                  accept_draws: torch.Tensor, pick_draws: torch.Tensor, accepted: torch.Tensor, picked: torch.Tensor,
                  draft_logits: Optional[torch.Tensor], workspace) -> None:
    """Which drafted tokens the target keeps, and the token after them, from given random numbers.

    Sequence b has k drafts and k + 1 packed rows of ``logits`` (float32 [rows, vocab]; row i follows i drafts),
    from ``first_row[b]`` on (int32, one number more than sequences, the last one the number of rows).  ``drafts`` (int32),
    ``accept_draws`` (float64 in [0, 1)) and ``draft_logits`` (float32 [drafts, vocab], what the drafts were drawn from
    at the same temperature; None: nobody drew them) are packed the same way without the sequences' last rows.
    With p and q the softmax of the rows over the temperature, a draft is kept iff draw * q(draft) < p(draft)
    (q = 1 without draft logits).  ``accepted[b]`` (int32): the drafts before the first that is not kept; ``picked[b]``
    (int32): the token after them, drawn with ``pick_draws[b]`` (float64) in id order from max(p - q, 0) where a draft was
    not kept and from p where all were (a draw outside [0, 1] is taken for its next end, NaN for 0).  Temperature 0 (or less): a draft is kept iff it is the argmax, which is also the pick.
    An id outside the vocabulary is never kept.  A row without probability (all logits -inf, a NaN or +inf among
    them) ends its sequence there: picked is -1.  Offsets that no packed rows have give 0 and -1."""
    ops.verify_drafts(logits, drafts, first_row, temperatures, accept_draws, pick_draws, accepted, picked, draft_logits,
                      workspace)


class DraftVerifier:
    """``verify_drafts`` for one sequence whose drafts are host numbers: draws from a SplitMix64 of the policy's seed, an
    accept draw a draft and then the pick's, every time; without a policy greedy."""

    def __init__(self, device, workspace, sampling: Optional[SamplingConfig]):
        self.device, self.workspace = device, workspace
        self.temperature = 0.0 if sampling is None else float(sampling.temperature)
        self._rng = SplitMix64(0 if sampling is None else sampling.seed)
        self._temperatures = torch.full((1,), self.temperature, dtype=torch.float32, device=device)
        self._out = torch.empty((2, 1), dtype=torch.int32, device=device)

    def verify(self, logits: torch.Tensor, drafts, draft_logits: Optional[torch.Tensor]):
        """(drafts kept, the token after them) by the logits' k + 1 rows; ``SamplingError`` where a row has no probability."""
        k = len(drafts)
        draws = torch.tensor([self._rng.next_unit_f64() for _ in range(k + 1)], dtype=torch.float64, device=self.device)
        ints = torch.tensor([*drafts, 0, k + 1], dtype=torch.int32, device=self.device)
        verify_drafts(logits, ints[:k], ints[k:], self._temperatures, draws[:k], draws[k:], self._out[0], self._out[1],
                      draft_logits, self.workspace)
        kept, token = self._out.reshape(-1).tolist()
        if token < 0:
            raise SamplingError("sampling softmax produced no positive finite probability mass")
        return kept, token
