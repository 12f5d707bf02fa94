"""Verification of drafts, called as a program may call it."""
import pytest
import torch

from test_verify_drafts_gpu import make_case, plain, run

pytestmark = pytest.mark.gpu
LOW, HIGH = -(1 << 31), (1 << 31) - 1


@pytest.mark.parametrize("model", [True, False])
@pytest.mark.parametrize("first", [[0, LOW, 6], [0, HIGH, 6], [LOW, 3, 6], [HIGH, 3, 6], [0, LOW + 1, LOW], [0, 3, HIGH], [LOW, LOW, LOW],
                                   [HIGH, HIGH, HIGH], [LOW, HIGH, LOW], [0, 3, LOW], [1, LOW + 1, 6]])
def test_offsets_at_the_ends_of_their_type(first, model):
    """Sequences whose offsets no packed rows have give 0 and -1; one whose own are good is answered."""
    case = make_case(31, [2, 2], 301, model=model)
    want = plain(*case)
    accepted, picked = run(*case, first=first)
    for b, good in enumerate(([0, 3], [3, 6])):
        got = (accepted[b], picked[b])
        if first[b:b + 2] == good:
            assert got == (want[0][b], want[1][b])
        else:
            assert got == (0, -1)


@pytest.mark.parametrize("model", [True, False])
@pytest.mark.parametrize("counts", [[32766], [9000, 0, 9000, 3]])
def test_as_many_drafts_as_a_call_takes(counts, model):
    """Drafts are kept for thousands of rows, then refused."""
    logits, counts, drafts, temps, accept, picks, draft_logits = make_case(41, counts, 23, model=model)
    at = 0
    for n in counts:
        accept[at:at + n // 2] = [0.0] * (n // 2)
        at += n
    case = (logits, counts, drafts, temps, accept, picks, draft_logits)
    assert run(*case) == plain(*case)


@pytest.mark.parametrize("model", [True, False])
def test_as_many_sequences_as_a_call_takes(model):
    """32,767 of them without drafts."""
    n, g = 32767, torch.Generator().manual_seed(43)
    case = (3.0 * torch.randn((n, 23), generator=g), [0] * n, [], [0.8] * n, [], torch.rand(n, generator=g, dtype=torch.float64).tolist(),
            torch.zeros((0, 23)) if model else None)
    assert run(*case) == plain(*case)


def test_more_rows_than_a_call_takes_are_refused():
    from nnis_b200.csrc.ops import KernelError
    with pytest.raises(KernelError, match="32,767"):
        run(*make_case(42, [32767], 3, model=False))
