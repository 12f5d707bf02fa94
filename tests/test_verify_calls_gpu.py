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
