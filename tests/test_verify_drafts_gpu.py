"""Verification of drafted tokens, against the definition in 64 bits, sequence by sequence."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def run(logits, counts, drafts, temps, accept, picks, draft_logits=None, first=None):
    from nnis_b200.engine.workspace import Workspace
    from nnis_b200.sampling import device
    if first is None:
        first = [0]
        for c in counts:
            first.append(first[-1] + c + 1)
    b = len(counts)
    make = lambda x, t: torch.tensor(x, dtype=t, device=DEV)
    accepted = torch.full((b,), 77, dtype=torch.int32, device=DEV)
    picked = torch.full((b,), 77, dtype=torch.int32, device=DEV)
    device.verify_drafts(logits.to(DEV), make(drafts, torch.int32), make(first, torch.int32), make(temps, torch.float32),
                         make(accept, torch.float64), make(picks, torch.float64), accepted, picked,
                         None if draft_logits is None else draft_logits.to(DEV), Workspace(torch.device(DEV)))
    return accepted.tolist(), picked.tolist()


def plain(logits, counts, drafts, temps, accept, picks, draft_logits=None):
    """numpy float64; no mass: picked -1."""
    z_all, y_all = logits.double().numpy(), None if draft_logits is None else draft_logits.double().numpy()
    vocab = z_all.shape[1]

    def softmax(x, t):
        if np.isnan(x).any() or (x == math.inf).any() or x.max() == -math.inf:
            return None
        with np.errstate(invalid="ignore"):
            e = np.where(x == -math.inf, 0.0, np.exp((x - x.max()) / t))
        return e / e.sum()

    out, row, at = [], 0, 0
    for b, count in enumerate(counts):
        t = float(np.float32(temps[b]))
        a, pick = 0, -1
        while True:
            z = z_all[row + a]
            p = softmax(z, t if t > 0 else 1.0)
            if p is None:
                break
            if not t > 0:
                best = int(np.argmax(z))
                if a < count and drafts[at + a] == best:
                    a += 1
                    continue
                pick = best
                break
            if a == count:
                left = p
            else:
                d = drafts[at + a]
                if y_all is not None:
                    q = softmax(y_all[at + a], t)
                    if q is None:
                        break
                else:
                    q = np.zeros(vocab)
                    if 0 <= d < vocab:
                        q[d] = 1.0
                if 0 <= d < vocab and accept[at + a] * q[d] < p[d]:
                    a += 1
                    continue
                left = np.maximum(p - q, 0.0)
                if left.sum() <= 0:
                    left = p
            running = np.cumsum(left)
            over = np.nonzero((left > 0) & (running > picks[b] * running[-1]))[0]
            pick = int(over[0]) if over.size else int(np.nonzero(left)[0][-1])
            break
        out.append((a, pick))
        row += count + 1
        at += count
    return [x[0] for x in out], [x[1] for x in out]


def make_case(seed, counts, vocab, spread=3.0, model=True, temps=None):
    g = torch.Generator().manual_seed(seed)
    b, drafted = len(counts), sum(counts)
    logits = spread * torch.randn((drafted + b, vocab), generator=g)
    rows = [r for r in range(drafted + b)]
    ends = np.cumsum([c + 1 for c in counts]) - 1
    of_draft = [r for r in rows if r not in set(ends.tolist())]
    draft_logits = None
    temps = temps if temps is not None else [0.8] * b
    if model:
        draft_logits = logits[of_draft] + 0.6 * torch.randn((drafted, vocab), generator=g)
        noise = -torch.log(-torch.log(torch.rand((drafted, vocab), generator=g, dtype=torch.float64).clamp(1e-300, 1 - 1e-16)))
        drafts = torch.argmax(draft_logits.double() / 0.8 + noise, dim=1).tolist()
    else:
        likely = torch.argmax(logits[of_draft], dim=1) if drafted else torch.zeros(0, dtype=torch.long)
        other = torch.randint(0, vocab, (drafted,), generator=g)
        drafts = torch.where(torch.rand(drafted, generator=g) < 0.6, likely, other).tolist()
    accept = torch.rand(drafted, generator=g, dtype=torch.float64).tolist()
    picks = torch.rand(b, generator=g, dtype=torch.float64).tolist()
    return logits, counts, drafts, temps, accept, picks, draft_logits


@pytest.mark.parametrize("vocab", [1, 2, 31, 257, 4099, 49152, 49153, 300001])
@pytest.mark.parametrize("model", [True, False])
@pytest.mark.parametrize("counts", [[0], [1], [4], [3, 0, 0, 7, 1], [2] * 40])
def test_drafts_are_kept_and_tokens_picked_as_defined(vocab, model, counts):
    if vocab > 60000 and sum(counts) > 20:
        counts = counts[:4]
    case = make_case(vocab + sum(counts), counts, vocab, model=model)
    assert run(*case) == plain(*case)


def test_draws_next_to_a_border():
    """An accept draw one step of 64 bits to either side of p / q, and pick draws at a running sum: the sums in 32 bits
    would decide by their rounding.  Two logits make the sums exact: p = 1/4, 3/4 up to 64-bit rounding."""
    vocab = 6000
    z = torch.full((1, vocab), -math.inf)
    z[0, 17], z[0, 5000] = 0.0, 0.0
    y = torch.full((1, vocab), -math.inf)
    y[0, 17] = 1.0
    rows = z.repeat(2, 1)
    for u, keeps in ((0.5 - 1e-13, 1), (0.5, 0), (0.5 + 1e-13, 0)):
        a, p = run(rows, [1], [17], [1.0], [u], [0.25], y)
        # (what is left of (1/2, 1/2) without 17 is the other token alone; a bonus token at 0.25 is 17)
        assert a == [keeps] and p == [17 if keeps else 5000]
    for r, token in ((0.0, 17), (0.5 - 1e-13, 17), (0.5, 5000), (1 - 1e-16, 5000)):
        assert run(z, [0], [], [1.0], [], [r]) == ([0], [token])


def test_many_draws_fall_as_the_64_bit_sums_say():
    """A flat distribution of 49,152 tokens has a border every 2e-5; p and q nearly alike leave little, which 32-bit
    differences would lose."""
    g = torch.Generator().manual_seed(5)
    n, vocab = 24, 49152
    z = 0.3 * torch.randn((2 * n, vocab), generator=g)
    y = z[0::2] + 1e-3 * torch.randn((n, vocab), generator=g)
    drafts = torch.randint(0, vocab, (n,), generator=g).tolist()
    accept, picks = [1.0 - 1e-9] * n, torch.rand(n, generator=g, dtype=torch.float64).tolist()
    case = (z, [1] * n, drafts, [1.0] * n, accept, picks, y)
    got, want = run(*case), plain(*case)
    assert got == want and 0 < sum(want[0]) < n


@pytest.mark.parametrize("model", [True, False])
def test_temperatures_zero_tiny_and_huge(model):
    counts = [3, 3, 2, 3, 1, 2]
    temps = [0.0, 1e-30, 1e-3, 1e30, math.inf, -1.0]
    case = make_case(3, counts, 1031, model=model, temps=temps)
    logits = case[0]
    logits[0, 5] = logits[0, 900] = logits[0].max() + 1.0  # a tie: the lower id
    got, want = run(*case), plain(*case)
    assert got == want
    greedy = make_case(4, [2, 2], 700, model=model, temps=[0.0, 0.0])
    best = torch.argmax(greedy[0], dim=1).tolist()
    kept = list(greedy)
    kept[2] = [best[0], best[1], best[3], (best[4] + 1) % 700]
    assert run(*kept) == ([2, 1], [best[2], best[4]])


def test_masked_logits_and_rows_without_probability():
    """-inf and the type's lowest value are tokens without weight; a row of nothing but them, a NaN or +inf in it, ends
    its sequence with no token; ids outside the vocabulary are never kept; what lies behind is left."""
    vocab, low = 515, torch.finfo(torch.float32).min
    for model in (True, False):
        case = list(make_case(9, [2] * 8, vocab, model=model, temps=[0.9] * 7 + [0.0]))
        z = case[0]
        z[0, 3:400] = -math.inf
        z[3, :] = low
        z[3, 100] = 1.0
        z[6, :] = -math.inf
        z[9, 44] = math.nan
        z[12, 1] = math.inf
        z[22, 8] = math.nan
        case[2][0] = 50       # masked out: never kept
        case[2][9] = vocab    # no token
        case[2][10] = -1
        case[4][0] = 0.0
        got, want = run(*case), plain(*case)
        assert got == want
        assert [want[1][i] for i in (2, 3, 4)] == [-1, -1, -1]
    y_bad = make_case(10, [2, 2], vocab)
    y_bad[6][0, 3] = math.nan
    y_bad[6][2, :] = -math.inf
    assert run(*y_bad) == plain(*y_bad) == ([0, 0], [-1, -1])


def test_equal_distributions_leave_the_target_itself():
    """p = q: a draft is kept by every draw below one; a draw of one (which no generator gives) finds nothing left."""
    g = torch.Generator().manual_seed(2)
    z = torch.randn((2, 300), generator=g)
    y = z[:1].clone()
    assert run(z, [1], [7], [1.0], [1 - 1e-9], [0.4], y)[0] == [1]
    assert run(z, [1], [7], [1.0], [1.0], [0.4], y) == plain(z, [1], [7], [1.0], [1.0], [0.4], y)


def test_offsets_that_no_rows_have():
    z = torch.randn((6, 50), generator=torch.Generator().manual_seed(1))
    a, p = run(z, [1, 1, 1], [0, 0, 0], [1.0] * 3, [0.5] * 3, [0.5] * 3, first=[0, 5, 4, 9])
    assert a == [0, 0, 0] and p == [-1, -1, -1]  # (more drafts than there are, rows that run back, rows beyond the last)
    a, p = run(z, [1, 1, 1], [0, 0, 0], [1.0] * 3, [0.5] * 3, [0.5] * 3, first=[-2, 2, 2, 6])
    assert a[:2] == [0, 0] and p[:2] == [-1, -1]


@pytest.mark.parametrize("model", [True, False])
def test_pick_draws_of_another_range(model):
    """Below 0 and NaN: the first id with any mass; from 1 on: the last.  Nothing is left unwritten."""
    counts = [0, 1, 0, 1, 0, 1]
    logits, _, drafts, temps, accept, _, draft_logits = make_case(5, counts, 4099, model=model)
    logits[:, :3], logits[:, -2:] = -math.inf, -math.inf
    accept = [1.0 - 2.0 ** -53] * 3
    if draft_logits is not None:
        draft_logits = draft_logits.flip(0).contiguous()
    case = lambda picks: (logits, counts, drafts, temps, accept, picks, draft_logits)
    low, high = plain(*case([0.0] * 6)), plain(*case([1.0] * 6))
    assert run(*case([-0.25, -0.25, math.nan, math.nan, -math.inf, -1e-300])) == low
    assert run(*case([1.0, 1.0, 1.5, 1.5, math.inf, math.inf])) == high


def test_verify_in_a_graph_and_on_another_stream():
    from nnis_b200.engine.workspace import Workspace
    from nnis_b200.sampling import device
    case = make_case(21, [4, 2, 5], 2000)
    logits, counts, drafts, temps, accept, picks, y = case
    t = {"z": logits.to(DEV), "y": y.to(DEV), "d": torch.tensor(drafts, dtype=torch.int32, device=DEV),
         "f": torch.tensor([0, 5, 8, 14], dtype=torch.int32, device=DEV), "t": torch.tensor(temps, device=DEV),
         "a": torch.tensor(accept, dtype=torch.float64, device=DEV), "p": torch.tensor(picks, dtype=torch.float64, device=DEV)}
    out = torch.zeros((2, 3), dtype=torch.int32, device=DEV)
    ws = Workspace(torch.device(DEV))
    call = lambda: device.verify_drafts(t["z"], t["d"], t["f"], t["t"], t["a"], t["p"], out[0], out[1], t["y"], ws)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    assert (out[0].tolist(), out[1].tolist()) == plain(*case)
    ws.frozen = True
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    other = make_case(22, [4, 2, 5], 2000)
    t["z"].copy_(other[0]), t["y"].copy_(other[6]), t["d"].copy_(torch.tensor(other[2])), t["a"].copy_(torch.tensor(other[4]))
    t["p"].copy_(torch.tensor(other[5]))
    graph.replay()
    assert (out[0].tolist(), out[1].tolist()) == plain(*other)


def test_verify_refuses():
    from nnis_b200.csrc.ops import KernelError
    case = make_case(1, [1, 1], 40)
    for change in ({2: [0]}, {4: [0.5]}, {5: [0.1]}, {3: [1.0]}, {6: case[6][:1]}, {6: case[6][:, :9]}, {0: case[0].double()}, {0: case[0].t()}):
        bad = list(case)
        for i, x in change.items():
            bad[i] = x
        with pytest.raises(KernelError):
            run(*bad)
