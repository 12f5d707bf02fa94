"""Attention over the 8-bit cache where scales of values lie far apart or near the ends of their range, and other calls of the 8-bit operators
that are allowed and rare."""
import pytest
import torch

import int8_plain as plain
from int8_plain import PAGE
from test_int8_cache_gpu import TYPES, cuda, place

pytestmark = pytest.mark.gpu


def attend(q, k, v, ks, vs, positions, seqs, table, heads, kv_heads, window, scale):
    from nnis_b200.csrc import ops
    from nnis_b200.engine.workspace import Workspace
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda")
    i32 = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (positions, seqs, table)]
    ops.attention_int8(q.cuda(), q.shape[1], *cuda(k, v, ks, vs), *i32, out, heads, kv_heads, q.shape[1] // heads, window, scale,
                       Workspace(torch.device("cuda")))
    return out.cpu().double()


# (one sequence with slices or a cluster; many short ones, a warp each; several rows of a sequence)
SHAPES = [([700], 1), ([300 - i for i in range(150)], 1), ([400, 130], 5)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,d", [(9, 3, 64), (8, 2, 128), (2, 1, 40)])
@pytest.mark.parametrize("lengths,tokens", SHAPES)
@pytest.mark.parametrize("low", [86, 96, 101])
def test_values_of_the_smallest_scales(dtype, heads, kv_heads, d, lengths, tokens, low):
    """Rows whose largest value is at least 2^-100 have scales from 2^-107 on; the outputs are those of the same values 2^low times as
    large, to within the same bound 2^-low times as large (all are powers of two away from the ends of the types' ranges)."""
    gen = torch.Generator().manual_seed(low)
    table, pages = place(lengths, gen)
    k, ks = plain.store(pages, kv_heads, d, gen)
    v, vs = plain.store(pages, kv_heads, d, gen)
    vs = vs.clamp_min(2.0 ** -6)
    positions, seqs = [n - tokens + j for n in lengths for j in range(tokens)], [i for i in range(len(lengths)) for _ in range(tokens)]
    q = (1.5 * torch.randn((len(positions), heads * d), generator=gen)).to(dtype)
    shown = [i for i in range(len(positions)) if i < 6 or i > len(positions) - 4]
    want, bound = plain.attention(q[shown], k, v, ks, vs, [positions[i] for i in shown], [seqs[i] for i in shown], table, heads, kv_heads, 0,
                                  d ** -0.5, dtype == torch.float32)
    got = attend(q, k, v, ks, vs * 2.0 ** -low, positions, seqs, table, heads, kv_heads, 0, d ** -0.5)[shown] * 2.0 ** low
    assert ((got - want).abs() <= bound).all(), float(((got - want).abs() / bound).max())
