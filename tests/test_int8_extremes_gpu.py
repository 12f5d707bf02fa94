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


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,d", [(9, 3, 64), (8, 2, 128), (12, 4, 96), (4, 2, 32), (2, 1, 40)])
@pytest.mark.parametrize("lengths,tokens", SHAPES)
@pytest.mark.parametrize("at", ["first", "middle", "last"])
@pytest.mark.parametrize("large", [20, 40, 100])
def test_a_large_value_that_has_no_weight(dtype, heads, kv_heads, d, lengths, tokens, at, large):
    """One position of a page has values 2^large times the others' and a key that no query turns to: its scores lie at least 2 (large + 40)
    below the others' (in natural units), so its share is below 2^-(large + 60) of any other's and the outputs are those without it."""
    gen = torch.Generator().manual_seed(large + d)
    table, pages = place(lengths, gen)
    k, ks = plain.store(pages, kv_heads, d, gen)
    v, vs = plain.store(pages, kv_heads, d, gen)
    q = (1.5 * torch.randn((len(lengths) * tokens, heads * d), generator=gen)).to(dtype).view(-1, heads, d)
    scale = d ** -0.5
    # value 0 of every query is 4 and every key's is 0, but that of the large positions, which have nothing else
    q[..., 0] = 4.0
    k[..., 0] = 0
    for line, n in zip(table, lengths):
        for j in {"first": [0], "middle": [(n - tokens) // 2], "last": [n - tokens]}[at]:
            page, slot = line[j // PAGE], j % PAGE
            k[page, :, slot] = 0
            k[page, :, slot, 0] = -127
            ks[page, :, slot] = 2.0 * (large + 60) / (4 * 127 * scale)
            vs[page, :, slot] *= 2.0 ** large
    q = q.reshape(len(lengths) * tokens, heads * d)
    positions, seqs = [n - tokens + j for n in lengths for j in range(tokens)], [i for i in range(len(lengths)) for _ in range(tokens)]
    shown = [i for i in range(len(positions)) if i < 6 or i > len(positions) - 4]
    # (the bound is that of the others: one with this position's key of zeros and its value as large as theirs, whose share of some
    # hundredths moves theirs by as much)
    plain_ks, plain_vs = ks.clone(), vs.clone()
    for line, n in zip(table, lengths):
        j = {"first": 0, "middle": (n - tokens) // 2, "last": n - tokens}[at]
        plain_ks[line[j // PAGE], :, j % PAGE] = 0.0
        plain_vs[line[j // PAGE], :, j % PAGE] *= 2.0 ** -large
    rows = [positions[i] for i in shown], [seqs[i] for i in shown], table, heads, kv_heads, 0, scale, dtype == torch.float32
    want, _ = plain.attention(q[shown], k, v, ks, plain_vs, *rows)
    _, bound = plain.attention(q[shown], k, v, plain_ks, plain_vs, *rows)
    got = attend(q, k, v, ks, vs, positions, seqs, table, heads, kv_heads, 0, scale)[shown]
    assert ((got - want).abs() <= 1.05 * bound).all(), float(((got - want).abs() / bound).max())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,d", [(9, 3, 64), (20, 1, 64), (8, 2, 128), (12, 4, 96), (4, 2, 32), (2, 1, 40)])
@pytest.mark.parametrize("window,at", [(100, 296), (0, 399)])
@pytest.mark.parametrize("sequences", [1, 120])
def test_a_large_value_that_others_see(dtype, heads, kv_heads, d, window, at, sequences):
    """Five rows of a sequence, of which the first (the last) alone sees a position whose values are 2^60 times the others'."""
    gen = torch.Generator().manual_seed(at + d)
    table, pages = place([400] * sequences, gen)
    k, ks = plain.store(pages, kv_heads, d, gen)
    v, vs = plain.store(pages, kv_heads, d, gen)
    for line in table:
        vs[line[at // PAGE], :, at % PAGE] *= 2.0 ** 60
    q = (1.5 * torch.randn((5 * sequences, heads * d), generator=gen)).to(dtype)
    positions, seqs = [395, 396, 397, 398, 399] * sequences, [i for i in range(sequences) for _ in range(5)]
    shown = list(range(5)) if sequences == 1 else [*range(5), *range(5 * sequences - 10, 5 * sequences)]
    want, bound = plain.attention(q[shown], k, v, ks, vs, [positions[i] for i in shown], [seqs[i] for i in shown], table, heads, kv_heads, window,
                                  d ** -0.5, dtype == torch.float32)
    got = attend(q, k, v, ks, vs, positions, seqs, table, heads, kv_heads, window, d ** -0.5)[shown]
    assert ((got - want).abs() <= bound).all(), float(((got - want).abs() / bound).max())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,d,sequences,window,tokens", [(32, 8, 128, 8, 2100, 1), (9, 3, 64, 32, 2100, 1), (32, 8, 128, 8, 1300, 2),
                                                                     (9, 3, 64, 32, 2200, 2), (8, 8, 32, 16, 3000, 2), (12, 4, 96, 24, 1999, 2)])
def test_windows_that_several_slices_share(dtype, heads, kv_heads, d, sequences, window, tokens):
    """Windows cut into slices, at positions all over a piece; of several rows of a sequence some lie further apart than a window is long,
    so that what they see together is more than the slices' parts."""
    from nnis_b200.csrc import ops
    gen = torch.Generator().manual_seed(window)
    lengths = [4600 - 37 * i for i in range(sequences)]
    table, pages = place(lengths, gen)
    positions = [n - 1 - j * (1 if i % 2 else 1450) for i, n in enumerate(lengths) for j in range(tokens)]
    seqs = [i for i in range(sequences) for _ in range(tokens)]
    slices, pieces, rows, cluster, _ = ops.attention_int8_plan(len(positions), sequences, heads, kv_heads, d, len(table[0]), window,
                                                               ops.sm_count(torch.device("cuda:0")))
    assert rows == tokens and slices > 1 and ops.attention_int8_slice(slices, pieces, rows, d, window) < pieces
    k, ks = plain.store(pages, kv_heads, d, gen)
    v, vs = plain.store(pages, kv_heads, d, gen)
    q = (1.5 * torch.randn((len(positions), heads * d), generator=gen)).to(dtype)
    shown = list(range(6))
    want, bound = plain.attention(q[shown], k, v, ks, vs, positions[:6], seqs[:6], table, heads, kv_heads, window, d ** -0.5, dtype == torch.float32)
    got = attend(q, k, v, ks, vs, positions, seqs, table, heads, kv_heads, window, d ** -0.5)[shown]
    assert ((got - want).abs() <= bound).all(), float(((got - want).abs() / bound).max())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 40])
def test_angles_of_no_position(dtype, d):
    """Tables of angles without a row: every position lies beyond them, so nothing is written."""
    from nnis_b200.csrc import ops
    gen = torch.Generator().manual_seed(3)
    k, ks = plain.store(2, 1, d, gen)
    v, vs = plain.store(2, 1, d, gen)
    stores = cuda(k, v, ks, vs)
    q = torch.full((3, 2 * d), 7.0, dtype=dtype, device="cuda")
    i32 = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 5, 70], [0, 0, 0], [[1, 0]])]
    none = torch.empty((0, d // 2), device="cuda")
    ops.rope_store_int8(torch.randn((3, 4 * d), generator=gen).to(dtype).cuda(), q, *i32, none, none, *stores, 2, 1, d, PAGE)
    assert (q == 7).all() and all(torch.equal(a.cpu(), b) for a, b in zip(stores, (k, v, ks, vs)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k", [(5, 64), (130, 96), (3, 37), (40, 2048), (2, 9000)])
def test_rows_that_share_memory(dtype, rows, k):
    """Rows of any stride: one row many times over, and rows that overlap."""
    from nnis_b200.csrc import ops
    from nnis_b200.engine.workspace import Workspace
    gen = torch.Generator().manual_seed(k)
    flat = torch.randn(k + 8 * rows, generator=gen).to(dtype).cuda()
    w, w_scales = plain.codes_of(torch.randn((24, k), generator=gen))
    w = torch.nn.functional.pad(w, (0, ops.int8_width(k) - k)).cuda()
    w_scales = w_scales.cuda()
    for x in (flat[:k].expand(rows, k), flat.as_strided((rows, k), (8, 1)), flat.as_strided((rows, k), (1, 1))):
        got, want = ([torch.full((rows, ops.int8_width(k)), 9, dtype=torch.int8, device="cuda"), torch.full((rows,), 9.0, device="cuda")]
                     for _ in range(2))
        ops.quantize_rows(x, *got)
        ops.quantize_rows(x.contiguous(), *want)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        outs = [torch.empty((rows, 24), dtype=dtype, device="cuda") for _ in range(2)]
        for out, values in zip(outs, (x, x.contiguous())):
            ops.linear_int8(values, w, w_scales, None, out, ops.STORE, Workspace(torch.device("cuda")))
        assert torch.equal(*outs)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_far_apart(dtype):
    """Rows whose distance, in elements, passes 31 bits."""
    from nnis_b200.csrc import ops
    gen = torch.Generator().manual_seed(4)
    apart, k = (1 << 31) + 8, 96
    flat = torch.empty(2 * apart + k, dtype=dtype, device="cuda")
    x = flat.as_strided((3, k), (apart, 1))
    x.copy_(torch.randn((3, k), generator=gen).to(dtype))
    got, want = ([torch.full((3, k), 9, dtype=torch.int8, device="cuda"), torch.full((3,), 9.0, device="cuda")] for _ in range(2))
    ops.quantize_rows(x, *got)
    ops.quantize_rows(x.contiguous(), *want)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,d", [(32, 8, 128), (6, 3, 40)])
def test_a_store_of_more_than_2_31_codes(dtype, heads, kv_heads, d):
    """Pages at the far end of a store, and of what they are read back to, hold and give what they do in a small one."""
    from nnis_b200.csrc import ops
    gen = torch.Generator().manual_seed(d)
    pages = (1 << 31) // (kv_heads * PAGE * d) + 9
    lengths, n = [500, 130], 70
    table, small = place(lengths, gen)
    qkv = torch.randn((n, (heads + 2 * kv_heads) * d), generator=gen).to(dtype).cuda()
    at = [(i, p) for i, length in enumerate(lengths) for p in range(length - n // 2, length)]
    token_seq, token_pos = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in zip(*at))
    k, ks = plain.store(small, kv_heads, d, gen)
    v, vs = plain.store(small, kv_heads, d, gen)
    cos, sin = cuda(*plain.angles(500, d))
    results = []
    for count, first in ((small, 0), (pages, pages - small)):
        stores = [torch.empty((count, *t.shape[1:]), dtype=t.dtype, device="cuda") for t in (k, v, ks, vs)]
        for store, t in zip(stores, (k, v, ks, vs)):
            store[first:] = t.cuda()
        ids = torch.tensor(table, dtype=torch.int32)
        ids = torch.where(ids < 0, ids, ids + first).cuda()
        q = torch.empty((n, heads * d), dtype=dtype, device="cuda")
        ops.rope_store_int8(qkv, q, token_pos, token_seq, ids, cos, sin, *stores, heads, kv_heads, d, PAGE)
        outs = [torch.zeros((count, kv_heads, PAGE, d), dtype=dtype, device="cuda") for _ in range(2)]
        ops.read_pages_int8(*stores, ids, ids, *outs)
        from nnis_b200.engine.workspace import Workspace
        attn = torch.empty_like(q)
        ops.attention_int8(q, heads * d, *stores, token_pos, token_seq, ids, attn, heads, kv_heads, d, 0, d ** -0.5, Workspace(torch.device("cuda")))
        results.append([q, attn, *(t[first:].clone() for t in (*stores, *outs))])
        del stores, outs
    for a, b in zip(*results):
        assert torch.equal(a, b)
    assert results[0][1].abs().amax() > 0
