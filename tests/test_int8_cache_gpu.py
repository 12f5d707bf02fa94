"""The cache held in 8 bits: written, read back and attended over."""
import pytest
import torch

import int8_plain as plain
from int8_plain import PAGE

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float32]


def cuda(*tensors):
    return [t.cuda() for t in tensors]


def place(lengths, gen, spare=2):
    """Page tables of sequences of these lengths, pages in random places."""
    counts = [-(-n // PAGE) for n in lengths]
    ids = torch.randperm(sum(counts) + spare, generator=gen).tolist()
    cols = max(1, max(counts))
    return [[ids.pop() for _ in range(c)] + [-1] * (cols - c) for c in counts], sum(counts) + spare


# ---- writing and reading back --------------------------------------------------------------------
def write(ops, qkv, positions, seqs, table, k, v, ks, vs, heads, kv_heads, d, cos=None, sin=None):
    q = torch.full((qkv.shape[0], heads * d), 7.0, dtype=qkv.dtype, device="cuda")
    ops.rope_store_int8(qkv, q, torch.tensor(positions, dtype=torch.int32, device="cuda"),
                        torch.tensor(seqs, dtype=torch.int32, device="cuda"), torch.tensor(table, dtype=torch.int32, device="cuda"),
                        cos, sin, k, v, ks, vs, heads, kv_heads, d, PAGE)
    return q


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,d", [(9, 3, 64), (4, 4, 128), (3, 1, 96), (2, 2, 8), (5, 1, 2), (2, 1, 250), (4, 2, 256), (3, 3, 24),
                                              (1, 1, 16), (2, 1, 6)])
@pytest.mark.parametrize("rotates", [True, False])
def test_rows_are_written_as_codes(dtype, heads, kv_heads, d, rotates):
    """Queries, codes and scales to the last bit; what no row writes stays as it was."""
    from nnis_b200.csrc import ops
    gen = torch.Generator().manual_seed(d * heads)
    spans = [(0, 70), (63, 1), (64, 1), (190, 130)]  # (positions held, new ones)
    table, pages = place([s + c for s, c in spans], gen)
    positions = [p for s, c in spans for p in range(s, s + c)] + [-1]
    seqs = [i for i, (_, c) in enumerate(spans) for _ in range(c)] + [0]
    n = len(positions)
    qkv = torch.randn((n, (heads + 2 * kv_heads) * d), generator=gen).to(dtype)
    cos, sin = plain.angles(max(positions) + 1, d) if rotates else (None, None)
    k, ks = plain.store(pages, kv_heads, d, gen)
    v, vs = plain.store(pages, kv_heads, d, gen)
    got = cuda(k, v, ks, vs)
    q = write(ops, qkv.cuda(), positions, seqs, table, *got, heads, kv_heads, d, *(cuda(cos, sin) if rotates else (None, None)))
    rows = qkv.view(n, -1, d)
    turned = rows[:, :heads + kv_heads]
    if rotates:
        at = torch.tensor(positions).clamp_min(0)
        turned = plain.rotate(turned, cos[at][:, None], sin[at][:, None])
    new = [*plain.codes_of(turned[:, heads:]), *plain.codes_of(rows[:, heads + kv_heads:])]
    for r in range(n - 1):
        page, slot = table[seqs[r]][positions[r] // PAGE], positions[r] % PAGE
        for t, x in zip((k, ks, v, vs), new):
            t[page, :, slot] = x[r]
    want_q = turned[:, :heads].reshape(n, -1).clone()
    want_q[-1] = 7.0  # the padding row
    assert torch.equal(q.cpu(), want_q)
    for g, w in zip(got, (k, v, ks, vs)):
        assert torch.equal(g.cpu(), w)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_zeros_of_tiny_values_and_of_no_numbers(dtype):
    """Zeros and values below 2^-100 give zeros; an infinity or a NaN gives a scale that is no number."""
    from nnis_b200.csrc import ops
    d, kv_heads = 64, 2
    qkv = torch.randn((6, 3 * 2 * d), generator=torch.Generator().manual_seed(1)).to(dtype)
    rows = qkv.view(6, 6, d)  # heads: q q k k v v
    rows[0, 2] = 0
    rows[1, 4] *= 2.0 ** -110
    rows[2, 3, 5] = float("inf")
    rows[3, 5, 63] = float("nan")
    rows[4, 2] *= 2.0 ** 120
    rows[5, 2] *= 2.0 ** -90
    k, v = (torch.full((1, kv_heads, PAGE, d), 3, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.full((1, kv_heads, PAGE), 5.0, device="cuda") for _ in range(2))
    write(ops, qkv.cuda(), list(range(6)), [0] * 6, [[0]], k, v, ks, vs, 2, kv_heads, d)
    for store, scales, first in ((k, ks, 2), (v, vs, 4)):
        codes, want = plain.codes_of(rows[:, first:first + 2])
        assert torch.equal(store[0, :, :6].cpu(), codes.transpose(0, 1))
        assert torch.equal(torch.nan_to_num(scales[0, :, :6].cpu(), nan=-9.0), torch.nan_to_num(want.T, nan=-9.0))
    assert float(ks[0, 0, 0]) == 0.0 and float(vs[0, 0, 1]) == 0.0 and torch.isnan(ks[0, 1, 2]) and torch.isnan(vs[0, 1, 3])
    assert (k[0, :, 6:] == 3).all() and (vs[0, :, 6:] == 5).all()


def test_rows_whose_page_is_not_there_store_nothing():
    """Beyond the table, beyond the store, a page that was given back, a sequence that is not there, beyond the angles."""
    from nnis_b200.csrc import ops
    d, gen = 64, torch.Generator().manual_seed(2)
    qkv = torch.randn((6, 3 * d), generator=gen).cuda()
    cos, sin = cuda(*plain.angles(200, d))
    k, ks = cuda(*plain.store(2, 1, d, gen))
    v, vs = cuda(*plain.store(2, 1, d, gen))
    before = [t.clone() for t in (k, v, ks, vs)]
    q = write(ops, qkv, [128, 0, 64, 5, 5, 200], [0, 1, 0, 2, -1, 0], [[1, -1], [2, 0]], k, v, ks, vs, 1, 1, d, cos, sin)
    for t, b in zip((k, v, ks, vs), before):
        assert torch.equal(t, b)
    assert (q[5] == 7).all() and not (q[:5] == 7).all(1).any()  # (their queries are turned all the same)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kv_heads,d", [(3, 64), (2, 128), (1, 96), (2, 2), (1, 250), (3, 20)])
def test_pages_are_read_back(dtype, kv_heads, d):
    """Code times scale, rounded once; pages that nobody asks for, or that are not there, stay as they were."""
    from nnis_b200.csrc import ops
    gen = torch.Generator().manual_seed(d)
    pages, table = 7, torch.tensor([[4, 0, 2, -1], [6, 9, 1, 5]], dtype=torch.int32)
    local = torch.tensor([[0, 3, -1], [2, 1, 8]], dtype=torch.int32)
    k, ks = plain.store(pages, kv_heads, d, gen)
    v, vs = plain.store(pages, kv_heads, d, gen)
    outs = [torch.full((5, kv_heads, PAGE, d), 9.0, dtype=dtype) for _ in range(2)]
    got = cuda(*outs)
    ops.read_pages_int8(*cuda(k, v, ks, vs, table, local), *got)
    for out, codes, scales, g in ((outs[0], k, ks, got[0]), (outs[1], v, vs, got[1])):
        for to, page in ((0, 4), (3, 0), (2, 6)):
            out[to] = (codes[page].float() * scales[page][..., None]).to(dtype)
        assert torch.equal(g.cpu(), out)


# ---- attention ------------------------------------------------------------------------------------
def check(dtype, heads, kv_heads, d, positions, seqs, table, pages, window=0, seed=0, stride=None, change=None):
    from nnis_b200.csrc import ops
    from nnis_b200.engine.workspace import Workspace
    gen = torch.Generator().manual_seed(seed)
    k, ks = plain.store(pages, kv_heads, d, gen)
    v, vs = plain.store(pages, kv_heads, d, gen)
    q = (1.5 * torch.randn((len(positions), heads * d), generator=gen)).to(dtype)
    scale = d ** -0.5
    want, bound = plain.attention(q, k, v, ks, vs, positions, seqs, table, heads, kv_heads, window, scale, dtype == torch.float32)
    if change is not None:
        change(k, v, ks, vs)
    rows = torch.full((len(positions), stride or heads * d), float("nan"), dtype=dtype)
    rows[:, :heads * d] = q
    out = torch.full((len(positions), heads * d), 7.0, dtype=dtype, device="cuda")
    ops.attention_int8(rows.cuda(), rows.shape[1], *cuda(k, v, ks, vs, torch.tensor(positions, dtype=torch.int32),
                                                        torch.tensor(seqs, dtype=torch.int32), torch.tensor(table, dtype=torch.int32)),
                       out, heads, kv_heads, d, window, scale, Workspace(torch.device("cuda")))
    got = out.cpu().double()
    assert torch.isfinite(got).all()
    assert ((got - want).abs() <= bound).all(), float(((got - want).abs() / bound).max())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,d", [(9, 3, 64), (15, 5, 64), (4, 4, 64), (8, 1, 64), (20, 1, 64), (32, 8, 128), (3, 3, 128), (24, 1, 128),
                                              (12, 4, 96), (4, 2, 32), (6, 2, 256), (2, 1, 2), (4, 2, 80), (2, 2, 250), (3, 1, 18), (64, 1, 64)])
def test_single_rows(dtype, heads, kv_heads, d):
    """Positions around the ends of pages and of slices, with padding rows between them."""
    gen = torch.Generator().manual_seed(7)
    lengths = [1, 2, 63, 64, 65, 128, 129, 500]
    table, pages = place(lengths, gen)
    positions = [n - 1 for n in lengths] + [-1, 5]
    check(dtype, heads, kv_heads, d, positions, list(range(len(lengths))) + [0, 7], table, pages, seed=heads)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,d", [(9, 3, 64), (8, 2, 128), (6, 2, 96)])
@pytest.mark.parametrize("window", [1, 2, 64, 65, 100, 1000])
def test_windows(dtype, heads, kv_heads, d, window):
    gen = torch.Generator().manual_seed(8)
    lengths = [1, 64, 65, 130, 700]
    table, pages = place(lengths, gen)
    for i, n in enumerate(lengths):  # pages wholly before the window have been given back
        for j in range(max(0, n - window) // PAGE):
            table[i][j] = -1
    check(dtype, heads, kv_heads, d, [n - 1 for n in lengths], list(range(len(lengths))), table, pages, window=window, seed=window)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,d", [(9, 3, 64), (8, 2, 128)])
def test_several_rows_of_a_sequence(dtype, heads, kv_heads, d):
    """Drafted tokens, rows in any order, one twice; rows of the queries further apart than they are long."""
    gen = torch.Generator().manual_seed(9)
    table, pages = place([300, 66, 5], gen)
    positions, seqs = [299, 297, 298, 65, 64, 63, 4, 0, 0, 299], [0, 0, 0, 1, 1, 1, 2, 2, 2, 0]
    check(dtype, heads, kv_heads, d, positions, seqs, table, pages, seed=3, stride=(heads + 2 * kv_heads) * d)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,d", [(9, 3, 64), (8, 2, 128), (2, 1, 40)])
def test_a_long_context_is_cut_into_slices(dtype, heads, kv_heads, d):
    gen = torch.Generator().manual_seed(10)
    table, pages = place([5003, 4096, 1], gen)
    check(dtype, heads, kv_heads, d, [5002, 4095, 0], [0, 1, 2], table, pages, seed=4)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,d", [(9, 3, 64), (8, 2, 128), (2, 1, 40)])
def test_pages_that_are_not_there_hold_no_keys(dtype, heads, kv_heads, d):
    """Holes in a table, ids beyond the store, a row that sees nothing, a sequence that is not there."""
    gen = torch.Generator().manual_seed(11)
    table, pages = place([400, 200, 64], gen)
    table[0][1] = -1
    table[0][4] = pages
    table[1][3] = 1 << 30
    table[2][0] = -7
    check(dtype, heads, kv_heads, d, [399, 199, 63, 5, 9, 10 ** 6], [0, 1, 2, 3, -1, 0], table, pages, seed=5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,d", [(9, 3, 64), (8, 2, 128), (2, 1, 40)])
def test_what_lies_behind_a_sequence_is_never_read(dtype, heads, kv_heads, d):
    """Scales that are no numbers behind the positions, in front of the window and in pages of others change nothing."""
    gen = torch.Generator().manual_seed(12)
    table, pages = place([70, 130], gen)

    def spoil(k, v, ks, vs):
        seen = torch.zeros(pages, PAGE, dtype=torch.bool)
        for seq, pos in ((0, 69), (1, 129)):
            for t in range(pos - 59, pos + 1):
                seen[table[seq][t // PAGE], t % PAGE] = True
        for t, s in ((k, ks), (v, vs)):
            s.masked_fill_(~seen[:, None], float("nan"))
            t[(~seen)[:, None].expand(-1, kv_heads, -1)] = -128
    check(dtype, heads, kv_heads, d, [69, 129], [0, 1], table, pages, window=60, seed=6, change=spoil)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128, 40])
def test_a_row_that_is_no_number_is_seen(dtype, d):
    """A key or value whose scale is NaN makes NaN of the rows that see it, of no others."""
    from nnis_b200.csrc import ops
    from nnis_b200.engine.workspace import Workspace
    gen = torch.Generator().manual_seed(13)
    for spoiled in range(2):
        stores = [t for _ in range(2) for t in plain.store(3, 2, d, gen)]
        stores[1 + 2 * spoiled][1, 1, 10] = float("nan")  # head 1 of position 74
        k, ks, v, vs = cuda(*stores)
        q = torch.randn((3, 4 * d), generator=gen).to(dtype).cuda()
        out = torch.empty_like(q)
        ops.attention_int8(q, 4 * d, k, v, ks, vs, torch.tensor([73, 74, 180], dtype=torch.int32, device="cuda"),
                           torch.zeros(3, dtype=torch.int32, device="cuda"), torch.tensor([[0, 1, 2]], dtype=torch.int32, device="cuda"),
                           out, 4, 2, d, 0, d ** -0.5, Workspace(torch.device("cuda")))
        bad = torch.isnan(out.view(3, 4, d)).all(2)
        assert bad.tolist() == [[False] * 4, [False, False, True, True], [False, False, True, True]]
        assert torch.isfinite(out.view(3, 4, d)[~bad]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128])
def test_large_and_small_queries_and_scales(dtype, d):
    """Scores of some hundred: one key has all the weight; a query of zeros: all keys alike."""
    from nnis_b200.csrc import ops
    from nnis_b200.engine.workspace import Workspace
    gen = torch.Generator().manual_seed(14)
    k, ks = plain.store(4, 1, d, gen)
    v, vs = plain.store(4, 1, d, gen)
    q = torch.randn((4, 2 * d), generator=gen).to(dtype)
    q[0] *= 200.0
    q[1] = 0.0
    q[2] *= 2.0 ** -60
    q[3, :d] *= 2.0 ** 30
    ks[3] *= 2.0 ** -30
    positions, seqs, table = [255, 255, 255, 60], [0, 0, 0, 1], [[0, 1, 2, 3], [3, 0, 0, 0]]
    scale = d ** -0.5
    want, bound = plain.attention(q, k, v, ks, vs, positions, seqs, table, 2, 1, 0, scale, dtype == torch.float32)
    out = torch.empty_like(q, device="cuda")
    ops.attention_int8(q.cuda(), 2 * d, *cuda(k, v, ks, vs, torch.tensor(positions, dtype=torch.int32),
                                              torch.tensor(seqs, dtype=torch.int32), torch.tensor(table, dtype=torch.int32)),
                       out, 2, 1, d, 0, scale, Workspace(torch.device("cuda")))
    assert ((out.cpu().double() - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_a_step_is_written_read_back_and_attended_over(dtype):
    """A prompt in chunks, then tokens one by one, as a program runs them: pages read back hold what attention sees, on a stream of the
    caller's and captured into a graph that is replayed."""
    from nnis_b200.csrc import ops
    from nnis_b200.engine.workspace import Workspace
    gen = torch.Generator().manual_seed(15)
    heads, kv_heads, d, total = 6, 2, 64, 140
    qkv = torch.randn((total, (heads + 2 * kv_heads) * d), generator=gen).to(dtype).cuda()
    cos, sin = cuda(*plain.angles(total, d))
    table = torch.tensor([[2, 0, 3]], dtype=torch.int32, device="cuda")
    stores = []
    for steps in ([total], [1, 62, 3, 64, 9, 1]):  # (the same store whichever way the tokens come)
        k, v = (torch.zeros((4, kv_heads, PAGE, d), dtype=torch.int8, device="cuda") for _ in range(2))
        ks, vs = (torch.zeros((4, kv_heads, PAGE), device="cuda") for _ in range(2))
        at = 0
        for n in steps:
            q = torch.empty((n, heads * d), dtype=dtype, device="cuda")
            ops.rope_store_int8(qkv[at:at + n], q, torch.arange(at, at + n, dtype=torch.int32, device="cuda"),
                                torch.zeros(n, dtype=torch.int32, device="cuda"), table, cos, sin, k, v, ks, vs, heads, kv_heads, d, PAGE)
            at += n
        stores.append((k, v, ks, vs, q[-1:].clone()))
    for a, b in zip(*stores):
        assert torch.equal(a, b)
    k, v, ks, vs, q = stores[0]
    local = torch.tensor([[0, 1, 2]], dtype=torch.int32, device="cuda")
    pos, seq = torch.tensor([total - 1], dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    k_read, v_read = (torch.zeros((3, kv_heads, PAGE, d), dtype=torch.float32, device="cuda") for _ in range(2))
    out, ws = torch.zeros((1, heads * d), dtype=dtype, device="cuda"), Workspace(torch.device("cuda"))

    def step():
        ops.read_pages_int8(k, v, ks, vs, table, local, k_read, v_read)
        ops.attention_int8(q, heads * d, k, v, ks, vs, pos, seq, table, out, heads, kv_heads, d, 0, d ** -0.5, ws)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    stream.synchronize()
    first = out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, first)
    keys, values = (t.permute(1, 0, 2, 3).reshape(kv_heads, -1, d)[:, :total].double().cpu() for t in (k_read, v_read))
    x = q.cpu().double().view(kv_heads, heads // kv_heads, d)
    want = torch.softmax(torch.einsum("hgd,hnd->hgn", x, keys) * d ** -0.5, -1) @ values
    _, bound = plain.attention(q.cpu(), *(t.cpu() for t in (k, v, ks, vs)), [total - 1], [0], table.tolist(), heads, kv_heads, 0, d ** -0.5,
                               dtype == torch.float32)
    # (the values read back are rounded to float32: half a step of each)
    assert ((out.cpu().double() - want.reshape(1, -1)).abs() <= 1.01 * bound + 1e-6).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,d", [(6, 3, 64), (6, 3, 128), (3, 3, 96), (8, 4, 32)])
def test_many_short_rows(dtype, heads, kv_heads, d):
    """Two hundred sequences of one to three hundred positions, a key/value head of each the work of one warp; padding rows and holes."""
    gen = torch.Generator().manual_seed(16)
    lengths = (1 + torch.randint(0, 300, (200,), generator=gen)).tolist()
    table, pages = place(lengths, gen)
    table[7][0] = -1
    table[9] = [-1] * len(table[9])
    positions = [-1 if i % 50 == 3 else n - 1 for i, n in enumerate(lengths)]
    check(dtype, heads, kv_heads, d, positions, list(range(200)), table, pages, seed=7)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,d,tokens,context,window", [(20, 1, 64, 3, 700, 0), (20, 1, 128, 3, 300, 0), (20, 1, 64, 5, 200, 90)])
def test_many_rows_of_many_queries(dtype, heads, kv_heads, d, tokens, context, window):
    """Sixty sequences' drafted tokens with twenty queries a key/value head: tiles of sixteen queries, the last of a run partly empty."""
    gen = torch.Generator().manual_seed(17)
    lengths = [context - 7 * (i % 9) for i in range(60)]
    table, pages = place(lengths, gen)
    positions = [n - tokens + j for n in lengths for j in range(tokens)]
    check(dtype, heads, kv_heads, d, positions, [i for i in range(60) for _ in range(tokens)], table, pages, window=window, seed=8)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 96, 40])
def test_queries_and_stores_at_any_address(dtype, d):
    """Rows of queries an odd number of values apart; codes that begin at no multiple of sixteen bytes."""
    from nnis_b200.csrc import ops
    from nnis_b200.engine.workspace import Workspace
    gen = torch.Generator().manual_seed(18)
    table, pages = place([130, 70], gen)
    check(dtype, 4, 2, d, [129, 69, 3], [0, 1, 1], table, pages, seed=9, stride=4 * d + 1)
    k, ks = plain.store(pages, 2, d, gen)
    v, vs = plain.store(pages, 2, d, gen)
    moved = []
    for t in (k, v):
        flat = torch.empty(t.numel() + 4, dtype=torch.int8, device="cuda")[4:].view(t.shape)
        flat.copy_(t)
        moved.append(flat)
    q = torch.randn((3, 4 * d), generator=gen).to(dtype)
    want, bound = plain.attention(q, k, v, ks, vs, [129, 69, 3], [0, 1, 1], table, 4, 2, 0, d ** -0.5, dtype == torch.float32)
    out = torch.empty_like(q, device="cuda")
    i32 = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([129, 69, 3], [0, 1, 1], table)]
    ops.attention_int8(q.cuda(), 4 * d, *moved, *cuda(ks, vs), *i32, out, 4, 2, d, 0, d ** -0.5, Workspace(torch.device("cuda")))
    assert ((out.cpu().double() - want).abs() <= bound).all()
    with pytest.raises(ops.KernelError, match="misaligned"):
        ops.rope_store_int8(torch.zeros((3, 8 * d), dtype=dtype, device="cuda"), q.cuda(), *i32, None, None, *moved, *cuda(ks, vs), 4, 2, d, PAGE)


@pytest.mark.parametrize("dtype", TYPES)
def test_other_page_sizes(dtype):
    """Pages of 16 positions take the kernel of any size."""
    from nnis_b200.csrc import ops
    from nnis_b200.engine.workspace import Workspace
    gen = torch.Generator().manual_seed(19)
    d, page = 64, 16
    x = torch.randn((5, 2, page, d), generator=gen)
    k, ks = plain.codes_of(x)
    v, vs = plain.codes_of(torch.randn((5, 2, page, d), generator=gen))
    q = torch.randn((2, 4 * d), generator=gen).to(dtype)
    table, positions = [[3, 1, 4], [0, 2, -1]], [40, 17]
    out = torch.empty_like(q, device="cuda")
    ops.attention_int8(q.cuda(), 4 * d, *cuda(k, v, ks, vs, torch.tensor(positions, dtype=torch.int32), torch.tensor([0, 1], dtype=torch.int32),
                                              torch.tensor(table, dtype=torch.int32)), out, 4, 2, d, 0, 0.125, Workspace(torch.device("cuda")))
    for r, (pages, pos) in enumerate(zip(table, positions)):
        keys, values = ((c[pages].double() * s[pages].double()[..., None]).transpose(0, 1).reshape(2, -1, d)[:, :pos + 1]
                        for c, s in ((k, ks), (v, vs)))
        h = q[r].double().view(2, 2, d)
        want = torch.softmax(torch.einsum("hgd,hnd->hgn", h, keys) * 0.125, -1) @ values
        # (scores of at most some ten, weights and sums of float32, the output rounded once)
        tolerance = 1e-5 * values.abs().amax() + torch.finfo(dtype).eps / 2 * want.abs()
        assert ((out[r].cpu().double().view(2, 2, d) - want).abs() <= tolerance).all()


def test_tickets_and_records_serve_calls_of_all_sizes():
    """One workspace, calls that cut their keys into slices and calls that do not, in turn: each call's answer is its own, and repeats to
    the last bit."""
    from nnis_b200.csrc import ops
    from nnis_b200.engine.workspace import Workspace
    ws, gen, kept = Workspace(torch.device("cuda")), torch.Generator().manual_seed(20), []
    for lengths, heads, kv_heads in (([5000], 9, 3), ([300] * 40, 6, 2), ([4000, 100], 4, 1), ([16000], 3, 1), ([64], 9, 3)):
        table, pages = place(lengths, gen)
        k, ks = plain.store(pages, kv_heads, 64, gen)
        v, vs = plain.store(pages, kv_heads, 64, gen)
        q = torch.randn((len(lengths), heads * 64), generator=gen).to(torch.bfloat16)
        args = cuda(k, v, ks, vs, torch.tensor([n - 1 for n in lengths], dtype=torch.int32), torch.arange(len(lengths), dtype=torch.int32),
                    torch.tensor(table, dtype=torch.int32))
        kept.append((q.cuda(), args, heads, kv_heads))

    def run(q, args, heads, kv_heads, space):
        out = torch.empty_like(q)
        ops.attention_int8(q, heads * 64, *args, out, heads, kv_heads, 64, 0, 0.125, space)
        return out

    alone = [run(*c, Workspace(torch.device("cuda"))) for c in kept]
    for _ in range(3):
        for c, want in zip(kept, alone):
            assert torch.equal(run(*c, ws), want)
    ops.check_status("cuda:0")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,d", [(3, 1, 64), (2, 2, 32), (6, 2, 128), (20, 1, 96)])
@pytest.mark.parametrize("tokens", [[64, 64], [33, 31, 32], [100, 1, 70], [40, 0, 3, 150]])
def test_runs_of_many_rows(dtype, heads, kv_heads, d, tokens):
    """More rows of a sequence than a warp has lanes, than are taken together; runs that cross the ends of sequences, padding rows among
    them, in a sequence of their own and in others'."""
    gen = torch.Generator().manual_seed(19)
    lengths = [t + 90 * (i % 2) + 1 for i, t in enumerate(tokens)]
    table, pages = place(lengths, gen)
    positions, seqs = [], []
    for i, (t, n) in enumerate(zip(tokens, lengths)):
        rows = [n - t + j for j in range(t)]
        if t > 30:
            rows[t // 2] = rows[5] = -1
        positions += rows + [-1, -1]
        seqs += [i] * t + [i, -1]
    check(dtype, heads, kv_heads, d, positions, seqs, table, pages, window=37 if heads == 6 else 0, seed=11)
