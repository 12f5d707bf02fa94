"""Attention of rows whose sequences share pages, against the definition in 64 bits, row by row."""
import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def ops():
    from nnis_b200.csrc import ops as o
    return o


def build(seed, prefixes, members, alone, tails, tokens=1):
    """Page lists of sequences: ``members`` behind each of ``prefixes`` (whole pages), ``alone`` that share nothing; every
    sequence goes on for one of ``tails`` tokens.  Returns (tables, seqs, positions)."""
    rng = random.Random(seed)
    tables, lengths, nxt = [], [], 0
    for p in prefixes:
        shared = list(range(nxt, nxt + p))
        nxt += p
        for _ in range(members):
            n = rng.choice(tails)
            own = -(-n // 64)
            tables.append(shared + list(range(nxt, nxt + own)))
            nxt += own
            lengths.append(p * 64 + n)
    for _ in range(alone):
        n = rng.choice(tails) + 40
        own = -(-n // 64)
        tables.append(list(range(nxt, nxt + own)))
        nxt += own
        lengths.append(n)
    order = list(range(nxt))
    rng.shuffle(order)
    tables = [[order[p] for p in t] for t in tables]
    seqs = [i for i, n in enumerate(lengths) for j in range(tokens)]
    positions = [max(0, n - tokens + j) for n in lengths for j in range(tokens)]
    return tables, seqs, positions, nxt


def check(tables, seqs, positions, pages, heads, kv_heads, dim, dtype, seed=0, spread=1.0, dirty=True, stride=0, call=None):
    """``dirty``: NaN and infinities where no row may look: behind the last position of every sequence."""
    from nnis_b200.engine.workspace import Workspace
    g = torch.Generator().manual_seed(seed)
    n = len(seqs)
    k = torch.randn((pages + 1, kv_heads, 64, dim), generator=g).to(dtype)
    v = torch.randn((pages + 1, kv_heads, 64, dim), generator=g).to(dtype)
    q_stride = heads * dim + stride
    q = (spread * torch.randn((n, q_stride), generator=g)).to(dtype)
    cols = max(len(t) for t in tables) + 1
    scale = 1.0 / math.sqrt(dim)
    ends = {}
    for s, p in zip(seqs, positions):
        ends[s] = max(ends.get(s, 0), p + 1)
    if dirty:
        shared = {}
        for t in tables:
            for p in t:
                shared[p] = shared.get(p, 0) + 1
        for s, end in ends.items():
            page = tables[s][(end - 1) // 64]
            if shared[page] == 1 and end % 64:
                k[page, :, end % 64:] = math.nan
                v[page, :, end % 64:] = math.inf
        k[pages], v[pages] = math.nan, math.nan
    kd, vd, qd = k.to(DEV), v.to(DEV), q.to(DEV)
    table = torch.tensor([t + [-1] * (cols - len(t)) for t in tables], dtype=torch.int32, device=DEV)
    pos = torch.tensor(positions, dtype=torch.int32, device=DEV)
    out = torch.full((n, heads * dim), 77.0, dtype=dtype, device=DEV)
    plan = ops().attention_shared_plan(tables, seqs, positions, heads, kv_heads, dim, dtype, DEV)
    ws = Workspace(torch.device(DEV))
    go = lambda: ops().attention_shared(qd, q_stride, kd, vd, pos, table, plan, out, heads, kv_heads, dim, scale, ws)
    (call or (lambda f: f()))(go)
    group = heads // kv_heads
    want = torch.zeros((n, heads, dim), dtype=torch.float64)
    size = torch.zeros((n, heads, 1), dtype=torch.float64)
    for r, (s, p) in enumerate(zip(seqs, positions)):
        if p < 0:
            continue
        ids = tables[s][:p // 64 + 1]
        keys = k[ids].permute(1, 0, 2, 3).reshape(kv_heads, -1, dim)[:, :p + 1].double()
        values = v[ids].permute(1, 0, 2, 3).reshape(kv_heads, -1, dim)[:, :p + 1].double()
        qr = q[r, :heads * dim].double().view(kv_heads, group, dim)
        w = torch.softmax(torch.einsum("hgd,htd->hgt", qr, keys) * scale, dim=2)
        want[r] = torch.einsum("hgt,htd->hgd", w, values).reshape(heads, dim)
        size[r] = torch.einsum("hgt,htd->hgd", w, values.abs()).amax(2).reshape(heads, 1)
    got = out.cpu().double().view(n, heads, dim)
    # float32: scores are sums of dim products of size |q||k| <= about 4 dim spread, rounded to 2^-24 each: the weights are off
    # by 2^-24 * dim * 4, ten times under 2e-5 of the values; and 2e-5 holds 2^-24 * 8,000 additions.
    # bfloat16: the output's rounding (2^-8 / 2 of itself) and the weights' (2^-9 each, of either sign: of the
    # mean of the absolute values at most that), 2^-8 of the weighted absolute values together; half as much again for the scores.
    tol = 2e-5 if dtype == torch.float32 else 1.5 * 2 ** -8
    err = ((got - want).abs() / (size + 1e-30)).amax().item() if n else 0.0
    live = torch.tensor([p >= 0 for p in positions])
    assert torch.isfinite(got).all()
    assert not got[~live].any()
    assert ((got - want).abs() <= tol * size + 1e-30).all(), (err, tol)


SHAPES = [(9, 3, 64), (32, 32, 64), (16, 2, 128), (20, 1, 64), (6, 3, 48), (2, 1, 2), (4, 4, 256), (3, 1, 30)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES)
@pytest.mark.parametrize("layout", ["two", "batch", "groups", "alone", "drafts", "exact pages"])
def test_rows_that_share_pages(dtype, heads, kv_heads, dim, layout):
    """Sizes from one key on, head layouts on and off the tiles, pages that end inside and on a tile."""
    tables, seqs, positions, pages = {
        "two": lambda: build(1, [1], 2, 0, [1, 2]),
        "batch": lambda: build(2, [5], 9, 0, [1, 7, 64, 65, 130]),
        "groups": lambda: build(3, [2, 7, 1], 5, 2, [3, 63, 64, 100]),
        "alone": lambda: build(4, [], 0, 3, [1, 90, 300]),
        "drafts": lambda: build(5, [3], 6, 1, [5, 66, 70], tokens=5),
        "exact pages": lambda: build(6, [4], 4, 0, [64, 128])}[layout]()
    check(tables, seqs, positions, pages, heads, kv_heads, dim, dtype, seed=heads + dim)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_trees_of_prefixes_and_padding_rows(dtype):
    """A prompt shared by all, longer ones by some of them, sequences that are whole prefixes of others, rows at several
    positions of one sequence, padding rows between them."""
    for seed in range(12):
        rng = random.Random(seed)
        tables, nxt = [], 0
        for _ in range(rng.randrange(2, 10)):
            begin = rng.choice(tables) if tables and rng.random() < 0.8 else []
            t = list(begin[:rng.randrange(0, len(begin) + 1)])
            for _ in range(rng.randrange(0 if t else 1, 5)):
                t.append(nxt)
                nxt += 1
            tables.append(t)
        seqs, positions = [], []
        for i, t in enumerate(tables):
            top = rng.randrange(0, 64 * len(t))
            for j in range(rng.choice((1, 1, 3))):
                seqs.append(i)
                positions.append(max(0, top - j) if rng.random() < 0.85 else -1)
        if all(p < 0 for p in positions):
            positions[0] = 0
        check(tables, seqs, positions, nxt, 6, 2, 64, dtype, seed=seed, dirty=False)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim", [64, 128])
def test_long_shared_prompts(dtype, dim):
    """Many pages (several chunks, records merged) and many rows (several tiles), scores far apart."""
    tables, seqs, positions, pages = build(7, [130], 37, 1, [1, 64, 200])
    check(tables, seqs, positions, pages, 6, 2, dim, dtype, seed=1, spread=4.0)
    tables, seqs, positions, pages = build(8, [70, 3], 70, 0, [9])
    check(tables, seqs, positions, pages, 4, 4, dim, dtype, seed=2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_queries_in_rows_of_a_larger_stride(dtype):
    tables, seqs, positions, pages = build(9, [3], 4, 1, [70])
    check(tables, seqs, positions, pages, 8, 2, 64, dtype, stride=256)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_only_padding_rows(dtype):
    check([[0], [0, 1]], [0, 1], [-1, -1], 2, 4, 2, 64, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv_heads,dim", [(9, 3, 64), (32, 32, 64), (16, 2, 128), (6, 3, 48)])
@pytest.mark.parametrize("members", [2, 9, 70])
def test_a_query_that_is_no_number_gives_none(dtype, heads, kv_heads, dim, members):
    """All scores of one (row, head) are NaN: its output is, and no other's."""
    from nnis_b200.engine.workspace import Workspace
    tables, seqs, positions, pages = build(11, [5], members, 1, [1, 64, 100])
    g = torch.Generator().manual_seed(3)
    k = torch.randn((pages, kv_heads, 64, dim), generator=g).to(dtype).to(DEV)
    v = torch.randn((pages, kv_heads, 64, dim), generator=g).to(dtype).to(DEV)
    q = torch.randn((len(seqs), heads * dim), generator=g).to(dtype).to(DEV)
    cols = max(map(len, tables))
    table = torch.tensor([t + [-1] * (cols - len(t)) for t in tables], dtype=torch.int32, device=DEV)
    pos = torch.tensor(positions, dtype=torch.int32, device=DEV)
    plan = ops().attention_shared_plan(tables, seqs, positions, heads, kv_heads, dim, dtype, DEV)
    outs = []
    for spoilt in (False, True):
        if spoilt:
            q[1, 2 * dim + 1] = math.nan
        out = torch.empty_like(q)
        ops().attention_shared(q, heads * dim, k, v, pos, table, plan, out, heads, kv_heads, dim, 0.1, Workspace(torch.device(DEV)))
        outs.append(out.view(-1, heads, dim).double())
    clean, got = outs
    assert torch.isnan(got[1, 2]).all()
    got[1, 2] = clean[1, 2]
    # (either is off by at most 1.5 * 2^-8 of the largest value, see ``check``)
    assert ((got - clean).abs() <= 3 * 2 ** -8 * v.abs().max().item()).all()


def test_pages_beyond_32_bit_offsets():
    """A store of more than 2^32 bytes and 2^31 values: pages at its end."""
    from nnis_b200.engine.workspace import Workspace
    heads, kv, d, pages = 8, 8, 128, 34000
    k = torch.zeros((pages, kv, 64, d), dtype=torch.bfloat16, device=DEV)
    v = torch.zeros_like(k)
    top = pages - 3
    k[top:] = torch.randn((3, kv, 64, d), device=DEV).to(torch.bfloat16)
    v[top:] = torch.randn((3, kv, 64, d), device=DEV).to(torch.bfloat16)
    tables, seqs, positions = [[top, top + 1], [top, top + 2]], [0, 1], [100, 127]
    q = torch.randn((2, heads * d), device=DEV).to(torch.bfloat16)
    out = torch.empty_like(q)
    plan = ops().attention_shared_plan(tables, seqs, positions, heads, kv, d, torch.bfloat16, DEV)
    ops().attention_shared(q, heads * d, k, v, torch.tensor(positions, dtype=torch.int32, device=DEV),
                           torch.tensor(tables, dtype=torch.int32, device=DEV), plan, out, heads, kv, d, 0.1, Workspace(torch.device(DEV)))
    for r in range(2):
        keys = k[tables[r]].permute(1, 0, 2, 3).reshape(kv, -1, d)[:, :positions[r] + 1].double()
        values = v[tables[r]].permute(1, 0, 2, 3).reshape(kv, -1, d)[:, :positions[r] + 1].double()
        w = torch.softmax(torch.einsum("hd,htd->ht", q[r].double().view(kv, d), keys) * 0.1, 1)
        want = torch.einsum("ht,htd->hd", w, values)
        size = torch.einsum("ht,htd->hd", w, values.abs())
        assert ((out[r].double().view(kv, d) - want).abs() <= 1.5 * 2 ** -8 * size.amax()).all()
    del k, v
    torch.cuda.empty_cache()


def test_shared_attention_in_a_graph_and_on_another_stream():
    tables, seqs, positions, pages = build(10, [6], 5, 1, [10, 100])

    def on_side(go):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            go()
        torch.cuda.current_stream().wait_stream(side)

    def captured(go):
        go()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            go()
        graph.replay()
        graph.replay()
        torch.cuda.synchronize()

    for call in (on_side, captured):
        for dtype in (torch.bfloat16, torch.float32):
            check(tables, seqs, positions, pages, 9, 3, 64, dtype, call=call)


def test_shared_attention_refuses():
    from nnis_b200.engine.workspace import Workspace
    o = ops()
    plan_of = lambda **kw: o.attention_shared_plan(**{**dict(tables=[[0, 1], [0, 2]], seqs=[0, 1], positions=[70, 80], heads=4,
                                                             kv_heads=2, head_dim=64, dtype=torch.float32, device=DEV), **kw})
    for bad in (dict(seqs=[0, 2]), dict(positions=[70, 128]), dict(positions=[1]), dict(heads=3), dict(head_dim=63),
                dict(head_dim=258), dict(dtype=torch.float16), dict(seqs=[], positions=[]),
                dict(tables=[[0, -1], [0, 2]])):
        with pytest.raises(o.KernelError):
            plan_of(**bad)
    plan, ws = plan_of(), Workspace(torch.device(DEV))
    q = torch.zeros((2, 256), device=DEV)
    k = torch.zeros((3, 2, 64, 64), device=DEV)
    pos = torch.tensor([70, 80], dtype=torch.int32, device=DEV)
    table = torch.tensor([[0, 1], [0, 2]], dtype=torch.int32, device=DEV)
    args = dict(q=q, q_stride=256, k_cache=k, v_cache=k, token_pos=pos, page_table=table, plan=plan, out=torch.empty_like(q),
                heads=4, kv_heads=2, head_dim=64, scale=0.1, workspace=ws)
    o.attention_shared(**args)
    for bad in (dict(q=q[:1]), dict(out=torch.empty((3, 256), device=DEV)), dict(page_table=table[:, :1].contiguous()),
                dict(page_table=table[:1]), dict(k_cache=k.bfloat16()), dict(heads=2, out=torch.empty((2, 128), device=DEV)),
                dict(q_stride=200), dict(token_pos=pos[:1]), dict(out=torch.empty((2, 256), dtype=torch.bfloat16, device=DEV))):
        with pytest.raises(o.KernelError):
            o.attention_shared(**{**args, **bad})
