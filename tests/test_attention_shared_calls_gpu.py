"""Attention over shared pages, called as a program may call it: right behind the kernels that write what it reads."""
import math

import pytest
import torch

from test_attention_shared_gpu import build, check

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def ops():
    from nnis_b200.csrc import ops as o
    return o


FORMS = [(9, 3, 64, torch.bfloat16, 3), (32, 32, 64, torch.bfloat16, 40), (8, 2, 64, torch.bfloat16, 40), (16, 2, 128, torch.bfloat16, 9),
         (9, 3, 64, torch.float32, 9), (6, 2, 128, torch.float32, 20), (6, 3, 48, torch.bfloat16, 5), (4, 1, 96, torch.float32, 9)]


@pytest.mark.parametrize("heads,kv_heads,dim,dtype,members", FORMS)
def test_positions_and_page_tables_written_by_the_kernel_before(heads, kv_heads, dim, dtype, members):
    """Positions by a kernel that lets the next one start before it has written them, page tables just before that: every form sees
    what they wrote, call after call.  (Positions are right only in that kernel's results: one behind them before it, and tables
    name the wrong pages.)"""
    from nnis_b200.engine.workspace import Workspace
    o, held = ops(), {}
    tables, seqs, positions, pages = build(12, [5], members, 1, [2, 65, 130])

    def keep(go):
        held.update(zip(go.__code__.co_freevars, (c.cell_contents for c in go.__closure__)))
        pos, table, n = held["pos"], held["table"], len(positions)
        pos0, table0 = pos - 1, table.flip(0).contiguous()
        real_pos, real_table = pos.clone(), table.clone()
        none = torch.zeros(n, dtype=torch.int32, device=DEV)
        for _ in range(20):
            held["out"].fill_(77.0)
            pos.copy_(pos0)
            table.copy_(table0)
            table.copy_(real_table)
            o.advance(none.clone(), pos, none)
            go()
        assert torch.equal(pos, real_pos)

    check(tables, seqs, positions, pages, heads, kv_heads, dim, dtype, seed=5, call=keep)


@pytest.mark.parametrize("heads,kv_heads,dim,dtype,members", FORMS)
def test_a_row_beyond_the_end_of_its_plan_sets_the_status_word(heads, kv_heads, dim, dtype, members):
    """One row of a batch a page behind what its plan was made for; at the plan's own positions, on its last page and for padding rows
    nothing is set.  (Tables and store have the page: nothing is out of range.)"""
    from nnis_b200.engine.workspace import Workspace
    o = ops()
    tables, seqs, positions, pages = build(13, [5], members, 1, [2, 65, 130])
    plan = o.attention_shared_plan(tables, seqs, positions, heads, kv_heads, dim, dtype, DEV)
    k = torch.randn((pages, kv_heads, 64, dim), device=DEV).to(dtype)
    q = torch.randn((len(seqs), heads * dim), device=DEV).to(dtype)
    table = torch.zeros((len(tables), 12), dtype=torch.int32)
    for i, t in enumerate(tables):
        table[i, :len(t)] = torch.tensor(t)
    table, out = table.to(DEV), torch.empty_like(q)

    def run(at):
        o.attention_shared(q, heads * dim, k, k, torch.tensor(at, dtype=torch.int32, device=DEV), table, plan, out, heads, kv_heads, dim,
                           0.1, Workspace(torch.device(DEV)))

    o.check_status(DEV)
    run(positions)
    o.check_status(DEV)
    run([p // 64 * 64 + 63 for p in positions])
    run([-1] * len(positions))
    o.check_status(DEV)
    padded = o.attention_shared_plan(tables, seqs, [-1, *positions[1:-1], -1], heads, kv_heads, dim, dtype, DEV)
    o.attention_shared(q, heads * dim, k, k, torch.tensor([-1, *positions[1:-1], -1], dtype=torch.int32, device=DEV), table, padded, out,
                       heads, kv_heads, dim, 0.1, Workspace(torch.device(DEV)))
    o.check_status(DEV)
    for row in (0, len(positions) - 1):
        run([p // 64 * 64 + 64 if r == row else p for r, p in enumerate(positions)])
        with pytest.raises(o.KernelError, match="beyond the pages of its plan"):
            o.check_status(DEV)
        o.check_status(DEV)
    assert math.isfinite(float(out.float().sum()))


def test_two_threads_at_once():
    """Two head sizes of one kernel, each on a stream and a workspace of its own, as often as one alone: the same to the bit."""
    import threading
    from nnis_b200.engine.workspace import Workspace
    o, work = ops(), []
    for seed, dim in ((1, 30), (2, 62)):
        tables, seqs, positions, pages = build(20 + seed, [5], 6, 1, [2, 65, 130])
        g = torch.Generator(device=DEV).manual_seed(seed)
        k = torch.randn((pages, 2, 64, dim), generator=g, device=DEV)
        q = torch.randn((len(seqs), 6 * dim), generator=g, device=DEV)
        cols = max(map(len, tables))
        table = torch.tensor([t + [-1] * (cols - len(t)) for t in tables], dtype=torch.int32, device=DEV)
        at = torch.tensor(positions, dtype=torch.int32, device=DEV)
        plan = o.attention_shared_plan(tables, seqs, positions, 6, 2, dim, torch.float32, DEV)
        ws = Workspace(torch.device(DEV))
        work.append(lambda out, q=q, k=k, at=at, table=table, plan=plan, dim=dim, ws=ws:
                    o.attention_shared(q, 6 * dim, k, k, at, table, plan, out, 6, 2, dim, 0.1, ws))
        work[-1].like = q
    got, errors = [[], []], []

    def run(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream(DEV)):
                for _ in range(30):
                    got[i].append(torch.empty_like(work[i].like))
                    work[i](got[i][-1])
                torch.cuda.current_stream().synchronize()
        except Exception as error:
            errors.append(error)

    torch.cuda.synchronize()
    threads = [threading.Thread(target=run, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for i in (0, 1):
        want = torch.empty_like(work[i].like)
        work[i](want)
        assert all(torch.equal(x, want) for x in got[i])


@pytest.mark.parametrize("heads,kv_heads,dim,dtype,members", FORMS)
def test_the_same_call_gives_the_same_bits(heads, kv_heads, dim, dtype, members):
    """No order of units, records or merges changes a result, and neither does what the workspace held."""
    from nnis_b200.engine.workspace import Workspace
    o = ops()
    tables, seqs, positions, pages = build(14, [9], members, 2, [2, 65, 130])
    plan = o.attention_shared_plan(tables, seqs, positions, heads, kv_heads, dim, dtype, DEV)
    k, v = (torch.randn((pages, kv_heads, 64, dim), device=DEV).to(dtype) for _ in range(2))
    q = (2.0 * torch.randn((len(seqs), heads * dim), device=DEV)).to(dtype)
    cols = max(map(len, tables))
    table = torch.tensor([t + [-1] * (cols - len(t)) for t in tables], dtype=torch.int32, device=DEV)
    at, ws, first = torch.tensor(positions, dtype=torch.int32, device=DEV), Workspace(torch.device(DEV)), None
    for turn in range(30):
        out = torch.full_like(q, 77.0)
        if turn:
            ws.room("attn_shared_records", 1, torch.float32).fill_(math.nan if turn % 2 else 3.0)
        o.attention_shared(q, heads * dim, k, v, at, table, plan, out, heads, kv_heads, dim, 0.1, ws)
        first = out if first is None else first
        assert torch.equal(out, first)


@pytest.mark.parametrize("heads,kv_heads,dim,dtype", [(4, 1, 64, torch.bfloat16), (2, 2, 128, torch.bfloat16), (4, 1, 64, torch.float32),
                                                      (2, 1, 16, torch.bfloat16)])
def test_thousands_of_rows(heads, kv_heads, dim, dtype):
    """2,000 sequences behind two pages; 300 tokens of one sequence, the same position twice among them."""
    tables, seqs, positions, pages = build(15, [2], 2000, 0, [1, 40, 64, 70])
    check(tables, seqs, positions, pages, heads, kv_heads, dim, dtype, seed=6)
    positions = [399 - i for i in range(299)] + [399]
    check([list(range(7))], [0] * 300, positions, 7, heads, kv_heads, dim, dtype, seed=7)
