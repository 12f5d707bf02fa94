"""Pages copied inside the store: exact, and nothing but the targets' rows written."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def ops():
    from nnis_b200.csrc import ops as o
    return o


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layers,heads,dim,vdim", [(1, 1, 2, 2), (3, 3, 64, 64), (2, 5, 48, 30), (2, 1, 66, 0), (30, 2, 128, 64), (2, 1, 33, 0), (1, 3, 5, 7)])
@pytest.mark.parametrize("case", ["one row", "ragged", "whole", "one source", "mixed"])
def test_rows_of_pages_are_copied(dtype, layers, heads, dim, vdim, case):
    """Rows from one to all, words of 16, 4 and 2 bytes, values of another size or none, no rows at all."""
    g = torch.Generator().manual_seed(layers * dim)
    pages = 23
    k = torch.randn((layers, pages, heads, 64, dim), generator=g).to(dtype).to(DEV)
    v = torch.randn((layers, pages, heads, 64, vdim), generator=g).to(dtype).to(DEV) if vdim else None
    moves = {"one row": [(4, 9, 1)], "ragged": [(i, 22 - i, 1 + (i * 29) % 64) for i in range(11)],
             "whole": [(0, 22, 64), (21, 1, 64), (3, 2, 64)], "one source": [(7, d, 37) for d in range(23) if d != 7],
             "mixed": [(0, 1, 64), (2, 3, 63), (2, 4, 0), (5, 6, 2)]}[case]
    want = []
    for store in (k, v):
        expect = store.clone() if store is not None else None
        if expect is not None:
            for s, d, r in moves:
                expect[:, d, :, :r] = store[:, s, :, :r]
        want.append(expect)
    ops().copy_pages(k, v, moves)
    assert torch.equal(k, want[0])
    assert v is None or torch.equal(v, want[1])


def test_more_moves_than_a_launch_takes():
    """2,500 moves are three launches; source and target lie at either end of the store."""
    o = ops()
    k = torch.randn((2, 5000, 1, 64, 2), device=DEV)
    want = k.clone()
    want[:, 2500:] = k[:, :2500].flip(1)
    before = o.launch_count()
    o.copy_pages(k, None, [(i, 4999 - i, 64) for i in range(2500)])
    assert o.launch_count() - before == 3
    assert torch.equal(k, want)


def test_a_store_of_more_than_four_giga_elements_of_bytes():
    """Pages whose bytes lie beyond 32 bits from the store's first."""
    k = torch.zeros((2, 40000, 4, 64, 128), dtype=torch.bfloat16, device=DEV)  # 5 GB a layer
    k[1, 39999] = torch.randn((4, 64, 128), device=DEV).to(torch.bfloat16)
    ops().copy_pages(k, None, [(39999, 0, 64), (39998, 39997, 64)])
    assert torch.equal(k[1, 0], k[1, 39999]) and not k[0].any()
    del k
    torch.cuda.empty_cache()


def test_copies_run_on_the_current_stream_and_into_graphs():
    """A replayed copy copies what the source holds then."""
    o = ops()
    k = torch.randn((2, 6, 3, 64, 64), device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o.copy_pages(k, None, [(0, 1, 5)])
    side.synchronize()
    assert torch.equal(k[:, 1, :, :5], k[:, 0, :, :5])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o.copy_pages(k, None, [(2, 3, 64)])
    k[:, 2] = 7.0
    graph.replay()
    torch.cuda.synchronize()
    assert bool((k[:, 3] == 7.0).all())


def test_moves_that_are_refused():
    o = ops()
    k = torch.zeros((1, 4, 1, 64, 2), device=DEV)
    for moves in ([(0, 4, 1)], [(-1, 0, 1)], [(0, 1, 65)], [(0, 1, -1)], [(0, 1, 2), (2, 1, 3)], [(0, 1, 2), (1, 2, 2)], [(1, 1, 1)],
                  [(0, 1)], [(0, 1, 1), (2, 3)], [(0, 1, 2.5)], [(0, 1, 2 ** 40)]):
        with pytest.raises(o.KernelError):
            o.copy_pages(k, None, moves)
    with pytest.raises(o.KernelError):
        o.copy_pages(k[0], None, [(0, 1, 1)])
    with pytest.raises(o.KernelError):
        o.copy_pages(k, torch.zeros((1, 5, 1, 64, 2), device=DEV), [(0, 1, 1)])
    with pytest.raises(o.KernelError):
        o.copy_pages(k.transpose(1, 3), None, [(0, 1, 1)])
    o.copy_pages(k, None, [])
    assert not k.any()
