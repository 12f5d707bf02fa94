"""Which batches read shared pages once (no GPU)."""
import pytest
import torch

from nnis_b200.csrc import ops
from nnis_b200.engine import sharing

F32, BF16 = torch.float32, torch.bfloat16


def pays(heads, kv_heads, dim, dtype, rows, pages, ahead=0):
    """``rows`` sequences behind ``pages`` shared pages, 21 tokens of each one's own."""
    tables = [list(range(pages)) + [pages + r] for r in range(rows)]
    positions = [pages * 64 + 20] * rows
    tree = ops.shared_nodes(tables, range(rows), positions, ahead)
    return sharing.heads_share(tree, positions, (0, heads, kv_heads, dim), dtype, ahead)


# measured us a layer, row by row and shared
MEASURED = [(12, 12, 96, BF16, 2, 512, 107.45, 344.56), (12, 12, 96, BF16, 4, 303, 120.40, 205.24), (12, 12, 96, BF16, 16, 15, 32.08, 26.16),
            (12, 12, 96, BF16, 64, 4, 35.41, 55.47), (16, 4, 96, BF16, 2, 341, 73.71, 96.85), (16, 4, 96, BF16, 4, 228, 97.65, 74.60),
            (16, 4, 96, BF16, 64, 43, 230.91, 94.25), (8, 2, 256, BF16, 16, 34, 88.67, 74.16), (8, 8, 256, BF16, 2, 512, 248.78, 634.24),
            (24, 12, 96, BF16, 8, 130, 150.16, 95.77), (32, 4, 96, BF16, 2, 341, 135.74, 100.06), (8, 8, 72, BF16, 4, 512, 133.07, 198.18),
            (12, 12, 96, F32, 2, 114, 48.00, 87.91), (12, 12, 96, F32, 8, 16, 39.65, 21.08), (12, 12, 96, F32, 64, 2, 33.57, 50.82),
            (16, 4, 96, F32, 64, 3, 49.72, 37.29), (32, 32, 64, F32, 2, 64, 41.10, 48.49), (32, 32, 64, F32, 4, 21, 34.59, 24.43),
            (32, 32, 64, F32, 64, 1, 25.73, 54.55), (9, 3, 64, F32, 2, 341, 75.93, 33.83), (32, 8, 128, F32, 64, 2, 70.98, 34.96),
            (9, 3, 64, BF16, 64, 256, 137.0, 19.0), (32, 32, 64, BF16, 2, 64, 15.5, 11.0)]


@pytest.mark.parametrize("heads,kv_heads,dim,dtype,rows,pages,alone,shared", MEASURED)
@pytest.mark.parametrize("ahead", [0, 8])
def test_batches_share_where_that_was_measured_to_pay(heads, kv_heads, dim, dtype, rows, pages, alone, shared, ahead):
    """With room to grow or without: the room is not read."""
    assert pays(heads, kv_heads, dim, dtype, rows, pages, ahead) == (shared < alone)


def test_more_rows_and_more_heads_of_a_group_pay_sooner():
    for dtype, dim in ((BF16, 96), (F32, 96), (F32, 64)):
        assert not pays(4, 4, dim, dtype, 2, 30) and pays(4, 4, dim, dtype, 16, 30) and pays(64, 4, dim, dtype, 2, 30)


def test_padding_rows_count_for_nothing():
    tables, positions = [[0, 1, 2], [0, 1, 3]], [140, 141]
    tree = ops.shared_nodes(tables, [0, 1], positions)
    padded = ops.shared_nodes(tables, [0, 1, 0, 0], positions + [-1, -1])
    for heads in (2, 8, 16):
        key = (0, heads, 1, 96)
        assert sharing.heads_share(tree, positions, key, BF16) == sharing.heads_share(padded, positions + [-1, -1], key, BF16)
