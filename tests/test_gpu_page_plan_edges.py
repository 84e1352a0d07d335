"""The page plan where sums of the counts pass 32 bits."""
import pytest
import torch

import tda_b200

pytestmark = pytest.mark.gpu
DEV = "cuda"
TOP = 2 ** 31 - 1


def ints(*x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("B", [3, 40, 5000])
def test_sums_of_new_tokens_past_32_bits(B):
    """Every request asks for 2^31 - 1 tokens: the first takes the 64 places there are, the others none."""
    page, width, rows = 16, 4, 64
    new = torch.full((B,), TOP, dtype=torch.int32, device=DEV)
    table = torch.full((B, width), -1, dtype=torch.int32, device=DEV)
    free = ints(5, 3, 9, 7)
    p = tda_b200.plan_pages(torch.zeros_like(new), new, table, free, ints(0), page, rows)
    assert p.slots.tolist() == [q * page + i for q in (5, 3, 9, 7) for i in range(page)]
    assert p.positions.tolist() == list(range(rows)) and p.requests.tolist() == [0] * rows
    assert p.starts.tolist() == [0] + [TOP] * B
    assert p.lengths.tolist() == [64] + [0] * (B - 1)
    assert p.free_head.tolist() == [4] and p.dropped.tolist() == [TOP]
    assert table[0].tolist() == [5, 3, 9, 7] and (table[1:] == -1).all()


def test_a_large_request_behind_small_ones():
    """Its rows are those that are left; a negative length is an empty request."""
    page, width = 16, 8
    table = torch.full((4, width), -1, dtype=torch.int32, device=DEV)
    table[0, 0] = 60
    free = torch.arange(10, dtype=torch.int32, device=DEV)
    p = tda_b200.plan_pages(ints(3, 0, -5, 0), ints(10, 20, TOP, TOP), table, free, ints(0), page, 30 + width * page)
    assert p.starts.tolist() == [0, 10, 30, TOP, TOP]
    assert p.lengths.tolist() == [13, 20, 128, 0]
    assert p.slots.tolist() == [60 * page + i for i in range(3, 13)] + list(range(20)) + [2 * page + i for i in range(128)]
    assert p.requests.tolist() == [0] * 10 + [1] * 20 + [2] * 128
    assert p.free_head.tolist() == [10] and p.dropped.tolist() == [TOP]
    assert table.tolist() == [[60] + [-1] * 7, [0, 1] + [-1] * 6, list(range(2, 10)), [-1] * 8]


@pytest.mark.parametrize("rows,slots,lengths,taken", [
    (0, [], [3, 0, 20], 0),
    (4, [[0, 3], [0, 4], [0, 5], [0, 6]], [7, 0, 20], 0),
    (10, [[0, i] for i in range(3, 13)], [13, 0, 20], 0),
    (29, [[0, i] for i in range(3, 13)] + [[5, i] for i in range(16)] + [[6, i] for i in range(3)], [13, 19, 20], 2),
    (37, [[0, i] for i in range(3, 13)] + [[5, i] for i in range(16)] + [[6, i] for i in range(11)], [13, 27, 20], 2),
    (42, [[0, i] for i in range(3, 13)] + [[5, i] for i in range(16)] + [[6, i] for i in range(11)] + [[2, i] for i in range(4, 9)],
     [13, 27, 25], 2),
])
def test_fewer_rows_than_new_tokens(rows, slots, lengths, taken):
    """Tokens without a row are dropped: no page, no length, and they are counted."""
    page = 16
    table = torch.tensor([[0, -1, -1], [-1, -1, -1], [1, 2, -1]], dtype=torch.int32, device=DEV)
    p = tda_b200.plan_pages(ints(3, 0, 20), ints(10, 27, 5), table, ints(5, 6, 7), ints(0), page, rows)
    assert p.slots.tolist() == [q * page + i for q, i in slots]
    assert p.lengths.tolist() == lengths and p.free_head.tolist() == [taken]
    assert p.dropped.tolist() == [42 - rows] and p.starts.tolist() == [0, 10, 37, 42]
    assert table.tolist() == [[0, -1, -1], [5, 6, -1] if taken else [-1] * 3, [1, 2, -1]]


def test_rows_that_end_in_a_later_scan():
    """3000 requests of one token and rows for 2100 of them."""
    B, rows, page = 3000, 2100, 16
    zeros = torch.zeros(B, dtype=torch.int32, device=DEV)
    table = torch.full((B, 1), -1, dtype=torch.int32, device=DEV)
    p = tda_b200.plan_pages(zeros, zeros + 1, table, torch.arange(B, dtype=torch.int32, device=DEV), ints(0), page, rows)
    assert p.lengths.tolist() == [1] * rows + [0] * (B - rows)
    assert p.dropped.tolist() == [B - rows] and p.free_head.tolist() == [rows]
    assert table.flatten().tolist() == list(range(rows)) + [-1] * (B - rows)
    assert p.slots.tolist() == [page * i for i in range(rows)]
