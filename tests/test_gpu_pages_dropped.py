"""Compactions that leave requests out: the pages that only these held are free pages, and
a free page has a count of 0."""
import pytest
import torch

from _pages import pages_of

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("max_moves", [0, 1, 64])
@pytest.mark.parametrize("kept_row", [[40, 41, 42], [0, 5, 63], [7, 8, 9]])
def test_pages_of_omitted_requests_come_back_without_holders(kept_row, max_moves):
    """Rows 1 and 2 share pages and are left out; row 0 stays."""
    import atflash
    P, page, width = 64, 16, 4
    table = _i32([kept_row + [-1], [20, 21, 22, -1], [20, 21, 23, -1], [-1] * 4])
    shared, free = _i32([0] * P), _i32([0] * P)
    shared[20] = shared[21] = 1
    c = atflash.compact_pages(_i32([48]), table, page, P, max_moves=max_moves, free_pages=free, req_rows=_i32([0]),
                              shared=shared)
    head = c.free_head.item()
    assert head == 3
    listed = free[head:].tolist()
    assert sorted(listed + table[0, :3].tolist()) == list(range(P))
    assert shared.tolist() == [0] * P
    # a request that takes such pages and is freed gives them all back
    table[3] = free[head:head + width]
    took = table[3].tolist()
    after = atflash.free_requests(_i32([3]), _i32([page * width]), table, page, free_pages=free, free_head=_i32([head + width]),
                                  shared=shared)
    assert after.tolist() == [head] and sorted(free[head:head + width].tolist()) == sorted(took)
    assert shared.tolist() == [0] * P
    assert atflash.check_device_errors() == 0


def test_moved_pages_take_their_counts_into_pages_of_omitted_requests():
    """A shared page moves into a hole that had a count of its own, left by omitted rows."""
    import atflash
    P, page = 32, 16
    table = _i32([[30, 31], [30, 29], [0, 1], [0, 1]])
    shared, free = _i32([0] * P), _i32([0] * P)
    shared[30], shared[0], shared[1] = 1, 5, 1
    c = atflash.compact_pages(_i32([32, 32]), table, page, P, max_moves=P, free_pages=free, req_rows=_i32([0, 1]),
                              shared=shared)
    assert c.src.tolist()[:4] == [31, 30, 29, -1] and c.dst.tolist()[:4] == [0, 1, 2, -1]
    assert table[:2].tolist() == [[1, 0], [1, 2]]
    assert shared.tolist() == [0, 1] + [0] * (P - 2)
    assert c.free_head.tolist() == [pages_of(48, page)]
    assert atflash.check_device_errors() == 0
