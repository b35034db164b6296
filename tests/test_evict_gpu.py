"""Eviction of the 8-bit cache's pages on the GPU at the ends of its arguments' ranges."""

import pytest
import torch

from gfx906_amd import kv8

pytestmark = pytest.mark.gpu
DEV = "cuda"


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("W", [3, 700, 5000])
@pytest.mark.parametrize("first,recent", [(2 ** 31 - 1, 1), (2 ** 40, 1), (1, 2 ** 31 - 1), (0, 2 ** 40),
                                          (2 ** 31 - 1, 2 ** 31 - 1), (2 ** 31 - 500, 2)])
def test_rows_that_are_kept_whole(first, recent, W):
    """As many first or most recent pages as an int counts: nothing goes."""
    print(f"evict first {first} recent {recent} of {W} columns", flush=True)
    weights = torch.rand(2 * W, 2, 1, device=DEV)
    rows = torch.arange(2 * W, dtype=torch.int32, device=DEV).view(2, W)
    table, free = rows.clone(), i32([7, 8, 9])
    lens = i32([64 * W, 64 * W - 5])
    got = kv8.evict(weights, table, lens, i32([1, 0]), free, i32([2]), first, recent)
    assert torch.equal(table, rows) and free.tolist() == [7, 8, 9]
    assert torch.equal(got.lens, lens) and got.used.item() == 2 and got.lost.item() == 0


def test_all_but_the_row_s_ends_may_go():
    """first and recent that fit the row exactly, and by one less."""
    weights = torch.rand(6, 1, 1, device=DEV)
    for first, recent, left in ((3, 3, 6), (3, 2, 5), (6, 1, 6), (5, 1, 6), (4, 1, 5)):
        table, free = i32([list(range(6))]), i32([0] * 6)
        got = kv8.evict(weights, table, i32([64 * 6]), i32([0]), free, i32([6]), first, recent)
        assert got.lens.item() == 64 * left and got.used.item() == left
        if left == 5:
            assert free.tolist() == [0] * 5 + [first]
