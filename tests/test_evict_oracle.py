"""Eviction past an empty pool, on the CPU: table entries without a page leave their rows, but are no
pages that anyone could be handed again."""

import torch

from oracle import longctx as oc
from oracle import serving as sv


def test_an_entry_without_a_page_takes_no_place_in_the_free_list():
    w = torch.tensor([5.0, 1, 2, 2, 9, 0.5, 4, 3]).view(8, 1, 1)
    # five columns, two stay: -1 goes before the pages of weight 1 and 2, and only those come back
    table, free, lens, used, lost = sv.evict(w, 64, [[6, 1, -1, 3, 4]], [320], [2], [9, 9], 2, 0, 1)
    assert table == [[6, 4, -1, -1, -1]] and lens == [128]
    assert free == [1, 3] and used == 0 and lost == 0
    # over requests: places and counts go by pages alone
    rows = [[0, -1, 8, 4], [-1, 2 ** 31 - 1, 5, 6], [-1, -1, -1, 7]]
    table, free, lens, used, lost = sv.evict(w, 64, rows, [256, 250, 256], [1, 1, 1],
                                             [10, 11, 12, 13], 3, 0, 1)
    assert table == [[4, -1, -1, -1], [6, -1, -1, -1], [7, -1, -1, -1]]
    assert lens == [64, 58, 64] and free == [10, 0, 5, 13] and used == 1 and lost == 0
    # no room: what is lost are pages
    table, free, lens, used, lost = sv.evict(w, 64, [[-1, 2, -1, 3, 1]], [320], [1], [9], 1, 0, 1)
    assert free == [2] and used == 0 and lost == 1


def test_the_pool_recovers():
    """6 pages, two requests that together ask for more: every page stays held or free, once."""
    free, used, table, lens = list(range(6)), 0, [[-1] * 6, [-1] * 6], [0, 0]
    w = torch.arange(1.0, 7).view(6, 1, 1)
    lacking = 0
    for new in ([128, 128], [128, 128], [128, 64], [64, 128], [64, 64], [64, 128]):
        _, _, lens, used, missing, table = oc.plan_pages(lens, new, table, free, used, 64, sum(new))
        lacking += missing
        table, free, lens, used, lost = sv.evict(w, 64, table, lens, [3, 3], free, used, 1, 1)
        held = [p for r in table for p in r if p >= 0]
        assert sorted(held + free[used:]) == list(range(6)) and lost == 0
    assert lacking
