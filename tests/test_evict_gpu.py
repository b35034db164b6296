"""Eviction of the 8-bit cache's pages on the GPU at the ends of its arguments' ranges."""

import pytest
import torch

from gfx906_amd import kv8
from oracle import serving as sv

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


BAD = [-1, 2 ** 31 - 1, -2 ** 31, -7]


@pytest.mark.parametrize("less", [0, 3, 1000])
@pytest.mark.parametrize("B,W,page", [(1, 9, 64), (1, 700, 128), (2, 30, 256), (9, 40, 64), (70, 513, 64),
                                      (300, 300, 64), (2, 4500, 64), (33, 4100, 128), (4096, 5, 64)])
def test_entries_without_a_page(B, W, page, less):
    """Few, many or only entries that name no page, in every part of the rows: they leave the rows,
    and pages alone are counted and given back."""
    print(f"evict {B} x {W} pages of {page}, {less} fewer used", flush=True)
    g = torch.Generator().manual_seed(B + W)
    held = [int(torch.randint(0, W + 1, (1,), generator=g)) for _ in range(B)]
    held[0] = W
    pages = sum(held) + 3
    phys, at, rows = torch.randperm(pages, generator=g).tolist(), 0, []
    for b, n in enumerate(held):
        row, at = phys[at:at + n], at + n
        part = [0.0, 0.02, 0.5, 0.9, 1.0][(b + B) % 5] if B > 1 else 0.3
        hit = (torch.rand(n, generator=g) < part).tolist()
        rows.append([[*BAD, pages][(b + c) % 5] if x else p for c, (p, x) in enumerate(zip(row, hit))]
                    + [-1] * (W - n))
    weights = torch.exp(2 * torch.randn(pages, 2, page // 64, generator=g))
    weights[::7] = float("nan")
    weights[3::7] = -float("inf")
    lens = [max(0, n * page - b % 50) for b, n in enumerate(held)]
    keep = [max(0, n // 3 - b % 3) for b, n in enumerate(held)]
    free, used = list(range(10 ** 6, 10 ** 6 + sum(held) + 5)), max(0, sum(held) - less)
    for first, recent in ((1, 1), (0, 3)):
        table, pool = i32(rows), i32(free)
        got = kv8.evict(weights.to(DEV), table, i32(lens), i32(keep), pool, i32([used]), first, recent)
        want = sv.evict(weights, page, rows, lens, keep, free, used, first, recent)
        for name, a, b in zip(("table", "free", "lens", "used", "lost"), (table, pool, *got),
                              (want[0], want[1], want[2], [want[3]], [want[4]])):
            assert a.tolist() == b, name


def test_serving_past_an_empty_pool():
    """Requests ask for more pages than there are, step after step: what finds no page is passed over
    and counted, and every page stays some request's or free, once."""
    B, Hq, Hkv, D, page, pages, keep = 3, 4, 2, 64, 64, 10, 3
    g = torch.Generator().manual_seed(0)
    cache, held = kv8.new_cache(pages, page, Hkv, D), sv.Cache(pages, page, Hkv, D)
    weights = kv8.new_weights(cache)
    table = torch.full((B, 8), -1, dtype=torch.int32, device=DEV)
    free, lens, used = i32(torch.randperm(pages, generator=g).tolist()), i32([0] * B), i32([0])
    lacking = 0
    for news in ([200, 130, 64], [130, 200, 1], [1, 1, 129], [64, 64, 64], [1, 1, 1], [200, 1, 70],
                 [1, 130, 130], [1, 1, 1]):
        plan = kv8.plan_pages(lens, i32(news), table, free, used, page, sum(news))
        lacking += plan.missing.item()
        x = torch.randn(sum(news), Hq + 2 * Hkv, D, generator=g).half().to(DEV)
        q, k, v = x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:]
        kv8.store(cache, k, v, table, plan.lens, plan.cu_new, weights)
        out, lse = kv8.attn(q, cache, table, plan.lens, D ** -0.5, cu_q=plan.cu_new, max_q=max(news),
                            lse=True)
        kv8.weigh(weights, q, lse, cache, table, plan.lens, D ** -0.5, cu_q=plan.cu_new, max_q=max(news))
        rows, n, cu = table.tolist(), plan.lens.tolist(), plan.cu_new.tolist()
        held.store(k.cpu(), v.cpu(), rows, n, cu)
        for r, (o, tol, l, ltol) in sv.attention(q.cpu(), held, rows, n, D ** -0.5, cu).items():
            assert ((out[r].double().cpu() - o).abs() <= tol).all()
            blind = l.isinf()
            assert torch.equal(lse[r].cpu().isinf(), blind)
            assert ((lse[r].double().cpu() - l).abs() <= ltol)[~blind].all()
        w, f, u = weights.cpu(), free.tolist(), plan.used.item()
        gone = kv8.evict(weights, table, plan.lens, i32([keep] * B), free, plan.used)
        want = sv.evict(w, page, rows, n, [keep] * B, f, u, 1, 1)
        for a, b in zip((table, free, gone.lens, gone.used, gone.lost),
                        (want[0], want[1], want[2], [want[3]], [want[4]])):
            assert a.tolist() == b
        lens, used = gone.lens, gone.used
        mine = [p for r in table.tolist() for p in r if p >= 0]
        assert sorted(mine + free[used.item():].tolist()) == list(range(pages))
        assert gone.lost.item() == 0
    assert lacking


def test_replayed_with_other_tables():
    """One captured call, replayed with tables that lack other pages; eager work in between."""
    B, W = 5, 40
    g = torch.Generator().manual_seed(3)
    weights = torch.rand(B * W, 1, 1, device=DEV)
    table, free, used = torch.zeros(B, W, dtype=torch.int32, device=DEV), i32([0] * B * W), i32([B * W])
    lens, keep = i32([64 * W] * B), i32([W // 4] * B)
    graph = torch.cuda.CUDAGraph()
    kv8.evict(weights, table, lens, keep, free, used)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = kv8.evict(weights, table, lens, keep, free, used)
    for n in range(4):
        rows = torch.randperm(B * W, generator=g).int().view(B, W)
        rows[torch.rand(B, W, generator=g) < 0.2 * n] = -1
        table.copy_(rows)
        free.zero_()
        graph.replay()
        replayed = [t.clone() for t in (table, free, *got)]
        table.copy_(rows)
        free.zero_()
        again = kv8.evict(weights, table, lens, keep, free, used)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(replayed, (table, free, *again))), n
