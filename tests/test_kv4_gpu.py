"""The 4-bit cache on the GPU against the CPU oracle in 64 bits: pages and slots,
storing and reading, attention over it, and a run of them together."""

import math

import pytest
import torch

from gfx906_amd import kv4
from oracle import longctx as oc

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float16, torch.bfloat16]


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


# -- pages and slots ----------------------------------------------------------------------

PLANS = [  # lens, new, page, table width, free pages, used, extra slots
    ([0], [1], 64, 1, 1, 0, 0),
    ([0, 0], [0, 0], 64, 2, 0, 0, 3),
    ([63, 64, 65], [1, 1, 1], 64, 3, 2, 1, 0),
    ([5, 0, 700, 128, 1], [300, 1, 0, 129, 64], 128, 7, 12, 2, 9),
    ([0, 10, 20], [1000, 2000, 3], 256, 20, 30, 0, 0),
    ([0, 100, 60], [500, 100, 300], 64, 4, 6, 0, 2),      # list and rows end early
    ([-3, 7], [5, -2], 64, 2, 2, 0, 0),                   # negative counts are 0
    (list(range(300)), [k % 5 for k in range(300)], 64, 8, 300, 0, 5),
    ([17] * 4096, [1] * 4096, 64, 1, 0, 0, 0),
]


@pytest.mark.parametrize("case", range(len(PLANS)))
def test_plan_pages(case):
    lens, new, page, W, n_free, used, extra = PLANS[case]
    print(f"plan {case}", flush=True)
    g = torch.Generator().manual_seed(case)
    phys = torch.randperm(n_free + len(lens) * W, generator=g).tolist()
    free, phys = phys[:n_free], phys[n_free:]
    table = [[phys[b * W + k] if k < -(-max(0, n) // page) else -1 for k in range(W)]
             for b, n in enumerate(lens)]
    tokens = sum(max(0, n) for n in new) + extra
    wide = torch.full((len(lens), W + 3), -7, dtype=torch.int32, device=DEV)  # strided rows
    wide[:, :W] = i32(table)
    plan = kv4.plan_pages(i32(lens), i32(new), wide[:, :W], i32(free), i32([used]), page, tokens)
    want = oc.plan_pages(lens, new, table, free, used, page, tokens)
    for got, ref in zip((*plan, wide[:, :W]), (want[0], want[1], want[2], [want[3]], [want[4]],
                                               want[5])):
        assert got.tolist() == ref
    assert wide[:, W:].eq(-7).all()
    # The call reads what it does not write: again with the same arguments, the same result.
    again = kv4.plan_pages(i32(lens), i32(new), wide[:, :W], i32(free), i32([used]), page, tokens)
    assert all(torch.equal(a, b) for a, b in zip(plan, again))


def test_plan_pages_with_a_short_slot_list():
    plan = kv4.plan_pages(i32([0, 0]), i32([70, 3]), i32([[-1, -1], [-1, -1]]), i32([4, 5, 6]),
                          i32([0]), 64, 10)
    assert plan.slots.tolist() == list(range(256, 266)) and plan.cu_new.tolist() == [0, 70, 73]


def test_plan_pages_with_counts_up_to_an_int():
    """Sums past 31 bits saturate; what comes before them is as ever."""
    top = 2 ** 31 - 1
    table = i32([[3, 4, 5], [6, 7, 9], [9, 9, 9]])
    plan = kv4.plan_pages(i32([top, 100, 0]), i32([top, top, 5]), table, i32([11, 12, 13, 14]),
                          i32([0]), 64, 70)
    assert plan.slots.tolist() == [-1] * 70      # all of request 0, behind its row's three pages
    assert plan.cu_new.tolist() == [0, top, top, top] and plan.lens.tolist() == [top, top, 5]
    # 2^26 - 2^25 pages lacked, ceil((2^31 + 99) / 64) - 2 = 2^25, and 1: none is left for the others
    assert plan.used.item() == 4 and plan.missing.item() == 2 ** 26 + 1
    assert table.tolist() == [[3, 4, 5], [6, 7, -1], [-1, 9, 9]]

    table = i32([[-1, -1], [9, -1]])
    plan = kv4.plan_pages(i32([0, 5]), i32([3, top]), table, i32([7, 8]), i32([0]), 64, 200)
    want = [448, 449, 450] + [9 * 64 + p for p in range(5, 64)] + [512 + p for p in range(64)]
    assert plan.slots.tolist() == want + [-1] * (200 - len(want))
    assert plan.cu_new.tolist() == [0, 3, top] and plan.lens.tolist() == [3, top]
    # request 1 lacks ceil((2^31 + 4) / 64) - 1 = 2^25 pages and gets one
    assert plan.used.item() == 2 and plan.missing.item() == 2 ** 25 - 1
    assert table.tolist() == [[7, -1], [9, 8]]


def test_plan_pages_of_no_requests():
    none = i32([])
    plan = kv4.plan_pages(none, none, i32([]).view(0, 3), i32([1, 2]), i32([1]), 64, 3)
    assert plan.slots.tolist() == [-1] * 3 and plan.cu_new.tolist() == [0]
    assert plan.lens.numel() == 0 and plan.used.item() == 1 and plan.missing.item() == 0


def test_plan_pages_refuses():
    a = dict(lens=i32([1]), new_lens=i32([1]), table=i32([[0]]), free_pages=i32([1]), used=i32([0]),
             page=64, tokens=1)
    for bad in (dict(lens=i32([1]).long()), dict(new_lens=i32([1, 2])), dict(page=100),
                dict(tokens=-1), dict(table=i32([0])), dict(table=i32([[0], [1]])),
                dict(used=i32([0, 0])), dict(free_pages=torch.zeros(2, dtype=torch.int32)),
                dict(lens=i32([1, 1]), new_lens=i32([1, 1]), table=i32([[0]]).expand(2, 1)),
                dict(free_pages=None)):
        with pytest.raises((RuntimeError, TypeError)):
            kv4.plan_pages(**(a | bad))
    t = i32([[0]])
    with pytest.raises(RuntimeError):
        kv4.plan_pages(**(a | dict(table=t, free_pages=t[0])))


# -- storing and reading ------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,H,D,page", [(1, 1, 64, 64), (5, 3, 128, 64), (130, 2, 64, 128),
                                        (300, 5, 128, 256)])
def test_store_is_exact(T, H, D, page, dtype):
    print(f"store T{T} H{H} D{D} page {page} {dtype}", flush=True)
    g = torch.Generator().manual_seed(T + H)
    pages = T // page + 3
    x = torch.randn(2, T, H, D, generator=g) * torch.exp2(
        torch.randint(-12, 9, (2, T, H, 1), generator=g).float())
    x[0, 0, 0, :32] = 0
    x[1, -1, -1, 32:40] = torch.tensor([6.0, 7.0, 5.0, 2.5, 0.75, 0.25, 3.5, 1.25])
    if T > 4:   # special blocks
        x[0, 1, 0, 3], x[0, 2, 0, 33], x[0, 3, 0, 0] = math.nan, math.inf, -math.inf
        x[1, 1, 0, :32] = 2.0 ** -24
        x[1, 2, 0, :32] = 65504.0 if dtype == torch.float16 else 3.0e38
    k, v = (t.to(dtype) for t in x)
    slots = torch.randperm(pages * page, generator=g)[:T].int()
    cache = kv4.new_cache(pages, page, H, D)
    kv4.store(cache, k.to(DEV), v.to(DEV), slots.to(DEV))
    host = kv4.Cache(*(t.cpu() for t in cache))
    for x, codes, scales in ((k, host.k, host.k_scale), (v, host.v, host.v_scale)):
        c, e = oc.quantise(x)
        held = torch.zeros(pages, page, dtype=torch.bool)
        for t, s in enumerate(slots.tolist()):
            gc, ge = oc.read_cache(codes, scales, s // page, s % page)
            ok = (ge != 255).repeat_interleave(32, -1)
            assert torch.equal(ge, e[t]) and torch.equal(gc[ok], c[t].int()[ok]), (t, s)
            held[s // page, s % page] = True
        assert codes.transpose(1, 2)[~held].eq(0).all()   # other tokens untouched
    gk, gv = kv4.load(cache, slots.to(DEV), dtype)
    for x, got in ((k, gk), (v, gv)):
        want = oc.dequantise(*oc.quantise(x)).to(dtype)
        assert torch.equal(got.cpu().nan_to_num(9.0, 8.0, 7.0), want.nan_to_num(9.0, 8.0, 7.0))


def test_store_and_load_pass_over_slots_outside_and_read_strided_rows():
    T, H, D, page = 70, 2, 64, 64
    big = torch.randn(T, 3, 3, 96, device=DEV).half()
    k, v = big[:, 0, :H, :D], big[:, 1, 1:, 3:3 + D]   # v: not 16-byte aligned, copied
    slots = torch.arange(T, dtype=torch.int32, device=DEV)
    slots[3], slots[4], slots[5] = -1, 2 * page, 2 ** 31 - 1
    cache = kv4.new_cache(2, page, H, D)
    kv4.store(cache, k, v, slots)
    gk, gv = kv4.load(cache, slots)
    for x, got in ((k, gk), (v, gv)):
        want = oc.dequantise(*oc.quantise(x.cpu())).half()
        want[3:6] = 0
        assert torch.equal(got.cpu(), want)
    empty = torch.empty(0, dtype=torch.int32, device=DEV)
    kv4.store(cache, k[:0], v[:0], empty)
    assert kv4.load(cache, empty)[0].shape == (0, H, D)


def test_store_and_load_refuse():
    cache = kv4.new_cache(2, 64, 2, 64)
    x, s = torch.zeros(3, 2, 64, device=DEV).half(), i32([0, 1, 2])
    for k, v, slots in ((x.float(), x.float(), s), (x, x.bfloat16(), s), (x, x[:2], s),
                        (x, x, s[:2]), (x, x, s.long()), (x[:, :1], x[:, :1], s),
                        (x.cpu(), x, s), (x, x, s.cpu())):
        with pytest.raises(RuntimeError):
            kv4.store(cache, k, v, slots)
    for bad in (cache._replace(k=cache.k.int()), cache._replace(v=cache.v[:1]),
                cache._replace(k_scale=cache.k_scale[:, :1]), cache._replace(v=cache.v[:, :, ::2])):
        with pytest.raises(RuntimeError):
            kv4.load(bad, s)
    with pytest.raises(RuntimeError):
        kv4.load(cache, s, torch.float32)


# -- attention ----------------------------------------------------------------------------

def filled(lens, page, Hkv, D, dtype, seed, spare=2, gain=2.0):
    """(cache on the GPU, its CPU copy, table) of random rows in shuffled pages. What no
    token fills holds NaN scales: nothing may read it."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    pages = sum(need) + spare
    phys = torch.randperm(pages, generator=g).tolist()
    W = max(max(need, default=0), 1) + 1
    table = torch.full((len(lens), W), -1, dtype=torch.int32)
    cache = kv4.new_cache(pages, page, Hkv, D)
    for t in cache:
        t.fill_(255)
    at, slots = 0, []
    for b, n in enumerate(lens):
        table[b, :need[b]] = torch.tensor(phys[at:at + need[b]], dtype=torch.int32)
        slots += [phys[at + t // page] * page + t % page for t in range(n)]
        at += need[b]
    T = len(slots)
    if T:
        k = (torch.randn(T, Hkv, D, generator=g) * gain).to(dtype)
        v = torch.randn(T, Hkv, D, generator=g).to(dtype)
        kv4.store(cache, k.to(DEV), v.to(DEV), i32(slots))
    return cache, [t.cpu() for t in cache], table


def check(out, rows, untouched=None):
    """Computed rows within the bound, the others as they were."""
    out = out.double().cpu()
    worst = 0.0
    for r in range(out.shape[0]):
        if r not in rows:
            if untouched is not None:
                assert torch.equal(out[r], untouched[r].double().cpu()), f"row {r} written"
            continue
        o, tol = rows[r]
        nan = o.isnan()
        assert torch.equal(out[r].isnan(), nan), f"row {r}: NaN"
        err = ((out[r] - o).abs() / tol)[~nan]
        if err.numel():
            worst = max(worst, err.max().item())
            assert worst <= 1.0, f"row {r}: {worst} of the bound"
    print(f"  worst {worst:.3f} of the bound", flush=True)


HEADS = [(1, 1), (8, 2), (5, 5), (16, 1), (24, 2), (40, 1), (6, 2)]
DECODES = [[1], [0, 5], [63, 64, 65], [0, 1, 130, 700, 33], [2050, 1, 300]]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,page", [(64, 64), (128, 64), (128, 128), (64, 256), (128, 256)])
@pytest.mark.parametrize("lens", DECODES)
def test_single_tokens(lens, D, page, dtype):
    Hq, Hkv = HEADS[(len(lens) + D // 64 + page // 64) % len(HEADS)]
    print(f"decode lens {lens} heads {Hq}/{Hkv} D{D} page {page} {dtype}", flush=True)
    cache, host, table = filled(lens, page, Hkv, D, dtype, seed=sum(lens))
    q = torch.randn(len(lens), Hq, D, generator=torch.Generator().manual_seed(7)).to(dtype)
    out = kv4.attn(q.to(DEV), cache, table.to(DEV), i32(lens), D ** -0.5)
    check(out, oc.cache_attn(q, host, page, table, lens, D ** -0.5))


CHUNKS = [  # lens, queries of each request, rows behind the last
    ([1], [1], 0), ([64], [64], 0), ([130, 77, 300], [130, 1, 45], 5),
    ([500, 0, 20, 9], [3, 0, 20, 0], 1), ([5, 200], [9, 2], 0),   # more queries than tokens
    ([700], [300], 0), ([129, 1025], [2, 17], 3),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads", [(4, 4), (6, 2), (8, 1)])
@pytest.mark.parametrize("case", range(len(CHUNKS)))
def test_chunks(case, heads, dtype, causal):
    lens, news, behind = CHUNKS[case]
    Hq, Hkv = heads
    D, page = (64, 128)[case % 2], (64, 128, 256)[(case + Hq) % 3]
    print(f"chunks {case} heads {heads} D{D} page {page} {dtype} causal {causal}", flush=True)
    cache, host, table = filled(lens, page, Hkv, D, dtype, seed=case)
    cu = [0]
    for m in news:
        cu.append(cu[-1] + m)
    T = cu[-1] + behind
    q = torch.randn(T, Hq, D, generator=torch.Generator().manual_seed(case)).to(dtype)
    out = torch.full((T, Hq, D), 3.0, dtype=dtype, device=DEV)
    before = out.clone()
    got = kv4.attn(q.to(DEV), cache, table.to(DEV), i32(lens), D ** -0.5, cu_q=i32(cu),
                   max_q=max(news), causal=causal, out=out)
    assert got.data_ptr() == out.data_ptr()
    check(out, oc.cache_attn(q, host, page, table, lens, D ** -0.5, cu, causal=causal), before)


LONG = [  # lens, queries of each request, heads: runs that end inside a head or a tile
    ([5000], [4], (16, 2)), ([3000, 70, 2600], [1, 1, 1], (6, 2)), ([4100], [200], (4, 2)),
    ([2500, 3000, 64], [300, 1, 64], (4, 1)), ([2300], [1], (96, 1)), ([300, 20], [3, 1], (96, 1)),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", range(len(LONG)))
def test_long_contexts(case, dtype, causal):
    lens, news, (Hq, Hkv) = LONG[case]
    D = (128, 64)[case % 2]
    print(f"long {case} {dtype} causal {causal}", flush=True)
    cache, host, table = filled(lens, 64, Hkv, D, dtype, seed=case)
    cu = [0]
    for m in news:
        cu.append(cu[-1] + m)
    q = torch.randn(cu[-1], Hq, D, generator=torch.Generator().manual_seed(case)).to(dtype)
    out = kv4.attn(q.to(DEV), cache, table.to(DEV), i32(lens), D ** -0.5, cu_q=i32(cu),
                   max_q=max(news), causal=causal)
    check(out, oc.cache_attn(q, host, 64, table, lens, D ** -0.5, cu, causal=causal))


@pytest.mark.parametrize("wide", [False, True])
def test_many_requests(wide):
    """A thousand requests, some without tokens; with a wide table too (runs of units)."""
    g = torch.Generator().manual_seed(12)
    lens = [int(n) for n in torch.randint(0, 90, (1000,), generator=g)]
    cache, host, table = filled(lens, 64, 1, 64, torch.float16, seed=12)
    if wide:
        table = torch.cat((table, torch.full((1000, 60), -1, dtype=torch.int32)), 1)
    q = torch.randn(1000, 2, 64, generator=g).half()
    out = kv4.attn(q.to(DEV), cache, table.to(DEV), i32(lens), 0.125)
    check(out, oc.cache_attn(q, host, 64, table, lens, 0.125))


@pytest.mark.parametrize("dtype", DTYPES)
def test_prompts_among_many_requests(dtype):
    """Three hundred requests, four of them prompts (their tiles are summed up by a kernel of
    its own), and the prompts by themselves."""
    g = torch.Generator().manual_seed(2)
    lens = [int(n) for n in torch.randint(0, 70, (300,), generator=g)]
    news = [min(1, n) for n in lens]
    for b, n in ((5, 400), (6, 130), (170, 700), (299, 257)):
        lens[b], news[b] = n, max(129, n - 100)
    cache, host, table = filled(lens, 64, 1, 64, dtype, seed=2)
    cu = [0]
    for m in news:
        cu.append(cu[-1] + m)
    q = torch.randn(cu[-1], 2, 64, generator=g).to(dtype)
    out = kv4.attn(q.to(DEV), cache, table.to(DEV), i32(lens), 0.125, cu_q=i32(cu),
                   max_q=max(news))
    check(out, oc.cache_attn(q, host, 64, table, lens, 0.125, cu))
    rows = oc.cache_attn(q, host, 64, table, lens, 0.125, cu)
    b = 170
    alone = kv4.attn(q[cu[b]:cu[b + 1]].to(DEV), cache, table[b:b + 1].to(DEV), i32(lens[b:b + 1]),
                     0.125, cu_q=i32([0, news[b]]), max_q=news[b])
    check(alone, {r - cu[b]: rows[r] for r in range(cu[b], cu[b + 1])})


@pytest.mark.parametrize("n", [255, 256, 257])
def test_row_counts_around_the_prompt_kernels(n):
    cache, host, table = filled([700], 64, 1, 128, torch.float16, seed=n)
    q = torch.randn(n, 1, 128, generator=torch.Generator().manual_seed(n)).half()
    out = kv4.attn(q.to(DEV), cache, table.to(DEV), i32([700]), 0.1, cu_q=i32([0, n]), max_q=n)
    check(out, oc.cache_attn(q, host, 64, table, [700], 0.1, [0, n]))


@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
def test_scales(scale):
    lens = [200, 3]
    cache, host, table = filled(lens, 64, 2, 64, torch.float16, seed=5)
    q = torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(5)).half()
    out = kv4.attn(q.to(DEV), cache, table.to(DEV), i32(lens), scale)
    check(out, oc.cache_attn(q, host, 64, table, lens, scale))


@pytest.mark.parametrize("news", [[1, 1, 1], [40, 3, 90]])
def test_bad_pages_narrow_tables_and_hostile_lengths(news):
    lens, page, D = [300, 150, 200], 64, 128
    cache, host, table = filled(lens, page, 2, D, torch.bfloat16, seed=11)
    table[0, 1], table[0, 3], table[1, 0], table[1, 1], table[1, 2] = -1, 10 ** 9, -5, 10 ** 6, -1
    table = table[:, :4].contiguous()          # request 0 has 5 pages
    for lens in ([300, 150, 200], [2 ** 31 - 1, -4, 10 ** 6]):
        cu = [0]
        for m in news:
            cu.append(cu[-1] + m)
        q = torch.randn(cu[-1], 4, D, generator=torch.Generator().manual_seed(3)).bfloat16()
        print(f"bad pages, lens {lens}", flush=True)
        # Tokens past what was stored hold NaN; a causal row past the table sees all of it.
        host_lens = [min(n, 4 * page) for n in lens]
        out = kv4.attn(q.to(DEV), cache, table.to(DEV), i32(lens), 0.1, cu_q=i32(cu),
                       max_q=max(news), causal=False)
        check(out, oc.cache_attn(q, host, page, table, host_lens, 0.1, cu, causal=False))


@pytest.mark.parametrize("cu", [[0, 5, 3, 9], [-4, 2, 100, 200], [7, 7, 7, 7], [9, 0, 0, 9]])
def test_query_bounds_out_of_order_are_safe(cu):
    lens = [100, 70, 64]
    cache, host, table = filled(lens, 64, 1, 64, torch.float16, seed=2)
    q = torch.randn(9, 2, 64, generator=torch.Generator().manual_seed(1)).half()
    out = torch.full((9, 2, 64), 3.0, dtype=torch.float16, device=DEV)
    before = out.clone()
    kv4.attn(q.to(DEV), cache, table.to(DEV), i32(lens), 0.1, cu_q=i32(cu), out=out)
    if cu == [0, 5, 3, 9]:
        return   # rows 3 and 4 belong to two requests: either's result
    check(out, oc.cache_attn(q, host, 64, table, lens, 0.1, cu), before)


def test_queries_past_max_q_are_left():
    lens, cu = [100, 90], [0, 40, 43]
    cache, host, table = filled(lens, 64, 2, 128, torch.float16, seed=4)
    q = torch.randn(43, 2, 128, generator=torch.Generator().manual_seed(1)).half()
    for max_q in (0, 1, 3, 33):
        out = torch.full((43, 2, 128), 3.0, dtype=torch.float16, device=DEV)
        before = out.clone()
        kv4.attn(q.to(DEV), cache, table.to(DEV), i32(lens), 0.1, cu_q=i32(cu), max_q=max_q, out=out)
        check(out, oc.cache_attn(q, host, 64, table, lens, 0.1, cu, max_q=max_q), before)


def test_infinite_and_nan_blocks():
    """A NaN or infinite key block makes the rows that see it NaN and no others; values
    likewise; where no row sees them they change nothing."""
    lens, D = [70, 70], 64
    g = torch.Generator().manual_seed(8)
    for where in ("k", "v"):
        cache, host, table = filled(lens, 64, 1, D, torch.float16, seed=8)
        bad = torch.randn(1, 1, D, generator=g).half()
        bad[0, 0, 40] = math.inf
        ok = torch.randn(1, 1, D, generator=g).half()
        slot = i32([table[0, 1].item() * 64 + 3])      # token 67 of request 0
        kv4.store(cache, (bad if where == "k" else ok).to(DEV), (bad if where == "v" else ok).to(DEV),
                  slot)
        q = torch.randn(10, 2, D, generator=g).half()
        out = kv4.attn(q.to(DEV), cache, table.to(DEV), i32(lens), 0.1, cu_q=i32([0, 5, 10]),
                       max_q=5).cpu()
        nan = out.isnan()
        dims = slice(0, D) if where == "k" else slice(32, D)
        assert nan[2:5, :, dims].all() and not nan[:2].any() and not nan[5:].any()
        if where == "v":
            assert not nan[:, :, :32].any()


@pytest.mark.parametrize("n,news,Hq", [(70, 5, 2), (2600, 6, 4), (300, 150, 2), (2600, 150, 2)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_hidden_tokens_may_hold_anything(n, news, Hq, dtype):
    """Tokens that hold NaN or infinities, late enough that some rows do not see them: single
    and several query rows, tables narrow and wide, prompts in one run and in several."""
    D = 128
    for where in ("k", "v"):
        cache, host, table = filled([n], 64, 1, D, dtype, seed=8)
        bad = torch.randn(2, 1, D, generator=torch.Generator().manual_seed(3)).to(dtype)
        bad[0, 0, 40], bad[1, 0, 100] = math.nan, -math.inf
        ok = torch.randn(2, 1, D, generator=torch.Generator().manual_seed(4)).to(dtype)
        late = [n - 2, n - 4]
        slots = i32([table[0, t // 64].item() * 64 + t % 64 for t in late])
        kv4.store(cache, (bad if where == "k" else ok).to(DEV), (bad if where == "v" else ok).to(DEV),
                  slots)
        host = [t.cpu() for t in cache]
        q = torch.randn(news, Hq, D, generator=torch.Generator().manual_seed(5)).to(dtype)
        wide = torch.cat((table, torch.full((1, 40), -1, dtype=torch.int32)), 1)
        for t in (table, wide):
            out = kv4.attn(q.to(DEV), cache, t.to(DEV), i32([n]), 0.1, cu_q=i32([0, news]),
                           max_q=news)
            rows = oc.cache_attn(q, host, 64, t, [n], 0.1, [0, news])
            assert not out[:news - 4].isnan().any() and out[news - 1].isnan().any()
            check(out, rows)


def test_strided_queries_and_outputs():
    lens, D = [90, 300], 64
    cache, host, table = filled(lens, 64, 2, D, torch.bfloat16, seed=9)
    big = torch.randn(3, 8, 4, D, device=DEV).bfloat16()
    for q in (big[0, :4].transpose(0, 1)[:2], big[1, :2, :, :], big[:2, 1, :, :],
              torch.randn(2, 4, D + 1, device=DEV).bfloat16()[:, :, 1:]):
        hold = torch.full((4, 2, D + 4), 3.0, dtype=torch.bfloat16, device=DEV)
        out = hold.transpose(0, 1)[:, :, :D]
        kv4.attn(q, cache, table.to(DEV), i32(lens), 0.1, out=out)
        check(out, oc.cache_attn(q.cpu(), host, 64, table, lens, 0.1))
        assert hold[:, :, D:].eq(3.0).all()
    q = big[0, :2].clone()
    want = kv4.attn(q, cache, table.to(DEV), i32(lens), 0.1)
    kv4.attn(q, cache, table.to(DEV), i32(lens), 0.1, out=q)   # in place
    assert torch.equal(q, want)


def test_attention_refuses():
    cache, _, table = filled([70], 64, 2, 64, torch.float16, seed=1)
    table = table.to(DEV)
    q = torch.zeros(1, 4, 64, device=DEV).half()
    n = i32([70])
    for kw in (dict(q=q.float()), dict(q=q[:, :3]), dict(q=q[:, :, :32]), dict(q=q.cpu()),
               dict(lens=n.long()), dict(lens=i32([70, 70])), dict(table=table[0]),
               dict(table=table.long()), dict(cu_q=i32([0])), dict(out=q.float()),
               dict(out=q.bfloat16()), dict(out=torch.zeros(1, 1, 64, device=DEV).half().expand(1, 4, 64)),
               dict(scale=math.nan), dict(scale=math.inf)):
        a = dict(q=q, cache=cache, table=table, lens=n, scale=0.1) | kw
        with pytest.raises(RuntimeError):
            kv4.attn(**a)
    x = torch.zeros(2, 4, 64, device=DEV).half()
    with pytest.raises(RuntimeError):   # out partly q
        kv4.attn(x[:1], cache, table, n, 0.1, out=x.view(-1)[64:320].view(1, 4, 64))


def test_caches_without_heads_and_sizes_past_an_int_are_refused():
    q, n, table = torch.zeros(1, 4, 64, device=DEV).half(), i32([1]), i32([[0]])
    none = kv4.new_cache(2, 64, 0, 64)
    for call in (lambda: kv4.attn(q, none, table, n, 0.1), lambda: kv4.load(none, n),
                 lambda: kv4.store(none, q[:, :0], q[:, :0], n),
                 lambda: kv4.plan_pages(n, n, table, n, n, 2 ** 32 + 64, 1)):
        with pytest.raises(RuntimeError):
            call()
    cache = kv4.new_cache(2, 64, 1, 64)
    wide = torch.zeros(1, 2 ** 25, dtype=torch.int32, device=DEV)
    with pytest.raises(RuntimeError):
        kv4.attn(q, cache, wide, n, 0.1)


@pytest.mark.parametrize("news", [1, 20])
@pytest.mark.parametrize("D", [64, 128])
def test_requests_without_keys_read_no_table(D, news):
    """No tokens, no columns in the table, or no pages: rows of zeros."""
    cache = kv4.new_cache(2, 64, 2, D)
    q = torch.randn(2 * news, 8, D, device=DEV).half()
    kw = dict(cu_q=i32([0, news, 2 * news]), max_q=news)
    for c, table, lens in ((cache, torch.empty(2, 0, dtype=torch.int32, device=DEV), [0, 90]),
                           (cache, i32([[1], [-1]]), [0, 9]),
                           (kv4.new_cache(0, 64, 2, D), i32([[1], [0]]), [70, 64])):
        assert kv4.attn(q, c, table, i32(lens), 0.1, **kw).eq(0).all()


def test_no_queries_and_an_empty_cache():
    cache = kv4.new_cache(0, 64, 2, 64)
    table = torch.empty(2, 0, dtype=torch.int32, device=DEV)
    q = torch.randn(2, 4, 64, device=DEV).half()
    assert kv4.attn(q, cache, table, i32([0, 9]), 0.1).eq(0).all()
    assert kv4.attn(q[:0], cache, table[:0], i32([]), 0.1).shape == (0, 4, 64)


# -- together -----------------------------------------------------------------------------

def serve(steps, dtype, D=128, Hq=8, Hkv=2, page=64, seed=0):
    """Prompts and then single tokens through plan, store and attention; returns every
    step's output and what the oracle needs."""
    g = torch.Generator().manual_seed(seed)
    B, W, pages = 3, 6, 14
    cache = kv4.new_cache(pages, page, Hkv, D)
    table = torch.full((B, W), -1, dtype=torch.int32, device=DEV)
    free = torch.randperm(pages, generator=g).int().to(DEV)
    lens, used = i32([0] * B), i32([0])
    done = []
    for news in steps:
        T = sum(news) + 2                       # padded batch
        q, k, v = (torch.randn(T, h, D, generator=g).to(dtype).to(DEV) for h in (Hq, Hkv, Hkv))
        plan = kv4.plan_pages(lens, i32(news), table, free, used, page, T)
        kv4.store(cache, k, v, plan.slots)
        out = torch.full((T, Hq, D), 3.0, dtype=dtype, device=DEV)
        kv4.attn(q, cache, table, plan.lens, D ** -0.5, cu_q=plan.cu_new, max_q=max(news), out=out)
        lens, used = plan.lens, plan.used
        done.append((out, q, [t.cpu() for t in cache], table.cpu(), lens.tolist(),
                     plan.cu_new.tolist()))
        assert plan.missing.item() == 0
    return done


@pytest.mark.parametrize("dtype", DTYPES)
def test_prompts_then_single_tokens(dtype):
    steps = [[100, 1, 37], [1, 1, 1], [1, 64, 1], [1, 0, 1], [5, 1, 2]]
    for out, q, host, table, lens, cu in serve(steps, dtype):
        rows = oc.cache_attn(q.cpu(), host, 64, table, lens, 128 ** -0.5, cu)
        check(out, rows, torch.full_like(out, 3.0))


def test_captured_step_replays():
    """Plan, store and attention in one graph, replayed with new inputs in the same
    buffers and eager work in between, against eager calls."""
    D, Hq, Hkv, page, B = 128, 8, 2, 64, 5
    g = torch.Generator(device=DEV).manual_seed(3)
    lens0 = [100, 63, 0, 700, 128]
    cache, _, table = filled(lens0, page, Hkv, D, torch.float16, seed=3, spare=9)
    table = table.to(DEV)
    taken = set(table[table >= 0].tolist())
    free = i32([p for p in range(cache.k.shape[0]) if p not in taken])
    lens, new, used = i32(lens0), i32([1] * B), i32([0])
    q, k, v = (torch.randn(B, h, D, device=DEV, generator=g).half() for h in (Hq, Hkv, Hkv))
    out = torch.zeros(B, Hq, D, device=DEV).half()

    def step():
        plan = kv4.plan_pages(lens, new, table, free, used, page, B)
        kv4.store(cache, k, v, plan.slots)
        kv4.attn(q, cache, table, plan.lens, 0.1, cu_q=plan.cu_new, max_q=1, out=out)
        return plan

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(4):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, device=DEV, generator=g).half())
        graph.replay()
        got = out.clone()
        torch.randn(1 << 18, device=DEV).sum().item()
        out.zero_()
        plan = step()
        assert torch.equal(out, got), f"replay {i}"
        lens.copy_(plan.lens)
        used.copy_(plan.used)
        torch.cuda.synchronize()


def test_captured_prompts_replay():
    """A batch of prompts and single tokens, captured and replayed with new queries."""
    lens, cu = [2500, 40, 700], [0, 150, 151, 300]
    cache, _, table = filled(lens, 64, 2, 128, torch.bfloat16, seed=4)
    table, n, cu = table.to(DEV), i32(lens), i32(cu)
    q = torch.randn(300, 8, 128, device=DEV).bfloat16()
    out = torch.zeros_like(q)
    call = lambda o=None: kv4.attn(q, cache, table, n, 0.1, cu_q=cu, max_q=150, out=o)  # noqa: E731
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call(out)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out)
    for i in range(4):
        q.copy_(torch.randn(q.shape, device=DEV).bfloat16())
        out.zero_()
        graph.replay()
        torch.randn(1 << 18, device=DEV).sum().item()
        assert torch.equal(out, call()), f"replay {i}"
        torch.cuda.synchronize()


def test_two_streams_at_once():
    lens = [3000, 500, 1]
    cache, host, table = filled(lens, 128, 2, 64, torch.float16, seed=6)
    table, n = table.to(DEV), i32(lens)
    qs = [torch.randn(3, 8, 64, device=DEV).half() for _ in range(6)]
    want = [kv4.attn(q, cache, table, n, 0.1) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for i, q in enumerate(qs):
        with torch.cuda.stream(streams[i % 3]):
            got.append(kv4.attn(q, cache, table, n, 0.1))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_offsets_past_32_bits():
    """Rows whose codes start past 2^32 bytes."""
    page, D, Hkv = 256, 128, 8
    pages = 2 ** 32 // (Hkv * page * D // 2) + 3
    cache = kv4.new_cache(pages, page, Hkv, D)
    k, v = (torch.randn(300, Hkv, D, device=DEV).half() for _ in range(2))
    at = torch.arange(300, dtype=torch.int32, device=DEV)
    table = i32([[pages - 1, pages - 2]])
    slots = table[0, (at // page).long()] * page + at % page
    kv4.store(cache, k, v, slots)
    want = [oc.dequantise(*oc.quantise(x.cpu())) for x in (k, v)]
    for got, ref in zip(kv4.load(cache, slots), want):
        assert torch.equal(got.cpu().double(), ref)
    q = torch.randn(300, 8, D).half()
    small = kv4.new_cache(2, page, Hkv, D)
    kv4.store(small, k, v, at)
    for cu, m, n in ((None, 1, 1), (i32([0, 300]), 300, 300)):
        x = q[:n].to(DEV)
        far = kv4.attn(x, cache, table, i32([300]), 0.1, cu_q=cu, max_q=m)
        near = kv4.attn(x, small, i32([[0, 1]]), i32([300]), 0.1, cu_q=cu, max_q=m)
        assert torch.equal(far, near)


def as_fp16(q, host, page, table, n, scale):
    """{row: (o, tolerance)} of one request's last tokens, its values as fp16 holds them:
    infinities past 65504, multiples of 2^-24 below the smallest normal number."""
    T, Hq, D = q.shape
    at = [(table[0, t // page].item(), t % page) for t in range(n)]
    k, v = (torch.stack([oc.dequantise(*oc.read_cache(*host[i:i + 2], p, t)) for p, t in at])
            .half().double() for i in (0, 2))
    G = Hq // k.shape[1]
    hide = torch.arange(n)[None] > torch.arange(T)[:, None] + n - T
    got = [oc.softmax_rows(q[:, h], k[:, h // G], v[:, h // G], scale, hide) for h in range(Hq)]
    vmax = v.nan_to_num(0.0, 0.0, 0.0).abs().max().item()
    tols = [oc.tolerance(o, s.nan_to_num(0.0, 0.0, 0.0), z, q.dtype, D, n, vmax) for o, s, z in got]
    return {r: (torch.stack([g[0][r] for g in got]), torch.stack([t[r] for t in tols]))
            for r in range(T)}


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("n,news", [(90, 6), (2600, 6), (300, 200), (2600, 150)])
@pytest.mark.parametrize("what", ["large values", "small keys"])
def test_hidden_tokens_leave_bf16_rows_read_as_fp16(what, n, news, wide):
    """fp16 queries over a cache of bf16 rows that fp16 does not hold: a row's result is that of
    the rounded values, whether a token it does not see holds NaN or not."""
    D, Hq, page = 128, 4, 64
    print(f"{what} n {n} news {news} wide {wide}", flush=True)
    g = torch.Generator().manual_seed(n + news)
    k = torch.randn(n, 1, D, generator=g)
    v = torch.randn(n, 1, D, generator=g)
    q = torch.randn(news, Hq, D, generator=g).half()
    scale = 0.1
    if what == "large values":
        v[7, 0, 3] = 1e5        # the nearest code stands for 98304
    else:
        k, q, scale = k * 2.0 ** -26, q * 10000, 1500.0   # scores of some units
    pages = -(-n // page)
    perm = torch.randperm(pages, generator=g).int()
    table = perm[None]
    if wide:
        table = torch.cat((table, torch.full((1, 40), -1, dtype=torch.int32)), 1)
    t = torch.arange(n)
    slots = (perm[t // page] * page + t % page).int()
    outs = []
    for hidden in (1.0, math.nan):
        v[n - 1, 0, 64:] = hidden
        cache = kv4.new_cache(pages, page, 1, D)
        kv4.store(cache, k.bfloat16().to(DEV), v.bfloat16().to(DEV), slots.to(DEV))
        out = kv4.attn(q.to(DEV), cache, table.to(DEV), i32([n]), scale, cu_q=i32([0, news]),
                       max_q=news).cpu()
        rows = as_fp16(q, [x.cpu() for x in cache], page, table, n, scale)
        for r in range(news - 1):     # (the last row sees the token)
            o, tol = rows[r]
            inf = o.isinf()
            assert torch.equal(out[r].double()[inf], o[inf]), (r, hidden)
            err = ((out[r].double() - o).abs() / tol)[~inf].max().item()
            assert err <= 1.0, (r, hidden, err)
        assert rows[0][0].isinf().any() == (what == "large values")
        outs.append(out[:-1])
    assert torch.equal(outs[0].isfinite(), outs[1].isfinite())


@pytest.mark.parametrize("B,Hq,Hkv,W", [(32, 16, 4, 64), (64, 2, 2, 64), (32, 16, 4, 33), (40, 64, 1, 40)])
def test_single_tokens_with_room_for_more(B, Hq, Hkv, W):
    """Without cu_q a request has one query, whatever max_q allows for: tables on either side
    of the short form's limits."""
    g = torch.Generator().manual_seed(B + W)
    lens = [int(n) for n in torch.randint(1, 300, (B,), generator=g)]
    cache, host, table = filled(lens, 64, Hkv, 64, torch.float16, seed=B)
    table = torch.cat((table, torch.full((B, W), -1, dtype=torch.int32)), 1)[:, :W].contiguous()
    q = torch.randn(B, Hq, 64, generator=g).half()
    want = kv4.attn(q.to(DEV), cache, table.to(DEV), i32(lens), 0.125)
    check(want, oc.cache_attn(q, host, 64, table, lens, 0.125))
    for max_q in (2, 17, B, 1000, -1):
        got = kv4.attn(q.to(DEV), cache, table.to(DEV), i32(lens), 0.125, max_q=max_q)
        assert torch.equal(got, want), max_q


@pytest.mark.parametrize("n,news", [(200, 1), (2300, 2), (300, 200)])
@pytest.mark.parametrize("scale", [0.0, 1e-37, -1e-37])
def test_small_scales_of_large_bf16_scores(scale, n, news):
    """Products up to 1e38: a scale of 0 weighs every key alike, one of 1e-37 gives scores of
    some units."""
    cache, host, table = filled([n], 64, 1, 64, torch.bfloat16, seed=n, gain=2.0 ** 60)
    q = torch.randn(news, 2, 64, generator=torch.Generator().manual_seed(n))
    q = (q * 2.0 ** 60).bfloat16()
    out = kv4.attn(q.to(DEV), cache, table.to(DEV), i32([n]), scale, cu_q=i32([0, news]), max_q=news)
    check(out, oc.cache_attn(q, host, 64, table, [n], scale, [0, news]))


def test_rows_of_two_requests_are_one_of_theirs():
    """Bounds [0, 5, 3, 9]: rows 3 and 4 belong to requests 0 and 2, the others to one."""
    lens, cu = [100, 70, 64], [0, 5, 3, 9]
    cache, host, table = filled(lens, 64, 1, 64, torch.float16, seed=2)
    q = torch.randn(9, 2, 64, generator=torch.Generator().manual_seed(1)).half()
    out = kv4.attn(q.to(DEV), cache, table.to(DEV), i32(lens), 0.1, cu_q=i32(cu))
    first = oc.cache_attn(q, host, 64, table[:1], lens[:1], 0.1, [0, 5])
    last = oc.cache_attn(q, host, 64, table[2:], lens[2:], 0.1, [3, 9])
    check(out, {r: first[r] for r in range(3)} | {r: last[r] for r in range(5, 9)})
    for r in (3, 4):   # (four dims at a time may come from either)
        off = [(out[r].double().cpu() - o).abs() <= tol for o, tol in (first[r], last[r])]
        assert (off[0] | off[1]).all(), r
