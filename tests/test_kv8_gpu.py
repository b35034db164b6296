"""The 8-bit cache on the GPU against the CPU oracle in 64 bits: storing and reading, attention
over it, weights of its blocks, eviction, and a run of them together."""

import math

import pytest
import torch

from gfx906_amd import kv8
from oracle import serving as sv

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float16, torch.bfloat16]


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def offsets(news):
    cu = [0]
    for m in news:
        cu.append(cu[-1] + m)
    return cu


def tables(lens, page, seed, spare=2, wider=1):
    """(table as lists, pages of the cache): shuffled pages, -1 behind the last."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-max(0, n) // page) for n in lens]
    W = max(max(need, default=0), 1) + wider
    phys = torch.randperm(sum(need) + spare, generator=g).tolist()
    out, at = [], 0
    for n in need:
        out.append(phys[at:at + n] + [-1] * (W - n))
        at += n
    return out, sum(need) + spare


def dirty_cache(pages, page, H, D):
    """A cache whose every byte is a NaN and whose scales are nonsense: nothing may read it."""
    cache = kv8.new_cache(pages, page, H, D)
    for t in (cache.k, cache.v):
        t.fill_(0xff)
    for t in (cache.k_scale, cache.v_scale):
        t.fill_(math.nan)
    return cache


def same(cache, want, tables_, lens):
    """The tokens that requests hold are exactly what the oracle says."""
    got = [sv.decode(cache.k.cpu(), cache.k_scale.cpu(), False),
           sv.decode(cache.v.cpu(), cache.v_scale.cpu(), True)]
    for b, n in enumerate(lens):
        for t in range(n):
            page = tables_[b][t // cache.page] if t // cache.page < len(tables_[b]) else -1
            if not 0 <= page < len(cache.k):
                continue
            for g, x in zip(got, want.x):
                a, e = g[page, :, t % cache.page], x[page, :, t % cache.page]
                assert torch.equal(a.nan_to_num(9e9), e.nan_to_num(9e9)), (b, t)


# -- storing and reading ------------------------------------------------------------------

STORES = [  # lens before, rows of each request in turn, page
    ([0], [[1]], 64), ([0, 5, 63], [[1, 1, 1]] * 3, 64), ([0, 0], [[100, 3], [30, 130]], 128),
    ([10, 64, 120, 0], [[200, 0, 9, 64], [1, 1, 1, 1], [5, 63, 64, 65]], 256),
    ([7] * 70, [[1] * 70] * 2, 64),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,D", [(1, 64), (3, 128)])
@pytest.mark.parametrize("case", range(len(STORES)))
def test_store(case, H, D, dtype):
    lens, steps, page = STORES[case]
    print(f"store {case} H{H} D{D} {dtype}", flush=True)
    g = torch.Generator().manual_seed(case)
    final = [n + sum(s[b] for s in steps) for b, n in enumerate(lens)]
    table, pages = tables(final, page, case)
    cache, want = dirty_cache(pages, page, H, D), sv.Cache(pages, page, H, D)
    weights = kv8.new_weights(cache)
    steps = [lens] + steps       # the tokens that are there come in one call
    lens = [0] * len(lens)
    for step, news in enumerate(steps):
        lens = [n + m for n, m in zip(lens, news)]
        cu = offsets(news)
        # sizes over many powers of two, so that scales grow
        x = torch.randn(2, cu[-1], H, D, generator=g) * torch.exp2(
            torch.randint(-14, 8, (2, cu[-1], H, 1), generator=g).float())
        if cu[-1] > 1:
            x[0, 0, 0, :4] = torch.tensor([math.nan, math.inf, -math.inf, 1.0])
            x[1, -1, -1, :3] = torch.tensor([65504.0, -60000.0, 2.0 ** -24])
            if dtype == torch.bfloat16:
                x[1, 0, 0, 5] = -3e38
        k, v = x.to(dtype)
        weights.fill_(7.0)
        want.begun[:] = False
        one = all(m == 1 for m in news) and case % 2
        kv8.store(cache, k.to(DEV), v.to(DEV), i32(table), i32(lens), None if one else i32(cu),
                  weights if step else None)
        want.store(k, v, table, lens, cu)
        same(cache, want, table, lens)
        if step:
            begun = want.begun[:, None].expand(-1, H, -1)
            assert torch.equal(weights.cpu() == 0, begun) and weights.cpu()[~begun].eq(7).all()
    e = torch.stack(want.e)
    for b, n in enumerate(lens):     # scales are the least that hold the tokens so far
        for t in range(0, n, 64):
            at = table[b][t // page], slice(None), t % page // 64
            for scale, x in ((cache.k_scale, e[0]), (cache.v_scale, e[1])):
                assert torch.equal(scale.cpu()[at], torch.exp2(x[at].float()))
    slots = [table[b][t // page] * page + t % page for b, n in enumerate(lens) for t in range(n)]
    for got, x in zip(kv8.load(cache, i32(slots + [-1, pages * page, 2 ** 31 - 1]), dtype), want.x):
        rows = torch.stack([x[s // page, :, s % page] for s in slots])
        assert torch.equal(got[:len(slots)].double().cpu().nan_to_num(9e9), rows.nan_to_num(9e9))
        assert got[len(slots):].eq(0).all()


def test_every_code_is_held_exactly_in_both_types():
    """All codes at the ends of the scales' range, read as fp16 and bf16."""
    cache = kv8.new_cache(2, 64, 1, 64)
    codes = torch.arange(256, dtype=torch.uint8, device=DEV)
    cache.k.view(-1)[:256] = codes
    cache.v.view(-1)[:256] = codes
    for exp in (-15, 0, 7):
        cache.k_scale.fill_(2.0 ** exp)
        cache.v_scale.fill_(2.0 ** exp)
        want = (sv.decode(cache.k.cpu(), cache.k_scale.cpu(), False),
                sv.decode(cache.v.cpu(), cache.v_scale.cpu(), True))
        for dtype in DTYPES:
            got = kv8.load(cache, torch.arange(64, device=DEV).int(), dtype)
            for g, w in zip(got, want):
                assert torch.equal(g.double().cpu()[:, 0].nan_to_num(9e9), w[0, 0].nan_to_num(9e9))


def test_store_passes_over_rows_without_a_place():
    """Pages that lack, tables that end, more rows than tokens, offsets past the rows."""
    page, H, D = 64, 2, 64
    x = torch.randn(2, 300, H, D).half()
    table = [[0, -1, 2], [3, 99, 4], [5, 6, 7], [8, 9, 10]]
    lens, cu = [192, 130, 5, 500], [-5, 150, 200, 210, 400]
    cache = kv8.new_cache(11, page, H, D)
    untouched = sv.Cache(11, page, H, D)
    untouched.store(x[0], x[1], table, lens, cu)
    kv8.store(cache, x[0].to(DEV), x[1].to(DEV), i32(table), i32(lens), i32(cu))
    got = sv.decode(cache.k.cpu(), cache.k_scale.cpu(), False)
    assert torch.equal(got, untouched.x[0])       # rows not stored left the cache as it was
    got = sv.decode(cache.v.cpu(), cache.v_scale.cpu(), True)
    assert torch.equal(got, untouched.x[1])


def test_store_reads_strided_rows_and_wide_tables():
    T, H, D, page = 70, 2, 64, 64
    big = torch.randn(T, 3, 3, 96, device=DEV).half()
    k, v = big[:, 0, :H, :D], big[:, 1, 1:, 3:3 + D]   # v: not 16-byte aligned, copied
    wide = torch.full((1, 9), -7, dtype=torch.int32, device=DEV)
    wide[0, :2] = i32([1, 0])
    cache, want = kv8.new_cache(2, page, H, D), sv.Cache(2, page, H, D)
    kv8.store(cache, k, v, wide[:, :2], i32([T]), i32([0, T]))
    want.store(k.cpu(), v.cpu(), [[1, 0]], [T], [0, T])
    same(cache, want, [[1, 0]], [T])
    kv8.store(cache, k[:0], v[:0], wide[:, :2], i32([T]), i32([0, 0]))
    kv8.store(cache, k[:0], v[:0], wide[:0], i32([]), i32([0]))
    same(cache, want, [[1, 0]], [T])


def test_shorter_again():
    """Drafted tokens that were refused: the next ones take their places."""
    H, D = 1, 128
    x = torch.randn(2, 100, H, D).bfloat16()
    x[:, 60:70] *= 30
    cache, want, table = kv8.new_cache(3, 64, H, D), sv.Cache(3, 64, H, D), [[2, 1]]
    for lens, a, b in ((62, 0, 62), (70, 62, 70), (64, 70, 72), (66, 72, 74), (92, 74, 100)):
        n = b - a
        kv8.store(cache, *x[:, a:b].to(DEV), i32(table), i32([lens]), i32([0, n]))
        want.store(*x[:, a:b], table, [lens], [0, n])
        same(cache, want, table, [lens])


def test_store_and_load_refuse():
    cache = kv8.new_cache(2, 64, 2, 64)
    x, t, n, cu = torch.zeros(3, 2, 64, device=DEV).half(), i32([[0]]), i32([3]), i32([0, 3])
    w = kv8.new_weights(cache)
    ok = dict(cache=cache, k=x, v=x, table=t, lens=n, cu_new=cu, weights=w)
    for bad in (dict(k=x.float(), v=x.float()), dict(v=x.bfloat16()), dict(v=x[:2]),
                dict(k=x[:, :1], v=x[:, :1]), dict(k=x.cpu()), dict(cu_new=None),
                dict(cu_new=cu.long()), dict(cu_new=i32([0])), dict(lens=i32([3, 3])),
                dict(table=t[0]), dict(table=t.long()), dict(table=t.cpu()), dict(weights=w[:1]),
                dict(weights=w.half()), dict(weights=w.cpu()),
                dict(cache=cache._replace(k=cache.k.int())), dict(cache=cache._replace(v=cache.v[:1])),
                dict(cache=cache._replace(k_scale=cache.k_scale[:, :1])),
                dict(cache=cache._replace(v=cache.v.transpose(3, 4).contiguous().transpose(3, 4))),
                dict(cache=kv8.Cache(*(y.cpu() for y in cache)))):
        with pytest.raises(RuntimeError):
            kv8.store(**(ok | bad))
    for bad in (n.long(), n.cpu(), n[None]):
        with pytest.raises(RuntimeError):
            kv8.load(cache, bad)
    with pytest.raises(RuntimeError):
        kv8.load(cache, n, torch.float32)


def filled(lens, page, Hkv, D, dtype, seed, gain=2.0):
    """(cache on the GPU, what it holds, table) of random rows; the rest holds NaN."""
    g = torch.Generator().manual_seed(seed)
    table, pages = tables(lens, page, seed)
    cache, held = dirty_cache(pages, page, Hkv, D), sv.Cache(pages, page, Hkv, D)
    cu = offsets([max(0, n) for n in lens])
    k = (torch.randn(cu[-1], Hkv, D, generator=g) * gain).to(dtype)
    v = torch.randn(cu[-1], Hkv, D, generator=g).to(dtype)
    kv8.store(cache, k.to(DEV), v.to(DEV), i32(table), i32(lens), i32(cu))
    # (as the GPU holds it: the stores have tests of their own)
    held.x = [sv.decode(cache.k.cpu(), cache.k_scale.cpu(), False),
              sv.decode(cache.v.cpu(), cache.v_scale.cpu(), True)]
    return cache, held, table


# -- attention ----------------------------------------------------------------------------

def check(out, lse, rows, untouched=None):
    """Computed rows within the bound, the others as they were."""
    out = out.double().cpu()
    lse = None if lse is None else lse.double().cpu()
    worst = far = 0.0
    for r in range(out.shape[0]):
        if r not in rows:
            if untouched is not None:
                assert torch.equal(out[r], untouched[r].double().cpu()), f"row {r} written"
            continue
        o, tol, l, ltol = rows[r]
        nan = o.isnan()
        assert torch.equal(out[r].isnan(), nan), f"row {r}: NaN"
        err = ((out[r] - o).abs() / tol)[~nan]
        if err.numel():
            worst = max(worst, err.max().item())
            assert worst <= 1.0, f"row {r}: {worst} of the bound"
        if lse is not None:
            fin = torch.isfinite(l)
            assert torch.equal(lse[r][~fin].nan_to_num(9e9, 8e9, 7e9), l[~fin].nan_to_num(9e9, 8e9, 7e9))
            if fin.any():
                far = max(far, ((lse[r] - l).abs() / ltol)[fin].max().item())
                assert far <= 1.0, f"row {r}: lse {far} of the bound"
    print(f"  worst {worst:.3f} of the bound, lse {far:.3f}", flush=True)


HEADS = [(1, 1), (8, 2), (5, 5), (16, 1), (24, 2), (40, 1), (6, 2)]
DECODES = [[1], [0, 5], [63, 64, 65], [0, 1, 130, 700, 33], [2050, 1, 300]]


@pytest.mark.parametrize("lse", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,page", [(64, 64), (128, 64), (128, 128), (64, 256), (128, 256)])
@pytest.mark.parametrize("lens", DECODES)
def test_single_tokens(lens, D, page, dtype, lse):
    Hq, Hkv = HEADS[(len(lens) + D // 64 + page // 64) % len(HEADS)]
    print(f"decode lens {lens} heads {Hq}/{Hkv} D{D} page {page} {dtype}", flush=True)
    cache, held, table = filled(lens, page, Hkv, D, dtype, seed=sum(lens))
    q = torch.randn(len(lens), Hq, D, generator=torch.Generator().manual_seed(7)).to(dtype)
    out = kv8.attn(q.to(DEV), cache, i32(table), i32(lens), D ** -0.5, lse=lse)
    check(*(out if lse else (out, None)), sv.attention(q, held, table, lens, D ** -0.5))


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
    D, page = (64, 128)[(case + Hq // 3) % 2], (64, 128, 256)[(case + Hq) % 3]
    print(f"chunks {case} heads {heads} D{D} page {page} {dtype} causal {causal}", flush=True)
    cache, held, table = filled(lens, page, Hkv, D, dtype, seed=case)
    cu = offsets(news)
    T = cu[-1] + behind
    q = torch.randn(T, Hq, D, generator=torch.Generator().manual_seed(case)).to(dtype)
    out = torch.full((T, Hq, D), 3.0, dtype=dtype, device=DEV)
    before = out.clone()
    got, lse = kv8.attn(q.to(DEV), cache, i32(table), i32(lens), D ** -0.5, cu_q=i32(cu),
                        max_q=max(news), causal=causal, out=out, lse=True)
    assert got.data_ptr() == out.data_ptr()
    rows = sv.attention(q, held, table, lens, D ** -0.5, cu, causal=causal)
    check(out, lse, rows, before)
    plain = kv8.attn(q.to(DEV), cache, i32(table), i32(lens), D ** -0.5, cu_q=i32(cu),
                     max_q=max(news), causal=causal)
    keep = sorted(rows)
    assert torch.equal(plain[keep], out[keep])     # with or without lse, the same result


LONG = [  # lens, queries of each request, heads: runs that end inside a head or a tile
    ([5000], [4], (16, 2)), ([3000, 70, 2600], [1, 1, 1], (6, 2)), ([4100], [200], (4, 2)),
    ([2500, 3000, 64], [300, 1, 64], (4, 1)), ([2300], [1], (96, 1)), ([300, 20], [3, 1], (96, 1)),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("case", range(len(LONG)))
def test_long_contexts(case, D, dtype, causal):
    lens, news, (Hq, Hkv) = LONG[case]
    print(f"long {case} D{D} {dtype} causal {causal}", flush=True)
    cache, held, table = filled(lens, 64, Hkv, D, dtype, seed=case)
    cu = offsets(news)
    q = torch.randn(cu[-1], Hq, D, generator=torch.Generator().manual_seed(case)).to(dtype)
    out, lse = kv8.attn(q.to(DEV), cache, i32(table), i32(lens), D ** -0.5, cu_q=i32(cu),
                        max_q=max(news), causal=causal, lse=True)
    check(out, lse, sv.attention(q, held, table, lens, D ** -0.5, cu, causal=causal))


@pytest.mark.parametrize("wide", [False, True])
def test_many_requests(wide):
    """A thousand requests, some without tokens; with a wide table too (runs of units)."""
    g = torch.Generator().manual_seed(12)
    lens = [int(n) for n in torch.randint(0, 90, (1000,), generator=g)]
    cache, held, table = filled(lens, 64, 1, 64, torch.float16, seed=12)
    if wide:
        table = [row + [-1] * 60 for row in table]
    q = torch.randn(1000, 2, 64, generator=g).half()
    out, lse = kv8.attn(q.to(DEV), cache, i32(table), i32(lens), 0.125, lse=True)
    check(out, lse, sv.attention(q, held, table, lens, 0.125))


@pytest.mark.parametrize("longest", [700, 320])
def test_prompts_among_many_requests(longest):
    """Three hundred requests, four of them prompts (their tiles are summed up by a kernel of
    its own), long enough for large tiles or not."""
    g = torch.Generator().manual_seed(2)
    lens = [int(n) for n in torch.randint(0, 70, (300,), generator=g)]
    news = [min(1, n) for n in lens]
    for b, n in ((5, 300), (6, 130), (170, longest), (299, 257)):
        lens[b], news[b] = n, max(129, n - 100)
    cache, held, table = filled(lens, 64, 1, 64, torch.bfloat16, seed=2)
    cu = offsets(news)
    q = torch.randn(cu[-1], 2, 64, generator=g).bfloat16()
    out, lse = kv8.attn(q.to(DEV), cache, i32(table), i32(lens), 0.125, cu_q=i32(cu),
                        max_q=max(news), lse=True)
    check(out, lse, sv.attention(q, held, table, lens, 0.125, cu))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("news", [[5, 1], [150, 40], [230, 130]])
def test_nan_reaches_only_the_rows_that_see_it(news, D, dtype):
    """NaN and infinities among the keys and values of tokens that some rows do not see."""
    lens, page, H = [230, 130], 64, 2
    table, pages = tables(lens, page, 4)
    cache, held = dirty_cache(pages, page, H, D), sv.Cache(pages, page, H, D)
    g = torch.Generator().manual_seed(5)
    k, v = torch.randn(2, sum(lens), H, D, generator=g).to(dtype)
    v[lens[0] - 2, 0, 5], v[lens[0] - 3, 1, D - 1] = math.nan, math.inf
    v[10, 0, 7] = -math.inf                       # a token that all rows see
    v[lens[0] + 100, 1, 3] = math.nan
    k[lens[0] - 1, 1, 0] = math.nan
    cu = offsets(lens)
    kv8.store(cache, k.to(DEV), v.to(DEV), i32(table), i32(lens), i32(cu))
    held.store(k, v, table, lens, cu)
    cu = offsets(news)
    heads = 6 if news[0] > 200 else 4      # (large tiles of rows, or not)
    q = torch.randn(cu[-1], heads, D, generator=g).to(dtype)
    for causal in (True, False):
        out, lse = kv8.attn(q.to(DEV), cache, i32(table), i32(lens), 0.1, cu_q=i32(cu),
                            max_q=max(news), causal=causal, lse=True)
        rows = sv.attention(q, held, table, lens, 0.1, cu, causal=causal)
        assert any(r[0].isnan().any() for r in rows.values())
        check(out, lse, rows)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("wide", [0, 60])
def test_lost_pages_and_scores_that_vanish(wide, dtype):
    """Pages that lack, scores of -inf, far scores, and a negative scale."""
    lens, news, page, H, D = [300, 64, 500], [4, 1, 290], 64, 2, 64
    cache, held, table = filled(lens, page, H, D, dtype, seed=8, gain=30.0)
    table[0][1], table[1][0], table[2][3] = -1, 99, -7
    table = [row + [-1] * wide for row in table]
    cu = offsets(news)
    q = (torch.randn(cu[-1], 4, D, generator=torch.Generator().manual_seed(1)) * 5).to(dtype)
    for scale in (0.125, -0.3, 8.0):
        out, lse = kv8.attn(q.to(DEV), cache, i32(table), i32(lens), scale, cu_q=i32(cu),
                            max_q=290, lse=True)
        check(out, lse, sv.attention(q, held, table, lens, scale, cu))


def test_fewer_queries_than_there_are_in_place_and_strided():
    lens, news, page, H, D = [200, 90], [150, 7], 64, 1, 128
    cache, held, table = filled(lens, page, H, D, torch.float16, seed=6)
    cu = offsets(news)
    buf = torch.randn(cu[-1], 3, 2 * D, device=DEV).half()
    q = buf[:, :2, :D]
    rows = sv.attention(q.cpu(), held, table, lens, 0.1, cu, 9)
    out = torch.zeros(cu[-1], 5, D, device=DEV).half()
    kv8.attn(q, cache, i32(table), i32(lens), 0.1, cu_q=i32(cu), max_q=9, out=out[:, 1:3])
    check(out[:, 1:3], None, rows, torch.zeros(cu[-1], 2, D))
    assert out[:, 0].eq(0).all() and out[:, 3:].eq(0).all()
    want = kv8.attn(q, cache, i32(table), i32(lens), 0.1, cu_q=i32(cu))
    q = q.contiguous()
    assert kv8.attn(q, cache, i32(table), i32(lens), 0.1, cu_q=i32(cu), out=q).data_ptr() == q.data_ptr()
    assert torch.equal(q, want)


def test_attn_refuses():
    cache, _, table = filled([70], 64, 2, 64, torch.float16, seed=1)
    q = torch.zeros(1, 4, 64, device=DEV).half()
    ok = dict(q=q, cache=cache, table=i32(table), lens=i32([70]), scale=0.1)
    for bad in (dict(q=q.float()), dict(q=q[:, :3]), dict(q=q.cpu()), dict(q=q[..., :32]),
                dict(scale=math.inf), dict(scale=math.nan), dict(lens=i32([70, 1])),
                dict(cu_q=i32([0])), dict(table=i32(table)[0]), dict(lens=i32([70]).long()),
                dict(out=q[:, :2]), dict(out=q.float()),
                dict(out=cache.k.view(-1)[:512].view(torch.float16).view(1, 4, 64)),
                dict(out=torch.zeros(1, 4, 128, device=DEV).half()[..., ::2]),
                dict(cache=cache._replace(v=cache.k))):
        with pytest.raises(RuntimeError):
            kv8.attn(**(ok | bad))


def test_out_beside_q_in_one_buffer():
    """Results may lie in another part of q's projection; a part of q is refused."""
    cache, _, table = filled([70, 9], 64, 2, 64, torch.float16, seed=1)
    x = torch.randn(2, 12, 64, device=DEV).half()
    args = (cache, i32(table), i32([70, 9]), 0.1)
    want = kv8.attn(x[:, :4].contiguous(), *args)
    assert torch.equal(kv8.attn(x[:, :4], *args, out=x[:, 8:]), want)
    assert torch.equal(x[:, 8:], want)
    for out in (x[:, 1:5], x[:, 3:7], x.view(-1, 64)[:16].view(2, 8, 64)[:, :4]):
        with pytest.raises(RuntimeError, match="overlap"):
            kv8.attn(x[:, :4], *args, out=out)
    assert kv8.attn(x[:, :4], *args, out=x[:, :4]).data_ptr() == x.data_ptr()
    assert torch.equal(x[:, :4], want)


# -- weights of blocks --------------------------------------------------------------------

def weighed(got, want, tol, table, lens, page):
    """Blocks that hold tokens within the bound, the others as they were."""
    got = got.double().cpu()
    assert torch.equal(got.isnan(), want.isnan())
    worst = ((got - want).abs() / tol)[~want.isnan()].max().item()
    print(f"  worst {worst:.3f} of the bound", flush=True)
    assert worst <= 1.0


WEIGHS = [  # lens, queries of each request
    ([1], [1]), ([0, 5], [1, 1]), ([63, 64, 65], [1, 1, 1]), ([130, 77, 300], [130, 1, 45]),
    ([500, 0, 20, 9], [3, 0, 20, 0]), ([5, 200], [9, 2]), ([700], [300]), ([1030, 4], [1, 4]),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,page", [(64, 64), (128, 128), (128, 256)])
@pytest.mark.parametrize("case", range(len(WEIGHS)))
def test_weigh(case, D, page, dtype, causal):
    lens, news = WEIGHS[case]
    Hq, Hkv = HEADS[(case + D // 64 + page // 64) % len(HEADS)]
    print(f"weigh {case} heads {Hq}/{Hkv} D{D} page {page} {dtype} causal {causal}", flush=True)
    cache, held, table = filled(lens, page, Hkv, D, dtype, seed=case)
    cu = offsets(news)
    g = torch.Generator().manual_seed(case)
    q = torch.randn(cu[-1] + 1, Hq, D, generator=g).to(dtype)
    # any lse will do, the call takes what it is given
    lse = torch.randn(cu[-1] + 1, Hq, generator=g) + 8
    lse[0, 0] = -math.inf
    weights = torch.rand(len(cache.k), Hkv, page // 64, generator=g)
    got = weights.to(DEV)
    single = all(m == 1 for m in news)
    kv8.weigh(got, (q[:-1] if single else q).to(DEV), (lse[:-1] if single else lse).to(DEV), cache,
              i32(table), i32(lens), D ** -0.5, cu_q=None if single else i32(cu), max_q=max(news),
              causal=causal)
    want, tol = sv.weigh(weights, q, lse, held, table, lens, D ** -0.5, cu, causal=causal)
    weighed(got, want, tol, table, lens, page)
    again = weights.to(DEV)
    kv8.weigh(again, q.to(DEV), lse.to(DEV), cache, i32(table), i32(lens), D ** -0.5, cu_q=i32(cu),
              max_q=max(news), causal=causal)
    assert torch.equal(got, again) or single    # the order of sums is set by sizes


def test_weigh_with_lost_pages_negative_scale_fewer_queries_and_nan():
    cache, held, table = filled([300, 130], 64, 2, 64, torch.float16, seed=3)
    table[0][1], table[1][0] = -1, 99
    q = torch.randn(20, 4, 64).half()
    lse = torch.full((20, 4), 5.0)
    lse[3, 1] = math.nan            # reaches every block that the row sees
    lse[4, 2] = math.inf
    weights = torch.rand(len(cache.k), 2, 1)
    for cu, max_q in (([0, 2, 20], 7), ([0, 18, 20], None)):
        got = weights.to(DEV)
        kv8.weigh(got, q.to(DEV), lse.to(DEV), cache, i32(table), i32([300, 130]), -0.2,
                  cu_q=i32(cu), max_q=max_q)
        want, tol = sv.weigh(weights, q, lse, held, table, [300, 130], -0.2, cu, max_q)
        weighed(got, want, tol, table, [300, 130], 64)


@pytest.mark.parametrize("news", [1, 30])
def test_rows_that_see_nothing_weigh_nothing_whatever_the_keys_hold(news):
    """An lse of -inf counts for the row, also where keys hold NaN."""
    H, D, n = 1, 64, 100
    k = torch.randn(n, H, D).half()
    k[40] = math.nan
    cache, table = kv8.new_cache(2, 64, H, D), i32([[1, 0]])
    kv8.store(cache, k.to(DEV), k.nan_to_num().to(DEV), table, i32([n]), i32([0, n]))
    q = torch.randn(news, 2, D, device=DEV).half()
    lse = torch.full((news, 2), -math.inf, device=DEV)
    w = kv8.new_weights(cache) + 3
    kv8.weigh(w, q, lse, cache, table, i32([n]), 0.1, cu_q=i32([0, news]), max_q=news)
    assert w.eq(3).all()


def test_weigh_refuses():
    cache, _, table = filled([70], 64, 2, 64, torch.float16, seed=1)
    w, q = kv8.new_weights(cache), torch.zeros(1, 4, 64, device=DEV).half()
    ok = dict(weights=w, q=q, lse=torch.zeros(1, 4, device=DEV), cache=cache, table=i32(table),
              lens=i32([70]), scale=0.1)
    for bad in (dict(weights=w[:1]), dict(weights=w.double()), dict(q=q.float()), dict(q=q[:, :3]),
                dict(lse=torch.zeros(1, 3, device=DEV)), dict(lse=torch.zeros(1, 4)),
                dict(lse=torch.zeros(1, 4, device=DEV).half()), dict(scale=math.inf),
                dict(scale=math.nan), dict(lens=i32([70, 1])), dict(cu_q=i32([0])),
                dict(table=i32(table)[0]), dict(lens=i32([70]).long())):
        with pytest.raises(RuntimeError):
            kv8.weigh(**(ok | bad))


# -- eviction -----------------------------------------------------------------------------

EVICTS = [  # lens, keep, page, first, recent, used less than what is held
    ([64 * 9], [4], 64, 1, 1, 0), ([64 * 9 + 1, 30, 0, 640], [4, 1, 0, 20], 64, 1, 1, 0),
    ([3000, 500], [2, 0], 64, 5, 3, 0), ([256 * 40, 256 * 13 - 9], [3, 5], 256, 0, 1, 0),
    ([128 * 700], [100], 128, 1, 4, 0), ([64 * 30] * 90, list(range(90)), 64, 1, 1, 0),
    ([640, 640], [2, 2], 64, 0, 2, 7), ([640, 640], [2, 2], 64, 0, 2, 19),
    ([64 * 4500, 64 * 4200], [1000, 4199], 64, 1, 1, 0), ([64 * 6], [-5], 64, 4, 9, 0),
]


@pytest.mark.parametrize("kind", ["spread", "equal", "special"])
@pytest.mark.parametrize("case", range(len(EVICTS)))
def test_evict(case, kind):
    lens, keep, page, first, recent, less = EVICTS[case]
    print(f"evict {case} {kind}", flush=True)
    g = torch.Generator().manual_seed(case)
    table, pages = tables(lens, page, case, spare=3)
    H = 1 + case % 3
    weights = torch.exp(3 * torch.randn(pages, H, page // 64, generator=g))
    if kind == "equal":
        weights = (weights > 1).float()
    if kind == "special":
        weights[::3] = 0.0
        weights[1::5, 0] = math.inf
        weights[2::7, 0] = math.nan
        weights[::9] = -weights[::9]
        for row in table[:2]:
            row[1] = [-1, pages, 2 ** 31 - 1, -2 ** 31][case % 4]
    held = sum(-(-n // page) for n in lens)
    free = list(range(1000, 1000 + held + 4))
    used = max(0, held - less)
    dev_table = torch.full((len(lens), len(table[0]) + 2), -7, dtype=torch.int32, device=DEV)
    dev_table[:, :len(table[0])] = i32(table)
    t, f = dev_table[:, :len(table[0])], i32(free)
    got = kv8.evict(weights.to(DEV), t, i32(lens), i32(keep), f, i32([used]), first, recent)
    want = sv.evict(weights, page, table, lens, keep, free, used, first, recent)
    for name, a, b in zip(("table", "free", "lens", "used", "lost"), (t, f, *got),
                          (want[0], want[1], want[2], [want[3]], [want[4]])):
        assert a.tolist() == b, name
    assert dev_table[:, len(table[0]):].eq(-7).all()


def test_evict_of_nothing():
    w = torch.zeros(4, 2, 1, device=DEV)
    none = i32([])
    got = kv8.evict(w, none.view(0, 3), none, none, i32([5, 6]), i32([9]))
    assert got.lens.numel() == 0 and got.used.item() == 2 and got.lost.item() == 0
    t = i32([[0, 1], [2, 3]])
    got = kv8.evict(w, t, i32([100, -4]), i32([2, 0]), i32([]), i32([0]))
    assert t.tolist() == [[0, 1], [2, 3]] and got.lens.tolist() == [100, -4]
    # lengths past the table's row: what the row holds counts
    got = kv8.evict(w, t, i32([2 ** 31 - 1, 64]), i32([1, 1]), i32([9, 9]), i32([2]), first=0)
    assert t.tolist() == [[1, -1], [2, 3]] and got.lens.tolist() == [2 ** 31 - 1 - 64, 64]


def test_evict_refuses():
    w = torch.zeros(4, 2, 1, device=DEV)
    ok = dict(weights=w, table=i32([[0, 1]]), lens=i32([100]), keep=i32([1]), free_pages=i32([7, 8]),
              used=i32([1]))
    t = i32([[0, 1]])
    for bad in (dict(weights=w.half()), dict(weights=w.cpu()), dict(weights=w[..., None]),
                dict(weights=torch.zeros(4, 2, 3, device=DEV)), dict(keep=i32([1, 1])), dict(first=-1),
                dict(recent=0), dict(used=i32([1, 1])), dict(lens=i32([1, 1])),
                dict(table=i32([0, 1])), dict(free_pages=i32([7, 8]).long()),
                dict(table=t, free_pages=t[0]),
                dict(lens=i32([1, 1]), keep=i32([1, 1]), table=t.expand(2, 2))):
        with pytest.raises(RuntimeError):
            kv8.evict(**(ok | bad))


# -- what a program may do with all of it ---------------------------------------------------

def test_caches_without_pages_and_requests_without_keys():
    q = torch.randn(3, 4, 64, device=DEV).half()
    empty = kv8.new_cache(0, 64, 2, 64)
    for cache, table in ((empty, i32([[0], [0], [0]])), (kv8.new_cache(2, 64, 2, 64), i32([[], [], []]))):
        out, lse = kv8.attn(q, cache, table, i32([5, 0, 70]), 0.1, lse=True)
        assert out.eq(0).all() and lse.eq(-math.inf).all()
        w = kv8.new_weights(cache)
        kv8.weigh(w, q, lse, cache, table, i32([5, 0, 70]), 0.1)
        kv8.store(cache, q[:, :2], q[:, :2], table, i32([5, 0, 70]), weights=w)
        assert w.eq(0).all()
    none = kv8.attn(q[:0], kv8.new_cache(2, 64, 2, 64), i32([]).view(0, 4), i32([]), 0.1, lse=True)
    assert none[0].shape == (0, 4, 64) and none[1].shape == (0, 4)


@pytest.mark.parametrize("news", [1, 4, 200])
def test_hostile_lengths_tables_and_bounds_are_safe(news):
    """Any int in lens, table and cu_q: no access outside, rows of others right."""
    lens, H, D = [2 ** 31 - 1, -5, 130, 2 ** 31 - 1], 2, 64
    cache, held, table = filled([130], 64, H, D, torch.float16, seed=1)
    pages = len(cache.k)
    wild = [[2 ** 31 - 1, -2 ** 31, pages, -1], [0, 1, 0, 1], table[0] + [-1] * (4 - len(table[0])),
            [0, 0, 0, 0]]
    cu = offsets([news] * 4)
    q = torch.randn(cu[-1], 4, D, generator=torch.Generator().manual_seed(2)).half()
    out, lse = kv8.attn(q.to(DEV), cache, i32(wild), i32(lens), 0.1, cu_q=i32(cu), max_q=news, lse=True)
    rows = sv.attention(q[cu[2]:cu[3]], held, [wild[2]], [130], 0.1, [0, news])
    check(out[cu[2]:cu[3]], lse[cu[2]:cu[3]], rows)
    assert out[:cu[1]].eq(0).all() and out[cu[1]:cu[2]].eq(0).all()
    w = kv8.new_weights(cache)
    kv8.weigh(w, q.to(DEV), lse, cache, i32(wild), i32(lens), 0.1, cu_q=i32(cu), max_q=news)
    for bounds in ([0, 5, 3, 2, 4], [-9, 2 ** 31 - 1, 0, -1, 3], [4, 3, 2, 1, 0]):
        kv8.attn(q.to(DEV), cache, i32(wild), i32(lens), 0.1, cu_q=i32(bounds))
        kv8.weigh(w, q.to(DEV), lse, cache, i32(wild), i32(lens), 0.1, cu_q=i32(bounds))
    other = kv8.new_cache(pages, 64, H, D)
    x = torch.randn(cu[-1], H, D, device=DEV).half()
    wild[3] = [-1] * 4     # (page 0 is another request's)
    for bounds in ([0, 5, 3, 2, 4], [-9, 2 ** 31 - 1, 0, -1, 3], [4, 3, 2, 1, 0], cu):
        kv8.store(other, x, x, i32(wild), i32(lens), i32(bounds))
    torch.cuda.synchronize()


@pytest.mark.parametrize("n,news", [(200, 1), (2300, 2), (300, 200)])
@pytest.mark.parametrize("scale", [0.0, 1e-37, -1e-37])
def test_small_scales(scale, n, news):
    """A scale of 0 weighs every key alike; so do those that leave scores below rounding."""
    cache, held, table = filled([n], 64, 1, 64, torch.bfloat16, seed=n)
    q = torch.randn(news, 2, 64, generator=torch.Generator().manual_seed(n)).bfloat16() * 100
    out, lse = kv8.attn(q.to(DEV), cache, i32(table), i32([n]), scale, cu_q=i32([0, news]), max_q=news,
                        lse=True)
    check(out, lse, sv.attention(q, held, table, [n], scale, [0, news]))


@pytest.mark.parametrize("heads", [(4, 2), (32, 1)])
@pytest.mark.parametrize("lens,news", [([700, 64, 3], [1, 1, 1]), ([900, 300], [260, 5])])
def test_weights_of_all_blocks_add_up_to_the_rows(lens, news, heads):
    """With attention's own lse every row's weights add up to 1, whatever way they are added."""
    Hq, Hkv = heads
    cache, _, table = filled(lens, 64, Hkv, 128, torch.bfloat16, seed=9)
    cu = offsets(news)
    q = torch.randn(cu[-1], Hq, 128, device=DEV).bfloat16()
    _, lse = kv8.attn(q, cache, i32(table), i32(lens), 0.1, cu_q=i32(cu), max_q=max(news), lse=True)
    for max_q in (max(news), 2000):        # (the room for more queries may take another form)
        w = kv8.new_weights(cache)
        kv8.weigh(w, q, lse, cache, i32(table), i32(lens), 0.1, cu_q=i32(cu), max_q=max_q)
        got, rows = w.double().sum((0, 2)).cpu(), cu[-1] * Hq // Hkv
        # an lse of some units is off by some 2^-21 and a score in fp32 by as much
        assert ((got - rows).abs() <= rows * 2.0 ** -16).all(), got
    again = kv8.new_weights(cache)
    kv8.weigh(again, q, lse, cache, i32(table), i32(lens), 0.1, cu_q=i32(cu), max_q=2000)
    assert torch.equal(again, w)


def test_serving_with_eviction():
    """Prompts, then single tokens, every step through page planning, norm and rotation, storing,
    attention, weights and eviction; tokens, tables and pages against the oracle."""
    from gfx906_amd import qknorm
    B, Hq, Hkv, D, page, keep = 3, 4, 2, 64, 64, 4
    g = torch.Generator().manual_seed(0)
    cache, held = dirty_cache(24, page, Hkv, D), sv.Cache(24, page, Hkv, D)
    weights = kv8.new_weights(cache).fill_(5.0)
    table = torch.full((B, 8), -1, dtype=torch.int32, device=DEV)
    free = torch.randperm(24, generator=g).int().to(DEV)
    everything = sorted(free.tolist())
    lens, used, told = i32([0] * B), i32([0]), [0] * B
    cos, sin = qknorm.angles(4096, D // 2)
    went = 0
    for news in ([300, 70, 130], [1, 1, 1], [60, 1, 200], [1, 64, 1], [3, 100, 2], [1, 1, 1]):
        plan = kv8.plan_pages(lens, i32(news), table, free, used, page, sum(news))
        assert plan.missing.item() == 0
        cu = offsets(news)
        x = torch.randn(cu[-1], Hq + 2 * Hkv, D, generator=g).half().to(DEV)
        pos = i32([told[b] + t for b in range(B) for t in range(news[b])])
        told = [n + m for n, m in zip(told, news)]
        q, k = qknorm.norm_rotate(x[:, :Hq], x[:, Hq:Hq + Hkv], cos=cos, sin=sin, positions=pos)
        v = x[:, Hq + Hkv:]
        kv8.store(cache, k, v, table, plan.lens, plan.cu_new, weights)
        out, lse = kv8.attn(q, cache, table, plan.lens, D ** -0.5, cu_q=plan.cu_new, max_q=max(news),
                            lse=True)
        before = weights.clone()
        kv8.weigh(weights, q, lse, cache, table, plan.lens, D ** -0.5, cu_q=plan.cu_new,
                  max_q=max(news))
        rows, n = table.tolist(), plan.lens.tolist()
        held.store(k.cpu(), v.cpu(), rows, n, cu)
        same(cache, held, rows, n)
        check(out, lse, sv.attention(q.cpu(), held, rows, n, D ** -0.5, cu))
        want, tol = sv.weigh(before.cpu(), q.cpu(), lse.cpu(), held, rows, n, D ** -0.5, cu)
        weighed(weights, want, tol, rows, n, page)
        w, f, u = weights.cpu(), free.tolist(), plan.used.item()
        gone = kv8.evict(weights, table, plan.lens, i32([keep] * B), free, plan.used, first=1, recent=2)
        want = sv.evict(w, page, rows, n, [keep] * B, f, u, 1, 2)
        for a, b in zip((table, free, gone.lens, gone.used, gone.lost),
                        (want[0], want[1], want[2], [want[3]], [want[4]])):
            assert a.tolist() == b
        went += u - gone.used.item()
        lens, used = gone.lens, gone.used
        # every page is free or some request's, once
        mine = [p for r in table.tolist() for p in r if p >= 0]
        assert sorted(mine + free[used.item():].tolist()) == everything
    assert went > 0


def test_captured_step_replays():
    """A decoding step with all of it in one graph, replayed with new inputs in the same tensors;
    eager work and synchronisations in between."""
    B, Hq, Hkv, D, page = 3, 8, 2, 128, 64
    lens0 = [300, 63, 128]
    cache, _, rows = filled([n + 60 for n in lens0], page, Hkv, D, torch.float16, seed=3)
    table0, lens, cu = i32(rows), i32(lens0), i32(list(range(B + 1)))
    weights = kv8.new_weights(cache) + 1
    g = torch.Generator(device=DEV).manual_seed(1)
    q, k, v = (torch.randn(B, h, D, device=DEV, generator=g).half() for h in (Hq, Hkv, Hkv))
    out, table = torch.zeros_like(q), table0.clone()
    free, used, keep = i32([0] * 9), i32([9]), i32([3] * B)
    live = [cache.k, cache.k_scale, cache.v, cache.v_scale, weights, out, table, free]

    def step():
        kv8.store(cache, k, v, table, lens, cu, weights)
        _, lse = kv8.attn(q, cache, table, lens, 0.1, cu_q=cu, max_q=1, out=out, lse=True)
        kv8.weigh(weights, q, lse, cache, table, lens, 0.1, cu_q=cu, max_q=1)
        return lse, kv8.evict(weights, table, lens, keep, free, used)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lse, gone = step()
    for i in range(4):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, device=DEV, generator=g).half() * (1 + 3 * i))
        table.copy_(table0)
        lens.copy_(i32([n + i + 1 for n in lens0]))
        saved = [t.clone() for t in live]
        graph.replay()
        got = [t.clone() for t in (*live, lse, *gone)]
        torch.randn(1 << 18, device=DEV).sum().item()
        for t, x in zip(live, saved):
            t.copy_(x)
        l2, g2 = step()
        for a, b in zip(got, (*live, l2, *g2)):
            assert torch.equal(a.nan_to_num(9.0), b.nan_to_num(9.0)), f"replay {i}"
        torch.cuda.synchronize()


def test_captured_prompts_replay():
    lens, cu = [2500, 40, 700], [0, 150, 151, 300]
    cache, _, table = filled(lens, 64, 2, 128, torch.bfloat16, seed=4)
    table, n, cu = i32(table), i32(lens), i32(cu)
    q = torch.randn(300, 8, 128, device=DEV).bfloat16()

    def call():
        out, lse = kv8.attn(q, cache, table, n, 0.1, cu_q=cu, max_q=150, lse=True)
        w = kv8.new_weights(cache)
        kv8.weigh(w, q, lse, cache, table, n, 0.1, cu_q=cu, max_q=150)
        return out, lse, w

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for i in range(4):
        q.copy_(torch.randn(q.shape, device=DEV).bfloat16())
        graph.replay()
        torch.randn(1 << 18, device=DEV).sum().item()
        assert all(torch.equal(a, b) for a, b in zip(got, call())), f"replay {i}"
        torch.cuda.synchronize()


def test_streams_at_once():
    lens = [3000, 500, 1]
    cache, _, table = filled(lens, 128, 2, 64, torch.float16, seed=6)
    table, n = i32(table), i32(lens)
    qs = [torch.randn(3, 8, 64, device=DEV).half() for _ in range(6)]
    want = [kv8.attn(q, cache, table, n, 0.1, lse=True) for q in qs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    for i, q in enumerate(qs):
        with torch.cuda.stream(streams[i % 3]):
            got.append(kv8.attn(q, cache, table, n, 0.1, lse=True))
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for a, b in zip(got, want) for x, y in zip(a, b))


def test_offsets_past_32_bits():
    """Rows whose codes start past 2^32 bytes."""
    page, D, Hkv = 256, 128, 8
    pages = 2 ** 32 // (Hkv * page * D) + 3
    cache, small = kv8.new_cache(pages, page, Hkv, D), kv8.new_cache(2, page, Hkv, D)
    k, v = (torch.randn(300, Hkv, D, device=DEV).half() for _ in range(2))
    at = torch.arange(300, dtype=torch.int32, device=DEV)
    far, near, cu = i32([[pages - 1, pages - 2]]), i32([[0, 1]]), i32([0, 300])
    for c, t in ((cache, far), (small, near)):
        for a, b in ((0, 100), (100, 101), (101, 300)):     # parts of blocks, then a step
            kv8.store(c, k[a:b], v[a:b], t, i32([b]), i32([0, b - a]))
    slots = far[0, (at // page).long()] * page + at % page
    for a, b in zip(kv8.load(cache, slots), kv8.load(small, at)):
        assert torch.equal(a, b) and not a.eq(0).all()
    q = torch.randn(300, 16, D, device=DEV).half()
    for cu, m, n in ((None, 1, 1), (i32([0, 300]), 300, 300)):
        got = []
        for c, t in ((cache, far), (small, near)):
            w = kv8.new_weights(c)
            out, lse = kv8.attn(q[:n], c, t, i32([300]), 0.1, cu_q=cu, max_q=m, lse=True)
            kv8.weigh(w, q[:n], lse, c, t, i32([300]), 0.1, cu_q=cu, max_q=m)
            got.append((out, lse, w[t[0].long()]))
        assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.parametrize("B,Hq,Hkv,W", [(32, 16, 4, 64), (64, 2, 2, 64), (32, 16, 4, 33), (40, 64, 1, 40),
                                        (70, 4, 1, 50)])
def test_single_tokens_with_room_for_more(B, Hq, Hkv, W):
    """Without cu_q a request has one query, whatever max_q allows for: tables on either side
    of the short form's limits, requests on either side of 64."""
    g = torch.Generator().manual_seed(B + W)
    lens = [int(n) for n in torch.randint(1, 300, (B,), generator=g)]
    cache, held, table = filled(lens, 64, Hkv, 64, torch.float16, seed=B)
    table = [(row + [-1] * W)[:W] for row in table]
    q = torch.randn(B, Hq, 64, generator=g).half()
    want = kv8.attn(q.to(DEV), cache, i32(table), i32(lens), 0.125)
    check(want, None, sv.attention(q, held, table, lens, 0.125))
    for max_q in (2, 17, B, 1000, -1):
        got = kv8.attn(q.to(DEV), cache, i32(table), i32(lens), 0.125, max_q=max_q)
        assert torch.equal(got, want), max_q
