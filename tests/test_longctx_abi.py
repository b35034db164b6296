"""C entry points and Python layer of the 4-bit cache and sparse attention: sizes of
workspaces and refusals. No GPU: a refused call launches nothing."""

import ctypes

import pytest
import torch

import gfx906_amd
from gfx906_amd import kv4, sparse

P, I, L, F, Z = (ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_float, ctypes.c_size_t)
FAKE = 1 << 20  # an aligned address that nothing dereferences


@pytest.fixture(scope="module")
def lib():
    try:
        so = gfx906_amd.capi()
    except gfx906_amd.NotBuiltError:
        pytest.skip("libraries not built")
    S = ctypes.POINTER(L)
    so.kv4_last_error.restype = so.sparse_last_error.restype = ctypes.c_char_p
    so.kv4_plan_pages.argtypes = [P, P, P, L, I, P, I, P, I, I, I, P, P, P, P, P, P]
    so.kv4_store.argtypes = [P, P, S, S, I, I, I, I, P, P, P, P, P, I, I, P]
    so.kv4_load.argtypes = [P, P, I, I, I, I, P, P, P, P, P, I, I, P]
    so.kv4_attn_workspace_bytes.argtypes = [I] * 7
    so.kv4_attn_workspace_bytes.restype = Z
    so.kv4_attn.argtypes = [P, P, S, S, I, I, I, I, I, I, P, P, P, P, I, I, P, L, I, P, P, I, F, I,
                            P, Z, P]
    so.sparse_block_means.argtypes = [P, S, I, I, I, I, I, I, P, P]
    so.sparse_select_workspace_bytes.argtypes = [I] * 5
    so.sparse_select_workspace_bytes.restype = Z
    so.sparse_select.argtypes = [P, P] + [I] * 9 + [P, P, Z, P]
    so.sparse_attn_workspace_bytes.argtypes = [I] * 7
    so.sparse_attn_workspace_bytes.restype = Z
    so.sparse_attn.argtypes = [P, P, P, P, S, S, S, S] + [I] * 7 + [F, P, I, I, I, P, Z, P]
    return so


def strides(*s):
    return (L * len(s))(*s)


def kv4_attn(lib, **kw):
    a = dict(q=FAKE, o=2 * FAKE, qs=strides(1024, 128), os=strides(1024, 128), dtype=0, T=4, B=4, Hq=8,
             Hkv=2, D=128, kc=FAKE, ks=FAKE, vc=FAKE, vs=FAKE, pages=9, page=64, table=FAKE,
             stride=3, W=3, lens=FAKE, cu=None, max_q=1, scale=0.1, causal=1, ws=FAKE, n=1 << 40,
             stream=None) | kw
    return lib.kv4_attn(*a.values())


@pytest.mark.parametrize("bad,word", [
    (dict(D=96), b"head dim"), (dict(page=32), b"pages hold"), (dict(Hkv=0), b"kv heads"),
    (dict(Hkv=3), b"multiple of kv heads"), (dict(Hq=0), b"multiple of kv heads"),
    (dict(dtype=2), b"dtype"), (dict(T=-1), b"negative"), (dict(W=-1), b"negative"),
    (dict(B=5000, T=5000), b"requests"), (dict(T=5), b"one query"), (dict(q=None), b"null"),
    (dict(lens=None), b"null"), (dict(kc=None), b"null cache"), (dict(kc=FAKE + 8), b"aligned"),
    (dict(pages=1 << 25), b"2^31"), (dict(W=1 << 26), b"too wide"), (dict(q=FAKE + 2), b"aligned"),
    (dict(o=FAKE), b"must not be q"),
    (dict(W=1 << 24, stride=1 << 24, Hq=64, Hkv=64, os=strides(8192, 128)), b"too wide"),
    (dict(qs=strides(1024, 100)), b"multiples of 8"), (dict(os=strides(-4, 128)), b"non-negative"),
    (dict(os=strides(128, 128)), b"overlap"), (dict(scale=float("nan")), b"finite"),
    (dict(stride=-3), b"negative stride"), (dict(max_q=-1), b"negative")])
def test_cache_attention_refuses(lib, bad, word):
    assert kv4_attn(lib, **bad) == 1
    assert word in lib.kv4_last_error()


def test_cache_attention_workspace_is_checked(lib):
    big = dict(T=4, B=4, W=1000, stride=1000)
    need = lib.kv4_attn_workspace_bytes(4, 4, 8, 2, 128, 1, 64000)
    if need:
        assert kv4_attn(lib, **big, n=need - 1) == 1
        assert b"workspace" in lib.kv4_last_error()
        assert kv4_attn(lib, **big, ws=FAKE + 4) == 1


@pytest.mark.parametrize("empty", [dict(T=0, B=0), dict(T=0, B=4, cu=FAKE), dict(max_q=0)])
def test_cache_attention_with_no_queries_launches_nothing(lib, empty):
    assert kv4_attn(lib, **empty) == 0 and lib.kv4_last_error() is None


def plan(lib, **kw):
    a = dict(lens=FAKE, new=FAKE, table=FAKE, stride=4, W=4, free=FAKE, n_free=3, used=FAKE, B=2,
             page=64, n=9, slots=FAKE, cu=FAKE, out=FAKE, used_out=FAKE, missing=FAKE,
             stream=None) | kw
    return lib.kv4_plan_pages(*a.values())


@pytest.mark.parametrize("bad,word", [
    (dict(page=65), b"pages hold"), (dict(B=4097), b"requests"), (dict(B=-1), b"requests"),
    (dict(W=-1), b"negative"), (dict(stride=3), b"overlapping"), (dict(n=-1), b"negative"),
    (dict(lens=None), b"null"), (dict(slots=None), b"null"), (dict(used=None), b"null")])
def test_plan_refuses(lib, bad, word):
    assert plan(lib, **bad) == 1 and word in lib.kv4_last_error()


@pytest.mark.parametrize("bad,word", [
    (dict(D=32), b"head dim"), (dict(T=-1), b"negative"), (dict(k=FAKE + 2), b"aligned"),
    (dict(ks=strides(12, 8)), b"multiples of 8"), (dict(slots=None), b"null"),
    (dict(dtype=7), b"dtype")])
def test_store_refuses(lib, bad, word):
    a = dict(k=FAKE, v=FAKE, ks=strides(256, 128), vs=strides(256, 128), dtype=1, T=3, Hkv=2, D=128,
             slots=FAKE, a=FAKE, b=FAKE, c=FAKE, d=FAKE, pages=2, page=64, stream=None) | bad
    assert lib.kv4_store(*a.values()) == 1 and word in lib.kv4_last_error()


def test_load_refuses(lib):
    ok = [FAKE, FAKE, 0, 3, 2, 128, FAKE, FAKE, FAKE, FAKE, FAKE, 2, 64, None]
    for at, val in ((2, 3), (3, -1), (5, 100), (12, 63), (6, None), (0, FAKE + 4)):
        args = list(ok)
        args[at] = val
        assert lib.kv4_load(*args) == 1, (at, val)


def sparse_attn(lib, **kw):
    s = strides(1 << 20, 1 << 16, 128)
    a = dict(q=FAKE, k=FAKE, v=FAKE, o=FAKE, qs=s, ks=s, vs=s, os=s, dtype=0, B=2, Hq=4, Hkv=2,
             Sq=300, Skv=400, D=128, scale=0.1, index=FAKE, block=64, count=5, causal=0, ws=FAKE,
             n=1 << 40, stream=None) | kw
    return lib.sparse_attn(*a.values())


@pytest.mark.parametrize("bad,word", [
    (dict(D=72), b"head dim"), (dict(block=32), b"blocks"), (dict(Hkv=3), b"multiple"),
    (dict(Hkv=0), b"multiple"), (dict(dtype=2), b"dtype"), (dict(Sq=-1), b"negative"),
    (dict(Skv=1 << 30), b"2^30"), (dict(Skv=(1 << 21) + 64), b"key blocks"),
    (dict(count=0), b"count"), (dict(count=2049), b"count"), (dict(scale=float("inf")), b"finite"),
    (dict(index=None), b"null"), (dict(k=None), b"null"), (dict(q=FAKE + 8), b"aligned"),
    (dict(ks=strides(1 << 20, 1 << 16, 100)), b"multiples of 8"),
    (dict(ks=strides(0, 0, 1 << 23)), b"2^22"), (dict(os=strides(0, 1 << 16, 128)), b"overlap"),
    (dict(vs=strides(1 << 20, 1 << 16, 64)), b"rows overlap"), (dict(B=300, Hq=300), b"65535")])
def test_sparse_attention_refuses(lib, bad, word):
    assert sparse_attn(lib, **bad) == 1 and word in lib.sparse_last_error()


def test_sparse_attention_workspace_is_checked(lib):
    need = lib.sparse_attn_workspace_bytes(2, 4, 1, 32768, 128, 64, 64)
    if need:
        kw = dict(Sq=1, Skv=32768, count=64)
        assert sparse_attn(lib, **kw, n=need - 1) == 1 and b"workspace" in lib.sparse_last_error()
        assert sparse_attn(lib, **kw, ws=FAKE + 4) == 1


@pytest.mark.parametrize("bad,word", [
    (dict(count=2, causal=1), b"own positions"), (dict(D=40), b"head dim"), (dict(n=15), b"workspace"),
    (dict(km=None), b"null"), (dict(count=0), b"count")])
def test_select_refuses(lib, bad, word):
    a = dict(qm=FAKE, km=FAKE, B=2, Hq=4, Hkv=2, Sq=300, Skv=400, D=64, block=64, count=3, causal=0,
             index=FAKE, ws=FAKE, n=1 << 30, stream=None) | bad
    assert lib.sparse_select(*a.values()) == 1 and word in lib.sparse_last_error()


@pytest.mark.parametrize("bad,word", [
    (dict(dtype=2), b"dtype"), (dict(qs=None), b"null"), (dict(qs=strides(9, 8, 8)), b"multiples"),
    (dict(q=FAKE + 4), b"aligned"), (dict(km=FAKE + 8), b"aligned"),
    (dict(n=15, Sq=300000, Skv=300000), b"workspace"),
    (dict(causal=1, count=2), b"own positions"), (dict(Hkv=3), b"multiple of kv heads")])
def test_choose_refuses(lib, bad, word):
    lib.sparse_choose.argtypes = [P, ctypes.POINTER(L), I, P] + [I] * 9 + [P, P, Z, P]
    a = dict(q=FAKE, qs=strides(1 << 20, 1 << 16, 64), dtype=0, km=FAKE, B=2, Hq=4, Hkv=2, Sq=300,
             Skv=400, D=64, block=64, count=3, causal=0, index=FAKE, ws=FAKE, n=1 << 30,
             stream=None) | bad
    assert lib.sparse_choose(*a.values()) == 1 and word in lib.sparse_last_error()


def test_means_refuses(lib):
    s = strides(1 << 20, 1 << 16, 128)
    ok = [FAKE, s, 0, 2, 4, 300, 128, 64, FAKE, None]
    for at, val in ((2, 5), (3, -1), (6, 80), (7, 100), (8, None), (0, FAKE + 2),
                    (1, strides(8, 8, 4))):
        args = list(ok)
        args[at] = val
        assert lib.sparse_block_means(*args) == 1, (at, val)


def test_grids_past_what_a_launch_takes_are_refused(lib):
    """Sizes whose grid would have 2^32 threads or more: refused before the first launch."""
    many = dict(B=4096, T=4096, Hq=4096, Hkv=4096, W=1, stride=1, os=strides(4096 * 128, 128))
    assert kv4_attn(lib, **many) == 1 and b"too many" in lib.kv4_last_error()
    rows = dict(T=1 << 25, Hq=64, Hkv=8, cu=FAKE, max_q=1 << 25, os=strides(8192, 128))
    assert kv4_attn(lib, **rows) == 1 and b"too many" in lib.kv4_last_error()
    far = strides(0, 1 << 40, 128)
    assert sparse_attn(lib, B=1, Hq=4, Sq=1 << 29, os=far) == 1
    assert b"too many" in lib.sparse_last_error()
    a = (FAKE, FAKE, 1, 1, 1, 1 << 29, 400, 64, 64, 3, 0, FAKE, FAKE, 1 << 50, None)
    assert lib.sparse_select(*a) == 1 and b"too many" in lib.sparse_last_error()
    assert lib.sparse_block_means(FAKE, far, 0, 1, 8, 1 << 29, 128, 64, FAKE, None) == 1
    assert b"too many" in lib.sparse_last_error()


def test_python_layer_refuses_on_the_cpu(lib):
    with pytest.raises(ValueError):
        kv4.new_cache(4, 32, 2, 128, device="cpu")
    with pytest.raises(ValueError):
        kv4.new_cache(4, 64, 2, 80, device="cpu")
    cache = kv4.new_cache(4, 64, 2, 128, device="cpu")
    assert cache.page == 64
    q, lens = torch.zeros(1, 2, 128).half(), torch.ones(1, dtype=torch.int32)
    table = torch.zeros(1, 1, dtype=torch.int32)
    for call in (lambda: kv4.attn(q, cache, table, lens, 0.1),
                 lambda: kv4.store(cache, q, q, lens), lambda: kv4.load(cache, lens),
                 lambda: kv4.plan_pages(lens, lens, table, lens, lens, 64, 1)):
        with pytest.raises(RuntimeError):
            call()
    x = torch.zeros(1, 1, 64, 64).half()
    for call in (lambda: sparse.block_means(x, 64), lambda: sparse.attn(x, x, x, 0.1, 4)):
        with pytest.raises(RuntimeError):
            call()
    for scale in (0.0, -1.0, float("nan")):
        with pytest.raises(ValueError):
            sparse.attn(x, x, x, scale, 4)


@pytest.mark.parametrize("B,Hq,Hkv,W", [(32, 16, 4, 64), (64, 2, 2, 64), (40, 64, 1, 40)])
def test_without_cu_q_a_request_has_one_query(lib, B, Hq, Hkv, W):
    """The workspace of max_q = 1 is the one that is asked for, whatever max_q is: a larger
    one would have these tables in the form that needs none, or in the prompts'."""
    need = lib.kv4_attn_workspace_bytes(B, B, Hq, Hkv, 128, 1, 64 * W)
    assert need > 0
    assert lib.kv4_attn_workspace_bytes(B, B, Hq, Hkv, 128, B, 64 * W) != need
    for max_q in (1, 2, B, 1000):
        kw = dict(T=B, B=B, Hq=Hq, Hkv=Hkv, W=W, stride=W, max_q=max_q, os=strides(128 * Hq, 128))
        assert kv4_attn(lib, **kw, n=need - 1) == 1
        assert b"workspace" in lib.kv4_last_error()


@pytest.mark.parametrize("scale", [2.5e38, -3e38, float("inf"), float("-inf"), float("nan")])
def test_scales_past_fp32_in_log2_units_are_refused(lib, scale):
    """Scores are multiplied by scale * log2(e), which must not be infinite."""
    assert kv4_attn(lib, scale=scale) == 1 and b"finite" in lib.kv4_last_error()
    assert sparse_attn(lib, scale=scale) == 1 and b"finite" in lib.sparse_last_error()


def test_workspaces_that_calls_need_are_not_empty(lib):
    """Long tables and short query lists are split, and ask for all of what the sizing calls say."""
    need = lib.kv4_attn_workspace_bytes(4, 4, 8, 2, 128, 1, 64000)
    assert need > 0
    for bad in (dict(n=need - 1), dict(n=0), dict(ws=None), dict(ws=FAKE + 4, n=need)):
        assert kv4_attn(lib, W=1000, stride=1000, **bad) == 1
        assert b"workspace" in lib.kv4_last_error()
    prompt = lib.kv4_attn_workspace_bytes(400, 4, 8, 2, 128, 300, 64000)
    assert prompt > need
    assert kv4_attn(lib, W=1000, stride=1000, T=400, cu=FAKE, max_q=300, n=prompt - 1) == 1
    assert b"workspace" in lib.kv4_last_error()
    need = lib.sparse_attn_workspace_bytes(2, 4, 1, 32768, 128, 64, 64)
    assert need > 0
    for bad in (dict(n=need - 1), dict(n=0), dict(ws=None), dict(ws=FAKE + 4, n=need)):
        assert sparse_attn(lib, Sq=1, Skv=32768, count=64, **bad) == 1
        assert b"workspace" in lib.sparse_last_error()
