"""C entry points and Python layer of the serving operators: sizes of workspaces and refusals.
No GPU: a refused call launches nothing."""

import ctypes

import pytest
import torch

import gfx906_amd
from gfx906_amd import kv8, qknorm

P, I, L, F, Z = (ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_float, ctypes.c_size_t)
FAKE = 1 << 20  # an aligned address that nothing dereferences


@pytest.fixture(scope="module")
def lib():
    try:
        so = gfx906_amd.capi()
    except gfx906_amd.NotBuiltError:
        pytest.skip("libraries not built")
    S = ctypes.POINTER(L)
    so.kv8_last_error.restype = so.qk_norm_rotate_last_error.restype = ctypes.c_char_p
    so.qk_norm_rotate.argtypes = ([P] * 4 + [S] * 4 + [I] * 6 + [P, P, I, F, P, P, L, I, I, I, P, S, P])
    so.kv8_store.argtypes = [P, P, S, S, I, I, I, I, I, P, P, P, P, I, I, P, L, I, P, P, P, P]
    so.kv8_load.argtypes = [P, P, I, I, I, I, P, P, P, P, P, I, I, P]
    so.kv8_attn_workspace_bytes.argtypes = so.kv8_weigh_workspace_bytes.argtypes = [I] * 7
    so.kv8_evict_workspace_bytes.argtypes = [I] * 2
    for f in (so.kv8_attn_workspace_bytes, so.kv8_weigh_workspace_bytes, so.kv8_evict_workspace_bytes):
        f.restype = Z
    so.kv8_attn.argtypes = [P, P, P, S, S, I, I, I, I, I, I, P, P, P, P, I, I, P, L, I, P, P, I, F, I,
                            P, Z, P]
    so.kv8_weigh.argtypes = [P, P, S, I, P, I, I, I, I, I, P, P, I, I, P, L, I, P, P, I, F, I, P, Z, P]
    so.kv8_evict.argtypes = [P, I, I, I, P, L, I, P, P, I, I, I, P, I, P, P, P, P, P, Z, P]
    return so


def strides(*s):
    return (L * len(s))(*s)


def rotate(lib, **kw):
    s = strides(1 << 20, 2048, 128)
    a = dict(q=FAKE, k=FAKE, qo=2 * FAKE, ko=3 * FAKE, qs=s, ks=s, qos=s, kos=s, dtype=1, B=2, S=9, Hq=8,
             Hk=2, D=128, wq=None, wk=None, w32=0, eps=1e-6, cos=FAKE, sin=FAKE, stride=64, N=9, R=128,
             near=0, pos=None, ps=None, stream=None) | kw
    return lib.qk_norm_rotate(*a.values())


@pytest.mark.parametrize("bad,word", [
    (dict(dtype=2), b"dtype"), (dict(D=60), b"head dim"), (dict(D=520), b"head dim"),
    (dict(D=0), b"head dim"), (dict(B=-1), b"tokens or heads"), (dict(Hq=70000), b"tokens or heads"),
    (dict(B=1 << 16, S=1 << 16), b"too many tokens"), (dict(R=24), b"rotated dims"),
    (dict(R=4, near=1), b"rotated dims"), (dict(R=144), b"rotated dims"), (dict(R=-16), b"rotated dims"),
    (dict(eps=-1e-6), b"eps"), (dict(eps=float("nan")), b"eps"), (dict(eps=float("inf")), b"eps"),
    (dict(q=None), b"null"), (dict(ko=None), b"null"), (dict(cos=None), b"null"), (dict(pos=FAKE), b"null"),
    (dict(N=0), b"angles need rows"), (dict(stride=62), b"16-byte"), (dict(sin=FAKE + 4), b"16-byte"),
    (dict(N=8), b"fewer rows"), (dict(q=FAKE + 2), b"16-byte"), (dict(ko=FAKE + 8), b"16-byte"),
    (dict(qs=strides(8, 12, 8)), b"multiples of 8"), (dict(kos=strides(1 << 20, 2048, 64)), b"overlap"),
    (dict(qos=strides(0, 2048, 128)), b"overlap")])
def test_norm_rotate_refuses(lib, bad, word):
    assert rotate(lib, **bad) == 1
    assert word in lib.qk_norm_rotate_last_error()


@pytest.mark.parametrize("empty", [dict(B=0), dict(S=0), dict(Hq=0, Hk=0)])
def test_norm_rotate_of_nothing_launches_nothing(lib, empty):
    assert rotate(lib, **empty) == 0 and lib.qk_norm_rotate_last_error() is None


def store(lib, **kw):
    a = dict(k=FAKE, v=FAKE, ks=strides(256, 128), vs=strides(256, 128), dtype=1, T=3, B=3, Hkv=2, D=128,
             a=FAKE, b=FAKE, c=FAKE, d=FAKE, pages=2, page=64, table=FAKE, stride=2, W=2, lens=FAKE,
             cu=None, w=None, stream=None) | kw
    return lib.kv8_store(*a.values())


@pytest.mark.parametrize("bad,word", [
    (dict(D=32), b"head dim"), (dict(page=96), b"pages hold"), (dict(T=-1), b"negative"),
    (dict(B=5000, T=5000), b"requests"), (dict(T=4), b"one row"), (dict(k=FAKE + 2), b"aligned"),
    (dict(ks=strides(12, 8)), b"multiples of 8"), (dict(lens=None), b"null"), (dict(dtype=7), b"dtype"),
    (dict(table=None), b"null table"), (dict(W=-1), b"null table"), (dict(W=1 << 26), b"too wide"),
    (dict(stride=-1), b"negative stride"), (dict(a=FAKE + 8), b"aligned"), (dict(b=None), b"null cache"),
    (dict(Hkv=0), b"kv heads"), (dict(pages=1 << 25), b"2^31"),
    (dict(T=1 << 30, cu=FAKE, Hkv=4096), b"too many")])
def test_store_refuses(lib, bad, word):
    assert store(lib, **bad) == 1 and word in lib.kv8_last_error()


@pytest.mark.parametrize("empty", [dict(T=0, B=0), dict(T=0, cu=FAKE), dict(pages=0), dict(W=0)])
def test_store_of_nothing_launches_nothing(lib, empty):
    assert store(lib, **empty) == 0 and lib.kv8_last_error() is None


def test_load_refuses(lib):
    ok = [FAKE, FAKE, 0, 3, 2, 128, FAKE, FAKE, FAKE, FAKE, FAKE, 2, 64, None]
    for at, val in ((2, 3), (3, -1), (5, 100), (12, 63), (6, None), (0, FAKE + 4), (4, 40000), (7, None)):
        args = list(ok)
        args[at] = val
        assert lib.kv8_load(*args) == 1, (at, val)
    assert lib.kv8_load(*[*ok[:3], 0, *ok[4:]]) == 0


def attn(lib, **kw):
    a = dict(q=FAKE, o=2 * FAKE, lse=None, qs=strides(1024, 128), os=strides(1024, 128), dtype=0, T=4,
             B=4, Hq=8, Hkv=2, D=128, kc=FAKE, ks=FAKE, vc=FAKE, vs=FAKE, pages=9, page=64, table=FAKE,
             stride=3, W=3, lens=FAKE, cu=None, max_q=1, scale=0.1, causal=1, ws=FAKE, n=1 << 40,
             stream=None) | kw
    return lib.kv8_attn(*a.values())


@pytest.mark.parametrize("bad,word", [
    (dict(D=96), b"head dim"), (dict(page=32), b"pages hold"), (dict(Hkv=0), b"kv heads"),
    (dict(Hkv=3), b"multiple of kv heads"), (dict(Hq=0), b"multiple of kv heads"),
    (dict(dtype=2), b"dtype"), (dict(T=-1), b"negative"), (dict(W=-1), b"negative"),
    (dict(B=5000, T=5000), b"requests"), (dict(T=5), b"one query"), (dict(q=None), b"null"),
    (dict(lens=None), b"null"), (dict(kc=None), b"null cache"), (dict(kc=FAKE + 8), b"aligned"),
    (dict(pages=1 << 25), b"2^31"), (dict(W=1 << 26), b"too wide"), (dict(q=FAKE + 2), b"aligned"),
    (dict(o=FAKE), b"must not be q"), (dict(lse=FAKE + 2), b"aligned"),
    (dict(W=1 << 24, stride=1 << 24, Hq=64, Hkv=64, os=strides(8192, 128)), b"too wide"),
    (dict(qs=strides(1024, 100)), b"multiples of 8"), (dict(os=strides(-4, 128)), b"non-negative"),
    (dict(os=strides(128, 128)), b"overlap"), (dict(scale=float("nan")), b"finite"),
    (dict(scale=3e38), b"finite"), (dict(stride=-3), b"negative stride"), (dict(max_q=-1), b"negative"),
    (dict(T=1 << 25, Hq=64, Hkv=8, cu=FAKE, max_q=1 << 25, os=strides(8192, 128)), b"too many")])
def test_attention_refuses(lib, bad, word):
    assert attn(lib, **bad) == 1
    assert word in lib.kv8_last_error()


def test_workspaces_are_checked(lib):
    need = lib.kv8_attn_workspace_bytes(4, 4, 8, 2, 128, 1, 64000)
    assert need > 0 and lib.kv8_attn_workspace_bytes(4, 4, 8, 2, 128, 1, 640) == 0
    for bad in (dict(n=need - 1), dict(n=0), dict(ws=None), dict(ws=FAKE + 4, n=need)):
        assert attn(lib, W=1000, stride=1000, **bad) == 1
        assert b"workspace" in lib.kv8_last_error()
    prompt = lib.kv8_attn_workspace_bytes(400, 4, 8, 2, 128, 300, 64000)
    assert prompt > need
    assert attn(lib, W=1000, stride=1000, T=400, cu=FAKE, max_q=300, n=prompt - 1) == 1
    # without cu_q a request has one query, whatever max_q is
    for max_q in (1, 2, 1000):
        assert attn(lib, W=1000, stride=1000, max_q=max_q, n=need - 1) == 1

    few = lib.kv8_weigh_workspace_bytes(4, 4, 8, 2, 1, 1000, 64)
    many = lib.kv8_weigh_workspace_bytes(4000, 4, 8, 2, 2000, 1000, 64)
    assert few == 0 and many > 0
    for bad in (dict(n=many - 1), dict(ws=None), dict(ws=FAKE + 2, n=many)):
        assert weigh(lib, W=1000, stride=1000, T=4000, cu=FAKE, max_q=2000, **bad) == 1
        assert b"workspace" in lib.kv8_last_error()
    # parts are fewer where there are many blocks, and one needs no room
    assert lib.kv8_weigh_workspace_bytes(1 << 20, 4096, 64, 64, 4000, 4096, 256) == 0

    assert lib.kv8_evict_workspace_bytes(9, 4096) == 0
    need = lib.kv8_evict_workspace_bytes(9, 4097)
    assert need == 9 * 4097 * 8
    for bad in (dict(n=need - 1), dict(ws=None), dict(ws=FAKE + 4, n=need)):
        assert evict(lib, B=9, W=4097, stride=4097, **bad) == 1
        assert b"workspace" in lib.kv8_last_error()


def weigh(lib, **kw):
    a = dict(w=FAKE, q=FAKE, qs=strides(1024, 128), dtype=0, lse=FAKE, T=4, B=4, Hq=8, Hkv=2, D=128,
             kc=FAKE, ks=FAKE, pages=9, page=64, table=FAKE, stride=3, W=3, lens=FAKE, cu=None, max_q=1,
             scale=0.1, causal=1, ws=FAKE, n=1 << 40, stream=None) | kw
    return lib.kv8_weigh(*a.values())


@pytest.mark.parametrize("bad,word", [
    (dict(D=96), b"head dim"), (dict(page=32), b"pages hold"), (dict(Hkv=3), b"multiple of kv heads"),
    (dict(dtype=2), b"dtype"), (dict(T=-1), b"negative"), (dict(W=-1), b"negative"),
    (dict(B=5000, T=5000), b"requests"), (dict(T=5), b"one query"), (dict(q=None), b"null"),
    (dict(w=None), b"null"), (dict(lse=None), b"null"), (dict(kc=None), b"null cache"),
    (dict(W=1 << 26), b"too wide"), (dict(q=FAKE + 2), b"aligned"), (dict(w=FAKE + 2), b"aligned"),
    (dict(qs=strides(1024, 100)), b"multiples of 8"), (dict(scale=float("inf")), b"finite"),
    (dict(T=1 << 30, Hq=16, cu=FAKE, max_q=1 << 30), b"query rows"),
    (dict(W=1 << 24, stride=1 << 24, B=4096, T=4096), b"too wide")])
def test_weigh_refuses(lib, bad, word):
    assert weigh(lib, **bad) == 1
    assert word in lib.kv8_last_error()


@pytest.mark.parametrize("empty", [dict(T=0, B=0), dict(T=0, B=4, cu=FAKE), dict(max_q=0), dict(W=0),
                                   dict(pages=0)])
def test_weigh_of_nothing_launches_nothing(lib, empty):
    assert weigh(lib, **empty) == 0 and lib.kv8_last_error() is None


def evict(lib, **kw):
    a = dict(w=FAKE, pages=9, Hkv=2, page=64, table=FAKE, stride=3, W=3, lens=FAKE, keep=FAKE, B=2,
             first=1, recent=1, free=FAKE, n_free=5, used=FAKE, out=FAKE, used_out=FAKE, lost=FAKE,
             ws=FAKE, n=1 << 40, stream=None) | kw
    return lib.kv8_evict(*a.values())


@pytest.mark.parametrize("bad,word", [
    (dict(page=100), b"pages hold"), (dict(Hkv=0), b"kv heads"), (dict(pages=1 << 25), b"2^31"),
    (dict(B=-1), b"requests"), (dict(B=4097), b"requests"), (dict(n_free=-1), b"negative"),
    (dict(first=-1), b"first"), (dict(recent=0), b"recent"), (dict(W=-1), b"negative width"),
    (dict(table=None), b"null table"), (dict(stride=2), b"overlapping"), (dict(lens=None), b"null"),
    (dict(keep=None), b"null"), (dict(used=None), b"null"), (dict(lost=None), b"null"),
    (dict(free=None), b"null"), (dict(w=None), b"null"), (dict(out=None), b"null")])
def test_evict_refuses(lib, bad, word):
    assert evict(lib, **bad) == 1
    assert word in lib.kv8_last_error()


def test_python_layer_refuses_on_the_cpu(lib):
    for bad in ((4, 32, 2, 128), (4, 64, 2, 80)):
        with pytest.raises(ValueError):
            kv8.new_cache(*bad, device="cpu")
    cache = kv8.new_cache(4, 128, 2, 64, device="cpu")
    assert cache.page == 128 and cache.v.shape == (4, 2, 2, 64, 64)
    assert kv8.new_weights(cache).shape == (4, 2, 2)
    assert sum(t.numel() * t.element_size() for t in (cache.k, cache.v)) == 4 * 2 * 128 * 64 * 2
    q, n = torch.zeros(1, 2, 64).half(), torch.ones(1, dtype=torch.int32)
    table, w = torch.zeros(1, 1, dtype=torch.int32), kv8.new_weights(cache)
    for call in (lambda: kv8.attn(q, cache, table, n, 0.1), lambda: kv8.store(cache, q, q, table, n),
                 lambda: kv8.load(cache, n), lambda: kv8.weigh(w, q, torch.zeros(1, 2), cache, table, n, 0.1),
                 lambda: kv8.evict(w, table, n, n, n, n), lambda: qknorm.norm_rotate(q, q),
                 lambda: kv8.plan_pages(n, n, table, n, n, 64, 1)):
        with pytest.raises(RuntimeError):
            call()


def test_angles():
    cos, sin = qknorm.angles(70000, 4, base=100.0, device="cpu")
    assert cos.dtype == torch.float32 and cos.shape == sin.shape == (70000, 4)
    x = torch.tensor(69999 * 100.0 ** -0.25, dtype=torch.float64)
    assert abs(cos[69999, 1].double() - x.cos()) < 1e-7 and abs(sin[69999, 1].double() - x.sin()) < 1e-7
