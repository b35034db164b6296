"""kv8_evict refuses results that lie over its arguments (no GPU: a refused call launches nothing)."""

import ctypes

import pytest

import gfx906_amd

P, I, L, Z = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_size_t
FAR = 1 << 20  # addresses that nothing dereferences


@pytest.fixture(scope="module")
def lib():
    try:
        so = gfx906_amd.capi()
    except gfx906_amd.NotBuiltError:
        pytest.skip("libraries not built")
    so.kv8_last_error.restype = ctypes.c_char_p
    so.kv8_evict.argtypes = [P, I, I, I, P, L, I, P, P, I, I, I, P, I, P, P, P, P, P, Z, P]
    return so


def evict(lib, **kw):
    a = dict(w=FAR, pages=9, Hkv=2, page=64, table=2 * FAR, stride=3, W=3, lens=3 * FAR, keep=4 * FAR, B=2,
             first=1, recent=1, free=5 * FAR, n_free=5, used=6 * FAR, out=7 * FAR, used_out=8 * FAR,
             lost=9 * FAR, ws=10 * FAR, n=1 << 40, stream=None) | kw
    return lib.kv8_evict(*a.values())


@pytest.mark.parametrize("bad,word", [
    (dict(out=3 * FAR), b"arguments"), (dict(out=4 * FAR), b"arguments"), (dict(out=3 * FAR + 4), b"arguments"),
    (dict(out=4 * FAR - 4), b"arguments"), (dict(out=6 * FAR), b"arguments"), (dict(out=6 * FAR - 4), b"arguments"),
    (dict(used_out=6 * FAR), b"arguments"), (dict(lost=6 * FAR), b"arguments"),
    (dict(lost=3 * FAR + 4), b"arguments"), (dict(used_out=5 * FAR + 16), b"arguments"),
    (dict(out=5 * FAR - 4), b"arguments"), (dict(lost=8 * FAR), b"each other"),
    (dict(used_out=7 * FAR + 4), b"each other")])
def test_results_over_arguments(lib, bad, word):
    assert evict(lib, **bad) == 1
    assert word in lib.kv8_last_error()
