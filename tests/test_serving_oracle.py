"""The CPU oracle of the serving operators against hand-made examples and torch's own operations."""

import math

import torch

from oracle import serving as sv


def test_codes():
    v = sv.values()
    assert v[:9].tolist() == [0, 1 / 512, 2 / 512, 3 / 512, 4 / 512, 5 / 512, 6 / 512, 7 / 512, 1 / 64]
    assert v[0x7e] == 448 and v[0x38] == 1 and v[0xb8] == -1 and math.isnan(v[0x7f]) and math.isnan(v[0xff])
    f8 = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    assert torch.equal(v.nan_to_num(9e9), f8.nan_to_num(9e9))
    x = torch.randn(5000, generator=torch.Generator().manual_seed(0)).double() * 100
    x = x.float().double().clamp(-448, 448)
    assert torch.equal(sv.round_codes(x), x.float().to(torch.float8_e4m3fn).double())
    ties = torch.tensor([1 + 1 / 16, 1 + 3 / 16, 1 / 1024, 3 / 1024, 464.0, -1e6]).double()
    assert sv.round_codes(ties).tolist() == [1, 1.25, 0, 4 / 1024, 448, -448]


def test_places_are_a_permutation_and_the_products_order():
    assert sorted(map(sv.place, range(64))) == list(range(64))
    # 8 bytes of half h and lane group g are tokens 32 h + 4 g + 0..3, 32 h + 16 + 4 g + 0..3
    for h in range(2):
        for g in range(4):
            first = 16 * g + 8 * h
            got = sorted(range(64), key=sv.place)[first:first + 8]
            assert got == [32 * h + 16 * kb + 4 * g + r for kb in range(2) for r in range(4)]


def test_scales():
    one = torch.ones(1)
    for top, e in ((0.0, -15), (448 * 2.0 ** -15, -15), (0.014, -14), (448, 0), (449, 1), (57344, 7),
                   (65504, 7), (3e38, 7), (1.0, -8), (1.75, -8), (1.76, -7)):
        assert sv.scale_for(one * top) == e, top
    assert sv.scale_for(torch.tensor([math.nan, math.inf, 2.0])) == -7


def test_cache_scales_grow_and_nan_stays():
    c = sv.Cache(2, 64, 1, 64)
    k = torch.ones(3, 1, 64).half()
    k[0, 0, 0], k[0, 0, 1], k[0, 0, 2] = math.nan, 0.01, math.inf
    c.store(k[:1], k[:1], [[1]], [1], [0, 1])
    assert c.e[0][1, 0, 0] == -8 and c.x[0][1, 0, 0, :3].isnan().tolist() == [True, False, True]
    small = c.x[0][1, 0, 0, 1].item()
    assert abs(small - 0.01) <= 0.01 * 2 ** -4
    k[1] = 500.0
    c.store(k[1:2], k[1:2], [[1]], [2], [0, 1])
    assert c.e[0][1, 0, 0] == 1 and c.x[0][1, 0, 1, 0] == 512
    # 0.01 in steps of 2 / 512
    assert c.x[0][1, 0, 0, 1] == 0.01171875 or c.x[0][1, 0, 0, 1] == 0.0078125
    c.store(k[2:], k[2:], [[1]], [1], [0, 1])   # the block begins anew
    assert c.e[0][1, 0, 0] == -8


def test_decode_reads_what_is_laid_out():
    g = torch.Generator().manual_seed(1)
    v = torch.randint(0, 126, (2, 3, 2, 64, 64), generator=g, dtype=torch.uint8)
    s = torch.exp2(torch.randint(-3, 3, (2, 3, 2), generator=g).float())
    x = sv.decode(v, s, True)
    assert x.shape == (2, 3, 128, 64)
    assert x[1, 2, 64 + 37, 5] == sv.values()[v[1, 2, 1, 5, sv.place(37)].long()] * s[1, 2, 1]
    k = torch.randint(0, 126, (2, 3, 128, 64), generator=g, dtype=torch.uint8)
    assert sv.decode(k, s, False)[1, 0, 70, 9] == sv.values()[k[1, 0, 70, 9].long()] * s[1, 0, 1]


def test_norm_rotate_is_the_norm_and_a_rotation():
    g = torch.Generator().manual_seed(2)
    x = torch.randn(2, 5, 3, 64, generator=g).half()
    w = torch.randn(64, generator=g)
    plain, _ = sv.norm_rotate(x, w, None, None, None, 1e-6, False)
    want = torch.nn.functional.rms_norm(x.double(), (64,), w.double(), 1e-6)
    assert torch.allclose(plain, want)
    angle = torch.rand(9, 16, generator=g).double()
    pos = torch.randint(0, 9, (2, 5), generator=g)
    for near in (False, True):
        y, tol = sv.norm_rotate(x, w, angle.cos().float(), angle.sin().float(), pos, 1e-6, near)
        a = plain[..., :32]
        z = torch.view_as_complex((a.unflatten(-1, (16, 2)) if near else
                                   torch.stack((a[..., :16], a[..., 16:]), -1)).contiguous())
        z = torch.view_as_real(z * torch.polar(torch.ones_like(angle), angle)[pos][:, :, None])
        z = z.flatten(-2) if near else torch.cat((z[..., 0], z[..., 1]), -1)
        assert torch.allclose(y[..., :32], z, atol=1e-6) and torch.equal(y[..., 32:], plain[..., 32:])
        assert (tol > 0).all()


def test_attention_and_weights_are_softmax():
    g = torch.Generator().manual_seed(3)
    c = sv.Cache(4, 64, 2, 64)
    k, v = torch.randn(2, 150, 2, 64, generator=g).half()
    table = [[3, 0, 2, -1]]
    c.store(k, v, table, [150], [0, 150])
    q = torch.randn(4, 4, 64, generator=g).half()
    rows = sv.attention(q, c, table, [150], 0.2, [0, 4])
    kk, vv, ok = c.rows(table[0], 150, 1)
    assert ok.all()
    z = q[1, 2].double() @ kk.T * 0.2
    z[148:] = -math.inf                       # the second of four queries
    o, _, lse, _ = rows[1]
    assert torch.allclose(o[2], torch.softmax(z, 0) @ vv) and torch.allclose(lse[2], torch.logsumexp(z, 0))
    lse = torch.stack([rows[r][2] for r in range(4)]).float()
    w, tol = sv.weigh(torch.zeros(4, 2, 1), q, lse, c, table, [150], 0.2, [0, 4])
    # every row's weights add up to 1
    assert torch.allclose(w.sum((0, 2)), torch.full((2,), 8.0).double(), atol=1e-5)
    assert w[1].eq(0).all() and (tol[0] > 0).all()


def test_eviction_example():
    w = torch.tensor([5.0, 1, 2, 2, 9, 0.5, math.nan, 3]).view(8, 1, 1)
    table, free, lens, used, lost = sv.evict(w, 64, [[7, 1, 2, 3, 4], [0, 5, 6, -1, -1]], [64 * 4 + 7, 192],
                                             [3, 1], [10, 11, 12, 13], 3, 1, 1)
    assert table == [[7, 3, 4, -1, -1], [0, 6, -1, -1, -1]]     # of equal weights the earlier goes
    assert lens == [64 * 2 + 7, 128] and free == [1, 2, 5, 13] and used == 0 and lost == 0
    table, free, lens, used, lost = sv.evict(w, 64, [[6, 1, -1, 3, 4]], [320], [2], [9, 9], 2, 0, 1)
    # an entry outside the cache weighs least, NaN most
    assert table == [[6, 4, -1, -1, -1]] and free == [1, -1] and used == 0 and lost == 1
