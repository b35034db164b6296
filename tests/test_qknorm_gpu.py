"""Norms of queries and keys with the position rotation on the GPU against the CPU oracle in 64
bits."""

import math

import pytest
import torch

import gfx906_amd
from gfx906_amd import qknorm
from oracle import serving as sv
from oracle.attention import sdpa_math_fp32

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float16, torch.bfloat16]


def close(got, want, tol, where=""):
    got = got.double().cpu()
    assert torch.equal(got.isnan(), want.isnan()), f"{where}: NaN"
    err = ((got - want).abs() / tol)[~want.isnan()]
    worst = err.max().item() if err.numel() else 0.0
    print(f"  {where} worst {worst:.3f} of the bound", flush=True)
    assert worst <= 1.0, f"{where}: {worst} of the bound"


def check(q, k, wq, wk, cos, sin, positions, eps, neighbours, got):
    host = [None if t is None else t.cpu() for t in (cos, sin, positions)]
    for name, x, w, y in (("q", q, wq, got[0]), ("k", k, wk, got[1])):
        want, tol = sv.norm_rotate(x.cpu(), None if w is None else w.cpu(), *host, eps, neighbours)
        close(y, want, tol, name)


SHAPES = [  # B, S, Hq, Hk, D, R
    (1, 1, 1, 1, 8, 8), (1, 5, 3, 1, 16, 16), (2, 3, 2, 2, 24, 16), (1, 70, 8, 2, 128, 128),
    (2, 33, 5, 5, 64, 32), (1, 9, 40, 8, 128, 64), (3, 4, 2, 1, 80, 80), (1, 17, 6, 6, 40, 0),
    (1, 3, 1, 2, 512, 512), (2, 2, 3, 1, 256, 64), (1, 300, 24, 24, 64, 64), (1, 2, 2, 1, 504, 496),
]


@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", range(len(SHAPES)))
def test_norm_rotate(case, dtype, neighbours):
    B, S, Hq, Hk, D, R = SHAPES[case]
    R = R if neighbours else R // 16 * 16        # (pairs of halves come in sixteens of dims)
    print(f"norm_rotate {SHAPES[case]} {dtype} neighbours {neighbours}", flush=True)
    g = torch.Generator().manual_seed(case)
    x = (torch.randn(B, S, Hq + 2 * Hk, D, generator=g) * 3).to(dtype).to(DEV)
    q, k = x[:, :, :Hq], x[:, :, Hq:Hq + Hk]     # parts of one projection
    if case % 3 == 1:                            # [B, H, S, D] in memory
        q, k = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k))
    wt = torch.float32 if case % 2 else dtype
    wq, wk = ((1 + 0.3 * torch.randn(D, generator=g)).to(wt).to(DEV) for _ in range(2))
    cos = sin = positions = None
    if R:
        cos, sin = qknorm.angles(max(S, 50), R // 2)
        if case % 4 != 2:
            positions = torch.randint(0, 50, (B, S), generator=g).int().to(DEV)
    got = qknorm.norm_rotate(q, k, wq, wk, cos, sin, positions, 1e-5, neighbours)
    if case % 3 == 1:
        assert got[0].stride() == q.stride()     # dense inputs keep their order
    check(q, k, wq, wk, cos, sin, positions, 1e-5, neighbours, got)


MANY = [  # B, S, Hq, Hk, D, R: few heads of many tokens, whole and with a ragged end
    (1, 65600, 1, 1, 8, 8), (2, 16387, 1, 0, 16, 16), (3, 2731, 1, 1, 64, 64), (1, 4101, 1, 1, 128, 96),
    (1, 2049, 1, 1, 200, 192), (3, 2731, 3, 1, 512, 512), (2, 8193, 2, 4, 248, 64), (1, 1024, 1, 0, 512, 0),
]


@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("case", range(len(MANY)))
def test_few_heads_of_many_tokens(case, neighbours):
    B, S, Hq, Hk, D, R = MANY[case]
    R = R if neighbours else R // 16 * 16
    print(f"norm_rotate {MANY[case]} neighbours {neighbours}", flush=True)
    g = torch.Generator().manual_seed(case)
    dtype = DTYPES[case % 2]
    x = (torch.randn(B, S, Hq + 2 * Hk, D, generator=g) * 3).to(dtype).to(DEV)
    q, k = x[:, :, :Hq], x[:, :, Hq:Hq + Hk] if Hk else None
    w = (1 + 0.3 * torch.randn(D, generator=g)).to(DEV)
    cos = sin = positions = None
    if R:
        cos, sin = qknorm.angles(max(S, 50), R // 2)
        if case % 2:
            positions = torch.randint(0, 50, (B, S), generator=g).int().to(DEV)
            positions[-1, -1] = 2 ** 30          # (no such row: NaN, in its own rows only)
    want_nan = positions is not None
    got = qknorm.norm_rotate(q, k, w, w if Hk else None, cos, sin, positions, 1e-6, neighbours)
    if not Hk:
        got = (got,)
    host = [None if t is None else t.cpu() for t in (cos, sin, positions)]
    for name, t, y in zip("qk", (q, k), got):
        want, tol = sv.norm_rotate(t.cpu(), w.cpu(), *host, 1e-6, neighbours)
        assert want.isnan().any() == want_nan
        close(y, want, tol, name)
    # over the rows themselves
    again = qknorm.norm_rotate(q, k, w, w if Hk else None, cos, sin, positions, 1e-6, neighbours,
                               out=(q, k) if Hk else q)
    for one, two in zip(got, again if Hk else (again,)):
        assert torch.equal(one.nan_to_num(7.0), two.nan_to_num(7.0))


@pytest.mark.parametrize("dtype", DTYPES)
def test_flat_rows_one_tensor_and_no_weight(dtype):
    q = torch.randn(7, 4, 64, device=DEV).to(dtype)
    cos, sin = qknorm.angles(7, 32)
    got = qknorm.norm_rotate(q, cos=cos, sin=sin)
    want, tol = sv.norm_rotate(q.cpu()[None], None, cos.cpu(), sin.cpu(), None, 1e-6, False)
    close(got, want[0], tol[0])
    out = torch.empty(7, 4, 64, device=DEV, dtype=dtype)
    assert qknorm.norm_rotate(q, cos=cos, sin=sin, out=out) is not None
    assert torch.equal(out, got)
    assert qknorm.norm_rotate(q[:0], q[:0])[0].shape == (0, 4, 64)


@pytest.mark.parametrize("dtype", DTYPES)
def test_in_place_in_one_projection(dtype):
    """q' and k' over q and k, in the buffer that also holds v."""
    x = torch.randn(2, 19, 5 + 2 * 2, 128, device=DEV).to(dtype)
    q, k, v = x[:, :, :5], x[:, :, 5:7], x[:, :, 7:].clone()
    cos, sin = qknorm.angles(19, 64)
    want = qknorm.norm_rotate(q, k, None, None, cos, sin)
    got = qknorm.norm_rotate(q, k, None, None, cos, sin, out=(q, k))
    assert got[0].data_ptr() == q.data_ptr()
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(x[:, :, 7:], v)


def test_special_values():
    """Zeros, rows of one large number, numbers whose squares leave fp32, infinities and NaN."""
    x = torch.randn(1, 8, 1, 64).bfloat16()
    x[0, 0] = 0
    x[0, 1, 0, 5] = 1e30
    x[0, 2] = 3e38
    x[0, 3] = 1e-30
    x[0, 4, 0, 3] = math.inf
    x[0, 5, 0, 63] = math.nan
    x[0, 6] *= 1e25
    cos, sin = qknorm.angles(8, 32)
    for near in (False, True):
        got = qknorm.norm_rotate(x.to(DEV), cos=cos, sin=sin, neighbours=near)
        want, tol = sv.norm_rotate(x, None, cos.cpu(), sin.cpu(), None, 1e-6, near)
        close(got, want, tol)


def test_positions_outside_the_table_and_far_ones():
    cos, sin = qknorm.angles(100000, 16)
    pos = torch.tensor([99999, -1, 100000, 0, 2 ** 31 - 1, -2 ** 31, 65535], device=DEV).int()
    q = torch.randn(7, 2, 64, device=DEV).half()
    got = qknorm.norm_rotate(q, cos=cos, sin=sin, positions=pos)
    want, tol = sv.norm_rotate(q.cpu()[None], None, cos.cpu(), sin.cpu(), pos.cpu()[None], 1e-6, False)
    close(got, want[0], tol[0])
    assert got[1, :, :32].isnan().all() and not got[1, :, 32:].isnan().any()


def test_strides():
    """Rows that are copied (not 16-byte aligned), broadcast rows, rows of angles further apart."""
    base = torch.randn(2, 6, 3, 200, device=DEV).half()
    q, k = base[..., 3:67], base[:, :1, :1, 64:128].expand(2, 6, 2, 64)
    cos, sin = qknorm.angles(6, 40)
    cos, sin = cos[:, 4:36], sin[:, 4:36]
    pos = torch.arange(6, device=DEV).int().expand(2, 6)
    got = qknorm.norm_rotate(q, k, None, None, cos, sin, pos)
    check(q, k, None, None, cos, sin, pos, 1e-6, False, got)


def test_refuses():
    q = torch.zeros(2, 5, 3, 64, device=DEV).half()
    cos, sin = qknorm.angles(5, 32)
    w = torch.ones(64, device=DEV)
    ok = dict(q=q, k=q.clone(), q_weight=w, k_weight=w, cos=cos, sin=sin)
    wide = torch.zeros(2, 5, 7, 64, device=DEV).half()
    for bad in (dict(q=q.float()), dict(q=q.cpu()), dict(q=q[0, 0]), dict(k=q.bfloat16()),
                dict(k=q[:1]), dict(k=q[..., :32]), dict(q_weight=w[:32]), dict(k_weight=w.double()),
                dict(cos=cos[:4], sin=sin[:4]), dict(sin=None), dict(cos=cos[:, :8]),
                dict(cos=cos.half(), sin=sin.half()), dict(cos=cos[:, :12], sin=sin[:, :12]),
                dict(positions=torch.zeros(2, 4, device=DEV).int()), dict(eps=-1.0),
                dict(positions=torch.zeros(2, 5, device=DEV).long()), dict(eps=math.nan),
                dict(cos=None, sin=None, positions=torch.zeros(2, 5, device=DEV).int()),
                dict(out=(q[:1], None)), dict(out=(None, q)), dict(k=None), dict(out=(q.float(), None)),
                dict(q=wide[:, :, :3], out=(wide[:, :, 1:4], None)),
                dict(k=wide[:, :, :3], out=(wide[:, :, 2:5], None)),
                dict(q=torch.zeros(2, 5, 3, 520, device=DEV).half()),
                dict(q=torch.zeros(2, 5, 3, 60, device=DEV).half())):
        with pytest.raises(RuntimeError):
            qknorm.norm_rotate(**(ok | bad))


def test_other_stream_and_graph():
    q = torch.randn(40, 8, 128, device=DEV).bfloat16()
    k = torch.randn(40, 2, 128, device=DEV).bfloat16()
    cos, sin = qknorm.angles(40, 64)
    want = qknorm.norm_rotate(q, k, None, None, cos, sin)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = qknorm.norm_rotate(q, k, None, None, cos, sin)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = qknorm.norm_rotate(q, k, None, None, cos, sin)
    for n in range(3):
        q.normal_()
        graph.replay()
        want = qknorm.norm_rotate(q, k, None, None, cos, sin)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), n


def test_with_attention():
    """As a diffusion transformer's block calls it: norm and rotation, then attention."""
    B, H, S, D = 1, 4, 333, 64
    x = torch.randn(B, S, 3 * H, D, device=DEV).half()
    wq, wk = (1 + 0.1 * torch.randn(D, device=DEV) for _ in range(2))
    cos, sin = qknorm.angles(S, D // 2)
    q, k = qknorm.norm_rotate(x[:, :, :H], x[:, :, H:2 * H], wq, wk, cos, sin, neighbours=True)
    v = x[:, :, 2 * H:]
    out = gfx906_amd.attn(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2), D ** -0.5)
    want = sdpa_math_fp32(*(t.transpose(1, 2).cpu() for t in (q, k, v)), D ** -0.5)
    # the attention's own bound, as everywhere (the norms are checked above)
    assert (out.float().cpu() - want).abs().max() <= 2e-3
