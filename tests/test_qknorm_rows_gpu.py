"""Norms of queries and keys on the GPU: rows at the ends of their types' ranges, and layouts of rows that
need no copy or get their results elsewhere."""

import math

import pytest
import torch

from gfx906_amd import qknorm
from oracle import serving as sv

pytestmark = pytest.mark.gpu
DEV = "cuda"


def close(got, want, tol):
    got = got.double().cpu()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.isinf(), want.isinf())
    worst = ((got - want).abs() / tol)[torch.isfinite(want)].max().item()
    print(f"  worst {worst:.3f} of the bound", flush=True)
    assert worst <= 1.0


@pytest.mark.parametrize("D", [8, 64, 128, 504])
@pytest.mark.parametrize("odd", [0.0, math.inf, 3e38])
def test_a_row_s_result_does_not_depend_on_others(odd, D):
    """Zeros, infinities and squares past fp32 in some rows leave the bits of the others as they are."""
    dtype = torch.float16 if odd == 0 else torch.bfloat16
    x = torch.randn(40000, 3, D, device=DEV, generator=torch.Generator(DEV).manual_seed(D)).to(dtype)
    want = qknorm.norm_rotate(x, eps=0.0)
    y = x.clone()
    y[::3, 1] = odd
    got = qknorm.norm_rotate(y, eps=0.0)
    others = torch.ones(40000, 3, dtype=torch.bool, device=DEV)
    others[::3, 1] = False
    assert torch.equal(got[others], want[others])


@pytest.mark.parametrize("size", [1e-38, 1e-30, 1e-25, 1e-20, 1e-16, 1e-15, 1e-10])
@pytest.mark.parametrize("eps", [0.0, 1e-45, 1e-38])
def test_small_rows(eps, size):
    """Rows whose squares are below fp32's range, or have few bits there; of fp32's smallest numbers too."""
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(1, 50, 2, 128, generator=g) * size).bfloat16()
    x[0, 3, 0] = 0
    x[0, 4, 1] = 0
    x[0, 4, 1, 100] = 2.0 ** -133
    x[0, 5, 0, :100] = 0
    got = qknorm.norm_rotate(x.to(DEV), eps=eps)
    want, tol = sv.norm_rotate(x, None, None, None, None, torch.tensor(eps).float().item(), False)
    close(got, want, tol)


@pytest.mark.parametrize("eps", [0.0, 1e30, 3e38])
def test_large_rows_and_large_eps(eps):
    """Sums past fp32 that eps has a share in."""
    x = torch.randn(1, 9, 2, 64, generator=torch.Generator().manual_seed(2))
    x = (x * torch.logspace(10, 30, 9)[None, :, None, None]).bfloat16()
    got = qknorm.norm_rotate(x.to(DEV), eps=eps)
    want, tol = sv.norm_rotate(x, None, None, None, None, torch.tensor(eps).float().item(), False)
    close(got, want, tol)


@pytest.mark.parametrize("tokens", [5, 3000])
@pytest.mark.parametrize("flat", [False, True])
def test_dense_rows_whose_dims_are_not_side_by_side(flat, tokens):
    """[.., D, heads] in memory: copied, as every such input; the results are contiguous."""
    g = torch.Generator(DEV).manual_seed(3)
    lead = (tokens,) if flat else (2, tokens)
    q, k = (torch.randn(*lead, 128, h, device=DEV, generator=g).half().transpose(-1, -2) for h in (6, 2))
    cos, sin = qknorm.angles(tokens, 64)
    got = qknorm.norm_rotate(q, k, cos=cos, sin=sin)
    want = qknorm.norm_rotate(q.contiguous(), k.contiguous(), cos=cos, sin=sin)
    for a, b, x in zip(got, want, (q, k)):
        assert a.shape == x.shape and a.stride(-1) == 1 and torch.equal(a, b)
    # heads last of all, batches between tokens
    one = torch.randn(tokens, 2, 64, 3, device=DEV, generator=g).half().permute(1, 0, 3, 2)
    assert torch.equal(qknorm.norm_rotate(one), qknorm.norm_rotate(one.contiguous()))


PLACES = {  # q and k of one buffer, by how it lies in memory
    "each head's q, k and v": lambda B, S, H, D: ((B, S, H, 3, D), lambda x: (x[..., 0, :], x[..., 1, :])),
    "each token's, heads first": lambda B, S, H, D: (
        (B, H, S, 3, D), lambda x: tuple(x[..., i, :].transpose(1, 2) for i in range(2))),
    "each batch's": lambda B, S, H, D: ((B, 3, S, H, D), lambda x: (x[:, 0], x[:, 1])),
    "whole tensors": lambda B, S, H, D: ((3, B, S, H, D), lambda x: (x[0], x[1])),
    "each token's": lambda B, S, H, D: ((B, S, 3, H, D), lambda x: (x[:, :, 0], x[:, :, 1])),
}


@pytest.mark.parametrize("B", [1, 2])
@pytest.mark.parametrize("place", PLACES)
def test_over_themselves_wherever_they_lie(place, B):
    """q' and k' over q and k, however those share a buffer; the rest of it stays."""
    S, H, D = 37, 5, 64
    shape, parts = PLACES[place](B, S, H, D)
    x = torch.randn(*shape, device=DEV, generator=torch.Generator(DEV).manual_seed(4)).half()
    q, k = parts(x)
    cos, sin = qknorm.angles(S, D // 2)
    want = qknorm.norm_rotate(q, k, cos=cos, sin=sin)
    y = x.clone()
    for t, w in zip(parts(y), want):
        t.copy_(w)
    qknorm.norm_rotate(q, k, cos=cos, sin=sin, out=(q, k))
    assert torch.equal(x, y)
    # over parts that are not their own, or each other's
    for out in ((k, q), (q, q), (k, None)):
        with pytest.raises(RuntimeError):
            qknorm.norm_rotate(q, k, cos=cos, sin=sin, out=out)
