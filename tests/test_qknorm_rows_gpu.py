"""Norms of queries and keys on the GPU: rows at the ends of their types' ranges, and layouts of rows that
need no copy or get their results elsewhere."""

import math

import pytest
import torch

from gfx906_amd import qknorm

pytestmark = pytest.mark.gpu
DEV = "cuda"


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
