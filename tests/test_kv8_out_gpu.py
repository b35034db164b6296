"""Results of attention over the 8-bit cache beside the queries in one buffer."""

import pytest
import torch

from gfx906_amd import kv8

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("place", ["heads", "tokens", "heads first", "tensors"])
@pytest.mark.parametrize("news", [1, 3, 150])
def test_out_beside_q(news, place):
    """q and out are other parts of every head, token or of the whole: neither is refused or written over."""
    g = torch.Generator(DEV).manual_seed(news)
    cache, table = kv8.new_cache(4, 64, 2, 64), torch.tensor([[3, 1, 2]], dtype=torch.int32, device=DEV)
    lens, cu = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([190], [0, news]))
    k, v = torch.randn(2, 190, 2, 64, device=DEV, generator=g).half()
    kv8.store(cache, k, v, table, lens, torch.tensor([0, 190], dtype=torch.int32, device=DEV))
    H = 8
    shape, part = {"heads": ((news, H, 2, 64), lambda x, i: x[:, :, i]),
                   "tokens": ((news, 2, H, 64), lambda x, i: x[:, i]),
                   "heads first": ((H, news, 2, 64), lambda x, i: x[:, :, i].transpose(0, 1)),
                   "tensors": ((2, news, H, 64), lambda x, i: x[i])}[place]
    x = torch.randn(*shape, device=DEV, generator=g).half()
    q = part(x, 0)
    want, kept = kv8.attn(q, cache, table, lens, 0.125, cu_q=cu), q.clone()
    got = kv8.attn(q, cache, table, lens, 0.125, cu_q=cu, out=part(x, 1))
    assert got.data_ptr() == part(x, 1).data_ptr()
    assert torch.equal(got, want) and torch.equal(q, kept)
    if news > 1:
        with pytest.raises(RuntimeError):
            kv8.attn(q[:-1], cache, table, lens, 0.125, cu_q=cu - (cu > 0).int(), out=q[1:])
