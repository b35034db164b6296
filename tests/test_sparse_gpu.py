"""Sparse attention on the GPU against the CPU oracle in 64 bits: block means, the
choice of blocks, attention over them, and a run of them together."""

import math

import pytest
import torch

from gfx906_amd import sparse
from oracle import longctx as oc

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float16, torch.bfloat16]


def rand(*shape, seed=0, dtype=torch.float16, gain=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * gain).to(dtype)


def check(out, o, tol):
    out = out.double().cpu()
    assert torch.equal(out.isnan(), o.isnan())
    err = ((out - o).abs() / tol)[~o.isnan()]
    worst = err.max().item() if err.numel() else 0.0
    print(f"  worst {worst:.3f} of the bound", flush=True)
    assert worst <= 1.0


# -- means --------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,H,S,D,block", [(1, 1, 1, 64, 64), (2, 3, 64, 128, 64),
                                           (1, 2, 333, 64, 128), (2, 1, 1000, 128, 128)])
def test_means_are_exact(B, H, S, D, block, dtype):
    x = rand(B, H, S, D, seed=S, dtype=dtype, gain=3.0)
    x[0, 0, S // 2] *= 2.0 ** -9
    got = sparse.block_means(x.to(DEV), block)
    assert torch.equal(got.cpu(), oc.block_means(x, block))
    wide = torch.zeros(B, S, H, D + 8, dtype=dtype, device=DEV)
    wide[..., :D] = x.to(DEV).transpose(1, 2)
    assert torch.equal(sparse.block_means(wide[..., :D].transpose(1, 2), block), got)
    odd = torch.zeros(B, H, S, D + 1, dtype=dtype, device=DEV)   # copied
    odd[..., 1:] = x.to(DEV)
    assert torch.equal(sparse.block_means(odd[..., 1:], block), got)


def test_means_of_special_values_and_nothing():
    x = torch.zeros(1, 1, 200, 64).half()
    x[0, 0, 3, 0], x[0, 0, 70, 1], x[0, 0, 140, 2], x[0, 0, 150, 2] = (math.inf, math.nan, math.inf,
                                                                       -math.inf)
    m = sparse.block_means(x.to(DEV), 64).cpu()[0, 0]
    assert m[0, 0] == math.inf and m[1, 1].isnan() and m[2, 2].isnan() and m[3].eq(0).all()
    assert sparse.block_means(x[:, :, :0].to(DEV), 64).shape == (1, 1, 0, 64)


# -- choice -------------------------------------------------------------------------------

SELECTS = [  # B, Hq, Hkv, Sq, Skv, D, block, count
    (1, 1, 1, 1, 1, 64, 64, 3), (2, 4, 2, 300, 300, 64, 64, 3), (1, 2, 2, 128, 1000, 128, 128, 5),
    (1, 2, 1, 200, 50, 64, 64, 4), (1, 6, 2, 1, 20000, 128, 64, 40), (1, 1, 1, 700, 700, 64, 128, 64),
    (1, 1, 1, 3, 40000, 64, 64, 600), (2, 2, 1, 257, 1290, 128, 64, 7),
    (1, 1, 1, 130, 330000, 64, 64, 33), (1, 1, 1, 1, 70000, 64, 64, 2000),
    (1, 1, 1, 1, 2000000, 64, 64, 1500), (1, 3, 1, 1400, 1400, 128, 64, 9),
]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("case", range(len(SELECTS)))
def test_choice(case, causal):
    B, Hq, Hkv, Sq, Skv, D, block, count = SELECTS[case]
    print(f"select {case} causal {causal}", flush=True)
    g = torch.Generator().manual_seed(case)
    nq, nk = -(-Sq // 128), -(-Skv // block)
    qm = torch.randn(B, Hq, nq, D, generator=g)
    km = torch.randn(B, Hkv, nk, D, generator=g)
    if nk > 4:       # equal scores: the lower index
        km[0, 0, nk // 2] = km[0, 0, 1]
        km[0, 0, nk - 1] = km[0, 0, 1]
        km[-1, -1, 2:4] = 0
    got = sparse.select(qm.to(DEV), km.to(DEV), count, Sq, Skv, block, causal)
    assert torch.equal(got.cpu(), oc.select(qm, km, count, Sq, Skv, block, causal))


@pytest.mark.parametrize("count", [3, 9, 64])
def test_choice_among_equal_and_special_scores(count):
    """Many equal scores, zeros of both signs, infinities and NaN."""
    D, nk = 64, 500
    qm = torch.zeros(1, 1, 3, D)
    qm[..., 0] = 1
    km = torch.zeros(1, 1, nk, D)
    km[0, 0, :, 0] = torch.randint(-2, 3, (nk,), generator=torch.Generator().manual_seed(1)).float()
    km[0, 0, 7, 0], km[0, 0, 100, 0], km[0, 0, 450, 0], km[0, 0, 451, 0] = (
        -0.0, math.nan, math.inf, -math.inf)
    for causal in (False, True):
        got = sparse.select(qm.to(DEV), km.to(DEV), count, 384, nk * 64, 64, causal)
        assert torch.equal(got.cpu(), oc.select(qm, km, count, 384, nk * 64, 64, causal))
    same = torch.ones(1, 1, nk, D)
    got = sparse.select(qm.to(DEV), same.to(DEV), count, 384, nk * 64, 64, False)
    assert got[0, 0].tolist() == [list(range(count))] * 3


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,Hq,Hkv,Sq,Skv,D,block,count,causal", [
    (1, 1, 1, 1, 1, 64, 64, 2, False), (2, 6, 2, 1, 30000, 128, 64, 40, True),
    (1, 4, 1, 128, 9000, 64, 128, 5, True), (1, 2, 2, 77, 50, 128, 64, 4, True),
    (1, 2, 1, 100, 70000, 64, 64, 300, False), (1, 1, 1, 3, 262144, 64, 64, 7, True),
    (1, 1, 1, 3, 262145, 64, 64, 7, True), (2, 2, 1, 129, 3000, 128, 64, 9, True),
    (1, 2, 2, 500, 0, 64, 64, 3, False), (1, 2, 2, 5, 0, 64, 64, 3, True),
    (1, 4, 2, 6000, 6000, 64, 128, 9, True), (1, 1, 1, 40000, 70000, 128, 64, 5, False)])
def test_choice_from_rows(B, Hq, Hkv, Sq, Skv, D, block, count, causal, dtype):
    """In one kernel and in several, with equal scores among them."""
    q = rand(B, Sq, Hq, D, seed=Sq, dtype=dtype).transpose(1, 2)
    nk = -(-Skv // block)
    km = torch.randn(B, Hkv, nk, D, generator=torch.Generator().manual_seed(nk))
    if nk > 4:
        km[0, 0, nk // 2] = km[0, 0, nk - 1] = km[0, 0, 1]
    got = sparse.choose(q.to(DEV), km.to(DEV), count, Skv, block, causal)
    want = oc.select(oc.block_means(q, 128), km, count, Sq, Skv, block, causal)
    assert torch.equal(got.cpu(), want)
    assert torch.equal(got, sparse.select(sparse.block_means(q.to(DEV), 128), km.to(DEV), count, Sq,
                                          Skv, block, causal))


def test_choice_from_rows_refuses():
    q, km = rand(1, 4, 9, 64).to(DEV), torch.zeros(1, 2, 5, 64, device=DEV)
    a = dict(q=q, k_means=km, count=4, k_len=300)
    for kw in (dict(q=q.float()), dict(k_means=km.half()), dict(k_len=200), dict(count=0),
               dict(k_means=km[:, :, :, :32]), dict(q=q[:, :3]), dict(block=32), dict(k_len=-1),
               dict(k_means=km.cpu()), dict(q=q[0]), dict(causal=True, count=0)):
        with pytest.raises(RuntimeError):
            sparse.choose(**(a | kw))


def test_choice_refuses():
    qm, km = torch.zeros(1, 2, 2, 64, device=DEV), torch.zeros(1, 2, 4, 64, device=DEV)
    a = dict(q_means=qm, k_means=km, count=4, q_len=200, k_len=256)
    for kw in (dict(count=0), dict(count=4000), dict(q_len=300), dict(k_len=100), dict(block=32),
               dict(q_means=qm.half()), dict(k_means=km[:, :, :, :32]), dict(q_means=qm[0]),
               dict(q_means=qm.cpu()), dict(k_means=km.cpu()), dict(causal=True, count=2),
               dict(k_means=torch.zeros(1, 3, 4, 64, device=DEV)),
               dict(q_means=qm[..., :32], k_means=km[..., :32])):
        with pytest.raises(RuntimeError):
            sparse.select(**(a | kw))


# -- attention ----------------------------------------------------------------------------

def random_index(B, Hq, nq, nk, count, seed, fill=0.0):
    g = torch.Generator().manual_seed(seed)
    index = torch.full((B, Hq, nq, count), -1, dtype=torch.int32)
    for row in index.view(-1, count):
        n = min(count, nk)
        if fill:
            n = max(0, n - int(torch.rand(1, generator=g).item() * fill * n))
        row[:n] = torch.randperm(nk, generator=g)[:n].sort()[0]
    return index


ATTNS = [  # B, Hq, Hkv, Sq, Skv, D, block, count
    (1, 1, 1, 1, 1, 64, 64, 1), (1, 2, 1, 1, 700, 128, 64, 4), (2, 3, 3, 128, 128, 64, 128, 1),
    (1, 4, 2, 300, 300, 128, 64, 3), (2, 2, 2, 129, 1000, 64, 64, 9), (1, 2, 2, 200, 50, 128, 64, 2),
    (1, 6, 2, 3, 5000, 64, 128, 20), (1, 1, 1, 1000, 1000, 128, 128, 5),
    (1, 2, 1, 513, 777, 64, 64, 13), (1, 8, 8, 260, 520, 128, 64, 2),
    (1, 1, 1, 127, 9000, 128, 64, 100),
]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", range(len(ATTNS)))
def test_attention_over_blocks(case, dtype, causal):
    B, Hq, Hkv, Sq, Skv, D, block, count = ATTNS[case]
    print(f"sparse {case} {dtype} causal {causal}", flush=True)
    q = rand(B, Hq, Sq, D, seed=case, dtype=dtype, gain=2.0)
    k, v = (rand(B, Hkv, Skv, D, seed=case + s, dtype=dtype) for s in (100, 200))
    index = random_index(B, Hq, -(-Sq // 128), -(-Skv // block), count, case, fill=0.5)
    out = sparse.attn_blocks(q.to(DEV), k.to(DEV), v.to(DEV), D ** -0.5, index.to(DEV), block, causal)
    check(out, *oc.sparse_attn(q, k, v, D ** -0.5, index, block, causal))


@pytest.mark.parametrize("Sq", [2, 200])
def test_lists_with_bad_entries(Sq):
    """Entries out of range, repeated or out of order, and lists that name nothing."""
    D, Skv = 64, 500
    q, k, v = rand(1, 4, Sq, D, seed=1), rand(1, 2, Skv, D, seed=2), rand(1, 2, Skv, D, seed=3)
    lists = [[2, 2, 1, 7, -1, 3, 8, 2 ** 31 - 1], [-1] * 8, [-2 ** 31, 5, 0, 5, 6, 6, 99, 7],
             [7, 6, 5, 4, 3, 2, 1, 0]]
    index = torch.tensor(lists, dtype=torch.int32)[None, :, None].repeat(1, 1, -(-Sq // 128), 1)
    for causal in (False, True):
        out = sparse.attn_blocks(q.to(DEV), k.to(DEV), v.to(DEV), 0.1, index.to(DEV), 64, causal)
        check(out, *oc.sparse_attn(q, k, v, 0.1, index, 64, causal))
        assert out[0, 1].eq(0).all()


@pytest.mark.parametrize("scale", [0.0, -0.3, 4.0])
@pytest.mark.parametrize("D", [64, 128])
def test_scales(scale, D):
    q, k, v = rand(1, 2, 150, D, seed=1), rand(1, 2, 300, D, seed=2), rand(1, 2, 300, D, seed=3)
    index = random_index(1, 2, 2, 5, 4, 1)
    out = sparse.attn_blocks(q.to(DEV), k.to(DEV), v.to(DEV), scale, index.to(DEV), 64)
    check(out, *oc.sparse_attn(q, k, v, scale, index, 64, False))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Sq", [1, 200])
def test_what_no_row_sees_changes_nothing(D, Sq):
    """NaN and infinite keys and values in blocks that are not listed, or behind a
    causal row; an infinite key a row does see is NaN or weight 0 as in softmax."""
    Skv = 448
    q, k, v = rand(1, 2, Sq, D, seed=1), rand(1, 2, Skv, D, seed=2), rand(1, 2, Skv, D, seed=3)
    index = torch.tensor([0, 2, 6], dtype=torch.int32).expand(1, 2, -(-Sq // 128), 3).contiguous()
    want = sparse.attn_blocks(q.to(DEV), k.to(DEV), v.to(DEV), 0.1, index.to(DEV), 64, True)
    k2, v2 = k.clone(), v.clone()
    k2[:, :, 64:128], v2[:, :, 64:128] = math.nan, math.inf
    k2[:, :, 192:384], v2[:, :, 192:384] = math.inf, math.nan
    got = sparse.attn_blocks(q.to(DEV), k2.to(DEV), v2.to(DEV), 0.1, index.to(DEV), 64, True)
    assert torch.equal(got, want)
    if Sq > 1:   # the last key is seen by the last row only
        k2[:, :, -1], v2[:, :, -1] = math.nan, math.nan
        got = sparse.attn_blocks(q.to(DEV), k2.to(DEV), v2.to(DEV), 0.1, index.to(DEV), 64, True)
        assert got[:, :, -1].isnan().all()
        check(got, *oc.sparse_attn(q, k2, v2, 0.1, index, 64, True))


def test_very_low_and_high_scores():
    """Scores that all lie far below 0, that differ by the type's range, or are -inf."""
    D, Sq, Skv = 128, 130, 256
    for dtype, big in ((torch.float16, 60000.0), (torch.bfloat16, 1e18)):
        q, k, v = rand(1, 1, Sq, D, dtype=dtype), rand(1, 1, Skv, D, seed=1, dtype=dtype), rand(
            1, 1, Skv, D, seed=2, dtype=dtype)
        q[..., 0], k[..., 0] = big, -big
        # One key above the others by 7e9 (2e36): scores that close together as those of
        # several such keys would be are equal in fp32, whose step at 3.6e9 is 256.
        k[0, 0, 70, 0] = big
        index = torch.arange(4, dtype=torch.int32).expand(1, 1, 2, 4).contiguous()
        out = sparse.attn_blocks(q.to(DEV), k.to(DEV), v.to(DEV), 1.0, index.to(DEV), 64)
        assert torch.equal(out.cpu()[0, 0], v[0, 0, 70].expand(Sq, D))   # one weight, exactly 1
    q = torch.ones(1, 1, 1, D).half()
    k = torch.full((1, 1, 64, D), -math.inf).half()
    k[0, 0, 5] = 1
    v = rand(1, 1, 64, D, seed=5)
    index = torch.zeros(1, 1, 1, 1, dtype=torch.int32)
    out = sparse.attn_blocks(q.to(DEV), k.to(DEV), v.to(DEV), 0.1, index.to(DEV), 64)
    assert torch.equal(out.cpu()[0, 0, 0], v[0, 0, 5])


def test_strided_tensors_and_outputs():
    B, S, H, D = 2, 200, 3, 64
    buf = rand(B, S, 3, H, D, seed=4).to(DEV)
    q, k, v = (buf[:, :, i].transpose(1, 2) for i in range(3))
    index = random_index(B, H, 2, 4, 3, 4)
    hold = torch.full((B, S, H, D + 4), 3.0, dtype=torch.float16, device=DEV)
    out = hold[..., :D].transpose(1, 2)
    assert sparse.attn_blocks(q, k, v, 0.1, index.to(DEV), out=out).data_ptr() == hold.data_ptr()
    check(out, *oc.sparse_attn(q.cpu(), k.cpu(), v.cpu(), 0.1, index, 64, False))
    assert hold[..., D:].eq(3.0).all()
    odd = torch.zeros(B, H, S, D + 1, dtype=torch.float16, device=DEV)
    odd[..., 1:] = q
    assert torch.equal(sparse.attn_blocks(odd[..., 1:], k, v, 0.1, index.to(DEV)), out)
    one = k[:1].expand(B, H, S, D)      # broadcast keys
    got = sparse.attn_blocks(q, one, v, 0.1, index.to(DEV))
    assert torch.equal(got, sparse.attn_blocks(q, one.contiguous(), v, 0.1, index.to(DEV)))
    q2 = q.contiguous()
    want = sparse.attn_blocks(q2, k, v, 0.1, index.to(DEV))
    sparse.attn_blocks(q2, k, v, 0.1, index.to(DEV), out=q2)   # in place
    assert torch.equal(q2, want)


@pytest.mark.parametrize("D,block", [(64, 64), (128, 128)])
@pytest.mark.parametrize("Sq", [1, 300])
def test_heads_of_more_than_2_gib(D, block, Sq):
    """Keys and values of [B, S, H, D] buffers whose heads span 2^31 bytes and more, against
    copies of the same rows."""
    S, row = 1100, 1 << 20
    buf = torch.zeros(S * row + 4 * D, dtype=torch.float16, device=DEV)
    k = buf.as_strided((1, 2, S, D), (0, D, row, 1))
    v = buf.as_strided((1, 2, S, D), (0, D, row, 1), 2 * D)
    k.copy_(rand(1, 2, S, D, seed=1).to(DEV))
    v.copy_(rand(1, 2, S, D, seed=2).to(DEV))
    q = rand(1, 4, Sq, D, seed=3).to(DEV)
    index = random_index(1, 4, -(-Sq // 128), -(-S // block), 6, 7).to(DEV)
    for causal in (False, True):
        got = sparse.attn_blocks(q, k, v, 0.1, index, block, causal)
        want = sparse.attn_blocks(q, k.contiguous(), v.contiguous(), 0.1, index, block, causal)
        assert torch.equal(got, want)


def test_overlapping_rows_are_copied():
    buf = rand(1, 1, 1, 9000, seed=1).to(DEV).view(-1)
    k = buf.as_strided((1, 2, 200, 64), (0, 4096, 8, 1))     # rows 8 elements apart
    q = rand(1, 2, 200, 64, seed=2).to(DEV)
    index = random_index(1, 2, 2, 4, 2, 7).to(DEV)
    want = sparse.attn_blocks(q, k.contiguous(), k.contiguous(), 0.1, index)
    assert torch.equal(sparse.attn_blocks(q, k, k, 0.1, index), want)


def test_means_kept_for_other_heads_are_refused():
    q, k = rand(1, 4, 9, 64).to(DEV), rand(1, 2, 300, 64).to(DEV)
    means = sparse.block_means(k.repeat_interleave(2, 1), 64)
    with pytest.raises(ValueError):
        sparse.attn(q, k, k, 0.1, 3, k_means=means)
    with pytest.raises(RuntimeError):
        sparse.attn(q, k, k, 0.1, 3, block=128, k_means=sparse.block_means(k, 64))


def test_attention_refuses():
    q, k = torch.zeros(1, 4, 130, 64, device=DEV).half(), torch.zeros(1, 2, 70, 64, device=DEV).half()
    ix = torch.zeros(1, 4, 2, 2, dtype=torch.int32, device=DEV)
    a = dict(q=q, k=k, v=k, scale=0.1, index=ix)
    for kw in (dict(q=q.float()), dict(k=k.bfloat16()), dict(v=k[:, :, :60]), dict(q=q[:, :3]),
               dict(index=ix.long()), dict(index=ix[:, :, :1]), dict(index=ix[:, :3]),
               dict(index=ix[..., :0]), dict(index=ix.cpu()), dict(block=256), dict(q=q[..., :32]),
               dict(out=q.bfloat16()), dict(out=q[:, :, :5]), dict(scale=math.nan), dict(q=q[0]),
               dict(out=torch.zeros(1, 1, 130, 64, device=DEV).half().expand(1, 4, 130, 64))):
        with pytest.raises(RuntimeError):
            sparse.attn_blocks(**(a | kw))
    x = torch.zeros(1, 1, 300, 64, device=DEV).half()
    with pytest.raises(RuntimeError):
        sparse.attn_blocks(x[:, :, :64], x[:, :, 64:128], x[:, :, 128:192], 0.1, ix[:, :1, :1],
                           out=x[:, :, 100:164])


def test_no_keys_and_no_queries():
    q, k = rand(1, 2, 130, 64).to(DEV), rand(1, 1, 0, 64).to(DEV)
    ix = torch.zeros(1, 2, 2, 1, dtype=torch.int32, device=DEV)
    assert sparse.attn_blocks(q, k, k, 0.1, ix).eq(0).all()
    out, index = sparse.attn(q, k, k, 0.1, 4)
    assert out.eq(0).all() and index.eq(-1).all()
    out, index = sparse.attn(q[:, :, :0], q, q, 0.1, 4)
    assert out.shape == (1, 2, 0, 64) and index.shape == (1, 2, 0, 4)


# -- together -----------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,Hq,Hkv,Sq,Skv,D,block,count,causal", [
    (1, 4, 2, 700, 700, 128, 64, 4, True), (2, 2, 2, 300, 1100, 64, 128, 3, False),
    (1, 8, 2, 1, 5000, 128, 64, 16, True), (1, 2, 2, 100, 64, 64, 64, 5, False),
    (1, 2, 1, 300, 100, 64, 64, 5, True)])
def test_choice_and_attention(B, Hq, Hkv, Sq, Skv, D, block, count, causal, dtype):
    q = rand(B, Hq, Sq, D, seed=1, dtype=dtype)
    k, v = (rand(B, Hkv, Skv, D, seed=s, dtype=dtype) for s in (2, 3))
    out, index = sparse.attn(q.to(DEV), k.to(DEV), v.to(DEV), D ** -0.5, count, block=block,
                             causal=causal)
    want = oc.select(oc.block_means(q, 128), oc.block_means(k, block), count, Sq, Skv, block, causal)
    assert torch.equal(index.cpu(), want)
    check(out, *oc.sparse_attn(q, k, v, D ** -0.5, want, block, causal))
    kept = sparse.block_means(k.to(DEV), block)
    out2, index2 = sparse.attn(q.to(DEV), k.to(DEV), v.to(DEV), D ** -0.5, count, block=block,
                               causal=causal, k_means=kept)
    assert torch.equal(out, out2) and torch.equal(index, index2)


def test_every_block_chosen_is_dense_attention():
    import gfx906_amd
    q, k, v = (rand(1, 4, 600, 128, seed=s).to(DEV) for s in (1, 2, 3))
    out, _ = sparse.attn(q, k, v, 0.09, 10)
    assert (out - gfx906_amd.attn(q, k, v, 0.09)).abs().max() < 2e-3


def test_captured_call_replays():
    g = torch.Generator(device=DEV).manual_seed(1)
    for Sq, Skv in ((1, 9000), (700, 700)):
        q = torch.randn(1, 4, Sq, 128, device=DEV, generator=g).half()
        k, v = (torch.randn(1, 2, Skv, 128, device=DEV, generator=g).half() for _ in range(2))
        out = torch.zeros_like(q)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            sparse.attn(q, k, v, 0.1, 8, causal=True, out=out)
        torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            _, index = sparse.attn(q, k, v, 0.1, 8, causal=True, out=out)
        for i in range(4):
            for t in (q, k, v):
                t.copy_(torch.randn(t.shape, device=DEV, generator=g).half())
            graph.replay()
            got, chosen = out.clone(), index.clone()
            torch.randn(1 << 18, device=DEV).sum().item()
            want, ref = sparse.attn(q, k, v, 0.1, 8, causal=True)
            assert torch.equal(got, want) and torch.equal(chosen, ref), f"replay {i}"


def test_two_streams_at_once():
    q = [rand(1, 4, 1, 64, seed=i).to(DEV) for i in range(6)]
    k, v = rand(1, 2, 9000, 64, seed=8).to(DEV), rand(1, 2, 9000, 64, seed=9).to(DEV)
    want = [sparse.attn(x, k, v, 0.1, 32, causal=True)[0] for x in q]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for i, x in enumerate(q):
        with torch.cuda.stream(streams[i % 3]):
            got.append(sparse.attn(x, k, v, 0.1, 32, causal=True)[0])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_offsets_past_32_bits():
    """Keys whose rows start past 2^32 bytes of the tensor."""
    D, S, H = 64, 1 << 22, 9
    k = torch.zeros(1, H, S, D, dtype=torch.float16, device=DEV)
    last = rand(1, 1, 640, D, seed=3).to(DEV)
    k[:, H - 1:, S - 640 - 64:S - 64] = last
    q = rand(1, H, 1, D, seed=4).to(DEV)
    n = S // 128
    index = torch.arange(n - 6, n, dtype=torch.int32, device=DEV).expand(1, H, 1, 6)
    got = sparse.attn_blocks(q, k, k, 0.3, index.contiguous(), block=128)
    near = k[:, H - 1:, S - 768:].contiguous()
    small = torch.arange(6, dtype=torch.int32, device=DEV).expand(1, 1, 1, 6).contiguous()
    want = sparse.attn_blocks(q[:, H - 1:], near, near, 0.3, small, block=128)
    # (the lists may be split differently: two fp32 sums of the same weights)
    assert torch.allclose(got[:, H - 1:].float(), want.float(), atol=1e-6, rtol=2 ** -9)


@pytest.mark.parametrize("Sq", [1, 200])
@pytest.mark.parametrize("scale", [0.0, 1e-37, -1e-37])
def test_small_scales_of_large_bf16_scores(scale, Sq):
    """Products up to 1e38: a scale of 0 weighs every key alike, one of 1e-37 gives scores of
    some units."""
    q, k, v = (rand(1, h, S, 64, seed=h + S, dtype=torch.bfloat16) for h, S in ((2, Sq), (1, 300), (2, 300)))
    q, k, v = q * 2.0 ** 60, k * 2.0 ** 60, v[:, :1]
    index = random_index(1, 2, -(-Sq // 128), 5, 4, 1)
    out = sparse.attn_blocks(q.to(DEV), k.to(DEV), v.to(DEV), scale, index.to(DEV), 64)
    check(out, *oc.sparse_attn(q, k, v, scale, index, 64, False))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
def test_the_choice_is_the_same_by_every_way(D, dtype):
    """Scores whose sums nearly cancel, and differ in the last bits by the order in which they
    are added: choose, select, and a query alone or in a batch take the same blocks."""
    g = torch.Generator().manual_seed(D)
    nk, count = 500, 40
    # Permutations of one set of terms over 50 octaves: equal sums, in no order alike in fp64.
    terms = torch.randn(D // 2, generator=g)
    terms *= torch.exp2(torch.randint(-50, 1, terms.shape, generator=g).float())
    terms = torch.cat((terms, -terms * (1 + 2.0 ** -20)))
    km = torch.stack([terms[torch.randperm(D, generator=g)] for _ in range(nk)])[None, None]
    q = torch.ones(1, 1, 1, D, dtype=dtype)
    alone = sparse.choose(q.to(DEV), km.to(DEV), count, nk * 64)
    picked = sparse.select(sparse.block_means(q.to(DEV), 128), km.to(DEV), count, 1, nk * 64)
    assert torch.equal(alone, picked)
    # (so many heads go through three kernels)
    many = sparse.choose(q.expand(1, 400, 1, D).contiguous().to(DEV), km.to(DEV), count, nk * 64)
    assert torch.equal(many, alone.expand(1, 400, 1, count))


@pytest.mark.parametrize("Sq", [1, 100, 128, 300])
@pytest.mark.parametrize("D", [64, 128])
def test_means_of_wide_bf16_rows_are_the_same_by_every_way(D, Sq):
    """bf16 rows over 80 octaves, most of which cancel: fp64 sums depend on their order, and the
    choice from the rows is that from block_means all the same."""
    g = torch.Generator().manual_seed(D + Sq)
    x = torch.randn(2, Sq, 1, D, generator=g)
    x *= torch.exp2(torch.randint(-40, 41, x.shape, generator=g).float())
    x[:, Sq // 2:Sq // 2 * 2] = -x[:, :Sq // 2].flip(1)
    q = x.transpose(1, 2).bfloat16()
    km = torch.randn(2, 1, 300, D, generator=g).to(DEV)
    means = sparse.block_means(q.to(DEV), 128)
    want = sparse.select(means, km, 20, Sq, 300 * 64)
    assert torch.equal(sparse.choose(q.to(DEV), km, 20, 300 * 64), want)
    many = sparse.choose(q.expand(2, 200, Sq, D).contiguous().to(DEV), km, 20, 300 * 64)
    assert torch.equal(many, want.expand(2, 200, -1, 20))
