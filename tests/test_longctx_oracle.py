"""The CPU oracle of the 4-bit cache and of sparse attention against hand-made
examples and torch's own operations."""

import math

import torch

from oracle import longctx as oc


def test_format_examples():
    x = torch.tensor([0.0, 0.25, 0.26, 0.5, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 5.1, 6.0, 7.9, -0.75,
                      -6.0] + [0.0] * 17, dtype=torch.float16)
    code, byte = oc.quantise(x)
    assert byte.tolist() == [127]
    assert code[:15].tolist() == [0, 0, 1, 1, 2, 2, 4, 4, 6, 6, 7, 7, 7, 10, 15]
    vals = oc.dequantise(code, byte)
    assert vals[:15].tolist() == [0, 0, .5, .5, 1, 1, 2, 2, 4, 4, 6, 6, 6, -1, -6]
    code, byte = oc.quantise(torch.tensor([math.inf] + [1.0] * 31).half())
    assert byte.item() == 255 and oc.dequantise(code, byte).isnan().all()
    code, byte = oc.quantise(torch.zeros(32).half())
    assert byte.item() == 1 and code.eq(0).all()


def test_format_error_is_at_most_half_a_step_below_saturation():
    x = torch.randn(64, 128, generator=torch.Generator().manual_seed(0)).bfloat16()
    code, byte = oc.quantise(x)
    d = oc.dequantise(code, byte)
    unit = torch.exp2(byte.double() - 127).repeat_interleave(32, -1)
    a = x.double().abs() / unit
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    err = (d - x.double()).abs() / unit
    assert (err <= step / 2)[a <= 7].all() and a.max() < 8


def test_plan_example():
    slots, cu, lens, used, missing, table = oc.plan_pages(
        [0, 64, 70], [65, 1, 0], [[-1, -1], [5, -1], [6, 7]], [9, 8, 4], 0, 64, 70)
    assert slots == list(range(9 * 64, 10 * 64)) + [8 * 64] + [4 * 64] + [-1] * 4
    assert cu == [0, 65, 66, 66] and lens == [65, 65, 70] and used == 3 and missing == 0
    assert table == [[9, 8], [5, 4], [6, 7]]
    # the list ends after one page; the table's row after two
    slots, _, _, used, missing, table = oc.plan_pages([0, 100], [70, 100], [[-1, -1], [1, 2]], [9],
                                                      0, 64, 170)
    assert missing == 3 and used == 1 and table == [[9, -1], [1, 2]]
    assert slots[64:70] == [-1] * 6 and slots[70] == 2 * 64 + 36 and slots[98] == -1


def test_cache_attention_skips_bad_pages_and_empty_rows():
    g = torch.Generator().manual_seed(1)
    codes = torch.randint(0, 256, (3, 1, 64, 32), generator=g, dtype=torch.uint8)
    scales = torch.full((3, 1, 1, 16, 2, 4), 127, dtype=torch.uint8)
    q = torch.randn(3, 2, 64, generator=g).half()
    table = torch.tensor([[2, 99, 0], [-1, -1, -1], [1, -1, -1]], dtype=torch.int32)
    rows = oc.cache_attn(q, (codes, scales, codes, scales), 64, table, [190, 5, 0], 0.125)
    ref = [oc.dequantise(*oc.read_cache(codes, scales, p, t))[0]
           for p, n in ((2, 64), (0, 62)) for t in range(n)]
    ref = torch.stack(ref)
    w = torch.softmax(q[0].double() @ ref.T * 0.125, 1)
    assert torch.allclose(rows[0][0], w @ ref)
    assert rows[1][0].eq(0).all() and rows[2][0].eq(0).all()


def test_selection_examples():
    qm = torch.tensor([[[[1.0, 0.0]]]])
    km = torch.tensor([[[[1.0, 5.0], [3.0, 0.0], [3.0, 1.0], [-1.0, 0.0], [math.nan, 0.0]]]])
    assert oc.select(qm, km, 2, 100, 300, 64, False).tolist() == [[[[1, 4]]]]
    assert oc.select(qm, km, 3, 100, 300, 64, False).tolist() == [[[[1, 2, 4]]]]
    # causal, one query at position 200: block 3 is its own
    assert oc.select(qm, km[:, :, :4], 2, 1, 201, 64, True).tolist() == [[[[1, 3]]]]
    assert oc.select(qm, km[:, :, :1], 3, 1, 7, 64, True).tolist() == [[[[0, -1, -1]]]]


def test_sparse_attention_over_all_blocks_is_attention():
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(1, 2, 200, 64, generator=g).half() for _ in range(3))
    index = torch.arange(4, dtype=torch.int32).expand(1, 2, 2, 4)
    for causal in (False, True):
        o, _ = oc.sparse_attn(q, k, v, 0.125, index, 64, causal)
        z = q.double() @ k.double().transpose(2, 3) * 0.125
        if causal:
            z = z + torch.triu(torch.full((200, 200), -math.inf, dtype=torch.float64), 1)
        assert torch.allclose(o, torch.softmax(z, -1) @ v.double())
    # entries that repeat, fall back or name no block are passed over
    index = torch.tensor([2, 2, 1, 7, -1, 3], dtype=torch.int32).expand(1, 2, 2, 6)
    o, _ = oc.sparse_attn(q, k, v, 0.125, index, 64, False)
    z = q.double() @ k.double()[:, :, 128:].transpose(2, 3) * 0.125
    assert torch.allclose(o, torch.softmax(z, -1) @ v.double()[:, :, 128:])
