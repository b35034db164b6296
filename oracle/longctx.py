"""CPU oracle of the 4-bit cache and of sparse attention (test infrastructure only).

Plain loops in 64 bits over the definitions in ``include/gfx906_amd_attn.h``; nothing here comes from the kernels.
"""

from __future__ import annotations

import math

import torch

VALUES = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
Q_BLOCK = 128


# -- the format ---------------------------------------------------------------------------

def quantise(x):
    """(codes [..., D] as numbers 0..15, scale bytes [..., D/32]) of fp16/bf16 x."""
    x = x.double().unflatten(-1, (-1, 32))
    top = x.abs().amax(-1)
    bad = ~torch.isfinite(x).all(-1)
    e = torch.floor(torch.log2(top.clamp(min=2.0 ** -124))).nan_to_num(0.0, 0.0, 0.0) - 2
    byte = torch.where(bad, 255, (e + 127).int())
    a = (x.abs() / torch.exp2(e)[..., None]).nan_to_num(6.0, 6.0, 6.0).clamp(max=6.0)
    dist = (a[..., None] - VALUES).abs()
    near = dist == dist.amin(-1, keepdim=True)
    # the nearest code; of two equally near ones the even
    rank = torch.arange(8) + 8 * (torch.arange(8) % 2)
    code = torch.where(near, rank, 99).amin(-1) % 8
    code = code + 8 * torch.signbit(x).int()
    return code.flatten(-2), byte


def dequantise(codes, byte):
    """fp64 values of codes [..., D] and scale bytes [..., D/32]."""
    sign = torch.where(codes >= 8, -1.0, 1.0).double()
    scale = torch.where(byte == 255, math.nan, torch.exp2(byte.double() - 127))
    x = (sign * VALUES[(codes % 8).long()]).unflatten(-1, (-1, 32)) * scale[..., None]
    return x.flatten(-2)


def read_cache(codes, scales, page, token):
    """(codes [H, D], bytes [H, D/32]) of one token of a page."""
    c = codes[page, :, token].int()
    c = torch.stack((c & 15, c >> 4), -1).flatten(-2)
    return c, scales[page, :, token // 64, token % 16, :, token % 64 // 16].int()


def write_cache(codes, scales, page, token, c, byte):
    codes[page, :, token] = (c[..., 0::2] + 16 * c[..., 1::2]).to(torch.uint8)
    scales[page, :, token // 64, token % 16, :, token % 64 // 16] = byte.to(torch.uint8)


# -- pages and slots ----------------------------------------------------------------------

def plan_pages(lens, new_lens, table, free_pages, used, page, tokens):
    """(slots, cu, lens, used, missing, table) as lists of ints."""
    table = [list(r) for r in table]
    W = len(table[0]) if table else 0
    slots, cu, out, at, missing = [], [0], [], max(0, used), 0
    for b, (n, m) in enumerate(zip(lens, new_lens)):
        n, m = max(0, n), max(0, m)
        first, last = -(-n // page), -(-(n + m) // page)
        fresh = {}
        for k in range(first, last):
            got = free_pages[at] if k < W and at < len(free_pages) else None
            missing += got is None
            fresh[k] = -1 if got is None else got
            if k < W:
                table[b][k] = fresh[k]
            at += 1
        for p in range(n, n + m):
            k = p // page
            pg = fresh[k] if k in fresh else table[b][k] if k < W else -1
            slots.append(pg * page + p % page if 0 <= pg * page + p % page < 2 ** 31 and pg >= 0
                         else -1)
        cu.append(cu[-1] + m)
        out.append(n + m)
    slots = (slots + [-1] * tokens)[:tokens]
    return slots, cu, out, max(max(0, used), min(at, len(free_pages))), missing, table


# -- attention ----------------------------------------------------------------------------

def softmax_rows(q, k, v, scale, hide):
    """(o, weighted |v|, largest sum |q k| |scale|) in 64 bits; rows that see nothing
    are 0. hide: [rows, keys] bool."""
    q, k, v = q.double(), k.double(), v.double()
    z = (q @ k.T * scale).masked_fill(hide, -math.inf)
    top = z.amax(1, keepdim=True) if z.shape[1] else torch.full((len(q), 1), -math.inf)
    w = torch.exp(z - torch.where(top == -math.inf, torch.zeros_like(top, dtype=z.dtype), top))
    w = torch.where(hide, 0.0, w)
    l = w.sum(1, keepdim=True)
    inv = torch.where(l > 0, 1 / l, torch.zeros_like(l))
    inv = torch.where(torch.isnan(l), l, inv)
    # A key that a row does not see adds nothing to it, whatever the key holds.
    bad = ~torch.isfinite(v).all(1) & (~hide).any(0)
    used = torch.where((torch.isfinite(v).all(1) & (~hide).any(0))[:, None], v, torch.zeros_like(v))
    more = sum((torch.where(hide[:, j:j + 1], 0.0, w[:, j:j + 1] * v[j]) for j in bad.nonzero()),
               torch.zeros(()))
    size = ((q.abs() @ k.abs().T) * abs(scale)).masked_fill(hide, 0.0)
    size = size.nan_to_num(0.0, 0.0, 0.0).max().item() if z.numel() else 0.0
    return (w @ used + more) * inv, w @ used.abs() * inv, size


def tolerance(o, spread, size, dtype, D, keys, vmax):
    """Bound on the error of a correct kernel: the output's rounding (half an ulp),
    the rounding of every weight to the element type in numerator and denominator,
    fp32 scores (D products of total size `size`, added in fp32) and exp2, and for
    fp16 weights and outputs below the smallest normal number."""
    eps = torch.finfo(dtype).eps
    tol = eps / 2 * o.abs() + spread * (eps + 2 * (D * 2.0 ** -24 * size + 2.0 ** -21))
    if dtype == torch.float16:
        tol = tol + keys * 2.0 ** -25 * vmax + 2.0 ** -25
    return tol + 1e-30


def cache_attn(q, cache, page, table, lens, scale, cu=None, max_q=None, causal=True):
    """{row: (o [Hq, D], tolerance)} of every computed row, all on the CPU."""
    codes_k, scales_k, codes_v, scales_v = cache
    pages, Hkv, _, half = codes_k.shape
    T, Hq, D = q.shape
    G = Hq // Hkv
    cu = list(range(len(lens) + 1)) if cu is None else [min(max(c, 0), T) for c in cu]
    W = table.shape[1]
    rows = {}
    for b, n in enumerate(lens):
        n, m = max(0, n), max(0, cu[b + 1] - cu[b])
        keys, ks, vs = [], [], []
        for t in range(min(n, W * page)):
            pg = table[b, t // page].item()
            if 0 <= pg < pages:
                keys.append(t)
                ks.append(dequantise(*read_cache(codes_k, scales_k, pg, t % page)))
                vs.append(dequantise(*read_cache(codes_v, scales_v, pg, t % page)))
        pos = torch.tensor(keys)
        k = torch.stack(ks) if ks else torch.zeros(0, Hkv, D, dtype=torch.float64)
        v = torch.stack(vs) if vs else torch.zeros(0, Hkv, D, dtype=torch.float64)
        m = m if max_q is None else min(m, max_q)
        if m == 0:
            continue
        n_all = max(0, cu[b + 1] - cu[b])
        at = torch.arange(m)[:, None] + n - n_all
        hide = (pos[None] > at) if causal else torch.zeros(m, len(keys), dtype=torch.bool)
        hide = hide.expand(m, len(keys))
        got = [softmax_rows(q[cu[b]:cu[b] + m, h], k[:, h // G], v[:, h // G], scale, hide)
               for h in range(Hq)]
        vmax = v.nan_to_num(0.0).abs().max().item() if len(keys) else 0.0
        for r in range(m):
            o = torch.stack([g[0][r] for g in got])
            tol = torch.stack([tolerance(g[0][r], g[1][r], g[2], q.dtype, D, len(keys), vmax)
                               for g in got])
            rows[cu[b] + r] = (o, tol)
    return rows


# -- sparse attention ---------------------------------------------------------------------

def block_means(x, block):
    return torch.stack([x[:, :, r:r + block].double().mean(2).float()
                        for r in range(0, x.shape[2], block)], 2)


def select(q_means, k_means, count, q_len, k_len, block, causal):
    B, Hq, nq, _ = q_means.shape
    G, nk = Hq // k_means.shape[1], k_means.shape[2]
    index = torch.full((B, Hq, nq, count), -1, dtype=torch.int32)
    for b in range(B):
        for h in range(Hq):
            # (one sum a block, all in the same order: a matrix product may add up two
            # equal columns differently, and equal blocks must have equal scores)
            km = k_means[b, h // G].double()
            score = torch.stack([(x.double() * km).sum(1) for x in q_means[b, h]])
            for i in range(nq):
                lo = i * Q_BLOCK + k_len - q_len
                hi = min(q_len, (i + 1) * Q_BLOCK) - 1 + k_len - q_len
                seen = (hi // block + 1 if hi >= 0 else 0) if causal else nk
                own = min(seen, max(lo, 0) // block) if causal else nk
                key = [(j < own, -math.inf if math.isnan(s) else -s if j < own else 0.0, j)
                       for j, s in enumerate(score[i, :seen].tolist())]
                mine = sorted(j for _, _, j in sorted(key)[:count])
                index[b, h, i, :len(mine)] = torch.tensor(mine, dtype=torch.int32)
    return index


def sparse_attn(q, k, v, scale, index, block, causal):
    """(o, tolerance) in 64 bits."""
    B, Hq, Sq, D = q.shape
    G, Skv = Hq // k.shape[1], k.shape[2]
    nk = -(-Skv // block)
    o, tol = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for b in range(B):
        for h in range(Hq):
            for i in range(index.shape[2]):
                r0, r1 = i * Q_BLOCK, min(Sq, (i + 1) * Q_BLOCK)
                last, keys = -1, []
                for j in index[b, h, i].tolist():
                    if last < j < nk:
                        last = j
                        keys += range(j * block, min(Skv, (j + 1) * block))
                at = torch.tensor(keys, dtype=torch.long)
                kk, vv = k[b, h // G][at], v[b, h // G][at]
                pos = torch.arange(r0, r1)[:, None] + Skv - Sq
                hide = at[None] > pos if causal else torch.zeros(r1 - r0, len(at), dtype=torch.bool)
                oo, spread, size = softmax_rows(q[b, h, r0:r1], kk, vv, scale, hide)
                vmax = vv.double().nan_to_num(0.0, 0.0, 0.0).abs().max().item() if keys else 0.0
                o[b, h, r0:r1] = oo
                tol[b, h, r0:r1] = tolerance(oo, spread, size, q.dtype, D, len(at), vmax)
    return o, tol
