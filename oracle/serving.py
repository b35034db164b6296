"""CPU oracle of the serving operators (test infrastructure only): head norms with the
position rotation, the 8-bit cache, attention over it, weights of its blocks, eviction.

Plain loops in 64 bits over the definitions in ``include/gfx906_amd_attn.h``; nothing
here comes from the kernels.
"""

from __future__ import annotations

import math

import torch

from .longctx import softmax_rows, tolerance

BLOCK = 64
LOW, HIGH = -15, 7


# -- norms and rotation -------------------------------------------------------------------

def norm_rotate(x, weight, cos, sin, positions, eps, neighbours):
    """(y, bound) of rows x [B, S, H, D]; positions [B, S] or None. The bound: the result's
    rounding, and for the fp32 arithmetic 32 roundings of the numbers that a result is
    added up from (D <= 512 squares in 8 + 6 steps, root, quotient, products)."""
    dtype, D = x.dtype, x.shape[-1]
    x = x.double()
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    if weight is not None:
        y = y * weight.double()
    size = y.abs()
    R = 0 if cos is None else 2 * cos.shape[1]
    out = y.clone()
    for b in range(x.shape[0]):
        for s in range(x.shape[1] if R else 0):
            p = s if positions is None else int(positions[b, s])
            ok = 0 <= p < len(cos)
            c = cos[p].double() if ok else torch.full((R // 2,), math.nan).double()
            n = sin[p].double() if ok else c
            first = slice(0, R, 2) if neighbours else slice(0, R // 2)
            second = slice(1, R, 2) if neighbours else slice(R // 2, R)
            u, v = y[b, s, :, first], y[b, s, :, second]
            out[b, s, :, first], out[b, s, :, second] = u * c - v * n, u * n + v * c
            total = u.abs() * c.abs() + v.abs() * n.abs(), u.abs() * n.abs() + v.abs() * c.abs()
            size[b, s, :, first], size[b, s, :, second] = total
    tiny = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134
    return out, torch.finfo(dtype).eps / 2 * out.abs() + 33 * 2.0 ** -24 * size + tiny


# -- the format ---------------------------------------------------------------------------

def values():
    """fp64 values of the 256 codes."""
    out = []
    for c in range(256):
        e, m = c >> 3 & 15, c & 7
        a = m / 512 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        out.append(math.nan if c & 127 == 127 else -a if c & 128 else a)
    return torch.tensor(out, dtype=torch.float64)


def place(t):
    """Place of a block's token in a row of the values' codes."""
    return 16 * (t >> 2 & 3) + 8 * (t >> 5) + 4 * (t >> 4 & 1) + (t & 3)


def scale_for(rows):
    """Exponent of the scale that fp16/bf16 rows ask for by themselves."""
    a = rows.double().abs()
    a = a[torch.isfinite(a)]
    top = a.max().item() if a.numel() else 0.0
    e = LOW
    while e < HIGH and top > 448 * 2.0 ** e:
        e += 1
    return e


def round_codes(x):
    """Numbers in scales to the nearest code's value, ties to even, at most 448."""
    grid = values()[:127]
    a = x.abs().clamp(max=448)
    hi = torch.searchsorted(grid, a).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    up, down = grid[hi] - a, a - grid[lo]
    take = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    take = torch.where(grid[hi] == a, hi, take)
    return torch.copysign(grid[take], x)


class Cache:
    """What a cache should hold: values [pages, heads, page, D] fp64 and exponents."""

    def __init__(self, pages, page, heads, D):
        self.page = page
        self.x = [torch.zeros(pages, heads, page, D, dtype=torch.float64) for _ in range(2)]
        self.e = [torch.full((pages, heads, page // BLOCK), LOW) for _ in range(2)]
        self.begun = torch.zeros(pages, page // BLOCK, dtype=torch.bool)

    def store(self, k, v, table, lens, cu):
        T = len(k)
        for b, n in enumerate(lens):
            r0, r1 = (min(max(c, 0), T) for c in cu[b:b + 2])
            old = max(0, n) - max(0, r1 - r0)
            p = max(0, old)
            while p < n:
                j = p // BLOCK
                end = min(n, (j + 1) * BLOCK)
                col = p // self.page
                page = table[b][col] if col < len(table[b]) else -1
                if 0 <= page < len(self.x[0]):
                    part, t0 = j % (self.page // BLOCK), j * BLOCK % self.page
                    self.begun[page, part] |= p == j * BLOCK
                    rows = slice(r0 + p - old, r0 + end - old)
                    for x, e, new in ((self.x[0], self.e[0], k), (self.x[1], self.e[1], v)):
                        for h in range(x.shape[1]):
                            was = int(e[page, h, part]) if p > j * BLOCK else LOW
                            now = max(was, scale_for(new[rows, h]))
                            e[page, h, part] = now
                            held = x[page, h, t0:t0 + p - j * BLOCK]
                            u = 2.0 ** now
                            x[page, h, t0:t0 + p - j * BLOCK] = torch.where(
                                torch.isnan(held), held, round_codes(held / u) * u)
                            r = new[rows, h].double()
                            x[page, h, t0 + p - j * BLOCK:t0 + end - j * BLOCK] = torch.where(
                                torch.isfinite(r), round_codes(r / u) * u, math.nan)
                p = end

    def rows(self, table_row, n, h):
        """(k, v) of the first n tokens of a table's row, and which of them have a page."""
        k, v, ok = [], [], []
        for t in range(n):
            col = t // self.page
            page = table_row[col] if col < len(table_row) else -1
            good = 0 <= page < len(self.x[0])
            ok.append(good)
            for out, x in ((k, self.x[0]), (v, self.x[1])):
                out.append(x[page, h, t % self.page] if good else torch.zeros(x.shape[-1]).double())
        D = self.x[0].shape[-1]
        k, v = (torch.stack(r) if r else torch.zeros(0, D, dtype=torch.float64) for r in (k, v))
        return k, v, torch.tensor(ok, dtype=torch.bool)


def decode(codes, scales, is_v):
    """fp64 values [pages, heads, page, D] of a cache's tensors (on the CPU)."""
    x = values()[codes.long()]
    if is_v:
        x = x[..., [place(t) for t in range(BLOCK)]].transpose(3, 4)
    else:
        x = x.unflatten(2, (-1, BLOCK))
    return (x * scales.double()[..., None, None]).flatten(2, 3)


# -- attention ----------------------------------------------------------------------------

def attention(q, cache, table, lens, scale, cu=None, max_q=None, causal=True):
    """{row: (o [Hq, D], bound, lse [Hq], bound of lse)} of every computed row. The bound of o is
    the one of the 4-bit cache's attention. An lse is off by its scores' errors (D products added in
    fp32) and by 2^-21 of the exponentials and their sum, and of its own size: it is ln 2 times the sum
    of a maximum and a logarithm, so by 2^-23 (the logarithm, 1 ulp), 2^-24 (the sum), 2^-25 (ln 2) and
    2^-24 (the product) of numbers no larger than |lse| and the scores, 2.3 * 2^-23 in all."""
    T, Hq, D = q.shape
    cu = list(range(T + 1)) if cu is None else [min(max(c, 0), T) for c in cu]
    G, out = Hq // cache.x[0].shape[1], {}
    for b, n in enumerate(lens):
        n = max(0, n)
        m = max(0, cu[b + 1] - cu[b])
        count = m if max_q is None else min(m, max_q)
        keys = min(n, len(table[b]) * cache.page)
        if not count:
            continue
        res = torch.zeros(count, Hq, D, dtype=torch.float64)
        tol, lse, ltol = torch.zeros_like(res), torch.zeros(count, Hq).double(), torch.zeros(count, Hq).double()
        seen = torch.arange(count) + (n - m) + 1 if causal else torch.full((count,), keys)
        for h in range(Hq):
            k, v, ok = cache.rows(table[b], keys, h // G)
            hide = ~ok[None] | (torch.arange(keys)[None] >= seen[:, None])
            x = q[cu[b]:cu[b] + count, h]
            o, spread, size = softmax_rows(x, k, v, scale, hide)
            top = v.abs().nan_to_num(0.0).max().item() if keys else 0.0
            res[:, h] = o
            tol[:, h] = tolerance(o, spread, size, q.dtype, D, keys, top)
            z = (x.double() @ k.T * scale).masked_fill(hide, -math.inf)
            lse[:, h] = torch.logsumexp(z, 1) if keys else -math.inf
            own = lse[:, h].abs().nan_to_num(0.0, 0.0)
            ltol[:, h] = D * 2.0 ** -24 * size + 2.0 ** -21 * (1 + size + own)
        for i in range(count):
            out[cu[b] + i] = (res[i], tol[i], lse[i], ltol[i])
    return out


def weigh(weights, q, lse, cache, table, lens, scale, cu=None, max_q=None, causal=True):
    """(weights after the call, bound). A weight is exp of a score less the lse: off by the errors
    of both in fp32, and its sum by a rounding for every addition of a lane's or a wave's."""
    T, Hq, D = q.shape
    cu = list(range(T + 1)) if cu is None else [min(max(c, 0), T) for c in cu]
    Hkv = cache.x[0].shape[1]
    out = weights.double().clone()
    tol = out.abs() * 2.0 ** -24
    for b, n in enumerate(lens):
        n = max(0, n)
        m = max(0, cu[b + 1] - cu[b])
        count = m if max_q is None else min(m, max_q)
        keys = min(n, len(table[b]) * cache.page)
        seen = torch.arange(count) + (n - m) + 1 if causal else torch.full((count,), keys)
        for h in range(Hq if keys and count else 0):
            k, _, ok = cache.rows(table[b], keys, h * Hkv // Hq)
            hide = ~ok[None] | (torch.arange(keys)[None] >= seen[:, None])
            x, l = q[cu[b]:cu[b] + count, h].double(), lse[cu[b]:cu[b] + count, h].double()
            hide = hide | (l == -math.inf)[:, None]
            size = ((x.abs() @ k.abs().T) * abs(scale)).masked_fill(hide, 0).max().item()
            shift = l[torch.isfinite(l)].abs().max().item() if torch.isfinite(l).any() else 0.0
            w = torch.where(hide, 0.0, torch.exp(x @ k.T * scale - l[:, None])).sum(0)
            rel = 2.0 ** -24 * (2 * D * size + 4 * shift + 16 * count * Hq // Hkv + 100)
            for t in range(keys):
                if ok[t]:
                    at = table[b][t // cache.page], h * Hkv // Hq, t % cache.page // BLOCK
                    out[at] += w[t]
                    tol[at] += w[t] * rel
    return out, tol + out.abs() * 2.0 ** -23


# -- eviction -----------------------------------------------------------------------------

def evict(weights, page, table, lens, keep, free_pages, used, first, recent):
    """(table, free pages, lens, used, lost) as lists. Table entries without a page go first; they are
    none that could be given back."""
    table, free, lens = [list(r) for r in table], list(free_pages), list(lens)
    used = min(max(used, 0), len(free))
    score = weights.double().flatten(1).sum(1).tolist() if len(weights) else []
    given = []
    for b in range(len(lens)):
        row = table[b]
        n = min(-(-max(0, lens[b]) // page), len(row))
        may = [c for c in range(n) if first <= c < n - recent]

        def rank(c):
            if not 0 <= row[c] < len(score):
                return (0, 0.0, c)
            s = score[row[c]]
            return (2, 0.0, c) if math.isnan(s) else (1, s, c)

        gone = sorted(sorted(may, key=rank)[:max(0, n - keep[b])])
        given += [row[c] for c in gone if 0 <= row[c] < len(score)]
        left = [row[c] for c in range(n) if c not in set(gone)]
        row[:n] = left + [-1] * len(gone)
        lens[b] -= page * len(gone)
    back = max(0, used - len(given))
    free[back:used] = given[:used - back]
    return table, free, lens, back, max(0, len(given) - used)
