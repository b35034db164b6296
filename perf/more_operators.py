"""Performance cases of the serving operators around the 8-bit cache: norms of
queries and keys with the position rotation, storing into the cache and
attention over it, accumulated attention weights and eviction by them.

``listed()`` returns the named cases and ``draw(rng)`` one more of the same
ranges. ``prepare`` makes a case's inputs on the GPU, ``run`` makes one pass
(in plain torch operations, or through the package where ``own`` is set),
``work`` counts what it cannot do without and ``exact`` gives the result in 64
bits.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BLOCK = 64                    # tokens of a head that share a scale
LOW, HIGH = -15, 7            # exponents of scales
# Place of a block's token in the rows of the values' codes [D, 64].
PLACE = [16 * (t >> 2 & 3) + 8 * (t >> 5) + 4 * (t >> 4 & 1) + (t & 3) for t in range(BLOCK)]


# -- cases --------------------------------------------------------------------------------

def _rotate(B, S, Hq, Hkv, D, R, dtype, wtype, neighbours, heads_first, far, **name):
    """Norm and rotation of B x S tokens; `R` dims of a head are rotated (0: none), in
    pairs of neighbours or of halves; heads_first: tensors [B, H, S, D] in memory, else
    parts of one [B, S, Hq + 2 Hkv, D] projection; `far`: length of the angles' table
    that positions are drawn from (0: row s of it for token s)."""
    return dict(op="rotate", B=B, S=S, Hq=Hq, Hkv=Hkv, D=D, R=R, dtype=dtype, wtype=wtype,
                neighbours=neighbours, heads_first=heads_first, far=far, **name)


def _store(B, lo, ctx, new_lo, new, Hkv, D, dtype, page, **name):
    """new_lo..new rows of K and V of each of B requests with lo..ctx cached tokens."""
    return dict(op="store", B=B, lo=lo, ctx=ctx, new_lo=new_lo, new=new, Hkv=Hkv, D=D,
                dtype=dtype, page=page, **name)


def _cache(op, B, lo, ctx, new_lo, new, Hq, Hkv, D, dtype, page, **name):
    """Attention over the cache ("attn") or the weights of its blocks ("weigh"): B
    requests with lo..ctx cached tokens and new_lo..new query tokens each (the last
    ones of the request)."""
    return dict(op=op, B=B, lo=lo, ctx=ctx, new_lo=new_lo, new=new, Hq=Hq, Hkv=Hkv, D=D,
                dtype=dtype, page=page, **name)


def _evict(B, lo, held, Hkv, page, share, **name):
    """B requests of lo..held pages, each with a budget of about `share` of `held`."""
    return dict(op="evict", B=B, lo=lo, held=held, Hkv=Hkv, page=page, share=share, **name)


def listed():
    return [
        # one decoding step of a serving batch: latency
        _rotate(1, 32, 32, 8, 128, 128, "bf16", "bf16", False, False, 131072, name="rotate_step"),
        # q and k of a diffusion transformer's block, image tokens, before its attention
        _rotate(2, 8192, 24, 24, 64, 64, "fp16", "fp32", True, True, 0, name="rotate_image"),
        # the new token of every request of a batch goes into the cache
        _store(64, 100, 4096, 1, 1, 8, 128, "bf16", 64, name="store8_step"),
        # prompts admitted together, behind cached prefixes
        _store(8, 30, 1000, 500, 4096, 16, 128, "fp16", 128, name="store8_prompts"),
        # one short conversation, one token: latency
        _cache("attn", 1, 1024, 1024, 1, 1, 16, 16, 64, "fp16", 64, name="attn8_single"),
        # a ragged serving batch, one token each
        _cache("attn", 32, 100, 16384, 1, 1, 32, 8, 128, "bf16", 64, name="attn8_batch"),
        # one 131072-token context, four drafted tokens at once
        _cache("attn", 1, 131068, 131068, 4, 4, 16, 2, 128, "fp16", 128, name="attn8_long"),
        # prompt chunks behind cached prefixes, ragged
        _cache("attn", 3, 300, 8192, 77, 2111, 16, 4, 128, "bf16", 64, name="attn8_prompts"),
        # the weights of a decoding step's tokens
        _cache("weigh", 32, 100, 16384, 1, 1, 32, 8, 128, "bf16", 64, name="weigh_step"),
        # the weights that prompt chunks give
        _cache("weigh", 3, 300, 8192, 77, 2111, 16, 4, 128, "bf16", 64, name="weigh_prompts"),
        # a serving batch of which many are over their budgets
        _evict(64, 20, 512, 8, 64, 0.5, name="evict_batch"),
        # one context of 131072 tokens, a quarter of it kept
        _evict(1, 2048, 2048, 8, 64, 0.25, name="evict_long"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    """One more case of the listed cases' ranges."""
    op = rng.choice(("rotate", "rotate", "store", "attn", "attn", "prompt", "weigh", "weigh_prompt",
                     "evict"))
    page = rng.choice((64, 128, 256))
    dtype = rng.choice(("fp16", "bf16"))
    D = rng.choice((64, 128))
    if op == "rotate":
        D = rng.choice((40, 64, 80, 128, 128, 256, 512))
        R = rng.choice((D // 16 * 16, D // 32 * 16, D // 16 * 16, 0))
        Hkv, G = rng.choice((1, 2, 4, 5, 8)), rng.choice((1, 3, 4, 7))
        tokens = _log(rng, 1, max(1, 50_000_000 // ((G + 1) * Hkv * D)))
        B = rng.choice((1, 1, 2, 3))
        S = max(1, tokens // B)
        return _rotate(B, S, G * Hkv, Hkv, D, R, dtype, rng.choice((dtype, "fp32")),
                       rng.random() < 0.5, rng.random() < 0.5, rng.choice((0, 4096, 131072)))
    Hkv = rng.choice((1, 2, 4, 5, 8))
    G = rng.choice((1, 2, 3, 4, 7, 8))
    if op == "store":
        B = _log(rng, 1, 128)
        new = _log(rng, 1, max(1, 40000 // B // Hkv))
        return _store(B, 1, _log(rng, 1, 4000), max(1, new // 8), new, Hkv, D, dtype, page)
    if op in ("attn", "weigh"):
        B = _log(rng, 1, 64)
        ctx = _log(rng, 1, max(64, min(131072, (1 << 20) // (B * Hkv))))
        return _cache(op, B, max(1, ctx // 20), ctx, 1, rng.choice((1, 1, 1, 2, 5)), G * Hkv, Hkv, D,
                      dtype, page)
    if op in ("prompt", "weigh_prompt"):
        Hkv, G, B = rng.choice((1, 2, 4)), rng.choice((1, 2, 3, 4)), rng.choice((1, 2, 3, 5))
        new = _log(rng, 17, 2111)
        return _cache("attn" if op == "prompt" else "weigh", min(B, 3), 1, _log(rng, 1, 8192),
                      max(1, new // 10), new, G * Hkv, Hkv, D, dtype, page)
    B = _log(rng, 1, 64)
    held = _log(rng, 2, 32768 // B)
    return _evict(B, 1, held, Hkv, page, rng.choice((0.1, 0.25, 0.5, 0.9)))


# -- sizes that follow from a case --------------------------------------------------------

def _spread(lo, hi, n, salt):
    """n lengths spread over lo..hi (over their logarithm), hi among them."""
    rng = random.Random(f"{salt} {lo} {hi} {n}")
    return [hi] + [_log(rng, lo, hi) for _ in range(n - 1)]


def _lengths(case):
    """(cached tokens, new tokens) of every request."""
    return (_spread(case["lo"], case["ctx"], case["B"], "ctx"),
            _spread(case["new_lo"], case["new"], case["B"], "new"))


def _held(case):
    """(pages held, budget) of every request."""
    held = _spread(case["lo"], case["held"], case["B"], "held")
    return held, [max(3, int(case["held"] * case["share"]))] * case["B"]


def work(case):
    op = case["op"]
    if op == "rotate":
        n = case["B"] * case["S"]
        rows = n if case["far"] else case["S"]
        x = n * (case["Hq"] + case["Hkv"]) * case["D"]
        return {"bytes": 4 * x + 4 * rows * case["R"], "flops": 8 * x}
    if op == "evict":
        held, keep = _held(case)
        gone = sum(max(0, min(n - m, n - 2)) for n, m in zip(held, keep))
        return {"bytes": 4 * case["Hkv"] * (case["page"] // BLOCK) * sum(held) + 8 * sum(held) + 4 * gone,
                "flops": case["Hkv"] * sum(held)}
    old, new = _lengths(case)
    D, Hkv, T = case["D"], case["Hkv"], sum(new)
    if op == "store":
        n = 2 * Hkv * D
        shared = sum(a % BLOCK for a in old)
        return {"bytes": n * (2 * T + T + 2 * (T + shared)), "flops": 3 * n * T}
    pairs = sum(b * (a + b) - b * (b - 1) // 2 for a, b in zip(old, new))
    tokens, Hq = sum(old) + T, case["Hq"]
    if op == "weigh":
        return {"bytes": Hkv * D * tokens + 2 * T * Hq * D + 4 * T * Hq + 8 * Hkv * tokens // BLOCK,
                "flops": 2 * D * Hq * pairs}
    return {"bytes": 2 * Hkv * D * tokens + 4 * T * Hq * D, "flops": 4 * D * Hq * pairs}


# -- the format ---------------------------------------------------------------------------

def _exponent(top):
    """Exponent of the smallest scale for a largest value `top` (fp32, finite)."""
    m, e = torch.frexp(top.clamp(2.0 ** -14, 448 * 2.0 ** HIGH))   # top = m 2^e, 0.5 <= m < 1
    return (e - 9 + (m > 0.875).int()).clamp(LOW, HIGH)


def _codes(x, e):
    """E4M3 bytes of fp32 x at scales 2^e."""
    y = torch.ldexp(x, -e).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    return torch.where(torch.isfinite(x), y, 127)


def _values(codes, e):
    return torch.ldexp(codes.view(torch.float8_e4m3fn).float(), e)


def _finite_top(x, dims):
    return torch.where(torch.isfinite(x), x.abs(), 0).amax(dims)


def _blocks(x):
    """Codes [n, H, page, D] and exponents [n, H, page/64] of whole pages of fp32 rows."""
    e = _exponent(_finite_top(x.unflatten(2, (-1, BLOCK)), (3, 4)))
    return _codes(x, e.repeat_interleave(BLOCK, 2)[..., None]), e


def _turned(codes):
    """Codes of values [n, H, page, D] in the cache's order [n, H, page/64, D, 64]."""
    place = torch.tensor(PLACE, device=codes.device)
    out = torch.empty_like(codes.unflatten(2, (-1, BLOCK)).transpose(3, 4),
                           memory_format=torch.contiguous_format)
    out[..., place] = codes.unflatten(2, (-1, BLOCK)).transpose(3, 4)
    return out


def _straight(codes):
    """The other way round."""
    place = torch.tensor(PLACE, device=codes.device)
    return codes[..., place].transpose(3, 4).flatten(2, 3)


# -- inputs -------------------------------------------------------------------------------

def _paged(case, lens, g, dev):
    """A cache of unit-normal keys and values in shuffled pages: keys' codes [pages, heads,
    page, D], values' [pages, heads, page/64, D, 64], a power of two for every 64
    tokens of a head."""
    D, Hkv, P = case["D"], case["Hkv"], case["page"]
    need = [-(-n // P) for n in lens]
    pages = sum(need) + 3
    phys = torch.randperm(pages, generator=g, device=dev).int()
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = phys[at:at + n]
        at += n
    parts = []
    for is_v, gain in ((False, 2.0), (True, 1.0)):   # keys with some spread of scores, unit values
        shape = (pages, Hkv, P // BLOCK, D, BLOCK) if is_v else (pages, Hkv, P, D)
        codes = torch.empty(shape, dtype=torch.uint8, device=dev)
        scale = torch.empty(pages, Hkv, P // BLOCK, device=dev)
        for p in range(0, pages, 256):
            n = min(256, pages - p)
            c, e = _blocks(torch.randn(n, Hkv, P, D, generator=g, device=dev) * gain)
            codes[p:p + n] = _turned(c) if is_v else c
            scale[p:p + n] = torch.ldexp(torch.ones_like(scale[p:p + n]), e)
        parts += [codes, scale]
    return table, parts


def _prepare_rotate(case, g, dev):
    B, S, Hq, Hkv, D, R = (case[x] for x in ("B", "S", "Hq", "Hkv", "D", "R"))
    dt, wt = DTYPES[case["dtype"]], DTYPES[case["wtype"]]
    if case["heads_first"]:
        q, k = ((torch.randn(B, H, S, D, generator=g, device=dev) * 3).to(dt).transpose(1, 2)
                for H in (Hq, Hkv))
    else:
        x = torch.empty(B, S, Hq + 2 * Hkv, D, dtype=dt, device=dev)
        for b in range(B):
            x[b] = torch.randn(S, Hq + 2 * Hkv, D, generator=g, device=dev) * 3
        q, k = x[:, :, :Hq], x[:, :, Hq:Hq + Hkv]
    wq, wk = ((1 + 0.2 * torch.randn(D, generator=g, device=dev)).to(wt) for _ in range(2))
    cos = sin = positions = None
    if R:
        n = case["far"] or S
        rate = 10000.0 ** (-torch.arange(R // 2, dtype=torch.float64, device=dev) * 2 / R)
        angle = torch.arange(n, dtype=torch.float64, device=dev)[:, None] * rate
        cos, sin = angle.cos().float(), angle.sin().float()
        if case["far"]:
            positions = torch.randint(0, n, (B, S), generator=g, device=dev).int()
    return dict(q=q, k=k, wq=wq, wk=wk, cos=cos, sin=sin, positions=positions)


def _prepare_store(case, g, dev, order):
    i32 = dict(dtype=torch.int32, device=dev)
    D, Hkv, P = case["D"], case["Hkv"], case["page"]
    old, new = ([x[i] for i in order] for x in _lengths(case))
    lens = [a + b for a, b in zip(old, new)]
    table, cache = _paged(case, lens, g, dev)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    k, v = ((torch.randn(cu[-1], Hkv, D, generator=g, device=dev) * s).to(DTYPES[case["dtype"]])
            for s in (2.0, 1.0))
    # Blocks that are written, and for each place of one: its row (-1: none) and whether
    # it holds a token already.
    where, row, held = [], [], []
    for b, (a, n) in enumerate(zip(old, lens)):
        for j in range(a // BLOCK, -(-n // BLOCK)):
            where.append((b, j))
            pos = range(j * BLOCK, (j + 1) * BLOCK)
            row.append([cu[b] + p - a if a <= p < n else -1 for p in pos])
            held.append([p < a for p in pos])
    where, row = torch.tensor(where, device=dev), torch.tensor(row, device=dev)
    held = torch.tensor(held, device=dev)
    per = P // BLOCK
    page, part = table[where[:, 0], where[:, 1] // per].long(), where[:, 1] % per
    slots = (page * P + part * BLOCK)[:, None] + torch.arange(BLOCK, device=dev)
    return dict(k=k, v=v, cache=cache, table=table, lens=torch.tensor(lens, **i32),
                cu=torch.tensor(cu, **i32), page=page, part=part, row=row, held=held,
                slots=slots[held | (row >= 0)].int())


def _prepare_evict(case, g, dev, order):
    i32 = dict(dtype=torch.int32, device=dev)
    P = case["page"]
    held, keep = ([x[i] for i in order] for x in _held(case))
    pages = sum(held) + 5
    phys = torch.randperm(pages, generator=g, device=dev).int()
    table = torch.full((len(held), max(held)), -1, **i32)
    at = 0
    for b, n in enumerate(held):
        table[b, :n] = phys[at:at + n]
        at += n
    # attention weight is spread unevenly, over many orders
    weights = torch.exp(2 * torch.randn(pages, case["Hkv"], P // BLOCK, generator=g, device=dev))
    last = torch.randint(1, P + 1, (len(held),), generator=g, device=dev)
    lens = ((torch.tensor(held, device=dev) - 1) * P + last).int()
    return dict(weights=weights, table=table, lens=lens, keep=torch.tensor(keep, **i32),
                free=torch.cat((phys[:at], phys[at:])), used=torch.tensor([at], **i32),
                first=1, recent=1)


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    if case["op"] == "rotate":
        return dict(case=case) | _prepare_rotate(case, g, dev)
    order = torch.randperm(case["B"], generator=g, device=dev).tolist()
    if case["op"] == "store":
        return dict(case=case) | _prepare_store(case, g, dev, order)
    if case["op"] == "evict":
        return dict(case=case) | _prepare_evict(case, g, dev, order)
    i32 = dict(dtype=torch.int32, device=dev)
    old, news = ([x[i] for i in order] for x in _lengths(case))
    lens = [a + b for a, b in zip(old, news)]
    table, cache = _paged(case, lens, g, dev)
    q = torch.randn(sum(news), case["Hq"], case["D"], generator=g, device=dev)
    cu = [0]
    for n in news:
        cu.append(cu[-1] + n)
    state = dict(case=case, q=q.to(DTYPES[case["dtype"]]), cache=cache, table=table,
                 lens=torch.tensor(lens, **i32), cu=torch.tensor(cu, **i32), host_lens=lens,
                 host_new=news, scale=case["D"] ** -0.5)
    if case["op"] == "weigh":
        pages = cache[0].shape[0]
        state["weights"] = torch.rand(pages, case["Hkv"], case["page"] // BLOCK, generator=g, device=dev)
        state["lse"] = torch.empty(q.shape[:2], device=dev)
        for at, c, x in _scores(state):
            state["lse"][at:at + c] = torch.logsumexp(x, -1).flatten(0, 1).T
    return state


# -- one pass -----------------------------------------------------------------------------

def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    case = s["case"]
    if case["op"] == "rotate":
        from gfx906_amd import qknorm
        return qknorm.norm_rotate(s["q"], s["k"], s["wq"], s["wk"], s["cos"], s["sin"],
                                  positions=s["positions"], neighbours=case["neighbours"])
    from gfx906_amd import kv8
    if case["op"] == "evict":
        table, free = s["table"].clone(), s["free"].clone()
        e = kv8.evict(s["weights"], table, s["lens"], s["keep"], free, s["used"], first=s["first"],
                      recent=s["recent"])
        return table, free, e.lens, e.used, e.lost
    cache = kv8.Cache(*s["cache"])
    if case["op"] == "store":
        kv8.store(cache, s["k"], s["v"], s["table"], s["lens"], s["cu"])
        return kv8.load(cache, s["slots"], s["k"].dtype)
    if case["op"] == "attn":
        return kv8.attn(s["q"], cache, s["table"], s["lens"], s["scale"], cu_q=s["cu"],
                        max_q=max(s["host_new"]))
    weights = s["weights"].clone()
    kv8.weigh(weights, s["q"], s["lse"], cache, s["table"], s["lens"], s["scale"], cu_q=s["cu"],
              max_q=max(s["host_new"]))
    return weights


def _run_plain(s):
    return {"rotate": _plain_rotate, "store": _plain_store, "attn": _plain_attn,
            "weigh": _plain_weigh, "evict": _plain_evict}[s["case"]["op"]](s)


def _plain_rotate(s):
    case, out = s["case"], []
    R, near = case["R"], case["neighbours"]
    if R:
        rows = slice(0, case["S"]) if s["positions"] is None else s["positions"].long()
        c, n = s["cos"][rows], s["sin"][rows]
        c, n = (t[None, :, None] if t.dim() == 2 else t[:, :, None] for t in (c, n))
    for x, w in ((s["q"], s["wq"]), (s["k"], s["wk"])):
        dt, x = x.dtype, x.float()
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.float()
        if R:
            r = x[..., :R]
            a, b = (r[..., 0::2], r[..., 1::2]) if near else (r[..., :R // 2], r[..., R // 2:])
            a, b = a * c - b * n, a * n + b * c
            r = torch.stack((a, b), -1).flatten(-2) if near else torch.cat((a, b), -1)
            x = torch.cat((r, x[..., R:]), -1) if R < x.shape[-1] else r
        out.append(x.to(dt))
    return tuple(out)


def _plain_store(s):
    page, part, row, held = s["page"], s["part"], s["row"], s["held"]
    n, D = len(page), s["case"]["D"]
    place = torch.tensor(PLACE, device=page.device)
    at = part[:, None] * BLOCK + torch.arange(BLOCK, device=page.device)
    fresh = ~held.any(1)
    write = (held | (row >= 0))[:, None, :, None]
    for is_v, x, codes, scale in ((False, s["k"], *s["cache"][:2]), (True, s["v"], *s["cache"][2:])):
        if is_v:
            was = codes[page, :, part][..., place].transpose(2, 3)         # [n, H, 64, D]
        else:
            was = codes[page[:, None], :, at].transpose(1, 2)
        old_e = torch.frexp(scale[page, :, part])[1] - 1
        rows = x.float()[row.clamp(min=0)].transpose(1, 2)                 # [n, H, 64, D]
        rows = torch.where((row >= 0)[:, None, :, None], rows, 0)
        e = _exponent(_finite_top(rows, (2, 3)))
        e = torch.where(fresh[:, None], e, torch.maximum(e, old_e))[..., None, None]
        kept = was.view(torch.float8_e4m3fn).float()
        kept = _codes(torch.ldexp(kept, old_e[..., None, None] - e), torch.zeros_like(e))
        c = torch.where(held[:, None, :, None], kept, _codes(rows, e))
        c = torch.where(write, c, was)
        if is_v:
            turned = torch.empty(n, c.shape[1], D, BLOCK, dtype=torch.uint8, device=c.device)
            turned[..., place] = c.transpose(2, 3)
            codes[page, :, part] = turned
        else:
            codes[page[:, None], :, at] = c.transpose(1, 2)
        scale[page, :, part] = torch.ldexp(torch.ones_like(e[..., 0, 0], dtype=torch.float32), e[..., 0, 0])
    return _plain_load(s)


def _plain_load(s):
    """Rows of the touched blocks' tokens."""
    P, dt, slots = s["case"]["page"], DTYPES[s["case"]["dtype"]], s["slots"].long()
    page, t = slots // P, slots % P
    kc, ks, vc, vs = s["cache"]
    place = torch.tensor(PLACE, device=slots.device)
    ke, ve = (torch.frexp(x[page, :, t // BLOCK])[1][..., None] - 1 for x in (ks, vs))
    v = vc[page, :, t // BLOCK, :, place[t % BLOCK]]
    return _values(kc[page, :, t], ke).to(dt), _values(v.contiguous(), ve).to(dt)


def _gathered(codes, scale, pages, n):
    """fp32 [heads, n, D] of the first n tokens of the listed pages."""
    c = codes[pages]
    c = _straight(c).contiguous() if c.dim() == 5 else c
    e = (torch.frexp(scale[pages])[1] - 1).repeat_interleave(BLOCK, 2)[..., None]
    return _values(c, e).transpose(0, 1).flatten(1, 2)[:, :n]


def _scores(s):
    """(first row, rows, scores [Hkv, G, rows, keys]) of every request, up to 256 rows
    at a time; -inf where a row does not see a key."""
    case, q, at = s["case"], s["q"], 0
    G = case["Hq"] // case["Hkv"]
    for b, (n, m) in enumerate(zip(s["host_lens"], s["host_new"])):
        pages = s["table"][b, :-(-n // case["page"])].long()
        k = _gathered(s["cache"][0], s["cache"][1], pages, n)
        for r in range(0, m, 256):
            c = min(256, m - r)
            qb = q[at + r:at + r + c].float().transpose(0, 1).reshape(-1, G * c, case["D"])
            x = torch.matmul(qb, k.transpose(1, 2)).view(-1, G, c, n) * s["scale"]
            pos = torch.arange(n - m + r, n - m + r + c, device=q.device)
            x.masked_fill_(torch.arange(n, device=q.device)[None] > pos[:, None], -math.inf)
            yield at + r, c, x
        at += m


def _plain_attn(s):
    case, q, P = s["case"], s["q"], s["case"]["page"]
    out, b, end, v = torch.empty_like(q), -1, 0, None
    for at, c, x in _scores(s):
        if at >= end:
            b += 1
            end += s["host_new"][b]
            n = s["host_lens"][b]
            v = _gathered(s["cache"][2], s["cache"][3], s["table"][b, :-(-n // P)].long(), n)
        x -= x.amax(-1, keepdim=True)
        x.exp_()
        o = torch.matmul(x.flatten(1, 2), v).view(*x.shape[:3], case["D"]) / x.sum(-1, keepdim=True)
        out[at:at + c] = o.flatten(0, 1).transpose(0, 1).to(q.dtype)
    return out


def _plain_weigh(s):
    case, weights = s["case"], s["weights"].clone()
    Hkv, P, end, b = case["Hkv"], case["page"], 0, -1
    for at, c, x in _scores(s):
        if at >= end:
            b += 1
            end += s["host_new"][b]
            pages = s["table"][b, :-(-s["host_lens"][b] // P)].long()
            total = torch.zeros(Hkv, len(pages) * P, device=x.device)
        x -= s["lse"][at:at + c].T.reshape(x.shape[:3])[..., None]
        total[:, :x.shape[-1]] += x.exp_().sum((1, 2))
        if at + c == end:
            weights[pages] += total.view(Hkv, len(pages), P // BLOCK, BLOCK).sum(-1).transpose(0, 1)
    return weights


def _plain_evict(s):
    table, free, lens, P = s["table"].clone(), s["free"].clone(), s["lens"], s["case"]["page"]
    B, W = table.shape
    col = torch.arange(W, device=table.device)[None]
    held = ((lens + P - 1) // P)[:, None]
    mine = col < held
    score = s["weights"].double().sum((1, 2))[table.clamp(min=0).long()]
    may = mine & (col >= s["first"]) & (col < held - s["recent"])
    gone = torch.minimum((held[:, 0] - s["keep"]).clamp(min=0), may.sum(1))
    rank = torch.argsort(torch.argsort(score.masked_fill(~may, math.inf), dim=1, stable=True), dim=1)
    out = rank < gone[:, None]
    order = torch.argsort((~mine | out).int(), dim=1, stable=True)
    closed = torch.gather(table, 1, order)
    count = (held[:, 0] - gone)[:, None]
    total = gone.sum()
    back = (s["used"] - total).clamp(min=0)
    place = torch.cumsum(out.flatten(), 0) - 1 + back      # in the order of requests and columns
    place = torch.where(out.flatten() & (place < s["used"]), place, len(free))
    free = torch.cat((free, free[:1]))
    free[place] = torch.where(place < len(free) - 1, table.flatten(), free[-1])
    lost = (total - s["used"]).clamp(min=0)
    return (torch.where(col < count, closed, torch.where(mine, -1, table)), free[:-1],
            (lens - gone * P).int(), back.int(), lost.int())


# -- the result in 64 bits ----------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"rotate": _exact_rotate, "store": _exact_store, "attn": _exact_attn,
            "weigh": _exact_weigh, "evict": _exact_evict}[case["op"]](s)


def _exact_rotate(s):
    case, out = s["case"], []
    R, h = case["R"], case["R"] // 2
    for x, w in ((s["q"], s["wq"]), (s["k"], s["wk"])):
        x = x.double()
        y = x / torch.sqrt(x.square().sum(-1, keepdim=True) / case["D"] + 1e-6) * w.double()
        if R:
            for b in range(case["B"]):
                rows = (torch.arange(case["S"], device=x.device) if s["positions"] is None
                        else s["positions"][b].long())
                z = torch.complex(s["cos"][rows].double(), s["sin"][rows].double())[:, None]
                t = y[b, ..., :R].clone()
                if case["neighbours"]:
                    p = torch.view_as_complex(t.unflatten(-1, (h, 2)).contiguous()) * z
                    y[b, ..., :R] = torch.view_as_real(p).flatten(-2)
                else:
                    p = torch.complex(t[..., :h].contiguous(), t[..., h:].contiguous()) * z
                    y[b, ..., :h], y[b, ..., h:R] = p.real, p.imag
        out.append(y)
    return tuple(out)


def _decoded(codes):
    """fp64 values of E4M3 bytes, by the format's fields."""
    c = codes.long()
    e, m = c // 8 % 16, c % 8
    a = torch.where(e == 0, m / 512.0, (1 + m / 8.0) * torch.exp2(e.double() - 7))
    a = torch.where(c % 128 == 127, math.nan, a.double())
    return torch.where(c >= 128, -a, a)


def _rounded(a):
    """fp64 numbers to the nearest E4M3 value, ties to even."""
    step = torch.exp2(torch.floor(torch.log2(a.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(a / step) * step).clamp(-448, 448)


def _exact_store(s):
    """Block by block, as the rule says; K and V rows of the listed slots."""
    case, res = s["case"], []
    P, D, Hkv = case["page"], case["D"], case["Hkv"]
    table, lens, cu = s["table"].tolist(), s["lens"].tolist(), s["cu"].tolist()
    place = torch.tensor(PLACE, device="cuda")
    for is_v, x, codes, scale in ((False, s["k"], *s["cache"][:2]), (True, s["v"], *s["cache"][2:])):
        parts = []
        for b, n in enumerate(lens):
            m = cu[b + 1] - cu[b]
            new = x[cu[b]:cu[b + 1]].double()
            pos = n - m
            while pos < n:
                j = pos // BLOCK
                end = min(n, (j + 1) * BLOCK)
                rows = new[pos - (n - m):end - (n - m)].transpose(0, 1)          # [H, r, D]
                top = rows.abs().amax((1, 2)).clamp(2.0 ** -20, 57344.0)
                unit = torch.exp2(torch.ceil(torch.log2(top / 448)).clamp(LOW, HIGH))
                before = pos - j * BLOCK
                page, part = table[b][j * BLOCK // P], j % (P // BLOCK)
                if before:
                    c = (codes[page, :, part][..., place].transpose(1, 2) if is_v
                         else codes[page, :, part * BLOCK:(part + 1) * BLOCK])[:, :before]
                    u = scale[page, :, part].double()
                    unit = torch.maximum(unit, u)
                    kept = _rounded(_decoded(c) * (u / unit)[:, None, None])
                    rows = torch.cat((kept * unit[:, None, None],
                                      _rounded(rows / unit[:, None, None]) * unit[:, None, None]), 1)
                else:
                    rows = _rounded(rows / unit[:, None, None]) * unit[:, None, None]
                parts.append(rows.transpose(0, 1))
                pos = end
        res.append(torch.cat(parts))
    return tuple(res)


def _values64(codes, scale, h):
    """fp64 [tokens, D] of one head of the listed pages."""
    place = torch.tensor(PLACE, device="cuda")
    x = _decoded(codes[:, h])
    x = x[..., place].transpose(2, 3) if x.dim() == 4 else x.unflatten(1, (-1, BLOCK))
    return (x * scale[:, h].double()[..., None, None]).flatten(0, 2)


def _exact_weights(s, each):
    """each(request, query head, kv head, pages, scores [queries, keys]) in 64 bits."""
    case, at = s["case"], 0
    G = case["Hq"] // case["Hkv"]
    for b, (n, m) in enumerate(zip(s["host_lens"], s["host_new"])):
        pages = s["table"][b, :-(-n // case["page"])].long()
        late = torch.triu(torch.full((m, n), -math.inf, dtype=torch.float64, device="cuda"),
                          diagonal=n - m + 1)
        for h in range(case["Hkv"]):
            k = _values64(s["cache"][0][pages], s["cache"][1][pages], h)[:n]
            for j in range(h * G, h * G + G):
                each(at, m, j, h, pages, (s["q"][at:at + m, j].double() @ k.T) * s["scale"] + late)
        at += m


def _exact_attn(s):
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    held = {}

    def each(at, m, j, h, pages, z):
        if held.get("for") != (at, h):
            v = _values64(s["cache"][2][pages], s["cache"][3][pages], h)[:z.shape[1]]
            held.update({"for": (at, h), "v": v})
        w = torch.exp(z - z.amax(1, keepdim=True))
        out[at:at + m, j] = (w @ held["v"]) / w.sum(1, keepdim=True)

    _exact_weights(s, each)
    return out


def _exact_weigh(s):
    weights, per = s["weights"].double(), s["case"]["page"] // BLOCK

    def each(at, m, j, h, pages, z):
        w = torch.exp(z - s["lse"][at:at + m, j].double()[:, None]).sum(0)
        w = torch.nn.functional.pad(w, (0, len(pages) * per * BLOCK - len(w)))
        weights[pages, h] += w.view(len(pages), per, BLOCK).sum(2)

    _exact_weights(s, each)
    return weights


def _exact_evict(s):
    """Request by request on the host."""
    P, used, given = s["case"]["page"], s["used"].item(), []
    table, free, lens = s["table"].tolist(), s["free"].tolist(), s["lens"].tolist()
    score = s["weights"].double().flatten(1).cpu().numpy().sum(1)
    for b, (n, keep) in enumerate(zip(list(lens), s["keep"].tolist())):
        held = -(-n // P)
        may = range(s["first"], max(s["first"], held - s["recent"]))
        gone = sorted(may, key=lambda c: (score[table[b][c]], c))[:max(0, held - keep)]
        given += [table[b][c] for c in sorted(gone)]
        row = [table[b][c] for c in range(held) if c not in set(gone)]
        table[b][:held] = row + [-1] * len(gone)
        lens[b] = n - P * len(gone)
    back = max(0, used - len(given))
    free[back:used] = given[:used - back]
    i32 = dict(dtype=torch.int32, device="cuda")
    return (torch.tensor(table, **i32), torch.tensor(free, **i32), torch.tensor(lens, **i32),
            torch.tensor([back], **i32), torch.tensor([max(0, len(given) - used)], **i32))
