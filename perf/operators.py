"""Performance cases of the long-context operators: pages and slots of a paged
cache, the 4-bit cache with its attention, and sparse attention over selected
blocks.

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

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
Q_BLOCK = 128                 # query rows that share one choice of key blocks
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# -- cases --------------------------------------------------------------------------------

def _pages(B, ctx, new, page, **name):
    """Page table update and slot map of B requests with up to `ctx` cached and
    `new` new tokens each."""
    return dict(op="pages", B=B, ctx=ctx, new=new, page=page, **name)


def _store(T, Hkv, D, dtype, page, **name):
    """T rows of K and V into the 4-bit cache, and the values they then stand for."""
    return dict(op="store", T=T, Hkv=Hkv, D=D, dtype=dtype, page=page, **name)


def _cache(B, lo, ctx, new_lo, new, Hq, Hkv, D, dtype, page, **name):
    """Attention over the 4-bit cache: B requests with lo..ctx cached tokens and
    new_lo..new query tokens each (the last ones of the request)."""
    return dict(op="cache", B=B, lo=lo, ctx=ctx, new_lo=new_lo, new=new, Hq=Hq, Hkv=Hkv, D=D,
                dtype=dtype, page=page, **name)


def _sparse(B, Hq, Hkv, Sq, Skv, D, dtype, block, count, causal, kept=False, **name):
    """Block choice and attention over the chosen blocks; `kept`: the program
    holds the key blocks' means already (a decoder keeps them beside its keys)."""
    return dict(op="sparse", B=B, Hq=Hq, Hkv=Hkv, Sq=Sq, Skv=Skv, D=D, dtype=dtype, block=block,
                count=count, causal=causal, kept=kept, **name)


def listed():
    return [
        # one decoding step of a serving batch: every request gets one token
        _pages(64, 16384, 1, 64, name="pages_step"),
        # prompts admitted together: slots of some tens of thousands of tokens
        _pages(48, 4096, 2111, 128, name="pages_prompts"),
        # the new token of every request of a batch goes into the cache
        _store(64, 8, 128, "bf16", 64, name="store_step"),
        # a long prompt's keys and values go into the cache
        _store(16384, 16, 128, "fp16", 128, name="store_prompt"),
        # one short conversation, one token: latency
        _cache(1, 1024, 1024, 1, 1, 16, 16, 64, "fp16", 64, name="cache_single"),
        # a ragged serving batch, one token each
        _cache(32, 100, 16384, 1, 1, 32, 8, 128, "bf16", 64, name="cache_batch"),
        # one 131072-token context, four drafted tokens at once
        _cache(1, 131068, 131068, 4, 4, 16, 2, 128, "fp16", 128, name="cache_long"),
        # prompt chunks behind cached prefixes, ragged
        _cache(3, 300, 8192, 77, 2111, 16, 4, 128, "bf16", 64, name="cache_prompts"),
        # one token of a long context: the choice and its 64 blocks
        _sparse(4, 16, 4, 1, 32768, 128, "fp16", 64, 64, True, kept=True, name="sparse_token"),
        # a ragged causal prompt with grouped heads
        _sparse(1, 16, 4, 5003, 5003, 128, "bf16", 64, 16, True, name="sparse_prompt"),
        # 16 heads of 16384 tokens, an eighth of the blocks
        _sparse(1, 16, 16, 16384, 16384, 128, "fp16", 64, 32, False, name="sparse_16k"),
        # a video's 131072 tokens, a sixteenth of the blocks
        _sparse(1, 8, 8, 131072, 131072, 64, "bf16", 128, 64, False, name="sparse_131k"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    """One more case of the listed cases' ranges."""
    op = rng.choice(("pages", "store", "cache", "cache", "prompt", "sparse", "sparse", "token"))
    page = rng.choice((64, 128, 256))
    dtype = rng.choice(("fp16", "bf16"))
    D = rng.choice((64, 128))
    if op == "pages":
        B = _log(rng, 1, 256)
        return _pages(B, _log(rng, 1, 32768), _log(rng, 1, max(1, 100000 // B)), page)
    if op == "store":
        return _store(_log(rng, 1, 16384), rng.choice((1, 2, 3, 4, 8, 16)), D, dtype, page)
    Hkv = rng.choice((1, 2, 4, 5, 8))
    G = rng.choice((1, 2, 3, 4, 7, 8))
    if op == "cache":
        B = _log(rng, 1, 64)
        ctx = _log(rng, 1, max(64, min(131072, (1 << 20) // (B * Hkv))))
        return _cache(B, max(1, ctx // 20), ctx, 1, rng.choice((1, 1, 1, 2, 5)), G * Hkv, Hkv, D,
                      dtype, page)
    if op == "prompt":
        Hkv, G, B = rng.choice((1, 2, 4)), rng.choice((1, 2, 3, 4)), rng.choice((1, 2, 3, 5))
        new = _log(rng, 17, 2500)
        return _cache(B, 1, _log(rng, 1, 9000), max(1, new // 10), new, G * Hkv, Hkv, D, dtype, page)
    block = rng.choice((64, 128))
    if op == "token":
        B = _log(rng, 1, 8)
        Skv = _log(rng, 64, 65536 // B)
        return _sparse(B, G * Hkv, Hkv, rng.choice((1, 1, 3)), Skv, D, dtype, block,
                       rng.randint(4, 96), True, kept=rng.random() < 0.7)
    S = _log(rng, 200, 16384)
    H = _log(rng, 1, max(1, min(16, 131072 // S)))
    causal = rng.random() < 0.5
    Sq = S if causal or rng.random() < 0.6 else _log(rng, 100, S)
    G = rng.choice((1, 2))
    return _sparse(1, H * G, H, Sq, S, D, dtype, block, rng.randint(3, 48), causal)


# -- sizes that follow from a case --------------------------------------------------------

def _spread(lo, hi, n, salt):
    """n lengths spread over lo..hi (over their logarithm), hi among them."""
    rng = random.Random(f"{salt} {lo} {hi} {n}")
    return [hi] + [_log(rng, lo, hi) for _ in range(n - 1)]


def _lengths(case):
    """(cached tokens, new tokens) of every request."""
    if case["op"] == "pages":
        if case["new"] == 1:
            return _spread(1, case["ctx"], case["B"], "ctx"), [1] * case["B"]
        return ([x - 1 for x in _spread(1, case["ctx"] + 1, case["B"], "ctx")],
                _spread(1, case["new"], case["B"], "new"))
    return (_spread(case["lo"], case["ctx"], case["B"], "ctx"),
            _spread(case["new_lo"], case["new"], case["B"], "new"))


def _visible_pairs(case):
    """(query row, key) pairs of the chosen blocks of one head."""
    Sq, Skv, n, blk = case["Sq"], case["Skv"], case["count"], case["block"]
    total = 0.0
    for r0 in range(0, Sq, Q_BLOCK):
        rows = min(Q_BLOCK, Sq - r0)
        if not case["causal"]:
            total += rows * min(Skv, n * blk)
            continue
        p0, p1 = r0 + Skv - Sq, r0 + rows - 1 + Skv - Sq
        chosen = min(n, p1 // blk + 1)
        own_keys = p1 + 1 - (p0 // blk) * blk
        past = max(0, chosen - (p1 // blk - p0 // blk + 1)) * blk
        total += rows * (past + own_keys - (rows - 1) / 2)
    return total


def work(case):
    if case["op"] == "pages":
        old, new = _lengths(case)
        taken = sum(-(-(a + b) // case["page"]) - -(-a // case["page"]) for a, b in zip(old, new))
        return {"bytes": 4 * (4 * case["B"] + 2 * taken + sum(new)), "flops": 2 * sum(new)}
    if case["op"] == "store":
        n = 2 * case["T"] * case["Hkv"] * case["D"]
        return {"bytes": n * 2 + n * 17 // 32 + n * 2, "flops": 2 * n}
    if case["op"] == "cache":
        old, new = _lengths(case)
        row = 2 * case["Hkv"] * case["D"] * 17 // 32
        pairs = sum(b * (a + b) - b * (b - 1) // 2 for a, b in zip(old, new))
        return {"bytes": row * (sum(old) + sum(new)) + 4 * sum(new) * case["Hq"] * case["D"],
                "flops": 4 * case["D"] * case["Hq"] * pairs}
    D, B, Hq, Hkv = case["D"], case["B"], case["Hq"], case["Hkv"]
    nq, nk = -(-case["Sq"] // Q_BLOCK), -(-case["Skv"] // case["block"])
    pairs = _visible_pairs(case)
    keys = min(Hkv * case["Skv"], Hq * nq * case["count"] * case["block"])
    byts = B * (4 * Hq * case["Sq"] * D + 4 * keys * D)
    byts += B * 4 * Hkv * nk * D if case["kept"] else B * 2 * D * max(0, Hkv * case["Skv"] - keys)
    return {"bytes": byts + 4 * B * Hq * nq * case["count"],
            "flops": B * Hq * (4 * D * pairs + 2 * D * nq * nk)}


# -- inputs -------------------------------------------------------------------------------

def _rows_and_cache(case, g, dev):
    """A cache of unit-normal keys and values in shuffled pages, in the layout
    the package documents: codes [pages, heads, page, D/2] (low nibble first),
    scales [pages, heads, page/64, 16, D/32, 4] (token 64 a + 16 c + b of a page
    at [a, b, :, c])."""
    D, Hkv, P = case["D"], case["Hkv"], case["page"]
    old, new = _lengths(case)
    order = torch.randperm(case["B"], generator=g, device=dev).tolist()
    lens = [old[i] + new[i] for i in order]
    news = [new[i] for i in order]
    need = [-(-n // P) for n in lens]
    pages = sum(need) + 3
    phys = torch.randperm(pages, generator=g, device=dev).int()
    table = torch.full((case["B"], max(need)), -1, dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = phys[at:at + n]
        at += n
    parts = []
    for gain in (2.0, 1.0):      # keys with some spread of scores, unit values
        codes = torch.empty(pages, Hkv, P, D // 2, dtype=torch.uint8, device=dev)
        scales = torch.empty(pages, Hkv, P // 64, 16, D // 32, 4, dtype=torch.uint8, device=dev)
        for p in range(0, pages, 256):
            n = min(256, pages - p)
            x = torch.randn(n, Hkv, P, D, generator=g, device=dev) * gain
            c, s = _quantise(x)
            codes[p:p + n] = c
            scales[p:p + n] = _scale_order(s)
        parts += [codes, scales]
    return lens, news, table, parts


def _scale_order(s):
    """Scales [n, heads, page, D/32] in the cache's order."""
    n, H, P, nb = s.shape
    return s.view(n, H, P // 64, 4, 16, nb).permute(0, 1, 2, 4, 5, 3)


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    i32 = dict(dtype=torch.int32, device=dev)
    state = dict(case=case)
    if case["op"] == "pages":
        old, new = _lengths(case)
        P = case["page"]
        order = torch.randperm(case["B"], generator=g, device=dev).tolist()
        old, new = [old[i] for i in order], [new[i] for i in order]
        held = [-(-a // P) for a in old]
        need = [-(-(a + b) // P) for a, b in zip(old, new)]
        phys = torch.randperm(sum(need) + 7, generator=g, device=dev).int()
        table = torch.full((case["B"], max(need)), -1, **i32)
        at = 0
        for b, n in enumerate(held):
            table[b, :n] = phys[at:at + n]
            at += n
        return state | dict(lens=torch.tensor(old, **i32), new=torch.tensor(new, **i32), table=table,
                            free=phys[at:].contiguous(), used=torch.zeros(1, **i32),
                            tokens=sum(new))
    if case["op"] == "store":
        T, Hkv, D, P = case["T"], case["Hkv"], case["D"], case["page"]
        pages = -(-T // P) + 2
        k, v = ((torch.randn(T, Hkv, D, generator=g, device=dev) * s).to(DTYPES[case["dtype"]])
                for s in (2.0, 1.0))
        perm = torch.randperm(pages, generator=g, device=dev)
        t = torch.arange(T, device=dev)
        slots = (perm[t // P] * P + t % P).int()
        if T <= 256:   # a step's tokens lie in pages of their own requests
            slots = torch.randperm(pages * P, generator=g, device=dev)[:T].int()
        empty = [torch.zeros(pages, Hkv, P, D // 2, dtype=torch.uint8, device=dev),
                 torch.zeros(pages, Hkv, P // 64, 16, D // 32, 4, dtype=torch.uint8, device=dev)]
        return state | dict(k=k, v=v, slots=slots, cache=empty + [t.clone() for t in empty])
    if case["op"] == "cache":
        lens, news, table, cache = _rows_and_cache(case, g, dev)
        q = torch.randn(sum(news), case["Hq"], case["D"], generator=g, device=dev)
        cu = [0]
        for n in news:
            cu.append(cu[-1] + n)
        return state | dict(q=q.to(DTYPES[case["dtype"]]), cache=cache, table=table,
                            lens=torch.tensor(lens, **i32), cu=torch.tensor(cu, **i32),
                            host_lens=lens, host_new=news, scale=case["D"] ** -0.5)
    dt, D = DTYPES[case["dtype"]], case["D"]
    # Keys of a block share a direction that some queries look for, as
    # neighbouring tokens of a text or a video do.
    B, Hq, Hkv, Sq, Skv = (case[x] for x in ("B", "Hq", "Hkv", "Sq", "Skv"))
    nk = -(-Skv // 64)
    topic = torch.randn(B, Hkv, nk, D, generator=g, device=dev)
    k = torch.randn(B, Hkv, Skv, D, generator=g, device=dev)
    k += 0.7 * topic.repeat_interleave(64, 2)[:, :, :Skv]
    nt = -(-Sq // 64)
    pick = torch.randint(0, nk, (B, Hkv, nt), generator=g, device=dev)
    want = torch.gather(topic, 2, pick[..., None].expand(-1, -1, -1, D))
    want = want.repeat_interleave(Hq // Hkv, 1).repeat_interleave(64, 2)[:, :, :Sq]
    q = torch.randn(B, Hq, Sq, D, generator=g, device=dev) + 0.7 * want
    v = torch.randn(B, Hkv, Skv, D, generator=g, device=dev)
    q, k, v = q.to(dt), k.to(dt), v.to(dt)
    return state | dict(q=q, k=k, v=v, scale=D ** -0.5,
                        k_means=_means(k, case["block"]) if case["kept"] else None)


# -- one pass -----------------------------------------------------------------------------

def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    case = s["case"]
    if case["op"] == "sparse":
        from gfx906_amd import sparse
        return sparse.attn(s["q"], s["k"], s["v"], s["scale"], case["count"], block=case["block"],
                           causal=case["causal"], k_means=s["k_means"])
    from gfx906_amd import kv4
    if case["op"] == "pages":
        plan = kv4.plan_pages(s["lens"], s["new"], s["table"], s["free"], s["used"], case["page"],
                              s["tokens"])
        return plan.slots, plan.cu_new, plan.lens, plan.used, s["table"]
    cache = kv4.Cache(*s["cache"])
    if case["op"] == "store":
        kv4.store(cache, s["k"], s["v"], s["slots"])
        return kv4.load(cache, s["slots"], s["k"].dtype)
    return kv4.attn(s["q"], cache, s["table"], s["lens"], s["scale"], cu_q=s["cu"],
                    max_q=max(s["host_new"]))


def _run_plain(s):
    op = s["case"]["op"]
    return {"pages": _plain_pages, "store": _plain_store, "cache": _plain_cache,
            "sparse": _plain_sparse}[op](s)


def _plain_pages(s):
    P, lens, new, table = s["case"]["page"], s["lens"].long(), s["new"].long(), s["table"].clone()
    cu = torch.zeros(len(new) + 1, dtype=torch.long, device=new.device)
    cu[1:] = torch.cumsum(new, 0)
    held = (lens + P - 1) // P
    need = (lens + new + P - 1) // P - held
    first = torch.cumsum(need, 0) - need + s["used"]
    col = torch.arange(table.shape[1], device=new.device)[None]
    fresh = (col >= held[:, None]) & (col < (held + need)[:, None])
    take = (first[:, None] + col - held[:, None]).clamp(0, len(s["free"]) - 1)
    table = torch.where(fresh, s["free"][take], table)
    t = torch.arange(s["tokens"], device=new.device)
    b = torch.searchsorted(cu, t, right=True) - 1
    pos = lens[b] + t - cu[b]
    slots = table[b, pos // P] * P + (pos % P).int()
    used = (s["used"] + need.sum()).int()
    return slots.int(), cu.int(), (lens + new).int(), used, table


def _quantise(x):
    """E2M1 codes (two a byte, low nibble first) and E8M0 scales of fp32 x."""
    blocks = x.unflatten(-1, (-1, 32))
    top = blocks.abs().amax(-1, keepdim=True)
    e = (torch.frexp(top)[1] - 3).clamp(min=-126)
    e = torch.where(top > 0, e, -126)
    a = torch.ldexp(blocks.abs(), -e)
    code = ((a > 0.25).byte() + (a >= 0.75).byte() + (a > 1.25).byte() + (a >= 1.75).byte()
            + (a > 2.5).byte() + (a >= 3.5).byte() + (a > 5.0).byte())
    code += 8 * (blocks < 0).byte()
    code = code.flatten(-2)
    return code[..., 0::2] + 16 * code[..., 1::2], (e[..., 0] + 127).byte()


def _dequantise(codes, scales):
    """fp32 values of codes [..., D/2] and scales [..., D/32]."""
    lut = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=codes.device)
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    return torch.ldexp(lut[c.int()].unflatten(-1, (-1, 32)),
                       (scales.int() - 127)[..., None]).flatten(-2)


def _plain_store(s):
    case, slots = s["case"], s["slots"].long()
    P, dt = case["page"], DTYPES[case["dtype"]]
    page, t = slots // P, slots % P
    out = []
    for x, codes, scales in ((s["k"], *s["cache"][:2]), (s["v"], *s["cache"][2:])):
        c, e = _quantise(x.float())
        codes[page, :, t] = c
        scales[page, :, t // 64, t % 16, :, t % 64 // 16] = e
        out.append(_dequantise(codes[page, :, t],
                               scales[page, :, t // 64, t % 16, :, t % 64 // 16]).to(dt))
    return tuple(out)


def _gathered(codes, scales, pages, n):
    """fp32 [heads, n, D] of the first n tokens of the listed pages."""
    P = codes.shape[2]
    e = scales[pages].permute(0, 1, 2, 5, 3, 4).flatten(2, 4)
    x = _dequantise(codes[pages], e)
    return x.transpose(0, 1).flatten(1, 2)[:, :n]


def _plain_cache(s):
    case, q = s["case"], s["q"]
    P, G = case["page"], case["Hq"] // case["Hkv"]
    out = torch.empty_like(q)
    at = 0
    for b, (n, m) in enumerate(zip(s["host_lens"], s["host_new"])):
        pages = s["table"][b, :-(-n // P)].long()
        k = _gathered(s["cache"][0], s["cache"][1], pages, n)
        v = _gathered(s["cache"][2], s["cache"][3], pages, n)
        for r in range(0, m, 256):
            c = min(256, m - r)
            qb = q[at + r:at + r + c].float().transpose(0, 1).reshape(-1, G * c, case["D"])
            x = torch.matmul(qb, k.transpose(1, 2)).view(-1, G, c, n) * s["scale"]
            pos = torch.arange(n - m + r, n - m + r + c, device=q.device)
            late = torch.arange(n, device=q.device)[None] > pos[:, None]
            x.masked_fill_(late, -math.inf)
            x -= x.amax(-1, keepdim=True)
            x.exp_()
            total = x.sum(-1)
            o = torch.matmul(x.view(-1, G * c, n), v).view(-1, G, c, case["D"]) / total[..., None]
            out[at + r:at + r + c] = o.flatten(0, 1).transpose(0, 1).to(q.dtype)
        at += m
    return out


def _means(x, size):
    """Mean of every `size` rows (the last block may be short): summed in 64 bits,
    as the choice of blocks hangs on values next to a border, rounded to fp32."""
    S = x.shape[2]
    full = S // size * size
    parts = [x[:, :, :full].double().unflatten(2, (-1, size)).sum(3) / size]
    if full < S:
        parts.append(x[:, :, full:].double().sum(2, keepdim=True) / (S - full))
    return torch.cat(parts, 2).float()


def _ranked(score, visible, forced, n):
    """The n best visible columns of every row, ascending, -1 behind the last."""
    score = score.masked_fill(forced, math.inf).masked_fill(~visible, -math.inf)
    best = torch.sort(score, dim=-1, descending=True, stable=True)[1][..., :n]
    nk = score.shape[-1]
    best = torch.where(torch.gather(visible.expand_as(score), -1, best), best, nk)
    best = torch.sort(best, -1)[0]
    if best.shape[-1] < n:
        best = torch.nn.functional.pad(best, (0, n - best.shape[-1]), value=nk)
    return torch.where(best < nk, best, -1).int()


def _choice(case, qm, km):
    """Key blocks of every query block: [B, Hq, nq, count]."""
    blk, Sq, Skv = case["block"], case["Sq"], case["Skv"]
    km = km.repeat_interleave(case["Hq"] // case["Hkv"], 1)
    score = torch.matmul(qm.double(), km.double().transpose(2, 3).contiguous())
    nq, nk = score.shape[2:]
    dev = score.device
    j = torch.arange(nk, device=dev)[None]
    if case["causal"]:
        first = torch.arange(nq, device=dev)[:, None] * Q_BLOCK
        last = (first + Q_BLOCK).clamp(max=Sq) - 1
        visible = j * blk <= last + Skv - Sq
        forced = visible & (j >= (first + Skv - Sq).clamp(min=0) // blk)
    else:
        visible = torch.ones(nq, nk, dtype=torch.bool, device=dev)
        forced = torch.zeros_like(visible)
    return _ranked(score, visible, forced, case["count"])


def _plain_sparse(s):
    case, q, k, v = s["case"], s["q"], s["k"], s["v"]
    blk, Sq, Skv, D, G = (case["block"], case["Sq"], case["Skv"], case["D"],
                          case["Hq"] // case["Hkv"])
    km = s["k_means"] if case["kept"] else _means(k, blk)
    index = _choice(case, _means(q, Q_BLOCK), km)
    nq, n = index.shape[2:]
    out = torch.empty_like(q)
    step = max(1, (1 << 27) // (n * blk * D))
    lane = torch.arange(blk, device=q.device)
    for b in range(case["B"]):
        for h in range(case["Hq"]):
            for i in range(0, nq, step):
                c = min(step, nq - i)
                idx = index[b, h, i:i + c].long()
                at = (idx[..., None] * blk + lane).flatten(1)         # [c, n blk]
                bad = (idx < 0).repeat_interleave(blk, 1) | (at >= Skv)
                at = at.clamp(0, Skv - 1)
                kk, vv = k[b, h // G][at].float(), v[b, h // G][at].float()
                rows = (torch.arange(c, device=q.device)[:, None] * Q_BLOCK + i * Q_BLOCK
                        + torch.arange(min(Q_BLOCK, Sq), device=q.device))
                qq = q[b, h][rows.clamp(max=Sq - 1)].float()
                x = torch.bmm(qq, kk.transpose(1, 2).contiguous()) * s["scale"]
                if case["causal"]:
                    hide = bad[:, None] | (at[:, None] > (rows + Skv - Sq)[..., None])
                else:
                    hide = bad[:, None]
                x.masked_fill_(hide, -math.inf)
                x -= x.amax(-1, keepdim=True)
                x.exp_()
                o = torch.bmm(x, vv) / x.sum(-1, keepdim=True)
                out[b, h, i * Q_BLOCK:(i + c) * Q_BLOCK] = o.flatten(0, 1)[:Sq - i * Q_BLOCK].to(
                    q.dtype)
    return out, index


# -- the result in 64 bits ----------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"pages": _exact_pages, "store": _exact_store, "cache": _exact_cache,
            "sparse": _exact_sparse}[case["op"]](s)


def _exact_pages(s):
    """The table and slot map, request by request on the host."""
    P = s["case"]["page"]
    lens, new, free = s["lens"].tolist(), s["new"].tolist(), s["free"].tolist()
    table, used = s["table"].tolist(), s["used"].item()
    slots, cu = [], [0]
    for b, (a, m) in enumerate(zip(lens, new)):
        for page in range(-(-a // P), -(-(a + m) // P)):
            table[b][page] = free[used]
            used += 1
        slots += [table[b][p // P] * P + p % P for p in range(a, a + m)]
        cu.append(cu[-1] + m)
    i32 = dict(dtype=torch.int32, device="cuda")
    return (torch.tensor(slots, **i32), torch.tensor(cu, **i32),
            torch.tensor([a + m for a, m in zip(lens, new)], **i32), torch.tensor([used], **i32),
            torch.tensor(table, **i32))


def _exact_store(s):
    out = []
    for x in (s["k"], s["v"]):
        x = x.double().unflatten(-1, (-1, 32))
        top = x.abs().amax(-1, keepdim=True)
        unit = torch.exp2(torch.floor(torch.log2(top.clamp(min=2.0 ** -124))) - 2)
        a = x.abs() / unit
        a = torch.where(a < 2, torch.round(2 * a) / 2,
                        torch.where(a < 4, torch.round(a), 2 * torch.round(a / 2)))
        out.append((torch.copysign(a.clamp(max=6), x) * unit).flatten(-2))
    return tuple(out)


def _values64(codes, scales):
    """fp64 [pages, heads, page, D] of a cache's pages, by the format's fields."""
    c = torch.stack((codes % 16, codes // 16), -1).flatten(-2).double()
    sign = torch.where(c >= 8, -1.0, 1.0).double()
    c = c % 8
    e, m = torch.floor(c / 2), c % 2
    a = torch.where(e == 0, m / 2, (1 + m / 2) * torch.exp2(e - 1))
    n, H, A, _, nb, _ = scales.shape
    u = torch.exp2(scales.double() - 127).permute(0, 1, 2, 5, 3, 4).reshape(n, H, A * 64, nb)
    return sign * a * u.repeat_interleave(32, -1)


def _exact_cache(s):
    case = s["case"]
    P, G, D = case["page"], case["Hq"] // case["Hkv"], case["D"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for b, (n, m) in enumerate(zip(s["host_lens"], s["host_new"])):
        pages = s["table"][b, :-(-n // P)].long()
        for h in range(case["Hkv"]):
            k = _values64(s["cache"][0][pages][:, h:h + 1], s["cache"][1][pages][:, h:h + 1])
            v = _values64(s["cache"][2][pages][:, h:h + 1], s["cache"][3][pages][:, h:h + 1])
            k, v = k.reshape(-1, D)[:n], v.reshape(-1, D)[:n]
            for j in range(h * G, h * G + G):
                z = (s["q"][at:at + m, j].double() @ k.T) * s["scale"]
                z += torch.triu(torch.full((m, n), -math.inf, dtype=torch.float64, device="cuda"),
                                diagonal=n - m + 1)
                w = torch.exp(z - z.amax(1, keepdim=True))
                out[at:at + m, j] = (w @ v) / w.sum(1, keepdim=True)
        at += m
    return out


def _exact_sparse(s):
    case = s["case"]
    blk, Sq, Skv = case["block"], case["Sq"], case["Skv"]
    B, Hq, G, n = case["B"], case["Hq"], case["Hq"] // case["Hkv"], case["count"]
    nq, nk = -(-Sq // Q_BLOCK), -(-Skv // blk)
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    index = torch.full((B, Hq, nq, n), -1, dtype=torch.int32)
    ends = [min(Skv, (j + 1) * blk) for j in range(nk)]

    def means(x, size):
        c = torch.nn.functional.pad(x.double(), (0, 0, 0, -x.shape[0] % size))
        c = c.view(-1, size, x.shape[1]).sum(1)
        rows = torch.full((len(c), 1), float(size), dtype=torch.float64, device="cuda")
        rows[-1] = x.shape[0] - size * (len(c) - 1)
        return (c / rows).float().double()

    for b in range(B):
        for h in range(Hq):
            q, k, v = s["q"][b, h], s["k"][b, h // G].double(), s["v"][b, h // G].double()
            score = (means(q, Q_BLOCK) @ means(s["k"][b, h // G], blk).T).cpu().numpy()
            for i in range(nq):
                r0, r1 = i * Q_BLOCK, min(Sq, (i + 1) * Q_BLOCK)
                lo, hi = r0 + Skv - Sq, r1 - 1 + Skv - Sq
                seen = hi // blk + 1 if case["causal"] else nk
                must = list(range(max(lo, 0) // blk, seen)) if case["causal"] else []
                rest = (-score[i, :seen - len(must)]).argsort(kind="stable")[:n - len(must)]
                mine = sorted(must + rest.tolist())
                index[b, h, i, :len(mine)] = torch.tensor(mine, dtype=torch.int32)
                at = torch.cat([torch.arange(j * blk, ends[j]) for j in mine]).cuda()
                z = (q[r0:r1].double() @ k[at].T) * s["scale"]
                if case["causal"]:
                    pos = torch.arange(lo, hi + 1, device="cuda")
                    z = torch.where(at[None] <= pos[:, None], z, -math.inf)
                w = torch.exp(z - z.amax(1, keepdim=True))
                out[b, h, r0:r1] = (w @ v[at]) / w.sum(1, keepdim=True)
    return out, index.cuda()
