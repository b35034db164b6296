"""A paged key/value cache held in 8 bits, attention over it, and eviction by the
attention that its pages got.

Keys and values are E4M3 numbers with one power-of-two scale per 64 tokens and head: half
the bytes of fp16, twice those of :mod:`gfx906_amd.kv4` at 2^-4 relative error instead
of 2^-2. Requests, page tables and lengths are those of kv4, with its page planning:

    plan = kv8.plan_pages(lens, new_lens, table, free_pages, used, cache.page, tokens)
    kv8.store(cache, k, v, table, plan.lens, plan.cu_new, weights)
    out, lse = kv8.attn(q, cache, table, plan.lens, scale, cu_q=plan.cu_new, max_q=longest, lse=True)
    kv8.weigh(weights, q, lse, cache, table, plan.lens, scale, cu_q=plan.cu_new, max_q=longest)
    gone = kv8.evict(weights, table, plan.lens, keep, free_pages, plan.used)

and the next step goes on with ``gone.lens`` and ``gone.used``. Without eviction the weights, the lse and
the last two calls are left out. Everything stays on the GPU: no call synchronises, and
all of them may be captured into a HIP graph. The layout and what happens to values out of
range is described in ``include/gfx906_amd_attn.h``. All calls run on the current
stream, raise ``RuntimeError`` for what they do not accept, and have no fallback. The
reference has no counterpart.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from .kv4 import HEAD_DIMS, PAGE_SIZES, Plan, plan_pages  # noqa: F401
from .loader import extension

BLOCK = 64   # tokens of a head that share a scale


class Cache(NamedTuple):
    """Codes of the keys ``[pages, heads, page, D]`` and of the values ``[pages, heads,
    page/64, D, 64]``, uint8, each followed by its scales, fp32 ``[pages, heads, page/64]``
    (see :func:`new_cache`)."""

    k: torch.Tensor
    k_scale: torch.Tensor
    v: torch.Tensor
    v_scale: torch.Tensor

    @property
    def page(self) -> int:
        """Tokens in a page."""
        return self.k.shape[2]


class Evicted(NamedTuple):
    """What :func:`evict` returns, int32 on the GPU."""

    lens: torch.Tensor   # [B] tokens of every request that are left
    used: torch.Tensor   # [1] free pages that are still taken
    lost: torch.Tensor   # [1] pages that had no place in the free list


def new_cache(pages, page, heads, head_dim, device="cuda") -> Cache:
    """An empty cache (every value 0) of ``pages`` pages of ``page`` tokens."""
    if page not in PAGE_SIZES or head_dim not in HEAD_DIMS:
        raise ValueError(f"new_cache: page must be one of {PAGE_SIZES} and head_dim of {HEAD_DIMS}")
    blocks = (pages, heads, page // BLOCK)
    k = torch.zeros(pages, heads, page, head_dim, dtype=torch.uint8, device=device)
    v = torch.zeros(*blocks, head_dim, BLOCK, dtype=torch.uint8, device=device)
    return Cache(k, torch.full(blocks, 2.0 ** -15, device=device),
                 v, torch.full(blocks, 2.0 ** -15, device=device))


def new_weights(cache):
    """Weights of a cache's blocks, fp32 ``[pages, heads, page/64]``, all 0."""
    return torch.zeros_like(cache.k_scale)


def store(cache, k, v, table, lens, cu_new=None, weights=None) -> None:
    """Quantises rows of ``k`` and ``v`` (``[T, heads, D]``, fp16 or bf16) into the cache.

    Rows ``cu_new[b] .. cu_new[b+1]`` (int32 ``[B + 1]``; without it row b) are the last tokens
    of request b, which holds ``lens[b]`` tokens, these among them (int32 ``[B]``), in the pages of
    ``table``'s row b. A block of 64 tokens that gets larger values than it holds takes a larger scale,
    and its older tokens are rounded to it; no block may be written for two requests. Rows without a page
    are passed over. ``weights``: accumulated weights start at 0 for the blocks that begin here."""
    extension().kv8_store(k, v, *cache, table, lens, cu_new, weights)


def load(cache, slots, dtype=torch.float16):
    """The ``(k, v)`` rows ``[T, heads, D]`` that the cache holds at ``slots`` (page * page size +
    place, int32 ``[T]``), in ``dtype``, exactly; zeros for a slot outside the cache."""
    return tuple(extension().kv8_load(*cache, slots, dtype))


def attn(q, cache, table, lens, scale, cu_q=None, max_q=None, causal=True, out=None, lse=False):
    """softmax(scale * q k^T) v over the cache: ``q`` ``[T, Hq, D]`` (fp16 or bf16; Hq
    a multiple of the cache's heads), the result in a new tensor or in ``out``; with ``lse`` the pair of
    it and of the logarithms of the sums of exp(scale * q k), fp32 ``[T, Hq]``.

    Rows ``cu_q[b] .. cu_q[b+1]`` (int32 ``[B + 1]``) are the queries of request b,
    which holds ``lens[b]`` tokens (int32 ``[B]``) in the pages of ``table``'s row b;
    without ``cu_q`` row b is the one query of request b. With ``causal`` they are
    the request's last tokens and see none behind themselves. ``max_q``, for ``cu_q``: at
    least the most queries of a request (queries past it are not computed); without it
    T is taken, and a decoding step pays for what it does not need. Rows outside
    every request are left as they were (in a new tensor: unset). ``out`` may be ``q``
    itself and must not overlap the other arguments otherwise. Rows that see no
    key are 0, with an lse of -inf; keys without a page weigh nothing."""
    if max_q is None:
        max_q = 1 if cu_q is None else q.shape[0]
    res = extension().kv8_attn(q, *cache, table, lens, float(scale), cu_q, max_q, causal, out,
                               bool(lse))
    return tuple(res) if lse else res[0]


def weigh(weights, q, lse, cache, table, lens, scale, cu_q=None, max_q=None, causal=True) -> None:
    """Adds to ``weights`` (:func:`new_weights`) the attention that every block's tokens get
    from the queries: the softmax weights summed over tokens, queries and the query heads of
    a kv head. ``lse`` is what :func:`attn` returned for the same arguments; queries whose weights are not
    wanted can be left out with ``cu_q`` and ``causal`` as there."""
    if max_q is None:
        max_q = 1 if cu_q is None else q.shape[0]
    extension().kv8_weigh(weights, q, lse, *cache, table, lens, float(scale), cu_q, max_q, causal)


def evict(weights, table, lens, keep, free_pages, used, first=1, recent=1) -> Evicted:
    """Pages of requests over their budgets go back to the free list: request b keeps ``keep[b]``
    pages (int32 ``[B]``), the ones of least weight go (``weights``, summed over heads and blocks in 64
    bits; of equal ones the earlier), but never its ``first`` first ones or its ``recent`` last ones.

    ``table`` (int32 ``[B, W]``) closes up in place; the pages go into ``free_pages`` in front of
    entry ``used`` (int32 ``[1]``), from where :func:`plan_pages` takes them. Entries without a page, which
    :func:`plan_pages` leaves when there are none, leave the rows before all others, and only pages go back.
    What is left keeps its order, and whole pages go, so nothing in the cache moves. A page that requests share goes back once for
    each of them."""
    return Evicted(*extension().kv8_evict(weights, table, lens, keep, free_pages, used, first, recent))
