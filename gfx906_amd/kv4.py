"""A paged key/value cache held in 4 bits, and attention over it.

Keys and values are stored in the OCP MX format MXFP4: E2M1 numbers with one
E8M0 scale per 32 head dims of a token, 17 bytes per 32 values (fp16 takes 64),
which gfx950 converts in hardware. A serving step goes

    plan = kv4.plan_pages(lens, new_lens, table, free_pages, used, cache.page, tokens)
    kv4.store(cache, k, v, plan.slots)
    out = kv4.attn(q, cache, table, plan.lens, scale, cu_q=plan.cu_new, max_q=longest)

with every length, table and slot on the GPU: no call synchronises, and all of
them may be captured into a HIP graph. The layout and what happens to values out
of range is described in ``include/gfx906_amd_attn.h``. All calls run on the
current stream, raise ``RuntimeError`` for what they do not accept, and have no
fallback. The reference has no counterpart.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from .loader import extension

PAGE_SIZES = (64, 128, 256)   # tokens a page may hold
HEAD_DIMS = (64, 128)


class Cache(NamedTuple):
    """Codes ``[pages, heads, page, D/2]`` and scales ``[pages, heads, page/64, 16,
    D/32, 4]`` of the keys and of the values, uint8 (see :func:`new_cache`)."""

    k: torch.Tensor
    k_scale: torch.Tensor
    v: torch.Tensor
    v_scale: torch.Tensor

    @property
    def page(self) -> int:
        """Tokens in a page."""
        return self.k.shape[2]


class Plan(NamedTuple):
    """What :func:`plan_pages` returns, int32 on the GPU."""

    slots: torch.Tensor    # [tokens] slot of every new token (-1: none)
    cu_new: torch.Tensor   # [B + 1] first new token of every request, and their number
    lens: torch.Tensor     # [B] tokens of every request with the new ones
    used: torch.Tensor     # [1] free pages taken so far
    missing: torch.Tensor  # [1] pages that could not be taken


def new_cache(pages, page, heads, head_dim, device="cuda") -> Cache:
    """An empty cache (every value 0) of ``pages`` pages of ``page`` tokens."""
    if page not in PAGE_SIZES or head_dim not in HEAD_DIMS:
        raise ValueError(f"new_cache: page must be one of {PAGE_SIZES} and head_dim of {HEAD_DIMS}")
    codes = (pages, heads, page, head_dim // 2)
    scales = (pages, heads, page // 64, 16, head_dim // 32, 4)
    return Cache(*(torch.zeros(s, dtype=torch.uint8, device=device)
                   for s in (codes, scales, codes, scales)))


def plan_pages(lens, new_lens, table, free_pages, used, page, tokens) -> Plan:
    """Pages and slots for ``new_lens[b]`` tokens behind the ``lens[b]`` cached ones
    of every request (int32 ``[B]``, B <= 4096).

    ``table`` (int32 ``[B, W]``) names the pages of a request in its row; pages that
    are lacking are taken from ``free_pages[used:]`` (``used``: int32 ``[1]``) in the
    order of the requests and written into the table. ``tokens`` is the length of
    the slot list: at least the sum of ``new_lens`` (slots behind it are -1)."""
    return Plan(*extension().kv4_plan_pages(lens, new_lens, table, free_pages, used, page, tokens))


def store(cache, k, v, slots) -> None:
    """Quantises rows of ``k`` and ``v`` (``[T, heads, D]``, fp16 or bf16) into the
    cache at ``slots`` (int32 ``[T]``; a slot outside the cache is skipped; the others
    must differ)."""
    extension().kv4_store(k, v, slots, *cache)


def load(cache, slots, dtype=torch.float16):
    """The ``(k, v)`` rows ``[T, heads, D]`` that the cache holds at ``slots``, in
    ``dtype`` (zeros for a slot outside the cache)."""
    return tuple(extension().kv4_load(*cache, slots, dtype))


def attn(q, cache, table, lens, scale, cu_q=None, max_q=None, causal=True, out=None):
    """softmax(scale * q k^T) v over the cache: ``q`` ``[T, Hq, D]`` (fp16 or bf16; Hq
    a multiple of the cache's heads), the result in a new tensor or in ``out``.

    Rows ``cu_q[b] .. cu_q[b+1]`` (int32 ``[B + 1]``) are the queries of request b,
    which holds ``lens[b]`` tokens (int32 ``[B]``) in the pages of ``table``'s row b;
    without ``cu_q`` row b is the one query of request b. With ``causal`` they are
    the request's last tokens and see none behind themselves. ``max_q``, for ``cu_q``: at
    least the most queries of a request (queries past it are not computed); without it
    T is taken, and a decoding step pays for what it does not need. Rows outside
    every request are left as they were (in a new tensor: unset). ``out`` may be ``q``
    itself and must not overlap the other arguments otherwise. Rows that see no
    key are 0; keys without a page weigh nothing."""
    if max_q is None:
        max_q = 1 if cu_q is None else q.shape[0]
    return extension().kv4_attn(q, *cache, table, lens, float(scale), cu_q, max_q, causal, out)
