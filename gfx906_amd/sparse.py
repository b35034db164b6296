"""Sparse attention: every 128 query rows read the key blocks that suit them best.

``attn`` does all of it; its parts serve programs that keep some of the results:

    k_means = sparse.block_means(k, 64)             # a decoder keeps them beside its keys
    index = sparse.choose(q, k_means, 32, k.shape[2])
    out = sparse.attn_blocks(q, k, v, scale, index)

A block's score is the product of the query block's mean and the key block's mean,
added up in 64 bits in one order, so that the choice is the same whichever of these
calls makes it, and for a query alone or in a batch (see
``include/gfx906_amd_attn.h``). q is ``[B, Hq, Sq, D]``, k and v
``[B, Hkv, Skv, D]``, fp16 or bf16, D 64 or 128, Hq a multiple of Hkv; strided views
with a contiguous head dim are read in place. All calls run on the current stream
without synchronising, raise ``RuntimeError`` for what they do not accept, and have
no fallback. The reference has no counterpart: its attention reads every key.
"""

from __future__ import annotations

from .loader import extension

Q_BLOCK = 128   # query rows that share one choice


def block_means(x, block):
    """fp32 means ``[B, H, ceil(S/block), D]`` of every ``block`` (64 or 128) rows of
    ``x`` ``[B, H, S, D]``; the last block may be short."""
    return extension().sparse_block_means(x, block)


def select(q_means, k_means, count, q_len, k_len, block=64, causal=False):
    """int32 ``[B, Hq, ceil(q_len/128), count]``: the ``count`` key blocks with the
    largest products of means for every query block, ascending, -1 behind the last
    (equal products: the lower index first).

    With ``causal`` row r stands at key position ``r + k_len - q_len``; the blocks that
    hold a query block's own positions are always taken (``count`` must leave room
    for them: 128/block + 1, or as many as fewer queries span)."""
    return extension().sparse_select(q_means, k_means, count, q_len, k_len, block, causal)


def choose(q, k_means, count, k_len, block=64, causal=False):
    """``select`` for the query rows themselves, whose block means are taken on the way."""
    return extension().sparse_choose(q, k_means, count, k_len, block, causal)


def attn_blocks(q, k, v, scale, index, block=64, causal=False, out=None):
    """softmax(scale * q k^T) v over the keys of the blocks in ``index``
    (``[B, Hq, ceil(Sq/128), count]``, as ``select`` returns it), in a new tensor or
    in ``out`` (which may be ``q`` itself, and must not overlap ``k`` or ``v``). An entry
    that names no block, or is not above the valid entries before it, is passed over; a
    row that sees no key is 0."""
    return extension().sparse_attn(q, k, v, float(scale), index, block, causal, out)


def attn(q, k, v, scale, count, block=64, causal=False, k_means=None, out=None):
    """Attention over the ``count`` best key blocks of every query block; returns the
    output and the choice (see ``select``). ``k_means``: ``block_means(k, block)``
    where the program holds them (copied here unless packed). ``scale`` must be positive, as the choice takes the
    largest products."""
    if not scale > 0:
        raise ValueError("sparse.attn: scale must be positive")
    if k_means is None:
        k_means = block_means(k, block)
    elif k_means.shape[:2] != k.shape[:2]:
        raise ValueError("sparse.attn: k_means must have k's batches and heads")
    index = choose(q, k_means, count, k.shape[2], block, causal)
    return attn_blocks(q, k, v, scale, index, block, causal, out), index
