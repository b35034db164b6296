"""Norms of queries and keys for each head, with the position rotation in the same pass.

What models do with the rows of their projections before attention: an RMS norm over
every head's dims, times a weight, then pairs of dims turned by angles of the token's
position. The results are what :func:`gfx906_amd.attn`, :func:`gfx906_amd.kv4.store` and
:func:`gfx906_amd.kv8.store` read. Formulas and the C ABI are in
``include/gfx906_amd_attn.h``. The call runs on the current stream, raises
``RuntimeError`` for what it does not accept, has no fallback and no gradient. The
reference has no counterpart.
"""

from __future__ import annotations

import torch

from .loader import extension


def angles(rows, pairs, base=10000.0, device="cuda"):
    """``(cos, sin)`` tables, fp32 ``[rows, pairs]``: position p turns pair n by
    ``p * base ** (-n / pairs)``, computed in 64 bits."""
    rate = float(base) ** (-torch.arange(pairs, dtype=torch.float64, device=device) / pairs)
    angle = torch.arange(rows, dtype=torch.float64, device=device)[:, None] * rate
    return angle.cos().float(), angle.sin().float()


def norm_rotate(q, k=None, q_weight=None, k_weight=None, cos=None, sin=None, positions=None,
                eps=1e-6, neighbours=False, out=None):
    """``(q', k')`` of the rows of ``q`` and ``k``: ``x / sqrt(mean(x^2) + eps) * weight``, then the
    first ``R`` dims turned in pairs; in fp32, rounded once. Without ``k`` the result is ``q'``.

    ``q`` is ``[T, Hq, D]`` or ``[B, S, Hq, D]``, ``k`` the same with its own heads (fp16 or bf16, D
    a multiple of 8 up to 512). Strides are free: pass parts of a fused projection as they are, and a
    ``[B, H, S, D]`` tensor as ``x.transpose(1, 2)`` (results keep the order of dense inputs whose head dim
    is contiguous; other rows are copied).
    Weights are ``[D]``, of the rows' type or fp32 (None: 1). ``cos`` and ``sin`` are fp32 ``[N, R/2]``
    (None: no rotation); a token's row is its entry in ``positions`` (int32 ``[T]`` or ``[B, S]``) or,
    without them, its place in the sequence. A position outside the tables gives NaN in the turned
    dims. Pairs are ``(n, n + R/2)`` (R a multiple of 16), or with ``neighbours`` ``(2n, 2n + 1)``
    (R a multiple of 8). ``out``: tensors for the results, ``(q', k')``; they may be ``q`` and ``k``."""
    if out is None:
        out = (None, None)
    elif k is None and isinstance(out, torch.Tensor):
        out = (out, None)
    q_out, k_out = out
    res = extension().norm_rotate(q, k, q_weight, k_weight, cos, sin, positions, float(eps),
                                  bool(neighbours), q_out, k_out)
    return res[0] if k is None else tuple(res)
