"""Rotary positions on gfx950, alone or with the cache writes of key and value.

No reference counterpart: the reference's routed path knows positions only by the
router's distance buckets.  ``rotary_to_caches`` stands to an attention layer's
caches as ``packed_projection_to_caches`` stands to the sparse caches: the token
rows go where the next operator reads them, in the launch that computes them.

Inference only: the operators have no gradient.
"""
from __future__ import annotations

import torch
from torch import Tensor

from relation_lm import _native  # noqa: F401  (registers torch.ops.rlm)


def rotary_positions(query: Tensor, key: Tensor, positions: Tensor, frequencies: Tensor,
                     interleaved: bool = False, scale: float = 1.0) -> tuple[Tensor, Tensor]:
    """Rotates query [B,Tq,Hq,D] and key [B,Tq,Hk,D] by their positions.

    Pair i of a head turns by ``positions * frequencies[i]`` and is multiplied by
    ``scale``; pair i is the features (i, F + i), or (2 i, 2 i + 1) where
    ``interleaved``.  ``frequencies`` is [F] fp32 with 2 F <= D: features from 2 F on
    pass unchanged.  Long contexts are a matter of ``frequencies`` (stretched, or
    stretched per pair) and ``scale``.  ``positions`` is 0-d, [Tq] or [B,Tq]; the
    angle is reduced in float64, so far positions keep their turn's fraction, and its
    sine and cosine are fp32.
    query and key may be strided views (of one projection's rows, say).
    """
    return torch.ops.rlm.rotary_positions(query, key, positions, frequencies, interleaved, scale)


def rotary_to_caches(query: Tensor, key: Tensor, value: Tensor, position: Tensor,
                     frequencies: Tensor, key_cache: Tensor, value_cache: Tensor,
                     interleaved: bool = False, scale: float = 1.0, ring: bool = False,
                     lengths: Tensor | None = None) -> Tensor:
    """``rotary_positions`` of Tq tokens that follow each other from ``position`` (0-d, or
    [B] with one first position per batch row); returns the rotated query and writes the
    rotated key and the value [B,Tq,Hk,D] to the tokens' rows of ``key_cache`` and
    ``value_cache`` [B,T,Hk,D] (any strides with unit stride in D).

    Tokens from ``lengths[b]`` on (padding of a ragged prompt batch) and positions
    outside [0, T) leave the caches as they are, and so do tokens that would stand past
    int64's last position (they turn as that one does).  ``ring``: position p goes to row
    p mod T, T a power of two, Tq <= T.  A decode step passes Tq = 1; several tokens
    written into a ring at once overwrite what the first of them could still see.
    """
    return torch.ops.rlm.rotary_to_caches(query, key, value, position, frequencies, key_cache,
                                          value_cache, interleaved, scale, ring, lengths)
