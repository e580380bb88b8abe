"""Block routing by itself and attention over what it picks, on gfx950.

``relation_select_packed`` routes each query to a local window and the router's top
blocks and keeps one anchor and K partners of them.  Here the router's picks come
out (``block_route``) and all of those positions are attended to
(``routed_attention``), with the same scores, tie rule, window and ring-buffer
conventions (``kernels/relation_select.py``, ``kernels/ring.py``); the picks may also
come from any other source.  No reference counterpart.

Decode forms take one query per batch row and a position that is 0-d or, unlike the
selection's, [B] (requests of different lengths); sequence forms take a query axis and
one position per query, [Tq] or [B,Tq].  A query at a negative position (a padded row)
sees nothing: its picks are -1, its output 0, its log-sum-exp -inf.

Inference only: the operators have no gradient.
"""
from __future__ import annotations

import torch
from torch import Tensor

from relation_lm import _native  # noqa: F401  (registers torch.ops.rlm)


def block_route(router_query: Tensor, block_mean: Tensor, block_std: Tensor, gamma: Tensor,
                bias: Tensor, position: Tensor, block_size: int, local_window: int,
                top_blocks: int, strict_valid: bool, ring: bool = False
                ) -> tuple[Tensor, Tensor]:
    """The router's picks for one query per batch row.

    router_query [B,RD], or [B,S,RD] with S routings of a row (one per key head, say);
    block_mean / block_std [B,NB,H,HD] fp32 (``block_statistics``,
    ``router_cache_update``), gamma [H], bias [H,RB].  Returns (blocks int32 [B,(S,)TOP],
    scores fp32), best first, ties to the lowest block, -1 and -inf where fewer blocks are
    complete (``strict_valid``: wholly before the local window).  A block whose score is
    NaN or at most -1e30 is not picked; a head of -inf adds nothing to a score.  ``ring``: the statistics are a ring buffer's;
    blocks stay absolute.
    """
    return torch.ops.rlm.block_route(router_query, block_mean, block_std, gamma, bias, position,
                                     block_size, local_window, top_blocks, strict_valid, ring)


def block_route_seq(router_query: Tensor, block_mean: Tensor, block_std: Tensor, gamma: Tensor,
                    bias: Tensor, positions: Tensor, block_size: int, local_window: int,
                    top_blocks: int, strict_valid: bool) -> tuple[Tensor, Tensor]:
    """Sequence form: router_query [B,Tq,RD] or [B,Tq,S,RD], positions [Tq] or [B,Tq];
    returns (blocks [B,Tq,(S,)TOP], scores)."""
    return torch.ops.rlm.block_route_seq(router_query, block_mean, block_std, gamma, bias,
                                         positions, block_size, local_window, top_blocks,
                                         strict_valid)


def routed_attention(query: Tensor, key_cache: Tensor, value_cache: Tensor, blocks: Tensor,
                     position: Tensor, block_size: int, local_window: int,
                     scale: float | None = None, ring: bool = False) -> tuple[Tensor, Tensor]:
    """Attention of one token per batch row over its window and its picked blocks.

    query [B,Hq,D], key_cache / value_cache [B,T,Hk,D] (Hq a multiple of Hk; any strides
    with unit stride in D), blocks int32 [B,TOP] or, with picks per key head, [B,Hk,TOP];
    scale defaults to D^-1/2.  Positions [t - local_window + 1, t] and the picked blocks'
    positions before them, each once.  Returns (out [B,Hq,D] in query's dtype,
    log-sum-exp fp32 [B,Hq]).  Sums and exponentials are fp32; 16-bit types round each
    weight to the type before it meets the values (bf16: 2^-8 at most, relative).
    ``ring``: position p lives in row p mod T, and the rows hold (t - T, t]: a chunk whose
    later tokens are in the ring already has lost the earlier ones' farthest positions.
    D a multiple of 8 up to 256, TOP <= 64.
    """
    return torch.ops.rlm.routed_attention(query, key_cache, value_cache, blocks, position,
                                          block_size, local_window, scale, ring)


def routed_attention_seq(query: Tensor, key_cache: Tensor, value_cache: Tensor, blocks: Tensor,
                         positions: Tensor, block_size: int, local_window: int,
                         scale: float | None = None) -> tuple[Tensor, Tensor]:
    """Sequence form: query [B,Tq,Hq,D], blocks [B,Tq,TOP] or [B,Tq,Hk,TOP], positions [Tq]
    or [B,Tq]; returns (out [B,Tq,Hq,D], log-sum-exp fp32 [B,Tq,Hq]).  Linear caches
    only; weights are rounded as there."""
    return torch.ops.rlm.routed_attention_seq(query, key_cache, value_cache, blocks, positions,
                                              block_size, local_window, scale)
