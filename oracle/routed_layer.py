"""Oracle of the routed attention layer's operators -- TEST INFRASTRUCTURE ONLY (see
oracle/__init__.py).

Rotary positions, block routing, attention over a window and picked blocks, and the gated
residual norm, in float64 from their definitions.  Block scores and picks are those of
oracle/select.py.  ``attention`` also returns what its tolerance is made of: the sums of
weights times |value| and the sizes of the score products.
"""
from __future__ import annotations

import numpy as np

from oracle import select as osel


def _f64(x) -> np.ndarray:
    return np.asarray(x, dtype=np.float64)


def positions_of(positions, batch: int, queries: int) -> np.ndarray:
    """0-d, [Tq] or [B,Tq] as [B,Tq]."""
    return np.broadcast_to(np.asarray(positions, dtype=np.int64), (batch, queries))


def rotary(x, positions, frequencies, interleaved: bool, scale: float) -> np.ndarray:
    """x [B,Tq,H,D] as complex pairs times scale * exp(i position frequency)."""
    x = _f64(x).copy()
    n = len(frequencies)
    t = positions_of(positions, x.shape[0], x.shape[1]).astype(np.float64)
    turn = scale * np.exp(1j * t[..., None] * _f64(frequencies))[:, :, None, :]
    one = slice(0, 2 * n, 2) if interleaved else slice(0, n)
    two = slice(1, 2 * n, 2) if interleaved else slice(n, 2 * n)
    z = (x[..., one] + 1j * x[..., two]) * turn
    x[..., one], x[..., two] = z.real, z.imag
    return x


def rotary_to_caches(query, key, value, position, frequencies, key_cache, value_cache,
                     interleaved: bool, scale: float, ring: bool, lengths=None):
    """Returns (rotated query, key cache, value cache) with untouched rows as they were."""
    batch, queries = np.shape(query)[:2]
    rows = np.shape(key_cache)[1]
    first = np.broadcast_to(np.asarray(position, dtype=np.int64), (batch,))
    t = first[:, None] + np.arange(queries)
    rotated = rotary(key, t, frequencies, interleaved, scale)
    keys, values = _f64(key_cache).copy(), _f64(value_cache).copy()
    for b in range(batch):
        for i in range(queries):
            row = t[b, i] % rows if ring else t[b, i]
            if t[b, i] < 0 or row >= rows or (lengths is not None and i >= lengths[b]):
                continue
            keys[b, row], values[b, row] = rotated[b, i], _f64(value)[b, i]
    return rotary(query, t, frequencies, interleaved, scale), keys, values


def block_route(router_query, mean, std, gamma, bias, positions, block_size: int,
                local_window: int, top_blocks: int, strict_valid: bool, ring: bool = False):
    """router_query [B,Tq,S,RD]; returns (blocks int32, scores float32) [B,Tq,S,TOP]."""
    batch, queries, slots = np.shape(router_query)[:3]
    t = np.repeat(positions_of(positions, batch, queries)[..., None], slots, -1).reshape(-1)
    batch_of = np.repeat(np.arange(batch), queries * slots)
    flat = _f64(router_query).reshape(batch * queries * slots, -1)
    options = dict(block_size=block_size, local_window=local_window, strict_valid=strict_valid)
    if ring:
        scores, held = osel.ring_block_scores(flat, mean, std, gamma, bias, batch_of, t, **options)
        blocks, valid = osel.ring_pick_blocks(scores, held, top_blocks)
        order = np.argsort(held, axis=1, kind="stable")
        ranked = -np.sort(-np.take_along_axis(scores, order, 1), axis=1, kind="stable")
    else:
        scores = osel.block_scores(flat, mean, std, gamma, bias, batch_of, t, **options)
        blocks, valid = osel.pick_blocks(scores, top_blocks)
        ranked = -np.sort(-scores, axis=1, kind="stable")
    value = np.full((len(t), top_blocks), -np.inf, np.float32)
    take = min(top_blocks, ranked.shape[1])
    value[:, :take] = ranked[:, :take]
    shape = (batch, queries, slots, top_blocks)
    return (np.where(valid, blocks, -1).astype(np.int32).reshape(shape),
            np.where(valid, value, -np.inf).astype(np.float32).reshape(shape))


def seen_positions(t: int, picks, rows: int, block_size: int, local_window: int,
                   ring: bool) -> np.ndarray:
    """The positions that a query at t attends to, ascending."""
    low = max(0, t - rows + 1) if ring else 0
    high = t + 1 if ring else min(t + 1, rows)
    p = np.arange(low, max(high, low))
    near = p > t - local_window
    return p[near | np.isin(p // block_size, [j for j in np.asarray(picks) if j >= 0])]


def attention(query, key_cache, value_cache, blocks, positions, block_size: int,
              local_window: int, scale: float, ring: bool = False):
    """query [B,Tq,Hq,D], blocks [B,Tq,Hk or 1,TOP].  Returns out, lse, and per output
    sum_p w_p |v_p| and the largest sum_d |q_d k_d| * scale."""
    query = _f64(query)
    batch, queries, heads, dim = query.shape
    rows, kv_heads = np.shape(key_cache)[1:3]
    group = heads // kv_heads
    t = positions_of(positions, batch, queries)
    out = np.zeros(query.shape)
    spread = np.zeros(query.shape)
    lse = np.full(query.shape[:3], -np.inf)
    size = np.zeros(query.shape[:3])
    for b in range(batch):
        for i in range(queries):
            for h in range(kv_heads):
                picks = blocks[b, i, h if np.shape(blocks)[2] > 1 else 0]
                p = seen_positions(int(t[b, i]), picks, rows, block_size, local_window, ring)
                if not len(p):
                    continue
                k = _f64(key_cache[b, p % rows if ring else p, h])
                v = _f64(value_cache[b, p % rows if ring else p, h])
                mine = slice(h * group, (h + 1) * group)
                s = query[b, i, mine] @ k.T * scale
                most = s.max(axis=1, keepdims=True)
                w = np.exp(s - most)
                total = w.sum(axis=1, keepdims=True)
                w /= total
                out[b, i, mine] = w @ v
                spread[b, i, mine] = w @ np.abs(v)
                lse[b, i, mine] = (most + np.log(total))[:, 0]
                size[b, i, mine] = (np.abs(query[b, i, mine]) @ np.abs(k).T).max(axis=1) * scale
    return out, lse, spread, size


def gated_residual_norm(branch, residual, gate, norm_weight, norm_bias, norm_eps, post_weight,
                        post_bias, residual_scale, rms, post_eps):
    """[N,D] rows; returns (hidden, normalized)."""
    def norm(x, w, b, eps):
        if not rms:
            x = x - x.mean(-1, keepdims=True)
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * _f64(w)
        return x if b is None else x + _f64(b)

    y = _f64(branch)
    if post_weight is not None:
        y = norm(y, post_weight, post_bias, post_eps)
    hidden = residual_scale * _f64(residual) + y / (1 + np.exp(-_f64(gate)))
    return hidden, norm(hidden, norm_weight, norm_bias, norm_eps)
