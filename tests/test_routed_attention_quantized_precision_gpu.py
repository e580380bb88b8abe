"""How exact attention over 8-bit caches is: queries that see one key, whose outputs are that key's value and
whose log-sum-exp is its score, and few keys, within the bound of test_routed_attention_quantized_gpu.py for as
many as are seen.

One key, a query of one feature q (u = eps(fp32) / 2, h = half a step of the output's type, P = 1 to 3 bf16
parts; a matrix instruction is off by at most 2 u of the largest of its sums):
 - the score takes P products (2 P u), up to four roundings of the factors scale log2(e) ks and of their
   products, log2(sum) = 0 up to u |score| and 2 u, and ln 2's two: |lse - exact| <= (2 P + 8) u |lse| + 4 u.
   Without an fp32 query's third part it would be off by up to 2^-18 = 64 u.
 - the weight is 1 up to u |score|, of which the sum is the same: it leaves out by division.  Weight times
   scale rounds by u, its parts leave p (2^-18 for two, 2^-26 for three), their products 6 u, the reciprocal
   and its product 3 u:                       |out - exact| <= h |out| + (12 u + p) |out|.
   Without the last part it would be off by up to 2^-9 (of two), 2^-18 (of three).
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from launched import launched
from oracle import routed_layer
from relation_lm.kernels.routed_attention import routed_attention_quantized
from test_routed_attention_quantized_gpu import DTYPES, SEQ, U, case, host, raw_seq, values
from test_routed_attention_quantized_tiles_gpu import ROWS

pytestmark = pytest.mark.gpu

PARTS = {torch.bfloat16: 1, torch.float16: 2, torch.float32: 3}
LEFT = {torch.bfloat16: 2.0 ** -18, torch.float16: 2.0 ** -18, torch.float32: 2.0 ** -26}


def one_key(g, batch, queries, heads, kv_heads, dim, rows, block, top, dtype):
    """Queries of one feature, and no picks."""
    query, key, value, positions, picks = case(g, batch, queries, heads, kv_heads, dim, rows, block,
                                               top, 1, dtype)
    only = torch.randint(0, dim, query.shape[:-1], generator=g)
    query = torch.zeros_like(query).scatter_(-1, only[..., None], 8 * query[..., :1])
    return query, key, value, positions, torch.full_like(picks, -1)


def check_one_key(out, lse, parts, scale):
    query, key, value, positions, _ = parts
    k, v = values(key), values(value)
    group = query.shape[2] // k.shape[2]
    at = (np.arange(len(k))[:, None], positions.numpy())
    k, v = (np.repeat(x[at], group, 2) for x in (k, v))             # [B, Tq, Hq, D]
    dtype = query.dtype
    score = (host(query) * k).sum(-1) * scale
    off = np.abs(host(lse) - score)
    bound = (2 * PARTS[dtype] + 8) * U * np.abs(score) + 4 * U
    assert (off <= bound).all(), float((off / bound).max())
    least = 2.0 ** -25 if dtype == torch.float16 else 1e-35
    bound = (torch.finfo(dtype).eps / 2 + 12 * U + LEFT[dtype]) * np.abs(v) + least
    off = np.abs(host(out) - v)
    assert (off <= bound).all(), float((off / bound).max())


# queries, heads, key heads, dim, block: few queries
FEW = [(3, 9, 3, 64, 32), (1, 32, 4, 128, 64), (5, 4, 4, 96, 16), (2, 6, 1, 256, 64), (7, 2, 2, 32, 8)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", FEW, ids=str)
def test_one_key(device, shape, dtype):
    queries, heads, kv_heads, dim, block = shape
    print(f"one key {shape} {dtype}", flush=True)
    g = torch.Generator().manual_seed(sum(shape))
    parts = one_key(g, 2, queries, heads, kv_heads, dim, 100, block, 2, dtype)
    out, lse = raw_seq(device, parts, block, 1, scale=0.7)
    check_one_key(out, lse, parts, 0.7)
    query, key, value, positions, picks = parts

    def token():
        return routed_attention_quantized(
            query[:, 0].to(device), key[0].to(device), value[0].to(device), key[1].to(device),
            value[1].to(device), picks[:, 0, 0].contiguous().to(device),
            positions[:, 0].contiguous().to(device), block, 1, 0.7)

    out, lse = token()
    torch.cuda.synchronize()
    check_one_key(out[:, None], lse[:, None],
                  (query[:, :1], key, value, positions[:, :1], picks[:, :1]), 0.7)
    assert "attend_codes_kernel" in launched(token)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("queries, dim, block", [
    (301, 64, 64), (301, 32, 48), (301, 96, 12), (301, 128, 64), (301, 256, 64), (700, 64, 20),
    (700, 32, 64), (700, 96, 20), (700, 128, 64), (700, 160, 64)])
def test_one_key_on_shared_tiles(device, queries, dim, block, dtype):
    print(f"one key, shared tiles {queries} {dim} {block} {dtype}", flush=True)
    g = torch.Generator().manual_seed(queries + dim + block)
    parts = one_key(g, 2, queries, 32, 4, dim, ROWS, block, 4 if block == 64 else 16, dtype)
    out, lse = raw_seq(device, parts, block, 1, scale=0.7)
    check_one_key(out, lse, parts, 0.7)
    names = launched(lambda: raw_seq(device, parts, block, 1, scale=0.7))
    assert ("attend_codes_kernel" if block == 12 else "attend_tile_kernel") in names


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SEQ, ids=str)
def test_as_many_keys_as_are_seen(device, shape, dtype):
    batch, queries, heads, kv_heads, dim, rows, block, window, top, slots = shape
    print(f"seen keys {shape} {dtype}", flush=True)
    g = torch.Generator().manual_seed(sum(shape) + 1)
    parts = case(g, batch, queries, heads, kv_heads, dim, rows, block, top, slots, dtype)
    query, key, value, positions, picks = parts
    out, lse = raw_seq(device, parts, block, window, slots)
    want, want_lse, spread, size = routed_layer.attention(
        host(query), values(key), values(value), picks.numpy(), positions.numpy(), block, window,
        dim ** -0.5)
    n = np.zeros(want_lse.shape)
    for b, i, h in np.ndindex(n.shape):
        pick = picks[b, i, h // (heads // kv_heads) if slots > 1 else 0].numpy()
        n[b, i, h] = len(routed_layer.seen_positions(int(positions[b, i]), pick, rows, block, window,
                                                     False))
    e = (PARTS[dtype] * dim + 6) * U * size
    relative = 2 * e + 2 * size * U + (4 * n + 20) * U + LEFT[dtype]
    least = 2.0 ** -25 if dtype == torch.float16 else 1e-30
    off = np.abs(host(out) - want)
    bound = torch.finfo(dtype).eps / 2 * np.abs(want) + spread * relative[..., None] + least
    assert (off <= bound).all(), float((off / bound).max())
    seen = np.isfinite(want_lse)
    off = np.abs(host(lse)[seen] - want_lse[seen])
    bound = (e + size * U + (n + 16) * U)[seen] + U * np.abs(want_lse[seen])
    assert (off <= bound).all(), float((off / bound).max())
