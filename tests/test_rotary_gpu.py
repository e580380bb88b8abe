"""GPU parity of rotary positions (rlm::rotary_positions, rlm::rotary_to_caches) against
oracle/routed_layer.py in float64.

Tolerance (u = 2^-24, h = half a step of the output's type): the angle is exact to float64 and
its reduced half-turns are rounded to fp32 (u relative to at most 1, so pi u of angle), sine and
cosine are off by that plus 2 u, times scale u: (pi + 3) u each; a (c) - b (s) adds 2 roundings
of terms up to scale (|a| + |b|).  |got - exact| <= h |exact| + 10 u scale (|a| + |b|).
Features that do not turn, values and cache rows that are not written keep their bits.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import routed_layer
from relation_lm.kernels.rotary import rotary_positions, rotary_to_caches

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def host(t):
    return t.detach().double().cpu().numpy()


def frequencies(pairs, base=10000.0, stretch=1.0):
    return (base ** (-torch.arange(pairs, dtype=torch.float64) / pairs) / stretch).float()


def check(got, x, want, pairs, interleaved, scale, dtype):
    size = np.abs(host(x))
    one = slice(0, 2 * pairs, 2) if interleaved else slice(0, pairs)
    two = slice(1, 2 * pairs, 2) if interleaved else slice(pairs, 2 * pairs)
    both = size[..., one] + size[..., two]
    bound = torch.finfo(dtype).eps / 2 * np.abs(want)
    bound[..., one] += 10 * U * scale * both
    bound[..., two] += 10 * U * scale * both
    if dtype == torch.float16:
        bound += 2.0 ** -25          # below the type's normal numbers
    assert (np.abs(host(got) - want) <= bound).all()
    assert torch.equal(got[..., 2 * pairs:].cpu(), x[..., 2 * pairs:].cpu())


SHAPES = [
    # batch, queries, heads, kv_heads, dim, pairs
    (1, 1, 1, 1, 2, 1),
    (2, 7, 9, 3, 64, 32),
    (1, 33, 4, 4, 128, 32),
    (3, 5, 5, 1, 80, 13),
    (1, 70, 32, 8, 128, 64),
    (2, 3, 2, 2, 96, 47),
    (1, 2, 3, 1, 7, 3),
    (1, 4, 1, 2, 1024, 512),
    (40, 30, 6, 2, 64, 24),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=[str(s) for s in SHAPES])
def test_rotary_positions(device, shape, interleaved, dtype):
    batch, queries, heads, kv_heads, dim, pairs = shape
    print(f"rotary_positions {shape} {interleaved} {dtype}", flush=True)
    g = torch.Generator().manual_seed(sum(shape))
    query = torch.randn(batch, queries, heads, dim, generator=g).to(dtype)
    key = torch.randn(batch, queries, kv_heads, dim, generator=g).to(dtype)
    freq = frequencies(pairs)
    for positions, scale in ((torch.randint(-5, 1 << 20, (batch, queries), generator=g), 1.0),
                             (torch.arange(queries, dtype=torch.int32) + 99990, 1.25),
                             (torch.tensor(12345), 0.5)):
        got = rotary_positions(query.to(device), key.to(device), positions.to(device),
                               freq.to(device), interleaved, scale)
        torch.cuda.synchronize()
        for mine, x in zip(got, (query, key)):
            want = routed_layer.rotary(host(x), positions.numpy(), freq.numpy(), interleaved, scale)
            check(mine, x, want, pairs, interleaved, scale, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset", [0, 1])
def test_views_of_one_projection(device, dtype, offset):
    """Query, key and value as views of a projection's rows; offset 1: not 16-byte aligned."""
    g = torch.Generator().manual_seed(1)
    batch, queries, heads, kv_heads, dim, pairs = 2, 37, 6, 2, 64, 32
    width = (heads + 2 * kv_heads) * dim
    rows = torch.randn(batch, queries, width + offset, generator=g).to(dtype).to(device)[..., offset:]
    parts = rows.split((heads * dim, kv_heads * dim, kv_heads * dim), dim=-1)
    query, key, value = [p.view(batch, queries, -1, dim) for p in parts]
    freq, positions = frequencies(pairs), torch.arange(queries)
    got = rotary_positions(query, key, positions.to(device), freq.to(device))
    for mine, x in zip(got, (query, key)):
        want = routed_layer.rotary(host(x), positions.numpy(), freq.numpy(), False, 1.0)
        check(mine, x, want, pairs, False, 1.0, dtype)
    shared = key[:1].expand(batch, -1, -1, -1)          # one batch row's key for all
    got = rotary_positions(query, shared, positions.to(device), freq.to(device))
    assert torch.equal(got[1][0], got[1][1])


CACHE = [
    # batch, queries, heads, kv_heads, dim, pairs, rows, first, ring
    (8, 1, 9, 3, 64, 32, 512, 511, False),
    (3, 1, 4, 4, 80, 20, 64, 1000, True),
    (2, 50, 6, 2, 64, 32, 64, 0, False),
    (2, 50, 6, 2, 64, 32, 64, 30, False),     # runs past the cache's end
    (2, 50, 6, 2, 64, 32, 64, -20, False),    # starts before it
    (2, 64, 3, 1, 128, 9, 64, 100, True),     # wraps, every row
    (1, 9, 2, 2, 32, 16, 16, -3, True),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", CACHE, ids=[str(s) for s in CACHE])
@pytest.mark.parametrize("ragged", [False, True])
def test_rotary_to_caches(device, shape, ragged, dtype):
    batch, queries, heads, kv_heads, dim, pairs, rows, first, ring = shape
    print(f"rotary_to_caches {shape} {ragged} {dtype}", flush=True)
    g = torch.Generator().manual_seed(sum(shape[:6]))
    query, key, value = [torch.randn(batch, queries, n, dim, generator=g).to(dtype)
                         for n in (heads, kv_heads, kv_heads)]
    caches = [torch.randn(batch, rows, kv_heads, dim, generator=g).to(dtype) for _ in range(2)]
    freq = frequencies(pairs)
    position = torch.tensor(first)
    lengths = None
    if ragged:
        position = first - torch.arange(batch)
        lengths = torch.randint(0, queries + 1, (batch,), generator=g, dtype=torch.int32)
    for layout in ("rows", "heads"):
        kc, vc = [c.to(device) if layout == "rows" else
                  c.to(device).permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
                  for c in caches]
        got = rotary_to_caches(query.to(device), key.to(device), value.to(device),
                               position.to(device), freq.to(device), kc, vc, False, 1.0, ring,
                               None if lengths is None else lengths.to(device))
        torch.cuda.synchronize()
        want_q, want_k, want_v = routed_layer.rotary_to_caches(
            host(query), host(key), host(value), position.numpy(), freq.numpy(), host(caches[0]),
            host(caches[1]), False, 1.0, ring, None if lengths is None else lengths.numpy())
        check(got, query, want_q, pairs, False, 1.0, dtype)
        assert np.array_equal(host(vc), want_v)
        written = np.zeros((batch, rows), bool)
        t = np.broadcast_to(position.numpy(), (batch,))[:, None] + np.arange(queries)
        for b in range(batch):
            many = queries if lengths is None else int(lengths[b])
            mine = t[b, :many]
            mine = mine[mine >= 0] % rows if ring else mine[(mine >= 0) & (mine < rows)]
            written[b, mine] = True
        kept = host(kc)[~written]
        assert np.array_equal(kept, host(caches[0])[~written])
        off = np.abs(host(kc) - want_k)[written]
        half = torch.finfo(dtype).eps / 2
        # |a| + |b| of a pair is at most sqrt(2) of the pair's length, which turning keeps.
        largest = 2 * np.abs(host(key)).max()
        assert (off <= half * np.abs(want_k)[written] + 10 * U * largest
                + (2.0 ** -25 if dtype == torch.float16 else 0)).all()


def test_empty_calls(device):
    x = torch.empty(0, 4, 2, 64, device=device)
    got = rotary_positions(x, x, torch.arange(4, device=device), frequencies(32).to(device))
    assert got[0].shape == x.shape
    x = torch.empty(2, 0, 2, 64, device=device)
    cache = torch.ones(2, 8, 2, 64, device=device)
    got = rotary_to_caches(x, x, x, torch.tensor(0, device=device), frequencies(32).to(device),
                           cache, cache.clone())
    assert got.shape == x.shape and (cache == 1).all()
