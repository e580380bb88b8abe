"""GPU parity of 8-bit caches (rlm_quantized::rotary_to_quantized_caches, rlm_quantized::quantized_rows) against
oracle/few_bits.py and oracle/routed_layer.py.

A value row is not rotated: its scale and codes are those of the stated fp32 operations, bit for
bit.  A key row x is rotated in fp32 first, off by r = 10 u scale (|a| + |b|) per feature
(u = 2^-24; tests/test_rotary_gpu.py derives it), so its scale is off by at most
max r / 448 + 2 u relative, and what it reads back as by the code's rounding of x / s, half a step:
2^-4 of the value or 2^-10 of the scale (e4m3's subnormal step is 2^-9), with the scale's own error
(at most 448 times it) and the two fp32 roundings of quotient and product.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import few_bits, routed_layer
from relation_lm.kernels.quantized_cache import quantized_rows, rotary_to_quantized_caches

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def host(t):
    return t.detach().double().cpu().numpy()


def frequencies(pairs):
    return (10000.0 ** (-torch.arange(pairs, dtype=torch.float64) / pairs)).float()


def caches(g, batch, rows, kv_heads, dim):
    """(codes, scales) of random rows."""
    x = torch.randn(batch, rows, kv_heads, dim, generator=g)
    scale, code = few_bits.coded(x.numpy())
    return torch.from_numpy(code).float().to(torch.float8_e4m3fn), torch.from_numpy(scale)


SHAPES = [
    # batch, queries, heads, kv_heads, dim, pairs, rows, first, ring, interleaved
    (8, 1, 9, 3, 64, 32, 512, 511, False, False),
    (3, 1, 4, 4, 80, 20, 64, 1000, True, True),
    (2, 50, 6, 2, 64, 32, 64, 30, False, False),    # runs past the cache's end
    (2, 50, 6, 2, 128, 64, 64, -20, False, True),   # starts before it
    (2, 64, 3, 1, 128, 9, 64, 100, True, False),    # wraps, every row
    (1, 9, 2, 2, 32, 16, 16, -3, True, False),
    (2, 17, 3, 3, 7, 3, 40, 5, False, True),
    (1, 21, 5, 1, 256, 128, 30, 2, False, False),
    (2, 300, 2, 1, 200, 93, 310, 4, False, False),
    (1, 3, 1, 1, 2, 1, 8, 2, False, False),
]


def position_rows(position, batch, queries, rows, ring, lengths):
    """[(b, token, row)] that are written."""
    first = np.broadcast_to(position.numpy(), (batch,))
    found = []
    for b in range(batch):
        for i in range(queries if lengths is None else min(queries, int(lengths[b]))):
            at = int(first[b]) + i
            if at >= 0 and (ring or at < rows):
                found.append((b, i, at % rows))
    return found


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_rotary_to_quantized_caches(device, shape, ragged, dtype):
    batch, queries, heads, kv_heads, dim, pairs, rows, first, ring, interleaved = shape
    print(f"rotary_to_quantized_caches {shape} {ragged} {dtype}", flush=True)
    g = torch.Generator().manual_seed(sum(shape[:6]))
    query, key, value = [torch.randn(batch, queries, n, dim, generator=g).to(dtype)
                         for n in (heads, kv_heads, kv_heads)]
    key[:, ::7] *= 1000
    value[:, 1::5] = 0                       # rows of zeros
    value[:, 2::5] *= 2.0 ** -12
    before = [caches(g, batch, rows, kv_heads, dim) for _ in range(2)]
    freq = frequencies(pairs)
    position = torch.tensor(first)
    lengths = None
    if ragged:
        position = first - torch.arange(batch)
        lengths = torch.randint(0, queries + 1, (batch,), generator=g, dtype=torch.int32)
    want_q = routed_layer.rotary(host(query), np.broadcast_to(position.numpy(), (batch,))[:, None]
                                 + np.arange(queries), freq.numpy(), interleaved, 1.25)
    want_k = routed_layer.rotary(host(key), np.broadcast_to(position.numpy(), (batch,))[:, None]
                                 + np.arange(queries), freq.numpy(), interleaved, 1.25)
    written = position_rows(position, batch, queries, rows, ring, lengths)
    for layout in ("rows", "heads"):
        def place(x):
            x = x.to(device)
            if layout == "rows":
                return x
            order = (0, 2, 1) + tuple(range(3, x.dim()))
            return x.permute(order).contiguous().permute(order)
        (kc, ks), (vc, vs) = [(place(c.view(torch.uint8)).view(torch.float8_e4m3fn), place(s))
                              for c, s in before]
        got = rotary_to_quantized_caches(
            query.to(device), key.to(device), value.to(device), position.to(device),
            freq.to(device), kc, vc, ks, vs, interleaved, 1.25, ring,
            None if lengths is None else lengths.to(device))
        torch.cuda.synchronize()
        size = 2 * 1.25 * np.abs(host(query)).max(-1, keepdims=True)
        half = torch.finfo(dtype).eps / 2
        assert (np.abs(host(got) - want_q)
                <= half * np.abs(want_q) + 10 * U * size + 2.0 ** -25).all()
        codes = [host(c.float()) for c in (kc, vc)]
        scales = [s.cpu().numpy() for s in (ks, vs)]
        kept = np.ones((batch, rows), bool)
        for b, i, row in written:
            kept[b, row] = False
            scale, code = few_bits.coded(value[b, i].float().numpy())
            assert np.array_equal(scales[1][b, row], scale)
            assert np.array_equal(codes[1][b, row], code)
            x = want_k[b, i]
            largest = 2 * 1.25 * np.abs(host(key[b, i])).max(-1)
            r = 10 * U * largest
            s = np.abs(x).max(-1) / 448
            off = np.abs(scales[0][b, row] - s)
            assert (off <= r / 448 + 2 * U * s).all()
            back = codes[0][b, row] * scales[0][b, row][:, None].astype(np.float64)
            bound = np.maximum(np.abs(x) * 2.0 ** -4, s[:, None] * 2.0 ** -10) * (1 + 1e-6)
            assert (np.abs(back - x) <= bound + 2 * r[:, None] + 4 * U * np.abs(x)).all()
        for i in range(2):
            assert np.array_equal(codes[i][kept], host(before[i][0].float())[kept])
            assert np.array_equal(scales[i][kept], before[i][1].numpy()[kept])


def store(device, key, value, dim=64, pairs=32, **options):
    """One call at position 0 of a cache of the inputs' length; (kc, vc, ks, vs)."""
    batch, queries, kv_heads = key.shape[:3]
    kc, vc = [torch.full((batch, queries, kv_heads, dim), 1.0, device=device).to(
        torch.float8_e4m3fn) for _ in range(2)]
    ks, vs = [torch.full((batch, queries, kv_heads), 7.0, device=device) for _ in range(2)]
    rotary_to_quantized_caches(key.to(device), key.to(device), value.to(device),
                               torch.tensor(0, device=device), frequencies(pairs).to(device),
                               kc, vc, ks, vs, **options)
    torch.cuda.synchronize()
    return kc, vc, ks, vs


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_of_any_magnitude(device, dtype):
    """From the smallest subnormals to the type's largest: scales and codes as stated; rows that are
    not finite read back as NaN, their neighbours as they are."""
    g = torch.Generator().manual_seed(3)
    info = torch.finfo(dtype)
    x = torch.randn(1, 40, 2, 64, generator=g).to(dtype)
    sizes = [info.max / 8, 1.0, 2.0 ** -60, 2.0 ** -118, 2.0 ** -126, 2.0 ** -133]
    for i, s in enumerate(sizes):
        x[0, i] = (x[0, i].double().clamp(-4, 4) * s).to(dtype)
    x[0, 10, 0, 5], x[0, 11, 1, 63], x[0, 12, 0, 0] = float("inf"), float("nan"), -float("inf")
    x[0, 13, 0, 1], x[0, 13, 0, 2] = info.max, info.min
    kc, vc, ks, vs = store(device, x, x)
    scale, code = few_bits.coded(x.float().numpy())
    assert np.array_equal(vs.cpu().numpy(), scale, equal_nan=True)
    normal = scale >= 2.0 ** -115   # below, the quotient's correction falls out of fp32's range
    normal |= np.isnan(scale)
    assert np.array_equal(host(vc.float())[normal], code[normal])
    off = np.abs(host(vc.float()) - code)[~normal]
    assert (off <= 2.0 ** -3 * np.abs(code[~normal]) + 2.0 ** -9).all()
    back = quantized_rows(vc, vs, dtype=torch.float32)
    bad = torch.zeros(1, 40, 2, dtype=torch.bool)
    bad[0, 10, 0] = bad[0, 11, 1] = bad[0, 12, 0] = True
    assert torch.isnan(back.cpu()[bad]).all() and torch.isfinite(back.cpu()[~bad]).all()
    assert torch.equal(torch.isnan(ks.cpu()), bad)


def test_views_of_one_projection(device):
    """Query, key and value as views of a projection's rows, aligned and not: the same bits."""
    g = torch.Generator().manual_seed(1)
    batch, queries, heads, kv_heads, dim, pairs = 2, 37, 6, 2, 64, 32
    width = (heads + 2 * kv_heads) * dim
    rows = torch.randn(batch, queries, width, generator=g).to(torch.bfloat16)
    results = []
    for offset in (0, 1, 8):
        wide = torch.zeros(batch, queries, width + offset, dtype=torch.bfloat16, device=device)
        wide[..., offset:] = rows.to(device)
        parts = wide[..., offset:].split((heads * dim, kv_heads * dim, kv_heads * dim), dim=-1)
        query, key, value = [p.view(batch, queries, -1, dim) for p in parts]
        kc, vc = [torch.zeros(batch, 40, kv_heads, dim, dtype=torch.uint8, device=device).view(
            torch.float8_e4m3fn) for _ in range(2)]
        ks, vs = [torch.zeros(batch, kv_heads, 40, device=device).transpose(1, 2)
                  for _ in range(2)]
        out = rotary_to_quantized_caches(query, key, value, torch.tensor(3, device=device),
                                         frequencies(pairs).to(device), kc, vc, ks, vs)
        torch.cuda.synchronize()
        results.append((out, kc.view(torch.uint8), vc.view(torch.uint8), ks, vs))
    for other in results[1:]:
        for a, b in zip(results[0], other):
            assert torch.equal(a, b)


ROWS = [
    # batch, rows, kv_heads, dim, named
    (2, 100, 3, 64, 0), (8, 512, 3, 64, 640), (1, 7, 1, 8, 3), (3, 33, 2, 80, 50),
    (2, 19, 5, 13, 0), (2, 19, 5, 13, 40), (1, 5000, 4, 128, 0), (1, 1, 1, 1, 1),
    (2, 0, 2, 64, 5),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", ROWS, ids=str)
def test_quantized_rows(device, shape, dtype):
    batch, rows, kv_heads, dim, named = shape
    print(f"quantized_rows {shape} {dtype}", flush=True)
    g = torch.Generator().manual_seed(sum(shape))
    codes = torch.randint(0, 256, (batch, rows, kv_heads, dim), generator=g, dtype=torch.uint8)
    codes[(codes & 127) == 127] = 1      # every code but NaN
    scale = torch.rand(batch, rows, kv_heads, generator=g) * 3
    values = torch.from_numpy(np.concatenate([few_bits.E4M3, [0], -few_bits.E4M3, [0]]))
    want = (values[codes.long()].float() * scale[..., None])
    where = None
    if named:
        where = torch.randint(-3, rows + 3, (batch, named), generator=g)
        where[0, 0] = 2 ** 62
        there = (where >= 0) & (where < rows)
        if rows:
            at = torch.where(there, where, 0)
            want = want[torch.arange(batch)[:, None], at] * there[..., None, None]
        else:
            want = torch.zeros(batch, named, kv_heads, dim)
    want = want.to(dtype)
    for index in ((torch.int64, torch.int32) if named else (None,)):
        rows_arg = None
        if named:
            small = where.clamp(-2 ** 31, 2 ** 31 - 1) if index == torch.int32 else where
            rows_arg = small.to(index).to(device)
        got = quantized_rows(codes.to(device).view(torch.float8_e4m3fn), scale.to(device), rows_arg,
                             dtype)
        torch.cuda.synchronize()
        assert got.dtype == dtype and torch.equal(got.cpu(), want)


def test_quantized_rows_of_other_layouts(device):
    g = torch.Generator().manual_seed(2)
    codes, scale = caches(g, 2, 50, 4, 64)
    plain = quantized_rows(codes.to(device), scale.to(device))
    raw = codes.view(torch.uint8).to(device)
    by_head = raw.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3).view(torch.float8_e4m3fn)
    odd = torch.zeros(2, 50, 4, 67, dtype=torch.uint8, device=device)
    odd[..., 3:] = raw
    scales = scale.to(device).transpose(1, 2).contiguous().transpose(1, 2)
    for view in (by_head, odd[..., 3:].view(torch.float8_e4m3fn)):
        assert torch.equal(quantized_rows(view, scales), plain)
    shared = codes.to(device)[:1].expand(2, -1, -1, -1)      # one cache for two requests
    both = quantized_rows(shared, scale.to(device)[:1].expand(2, -1, -1))
    assert torch.equal(both[0], plain[0]) and torch.equal(both[1], plain[0])


def test_empty_calls(device):
    x = torch.empty(0, 4, 2, 64, device=device)
    kc = torch.empty(0, 8, 2, 64, device=device).to(torch.float8_e4m3fn)
    ks = torch.empty(0, 8, 2, device=device)
    got = rotary_to_quantized_caches(x, x, x, torch.tensor(0, device=device),
                                     frequencies(32).to(device), kc, kc.clone(), ks, ks.clone())
    assert got.shape == x.shape
    x = torch.empty(2, 0, 2, 64, device=device)
    kc = torch.ones(2, 8, 2, 64, device=device).to(torch.float8_e4m3fn)
    ks = torch.ones(2, 8, 2, device=device)
    rotary_to_quantized_caches(x, x, x, torch.tensor(0, device=device), frequencies(32).to(device),
                               kc, kc.clone(), ks, ks.clone())
    assert (kc.float() == 1).all() and (ks == 1).all()
    none = torch.empty(2, 0, dtype=torch.int64, device=device)
    assert quantized_rows(kc, ks, none).shape == (2, 0, 2, 64)
