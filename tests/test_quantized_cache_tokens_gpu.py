"""Many tokens written to 8-bit caches with the rotation: workgroups of several tokens, within the
bounds of test_quantized_cache_gpu.py, and bit for bit what fewer tokens get."""
from __future__ import annotations

import pytest
import torch

import test_quantized_cache_gpu as few
from launched import launched
from relation_lm.kernels.quantized_cache import rotary_to_quantized_caches

pytestmark = pytest.mark.gpu

SHAPES = [
    # batch, queries, heads, kv_heads, dim, pairs, rows, first, ring, interleaved
    (2, 4099, 2, 1, 64, 32, 4200, 30, False, False),
    (3, 2741, 1, 1, 48, 16, 2700, -20, False, False),   # starts before the cache, runs past it
    (1, 4099, 1, 2, 80, 40, 8192, 5000, True, False),   # wraps
    (1, 2051, 2, 1, 200, 96, 2100, 5, False, False),
    (1, 2051, 1, 1, 256, 64, 2051, 0, False, True),
    (1, 16401, 1, 1, 24, 8, 16401, 0, False, True),
    (1, 16401, 5, 2, 32, 16, 16500, 7, False, False),
    (1, 4101, 1, 1, 128, 64, 4101, 0, False, True),
]


@pytest.mark.parametrize("dtype", few.DTYPES)
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_many_tokens(device, shape, ragged, dtype):
    few.test_rotary_to_quantized_caches(device, shape, ragged, dtype)


def stored(device, parts, freq, interleaved, at=slice(None)):
    query, key, value = [x[:, at].to(device) for x in parts]
    batch, queries, kv_heads, dim = key.shape
    codes = [torch.full(key.shape, 1.0, device=device).to(torch.float8_e4m3fn) for _ in range(2)]
    scales = [torch.full(key.shape[:3], 7.0, device=device) for _ in range(2)]
    call = lambda: rotary_to_quantized_caches(
        query, key, value, torch.zeros(batch, dtype=torch.int64, device=device) + 0, freq.to(device),
        *codes, *scales, interleaved)
    names = launched(call)
    out = call()
    torch.cuda.synchronize()
    return names, [out] + [c.view(torch.uint8) for c in codes] + scales


@pytest.mark.parametrize("dtype", few.DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim, pairs", [(32, 16), (64, 32), (64, 16), (128, 64), (256, 128)])
def test_same_bits_as_fewer_tokens(device, dim, pairs, interleaved, dtype):
    print(f"same bits {dim} {pairs} {interleaved} {dtype}", flush=True)
    g = torch.Generator().manual_seed(dim + pairs)
    tokens = 1024 * 64 // max(dim // 8, 4) + 3
    parts = [torch.randn(1, tokens, n, dim, generator=g).to(dtype) for n in (3, 2, 2)]
    parts[1][0, 5, 0, 3], parts[2][0, 6, 1, 4] = float("inf"), float("nan")
    parts[2][0, 7] = 0
    freq = few.frequencies(pairs)
    names, many = stored(device, parts, freq, interleaved)
    assert "rotary_quantize_tokens_kernel" in names
    names, one = stored(device, parts, freq, interleaved, slice(0, 50))
    assert "rotary_quantize_kernel" in names
    for a, b in zip(many, one):
        a = a[:, :50].contiguous()
        same = (a == b) | ((a != a) & (b != b))
        assert same.all()
