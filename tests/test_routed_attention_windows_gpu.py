"""Attention on shared tiles (rlm::routed_attention_seq) whose blocks are whole tiles, over caches of
more than one window (256 tiles) of the kernel's walk: 16384 rows where a tile has 64 keys, 8192
where it has 32.  Tolerances: test_routed_attention_gpu.py's."""
from __future__ import annotations

import pytest
import torch

from relation_lm.kernels.routed_attention import routed_attention, routed_attention_seq
from test_routed_attention_gpu import case, run_seq, tile_kernel

pytestmark = pytest.mark.gpu

SHAPES = [
    # batch, queries, heads, kv_heads, dim, rows, block, window, top, slots, spread
    (1, 1100, 20, 4, 64, 40000, 64, 90, 9, 4, False),
    (1, 1500, 16, 4, 128, 20000, 128, 100, 6, 4, False),
    (1, 2400, 8, 8, 128, 33000, 64, 70, 6, 1, True),
    (2, 1100, 12, 4, 64, 21000, 128, 100, 6, 1, True),
    (1, 2000, 8, 8, 32, 40001, 64, 65, 8, 1, False),
    (1, 1800, 16, 2, 256, 17000, 64, 100, 6, 2, False),
    (2, 1700, 16, 2, 96, 20000, 192, 100, 4, 2, True),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES, ids=[str(s) for s in SHAPES])
def test_whole_blocks_over_several_windows(device, shape, dtype):
    """Picks over the whole cache; queries at its end, or (`spread`) anywhere."""
    batch, queries, heads, kv_heads, dim, rows, block, window, top, slots, spread = shape
    print(f"routed_attention_seq {shape} {dtype}", flush=True)
    g = torch.Generator().manual_seed(sum(shape))
    parts = case(g, batch, queries, heads, kv_heads, dim, rows, block, top, slots, dtype,
                 first=None if spread else rows - queries)
    run_seq(device, parts, block, window, slots)
    query, key, value, positions, picks = [x.to(device) for x in parts]
    blocks = picks if slots > 1 else picks[:, :, 0].contiguous()
    assert tile_kernel(lambda: routed_attention_seq(query, key, value, blocks, positions, block,
                                                    window))


def test_whole_blocks_in_a_cache_past_four_gib(device):
    """Picks at both ends of 140000 rows: the same rows in a small cache."""
    rows, kv_heads, dim, block, window, queries = 140_000, 64, 256, 64, 150, 1600
    head, low = 3200, 134_400        # multiples of the block size
    key = torch.empty(1, rows, kv_heads, dim, device=device, dtype=torch.bfloat16)
    value = torch.empty_like(key)
    assert key.numel() > 2**31
    gen = torch.Generator(device=device).manual_seed(4)
    small = [torch.randn(1, head + rows - low, kv_heads, dim, generator=gen, device=device,
                         dtype=torch.bfloat16) for _ in range(2)]
    for big, part in zip((key, value), small):
        big[:, :head], big[:, low:] = part[:, :head], part[:, head:]
    query = torch.randn(1, queries, 64, dim, generator=gen, device=device, dtype=torch.bfloat16)
    positions = torch.arange(rows - queries, rows, device=device)
    count = (head + rows - low) // block
    near = (head + rows - low - queries - window) // block      # blocks before every window
    picks = torch.randint(0, near, (1, queries, 3), generator=gen, device=device,
                          dtype=torch.int32)
    assert near < count and (picks < head // block).any() and (picks >= head // block).any()
    away = torch.where(picks < head // block, picks, picks + (low - head) // block)
    args = (query, key, value, away, positions, block, window)
    got = routed_attention_seq(*args)
    assert tile_kernel(lambda: routed_attention_seq(*args))
    want = routed_attention_seq(query, *small, picks, positions - (low - head), block, window)
    # (The kernels may sum in another order over the small cache: a step of the output, and of the
    # weights.)
    half = torch.finfo(torch.bfloat16).eps / 2
    assert torch.allclose(got[0].float(), want[0].float(), rtol=4 * half, atol=4 * half)
    assert torch.allclose(got[1], want[1], rtol=1e-5, atol=1e-5)
    one = routed_attention(query[:, 700], key, value, away[:, 700], positions[700], block, window)
    assert torch.allclose(one[0].float(), want[0][:, 700].float(), rtol=4 * half, atol=4 * half)
