"""Attention over 8-bit caches where many queries share key tiles: the instances that such calls
take, against oracle/routed_layer.py within the bound of test_routed_attention_quantized_gpu.py."""
from __future__ import annotations

import re

import pytest
import torch

from launched import launched
from oracle import routed_layer
from test_routed_attention_quantized_gpu import (DTYPES, case, check, host, raw_seq, run_seq,
                                                 values)

pytestmark = pytest.mark.gpu

ROWS, WINDOW = 250, 230
DIMS = [32, 48, 64, 80, 96, 128, 256, 16, 112, 160]


def instance(device, parts, block, window=WINDOW):
    """(head dim in 32s, whole, keys of a tile, waves, shares) of the tile kernel that the call takes."""
    names = launched(lambda: raw_seq(device, parts, block, window))
    plain = re.search(r"attend_tile_kernel<.*code8, (\d+), (\w+), (\d+), (\d+), (\d+)>", names)
    if plain:
        return int(plain[1]), plain[2] == "true", int(plain[3]), int(plain[4]), int(plain[5])
    mangled = re.search(r"attend_tile_kernel.*code8ELi(\d+)ELb(\d)ELi(\d+)ELi(\d+)ELi(\d+)E", names)
    assert mangled, names
    return int(mangled[1]), mangled[2] == "1", int(mangled[3]), int(mangled[4]), int(mangled[5])


def expected_instance(dim, block, waves, shares):
    dc = -(-dim // 32)
    dc = dc if dc <= 4 else 8
    return dc, block % 64 == 0, 64 if dc <= 2 else 32, waves, shares


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("block", [64, 48, 4])
@pytest.mark.parametrize("dim", DIMS)
def test_many_queries(device, dim, block, dtype):
    print(f"many queries dim {dim} block {block} {dtype}", flush=True)
    g = torch.Generator().manual_seed(dim + block)
    parts = case(g, 2, 700, 32, 4, dim, ROWS, block, 2, 1, dtype)
    run_seq(device, parts, block, WINDOW)
    if dtype != torch.float32:
        assert instance(device, parts, block) == expected_instance(dim, block, 4, 1)
    elif (dim, block) != (64, 4):        # (a query to a workgroup)
        shares = 2 if dim <= 64 else 1
        assert instance(device, parts, block) == expected_instance(dim, block, 1, shares)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim, block", [(d, 64) for d in DIMS] + [(32, 48), (64, 48), (96, 12)])
def test_fewer_queries(device, dim, block, dtype):
    print(f"fewer queries dim {dim} block {block} {dtype}", flush=True)
    g = torch.Generator().manual_seed(dim + block)
    parts = case(g, 2, 301, 32, 4, dim, ROWS, block, 2, 1, dtype)
    run_seq(device, parts, block, WINDOW)
    shares = 2 if dim <= 64 else 1
    assert instance(device, parts, block) == expected_instance(dim, block, 1, shares)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim, block", [(d, 64) for d in DIMS] + [(32, 4), (64, 48), (96, 12), (128, 48),
                                                                  (160, 20)])
def test_few_queries(device, dim, block, dtype):
    print(f"few queries dim {dim} block {block} {dtype}", flush=True)
    g = torch.Generator().manual_seed(dim + block)
    parts = case(g, 2, 199, 32, 4, dim, ROWS, block, 2, 1, dtype)
    run_seq(device, parts, block, WINDOW)
    assert dim == 160 or instance(device, parts, block) == expected_instance(dim, block, 1, 2)


# queries, block: two waves that share out tiles, four waves of 16-bit queries
SHARED = [(301, 64), (301, 20), (700, 64), (700, 20)]


@pytest.mark.parametrize("what", ["codes", "scale nan", "scale inf"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("queries, block", SHARED)
def test_unseen_rows_do_not_reach_the_output(device, queries, block, dtype, what):
    print(f"unseen rows {queries} {block} {dtype} {what}", flush=True)
    g = torch.Generator().manual_seed(11)
    query, key, value, positions, picks = case(g, 2, queries, 32, 4, 64, ROWS, block, 2, 1, dtype)
    positions = positions.clamp_max(240)
    parts = query, key, value, positions, picks
    clean = run_seq(device, parts, block, WINDOW)
    assert instance(device, parts, block)[0] == 2

    def spoil(rows, at):
        codes, scales = rows[0].clone(), rows[1].clone()
        if what == "codes":
            codes.view(torch.uint8)[:, at] = 0x7f    # NaN
        else:
            scales[:, at] = float(what.split()[1])
        return codes, scales

    past = slice(241, None)
    got = raw_seq(device, (query, spoil(key, past), spoil(value, past), positions, picks), block,
                  WINDOW)
    assert torch.equal(got[0], clean[0]) and torch.equal(got[1], clean[1])
    # A row that only the later queries see, in their windows.
    at = slice(200, 201)
    got = raw_seq(device, (query, spoil(key, at), spoil(value, at), positions, picks), block, WINDOW)
    for b in range(2):
        others = positions[b] < 200
        expected = routed_layer.attention(
            host(query[b:b + 1, others]), values(key)[b:b + 1], values(value)[b:b + 1],
            picks[b:b + 1, others].numpy(), positions[b:b + 1, others].numpy(), block, WINDOW,
            64 ** -0.5)
        check(got[0][b:b + 1, others], got[1][b:b + 1, others], expected, dtype, 64)
        assert torch.isnan(got[0][b, ~others]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("queries, block", SHARED)
def test_rows_that_see_nothing_and_positions_past_the_cache(device, queries, block, dtype):
    print(f"positions {queries} {block} {dtype}", flush=True)
    g = torch.Generator().manual_seed(5)
    parts = case(g, 2, queries, 32, 4, 64, ROWS, block, 2, 1, dtype)
    positions = parts[3]
    positions[0, ::3] = -1
    for i, t in enumerate([ROWS + 10, 10 ** 12, -10 ** 12, 2 ** 63 - 1, -2 ** 63]):
        positions[1, 5 + i] = t
    out, lse = run_seq(device, parts, block, WINDOW)
    assert instance(device, parts, block)[0] == 2
    assert (out[0, ::3] == 0).all() and torch.isneginf(lse[0, ::3]).all()
    assert (out[1, 9] == 0).all() and torch.isneginf(lse[1, 9]).all()


@pytest.mark.parametrize("queries, block", SHARED)
def test_scores_that_grow_along_the_cache(device, queries, block):
    g = torch.Generator().manual_seed(12)
    for dtype in DTYPES:
        print(f"growing scores {queries} {block} {dtype}", flush=True)
        query, key, value, positions, picks = case(g, 2, queries, 32, 4, 64, ROWS, block, 2, 1,
                                                   dtype)
        query = query.abs()
        codes = key[0].float().abs().to(torch.float8_e4m3fn)
        key = codes, key[1] * torch.linspace(0.1, 6.0, ROWS)[:, None]
        for scale in (0.5, 0.0, -0.3):
            run_seq(device, (query, key, value, positions, picks), block, WINDOW, scale=scale)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("queries, block", SHARED)
def test_caches_of_other_layouts(device, queries, block, dtype):
    print(f"layouts {queries} {block} {dtype}", flush=True)
    g = torch.Generator().manual_seed(7)
    parts = case(g, 2, queries, 32, 4, 80, ROWS, block, 2, 1, dtype)
    plain = raw_seq(device, parts, block, WINDOW)

    def raw(x):
        return x.to(device).view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x.to(device)

    def by_head(x):      # [B,Hk,T,...] storage
        order = (0, 2, 1) + tuple(range(3, x.dim()))
        y = raw(x).permute(order).contiguous().permute(order)
        return y.view(x.dtype)

    def inside(x):       # rows of a wider buffer
        y = raw(x)
        if x.dim() == 3:
            wide = torch.full((x.shape[0], x.shape[1] + 3, x.shape[2], 2), 9.0, device=device)
            wide[:, :-3, :, 1] = y
            return wide[:, :-3, :, 1]
        wide = torch.full((x.shape[0], x.shape[1] + 3, x.shape[2], x.shape[3] + 32), 0x7f,
                          dtype=torch.uint8, device=device)
        wide[:, :-3, :, 16:-16] = y
        return wide.view(x.dtype)[:, :-3, :, 16:-16]

    for layout in (by_head, inside):
        again = raw_seq(device, parts, block, WINDOW, layout=layout)
        assert torch.equal(plain[0], again[0]) and torch.equal(plain[1], again[1])


def test_long_caches_of_wide_rows(device):
    """Rows of a key head that reach over 2 GiB, of which the last are looked at."""
    rows, stride = 2 ** 19 + 192, 4352
    g = torch.Generator().manual_seed(3)
    query, key, value, positions, picks = case(g, 1, 1500, 8, 4, 64, 320, 64, 2, 1,
                                               torch.bfloat16)

    def move(x):
        if x.dim() == 3:
            far = torch.zeros(1, rows, 4, device=device)
            far[:, -320:] = x.to(device)
            return far
        store = torch.empty(1, rows * stride, dtype=torch.uint8, device=device)
        far = store.view(1, rows, stride)[..., :256].unflatten(-1, (4, 64))
        far[:, -320:] = x.to(device).view(torch.uint8)
        return far.view(torch.float8_e4m3fn)

    near = raw_seq(device, (query, key, value, positions, picks), 64, 150)
    shift = rows - 320
    assert shift % 64 == 0
    blocks = torch.where(picks >= 0, picks + shift // 64, -1).to(torch.int32)
    moved = query, key, value, positions + shift, blocks
    # What lies before the 320 rows is never seen.
    seen = positions[0] >= 149
    far = raw_seq(device, moved, 64, 150, layout=move)
    names = launched(lambda: raw_seq(device, moved, 64, 150, layout=move))
    assert "attend_tile_kernel" in names
    expected = routed_layer.attention(host(query[:, seen]), values(key), values(value),
                                      picks[:, seen].numpy(), positions[:, seen].numpy(), 64, 150,
                                      64 ** -0.5)
    check(far[0][:, seen], far[1][:, seen], expected, torch.bfloat16, 64)
    check(near[0][:, seen], near[1][:, seen], expected, torch.bfloat16, 64)
