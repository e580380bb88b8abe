"""GPU parity of attention over a local window and picked blocks (rlm::routed_attention[_seq])
against oracle/routed_layer.py in float64.

Tolerance, per output (u = eps(fp32) / 2, h = half a step of the output's type):
  a score is a sum of D products in fp32, off by at most (D + 4) u sum_d |q_d k_d| scale = e;
  a weight is then off by 2 e relative, plus 4 u from exp2 and its scaled argument (|s| u
  relative, |s| within `size`), the sums of n weights by n u: in all, relative to
  A = sum_p w_p |v_p|,
     |out - exact| <= h |out| + A (2 e + 2 size u + (2 n + 16) u + p),
  p = half a step of the 16-bit type in which the kernels round the weights (0 for fp32: its
  weights are not rounded), |lse - exact| <= e + size u + (n + 16) u + u |lse|.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from launched import launched
from oracle import routed_layer
from relation_lm.kernels.routed_attention import routed_attention, routed_attention_seq

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def host(t):
    return t.detach().double().cpu().numpy()


def check(out, lse, expected, dtype, dim):
    want, want_lse, spread, size = expected
    half = torch.finfo(dtype).eps / 2
    n = 4096
    e = (dim + 4) * U * size
    weights = 0.0 if dtype == torch.float32 else half
    relative = 2 * e + 2 * size * U + (2 * n + 16) * U + weights
    got, got_lse = host(out), host(lse)
    bound = half * np.abs(want) + spread * relative[..., None] + 1e-30
    off = np.abs(got - want)
    assert (off <= bound).all(), float((off / bound).max())
    seen = np.isfinite(want_lse)
    assert (np.isneginf(got_lse) == ~seen).all()
    off = np.abs(got_lse[seen] - want_lse[seen])
    assert (off <= (e + size * U)[seen] + (n + 16) * U + U * np.abs(want_lse[seen])).all()


def case(g, batch, queries, heads, kv_heads, dim, rows, block, top, slots, dtype, first=None,
         odd=True):
    """Random tensors on the CPU.  Picks: distinct blocks before the query's position, mixed
    (`odd`) with -1, repeats and blocks outside the cache."""
    query = torch.randn(batch, queries, heads, dim, generator=g).to(dtype)
    key = torch.randn(batch, rows, kv_heads, dim, generator=g).to(dtype)
    value = torch.randn(batch, rows, kv_heads, dim, generator=g).to(dtype)
    positions = (torch.randint(0, rows, (batch, queries), generator=g) if first is None
                 else first + torch.arange(queries).expand(batch, queries))
    count = -(-rows // block)
    picks = torch.rand(batch, queries, slots, count, generator=g).argsort(-1)[..., :top]
    if picks.shape[-1] < top:
        picks = torch.nn.functional.pad(picks, (0, top - picks.shape[-1]), value=-1)
    if odd and top:
        kind = torch.rand(picks.shape, generator=g)
        picks = torch.where(kind < 0.1, -1, picks)
        picks = torch.where((kind > 0.1) & (kind < 0.2), picks[..., :1], picks)
        picks = torch.where((kind > 0.2) & (kind < 0.25), count + 7, picks)
    return query, key, value, positions.contiguous(), picks.to(torch.int32)


def run_seq(device, parts, block, window, slots, scale=None, key_layout=None):
    query, key, value, positions, picks = parts
    blocks = picks if slots > 1 else picks[:, :, 0]
    move = key_layout or (lambda x: x.to(device))
    out, lse = routed_attention_seq(query.to(device), move(key), move(value),
                                    blocks.contiguous().to(device), positions.to(device), block,
                                    window, scale)
    torch.cuda.synchronize()
    dim = query.shape[-1]
    expected = routed_layer.attention(host(query), host(key), host(value), picks.numpy(),
                                      positions.numpy(), block, window,
                                      dim ** -0.5 if scale is None else scale)
    check(out, lse, expected, query.dtype, dim)
    return out, lse


SEQ = [
    # batch, queries, heads, kv_heads, dim, rows, block, window, top, slots
    (1, 1, 1, 1, 64, 1, 1, 1, 1, 1),
    (2, 70, 4, 4, 64, 128, 16, 32, 2, 1),
    (1, 130, 12, 4, 64, 256, 64, 128, 3, 1),
    (1, 65, 16, 1, 128, 192, 32, 64, 4, 1),
    (2, 33, 8, 2, 128, 512, 64, 128, 4, 2),
    (1, 100, 6, 2, 80, 333, 9, 17, 5, 2),
    (1, 40, 9, 3, 96, 200, 8, 16, 8, 3),
    (1, 37, 40, 2, 32, 160, 32, 33, 3, 1),
    (1, 19, 2, 1, 256, 300, 60, 100, 2, 1),
    (1, 50, 5, 1, 8, 100, 4, 0, 6, 1),
    (1, 21, 3, 3, 128, 700, 128, 1, 5, 3),
    (1, 9, 128, 1, 64, 90, 10, 7, 64, 1),
    (3, 5, 7, 7, 24, 50, 16, 50, 0, 1),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", SEQ, ids=[str(s) for s in SEQ])
def test_sequence_form(device, shape, dtype):
    batch, queries, heads, kv_heads, dim, rows, block, window, top, slots = shape
    print(f"routed_attention_seq {shape} {dtype}", flush=True)
    g = torch.Generator().manual_seed(hash(shape) % 2**31)
    parts = case(g, batch, queries, heads, kv_heads, dim, rows, block, top, slots, dtype)
    run_seq(device, parts, block, window, slots)


# Enough queries for the tiles that the rows of a workgroup share.
TILES = [
    # batch, queries, heads, kv_heads, dim, rows, block, window, top, slots
    (2, 1100, 12, 4, 64, 1100, 64, 128, 3, 1),
    (2, 1300, 16, 2, 128, 1400, 64, 100, 8, 2),
    (1, 2000, 8, 8, 32, 2048, 16, 32, 8, 1),
    (1, 2500, 18, 2, 80, 2501, 20, 33, 30, 2),
    (2, 900, 10, 10, 96, 900, 60, 64, 5, 1),
    (1, 900, 40, 2, 256, 900, 128, 70, 4, 2),
    (1, 4000, 5, 1, 64, 4000, 4, 16, 60, 1),
    (2, 1024, 15, 3, 56, 1100, 48, 300, 0, 1),
    (1, 1000, 20, 4, 64, 40000, 100, 90, 7, 4),     # more than one window of the cache
    (4, 1200, 4, 4, 64, 1200, 12, 0, 16, 1),
]


def tile_kernel(call):
    return "attend_tile_kernel" in launched(call)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", TILES, ids=[str(s) for s in TILES])
def test_sequence_form_on_shared_tiles(device, shape, dtype):
    batch, queries, heads, kv_heads, dim, rows, block, window, top, slots = shape
    print(f"routed_attention_seq {shape} {dtype}", flush=True)
    g = torch.Generator().manual_seed(hash(shape) % 2**31)
    first = None if rows < queries + 90 else rows - queries
    parts = case(g, batch, queries, heads, kv_heads, dim, rows, block, top, slots, dtype,
                 first=first)
    run_seq(device, parts, block, window, slots, scale=-0.2 if heads == 10 else None)
    query, key, value, positions, picks = [x.to(device) for x in parts]
    blocks = picks if slots > 1 else picks[:, :, 0].contiguous()
    assert tile_kernel(lambda: routed_attention_seq(query, key, value, blocks, positions, block,
                                                    window))


def many(g, dtype, heads=4, kv_heads=2, queries=1500, rows=1600, block=16, top=3):
    return case(g, 2, queries, heads, kv_heads, 64, rows, block, top, 1, dtype, first=60)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tiles", [False, True])
def test_rows_that_see_nothing_and_positions_past_the_cache(device, tiles, dtype):
    g = torch.Generator().manual_seed(5)
    query, key, value, positions, picks = (many(g, dtype, 8, 4) if tiles else
                                           case(g, 2, 40, 4, 2, 64, 96, 16, 3, 1, dtype))
    rows = key.shape[1]
    positions[0, ::3] = -1
    positions[1, 5] = rows + 10      # window partly past the cache
    positions[1, 6] = 10 ** 12       # window wholly past it: the picks alone
    positions[1, 7] = -10 ** 12
    out, lse = run_seq(device, (query, key, value, positions, picks), 16, 24, 1)
    assert (out[0, ::3] == 0).all() and torch.isneginf(lse[0, ::3]).all()
    if tiles:
        args = [x.to(device) for x in (query, key, value, picks[:, :, 0].contiguous(), positions)]
        assert tile_kernel(lambda: routed_attention_seq(*args, 16, 24))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tiles", [False, True])
def test_positions_at_the_ends_of_int64(device, tiles, dtype):
    """The last one sees what was picked, as any position past the window does; the first one
    nothing."""
    g = torch.Generator().manual_seed(14)
    query, key, value, positions, picks = (many(g, dtype, 8, 4) if tiles else
                                           case(g, 2, 40, 4, 2, 64, 96, 16, 3, 1, dtype))
    positions[0, 1::4] = 2 ** 63 - 1
    positions[1, 2::4] = -2 ** 63
    out, lse = run_seq(device, (query, key, value, positions, picks), 16, 24, 1)
    assert (out[1, 2::4] == 0).all() and torch.isneginf(lse[1, 2::4]).all()


def test_scores_past_a_tiles_limit(device):
    """Keys that grow along the cache: every tile's scores pass the base of the one before, by
    more than fp16 weights could hold; and all scores equal (a scale of 0)."""
    g = torch.Generator().manual_seed(12)
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        query, key, value, positions, picks = many(g, dtype, 8, 4, rows=1600)
        query = query.abs()
        key = (key.abs() * torch.linspace(0.1, 3.0, 1600)[:, None, None]).to(dtype)
        parts = (query, key, value, positions, picks)
        run_seq(device, parts, 16, 400, 1, scale=0.5)
        run_seq(device, parts, 16, 400, 1, scale=0.0)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"),
                                 torch.finfo(torch.bfloat16).min])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tiles", [False, True])
def test_unseen_rows_do_not_reach_the_output(device, tiles, bad, dtype):
    """Rows that no query sees and, in the same tiles, rows that only later queries see."""
    g = torch.Generator().manual_seed(6)
    query, key, value, positions, picks = (many(g, dtype, 8, 4) if tiles else
                                           case(g, 1, 48, 4, 2, 64, 128, 16, 2, 1, dtype, first=60))
    picks = picks.clamp_max(1)                       # blocks 0 and 1: rows 0..31
    parts = (query, key, value, positions, picks)
    clean = run_seq(device, parts, 16, 8, 1)
    if tiles:
        args = [x.to(device) for x in (query, key, value, picks[:, :, 0].contiguous(), positions)]
        assert tile_kernel(lambda: routed_attention_seq(*args, 16, 8))
    key, value = key.clone(), value.clone()
    end = int(positions.max()) + 1
    key[:, end:], value[:, end:] = bad, bad          # past every query
    got = run_seq_raw(device, (query, key, value, positions, picks), 16, 8)
    assert torch.equal(got[0], clean[0]) and torch.equal(got[1], clean[1])
    # Seen by the queries at 80 .. 87 alone (window 8): the others' outputs stay, within the bound
    # that the file states (a row with bad values among its neighbours' may be summed in another
    # order than before).
    key[:, 80], value[:, 80] = bad, bad
    got = run_seq_raw(device, (query, key, value, positions, picks), 16, 8)
    others = (positions[0] < 80) | (positions[0] > 87)
    expected = routed_layer.attention(host(query[:, others]), host(key), host(value),
                                      picks[:, others].numpy(), positions[:, others].numpy(), 16, 8,
                                      64 ** -0.5)
    check(got[0][:, others], got[1][:, others], expected, dtype, 64)
    if bad != bad:
        assert torch.isnan(got[0][:, ~others]).all()


def run_seq_raw(device, parts, block, window):
    query, key, value, positions, picks = parts
    result = routed_attention_seq(query.to(device), key.to(device), value.to(device),
                                  picks[:, :, 0].contiguous().to(device), positions.to(device),
                                  block, window)
    torch.cuda.synchronize()
    return result


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tiles", [False, True])
def test_caches_of_other_layouts(device, tiles, dtype):
    g = torch.Generator().manual_seed(7)
    parts = (case(g, 2, 1500, 8, 4, 64, 1500, 20, 3, 1, dtype) if tiles else
             case(g, 2, 33, 6, 3, 64, 100, 20, 3, 1, dtype))
    plain = run_seq(device, parts, 20, 24, 1)

    def by_head(x):      # [B,Hk,T,D] storage
        return x.to(device).permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)

    def inside(x):       # rows of a wider buffer
        wide = torch.full((x.shape[0], x.shape[1] + 3, x.shape[2], x.shape[3] + 16), 9.0,
                          dtype=dtype, device=device)
        wide[:, :-3, :, 8:-8] = x.to(device)
        return wide[:, :-3, :, 8:-8]

    for layout in (by_head, inside):
        again = run_seq(device, parts, 20, 24, 1, key_layout=layout)
        assert torch.equal(plain[0], again[0]) and torch.equal(plain[1], again[1])


@pytest.mark.parametrize("positions_form", ["shared", "scalar"])
def test_position_forms(device, positions_form):
    g = torch.Generator().manual_seed(8)
    query, key, value, _, picks = case(g, 2, 20, 4, 4, 32, 64, 8, 2, 1, torch.float32)
    positions = torch.arange(30, 50) if positions_form == "shared" else torch.tensor(41)
    run_seq(device, (query, key, value, positions.to(torch.int32), picks), 8, 12, 1, scale=0.3)


DECODE = [
    # batch, heads, kv_heads, dim, rows, block, window, top, slots
    (1, 9, 3, 64, 512, 32, 64, 4, 1),
    (8, 9, 3, 64, 512, 32, 64, 4, 3),
    (3, 32, 4, 128, 4096, 64, 512, 16, 4),
    (40, 8, 8, 96, 300, 20, 31, 6, 1),
    (2, 48, 1, 256, 1000, 50, 100, 3, 1),
    (1, 1, 1, 8, 1, 1, 1, 1, 1),
    (2, 16, 16, 128, 2000, 1000, 0, 2, 16),
    (70, 16, 8, 80, 640, 16, 40, 64, 1),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", DECODE, ids=[str(s) for s in DECODE])
def test_decode_form(device, shape, dtype):
    batch, heads, kv_heads, dim, rows, block, window, top, slots = shape
    print(f"routed_attention {shape} {dtype}", flush=True)
    g = torch.Generator().manual_seed(hash(shape) % 2**31)
    query, key, value, positions, picks = case(g, batch, 1, heads, kv_heads, dim, rows, block, top,
                                               slots, dtype)
    blocks = picks[:, 0] if slots > 1 else picks[:, 0, 0]
    for position in (positions[:, 0], torch.tensor(rows - 1, dtype=torch.int32)):
        out, lse = routed_attention(query[:, 0].to(device), key.to(device), value.to(device),
                                    blocks.contiguous().to(device), position.to(device), block,
                                    window)
        torch.cuda.synchronize()
        each = position.long()[:, None] if position.ndim else position.long()
        expected = routed_layer.attention(host(query), host(key), host(value), picks.numpy(),
                                          each.numpy(), block, window, dim ** -0.5)
        check(out[:, None], lse[:, None], expected, dtype, dim)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("items", [64, 65, 85, 86, 128, 129, 170, 171, 257])
@pytest.mark.parametrize("dim", [40, 72, 96, 104, 136, 200])
def test_features_shared_by_workgroups(device, dim, items, dtype):
    """Both sides of every number of (row, key head) items where the value features are shared
    by one workgroup more, and head dims that leave the last of them part of its share or none."""
    g = torch.Generator().manual_seed(items + dim)
    query, key, value, positions, picks = case(g, items, 1, 3, 1, dim, 150, 16, 3, 1, dtype)
    out, lse = routed_attention(query[:, 0].to(device), key.to(device), value.to(device),
                                picks[:, 0, 0].to(device), positions[:, 0].to(device), 16, 50)
    torch.cuda.synchronize()
    expected = routed_layer.attention(host(query), host(key), host(value), picks.numpy(),
                                      positions.numpy(), 16, 50, dim ** -0.5)
    check(out[:, None], lse[:, None], expected, dtype, dim)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t", [0, 5, 63, 64, 100, 127, 128, 1000, 2**33 + 77])
def test_ring_decode(device, t, dtype):
    """Absolute picks over a ring of 128 rows, window and blocks wrapping; blocks that the ring
    no longer holds, or not yet, name nothing."""
    g = torch.Generator().manual_seed(t % 1000)
    rows, block, window, top = 128, 16, 40, 8
    query, key, value, _, _ = case(g, 3, 1, 4, 2, 64, rows, block, top, 1, dtype)
    now = t // block
    if now >= 2**31 - 9:
        pytest.skip("block index past int32")
    picks = now + 1 - torch.stack([torch.randperm(11, generator=g)[:top] for _ in range(3)])
    picks = picks[:, None, None].to(torch.int32)
    out, lse = routed_attention(query[:, 0].to(device), key.to(device), value.to(device),
                                picks[:, 0, 0].to(device), torch.tensor(t, device=device), block,
                                window, None, True)
    torch.cuda.synchronize()
    expected = routed_layer.attention(host(query), host(key), host(value), picks.numpy(),
                                      np.array(t), block, window, 64 ** -0.5, ring=True)
    check(out[:, None], lse[:, None], expected, dtype, 64)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("batch,window,top", [(1, 1, 0), (2, 20, 3), (300, 33, 1)])
def test_an_infinity_that_is_seen_stays_one(device, batch, window, top, dtype):
    """The window's last row holds an infinite value feature: that feature is infinite, whatever
    keys of the same tile do not count, and the other features are as they were."""
    g = torch.Generator().manual_seed(13)
    query, key, value, _, picks = case(g, batch, 1, 4, 2, 64, 100, 7, top, 1, dtype)
    args = [x.to(device) for x in (query[:, 0], key, value, picks[:, 0, 0], torch.tensor(90))]
    clean, lse = routed_attention(*args, 7, window)
    args[2] = args[2].clone()
    args[2][:, 90, :, 5] = float("inf")
    out, again = routed_attention(*args, 7, window)
    torch.cuda.synchronize()
    assert torch.isposinf(out[..., 5]).all()
    rest = [i for i in range(64) if i != 5]
    assert torch.equal(out[..., rest], clean[..., rest]) and torch.equal(lse, again)


def test_ring_equals_linear_before_it_wraps(device):
    g = torch.Generator().manual_seed(9)
    query, key, value, positions, picks = case(g, 5, 1, 8, 2, 128, 256, 32, 4, 1, torch.bfloat16)
    args = [x.to(device) for x in (query[:, 0], key, value, picks[:, 0, 0], positions[:, 0])]
    linear = routed_attention(*args, 32, 48)
    ring = routed_attention(*args, 32, 48, None, True)
    assert torch.equal(linear[0], ring[0]) and torch.equal(linear[1], ring[1])


@pytest.mark.parametrize("queries", [3, 1600])
def test_cache_past_four_gib(device, queries):
    """Rows whose offsets pass 2^32 bytes and 2^31 elements: the same rows in a small cache."""
    rows, kv_heads, dim, block, window = 140_000, 64, 256, 100, 150
    key = torch.empty(1, rows, kv_heads, dim, device=device, dtype=torch.bfloat16)
    value = torch.empty_like(key)
    assert key.numel() > 2**31
    low = 134_400        # a multiple of the block size and of every key tile
    gen = torch.Generator(device=device).manual_seed(3)
    tail = [torch.randn(1, rows - low, kv_heads, dim, generator=gen, device=device,
                        dtype=torch.bfloat16) for _ in range(2)]
    key[:, low:], value[:, low:] = tail
    query = torch.randn(1, queries, 64, dim, generator=gen, device=device, dtype=torch.bfloat16)
    positions = torch.arange(rows - queries, rows, device=device)
    picks = torch.randint(0, (rows - low) // block - 20, (1, queries, 2), generator=gen,
                          device=device, dtype=torch.int32)
    args = (query, key, value, picks + low // block, positions, block, window)
    big = routed_attention_seq(*args)
    assert tile_kernel(lambda: routed_attention_seq(*args)) == (queries > 1000)
    small = routed_attention_seq(query, *[x.contiguous() for x in tail], picks, positions - low,
                                 block, window)
    half = torch.finfo(torch.bfloat16).eps / 2
    if queries == 3:
        assert torch.equal(big[0], small[0]) and torch.equal(big[1], small[1])
        one = routed_attention(query[:, 0], key, value, picks[:, 0] + low // block, positions[:1],
                               block, window)
        assert torch.allclose(one[0].float(), small[0][:, 0].float(), rtol=4 * half, atol=4 * half)
    else:   # (the model of the kernels' times may choose another for the small cache)
        assert torch.allclose(big[0].float(), small[0].float(), rtol=4 * half, atol=4 * half)
        assert torch.allclose(big[1], small[1], rtol=1e-5, atol=1e-5)


def test_one_answer_whatever_runs_beside(device):
    """The same bits on every call, and on another stream."""
    g = torch.Generator().manual_seed(11)
    for queries in (200, 4000):      # one query to a workgroup, shared tiles
        query, key, value, positions, picks = case(g, 2, queries, 8, 2, 64, 512, 32, 6, 1,
                                                   torch.bfloat16)
        args = [x.to(device) for x in (query, key, value, picks[:, :, 0].contiguous(), positions)]
        first = routed_attention_seq(*args, 32, 64)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            second = routed_attention_seq(*args, 32, 64)
        torch.cuda.current_stream().wait_stream(stream)
        assert torch.equal(first[0], second[0]) and torch.equal(first[1], second[1])
        assert tile_kernel(lambda: routed_attention_seq(*args, 32, 64)) == (queries == 4000)
