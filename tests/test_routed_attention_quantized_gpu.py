"""GPU parity of attention over 8-bit caches (rlm_quantized::routed_attention_quantized[_seq]) against
oracle/routed_layer.py in float64, whose keys and values are codes times scales.

Tolerance, per output (u = eps(fp32) / 2, h = half a step of the output's type, P = 1 to 3 bf16
parts): a score is a sum of P D products in fp32 times two factors, off by at most
(P D + 6) u sum_d |q_d k_d| scale = e; a weight is then off by 2 e relative, plus 4 u from exp2 and
its scaled argument (|s| u relative, |s| within `size`), u from its value scale, p from its bf16
parts (2^-18 for two, 2^-26 for three), the sums of n weights by P n u: in all, relative to
A = sum_p w_p |v_p|,
   |out - exact| <= h |out| + A (2 e + 2 size u + (4 n + 20) u + p),
   |lse - exact| <= e + size u + (n + 16) u + u |lse|.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import few_bits, routed_layer
from relation_lm.kernels.routed_attention import (routed_attention_quantized,
                                                  routed_attention_quantized_seq)

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def host(t):
    return t.detach().double().cpu().numpy()


def check(out, lse, expected, dtype, dim):
    want, want_lse, spread, size = expected
    size = np.abs(size)              # the oracle's has the sign of the scale
    half = torch.finfo(dtype).eps / 2
    n = 4096
    e = (3 * dim + 6) * U * size
    parts = 2.0 ** -26 if dtype == torch.float32 else 2.0 ** -18
    relative = 2 * e + 2 * size * U + (4 * n + 20) * U + parts
    got, got_lse = host(out), host(lse)
    bound = half * np.abs(want) + spread * relative[..., None] + 1e-30
    if dtype == torch.float16:
        bound = bound + 2.0 ** -25
    off = np.abs(got - want)
    assert (off <= bound).all(), float((off / bound).max())
    seen = np.isfinite(want_lse)
    assert (np.isneginf(got_lse) == ~seen).all()
    off = np.abs(got_lse[seen] - want_lse[seen])
    assert (off <= (e + size * U)[seen] + (n + 16) * U + U * np.abs(want_lse[seen])).all()


def coded(x):
    scale, code = few_bits.coded(x.numpy())
    return torch.from_numpy(code).float().to(torch.float8_e4m3fn), torch.from_numpy(scale)


def case(g, batch, queries, heads, kv_heads, dim, rows, block, top, slots, dtype, first=None,
         odd=True):
    """Random tensors on the CPU: query, (key codes, scales), (value codes, scales), positions and
    picks -- distinct blocks before the query's position, mixed (`odd`) with -1, repeats and blocks
    outside the cache."""
    query = torch.randn(batch, queries, heads, dim, generator=g).to(dtype)
    key = coded(torch.randn(batch, rows, kv_heads, dim, generator=g))
    value = coded(torch.randn(batch, rows, kv_heads, dim, generator=g)
                  * torch.rand(batch, rows, kv_heads, 1, generator=g))
    positions = (torch.randint(0, rows, (batch, queries), generator=g) if first is None
                 else first + torch.arange(queries).expand(batch, queries))
    count = -(-rows // block)
    picks = torch.rand(batch, queries, slots, count, generator=g).argsort(-1)[..., :top]
    picks = torch.nn.functional.pad(picks, (0, top - picks.shape[-1]), value=-1)
    if odd and top:
        kind = torch.rand(picks.shape, generator=g)
        picks = torch.where(kind < 0.1, -1, picks)
        picks = torch.where((kind > 0.1) & (kind < 0.2), picks[..., :1], picks)
        picks = torch.where((kind > 0.2) & (kind < 0.25), count + 7, picks)
    return query, key, value, positions.contiguous(), picks.to(torch.int32)


def values(rows):
    """Codes times scales, float64."""
    codes, scales = rows
    return host(codes.float()) * host(scales)[..., None]


def raw_seq(device, parts, block, window, slots=1, scale=None, layout=None):
    query, key, value, positions, picks = parts
    blocks = picks if slots > 1 else picks[:, :, 0]
    move = layout or (lambda x: x.to(device))
    result = routed_attention_quantized_seq(
        query.to(device), move(key[0]), move(value[0]), move(key[1]), move(value[1]),
        blocks.contiguous().to(device), positions.to(device), block, window, scale)
    torch.cuda.synchronize()
    return result


def run_seq(device, parts, block, window, slots=1, scale=None, layout=None):
    query, key, value, positions, picks = parts
    out, lse = raw_seq(device, parts, block, window, slots, scale, layout)
    dim = query.shape[-1]
    check(out, lse, routed_layer.attention(host(query), values(key), values(value), picks.numpy(),
                                           positions.numpy(), block, window,
                                           dim ** -0.5 if scale is None else scale),
          query.dtype, dim)
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
    (1, 50, 5, 1, 16, 100, 4, 0, 6, 1),
    (1, 21, 3, 3, 128, 700, 128, 1, 5, 3),
    (1, 9, 128, 1, 64, 90, 10, 7, 64, 1),
    (3, 5, 7, 7, 48, 50, 16, 50, 0, 1),
    (1, 300, 3, 3, 112, 310, 12, 5, 9, 1),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SEQ, ids=str)
def test_sequence_form(device, shape, dtype):
    batch, queries, heads, kv_heads, dim, rows, block, window, top, slots = shape
    print(f"routed_attention_quantized_seq {shape} {dtype}", flush=True)
    g = torch.Generator().manual_seed(hash(shape) % 2**31)
    parts = case(g, batch, queries, heads, kv_heads, dim, rows, block, top, slots, dtype)
    run_seq(device, parts, block, window, slots)


# Enough queries that their key tiles would be shared.
MANY = [
    # batch, queries, heads, kv_heads, dim, rows, block, window, top, slots
    (2, 1100, 12, 4, 64, 1100, 64, 128, 3, 1),
    (1, 1300, 16, 2, 128, 1400, 64, 100, 8, 2),
    (1, 2000, 8, 8, 32, 2048, 16, 32, 8, 1),
    (1, 1500, 18, 2, 80, 1501, 20, 33, 30, 2),
    (1, 900, 10, 10, 96, 900, 60, 64, 5, 1),
    (1, 700, 40, 2, 256, 900, 128, 70, 4, 2),
    (1, 2000, 5, 1, 64, 4000, 4, 16, 60, 1),
    (2, 1024, 15, 3, 48, 1100, 48, 300, 0, 1),
    (1, 800, 20, 4, 64, 40000, 100, 90, 7, 4),
    (2, 1200, 4, 4, 64, 1200, 12, 0, 16, 1),
    (1, 999, 12, 4, 64, 4096, 64, 128, 8, 1),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", MANY, ids=str)
def test_sequence_form_of_many_queries(device, shape, dtype):
    batch, queries, heads, kv_heads, dim, rows, block, window, top, slots = shape
    print(f"routed_attention_quantized_seq {shape} {dtype}", flush=True)
    g = torch.Generator().manual_seed(hash(shape) % 2**31)
    first = None if rows < queries + 90 else rows - queries
    parts = case(g, batch, queries, heads, kv_heads, dim, rows, block, top, slots, dtype,
                 first=first)
    run_seq(device, parts, block, window, slots, scale=-0.2 if heads == 10 else None)


def either(g, many, dtype, **options):
    """A call of many queries, or of a few."""
    return (case(g, 2, 1500, 8, 4, 64, 1600, 16, 3, 1, dtype, first=60, **options) if many else
            case(g, 2, 40, 4, 2, 64, 96, 16, 3, 1, dtype, **options))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("many", [False, True])
def test_rows_that_see_nothing_and_positions_past_the_cache(device, many, dtype):
    g = torch.Generator().manual_seed(5)
    parts = either(g, many, dtype)
    positions, rows = parts[3], parts[1][0].shape[1]
    positions[0, ::3] = -1
    positions[1, 5] = rows + 10      # window partly past the cache
    positions[1, 6] = 10 ** 12       # window wholly past it: the picks alone
    positions[1, 7] = -10 ** 12
    positions[1, 8] = 2 ** 63 - 1
    positions[1, 9] = -2 ** 63
    out, lse = run_seq(device, parts, 16, 24)
    assert (out[0, ::3] == 0).all() and torch.isneginf(lse[0, ::3]).all()
    assert (out[1, 9] == 0).all() and torch.isneginf(lse[1, 9]).all()


def test_scores_that_grow_along_the_cache(device):
    g = torch.Generator().manual_seed(12)
    for dtype in DTYPES:
        query, key, value, positions, picks = either(g, True, dtype)
        query = query.abs()
        codes = key[0].float().abs().to(torch.float8_e4m3fn)
        key = codes, key[1] * torch.linspace(0.1, 3.0, 1600)[:, None]
        parts = (query, key, value, positions, picks)
        run_seq(device, parts, 16, 400, scale=0.5)
        run_seq(device, parts, 16, 400, scale=0.0)


def test_scales_of_any_size(device):
    """Scales over the whole of fp32's range, zero among them."""
    g = torch.Generator().manual_seed(13)
    for many in (False, True):
        for dtype in DTYPES:
            query, key, value, positions, picks = either(g, many, dtype)
            exponent = torch.randint(-30, 10, value[1].shape, generator=g)
            value = value[0], torch.where(exponent < -25, 0.0, value[1] * 2.0 ** exponent)
            if dtype == torch.float16:
                value = value[0], value[1].clamp_max(100)
            key = key[0], torch.where(torch.rand(key[1].shape, generator=g) < 0.2, 0.0, key[1])
            run_seq(device, (query, key, value, positions, picks), 16, 24)


@pytest.mark.parametrize("what", ["codes", "scale nan", "scale inf"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("many", [False, True])
def test_unseen_rows_do_not_reach_the_output(device, many, what, dtype):
    """Rows that no query sees and, in the same tiles, rows that only later queries see."""
    g = torch.Generator().manual_seed(6)
    query, key, value, positions, picks = (
        case(g, 2, 1500, 8, 4, 64, 1600, 16, 2, 1, dtype, first=60) if many else
        case(g, 1, 48, 4, 2, 64, 128, 16, 2, 1, dtype, first=60))
    picks = picks.clamp_max(1)                       # blocks 0 and 1: rows 0..31
    clean = run_seq(device, (query, key, value, positions, picks), 16, 8)

    def spoil(rows, at):
        codes, scales = rows[0].clone(), rows[1].clone()
        if what == "codes":
            codes.view(torch.uint8)[:, at] = 0x7f    # NaN
        else:
            scales[:, at] = float(what.split()[1])
        return codes, scales

    end = slice(int(positions.max()) + 1, None)      # past every query
    key, value = spoil(key, end), spoil(value, end)
    got = raw_seq(device, (query, key, value, positions, picks), 16, 8)
    assert torch.equal(got[0], clean[0]) and torch.equal(got[1], clean[1])
    # Seen by the queries at 80 .. 87 alone (window 8): the others' outputs stay, within the bound
    # (their sums may be taken in another order), and those are no numbers.
    good = key, value
    key, value = spoil(key, slice(80, 81)), spoil(value, slice(80, 81))
    got = raw_seq(device, (query, key, value, positions, picks), 16, 8)
    others = (positions[0] < 80) | (positions[0] > 87)
    expected = routed_layer.attention(host(query[:, others]), values(good[0]), values(good[1]),
                                      picks[:, others].numpy(), positions[:, others].numpy(), 16, 8,
                                      64 ** -0.5)
    check(got[0][:, others], got[1][:, others], expected, dtype, 64)
    assert torch.isnan(got[0][:, ~others]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("many", [False, True])
def test_caches_of_other_layouts(device, many, dtype):
    g = torch.Generator().manual_seed(7)
    parts = (case(g, 2, 1500, 8, 4, 64, 1500, 20, 3, 1, dtype) if many else
             case(g, 2, 33, 6, 3, 64, 100, 20, 3, 1, dtype))
    plain = raw_seq(device, parts, 20, 24)

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
        again = raw_seq(device, parts, 20, 24, layout=layout)
        assert torch.equal(plain[0], again[0]) and torch.equal(plain[1], again[1])


@pytest.mark.parametrize("positions_form", ["shared", "scalar"])
def test_position_forms(device, positions_form):
    g = torch.Generator().manual_seed(8)
    query, key, value, _, picks = case(g, 2, 20, 4, 4, 32, 64, 8, 2, 1, torch.float32)
    positions = torch.arange(30, 50) if positions_form == "shared" else torch.tensor(41)
    run_seq(device, (query, key, value, positions.to(torch.int32), picks), 8, 12, scale=0.3)


DECODE = [
    # batch, heads, kv_heads, dim, rows, block, window, top, slots, ring
    (1, 9, 3, 64, 512, 32, 64, 4, 1, False),
    (8, 9, 3, 64, 512, 32, 64, 4, 3, False),
    (3, 32, 4, 128, 4096, 64, 512, 16, 4, False),
    (40, 8, 8, 96, 300, 20, 31, 6, 1, False),
    (2, 48, 1, 256, 1000, 50, 100, 3, 1, False),
    (1, 1, 1, 16, 1, 1, 1, 1, 1, False),
    (2, 16, 16, 128, 2000, 1000, 0, 2, 16, False),
    (70, 16, 8, 80, 640, 16, 40, 64, 1, False),
    (3, 8, 2, 64, 256, 32, 40, 5, 2, True),
    (2, 4, 4, 128, 64, 16, 100, 4, 1, True),
    (300, 4, 4, 112, 96, 8, 16, 3, 1, False),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", DECODE, ids=str)
def test_decode_form(device, shape, dtype):
    batch, heads, kv_heads, dim, rows, block, window, top, slots, ring = shape
    print(f"routed_attention_quantized {shape} {dtype}", flush=True)
    g = torch.Generator().manual_seed(hash(shape) % 2**31)
    query, key, value, positions, picks = case(g, batch, 1, heads, kv_heads, dim, rows, block, top,
                                               slots, dtype)
    if ring:
        positions = positions + torch.randint(0, 3, positions.shape, generator=g) * rows + 7
        now = positions[:, :, None, None] // block
        picks = torch.where(picks >= 0, now - (now - picks) % (rows // block), -1).to(torch.int32)
    blocks = picks[:, 0] if slots > 1 else picks[:, 0, 0]
    for position in (positions[:, 0], torch.tensor(rows - 1, dtype=torch.int32)):
        out, lse = routed_attention_quantized(
            query[:, 0].to(device), key[0].to(device), value[0].to(device), key[1].to(device),
            value[1].to(device), blocks.contiguous().to(device), position.to(device), block, window,
            None, ring)
        torch.cuda.synchronize()
        t = np.broadcast_to(position.numpy().reshape(-1, 1), (batch, 1))
        check(out[:, None], lse[:, None],
              routed_layer.attention(host(query), values(key), values(value), picks.numpy(), t,
                                     block, window, dim ** -0.5, ring), dtype, dim)


def test_rows_past_4_gib(device):
    """A cache of more than 2^32 bytes: rows at its end, and a row stride beyond it."""
    rows, dim = 70_000_000, 64
    if torch.cuda.mem_get_info()[0] < 3 * rows * dim:
        pytest.skip("too little free memory")
    g = torch.Generator().manual_seed(9)
    query, key, value, _, picks = case(g, 1, 2, 2, 1, dim, 256, 64, 2, 1, torch.bfloat16)
    codes = torch.zeros(1, rows, 1, dim, dtype=torch.uint8, device=device)
    scales = torch.zeros(1, rows, 1, device=device)
    at = rows - 256
    positions = torch.tensor([[rows - 1, rows - 100]])
    picks = torch.full((1, 2, 1, 2), -1, dtype=torch.int32)
    picks[0, :, 0, 0] = (at + 64) // 64
    big = []
    for codes_of, scales_of in (key, value):
        codes[:, at:] = codes_of.view(torch.uint8).to(device)
        scales[:, at:] = scales_of.to(device)
        big.append((codes.clone().view(torch.float8_e4m3fn), scales.clone()))
    out, lse = routed_attention_quantized_seq(
        query.to(device), big[0][0], big[1][0], big[0][1], big[1][1],
        picks[:, :, 0].to(device), positions.to(device), 64, 40)
    torch.cuda.synchronize()
    assert at % 64 == 0
    want = routed_layer.attention(host(query), values(key), values(value),
                                  np.where(picks.numpy() >= 0, picks.numpy() - at // 64, -1),
                                  positions.numpy() - at, 64, 40, dim ** -0.5)
    check(out, lse, want, torch.bfloat16, dim)


def test_empty_calls(device):
    kc = torch.ones(2, 8, 2, 64, device=device).to(torch.float8_e4m3fn)
    ks = torch.ones(2, 8, 2, device=device)
    query = torch.empty(2, 0, 4, 64, device=device)
    out, lse = routed_attention_quantized_seq(
        query, kc, kc, ks, ks, torch.empty(2, 0, 3, dtype=torch.int32, device=device),
        torch.empty(0, dtype=torch.int64, device=device), 4, 4)
    assert out.shape == (2, 0, 4, 64) and lse.shape == (2, 0, 4)
    query = torch.randn(2, 3, 4, 64, device=device)
    none = kc[:, :0], kc[:, :0], ks[:, :0], ks[:, :0]
    out, lse = routed_attention_quantized_seq(
        query, *none, torch.zeros(2, 3, 1, dtype=torch.int32, device=device),
        torch.tensor(5, device=device), 4, 4)
    assert (out == 0).all() and torch.isneginf(lse).all()
