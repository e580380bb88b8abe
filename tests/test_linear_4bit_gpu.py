"""GPU parity of products with 4-bit weights (rlm_quantized::linear_4bit, rlm_quantized::gated_linear_4bit) against
oracle/few_bits.py in float64.

Tolerance (u = eps(fp32) / 2, h = half a step of the type): a group's L <= 128 inputs are summed in
fp32 with the codes as 16 + c (fp32: c - 8), in up to 3 parts, and so are the inputs alone, which are
then multiplied by 16 + z: each of the (3 L + 4) sums and three roundings is off by u of at most
S = sum |x| s (32 + c + |z|); the scaled groups (their number and the waves' and chunks') add u each
of T = sum |x| s |c - z|:
   d = u ((3 * 128 + 8) S + (K / 32 + 24) T),   |out - exact| <= h |out| + d.
(S and T of all groups together.)  The fp32 parts leave 2^-26 of T.  Gated: the activation's slope is
at most 1.13, its own error 8 u relative (silu) or |g| (0.75e-7 + 8 u) (GELU).
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import few_bits
from relation_lm.kernels.linear_4bit import (gated_linear_4bit, linear_4bit, pack_4bit,
                                             quantize_4bit)

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def host(t):
    return t.detach().double().cpu().numpy()


def weight(g, n, k, group, zeros, dtype):
    """codes, scales, zeros on the CPU."""
    codes = torch.randint(0, 16, (n, k), generator=g, dtype=torch.uint8)
    groups = -(-k // group)
    scales = ((torch.rand(groups, n, generator=g) + 0.1) * (1 - 2 * (torch.rand(
        groups, n, generator=g) < 0.1)) * 0.3 * k ** -0.5).to(dtype)
    scales[0, ::5] = 0
    z = None
    if zeros:   # whole ones and others
        z = torch.randint(0, 16, (groups, n), generator=g).to(dtype)
        z[:, 1::3] = (torch.rand(z[:, 1::3].shape, generator=g) * 15).to(dtype)
    return codes, scales, z


def product(x, w, group):
    """Exact product and how far a kernel's may be off before it is rounded."""
    codes, scales, zeros = w
    out, s, t = few_bits.product(host(x).reshape(-1, x.shape[-1]), codes.numpy(), host(scales),
                                 None if zeros is None else host(zeros), group)
    d = U * ((3 * 128 + 8) * s + (x.shape[-1] / 32 + 24) * t) + 2.0 ** -26 * t
    return out, d


def check(got, want, d, dtype):
    half = torch.finfo(dtype).eps / 2
    bound = half * (np.abs(want) + d) + d + (2.0 ** -25 if dtype == torch.float16 else 1e-35)
    off = np.abs(host(got).reshape(want.shape) - want)
    assert (off <= bound).all(), float((off / bound).max())


def on(device, w):
    codes, scales, zeros = w
    return (pack_4bit(codes).to(device), scales.to(device),
            None if zeros is None else zeros.to(device))


SHAPES = [
    # tokens, width, outputs, group
    (1, 1, 1, 32), (1, 576, 2304, 64), (1, 4096, 512, 128), (2, 128, 16, 128), (3, 100, 37, 32),
    (5, 640, 50, 256), (16, 768, 96, 64), (17, 768, 64, 128), (31, 2304, 576, 32),
    (33, 333, 130, 64), (64, 512, 256, 128), (65, 512, 256, 128), (100, 1000, 333, 384),
    (129, 576, 640, 64), (200, 2048, 200, 128), (300, 96, 1000, 32), (513, 260, 514, 128),
    (1, 14000, 40, 128), (7, 2050, 1030, 32), (1000, 72, 24, 32),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_linear(device, shape, zeros, dtype):
    tokens, width, outputs, group = shape
    print(f"linear_4bit {shape} {zeros} {dtype}", flush=True)
    g = torch.Generator().manual_seed(sum(shape))
    x = torch.randn(tokens, width, generator=g).to(dtype)
    for scale_dtype in {dtype, torch.float32}:
        w = weight(g, outputs, width, group, zeros, scale_dtype)
        bias = torch.randn(outputs, generator=g).to(torch.float16) if tokens % 2 else None
        got = linear_4bit(x.to(device), *on(device, w), group,
                          None if bias is None else bias.to(device))
        torch.cuda.synchronize()
        want, d = product(x, w, group)
        if bias is not None:
            want = want + host(bias)
            d = d + U * (np.abs(want) + d)
        check(got, want, d, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_gated_linear(device, shape, activation, dtype):
    tokens, width, outputs, group = shape
    print(f"gated_linear_4bit {shape} {activation} {dtype}", flush=True)
    g = torch.Generator().manual_seed(sum(shape) + 1)
    x = (2 * torch.randn(tokens, width, generator=g)).to(dtype)
    zeros = tokens % 2 == 0
    gate, up = [weight(g, outputs, width, group, zeros, dtype) for _ in range(2)]
    (gc, gs, gz), (uc, us, uz) = on(device, gate), on(device, up)
    got = gated_linear_4bit(x.to(device), gc, gs, uc, us, gz, uz, group, activation)
    torch.cuda.synchronize()
    (a, da), (b, db) = product(x, gate, group), product(x, up, group)
    t = torch.from_numpy(a)
    act = (torch.nn.functional.silu(t) if activation == "silu" else
           torch.nn.functional.gelu(t)).numpy()
    own = (8 * U * np.abs(act) if activation == "silu" else np.abs(a) * (0.75e-7 + 8 * U))
    d_act = 1.13 * da + own
    d = d_act * (np.abs(b) + db) + np.abs(act) * db
    check(got, act * b, d + U * np.abs(act * b), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_leading_dims_and_strides(device, dtype):
    """Rows of a wider tensor, not 16-byte aligned rows, any leading dims: the same bits."""
    g = torch.Generator().manual_seed(2)
    x = torch.randn(3, 7, 200, generator=g).to(dtype).to(device)
    w = on(device, weight(g, 90, 200, 64, True, dtype))
    plain = linear_4bit(x, *w, 64)
    assert plain.shape == (3, 7, 90)
    for offset in (1, 8):
        wide = torch.zeros(3, 7, 200 + 2 * offset, dtype=dtype, device=device)
        wide[..., offset:-offset] = x
        assert torch.equal(linear_4bit(wide[..., offset:-offset], *w, 64), plain)
    assert torch.equal(linear_4bit(x.transpose(0, 1), *w, 64), plain.transpose(0, 1))
    assert torch.equal(linear_4bit(x[1, 2], *w, 64), linear_4bit(x[1, 2:3], *w, 64)[0])
    same = x[:1].expand(3, -1, -1)
    assert torch.equal(linear_4bit(same, *w, 64)[2], linear_4bit(same, *w, 64)[0])
    assert linear_4bit(x[:0], *w, 64).shape == (0, 7, 90)


def test_scales_at_any_address(device):
    """Scales and zero points that start inside a buffer, and an odd number of outputs."""
    g = torch.Generator().manual_seed(4)
    x = torch.randn(3, 256, generator=g).bfloat16().to(device)
    codes, scales, zeros = on(device, weight(g, 64, 256, 32, True, torch.bfloat16))
    plain = linear_4bit(x, codes, scales, zeros, 32)
    buffer = torch.zeros(scales.numel() + 1, dtype=torch.bfloat16, device=device)
    buffer[1:] = scales.flatten()
    assert torch.equal(linear_4bit(x, codes, buffer[1:].view_as(scales), zeros, 32), plain)


def test_codes_past_the_ends_do_not_matter(device):
    """Codes of rows past N and of inputs past K hold anything."""
    g = torch.Generator().manual_seed(5)
    for dtype in DTYPES:
        for tokens in (1, 70, 300):
            x = torch.randn(tokens, 70, generator=g).to(dtype).to(device)
            w = weight(g, 21, 70, 32, True, dtype)
            codes, scales, zeros = on(device, w)
            wide = torch.randint(0, 16, (32, 128), generator=g, dtype=torch.uint8)
            wide[:21, :70] = w[0]
            assert torch.equal(linear_4bit(x, codes, scales, zeros, 32),
                               linear_4bit(x, pack_4bit(wide).to(device), scales, zeros, 32))


@pytest.mark.parametrize("tokens", [2, 40, 300])
def test_inputs_that_are_not_finite(device, tokens):
    """A token with an infinity or NaN gives NaN; the others are as they were."""
    g = torch.Generator().manual_seed(6)
    x = torch.randn(tokens, 256, generator=g).bfloat16().to(device)
    w = on(device, weight(g, 48, 256, 64, False, torch.bfloat16))
    plain = linear_4bit(x, *w, 64)
    for bad in (float("inf"), float("nan")):
        y = x.clone()
        y[1, 77] = bad
        got = linear_4bit(y, *w, 64)
        assert torch.isnan(got[1]).all()
        keep = [i for i in range(tokens) if i != 1]
        assert torch.equal(got[keep], plain[keep])


def test_quantize_and_pack(device):
    """quantize_4bit's codes stand for values within half a scale of the weight's, and the product
    of packed weights is that of the values they stand for."""
    g = torch.Generator().manual_seed(7)
    original = torch.randn(96, 300, generator=g)
    original[3] = 0
    original[4] = original[4].abs()
    for symmetric in (False, True):
        codes, scales, zeros = quantize_4bit(original.to(device), 64, symmetric)
        pick = torch.arange(300) // 64
        s = scales.cpu()[pick].T
        z = torch.full_like(s, 8) if zeros is None else zeros.cpu()[pick].T
        stands_for = (codes.cpu().float() - z) * s
        assert ((stands_for - original).abs() <= s * 0.5 * (1 + 1e-5)).all()
        assert (stands_for[3] == 0).all()
        x = torch.randn(4, 300, generator=g)
        got = linear_4bit(x.to(device), pack_4bit(codes), scales, zeros, 64)
        want, d = product(x, (codes.cpu(), scales.cpu(), None if zeros is None else zeros.cpu()),
                          64)
        check(got, want, d, torch.float32)
