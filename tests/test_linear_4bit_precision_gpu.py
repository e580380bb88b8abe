"""How exact products with 4-bit weights are: tokens of one input that is not 0, whose products have few
roundings, and tokens of one sign, whose sums would cancel had the codes an offset.

u = eps(fp32) / 2, h = half a step of the output's type.  A matrix instruction is off by at most 2 u of the
largest of its sums.

One input x of 24 bits (fp32 tokens): codes enter as c - 8, x as three bf16 parts, in three
instructions.  These are off by 6 u |x| |c - 8|, the scale's multiply-add by u of the same.  With
zero points few tokens round z - 8, and once where x (z - 8) is taken off; tiles round z - 8 and its
product with s, and take x off in six instructions (12 u) that leave u / 4:
   |out - exact| <= u (8 |x s (c - 8)| + 16 |x s (z - 8)| + |exact|).
Without x's third part it would be off by up to 2^-18 = 64 u of |x s (c - 8)|.

One input of 16 bits, scales and zero points of 24: codes enter as 16 + c, the first product is exact and
the others are as above, so
   |out - exact| <= h |exact| + 16 u |x s| (32 + c + |z|)    (fp16: + 2^-25),
where scales of 16 bits would add up to 2^-8 (2^-11) of the exact value.

Tokens of one sign: the parts of a chunk of up to 128 inputs (three to each 32) are off by 2 u each of
the chunk's largest sum up to there; chunks are off by signs of their own, and so
are the sums of chunks and waves, so that with v a chunk's sums
   rms(out - exact)^2 <= mean over outputs of sum over chunks (s sum over instructions 2 u |v|)^2
                         + (chunks + 8) (u |total|)^2.
Had the codes an offset of 16, v would hold 24 sum x instead of its few percent.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from relation_lm.kernels.linear_4bit import gated_linear_4bit, linear_4bit
from test_linear_4bit_gpu import U, check, host, on, product, weight
from test_linear_4bit_tiles_gpu import SHAPES, instance

pytestmark = pytest.mark.gpu

# tile, group, tokens, outputs, width
FP32 = [
    ("few", 32, 1, 100, 576), ("few", 128, 7, 333, 260), ("few", 64, 31, 128, 1000),
    ("few", 64, 65, 1000, 304), ("wide", 32, 2099, 2000, 304), ("wide", 64, 2099, 2000, 1104),
    ("wide", 256, 2099, 2000, 304), ("middle", 32, 1299, 1000, 1104), ("middle", 64, 1299, 1000, 304),
    ("middle", 128, 701, 1000, 1104), ("odd outputs", 32, 301, 777, 1104),
    ("odd outputs", 128, 301, 777, 1104), ("odd", 64, 301, 777, 1001), ("odd", 128, 301, 777, 1001),
]
EXPECTED = {"odd outputs": (2, 1, 2, True), "odd": (2, 1, 2, False), **SHAPES}


def single(g, tokens, width, dtype):
    """Tokens with one input each, its place, and its value."""
    at = torch.randint(0, width, (tokens,), generator=g)
    value = torch.randn(tokens, generator=g).to(dtype)
    x = torch.zeros(tokens, width, dtype=dtype)
    x[torch.arange(tokens), at] = value
    return x, at.numpy(), host(value)


def of_single(at, value, w, group):
    """x s, c and z of every output of such tokens, [tokens, N]."""
    codes, scales, zeros = w
    s = host(scales)[at // group]
    z = np.full_like(s, 8.0) if zeros is None else host(zeros)[at // group]
    return value[:, None] * s, host(codes.float())[:, at].T, z


def within(got, want, bound):
    off = np.abs(host(got) - want)
    assert (off <= bound).all(), (float((off - bound).max()), float((off > bound).mean()))


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("shape", FP32, ids=str)
def test_fp32_inputs_keep_24_bits(device, shape, zeros):
    tile, group, tokens, outputs, width = shape
    print(f"24 bits {shape} {zeros}", flush=True)
    g = torch.Generator().manual_seed(sum(shape[1:]))
    x, at, value = single(g, tokens, width, torch.float32)
    weights = [weight(g, outputs, width, group, zeros, torch.float32) for _ in range(2)]
    args = (x.to(device), *on(device, weights[0]), group)
    got = linear_4bit(*args)
    torch.cuda.synchronize()
    exact, bound = [], []
    for w in weights:
        xs, c, z = of_single(at, value, w, group)
        exact.append(xs * (c - z))
        bound.append(U * (8 * np.abs(xs * (c - 8)) + 16 * np.abs(xs * (z - 8)) + np.abs(exact[-1]))
                     + 1e-37)
    within(got, exact[0], bound[0])
    assert instance(lambda: linear_4bit(*args)) == EXPECTED.get(tile)
    (gc, gs, gz), (uc, us, uz) = [on(device, w) for w in weights]
    got = gated_linear_4bit(x.to(device), gc, gs, uc, us, gz, uz, group, "silu")
    torch.cuda.synchronize()
    act = torch.nn.functional.silu(torch.from_numpy(exact[0])).numpy()
    d_act = 1.13 * bound[0] + 8 * U * np.abs(act)
    within(got, act * exact[1], d_act * (np.abs(exact[1]) + bound[1]) + np.abs(act) * bound[1]
           + 2 * U * np.abs(act * exact[1]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [
    ("few", 64, 3, 100, 576), ("few", 128, 31, 333, 260), ("wide", 64, 2099, 2000, 1104),
    ("middle", 32, 701, 2000, 304), ("small", 64, 499, 1000, 2104), ("odd outputs", 32, 301, 777, 1104),
    ("odd", 64, 333, 777, 1001)], ids=str)
def test_scales_keep_24_bits(device, shape, dtype):
    tile, group, tokens, outputs, width = shape
    print(f"scales of 24 bits {shape} {dtype}", flush=True)
    g = torch.Generator().manual_seed(sum(shape[1:]))
    x, at, value = single(g, tokens, width, dtype)
    for zeros in (False, True):
        w = weight(g, outputs, width, group, zeros, torch.float32)
        args = (x.to(device), *on(device, w), group)
        got = linear_4bit(*args)
        torch.cuda.synchronize()
        xs, c, z = of_single(at, value, w, group)
        exact = xs * (c - z)
        least = 2.0 ** -25 if dtype == torch.float16 else 1e-37
        within(got, exact, torch.finfo(dtype).eps / 2 * np.abs(exact)
               + 16 * U * np.abs(xs) * (32 + c + np.abs(z)) + least)
    assert instance(lambda: linear_4bit(*args)) == EXPECTED.get(tile)


def spread(x, w, group):
    """The mean square of the error that the roundings of fp32 tokens give an output."""
    codes, scales, _ = w
    x, c, s = host(x), host(codes.float()) - 8, host(scales)
    square, total, chunks = 0.0, np.zeros((len(x), len(c))), 0
    for first in range(0, x.shape[1], min(group, 128)):
        last = min(first + min(group, 128), x.shape[1])
        v, off = np.zeros_like(total), np.zeros_like(total)
        for at in range(first, last, 32):
            some = slice(at, min(at + 32, last))
            before, v = v, v + x[:, some] @ c[:, some].T
            off += 3 * 2 * U * np.maximum(np.abs(before), np.abs(v))
        square = square + (s[first // group] * off) ** 2
        total += s[first // group] * v
        chunks += 1
    return total, np.mean(square + (chunks + 8) * (U * total) ** 2)


@pytest.mark.parametrize("shape", [
    ("few", 128, 5, 400, 2304), ("few", 64, 65, 1000, 304), ("wide", 32, 2099, 2000, 304),
    ("wide", 128, 2099, 2000, 1104), ("middle", 64, 1299, 1000, 304), ("middle", 128, 701, 1000, 1104),
    ("odd outputs", 128, 301, 777, 1104), ("odd", 64, 301, 777, 1001)], ids=str)
def test_fp32_inputs_of_one_sign(device, shape):
    tile, group, tokens, outputs, width = shape
    print(f"one sign {shape}", flush=True)
    g = torch.Generator().manual_seed(sum(shape[1:]))
    x = 4 + torch.randn(tokens, width, generator=g)
    w = weight(g, outputs, width, group, False, torch.float32)
    args = (x.to(device), *on(device, w), group)
    got = linear_4bit(*args)
    torch.cuda.synchronize()
    want, square = spread(x, w, group)
    off = np.sqrt(np.mean((host(got) - want) ** 2))
    print(f"  rms {off:.3g}, bound {np.sqrt(square):.3g}", flush=True)
    assert off <= np.sqrt(square), float(off / np.sqrt(square))
    assert instance(lambda: linear_4bit(*args)) == EXPECTED.get(tile)


@pytest.mark.parametrize("shape", [
    (torch.bfloat16, "wide", 32, 2099, 2000, 304), (torch.bfloat16, "middle", 32, 701, 2000, 304),
    (torch.float16, "small", 32, 499, 2000, 304), (torch.float16, "odd outputs", 64, 301, 777, 1104),
    (torch.bfloat16, "odd", 64, 333, 777, 1001), (torch.float32, "wide", 32, 2099, 2000, 304),
    (torch.float32, "middle", 64, 1299, 1000, 304), (torch.float32, "odd", 64, 301, 777, 1001),
    (torch.float32, "few", 64, 65, 1000, 304)], ids=str)
def test_inputs_that_are_not_finite(device, shape):
    """An infinity or NaN makes all of its token's outputs NaN, and no other's."""
    dtype, tile, group, tokens, outputs, width = shape
    print(f"not finite {shape}", flush=True)
    g = torch.Generator().manual_seed(sum(shape[2:]))
    x = torch.randn(tokens, width, generator=g).to(dtype)
    for zeros in (False, True):
        w = on(device, weight(g, outputs, width, group, zeros, dtype))
        plain = linear_4bit(x.to(device), *w, group)
        y = x.clone()
        bad = {0: float("inf"), 17: float("-inf"), 40: float("nan"), tokens - 1: float("inf")}
        for i, (token, what) in enumerate(bad.items()):
            y[token, (37 * i + width - 1) % width] = what
        y = y.to(device)
        got = linear_4bit(y, *w, group)
        assert torch.isnan(got[list(bad)]).all()
        others = [i for i in range(tokens) if i not in bad]
        assert torch.equal(got[others], plain[others])
    assert instance(lambda: linear_4bit(y, *w, group)) == EXPECTED.get(tile)
