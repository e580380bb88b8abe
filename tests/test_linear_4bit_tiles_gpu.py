"""Products with 4-bit weights of many tokens: every shape of tile that such calls take, against
oracle/few_bits.py within the bounds of test_linear_4bit_gpu.py."""
from __future__ import annotations

import re

import numpy as np
import pytest
import torch

from launched import launched
from relation_lm.kernels.linear_4bit import gated_linear_4bit, linear_4bit
from test_linear_4bit_gpu import U, check, host, on, product, weight

pytestmark = pytest.mark.gpu

# Waves along rows, tokens and parts of the inputs; whether inputs come by DMA.
SHAPES = {"wide": (4, 2, 1, True), "middle": (2, 1, 2, True), "small": (1, 1, 4, True)}


def instance(call):
    """(waves' rows, tokens, parts, aligned) of the tile kernel that the call takes, or None."""
    names = launched(call)
    if "linear_4bit_kernel" in names:
        return None
    plain = re.search(r"linear_4bit_tile_kernel<.*, \d+, \d+, (\d+), (\d+), (\d+), (\w+), \w+>", names)
    if plain:
        return int(plain[1]), int(plain[2]), int(plain[3]), plain[4] == "true"
    mangled = re.search(r"linear_4bit_tile_kernel.*Li\d+ELi\d+ELi(\d+)ELi(\d+)ELi(\d+)ELb(\d)ELb\dE", names)
    assert mangled, names
    return tuple(int(mangled[i]) for i in (1, 2, 3)) + (mangled[4] == "1",)


PLAIN = [
    # tile, group, tokens, outputs, width
    ("wide", 32, 2099, 2000, 304), ("wide", 64, 2099, 2000, 1104), ("wide", 128, 2099, 2000, 1104),
    ("wide", 128, 2099, 2000, 2104), ("wide", 256, 2099, 2000, 304), ("wide", 32, 2099, 2000, 1104),
    ("middle", 32, 701, 2000, 304), ("middle", 32, 2099, 504, 2104), ("middle", 64, 2099, 1000, 1104),
    ("middle", 128, 701, 2000, 1104), ("middle", 256, 2099, 1000, 2104),
    ("middle", 128, 2099, 1000, 1104), ("middle", 256, 701, 2000, 304),
    ("small", 32, 499, 2000, 304), ("small", 32, 701, 1000, 1104), ("small", 64, 499, 1000, 2104),
    ("small", 128, 499, 2000, 304), ("small", 256, 701, 1000, 1104), ("small", 64, 299, 2000, 1104),
    ("few", 32, 299, 2000, 304), ("few", 128, 201, 2000, 304), ("few", 256, 499, 1000, 1104),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", PLAIN, ids=str)
def test_linear(device, shape, dtype):
    tile, group, tokens, outputs, width = shape
    print(f"tiles {shape} {dtype}", flush=True)
    g = torch.Generator().manual_seed(sum(shape[1:]))
    x = torch.randn(tokens, width, generator=g).to(dtype)
    bias = torch.randn(outputs, generator=g)
    for scale_dtype, zeros in ((dtype, True), (torch.float32, False)):
        w = weight(g, outputs, width, group, zeros, scale_dtype)
        args = (x.to(device), *on(device, w), group, bias.to(device))
        got = linear_4bit(*args)
        torch.cuda.synchronize()
        want, d = product(x, w, group)
        want = want + host(bias)
        check(got, want, d + U * (np.abs(want) + d), dtype)
        assert instance(lambda: linear_4bit(*args)) == SHAPES.get(tile)


GATED = [
    ("wide", 32, 2099, 1000, 304), ("wide", 64, 2099, 1000, 1104), ("wide", 128, 2099, 1000, 1104),
    ("middle", 32, 701, 1000, 1104), ("middle", 64, 701, 2000, 1104),
    ("middle", 128, 1499, 504, 1104), ("middle", 256, 499, 2000, 304),
    ("small", 32, 499, 1000, 1104), ("small", 64, 201, 2000, 1104), ("small", 128, 299, 1000, 2104),
    ("few", 32, 201, 2000, 304),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", GATED, ids=str)
def test_gated_linear(device, shape, dtype):
    tile, group, tokens, outputs, width = shape
    print(f"gated tiles {shape} {dtype}", flush=True)
    g = torch.Generator().manual_seed(sum(shape[1:]) + 1)
    x = (2 * torch.randn(tokens, width, generator=g)).to(dtype)
    for scale_dtype, zeros in ((dtype, True), (torch.float32, False)):
        gate, up = [weight(g, outputs, width, group, zeros, scale_dtype) for _ in range(2)]
        (gc, gs, gz), (uc, us, uz) = on(device, gate), on(device, up)
        args = (x.to(device), gc, gs, uc, us, gz, uz, group, "silu")
        got = gated_linear_4bit(*args)
        torch.cuda.synchronize()
        (a, da), (b, db) = product(x, gate, group), product(x, up, group)
        act = torch.nn.functional.silu(torch.from_numpy(a)).numpy()
        d_act = 1.13 * da + 8 * U * np.abs(act)
        d = d_act * (np.abs(b) + db) + np.abs(act) * db
        check(got, act * b, d + U * np.abs(act * b), dtype)
        assert instance(lambda: gated_linear_4bit(*args)) == SHAPES.get(tile)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_any_alignment(device, group, dtype):
    print(f"unaligned {group} {dtype}", flush=True)
    g = torch.Generator().manual_seed(group)
    x = torch.randn(333, 1001, generator=g).to(dtype)
    w = weight(g, 777, 1001, group, True, dtype)
    args = (x.to(device), *on(device, w), group)
    got = linear_4bit(*args)
    torch.cuda.synchronize()
    check(got, *product(x, w, group), dtype)
    assert instance(lambda: linear_4bit(*args)) == (2, 1, 2, False)


def test_inputs_that_are_not_finite(device):
    """An infinity or NaN reaches its own token's outputs and no other's."""
    g = torch.Generator().manual_seed(9)
    for tile, group, tokens, outputs, width in (PLAIN[0], PLAIN[6], PLAIN[13]):
        x = torch.randn(tokens, width, generator=g).to(torch.bfloat16)
        w = on(device, weight(g, outputs, width, group, True, torch.bfloat16))
        plain = linear_4bit(x.to(device), *w, group)
        x[17, 5], x[90, width - 1] = float("inf"), float("nan")
        got = linear_4bit(x.to(device), *w, group)
        assert not torch.isfinite(got[17, 1]) and torch.isnan(got[90, 1])
        others = torch.ones(tokens, dtype=torch.bool)
        others[17] = others[90] = False
        assert torch.equal(got[others.to(device)], plain[others.to(device)])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize("scale_dtype", ["same", "fp32"])
def test_odd_outputs(device, group, scale_dtype, dtype):
    """Whole accesses of inputs, none of scales; plain and gated."""
    print(f"odd outputs {group} {scale_dtype} {dtype}", flush=True)
    g = torch.Generator().manual_seed(group)
    kind = torch.float32 if scale_dtype == "fp32" else dtype
    x = torch.randn(301, 1104, generator=g).to(dtype)
    gate, up = [weight(g, 777, 1104, group, True, kind) for _ in range(2)]
    args = (x.to(device), *on(device, gate), group)
    got = linear_4bit(*args)
    torch.cuda.synchronize()
    (a, da), (b, db) = product(x, gate, group), product(x, up, group)
    check(got, a, da, dtype)
    assert instance(lambda: linear_4bit(*args)) == (2, 1, 2, True)
    (gc, gs, gz), (uc, us, uz) = on(device, gate), on(device, up)
    got = gated_linear_4bit(x.to(device), gc, gs, uc, us, gz, uz, group, "silu")
    torch.cuda.synchronize()
    act = torch.nn.functional.silu(torch.from_numpy(a)).numpy()
    d_act = 1.13 * da + 8 * U * np.abs(act)
    check(got, act * b, d_act * (np.abs(b) + db) + np.abs(act) * db + U * np.abs(act * b), dtype)


FP32 = [
    # tile, group, tokens, outputs, width
    ("wide", 32, 2099, 2000, 304), ("wide", 64, 2099, 2000, 1104), ("wide", 256, 2099, 2000, 304),
    ("middle", 32, 1299, 1000, 1104), ("middle", 64, 1299, 1000, 304), ("middle", 128, 701, 1000, 1104),
    ("middle", 384, 299, 2000, 1104), ("odd outputs", 32, 301, 777, 1104),
    ("odd outputs", 64, 301, 1777, 1104), ("odd outputs", 128, 301, 777, 1104),
    ("odd", 32, 301, 777, 1001), ("odd", 64, 301, 777, 1001), ("odd", 128, 301, 777, 1001),
    ("few", 64, 65, 1000, 304),
]


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("shape", FP32, ids=str)
def test_fp32(device, shape, zeros):
    tile, group, tokens, outputs, width = shape
    print(f"fp32 tiles {shape} {zeros}", flush=True)
    g = torch.Generator().manual_seed(sum(shape[1:]))
    x = torch.randn(tokens, width, generator=g)
    gate, up = [weight(g, outputs, width, group, zeros, torch.float32) for _ in range(2)]
    args = (x.to(device), *on(device, gate), group)
    got = linear_4bit(*args)
    torch.cuda.synchronize()
    (a, da), (b, db) = product(x, gate, group), product(x, up, group)
    check(got, a, da, torch.float32)
    expected = {"odd outputs": (2, 1, 2, True), "odd": (2, 1, 2, False), **SHAPES}.get(tile)
    assert instance(lambda: linear_4bit(*args)) == expected
    (gc, gs, gz), (uc, us, uz) = on(device, gate), on(device, up)
    got = gated_linear_4bit(x.to(device), gc, gs, uc, us, gz, uz, group, "silu")
    torch.cuda.synchronize()
    act = torch.nn.functional.silu(torch.from_numpy(a)).numpy()
    d_act = 1.13 * da + 8 * U * np.abs(act)
    check(got, act * b, d_act * (np.abs(b) + db) + np.abs(act) * db + U * np.abs(act * b),
          torch.float32)
