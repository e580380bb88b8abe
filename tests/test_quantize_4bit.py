"""quantize_4bit of weights that are not finite and of zeros (no GPU needed)."""
from __future__ import annotations

import pytest
import torch

from relation_lm.kernels.linear_4bit import pack_4bit, quantize_4bit


def stands_for(codes, scales, zeros, group):
    pick = torch.arange(codes.shape[1]) // group
    z = 8.0 if zeros is None else zeros[pick].T
    return (codes.float() - z) * scales[pick].T


@pytest.mark.parametrize("symmetric", [False, True])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), float("-inf")])
def test_groups_that_are_not_finite(symmetric, what):
    """Such a group's values are no numbers where the weight is none, its codes are codes, and the other groups
    stay as they are."""
    g = torch.Generator().manual_seed(1)
    weight = torch.randn(5, 96, generator=g)
    plain = stands_for(*quantize_4bit(weight, 32, symmetric), 32)
    weight[2, 40] = what
    codes, scales, zeros = quantize_4bit(weight, 32, symmetric)
    assert int(codes.max()) <= 15
    pack_4bit(codes)
    values = stands_for(codes, scales, zeros, 32)
    assert not torch.isfinite(values[2, 32:64]).any()
    rest = torch.ones_like(weight, dtype=torch.bool)
    rest[2, 32:64] = False
    assert torch.equal(values[rest], plain[rest])


@pytest.mark.parametrize("symmetric", [False, True])
def test_groups_of_zeros(symmetric):
    weight = torch.zeros(3, 70)
    weight[1, 65] = 1.0
    codes, scales, zeros = quantize_4bit(weight, 32, symmetric)
    assert (scales[:2] == 1).all() and torch.equal(stands_for(codes, scales, zeros, 32), weight)
