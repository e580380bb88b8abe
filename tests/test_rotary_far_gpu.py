"""Rotary positions (rlm::rotary_to_caches) where the tokens' positions reach the end of int64."""
from __future__ import annotations

import pytest
import torch

from oracle import routed_layer
from relation_lm.kernels.rotary import rotary_to_caches
from test_rotary_gpu import check, host

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("ring", [False, True])
def test_positions_past_the_end_of_int64(device, ring, dtype):
    """Tokens that would stand past 2^63 - 1 turn as the last position does and leave the caches as
    they are.  (2^63 - 1 and its neighbours are 2^63 in float64: an angle of 2 at a frequency of
    2^-62, where a sum that had wrapped would turn by -2.)"""
    g = torch.Generator().manual_seed(1)
    query, key, value = (torch.randn(2, 5, 2, 16, generator=g).to(dtype) for _ in range(3))
    caches = [torch.randn(2, 8, 2, 16, generator=g).to(dtype) for _ in range(2)]
    mine = [c.to(device) for c in caches]
    freq = torch.tensor([2.0 ** -62, 2.0 ** -63, 3 * 2.0 ** -64])
    first = torch.tensor([2 ** 63 - 2, 2 ** 63 - 4])
    got = rotary_to_caches(query.to(device), key.to(device), value.to(device), first.to(device),
                           freq.to(device), *mine, False, 1.0, ring)
    torch.cuda.synchronize()
    last = torch.tensor(2 ** 63 - 1).numpy()
    check(got, query, routed_layer.rotary(host(query), last, freq.numpy(), False, 1.0), 3, False,
          1.0, dtype)
    turned = routed_layer.rotary(host(key), last, freq.numpy(), False, 1.0)
    left = torch.ones(2, 8, dtype=torch.bool)
    if ring:
        for b, many in ((0, 2), (1, 4)):      # tokens at positions up to 2^63 - 1
            rows = [(int(first[b]) + i) % 8 for i in range(many)]
            left[b, rows] = False
            check(mine[0][b:b + 1, rows], key[b:b + 1, :many], turned[b:b + 1, :many], 3, False, 1.0,
                  dtype)
            assert torch.equal(mine[1][b, rows].cpu(), value[b, :many])
    for cache, before in zip(mine, caches):
        assert torch.equal(cache.cpu()[left], before[left])
