"""Cache rows whose key scale or whose value scale is not finite: NaN for the queries that see one, whatever the
score's sign, and nothing for the others."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from launched import launched
from oracle import routed_layer
from relation_lm.kernels.routed_attention import routed_attention_quantized
from test_routed_attention_quantized_gpu import DTYPES, U, case, check, host, raw_seq, values
from test_routed_attention_quantized_tiles_gpu import ROWS

pytestmark = pytest.mark.gpu

BAD = [float("inf"), float("-inf"), float("nan")]


def spoil(rows, at, what):
    codes, scales = rows[0], rows[1].clone()
    scales[:, at] = what
    return codes, scales


# A query to a workgroup, shared tiles, and one that takes either by its type.
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("which", ["key", "value"])
@pytest.mark.parametrize("kernel, queries, dim, block", [
    ("attend_codes", 40, 64, 64), ("attend_codes", 9, 256, 20), ("attend_tile", 301, 64, 64),
    ("attend", 301, 96, 12), ("attend_tile", 301, 64, 20), ("attend_tile", 301, 128, 64),
    ("attend_tile", 700, 64, 20), ("attend_tile", 700, 96, 64)])
def test_scales_that_are_not_finite(device, kernel, queries, dim, block, which, dtype):
    print(f"scales {kernel} {queries} {dim} {block} {which} {dtype}", flush=True)
    g = torch.Generator().manual_seed(queries + dim + block)
    window, at = 30, 200
    query, key, value, positions, picks = case(g, 2, queries, 32, 4, dim, ROWS, block,
                                               4 if block == 64 else 16, 1, dtype)
    picks = torch.where(picks == at // block, -1, picks)      # windows alone see the row
    positions[:, 0] = at
    expected = routed_layer.attention(host(query), values(key), values(value), picks.numpy(),
                                      positions.numpy(), block, window, dim ** -0.5)
    sees = ((positions >= at) & (positions < at + window)).numpy()
    assert (sees.sum(1) > 1).all() or queries < 40
    for what in BAD:
        spoiled = {"key": key, "value": value}
        spoiled[which] = spoil(spoiled[which], at, what)
        parts = query, spoiled["key"], spoiled["value"], positions, picks
        out, lse = raw_seq(device, parts, block, window)
        assert torch.isnan(out[sees]).all()
        check(out[~sees], lse[~sees], [x[~sees] for x in expected], dtype, dim)
        if which == "key":
            assert torch.isnan(lse[sees]).all()
        else:                               # the log-sum-exp has no values
            bound = U * ((3 * dim + 7) * expected[3] + ROWS + 16 + np.abs(expected[1]))
            assert (np.abs(host(lse) - expected[1]) <= bound)[sees].all()
    assert kernel in launched(lambda: raw_seq(device, parts, block, window))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ring", [False, True])
@pytest.mark.parametrize("which", ["key", "value"])
def test_one_token(device, which, ring, dtype):
    print(f"one token {which} {ring} {dtype}", flush=True)
    g = torch.Generator().manual_seed(3)
    query, key, value, _, _ = case(g, 4, 1, 8, 2, 64, 128, 16, 2, 1, dtype)
    position = torch.tensor([60, 90, 100, 127])
    picks = torch.tensor([[0, 1]], dtype=torch.int32).expand(4, 2).contiguous()
    for what in BAD:
        # Row 70 is in the window of the second request alone, row 20 among everybody's picks.
        for row, sees in ((70, [1]), (20, [0, 1, 2, 3])):
            spoiled = {"key": key, "value": value}
            spoiled[which] = spoil(spoiled[which], row, what)
            out, lse = routed_attention_quantized(
                query[:, 0].to(device), *(spoiled[n][0].to(device) for n in ("key", "value")),
                *(spoiled[n][1].to(device) for n in ("key", "value")), picks.to(device),
                position.to(device), 16, 24, None, ring)
            bad = torch.isnan(out).all(-1).all(-1).cpu()
            assert bad.tolist() == [b in sees for b in range(4)]
            assert torch.isfinite(out[~bad.to(device)]).all()
            assert torch.isnan(lse).all(-1).cpu().tolist() == (
                bad.tolist() if which == "key" else [False] * 4)
