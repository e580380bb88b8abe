"""Scores of block routing (rlm::block_route[_seq]) where its running log-sum-exp over the heads
could lose them: heads of infinite terms."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from relation_lm.kernels.routed_attention import block_route, block_route_seq
from test_block_route_gpu import check, inputs, oracle

pytestmark = pytest.mark.gpu

STATISTICS = ("mean", "std", "gamma", "bias")
# queries, blocks, head_dim: one query to a workgroup, four, four to a wave; a block to four lanes
# and to one.
FORMS = [(5, 20, 16), (5, 20, 12), (1030, 300, 16), (1030, 300, 12), (17000, 40, 16),
         (17000, 40, 12)]


def route(device, x, positions, block, window, top):
    got = block_route_seq(x["query"][:, :, 0].to(device), *(x[k].to(device) for k in STATISTICS),
                          positions.to(device), block, window, top, False)
    torch.cuda.synchronize()
    return got


@pytest.mark.parametrize("queries,blocks,head_dim", FORMS)
def test_heads_without_a_term(device, queries, blocks, head_dim):
    """A bias of -inf takes a head out of the blocks at its distance, the first heads too; with
    every head taken out a block is not picked."""
    print(f"block_route_seq {queries} {blocks} {head_dim} -inf", flush=True)
    g = torch.Generator().manual_seed(queries + head_dim)
    x = inputs(g, 1, queries, 1, 4, head_dim, blocks, 9, torch.bfloat16)
    for bucket, heads in ((2, [0, 1]), (3, [0, 1, 2]), (4, [1, 2, 3]), (5, [0]), (6, [0, 1, 2, 3])):
        x["bias"][heads, bucket] = -float("inf")
    positions = torch.randint(0, blocks * 8 + 20, (1, queries), generator=g)
    got = route(device, x, positions, 8, 20, 12)
    # For the oracle all of a block's heads at -1e200: below what is picked.
    x["bias"] = x["bias"].double()
    x["bias"][:, 6] = -1e200
    with np.errstate(over="ignore"):
        want = oracle(x, positions.numpy(), 8, 20, 12, False)
    check(got, [w[:, :, 0] for w in want])


@pytest.mark.parametrize("queries,blocks,head_dim", FORMS)
def test_two_heads_of_infinite_terms(device, queries, blocks, head_dim):
    """log(inf + inf + ..) is infinite: that block is first, and the others as without it."""
    print(f"block_route_seq {queries} {blocks} {head_dim} inf", flush=True)
    g = torch.Generator().manual_seed(queries + head_dim)
    x = inputs(g, 1, queries, 1, 4, head_dim, blocks, 9, torch.float32)
    positions = torch.full((1, queries), blocks * 8 - 1)
    want = route(device, x, positions, 8, 20, 20)
    x["std"][0, 9, :2, 0] = float("inf")
    got = route(device, x, positions, 8, 20, 20)
    assert (got[0][..., 0] == 9).all() and torch.isposinf(got[1][..., 0]).all()
    rest = want[0] != 9
    for row in range(0, queries, max(1, queries // 50)):
        kept = rest[0, row]
        n = min(19, int(kept.sum()))
        for mine, theirs in zip(got, want):
            assert torch.equal(mine[0, row, 1:1 + n], theirs[0, row][kept][:n])


def test_one_token_whose_first_heads_have_no_term(device):
    g = torch.Generator().manual_seed(3)
    x = inputs(g, 6, 1, 2, 4, 16, 70, 9, torch.float16)
    x["bias"][:2] = -float("inf")
    position = torch.tensor(70 * 8 - 1)
    got = block_route(x["query"][:, 0].to(device), *(x[k].to(device) for k in STATISTICS),
                      position.to(device), 8, 20, 12, False)
    torch.cuda.synchronize()
    check(got, [w[:, 0] for w in oracle(x, position.numpy(), 8, 20, 12, False)])
