"""GPU parity of block routing (rlm::block_route[_seq]) against the oracle's float64 scores:
the picks are equal, ties to the lowest block; the scores are the float64 ones rounded to fp32
(one step at most where the two float64 values straddle a rounding border)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import routed_layer
from relation_lm.kernels.routed_attention import block_route, block_route_seq

pytestmark = pytest.mark.gpu


def inputs(g, batch, queries, slots, heads, head_dim, blocks, buckets, dtype):
    width = heads * head_dim
    return dict(
        query=torch.randn(batch, queries, slots, width, generator=g).to(dtype),
        mean=0.5 * torch.randn(batch, blocks, heads, head_dim, generator=g),
        std=0.5 + torch.rand(batch, blocks, heads, head_dim, generator=g),
        gamma=torch.randn(heads, generator=g), bias=torch.randn(heads, buckets, generator=g))


def check(got, want):
    blocks, scores = (x.cpu().numpy() for x in got)
    assert np.array_equal(blocks, want[0])
    seen = np.isfinite(want[1])
    assert (np.isneginf(scores) == ~seen).all()
    assert (np.abs(scores[seen] - want[1][seen]) <= np.spacing(np.abs(want[1][seen]))).all()


def oracle(x, positions, block, window, top, strict, ring=False):
    return routed_layer.block_route(
        x["query"].double().numpy(), x["mean"].numpy(), x["std"].numpy(),
        x["gamma"].double().numpy(), x["bias"].double().numpy(), positions, block, window, top,
        strict, ring)


SEQ = [
    # batch, queries, slots, heads, head_dim, blocks, buckets, block, window, top
    (1, 1, 1, 4, 16, 1, 16, 8, 16, 1),
    (2, 700, 1, 4, 16, 64, 16, 16, 32, 8),
    (1, 333, 4, 8, 8, 37, 5, 9, 13, 4),
    (3, 515, 1, 1, 64, 20, 16, 30, 64, 16),
    (1, 1030, 2, 3, 12, 130, 1, 8, 17, 20),
    (1, 600, 1, 2, 4, 70, 16, 9, 5, 64),
    (1, 90, 1, 4, 100, 12, 16, 8, 16, 3),
    (2, 520, 1, 16, 16, 9, 16, 64, 128, 12),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("strict", [False, True])
@pytest.mark.parametrize("shape", SEQ, ids=[str(s) for s in SEQ])
def test_sequence_form(device, shape, strict, dtype):
    batch, queries, slots, heads, head_dim, blocks, buckets, block, window, top = shape
    print(f"block_route_seq {shape} {strict} {dtype}", flush=True)
    g = torch.Generator().manual_seed(sum(shape))
    x = inputs(g, batch, queries, slots, heads, head_dim, blocks, buckets, dtype)
    random = torch.randint(-2, blocks * block + 40, (batch, queries), generator=g)
    for positions in (random, torch.arange(queries, dtype=torch.int32)):
        query = x["query"] if slots > 1 else x["query"][:, :, 0]
        got = block_route_seq(query.to(device), *(x[k].to(device) for k in
                                                  ("mean", "std", "gamma", "bias")),
                              positions.to(device), block, window, top, strict)
        torch.cuda.synchronize()
        want = oracle(x, positions.numpy(), block, window, top, strict)
        check(got, want if slots > 1 else [w[:, :, 0] for w in want])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("batch,blocks,top,slots", [(1, 16, 4, 1), (8, 16, 4, 3), (20, 2048, 16, 4),
                                                    (3, 333, 64, 1), (1, 5, 9, 2)])
def test_decode_form(device, batch, blocks, top, slots, dtype):
    print(f"block_route {batch} {blocks} {top} {slots} {dtype}", flush=True)
    g = torch.Generator().manual_seed(batch + blocks)
    x = inputs(g, batch, 1, slots, 4, 16, blocks, 16, dtype)
    each = torch.randint(0, blocks * 32, (batch,), generator=g)
    for position in (each, torch.tensor(blocks * 32 - 1)):
        query = x["query"][:, 0] if slots > 1 else x["query"][:, 0, 0]
        got = block_route(query.to(device), *(x[k].to(device) for k in
                                              ("mean", "std", "gamma", "bias")),
                          position.to(device), 32, 64, top, False)
        torch.cuda.synchronize()
        want = oracle(x, position.numpy().reshape(-1, 1), 32, 64, top, False)
        check(got, [w[:, 0] if slots > 1 else w[:, 0, 0] for w in want])


@pytest.mark.parametrize("queries,blocks,head_dim,top", [
    (256, 300, 16, 9), (257, 300, 16, 9),        # one query / four to a workgroup, 16 waves
    (1030, 300, 16, 64), (1030, 300, 12, 20),    # four, fewer waves; a lane to a block
    (4095, 16, 16, 3), (4097, 16, 16, 3),        # one wave for all blocks: one query / four
    (17000, 40, 16, 5),                          # four queries to a wave
])
def test_queries_that_share_workgroups(device, queries, blocks, head_dim, top):
    g = torch.Generator().manual_seed(queries)
    x = inputs(g, 1, queries, 1, 2, head_dim, blocks, 9, torch.bfloat16)
    positions = torch.randint(-1, blocks * 8 + 20, (1, queries), generator=g)
    got = block_route_seq(x["query"][:, :, 0].to(device), *(x[k].to(device) for k in
                                                            ("mean", "std", "gamma", "bias")),
                          positions.to(device), 8, 20, top, False)
    torch.cuda.synchronize()
    check(got, [w[:, :, 0] for w in oracle(x, positions.numpy(), 8, 20, top, False)])


@pytest.mark.parametrize("batch,blocks", [(300, 300), (4100, 16)])
def test_large_decode_batches(device, batch, blocks):
    g = torch.Generator().manual_seed(batch)
    x = inputs(g, batch, 1, 1, 2, 16, blocks, 9, torch.bfloat16)
    position = torch.randint(0, blocks * 8, (batch,), generator=g)
    got = block_route(x["query"][:, 0, 0].to(device), *(x[k].to(device) for k in
                                                        ("mean", "std", "gamma", "bias")),
                      position.to(device), 8, 20, 4, False)
    torch.cuda.synchronize()
    want = oracle(x, position.numpy()[:, None], 8, 20, 4, False)
    check(got, [w[:, 0, 0] for w in want])


@pytest.mark.parametrize("strict", [False, True])
@pytest.mark.parametrize("t", [-1, 0, 31, 32, 500, 511, 512, 700, 4095, 2**35 + 3])
def test_ring(device, t, strict):
    g = torch.Generator().manual_seed(t % 1000)
    x = inputs(g, 3, 1, 2, 4, 16, 16, 16, torch.bfloat16)
    got = block_route(x["query"][:, 0].to(device), *(x[k].to(device) for k in
                                                     ("mean", "std", "gamma", "bias")),
                      torch.tensor(t, device=device), 32, 64, 5, strict, True)
    torch.cuda.synchronize()
    want = oracle(x, np.array(t), 32, 64, 5, strict, True)
    check(got, [w[:, 0] for w in want])


def test_ring_blocks_past_int32_are_not_picked(device):
    """16 blocks on both sides of number 2^31: the picks are those below it."""
    g = torch.Generator().manual_seed(7)
    x = inputs(g, 3, 1, 2, 4, 16, 16, 16, torch.bfloat16)
    t = 32 * (2**31 + 4) + 31
    got = block_route(x["query"][:, 0].to(device), *(x[k].to(device) for k in
                                                     ("mean", "std", "gamma", "bias")),
                      torch.tensor(t, device=device), 32, 64, 14, False, True)
    torch.cuda.synchronize()
    ranked = oracle(x, np.array(t), 32, 64, 16, False, True)     # blocks from 2^31 on: negative
    want = [np.full((3, 2, 14), -1, np.int32), np.full((3, 2, 14), -np.inf, np.float32)]
    for row in np.ndindex(3, 2):
        blocks, scores = (w[row[0], 0, row[1]] for w in ranked)
        held = blocks >= 0
        assert held.sum() == 11
        want[0][row][:11], want[1][row][:11] = blocks[held], scores[held]
    check(got, want)


@pytest.mark.parametrize("queries", [5, 700])
def test_positions_at_the_ends_of_int64(device, queries):
    """The last one has every block of the cache, all in the farthest bucket; the first none."""
    g = torch.Generator().manual_seed(8)
    x = inputs(g, 1, queries, 1, 4, 16, 20, 16, torch.bfloat16)
    positions = torch.full((queries,), 2**62)
    want = oracle(x, positions.numpy(), 8, 16, 20, True)
    want[0][:, 1::2], want[1][:, 1::2] = -1, -np.inf
    positions[::4], positions[1::2] = 2**63 - 1, -2**63
    got = block_route_seq(x["query"][:, :, 0].to(device), *(x[k].to(device) for k in
                                                            ("mean", "std", "gamma", "bias")),
                          positions.to(device), 8, 16, 20, True)
    torch.cuda.synchronize()
    check(got, [w[:, :, 0] for w in want])


def test_widest_tables(device):
    """64 heads of 4 features with 32 buckets, four queries to a wave: the most shared memory."""
    g = torch.Generator().manual_seed(9)
    x = inputs(g, 1, 530, 1, 64, 4, 70, 32, torch.bfloat16)
    positions = torch.arange(530)
    got = block_route_seq(x["query"][:, :, 0].to(device), *(x[k].to(device) for k in
                                                            ("mean", "std", "gamma", "bias")),
                          positions.to(device), 7, 9, 11, False)
    torch.cuda.synchronize()
    check(got, [w[:, :, 0] for w in oracle(x, positions.numpy(), 7, 9, 11, False)])


@pytest.mark.parametrize("queries,blocks", [(300, 300), (17000, 20), (200, 300)])
def test_widest_router_with_most_buckets(device, queries, blocks):
    """16 heads of 16 with 128 buckets: the most shared memory of each launch form."""
    g = torch.Generator().manual_seed(queries)
    x = inputs(g, 1, queries, 1, 16, 16, blocks, 128, torch.bfloat16)
    positions = torch.randint(0, blocks * 8, (1, queries), generator=g)
    got = block_route_seq(x["query"][:, :, 0].to(device), *(x[k].to(device) for k in
                                                            ("mean", "std", "gamma", "bias")),
                          positions.to(device), 8, 20, 64, False)
    torch.cuda.synchronize()
    check(got, [w[:, :, 0] for w in oracle(x, positions.numpy(), 8, 20, 64, False)])


@pytest.mark.parametrize("queries", [1, 600])
@pytest.mark.parametrize("ring", [False, True])
def test_ties_go_to_the_lowest_block(device, queries, ring):
    """Blocks with the same statistics, in one distance bucket, score the same bits."""
    if ring and queries > 1:
        pytest.skip("the ring form takes one query")
    g = torch.Generator().manual_seed(4)
    x = inputs(g, 1, queries, 1, 4, 16, 64, 1, torch.float32)
    kinds = torch.randint(0, 3, (64,), generator=g)
    x["mean"] = x["mean"][:, kinds].contiguous()
    x["std"] = x["std"][:, kinds].contiguous()
    t = 64 * 8 + (100 if ring else -1)
    want = oracle(x, np.array(t), 8, 16, 12, False, ring)
    args = [x[k].to(device) for k in ("mean", "std", "gamma", "bias")]
    if queries == 1:
        got = block_route(x["query"][:, 0, 0].to(device), *args, torch.tensor(t, device=device), 8,
                          16, 12, False, ring)
        check(got, [w[:, 0, 0] for w in want])
    else:
        got = block_route_seq(x["query"][:, :, 0].to(device), *args,
                              torch.tensor(t, device=device), 8, 16, 12, False)
        check(got, [w[:, :, 0] for w in want])


def test_scores_that_are_no_numbers_are_not_picked(device):
    g = torch.Generator().manual_seed(5)
    x = inputs(g, 1, 600, 1, 4, 16, 20, 16, torch.float32)
    x["mean"][0, 3, 1, 2] = float("nan")
    x["mean"][0, 7] = -float("inf")
    x["std"][0, 9, 0, 0] = float("inf")          # an infinite score: first
    blocks, scores = block_route_seq(x["query"][:, :, 0].to(device),
                                     *(x[k].to(device) for k in ("mean", "std", "gamma", "bias")),
                                     torch.tensor(20 * 8 - 1, device=device), 8, 16, 20, False)
    blocks, scores = blocks.cpu(), scores.cpu()
    assert not torch.isin(blocks, torch.tensor([3, 7])).any()
    assert not torch.isnan(scores).any()
    assert (blocks[..., 0] == 9).all() and torch.isposinf(scores[..., 0]).all()
    assert (blocks[..., 18:] == -1).all() and torch.isneginf(scores[..., 18:]).all()


def test_query_views(device):
    g = torch.Generator().manual_seed(6)
    x = inputs(g, 2, 300, 2, 4, 16, 20, 16, torch.bfloat16)
    args = [x[k].to(device) for k in ("mean", "std", "gamma", "bias")]
    positions = torch.arange(300, device=device)
    want = block_route_seq(x["query"].to(device), *args, positions, 8, 16, 4, False)
    wide = torch.randn(2, 300, 5, 70, generator=g).to(torch.bfloat16).to(device)
    wide[:, :, 1:5:2, 3:67] = x["query"].to(device)
    got = block_route_seq(wide[:, :, 1:5:2, 3:67], *args, positions, 8, 16, 4, False)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
