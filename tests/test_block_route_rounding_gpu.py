"""Block routing (rlm::block_route_seq) ranks by the scores that the selection ranks by: float64
log-sum-exps, rounded to fp32 once.

The scores of the first test lie within a few of 0, where fp32 numbers are close.  A head's term is a
sum of up to 33 float64 numbers with partial sums below 4; the roundings, 2^-53 of a partial sum at
most and independent of each other, add up to some sqrt(33) 2^-53 2 = 1.3e-15; the exponentials and
the logarithm add less than 1e-15, and the oracle is off as much.  Two such numbers round to
different fp32 numbers only where a border lies between them: for a share of 5e-15 over the spacing
of fp32 numbers, 3e-8 for scores of a quarter, less for larger ones and 2^n times as much for the
2^-n of the scores that are 2^n times smaller: some 2e-7 to 1e-6 of the scores.  Of the 0.3 to 0.9
million of a case none or one is expected; four are allowed.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from relation_lm.kernels.relation_select import relation_select_packed_seq
from relation_lm.kernels.routed_attention import block_route_seq
from relation_lm.workloads import RelationConfig, select_args, selection_inputs
from test_block_route_gpu import inputs, oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("batch,queries,blocks,head_dim", [
    (4, 4500, 64, 16), (4, 4500, 64, 8), (8, 600, 300, 16)])
def test_scores_are_float64_ones_rounded_once(device, batch, queries, blocks, head_dim):
    print(f"block_route_seq {batch} {queries} {blocks} {head_dim}", flush=True)
    g = torch.Generator().manual_seed(queries + head_dim)
    x = inputs(g, batch, queries, 1, 4, head_dim, blocks, 16, torch.bfloat16)
    x["gamma"] -= 6.0                           # content and spread of about one half,
    x["bias"] = 0.5 * x["bias"] - 1.4           # less log 4
    positions = torch.randint(blocks * 4, blocks * 8, (batch, queries), generator=g)
    got = block_route_seq(x["query"][:, :, 0].to(device), *(x[k].to(device) for k in
                                                            ("mean", "std", "gamma", "bias")),
                          positions.to(device), 8, 20, 64, False)
    torch.cuda.synchronize()
    scores = got[1].cpu().numpy()
    many = wrong = 0
    for b in range(batch):
        one = {k: v[b:b + 1] if k in ("query", "mean", "std") else v for k, v in x.items()}
        want = oracle(one, positions[b:b + 1].numpy(), 8, 20, 64, False)[1][0, :, 0]
        seen = np.isfinite(want)
        assert np.abs(want[seen]).max() < 8 and np.median(np.abs(want[seen])) > 0.2
        many += int(seen.sum())
        wrong += int((scores[b][seen] != want[seen]).sum())
    print(f"{wrong} of {many} scores differ", flush=True)
    assert many > 250_000 and wrong <= 4


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("strict", [False, True])
def test_first_pick_is_the_selections(device, strict, dtype):
    """Keys whose scores fall along the cache: with a window of one position and one routed block
    the anchor is the first position of the block that the selection's router picks."""
    cfg = RelationConfig(name="router", batch=3, context=512, d_model=256, block_size=8,
                         local_window=1, top_blocks=1, k_out=1, dtype=dtype, seed=77,
                         strict_valid=strict)
    inp = selection_inputs(cfg, device=device)
    for part in ("anchor_block_mean", "anchor_block_std"):
        # Pairs of blocks that differ in few bits: their scores tie or are next to each other.
        inp[part] = inp[part].float()
        inp[part][:, 1::2] = inp[part][:, ::2]
    inp["anchor_block_mean"][:, 1::2, 0, 0] *= 1 + 2.0 ** -23
    row = torch.arange(512, device=device)
    inp["anchor_query"].zero_()
    inp["anchor_query"][..., 0], inp["anchor_query"][..., 1] = 256, 1
    inp["anchor_keys"].zero_()
    inp["anchor_keys"][..., 0] = -(row // 256).to(inp["anchor_keys"].dtype)
    inp["anchor_keys"][..., 1] = -(row % 256).to(inp["anchor_keys"].dtype)
    anchor = relation_select_packed_seq(*select_args(inp, cfg))[0]
    blocks, _ = block_route_seq(inp["anchor_router_query"], inp["anchor_block_mean"],
                                inp["anchor_block_std"], inp["anchor_gamma"], inp["anchor_bias"],
                                inp["positions"], 8, 1, 1, strict)
    torch.cuda.synchronize()
    t = inp["positions"].expand(blocks.shape[:2])
    want = torch.where(blocks[..., 0] >= 0, blocks[..., 0] * 8, t.int())
    assert torch.equal(anchor, want.int())
