"""Operators of a routed attention layer, measured through the public entry points.

Families (a case's ``kind``):

  rotary   rotary positions of query and key; with ``cache``, the key and value rows also go
           into their cache rows (a prompt, or one token of a serving batch)
  route    the block router's scores and its ``top`` picks for each query
  attend   attention over the local window and the picked blocks (one token, or a prompt)
  norm     the norm after a block, its gate, the residual sum and the next block's norm

``listed`` takes its widths from ``relation_lm.workloads`` (d_model 576 and 768 in heads of 64,
block 32 / window 64 / top 4 and block 64 / window 128 / top 8) or generic ones; ``draw`` varies
batch, length, heads, head dims, routing, layout and type around them.

Plain forms are dense or gathered torch operations in 32 bits (angles and router scores, where
near values change the result, in 64).
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

EPS = 1e-5
BUCKETS = 16
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}
_entries = None


def _framework():
    """The framework's entry points (imported only where they are measured)."""
    global _entries
    if _entries is None:
        sys.path.insert(1, os.path.join(os.getcwd(), "relation-lm_amd"))
        from relation_lm.kernels import gated_norm, rotary, routed_attention

        _entries = (rotary, routed_attention, gated_norm)
    return _entries


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # The next token of eight users: a 576-wide model's nine heads of 64 on three key heads,
        # written into a full 512-row cache.  All latency.
        dict(name="rotary_decode_8", kind="rotary", batch=8, queries=1, rows=512, first=511,
             heads=9, kv_heads=3, dim=64, pairs=32, interleaved=False, base=10000.0, stretch=1.0,
             scale=1.0, cache=True, ring=False, ragged=False, dtype="bf16"),
        # A prompt batch of the 768-wide stack, into the caches that its attention reads.
        dict(name="rotary_prompt_4096", kind="rotary", batch=4, queries=4096, rows=4096, first=0,
             heads=12, kv_heads=4, dim=64, pairs=32, interleaved=False, base=10000.0, stretch=1.0,
             scale=1.0, cache=True, ring=False, ragged=True, dtype="bf16"),
        # A chunk deep in a long document: interleaved pairs over three quarters of the head,
        # frequencies stretched eightfold, odd length, fp32.
        dict(name="rotary_far_1999_fp32", kind="rotary", batch=2, queries=1999, rows=0,
             first=250000, heads=8, kv_heads=8, dim=64, pairs=24, interleaved=True, base=500000.0,
             stretch=8.0, scale=1.1, cache=False, ring=False, ragged=False, dtype="fp32"),
        # Where a serving batch's next tokens look: 16 blocks of 32, four picks.
        dict(name="route_decode_8", kind="route", batch=8, queries=1, rows=512, first=511, slots=1,
             heads=4, head_dim=16, block=32, local=64, top=4, strict=False, ring=False,
             ragged=False, dtype="bf16"),
        # Every query of a prompt batch over 64 blocks, eight picks.
        dict(name="route_prompt_4096", kind="route", batch=4, queries=4096, rows=4096, first=0,
             slots=1, heads=4, head_dim=16, block=64, local=128, top=8, strict=False, ring=False,
             ragged=False, dtype="bf16"),
        # The attention of the first case's step: the smallest call.
        dict(name="attend_decode_8", kind="attend", batch=8, queries=1, rows=512, first=511,
             heads=9, kv_heads=3, dim=64, block=32, local=64, top=4, slots=1, strict=False,
             ring=False, ragged=False, dtype="bf16"),
        # A serving batch over caches of 131072 rows (past 4 GiB), each request at a length of its
        # own, eight query heads to a key head, 16 blocks and a window of 512.
        dict(name="attend_decode_131072", kind="attend", batch=20, queries=1, rows=131072,
             first=131071, heads=32, kv_heads=4, dim=128, block=64, local=512, top=16, slots=4,
             strict=True, ring=False, ragged=True, dtype="fp16"),
        # A prompt batch of the 768-wide stack, 64 blocks, eight picks and a window of 128.
        dict(name="attend_prompt_4096", kind="attend", batch=4, queries=4096, rows=4096, first=0,
             heads=12, kv_heads=4, dim=64, block=64, local=128, top=8, slots=1, strict=False,
             ring=False, ragged=False, dtype="bf16"),
        # A later chunk of a short prompt, small blocks, every head with keys of its own, fp32.
        dict(name="attend_chunk_333_fp32", kind="attend", batch=2, queries=333, rows=1008,
             first=667, heads=8, kv_heads=8, dim=32, block=16, local=32, top=8, slots=1,
             strict=False, ring=False, ragged=False, dtype="fp32"),
        # One long document, eight query heads to a key head that picks for itself.
        dict(name="attend_prompt_8192", kind="attend", batch=1, queries=8192, rows=8192, first=0,
             heads=16, kv_heads=2, dim=128, block=64, local=256, top=8, slots=2, strict=True,
             ring=False, ragged=False, dtype="bf16"),
        # Between two blocks of a decode step.
        dict(name="norm_decode_8", kind="norm", rows=8, width=576, post=True, gate="one",
             residual_scale=1.0, rms=False, bias=True, dtype="bf16"),
        # Between two blocks of a prompt batch of the 768-wide stack.
        dict(name="norm_prompt_16384", kind="norm", rows=16384, width=768, post=True, gate="one",
             residual_scale=1.0, rms=False, bias=True, dtype="bf16"),
    ]


def _spread(rng, low, high):
    """A whole number, uniform in its logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))) - 0.5)))


def draw(rng):
    kind = rng.choice(["rotary", "route", "attend", "attend", "norm"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind == "norm":
        width = rng.choice([rng.choice([256, 512, 576, 768, 1024, 2048, 4096]),
                            _spread(rng, 33, 5000)])
        return dict(kind="norm", rows=_spread(rng, 1, 10_000_000 // width), width=width,
                    post=rng.random() < 0.6, gate=rng.choice(["one", "columns", "rows"]),
                    residual_scale=rng.choice([1.0, round(rng.uniform(0.5, 2.5), 3)]),
                    rms=rng.random() < 0.5, bias=rng.random() < 0.5, dtype=dtype)
    single = rng.random() < 0.4
    ring = single and rng.random() < 0.3
    block = rng.choice([8, 16, 32, 64])
    if kind == "rotary":
        kv_heads = rng.choice([1, 2, 3, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 3, 4, 8])
        dim = rng.choice([32, 64, 64, 96, 128, 128, 256])
        batch = _spread(rng, 1, 48 if single else 4)
        queries = 1 if single else _spread(rng, 2, max(2, 3_000_000 // (batch * heads * dim)))
        cache = single or rng.random() < 0.5
        if ring:
            rows = 2 ** rng.randint(8, 11)
            first = _spread(rng, 1, 200000)
        else:
            first = _spread(rng, 1, 3000 if cache else 300000)
            rows = first + queries + rng.randint(0, 40) if cache else 0
        return dict(kind="rotary", batch=batch, queries=queries, rows=rows, first=first,
                    heads=heads, kv_heads=kv_heads, dim=dim,
                    pairs=rng.choice([dim // 2, dim // 2, dim // 4, rng.randint(1, dim // 2)]),
                    interleaved=rng.random() < 0.5, base=rng.choice([10000.0, 500000.0]),
                    stretch=rng.choice([1.0, 1.0, 4.0, 32.0]),
                    scale=rng.choice([1.0, round(rng.uniform(1.0, 1.4), 3)]), cache=cache,
                    ring=ring and cache, ragged=rng.random() < 0.5, dtype=dtype)
    if kind == "route":
        batch = _spread(rng, 1, 40 if single else 6)
        # Positions far enough in for a whole block before the window.
        if ring:
            rows = 2 ** rng.randint(10, 14)
            queries, first = 1, _spread(rng, rows // 2, 200000)
        else:
            rows = block * _spread(rng, 12, 500)
            queries = 1 if single else min(rows // 2, _spread(rng, 2, 6000 // batch))
            first = rng.randint(rows // 2, rows - queries)
        local = min(rng.choice([block, 2 * block, 128, rng.randint(1, 300)]), rows // 32)
        return dict(kind="route", batch=batch, queries=queries, rows=rows, first=first,
                    slots=rng.choice([1, 1, 2, 4]), heads=rng.choice([1, 2, 4, 8]),
                    head_dim=rng.choice([8, 16, 32]), block=block,
                    local=max(1, local), top=rng.randint(1, 16), strict=rng.random() < 0.5,
                    ring=ring, ragged=rng.random() < 0.4, dtype=dtype)
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 6, 8, 16])
    dim = rng.choice([32, 64, 64, 80, 96, 128, 128, 256])
    if single:
        batch = _spread(rng, 1, 48)
        rows = 2 ** rng.randint(8, 13) if ring else block * _spread(rng, 2, 1500)
        queries, first = 1, _spread(rng, 1, 100000) if ring else rng.randint(0, rows - 1)
    else:
        batch = _spread(rng, 1, 3)
        longest = 3000 if heads * dim <= 1024 else 1500
        rows = block * max(2, _spread(rng, 64, longest) // block)
        queries = min(rows, _spread(rng, 2, rows))
        first = rng.randint(0, rows - queries)
    return dict(kind="attend", batch=batch, queries=queries, rows=rows, first=first, heads=heads,
                kv_heads=kv_heads, dim=dim, block=block,
                local=rng.choice([block, 2 * block, 128, rng.randint(1, 300)]),
                top=rng.randint(1, 16), slots=rng.choice([1, kv_heads]),
                strict=rng.random() < 0.5, ring=ring, ragged=rng.random() < 0.4, dtype=dtype)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _positions(case, gen):
    """One position per query, [B, Tq].  Ragged: requests of different lengths -- a single token at
    a position of its own, a prompt with its last rows empty (position -1)."""
    b, tq, first = case["batch"], case["queries"], case["first"]
    steps = torch.arange(tq, device="cuda")
    if not case["ragged"]:
        return (first + steps).expand(b, tq).contiguous()
    share = 0.25 + 0.75 * torch.rand(b, 1, generator=gen, device="cuda", dtype=torch.float64)
    if tq == 1:
        return (first * share).long()
    return torch.where(steps < (tq * share).long().clamp_min(1), first + steps, -1)


def _likeness(gen, *shape):
    """Standard normal values over [B, S, Tq, ...] of which half the variance is common to 64
    neighbouring queries: neighbouring tokens of a text ask alike."""
    b, s, tq, n = shape
    common = torch.randn(b, s, -(-tq // 64), n, generator=gen, device="cuda")
    own_part = torch.randn(b, s, tq, n, generator=gen, device="cuda")
    return (common.repeat_interleave(64, 2)[:, :, :tq] + own_part) * 0.5 ** 0.5


def _held(t, count, block, ring):
    """Absolute block that slot j of `count` holds at position t: [..., count]."""
    slot = torch.arange(count, device="cuda")
    if not ring:
        return slot.expand(t.shape + (count,))
    now = torch.div(t, block, rounding_mode="floor")[..., None]
    return now - (now - slot) % count


def _eligible(t, held, case):
    end = (held + 1) * case["block"] - 1
    ok = (held >= 0) & (end <= t[..., None])
    if case["strict"]:
        ok &= end < (t[..., None] - case["local"] + 1).clamp_min(0)
    return ok


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(1 + seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, kind=dtype):
        return torch.randn(shape, generator=gen, device="cuda", dtype=kind)

    state = {"case": case}
    if case["kind"] == "norm":
        n, d = case["rows"], case["width"]
        shape = {"one": (), "columns": (d,), "rows": (n, d)}[case["gate"]]
        state.update(branch=normal(n, d), residual=2 * normal(n, d),
                     gate=(normal(*shape, kind=torch.float32) - 0.5).to(dtype),
                     weight=(1 + 0.1 * normal(d, kind=torch.float32)).to(dtype),
                     bias=(0.1 * normal(d, kind=torch.float32)).to(dtype) if case["bias"] else None,
                     post_weight=None, post_bias=None)
        if case["post"]:
            state["post_weight"] = (1 + 0.1 * normal(d, kind=torch.float32)).to(dtype)
            if case["bias"]:
                state["post_bias"] = (0.1 * normal(d, kind=torch.float32)).to(dtype)
        return state
    b, tq = case["batch"], case["queries"]
    positions = _positions(case, gen)
    state["positions"] = positions
    if case["kind"] == "rotary":
        hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
        # Query, key and value as the layer's one projection leaves them: views of its rows.
        rows = normal(b, tq, (hq + 2 * hk) * d)
        state["query"] = rows[..., :hq * d].view(b, tq, hq, d)
        state["key"] = rows[..., hq * d:(hq + hk) * d].view(b, tq, hk, d)
        state["value"] = rows[..., (hq + hk) * d:].view(b, tq, hk, d)
        pairs = torch.arange(case["pairs"], device="cuda", dtype=torch.float64) / case["pairs"]
        state["frequencies"] = (case["base"] ** -pairs / case["stretch"]).float()
        if case["cache"]:
            state["key_cache"] = normal(b, case["rows"], hk, d)
            state["value_cache"] = normal(b, case["rows"], hk, d)
            # Tokens follow each other from a row's first position; lengths[b] of them are real.
            state["position"] = (positions[:, 0] if case["ragged"] and tq == 1
                                 else torch.tensor(case["first"], device="cuda"))
            state["lengths"] = ((positions >= 0).sum(1) if case["ragged"] and tq > 1 else None)
        return state
    blocks = case["rows"] // case["block"]
    if case["kind"] == "route":
        s, h, hd = case["slots"], case["heads"], case["head_dim"]
        query = _likeness(gen, b, s, tq, h * hd).transpose(1, 2).to(dtype).contiguous()
        state["router_query"] = query if s > 1 else query[:, :, 0]
        # Block statistics of router keys that drift: means apart from each other, spread about 1.
        state["mean"] = 0.5 * normal(b, blocks, h, hd, kind=torch.float32)
        state["std"] = 0.5 + torch.rand(b, blocks, h, hd, generator=gen, device="cuda")
        state["gamma"] = normal(h, kind=torch.float32)
        state["bias"] = normal(h, BUCKETS, kind=torch.float32)
        return state
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    state["query"] = normal(b, tq, hq, d)
    state["key_cache"] = normal(b, case["rows"], hk, d)
    state["value_cache"] = normal(b, case["rows"], hk, d)
    # A router's picks: best first, -1 where a query has fewer blocks to pick from.
    t = positions[:, None].expand(b, case["slots"], tq)
    held = _held(t, blocks, case["block"], case["ring"])
    liking = _likeness(gen, b, case["slots"], tq, blocks)
    liking = liking.masked_fill(~_eligible(t, held, case), -math.inf)
    best = liking.topk(min(case["top"], blocks), dim=-1)
    picks = torch.where(best.values > -math.inf, held.gather(-1, best.indices), -1)
    if case["top"] > blocks:
        picks = torch.nn.functional.pad(picks, (0, case["top"] - blocks), value=-1)
    picks = picks.transpose(1, 2).to(torch.int32)
    state["blocks"] = (picks if case["slots"] > 1 else picks[:, :, 0]).contiguous()
    return state


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------

def _turned(x, angle, case):
    """Rotates the first 2 * pairs features of x [B, Tq, H, D] by angle [B, Tq, pairs]."""
    n = case["pairs"]
    x = x.float()
    cos = (angle.cos() * case["scale"]).float()[:, :, None]
    sin = (angle.sin() * case["scale"]).float()[:, :, None]
    head, rest = x[..., :2 * n], x[..., 2 * n:]
    if case["interleaved"]:
        a, b = head[..., 0::2], head[..., 1::2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = head[..., :n], head[..., n:]
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((turned, rest), -1)


def _plain_rotary(state):
    case, dtype = state["case"], DTYPES[state["case"]["dtype"]]
    b, tq = case["batch"], case["queries"]
    if not case["cache"]:
        angle = state["positions"].double()[..., None] * state["frequencies"].double()
        return {"query": _turned(state["query"], angle, case).to(dtype),
                "key": _turned(state["key"], angle, case).to(dtype)}
    steps = torch.arange(tq, device="cuda")
    t = (state["position"].reshape(-1, 1) + steps).expand(b, tq)
    angle = t.double()[..., None] * state["frequencies"].double()
    key_cache, value_cache = state["key_cache"], state["value_cache"]
    key = _turned(state["key"], angle, case).to(dtype)
    real = (torch.ones_like(t, dtype=torch.bool) if state["lengths"] is None
            else steps < state["lengths"][:, None])
    row = t % case["rows"] if case["ring"] else t
    batch, token = real.nonzero(as_tuple=True)
    key_cache[batch, row[batch, token]] = key[batch, token]
    value_cache[batch, row[batch, token]] = state["value"][batch, token]
    return {"query": _turned(state["query"], angle, case).to(dtype), "key_cache": key_cache,
            "value_cache": value_cache}


def _plain_route(state):
    case = state["case"]
    b, tq, s, h, hd = (case[k] for k in ("batch", "queries", "slots", "heads", "head_dim"))
    blocks = case["rows"] // case["block"]
    t = state["positions"]
    held = _held(t, blocks, case["block"], case["ring"])                        # [B, Tq, NB]
    q = state["router_query"].double().view(b, tq * s, h, hd).transpose(1, 2)   # [B, H, Tq*S, HD]
    mean = state["mean"].double().permute(0, 2, 3, 1).contiguous()              # [B, H, HD, NB]
    std = state["std"].double().permute(0, 2, 3, 1).contiguous()
    spread = (1 + state["gamma"].double().exp()).log()[:, None, None]
    score = (torch.matmul(q.contiguous(), mean)
             + spread * torch.matmul(q.abs().contiguous(), std)) * hd ** -0.5
    away = (t[..., None] - ((held + 1) * case["block"] - 1)).clamp_min(0) + 1
    bucket = (torch.frexp(away.double()).exponent.long() - 1).clamp_max(BUCKETS - 1)
    score = score.view(b, h, tq, s, blocks) + state["bias"].double()[:, bucket].transpose(0, 1)[
        :, :, :, None]
    most = score.amax(1, keepdim=True)
    score = (most[:, 0] + (score - most).exp().sum(1).log()).float()            # [B, Tq, S, NB]
    score = score.masked_fill(~_eligible(t, held, case)[:, :, None], -math.inf)
    if case["ring"]:    # lowest absolute block first among equals
        order = held.argsort(-1)
        held = held.gather(-1, order)
        score = score.gather(-1, order[:, :, None].expand_as(score))
    value, index = score.sort(dim=-1, descending=True, stable=True)
    value, index = value[..., :case["top"]], index[..., :case["top"]]
    pick = held[:, :, None].expand_as(score).gather(-1, index)
    pick = torch.where(value > -math.inf, pick, -1)
    if case["top"] > blocks:
        pad = (0, case["top"] - blocks)
        pick = torch.nn.functional.pad(pick, pad, value=-1)
        value = torch.nn.functional.pad(value, pad, value=-math.inf)
    if s == 1:
        pick, value = pick[:, :, 0], value[:, :, 0]
    return {"blocks": pick.to(torch.int32), "scores": value}


def _weighted(score, value):
    """softmax(score) . value over the last axis of score; an empty row gives 0 and lse -inf."""
    most = score.amax(-1, keepdim=True)
    weight = (score - most.clamp_min(-3e38)).exp_()
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight, value) / total.where(total > 0, 1.0)
    return out, (most + total.log())[..., 0]


def _plain_attend(state):
    case, dtype = state["case"], DTYPES[state["case"]["dtype"]]
    b, tq, hq, hk, d = (case[k] for k in ("batch", "queries", "heads", "kv_heads", "dim"))
    g, block, rows, s = hq // hk, case["block"], case["rows"], case["slots"]
    t = state["positions"][:, None]                                             # [B, 1, Tq]
    start = (t - case["local"] + 1).clamp_min(0)
    picks = state["blocks"].long().view(b, tq, s, case["top"]).transpose(1, 2)  # [B, S, Tq, TOP]
    query = state["query"].float().view(b, tq, hk, g, d).transpose(1, 2)        # [B, HK, Tq, G, D]
    query = query * d ** -0.5
    key, value = (state[k].permute(0, 2, 1, 3) for k in ("key_cache", "value_cache"))
    if tq == 1:
        # Gathered: the window's rows, then the picked blocks' rows before the window.
        p = (picks[..., None] * block + torch.arange(block, device="cuda")).flatten(-2)
        ok = (picks >= 0).repeat_interleave(block, -1) & (p < start[..., None])
        near = (start[..., None] + torch.arange(case["local"], device="cuda")).expand(b, s, 1, -1)
        p, ok = torch.cat((near, p), -1), torch.cat((torch.ones_like(near, dtype=torch.bool), ok),
                                                    -1)
        ok = ok & (p <= t[..., None])
        if case["ring"]:
            ok, row = ok & (p > t[..., None] - rows), p % rows
        else:
            ok, row = ok & (p < rows), p
        row = torch.where(ok, row, 0).expand(b, hk, 1, -1)[:, :, 0]             # [B, HK, C]
        at = (torch.arange(b, device="cuda")[:, None, None],
              torch.arange(hk, device="cuda")[:, None], row)
        score = torch.matmul(query[:, :, 0], key[at].float().transpose(-1, -2).contiguous())
        score = score.masked_fill(~ok, -math.inf)
        out, lse = _weighted(score, value[at].float())
        return {"out": out.reshape(b, 1, hq, d).to(dtype), "lse": lse.reshape(b, 1, hq)}
    count = rows // block
    chosen = torch.zeros(b, s, tq, count + 1, dtype=torch.bool, device="cuda")
    chosen = chosen.scatter_(-1, picks.where(picks >= 0, count), True)[..., :count]
    p = torch.arange(rows, device="cuda")
    ok = (chosen.repeat_interleave(block, -1) | (p >= start[..., None])) & (p <= t[..., None])
    score = torch.matmul(query.reshape(b, hk, tq * g, d),
                         key.float().transpose(-1, -2).contiguous()).view(b, hk, tq, g, rows)
    score.masked_fill_(~ok[:, :, :, None], -math.inf)
    out, lse = _weighted(score.view(b, hk, tq * g, rows), value.float().contiguous())
    out = out.view(b, hk, tq, g, d).transpose(1, 2).reshape(b, tq, hq, d)
    return {"out": out.to(dtype), "lse": lse.view(b, hk, tq, g).transpose(1, 2).reshape(b, tq, hq)}


def _plain_normed(x, weight, bias, rms):
    if not rms:
        x = x - x.mean(-1, keepdim=True)
    x = x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt() * weight.float()
    return x if bias is None else x + bias.float()


def _plain_norm(state):
    case, dtype = state["case"], DTYPES[state["case"]["dtype"]]
    branch = state["branch"].float()
    if case["post"]:
        branch = _plain_normed(branch, state["post_weight"], state["post_bias"], case["rms"])
    gate = 1 / (1 + (-state["gate"].float()).exp())
    hidden = case["residual_scale"] * state["residual"].float() + gate * branch
    return {"hidden": hidden.to(dtype),
            "normalized": _plain_normed(hidden, state["weight"], state["bias"],
                                        case["rms"]).to(dtype)}


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

def _own_rotary(state):
    rotary, case = _framework()[0], state["case"]
    if not case["cache"]:
        query, key = rotary.rotary_positions(state["query"], state["key"], state["positions"],
                                             state["frequencies"], case["interleaved"],
                                             case["scale"])
        return {"query": query, "key": key}
    query = rotary.rotary_to_caches(state["query"], state["key"], state["value"],
                                    state["position"], state["frequencies"], state["key_cache"],
                                    state["value_cache"], case["interleaved"], case["scale"],
                                    case["ring"], state["lengths"])
    return {"query": query, "key_cache": state["key_cache"], "value_cache": state["value_cache"]}


def _own_route(state):
    attention, case = _framework()[1], state["case"]
    if case["queries"] == 1:
        blocks, scores = attention.block_route(
            state["router_query"][:, 0], state["mean"], state["std"], state["gamma"],
            state["bias"], state["positions"][:, 0], case["block"], case["local"], case["top"],
            case["strict"], case["ring"])
        return {"blocks": blocks[:, None], "scores": scores[:, None]}
    blocks, scores = attention.block_route_seq(
        state["router_query"], state["mean"], state["std"], state["gamma"], state["bias"],
        state["positions"], case["block"], case["local"], case["top"], case["strict"])
    return {"blocks": blocks, "scores": scores}


def _own_attend(state):
    attention, case = _framework()[1], state["case"]
    if case["queries"] == 1:
        out, lse = attention.routed_attention(
            state["query"][:, 0], state["key_cache"], state["value_cache"], state["blocks"][:, 0],
            state["positions"][:, 0], case["block"], case["local"], None, case["ring"])
        return {"out": out[:, None], "lse": lse[:, None]}
    out, lse = attention.routed_attention_seq(
        state["query"], state["key_cache"], state["value_cache"], state["blocks"],
        state["positions"], case["block"], case["local"])
    return {"out": out, "lse": lse}


def _own_norm(state):
    gated_norm, case = _framework()[2], state["case"]
    hidden, normalized = gated_norm.gated_residual_norm(
        state["branch"], state["residual"], state["gate"], state["weight"], state["bias"], EPS,
        state["post_weight"], state["post_bias"], case["residual_scale"], case["rms"])
    return {"hidden": hidden, "normalized": normalized}


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"rotary": _own_rotary, "route": _own_route, "attend": _own_attend,
                "norm": _own_norm}[kind](state)
    return {"rotary": _plain_rotary, "route": _plain_route, "attend": _plain_attend,
            "norm": _plain_norm}[kind](state)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------

def _reach(case):
    """Keys that the queries of a case attend to, in all (every request taken at full length)."""
    total = 0
    for i in range(case["queries"]):
        t = case["first"] + i
        if case["ring"]:
            far, seen = case["rows"] - case["local"], min(t + 1, case["rows"])
        else:
            far, seen = case["rows"], min(t + 1, case["rows"])
        near = min(seen, case["local"])
        total += near + min(max(0, min(far, seen - near)), case["top"] * case["block"])
    return case["batch"] * total


def work(case):
    size = SIZES[case["dtype"]]
    if case["kind"] == "norm":
        n, d = case["rows"], case["width"]
        gates = {"one": 1, "columns": d, "rows": n * d}[case["gate"]]
        return {"bytes": size * (4 * n * d + gates + 4 * d), "flops": 20 * n * d}
    tokens = case["batch"] * case["queries"]
    if case["kind"] == "rotary":
        hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
        moved = 2 * tokens * (hq + (2 if case["cache"] else 1) * hk) * d * size
        return {"bytes": moved, "flops": 6 * tokens * (hq + hk) * case["pairs"]}
    blocks = case["rows"] // case["block"]
    if case["kind"] == "route":
        width = case["heads"] * case["head_dim"]
        asked = tokens * case["slots"]
        return {"bytes": asked * (width * size + 8 * case["top"])
                + 8 * case["batch"] * blocks * width,
                "flops": 4 * asked * blocks * width}
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    keys = _reach(case)
    read = min(keys, case["batch"] * min(case["rows"], case["first"] + case["queries"]))
    return {"bytes": 2 * tokens * hq * d * size + 4 * tokens * hq + 2 * read * hk * d * size
            + 4 * tokens * case["slots"] * case["top"],
            "flops": 4 * keys * hq * d}


# ---------------------------------------------------------------------------
# From the definition, in 64 bits
# ---------------------------------------------------------------------------

def _exact_rotary(state, case):
    b, tq, n = case["batch"], case["queries"], case["pairs"]
    if case["cache"]:
        t = (state["position"].reshape(-1, 1)
             + torch.arange(tq, device="cuda")).expand(b, tq).double()
    else:
        t = state["positions"].double()
    turn = torch.polar(torch.full((), case["scale"], dtype=torch.float64, device="cuda").expand(
        b, tq, n), t[..., None] * state["frequencies"].double())[:, :, None]

    def rotated(x):
        y = x.double().clone()
        one = slice(0, 2 * n, 2) if case["interleaved"] else slice(0, n)
        two = slice(1, 2 * n, 2) if case["interleaved"] else slice(n, 2 * n)
        z = torch.complex(y[..., one], y[..., two]) * turn
        y[..., one], y[..., two] = z.real, z.imag
        return y

    if not case["cache"]:
        return {"query": rotated(state["query"]), "key": rotated(state["key"])}
    caches = state["key_cache"].double(), state["value_cache"].double()
    keys = rotated(state["key"])
    for i in range(b):
        many = tq if state["lengths"] is None else int(state["lengths"][i])
        row = t[i, :many].long()
        row = row % case["rows"] if case["ring"] else row
        caches[0][i].index_copy_(0, row, keys[i, :many])
        caches[1][i].index_copy_(0, row, state["value"][i, :many].double())
    return {"query": rotated(state["query"]), "key_cache": caches[0], "value_cache": caches[1]}


def _exact_attend(state, case):
    b, tq, hq, hk, d = (case[k] for k in ("batch", "queries", "heads", "kv_heads", "dim"))
    g, rows, block, s = hq // hk, case["rows"], case["block"], case["slots"]
    out = torch.zeros(b, tq, hq, d, dtype=torch.float64, device="cuda")
    lse = torch.zeros(b, tq, hq, dtype=torch.float64, device="cuda")
    row = torch.arange(rows, device="cuda")
    picks = state["blocks"].long().view(b, tq, s, -1)
    for i in range(b):
        for low in range(0, tq, 1024):
            t = state["positions"][i, low:low + 1024, None]
            # The position that each row of the cache holds.
            p = t - (t - row) % rows if case["ring"] else row.expand(len(t), rows)
            seen = (p >= 0) & (p <= t)
            for h in range(hk):
                mine = picks[i, low:low + 1024, h if s > 1 else 0]
                near = p > t - case["local"]
                # Blocks by their remainder: a cache holds one block of each.
                mark = torch.zeros(len(t), rows // block + 1, dtype=torch.int64, device="cuda")
                mark.scatter_(1, torch.where(mine < 0, rows // block, mine % (rows // block)),
                              mine + 1)
                whose = (p // block) if not case["ring"] else torch.where(p >= 0, p // block, -1)
                picked = mark.gather(1, torch.where(whose < 0, rows // block,
                                                    whose % (rows // block))) == whose + 1
                ok = seen & (near | (picked & (whose >= 0)))
                q = state["query"][i, low:low + 1024, h * g:(h + 1) * g].double()
                a = torch.matmul(q, state["key_cache"][i, :, h].double().T.contiguous())
                a = (a / math.sqrt(d)).masked_fill(~ok[:, None], -math.inf)
                z = torch.logsumexp(a, -1)
                w = (a - z.clamp_min(-1e300)[..., None]).exp()
                out[i, low:low + 1024, h * g:(h + 1) * g] = torch.matmul(
                    w, state["value_cache"][i, :, h].double())
                lse[i, low:low + 1024, h * g:(h + 1) * g] = z
    return {"out": out, "lse": lse}


def _exact_route(state, case):
    """Scores of the picks alone: which blocks they are is compared with the plain form's."""
    b, tq, s, h, hd = (case[k] for k in ("batch", "queries", "slots", "heads", "head_dim"))
    blocks = case["rows"] // case["block"]
    q = state["router_query"].double().view(b, tq, s, h, hd)
    score = torch.empty(b, tq, s, blocks, dtype=torch.float64, device="cuda")
    slot = torch.arange(blocks, device="cuda")
    powers = 2 ** torch.arange(1, BUCKETS, device="cuda")
    for i in range(b):
        t = state["positions"][i, :, None]
        held = slot.expand(tq, blocks)
        if case["ring"]:
            held = t // case["block"] - (t // case["block"] - slot) % blocks
        last = held * case["block"] + case["block"] - 1
        # floor(log2(n)) of a whole n >= 1 is the number of powers 2, 4, 8, ... up to n.
        bucket = ((t - last).clamp_min(0)[..., None] + 1 >= powers).sum(-1)
        heads = []
        for k in range(h):
            like = q[i, :, :, k] @ state["mean"][i, :, k].double().T.contiguous()
            wide = q[i, :, :, k].abs() @ state["std"][i, :, k].double().T.contiguous()
            heads.append((like + torch.nn.functional.softplus(
                state["gamma"][k].double(), threshold=1e9) * wide) / math.sqrt(hd)
                + state["bias"][k].double()[bucket][:, None])
        all_heads = torch.logsumexp(torch.stack(heads), 0)
        free = (held >= 0) & (last <= t)
        if case["strict"]:
            free &= last < (t - case["local"] + 1).clamp_min(0)
        score[i] = all_heads.masked_fill(~free[:, None], -math.inf)
    value = score.topk(min(case["top"], blocks), dim=-1).values
    if case["top"] > blocks:
        value = torch.nn.functional.pad(value, (0, case["top"] - blocks), value=-math.inf)
    return {"blocks": None, "scores": value if s > 1 else value[:, :, 0]}


def _exact_norm(state, case):
    def normed(x, weight, bias):
        if not case["rms"]:
            x = x - x.mean(-1, keepdim=True)
        x = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * weight.double()
        return x if bias is None else x + bias.double()

    y = state["branch"].double()
    if case["post"]:
        y = normed(y, state["post_weight"], state["post_bias"])
    hidden = case["residual_scale"] * state["residual"].double() + y * torch.sigmoid(
        state["gate"].double())
    return {"hidden": hidden, "normalized": normed(hidden, state["weight"], state["bias"])}


def exact(case, seed):
    state = prepare(case, seed)
    return {"rotary": _exact_rotary, "route": _exact_route, "attend": _exact_attend,
            "norm": _exact_norm}[case["kind"]](state, case)
