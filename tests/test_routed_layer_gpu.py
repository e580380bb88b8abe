"""The routed attention layer's operators (torch.ops.rlm.*) together, as a layer runs them: a prompt
and then single tokens, under HIP graphs, torch.compile, other streams, and opcheck's sweep of
schemas, fake kernels and declared mutations."""
from __future__ import annotations

import pytest
import torch

from oracle import routed_layer
from relation_lm.kernels.gated_norm import gated_residual_norm
from relation_lm.kernels.rotary import rotary_positions, rotary_to_caches
from relation_lm.kernels.routed_attention import (block_route, block_route_seq, routed_attention,
                                                  routed_attention_seq)

pytestmark = pytest.mark.gpu
ops = torch.ops.relation_lm

BLOCK, WINDOW, TOP = 16, 24, 3
HEADS, KV_HEADS, DIM, RD = 8, 2, 32, 32        # router: 4 heads of 8
WIDTH = HEADS * DIM


def host(t):
    return t.detach().double().cpu().numpy()


class Layer:
    """Weights and caches of one layer over 128 rows; router keys are a projection of its own."""

    def __init__(self, device, dtype, batch, rows=128, seed=0):
        g = torch.Generator().manual_seed(seed)

        def weight(*shape, scale=1.0):
            return (scale * torch.randn(*shape, generator=g)).to(dtype).to(device)

        self.dtype, self.batch, self.rows = dtype, batch, rows
        parts = (HEADS + 2 * KV_HEADS) * DIM
        self.projection = weight(parts + 2 * RD, WIDTH, scale=WIDTH ** -0.5)
        self.output = weight(WIDTH, WIDTH, scale=WIDTH ** -0.5)
        self.norms = [(1 + weight(WIDTH, scale=0.1)).to(dtype) for _ in range(2)]
        self.bias = weight(WIDTH, scale=0.1)
        self.gate = torch.tensor(0.3, device=device)
        self.gamma = torch.randn(4, generator=g).to(device)
        self.bucket_bias = torch.randn(4, 16, generator=g).to(device)
        self.frequencies = (10000.0 ** (-torch.arange(16) / 16)).float().to(device)
        self.key_cache = torch.full((batch, rows, KV_HEADS, DIM), float("nan"), dtype=dtype,
                                    device=device)
        self.value_cache = self.key_cache.clone()
        self.router_keys = torch.zeros(batch, rows, RD, dtype=dtype, device=device)

    def split(self, normalized):
        rows = ops.relation_linear(normalized, self.projection)
        lead = rows.shape[:-1]
        sizes = (HEADS * DIM, KV_HEADS * DIM, KV_HEADS * DIM, RD, RD)
        q, k, v, router_query, router_key = rows.split(sizes, dim=-1)
        return (q.view(*lead, HEADS, DIM), k.view(*lead, KV_HEADS, DIM),
                v.view(*lead, KV_HEADS, DIM), router_query, router_key)

    def statistics(self):
        mean, std = ops.block_statistics(self.router_keys, BLOCK)
        shape = (self.batch, self.rows // BLOCK, 4, RD // 4)
        return mean.view(shape), std.view(shape)

    def finish(self, attended, hidden):
        branch = ops.relation_linear(attended.flatten(-2), self.output)
        return gated_residual_norm(branch, hidden, self.gate, self.norms[0], self.bias, 1e-5,
                                   self.norms[1], None, 1.0, False)

    def prompt(self, hidden, normalized, lengths=None):
        length = hidden.shape[1]
        start = torch.zeros((), dtype=torch.int64, device=hidden.device)
        q, k, v, router_query, router_key = self.split(normalized)
        self.router_keys[:, :length] = router_key
        q = rotary_to_caches(q, k, v, start, self.frequencies, self.key_cache, self.value_cache,
                             lengths=lengths)
        positions = torch.arange(length, device=hidden.device)
        blocks, _ = block_route_seq(router_query, *self.statistics(), self.gamma, self.bucket_bias,
                                    positions, BLOCK, WINDOW, TOP, True)
        attended, lse = routed_attention_seq(q, self.key_cache, self.value_cache, blocks, positions,
                                             BLOCK, WINDOW)
        return self.finish(attended, hidden) + (q, blocks, attended, lse)

    def token(self, hidden, normalized, position):
        """position [B] on the device; everything stays there."""
        q, k, v, router_query, router_key = self.split(normalized)
        rows = position[:, None, None].expand(-1, 1, RD)
        self.router_keys.scatter_(1, rows, router_key[:, None])
        q = rotary_to_caches(q[:, None], k[:, None], v[:, None], position, self.frequencies,
                             self.key_cache, self.value_cache)
        blocks, _ = block_route(router_query, *self.statistics(), self.gamma, self.bucket_bias,
                                position, BLOCK, WINDOW, TOP, True)
        attended, lse = routed_attention(q[:, 0], self.key_cache, self.value_cache, blocks,
                                         position, BLOCK, WINDOW)
        return self.finish(attended, hidden) + (q[:, 0], blocks, attended, lse)


def inputs(device, dtype, batch, length, seed=1):
    g = torch.Generator().manual_seed(seed)
    hidden = torch.randn(batch, length, WIDTH, generator=g).to(dtype).to(device)
    ones, zeros = torch.ones(WIDTH, device=device), torch.zeros(WIDTH, device=device)
    return hidden, ops.layer_norm(hidden, ones, zeros, 1e-5)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prompt_then_tokens(device, dtype):
    """A prompt's stages against the oracle, each on the GPU's own inputs; then tokens one by one:
    the rows of a prompt that holds them as well."""
    batch, length, more = 2, 101, 20
    hidden, normalized = inputs(device, dtype, batch, length + more)
    layer, whole = Layer(device, dtype, batch), Layer(device, dtype, batch)
    out = layer.prompt(hidden[:, :length], normalized[:, :length])
    q, k, v, router_query, _ = layer.split(normalized[:, :length])
    t = torch.arange(length).numpy()
    freq = layer.frequencies.cpu().numpy()
    turned = routed_layer.rotary(host(k), t, freq, False, 1.0)
    half = torch.finfo(dtype).eps / 2
    # One rounding to the type, and 20 u of a pair's size (tests/test_rotary_gpu.py).
    size = 20 * 2.0 ** -24 * abs(host(k)).max()
    off = abs(host(layer.key_cache)[:, :length] - turned)
    assert (off <= half * abs(turned) + size).all()
    assert torch.equal(layer.value_cache[:, :length], v)
    assert torch.isnan(layer.key_cache[:, length:]).all()
    mean, std = layer.statistics()
    want, _ = routed_layer.block_route(
        host(router_query)[:, :, None], mean.cpu().numpy(), std.cpu().numpy(), host(layer.gamma),
        host(layer.bucket_bias), t, BLOCK, WINDOW, TOP, True)
    blocks = out[3].cpu().numpy()
    assert (blocks == want[:, :, 0]).all()
    keys, values = host(layer.key_cache[:, :length]), host(layer.value_cache[:, :length])
    attended, lse, spread, score = routed_layer.attention(host(out[2]), keys, values,
                                                          blocks[:, :, None], t, BLOCK, WINDOW,
                                                          DIM ** -0.5)
    u = 2.0 ** -24
    relative = (2 * (DIM + 4) + 2) * u * score[..., None] + 300 * u
    relative = relative + (0 if dtype == torch.float32 else half)
    assert (abs(host(out[4]) - attended) <= half * abs(attended) + spread * relative).all()

    reference = whole.prompt(hidden, normalized)
    tight = dict(rtol=1e-5, atol=2e-5) if dtype == torch.float32 else dict(rtol=3e-2, atol=3e-2)
    for i in range(length, length + more):
        position = torch.full((batch,), i, device=device)
        step = layer.token(hidden[:, i], normalized[:, i].contiguous(), position)
        if dtype == torch.float32:      # (bf16 linears of one row and of many round differently)
            assert torch.equal(step[3], reference[3][:, i])
        else:
            continue
        for mine, theirs in zip(step[:2] + step[4:], reference[:2] + reference[4:]):
            torch.testing.assert_close(mine, theirs[:, i], **tight)
    assert torch.isnan(layer.key_cache[:, length + more:]).all()


def test_ragged_prompt(device):
    """Rows past a request's length: the caches stay as they were there, the others' are right."""
    hidden, normalized = inputs(device, torch.float32, 2, 60)
    short, full = Layer(device, torch.float32, 2), Layer(device, torch.float32, 2)
    lengths = torch.tensor([60, 41], device=device)
    a = short.prompt(hidden, normalized, lengths)
    b = full.prompt(hidden, normalized)
    assert torch.isnan(short.key_cache[1, 41:]).all() and torch.isnan(short.value_cache[1, 41:]).all()
    assert torch.equal(short.key_cache[1, :41], full.key_cache[1, :41])
    for mine, theirs in zip(a, b):
        assert torch.equal(mine[0], theirs[0]) and torch.equal(mine[1, :41], theirs[1, :41])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_tokens(device, dtype):
    """A step captured once and replayed at new positions and inputs equals the eager step, with
    eager work and a second captured graph between the replays."""
    batch, length, more = 3, 70, 12
    hidden, normalized = inputs(device, dtype, batch, length + more)
    layers = [Layer(device, dtype, batch) for _ in range(3)]     # two graphs', the eager one's
    for layer in layers:
        layer.prompt(hidden[:, :length], normalized[:, :length])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graphs = []
    for layer in layers[:2]:
        h, n = hidden[:, length].clone(), normalized[:, length].clone()
        position = torch.full((batch,), length, device=device)
        saved = [c.clone() for c in (layer.key_cache, layer.value_cache, layer.router_keys)]
        with torch.cuda.stream(stream):
            layer.token(h, n, position)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                out = layer.token(h, n, position)
        for c, s in zip((layer.key_cache, layer.value_cache, layer.router_keys), saved):
            c.copy_(s)
        graphs.append((graph, h, n, position, out))
    torch.cuda.synchronize()
    for i in range(length, length + more):
        eager = layers[2].token(hidden[:, i], normalized[:, i].contiguous(),
                                torch.full((batch,), i, device=device))
        for (graph, h, n, position, out), layer in zip(graphs, layers):
            h.copy_(hidden[:, i])
            n.copy_(normalized[:, i])
            position.fill_(i)
            graph.replay()
            torch.cuda.synchronize()
            for mine, theirs in zip(out, eager):
                assert torch.equal(mine, theirs)
            same = layers[2].key_cache[:, :i + 1]
            assert torch.equal(layer.key_cache[:, :i + 1], same)


def test_compiled_step(device):
    """torch.compile(fullgraph=True) of a step: fake kernels and the caches' mutation."""
    layer, eager = Layer(device, torch.bfloat16, 2), Layer(device, torch.bfloat16, 2)
    hidden, normalized = inputs(device, torch.bfloat16, 2, 53)
    for x in (layer, eager):
        x.prompt(hidden[:, :50], normalized[:, :50])

    def step(q, k, v, router_query, mean, std, position, key_cache, value_cache, residual):
        turned = rotary_to_caches(q[:, None], k[:, None], v[:, None], position, layer.frequencies,
                                  key_cache, value_cache)
        blocks, _ = block_route(router_query, mean, std, layer.gamma, layer.bucket_bias, position,
                                BLOCK, WINDOW, TOP, True)
        attended, _ = routed_attention(turned[:, 0], key_cache, value_cache, blocks, position,
                                       BLOCK, WINDOW)
        return gated_residual_norm(attended.flatten(-2), residual, layer.gate, layer.norms[0],
                                   None, 1e-5)

    compiled = torch.compile(step, fullgraph=True)
    for i in (50, 51, 52):
        q, k, v, router_query, _ = layer.split(normalized[:, i].contiguous())
        mean, std = layer.statistics()
        position = torch.full((2,), i, device=device)
        a = compiled(q, k, v, router_query, mean, std, position, layer.key_cache,
                     layer.value_cache, hidden[:, i])
        b = step(q, k, v, router_query, mean, std, position, eager.key_cache, eager.value_cache,
                 hidden[:, i])
        torch.cuda.synchronize()
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        assert torch.equal(layer.key_cache[:, :i + 1], eager.key_cache[:, :i + 1])


def op_cases(device):
    g = torch.Generator().manual_seed(3)

    def normal(*shape, dtype=torch.bfloat16):
        return torch.randn(*shape, generator=g).to(dtype).to(device)

    freq = (10000.0 ** (-torch.arange(8) / 8)).float().to(device)
    q, k, v = normal(2, 6, 4, 32), normal(2, 6, 2, 32), normal(2, 6, 2, 32)
    caches = normal(2, 64, 2, 32), normal(2, 64, 2, 32)
    positions = torch.arange(40, 46, device=device)
    position = torch.tensor([40, 50], device=device)
    stats = normal(2, 4, 4, 8, dtype=torch.float32), normal(2, 4, 4, 8, dtype=torch.float32).abs()
    router = normal(4, dtype=torch.float32), normal(4, 16, dtype=torch.float32)
    blocks = torch.randint(0, 4, (2, 6, 2), generator=g).to(torch.int32).to(device)
    ns = torch.ops.rlm
    w = normal(64)
    return [
        ("rotary_positions", ns.rotary_positions.default, (q, k, positions, freq, True, 1.1)),
        ("rotary_to_caches", ns.rotary_to_caches.default,
         (q, k, v, position, freq, *caches, False, 1.0, False, None)),
        ("block_route", ns.block_route.default,
         (normal(2, 32), *stats, *router, position, 16, 24, 3, True, False)),
        ("block_route_seq", ns.block_route_seq.default,
         (normal(2, 6, 3, 32), *stats, *router, positions, 16, 24, 3, False)),
        ("routed_attention", ns.routed_attention.default,
         (q[:, 0].contiguous(), *caches, blocks[:, 0].contiguous(), position, 16, 24, None, True)),
        ("routed_attention_seq", ns.routed_attention_seq.default,
         (q, *caches, blocks, positions, 16, 24, 0.2)),
        ("gated_residual_norm", ns.gated_residual_norm.default,
         (normal(5, 64), normal(5, 64), normal(64), w, w, 1e-5, w, None, 1.5, True, 1e-6)),
    ]


def test_opcheck_every_operator(device):
    cases = op_cases(device)
    registered = {n.split("::")[1] for n in torch._C._dispatch_get_all_op_names()
                  if n.startswith("rlm::")}
    assert registered == {name for name, _, _ in cases}
    for name, op, args in cases:
        print(f"opcheck {name}", flush=True)
        result = torch.library.opcheck(op, args)
        assert all(v == "SUCCESS" for v in result.values()), (name, result)


def test_refusals_raise(device):
    cases = {name: (op, args) for name, op, args in op_cases(device)}
    for name, (op, args) in cases.items():
        with pytest.raises((RuntimeError, NotImplementedError)):      # a tensor on the CPU
            op(args[0], args[1].cpu(), *args[2:])
    op, args = cases["routed_attention"]
    with pytest.raises(RuntimeError, match="blocks"):
        op(*args[:3], args[3].long(), *args[4:])
    with pytest.raises(RuntimeError, match="query"):
        op(args[0][0], *args[1:])
    op, args = cases["block_route"]
    with pytest.raises(RuntimeError, match="top_blocks"):
        op(*args[:8], 0, *args[9:])
    op, args = cases["gated_residual_norm"]
    with pytest.raises(RuntimeError, match="residual"):
        op(args[0], args[1][:4], *args[2:])
    with pytest.raises(RuntimeError, match="gate"):
        op(args[0], args[1], torch.zeros(5, 1, device=device), *args[3:])
    op, args = cases["rotary_positions"]
    with pytest.raises(RuntimeError, match="frequencies"):
        op(*args[:3], args[3].double(), *args[4:])


def test_leading_dims_of_the_norm(device):
    x = torch.randn(2, 3, 4, 5, 16, device=device)
    w = torch.rand(16, device=device)
    gate = torch.randn(2, 3, 4, 5, 16, device=device)
    a = gated_residual_norm(x, x, gate, w, None, 1e-5)
    b = gated_residual_norm(x.reshape(-1, 16), x.reshape(-1, 16), gate.reshape(-1, 16), w, None, 1e-5)
    assert a[0].shape == x.shape
    assert torch.equal(a[0].reshape(-1, 16), b[0]) and torch.equal(a[1].reshape(-1, 16), b[1])
    row = gated_residual_norm(x[0, 0, 0, 0], x[0, 0, 0, 0], gate[0, 0, 0, 0], w, None, 1e-5)
    assert torch.equal(row[0], a[0][0, 0, 0, 0])
    across = x.permute(3, 0, 1, 2, 4)           # no view as rows: copied
    c = gated_residual_norm(across, across, gate.permute(3, 0, 1, 2, 4), w, None, 1e-5)
    assert torch.equal(c[1], a[1].permute(3, 0, 1, 2, 4))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_calls_without_rows(device, dtype):
    """No queries, no batch rows, a cache without rows, no picks: outputs of the right shapes, and
    where there are queries, ones that saw nothing."""
    def some(*shape):
        return torch.randn(*shape, device=device).to(dtype)

    positions = torch.zeros(0, dtype=torch.int64, device=device)
    out, lse = routed_attention_seq(some(2, 0, 4, 32), some(2, 8, 2, 32), some(2, 8, 2, 32),
                                    torch.zeros(2, 0, 3, dtype=torch.int32, device=device),
                                    positions, 4, 4)
    assert out.shape == (2, 0, 4, 32) and lse.shape == (2, 0, 4)
    at = torch.tensor(3, device=device)
    for batch, rows, top in ((0, 8, 3), (2, 0, 3), (2, 0, 0)):
        picks = torch.zeros(batch, top, dtype=torch.int32, device=device)
        out, lse = routed_attention(some(batch, 4, 32), some(batch, rows, 2, 32),
                                    some(batch, rows, 2, 32), picks, at, 4, 4)
        assert (out == 0).all() and torch.isneginf(lse).all() and out.shape == (batch, 4, 32)
    freq = torch.ones(16, device=device)
    q, k = rotary_positions(some(2, 0, 4, 32), some(2, 0, 2, 32), positions, freq)
    assert q.shape == (2, 0, 4, 32) and k.shape == (2, 0, 2, 32)
    cache = some(2, 0, 2, 32)
    query = some(2, 1, 4, 32)
    turned = rotary_to_caches(query, some(2, 1, 2, 32), some(2, 1, 2, 32),
                              torch.tensor(0, device=device), freq, cache, cache.clone())
    assert torch.equal(turned, query)          # position 0, and no cache row to write
    blocks, scores = block_route_seq(some(2, 0, 32), torch.zeros(2, 3, 2, 16, device=device),
                                     torch.zeros(2, 3, 2, 16, device=device),
                                     torch.zeros(2, device=device), torch.zeros(2, 5, device=device),
                                     positions, 4, 4, 2, False)
    assert blocks.shape == scores.shape == (2, 0, 2)
    torch.cuda.synchronize()
