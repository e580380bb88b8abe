"""The operators for 8-bit caches and 4-bit weights (torch.ops.rlm_quantized.*) together, as a layer
runs them: a prompt and then single tokens, under HIP graphs, torch.compile, other streams, and
opcheck's sweep of schemas, fake kernels and declared mutations."""
from __future__ import annotations

import pytest
import torch

from relation_lm.kernels.gated_norm import gated_residual_norm
from relation_lm.kernels.linear_4bit import (gated_linear_4bit, linear_4bit, pack_4bit,
                                             quantize_4bit)
from relation_lm.kernels.quantized_cache import quantized_rows, rotary_to_quantized_caches
from relation_lm.kernels.rotary import rotary_positions
from relation_lm.kernels.routed_attention import (block_route, block_route_seq, routed_attention,
                                                  routed_attention_quantized,
                                                  routed_attention_quantized_seq)

pytestmark = pytest.mark.gpu
ops = torch.ops.relation_lm

BLOCK, WINDOW, TOP = 16, 24, 3
HEADS, KV_HEADS, DIM, RD = 8, 2, 32, 32        # router: 4 heads of 8
WIDTH, INNER, GROUP = HEADS * DIM, 640, 64


class Layer:
    """One layer over 128 rows: attention, then a gated feed-forward block, every weight in 4 bits
    and the caches in 8; router keys are a projection of their own."""

    def __init__(self, device, dtype, batch, rows=128, seed=0):
        g = torch.Generator().manual_seed(seed)

        def weight(n, k):
            w = torch.randn(n, k, generator=g) * k ** -0.5
            codes, scales, zeros = quantize_4bit(w, GROUP)
            return (pack_4bit(codes).to(device), scales.to(dtype).to(device),
                    zeros.to(dtype).to(device))

        self.dtype, self.batch, self.rows = dtype, batch, rows
        self.projection = weight((HEADS + 2 * KV_HEADS) * DIM + 2 * RD, WIDTH)
        self.output = weight(WIDTH, WIDTH)
        self.gate_up = weight(INNER, WIDTH), weight(INNER, WIDTH)
        self.down = weight(WIDTH, INNER)
        self.norms = [(1 + 0.1 * torch.randn(WIDTH, generator=g)).to(dtype).to(device)
                      for _ in range(2)]
        self.gate = torch.tensor(0.3, device=device)
        self.gamma = torch.randn(4, generator=g).to(device)
        self.bucket_bias = torch.randn(4, 16, generator=g).to(device)
        self.frequencies = (10000.0 ** (-torch.arange(16) / 16)).float().to(device)
        self.caches = [torch.full((batch, rows, KV_HEADS, DIM), 0x7f, dtype=torch.uint8,
                                  device=device).view(torch.float8_e4m3fn) for _ in range(2)]
        self.scales = [torch.full((batch, rows, KV_HEADS), float("nan"), device=device)
                       for _ in range(2)]
        self.router_keys = torch.zeros(batch, rows, RD, dtype=dtype, device=device)

    def state(self):
        return [c.view(torch.uint8) for c in self.caches] + self.scales + [self.router_keys]

    def split(self, normalized):
        rows = linear_4bit(normalized, *self.projection, GROUP)
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
        branch = linear_4bit(attended.flatten(-2), *self.output, GROUP)
        hidden, normalized = gated_residual_norm(branch, hidden, self.gate, self.norms[0], None,
                                                 1e-5)
        (gc, gs, gz), (uc, us, uz) = self.gate_up
        inner = gated_linear_4bit(normalized, gc, gs, uc, us, gz, uz, GROUP, "silu")
        return gated_residual_norm(linear_4bit(inner, *self.down, GROUP), hidden, self.gate,
                                   self.norms[1], None, 1e-5)

    def prompt(self, hidden, normalized, lengths=None):
        length = hidden.shape[1]
        start = torch.zeros((), dtype=torch.int64, device=hidden.device)
        q, k, v, router_query, router_key = self.split(normalized)
        self.router_keys[:, :length] = router_key
        q = rotary_to_quantized_caches(q, k, v, start, self.frequencies, *self.caches,
                                       *self.scales, lengths=lengths)
        positions = torch.arange(length, device=hidden.device)
        blocks, _ = block_route_seq(router_query, *self.statistics(), self.gamma, self.bucket_bias,
                                    positions, BLOCK, WINDOW, TOP, True)
        attended, lse = routed_attention_quantized_seq(q, *self.caches, *self.scales, blocks,
                                                       positions, BLOCK, WINDOW)
        return self.finish(attended, hidden) + (q, blocks, attended, lse)

    def token(self, hidden, normalized, position):
        """position [B] on the device; everything stays there."""
        q, k, v, router_query, router_key = self.split(normalized)
        rows = position[:, None, None].expand(-1, 1, RD)
        self.router_keys.scatter_(1, rows, router_key[:, None])
        q = rotary_to_quantized_caches(q[:, None], k[:, None], v[:, None], position,
                                       self.frequencies, *self.caches, *self.scales)
        blocks, _ = block_route(router_query, *self.statistics(), self.gamma, self.bucket_bias,
                                position, BLOCK, WINDOW, TOP, True)
        attended, lse = routed_attention_quantized(q[:, 0], *self.caches, *self.scales, blocks,
                                                   position, BLOCK, WINDOW)
        return self.finish(attended, hidden) + (q[:, 0], blocks, attended, lse)


def inputs(device, dtype, batch, length, seed=1):
    g = torch.Generator().manual_seed(seed)
    hidden = torch.randn(batch, length, WIDTH, generator=g).to(dtype).to(device)
    ones, zeros = torch.ones(WIDTH, device=device), torch.zeros(WIDTH, device=device)
    return hidden, ops.layer_norm(hidden, ones, zeros, 1e-5)


def test_prompt_against_the_16_bit_operators(device):
    """Attention over the 8-bit caches is that of the rows which quantized_rows reads back, to the
    rounding of those rows and weights in bf16; the query turns as rotary_positions turns it."""
    layer = Layer(device, torch.bfloat16, 2)
    hidden, normalized = inputs(device, torch.bfloat16, 2, 101)
    out = layer.prompt(hidden, normalized)
    q, k, _, _, _ = layer.split(normalized)
    positions = torch.arange(101, device=device)
    turned, _ = rotary_positions(q, k, positions, layer.frequencies)
    assert torch.equal(out[2], turned)
    keys, values = [quantized_rows(c, s)[:, :101].contiguous()
                    for c, s in zip(layer.caches, layer.scales)]
    from relation_lm.kernels.routed_attention import routed_attention_seq
    attended, lse = routed_attention_seq(out[2], keys, values, out[3], positions, BLOCK, WINDOW)
    # Keys rounded to bf16 move a score by 2^-8 of its products' size (up to 8 here), so weights by
    # 3%; values and outputs by 2^-8.
    size = values.float().abs().max()
    assert (out[4].float() - attended.float()).abs().max() <= 0.05 * size
    assert (out[5] - lse).abs().max() <= 0.04
    assert torch.isnan(layer.scales[0][:, 101:]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tokens_continue_a_prompt(device, dtype):
    """Tokens one by one write the caches that a prompt holding them writes, to a rounding of its
    products (which sum in another order): nearly every code is the same."""
    batch, length, more = 2, 60, 12
    hidden, normalized = inputs(device, dtype, batch, length + more)
    layer, whole = Layer(device, dtype, batch), Layer(device, dtype, batch)
    layer.prompt(hidden[:, :length], normalized[:, :length])
    reference = whole.prompt(hidden, normalized)
    for i in range(length, length + more):
        position = torch.full((batch,), i, device=device)
        step = layer.token(hidden[:, i], normalized[:, i].contiguous(), position)
        if dtype == torch.float32:
            assert torch.equal(step[3], reference[3][:, i])
            # A code that falls on the other side of a tie moves a row by 2^-4 of one feature.
            assert (step[4] - reference[4][:, i]).abs().max() <= 0.07 * reference[4].abs().max()
    mine, theirs = [torch.stack([quantized_rows(c, s, dtype=torch.float32)[:, :length + more]
                                 for c, s in zip(x.caches, x.scales)]) for x in (layer, whole)]
    limit = 1e-5 if dtype == torch.float32 else 2.0 ** -7
    close = (mine - theirs).abs() <= limit * theirs.abs() + 1e-6
    assert close.float().mean() > (0.9999 if dtype == torch.float32 else 0.9)
    assert ((mine - theirs).abs() <= (2.0 ** -3 + limit) * theirs.abs().amax(-1, True)).all()


def test_ragged_prompt(device):
    """Rows past a request's length: the caches stay as they were there, the others' are right."""
    hidden, normalized = inputs(device, torch.float32, 2, 60)
    short, full = Layer(device, torch.float32, 2), Layer(device, torch.float32, 2)
    lengths = torch.tensor([60, 41], device=device)
    a = short.prompt(hidden, normalized, lengths)
    b = full.prompt(hidden, normalized)
    for s, f in zip(short.state()[:4], full.state()[:4]):
        assert torch.equal(s[1, :41], f[1, :41])
    assert torch.isnan(short.scales[0][1, 41:]).all()
    assert (short.caches[1].view(torch.uint8)[1, 41:] == 0x7f).all()
    for mine, theirs in zip(a, b):
        assert torch.equal(mine[0], theirs[0]) and torch.equal(mine[1, :41], theirs[1, :41])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_tokens(device, dtype):
    """A step captured once and replayed at new positions and inputs equals the eager step, with
    eager work and a second captured graph between the replays."""
    batch, length, more = 3, 70, 8
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
        saved = [c.clone() for c in layer.state()]
        with torch.cuda.stream(stream):
            layer.token(h, n, position)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                out = layer.token(h, n, position)
        for c, s in zip(layer.state(), saved):
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
            for mine, theirs in zip(layer.state(), layers[2].state()):
                assert torch.equal(mine[:, :i + 1], theirs[:, :i + 1])


def test_two_streams_at_once(device):
    """Steps of two layers on two streams give what they give one after the other."""
    hidden, normalized = inputs(device, torch.bfloat16, 2, 40)
    layers = [Layer(device, torch.bfloat16, 2, seed=s) for s in (0, 1, 0, 1)]
    want = [layer.prompt(hidden, normalized) for layer in layers[:2]]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        got = []
        for layer, stream in zip(layers[2:], streams):
            with torch.cuda.stream(stream):
                got.append(layer.prompt(hidden, normalized))
        torch.cuda.synchronize()
        for mine, theirs in zip(got, want):
            assert all(torch.equal(a, b) for a, b in zip(mine, theirs))


def test_compiled_step(device):
    """torch.compile(fullgraph=True) of a step: fake kernels and the caches' mutation."""
    layer, eager = Layer(device, torch.bfloat16, 2), Layer(device, torch.bfloat16, 2)
    hidden, normalized = inputs(device, torch.bfloat16, 2, 53)
    for x in (layer, eager):
        x.prompt(hidden[:, :50], normalized[:, :50])

    def step(q, k, v, blocks, position, kc, vc, ks, vs, residual):
        turned = rotary_to_quantized_caches(q[:, None], k[:, None], v[:, None], position,
                                            layer.frequencies, kc, vc, ks, vs)
        attended, _ = routed_attention_quantized(turned[:, 0], kc, vc, ks, vs, blocks, position,
                                                 BLOCK, WINDOW)
        return layer.finish(attended, residual)

    compiled = torch.compile(step, fullgraph=True)
    for i in (50, 51, 52):
        q, k, v, router_query, _ = layer.split(normalized[:, i].contiguous())
        position = torch.full((2,), i, device=device)
        blocks, _ = block_route(router_query, *layer.statistics(), layer.gamma, layer.bucket_bias,
                                position, BLOCK, WINDOW, TOP, True)
        a = compiled(q, k, v, blocks, position, *layer.caches, *layer.scales, hidden[:, i])
        b = step(q, k, v, blocks, position, *eager.caches, *eager.scales, hidden[:, i])
        torch.cuda.synchronize()
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        for mine, theirs in zip(layer.state()[:4], eager.state()[:4]):
            assert torch.equal(mine[:, :i + 1], theirs[:, :i + 1])


def op_cases(device):
    g = torch.Generator().manual_seed(3)

    def normal(*shape, dtype=torch.bfloat16):
        return torch.randn(*shape, generator=g).to(dtype).to(device)

    freq = (10000.0 ** (-torch.arange(8) / 8)).float().to(device)
    q, k, v = normal(2, 6, 4, 32), normal(2, 6, 2, 32), normal(2, 6, 2, 32)
    caches = [normal(2, 64, 2, 32).to(torch.float8_e4m3fn) for _ in range(2)]
    scales = [normal(2, 64, 2, dtype=torch.float32).abs() for _ in range(2)]
    positions = torch.arange(40, 46, device=device)
    position = torch.tensor([40, 50], device=device)
    blocks = torch.randint(0, 4, (2, 6, 2), generator=g).to(torch.int32).to(device)
    rows = torch.randint(0, 64, (2, 9), generator=g).to(device)
    codes = [pack_4bit(torch.randint(0, 16, (24, 64), generator=g)).to(device) for _ in range(2)]
    s = [normal(2, 24).abs() for _ in range(2)]
    z = [normal(2, 24) for _ in range(2)]
    ns = torch.ops.rlm_quantized
    return [
        ("rotary_to_quantized_caches", ns.rotary_to_quantized_caches.default,
         (q, k, v, position, freq, *caches, *scales, False, 1.0, False, None)),
        ("quantized_rows", ns.quantized_rows.default, (caches[0], scales[0], rows, torch.float16)),
        ("routed_attention_quantized", ns.routed_attention_quantized.default,
         (q[:, 0].contiguous(), *caches, *scales, blocks[:, 0].contiguous(), position, 16, 24, None,
          True)),
        ("routed_attention_quantized_seq", ns.routed_attention_quantized_seq.default,
         (q, *caches, *scales, blocks, positions, 16, 24, 0.2)),
        ("linear_4bit", ns.linear_4bit.default,
         (normal(2, 3, 64), codes[0], s[0], z[0], 32, normal(24))),
        ("gated_linear_4bit", ns.gated_linear_4bit.default,
         (normal(5, 64), codes[0], s[0], codes[1], s[1], None, None, 32, "gelu")),
    ]


def test_opcheck_every_operator(device):
    cases = op_cases(device)
    registered = {n.split("::")[1] for n in torch._C._dispatch_get_all_op_names()
                  if n.startswith("rlm_quantized::")}
    assert registered == {name for name, _, _ in cases}
    for name, op, args in cases:
        print(f"opcheck {name}", flush=True)
        # (opcheck's test of the schema multiplies its inputs, which 8-bit floats do not do: what
        # such operators write is compared here.)
        codes = any(getattr(x, "dtype", None) == torch.float8_e4m3fn for x in args)
        utils = ("test_faketensor",) if codes else ("test_schema", "test_faketensor")
        before = [x.clone() if isinstance(x, torch.Tensor) else x for x in args]
        op(*args)
        torch.cuda.synchronize()
        for i, (x, y) in enumerate(zip(args, before)):
            written = name == "rotary_to_quantized_caches" and 5 <= i <= 8
            if isinstance(x, torch.Tensor):
                assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)) != written, (name, i)
        result = torch.library.opcheck(op, args, test_utils=utils)
        assert all(v == "SUCCESS" for v in result.values()), (name, result)


def test_refusals_raise(device):
    cases = {name: (op, args) for name, op, args in op_cases(device)}
    for name, (op, args) in cases.items():
        with pytest.raises((RuntimeError, NotImplementedError)):      # a tensor on the CPU
            op(args[0], args[1].cpu(), *args[2:])
    op, args = cases["routed_attention_quantized"]
    with pytest.raises(RuntimeError, match="key_cache"):
        op(args[0], args[1].float(), *args[2:])
    with pytest.raises(RuntimeError, match="key_scale"):
        op(*args[:3], args[3][:, :-1], *args[4:])
    op, args = cases["quantized_rows"]
    with pytest.raises(RuntimeError, match="dtype"):
        op(*args[:3], torch.float64)
    with pytest.raises(RuntimeError, match="rows"):
        op(*args[:2], args[2][0], args[3])
    with pytest.raises(RuntimeError, match="cache"):
        op(args[0][0], *args[1:])
    op, args = cases["linear_4bit"]
    with pytest.raises(RuntimeError, match="group_size"):
        op(*args[:4], 48, None)
    with pytest.raises(RuntimeError, match="codes"):
        op(args[0], args[1].view(-1), *args[2:])
    with pytest.raises(RuntimeError, match="scales"):
        op(*args[:2], args[2][0], *args[3:])
    op, args = cases["gated_linear_4bit"]
    with pytest.raises(RuntimeError, match="activation"):
        op(*args[:8], "relu")
    with pytest.raises(RuntimeError, match="both or neither"):
        op(*args[:5], args[2], None, *args[7:])
    # 8-bit caches are no input of the 16-bit operators.
    q, kc = cases["routed_attention_quantized_seq"][1][:2]
    blocks, positions = cases["routed_attention_quantized_seq"][1][5:7]
    with pytest.raises(RuntimeError, match="key_cache"):
        routed_attention(q[:, 0], kc, kc, blocks[:, 0], positions[0], 16, 24)
