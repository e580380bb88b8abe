"""GPU parity of the gated residual norm (rlm::gated_residual_norm) against
oracle/routed_layer.py in float64.

Tolerance (u = 2^-24, h = half a step of the output's type).  post: the centred values are off
by (D' + 2) u of the row's largest value, D' = 64 adds in sequence at most plus 8 of the tree;
1 / sqrt(var + eps) by 80 u relative; so post(branch) by P = 200 u (|post| + |w| amplitude),
amplitude = largest |x - mean| / sqrt(var + eps).  sigmoid: 6 u.  hidden: P plus 4 u of its
terms.  normalized: the same steps again over hidden, whose own error enters with 1 / sqrt(var).
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import routed_layer
from relation_lm.kernels.gated_norm import gated_residual_norm

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def host(t):
    return None if t is None else t.detach().double().cpu().numpy()


def check(got, branch, residual, gate, weight, bias, eps, post_weight, post_bias, scale, rms,
          post_eps, dtype):
    d = branch.shape[-1]
    args = [host(x) for x in (branch, residual, gate, weight, bias)]
    x, r = args[0].reshape(-1, d), args[1].reshape(-1, d)
    gate = args[2].reshape(-1, d) if args[2].ndim > 1 else args[2]
    pw, pb = host(post_weight), host(post_bias)
    hidden, normalized = routed_layer.gated_residual_norm(x, r, gate, args[3], args[4], eps, pw, pb,
                                                          scale, rms, post_eps)
    def inverse(y, e):
        y = y if rms else y - y.mean(-1, keepdims=True)
        return 1 / np.sqrt((y * y).mean(-1, keepdims=True) + e)

    y, off = x, 0.0
    if pw is not None:
        ones, zeros = np.ones(d), np.zeros(d)
        unit = routed_layer.gated_residual_norm(x, zeros, 1e9, ones, zeros, eps, ones, zeros, 0.0,
                                                rms, post_eps)[0]
        size = np.abs(x).max(-1, keepdims=True) * inverse(x, post_eps)
        y = unit * pw + (0 if pb is None else pb)
        off = 200 * U * (np.abs(unit) + size) * np.abs(pw) + 4 * U * np.abs(y)
    off_h = off + 8 * U * (np.abs(y) + np.abs(scale * r))
    half = torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -25 if dtype == torch.float16 else 1e-30
    got_h, got_n = (host(g).reshape(-1, d) for g in got)
    assert (np.abs(got_h - hidden) <= half * np.abs(hidden) + off_h + tiny).all()
    inv = inverse(hidden, eps)
    size = np.abs(hidden).max(-1, keepdims=True) * inv
    worst = off_h.max(-1, keepdims=True) * inv
    plain = hidden if rms else hidden - hidden.mean(-1, keepdims=True)
    unit = np.abs(plain * inv)
    off_n = (200 * U * (unit + size) + (2 + 2 * unit) * worst) * np.abs(args[3]) \
        + 4 * U * np.abs(normalized)
    assert (np.abs(got_n - normalized) <= half * np.abs(normalized) + off_n + tiny).all()


CASES = [
    # rows (leading dims), width, post, gate, scale, rms, bias, parameter dtype (None: rows')
    ((1,), 1, False, "one", 1.0, True, True, None),
    ((8,), 576, True, "one", 1.0, False, True, None),
    ((5,), 768, True, "columns", 1.0, True, False, torch.float32),
    ((2, 33), 512, False, "rows", 2.5, False, True, torch.float32),
    ((7,), 1000, True, "rows", 0.5, True, True, None),
    ((3,), 77, True, "columns", 1.0, False, False, None),
    ((9,), 2048, True, "one", 1.0, True, False, None),
    ((4,), 2049, False, "one", 1.0, False, True, torch.float32),
    ((2, 3), 4096, True, "rows", 1.0, False, True, None),
    ((3,), 8192, True, "columns", 1.0, False, True, torch.float32),
    ((2,), 8191, True, "one", 1.0, True, True, None),
    ((300, 7), 64, True, "one", 1.0, False, True, None),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", CASES, ids=[str(c[:6]) for c in CASES])
def test_gated_residual_norm(device, case, dtype):
    lead, width, post, gate_form, scale, rms, with_bias, parameters = case
    print(f"gated_residual_norm {case} {dtype}", flush=True)
    g = torch.Generator().manual_seed(width + len(lead))
    kind = parameters or dtype
    branch = (3 + 2 * torch.randn(*lead, width, generator=g)).to(dtype)
    residual = (torch.randn(*lead, width, generator=g) * 2).to(dtype)
    shape = {"one": (), "columns": (width,), "rows": lead + (width,)}[gate_form]
    gate = torch.randn(shape, generator=g).to(dtype if gate_form == "rows" else kind)
    vectors = [(1 + 0.2 * torch.randn(width, generator=g)).to(kind),
               (0.2 * torch.randn(width, generator=g)).to(kind),
               (1 + 0.2 * torch.randn(width, generator=g)).to(kind),
               (0.2 * torch.randn(width, generator=g)).to(kind)]
    weight, bias, post_weight, post_bias = vectors
    if not with_bias:
        bias = post_bias = None
    if not post:
        post_weight = post_bias = None
    args = (branch, residual, gate, weight, bias, 1e-5, post_weight, post_bias, scale, rms, 1e-3)
    got = gated_residual_norm(*(x.to(device) if isinstance(x, torch.Tensor) else x for x in args))
    torch.cuda.synchronize()
    assert got[0].shape == branch.shape and got[0].dtype == dtype
    check(got, *args, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", [520, 768, 1016, 2040])
@pytest.mark.parametrize("rows", [1024, 1025])
def test_rows_on_a_wave_and_on_a_workgroup(device, rows, width, dtype):
    """Up to 1024 rows of more than 64 accesses have a workgroup each, more of them a wave each."""
    g = torch.Generator().manual_seed(rows + width)
    branch, residual = (torch.randn(rows, width, generator=g).to(dtype) for _ in range(2))
    weight, bias, post = (torch.randn(width, generator=g).to(dtype) for _ in range(3))
    args = (branch, residual, torch.tensor(0.4), weight, bias, 1e-5, post, None, 1.5, False, 1e-5)
    got = gated_residual_norm(*(x.to(device) if isinstance(x, torch.Tensor) else x for x in args))
    torch.cuda.synchronize()
    check(got, *args, dtype)


def test_strided_rows_and_mixed_parameters(device):
    g = torch.Generator().manual_seed(2)
    for dtype, skip in ((torch.bfloat16, 8), (torch.bfloat16, 3), (torch.float32, 4)):
        wide = torch.randn(40, 3 * 128 + skip, generator=g).to(dtype).to(device)
        branch, residual, gate = (wide[:, skip + i * 128:skip + (i + 1) * 128] for i in range(3))
        weight = torch.randn(128, generator=g).to(device)
        bias = torch.randn(128, generator=g).half().to(device)
        post = torch.randn(128, generator=g).bfloat16().to(device)
        args = (branch, residual, gate, weight, bias, 1e-5, post, None, 1.0, False, 1e-5)
        got = gated_residual_norm(*args)
        torch.cuda.synchronize()
        check(got, *args, dtype)


def test_post_eps_defaults_to_norm_eps(device):
    g = torch.Generator().manual_seed(3)
    x, r, w = (torch.randn(4, 64, generator=g).to(device) for _ in range(3))
    w = w[0]
    one = torch.tensor(0.3, device=device)
    a = gated_residual_norm(x, r, one, w, None, 0.1, w)
    b = gated_residual_norm(x, r, one, w, None, 0.1, w, post_eps=0.1)
    c = gated_residual_norm(x, r, one, w, None, 0.1, w, post_eps=0.2)
    assert torch.equal(a[0], b[0]) and not torch.equal(a[0], c[0])


def test_extreme_gates_and_empty_rows(device):
    x = torch.randn(3, 64, device=device)
    r = torch.randn(3, 64, device=device)
    w = torch.ones(64, device=device)
    for logit, open_ in ((200.0, 1.0), (-200.0, 0.0), (float("inf"), 1.0), (-float("inf"), 0.0)):
        hidden, _ = gated_residual_norm(x, r, torch.tensor(logit, device=device), w, None, 1e-5)
        assert torch.equal(hidden, r + open_ * x)
    hidden, normalized = gated_residual_norm(x[:0], r[:0], torch.tensor(0.0, device=device), w, None,
                                             1e-5)
    assert hidden.shape == normalized.shape == (0, 64)
    # Constant rows: LayerNorm's variance is 0.
    hidden, normalized = gated_residual_norm(torch.ones(2, 64, device=device),
                                             torch.ones(2, 64, device=device),
                                             torch.tensor(0.0, device=device), w, None, 1e-5)
    assert torch.equal(normalized, torch.zeros_like(normalized))
