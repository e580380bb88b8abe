"""Products with 4-bit weights of more tokens than 65535 blocks of 32, against oracle/few_bits.py within the
bounds of test_linear_4bit_gpu.py."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from relation_lm.kernels.linear_4bit import gated_linear_4bit, linear_4bit
from test_linear_4bit_gpu import U, check, host, on, product, weight

pytestmark = pytest.mark.gpu

# tokens, outputs, width, group, dtype
SHAPES = [
    (2 ** 21 + 5, 16, 128, 128, torch.bfloat16), (2 ** 22 - 1, 9, 40, 32, torch.float16),
    (2 ** 21 - 31, 24, 64, 64, torch.float32), (2 ** 21 - 32, 16, 128, 64, torch.bfloat16),
]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_many_tokens(device, shape):
    tokens, outputs, width, group, dtype = shape
    print(f"many tokens {shape}", flush=True)
    g = torch.Generator().manual_seed(outputs + width)
    some = torch.cat((torch.arange(40), torch.randint(0, tokens, (100,), generator=g),
                      torch.arange(65535 * 32 - 9, min(65535 * 32 + 9, tokens)),
                      torch.arange(tokens - 40, tokens)))
    of = torch.Generator(device=device).manual_seed(1)
    x = torch.randn(tokens, width, generator=of, device=device, dtype=dtype)
    gate, up = [weight(g, outputs, width, group, True, dtype) for _ in range(2)]
    got = linear_4bit(x, *on(device, gate), group)
    torch.cuda.synchronize()
    few = x[some.to(device)].cpu()
    (a, da), (b, db) = product(few, gate, group), product(few, up, group)
    check(got[some.to(device)], a, da, dtype)
    (gc, gs, gz), (uc, us, uz) = on(device, gate), on(device, up)
    got = gated_linear_4bit(x, gc, gs, uc, us, gz, uz, group, "silu")
    torch.cuda.synchronize()
    act = torch.nn.functional.silu(torch.from_numpy(a)).numpy()
    d_act = 1.13 * da + 8 * U * np.abs(act)
    check(got[some.to(device)], act * b,
          d_act * (np.abs(b) + db) + np.abs(act) * db + U * np.abs(act * b), dtype)
    assert torch.isfinite(got).all()
