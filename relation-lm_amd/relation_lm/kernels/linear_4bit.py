"""Products with weights of 4 bits on gfx950.

A weight [N,K] is codes 0..15 with a scale, and optionally a zero point, for each output and
group of ``group_size`` inputs:

    W[n][k] = (codes[n][k] - zeros[k // group_size][n]) * scales[k // group_size][n]

``quantize_4bit`` makes them of a float weight, ``pack_4bit`` puts codes (from there, or from a
checkpoint) in the order in which the matrix instructions read them -- once per weight, as
``mfma_fragments`` -- and ``linear_4bit`` / ``gated_linear_4bit`` take them packed.  A token's
products read a quarter of the bytes that ``relation_linear`` with bf16 weights reads.

Inference only: the operators have no gradient.
"""
from __future__ import annotations

import torch
from torch import Tensor

from relation_lm import _native  # noqa: F401  (registers torch.ops.rlm_quantized)


def _check_group(group_size: int) -> None:
    if group_size not in (32, 64) and (group_size < 128 or group_size % 128 != 0):
        raise ValueError(f"group_size must be 32, 64 or a multiple of 128, got {group_size}")


def quantize_4bit(weight: Tensor, group_size: int = 128, symmetric: bool = False
                  ) -> tuple[Tensor, Tensor, Tensor | None]:
    """(codes uint8 [N,K], scales fp32 [groups,N], zeros fp32 [groups,N] or None) of a float
    weight [N,K], on its device.

    Each group's range, widened to hold 0, is cut into 15 steps of one scale with a whole zero
    point, and values rounded to the nearest; ``symmetric``: the scale is the largest magnitude
    / 7, the zero point 8 (no zeros).  A group of zeros has scale 1; one with an infinity or NaN
    stands for no finite values.
    """
    _check_group(group_size)
    if weight.dim() != 2 or not weight.is_floating_point():
        raise ValueError("weight must be a 2-d float tensor")
    n, k = weight.shape
    groups = -(-k // group_size)
    w = torch.nn.functional.pad(weight.float(), (0, groups * group_size - k))
    w = w.view(n, groups, group_size)
    if symmetric:
        scales = w.abs().amax(-1) / 7
        zeros = None
    else:
        low, high = w.amin(-1).clamp_max(0), w.amax(-1).clamp_min(0)
        scales = (high - low) / 15
    scales = torch.where(scales == 0, torch.ones_like(scales), scales)
    if not symmetric:
        zeros = (-low / scales).round().clamp(0, 15)
    codes = (w / scales[..., None]).round() + (8 if symmetric else zeros[..., None])
    codes = codes.nan_to_num(0).clamp(0, 15).to(torch.uint8).view(n, -1)[:, :k].contiguous()
    return (codes, scales.T.contiguous(),
            None if zeros is None else zeros.T.contiguous())


def pack_4bit(codes: Tensor) -> Tensor:
    """Codes 0..15 [N,K] (any integer type) in operand order, int32 [ceil(N/16), ceil(K/128),
    64, 4]: word s of lane 16 q + r of tile (i, j) holds row 16 i + r, inputs
    128 j + 32 s + 8 q + e (e = 0..7) at bit 4 (e // 2) + 16 (e % 2).  A packing step run once
    per weight, on the codes' device."""
    if codes.dim() != 2 or codes.dtype not in (torch.uint8, torch.int8, torch.int16, torch.int32,
                                               torch.int64):
        raise ValueError("codes must be a 2-d integer tensor")
    if codes.numel() and (int(codes.min()) < 0 or int(codes.max()) > 15):
        raise ValueError("codes must be in 0..15")
    n, k = codes.shape
    c = torch.nn.functional.pad(codes, (0, -k % 128, 0, -n % 16))
    c = c.view(-(-n // 16), 16, -(-k // 128), 4, 4, 8).permute(0, 2, 4, 1, 3, 5)
    words = torch.zeros(c.shape[:-1], dtype=torch.int32, device=codes.device)
    for e in range(8):
        words |= c[..., e].int() << (4 * (e // 2) + 16 * (e % 2))
    return words.reshape(c.shape[0], c.shape[1], 64, 4).contiguous()


def linear_4bit(input: Tensor, codes: Tensor, scales: Tensor, zeros: Tensor | None = None,
                group_size: int = 128, bias: Tensor | None = None) -> Tensor:
    """``input @ W.T + bias`` for input [..., K], in input's type (bfloat16, float16, float32).

    ``codes`` as ``pack_4bit`` gives them, ``scales`` [groups,N] in float32 or input's type,
    ``zeros`` the same or None (8 everywhere); ``group_size`` 32, 64 or a multiple of 128 (the
    last group may be short).  N and K are arbitrary.  Codes meet the input exactly, sums are
    fp32, and each group's sum is scaled in fp32.  An input that is not finite makes its
    token's outputs NaN, and so may inputs whose sums, of up to 31 times 128 of them, pass fp32
    (from about 2^115; 2^117 in fp32).
    """
    return torch.ops.rlm_quantized.linear_4bit(input, codes, scales, zeros, group_size, bias)


def gated_linear_4bit(input: Tensor, gate_codes: Tensor, gate_scales: Tensor, up_codes: Tensor,
                      up_scales: Tensor, gate_zeros: Tensor | None = None,
                      up_zeros: Tensor | None = None, group_size: int = 128,
                      activation: str = "silu") -> Tensor:
    """``act(input @ Wg.T) * (input @ Wu.T)``, the first half of a gated feed-forward block, in
    one launch; ``activation`` "silu" or "gelu" (exact).  Both weights have one shape and type,
    arguments as in ``linear_4bit``; neither product is rounded before the other."""
    return torch.ops.rlm_quantized.gated_linear_4bit(input, gate_codes, gate_scales, up_codes,
                                                     up_scales, gate_zeros, up_zeros, group_size,
                                                     activation)
