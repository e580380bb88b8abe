"""The norms before and after a block, fused with its gate and residual sum, on gfx950.

Generalises what the relation path does at its ends -- a block's
``hidden + sigmoid(residual_gate) * context`` followed by the next block's input_norm,
the head's ``output_norm(query + sigmoid(mix) * context)`` -- to any layer's branch.
No reference operator.  Inference only: no gradient.
"""
from __future__ import annotations

import torch
from torch import Tensor

from relation_lm import _native  # noqa: F401  (registers torch.ops.rlm)


def gated_residual_norm(branch: Tensor, residual: Tensor, gate: Tensor, norm_weight: Tensor,
                        norm_bias: Tensor | None, norm_eps: float,
                        post_weight: Tensor | None = None, post_bias: Tensor | None = None,
                        residual_scale: float = 1.0, rms: bool = False,
                        post_eps: float | None = None) -> tuple[Tensor, Tensor]:
    """Returns (hidden, normalized) of branch's shape [..., D] and dtype:

        hidden     = residual_scale * residual + sigmoid(gate) * post(branch)
        normalized = norm(hidden)

    norm is LayerNorm with norm_weight / norm_bias (``rms``: the root-mean-square norm);
    post the same with post_weight / post_bias and post_eps (default norm_eps), or nothing
    without a post_weight.  ``gate`` holds logits: 0-d, [D], or branch's shape.  The second
    norm reads hidden before its rounding.  D <= 8192.
    """
    return torch.ops.rlm.gated_residual_norm(branch, residual, gate, norm_weight, norm_bias,
                                             norm_eps, post_weight, post_bias, residual_scale,
                                             rms, post_eps)
