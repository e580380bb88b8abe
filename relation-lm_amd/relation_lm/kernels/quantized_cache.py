"""Key and value caches in 8 bits on gfx950: written with the rotation, and read back.

A cache is a float8_e4m3fn tensor [B,T,Hk,D] of codes and an fp32 tensor [B,T,Hk] of scales;
a row -- the features of one token and key head -- is its codes times its scale, about half
the bytes of a bf16 row.  ``rotary_to_quantized_caches`` stands to these caches as
``rotary_to_caches`` to 16-bit ones, ``routed_attention_quantized``
(``kernels/routed_attention.py``) attends over them, and ``quantized_rows`` gives their
rows in a float type to whatever else wants them.

Inference only: the operators have no gradient.
"""
from __future__ import annotations

import torch
from torch import Tensor

from relation_lm import _native  # noqa: F401  (registers torch.ops.rlm_quantized)


def rotary_to_quantized_caches(query: Tensor, key: Tensor, value: Tensor, position: Tensor,
                               frequencies: Tensor, key_cache: Tensor, value_cache: Tensor,
                               key_scale: Tensor, value_scale: Tensor,
                               interleaved: bool = False, scale: float = 1.0, ring: bool = False,
                               lengths: Tensor | None = None) -> Tensor:
    """``rotary_to_caches`` into 8-bit caches: returns the rotated query and writes the rows of
    the rotated key and of the value, as codes to ``key_cache`` / ``value_cache`` (float8_e4m3fn
    [B,T,Hk,D]) and scales to ``key_scale`` / ``value_scale`` (fp32 [B,T,Hk]); any strides with
    unit stride in D.

    A row x (fp32 after the rotation, not rounded to the key's type before) has the scale
    max |x| / 448, at least 2^-126, and the codes x / scale rounded to e4m3 (within 2^-4 of
    each value, or 2^-10 of the scale).  A row of zeros has scale 0; one that holds an
    infinity or NaN has scale NaN and reads back as NaN.  D <= 256; positions, ``lengths``
    and ``ring`` as in ``rotary_to_caches``.
    """
    return torch.ops.rlm_quantized.rotary_to_quantized_caches(
        query, key, value, position, frequencies, key_cache, value_cache, key_scale, value_scale,
        interleaved, scale, ring, lengths)


def quantized_rows(cache: Tensor, scale: Tensor, rows: Tensor | None = None,
                   dtype: torch.dtype = torch.bfloat16) -> Tensor:
    """Rows of an 8-bit cache in ``dtype`` (bfloat16, float16 or float32), each code times its
    row's scale as an fp32 product, rounded to it: all of them, [B,T,Hk,D], or the ``rows``
    [B,N] named (int32 or int64 cache rows in any order, repeats allowed), [B,N,Hk,D] with zeros
    where a row is outside [0, T)."""
    return torch.ops.rlm_quantized.quantized_rows(cache, scale, rows, dtype)
