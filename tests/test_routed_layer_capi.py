"""Refusals of the routed attention layer's entry points (no GPU needed): malformed descriptors
return hipErrorInvalidValue with a message before anything is launched."""
from __future__ import annotations

import ctypes

import pytest

from test_capi import (HIP_ERROR_INVALID_VALUE, RLM_BF16, RLM_F16, RLM_F32, RLM_I32, RLM_I64, lib,
                       tensor)  # noqa: F401  (lib: fixture)


def call(lib, name, tensors, *rest):
    """tensors: descriptors or None, in argument order up to the scalars of `rest`, which may hold
    descriptors as well (outputs)."""
    def arg(x):
        return None if x is None else ctypes.byref(x) if isinstance(x, ctypes.Structure) else x
    rc = getattr(lib, name)(*[arg(x) for x in tensors], *[arg(x) for x in rest], None)
    return rc, lib.rlm_last_error().decode()


def refused(result, *words):
    rc, message = result
    assert rc == HIP_ERROR_INVALID_VALUE, message
    for word in words:
        assert word in message, message


def i64(x):
    return ctypes.c_int64(x)


# ---------------------------------------------------------------------------
# Rotary positions
# ---------------------------------------------------------------------------

def rotary(lib, **change):
    d = dict(query=tensor([2, 5, 4, 64], RLM_BF16), key=tensor([2, 5, 2, 64], RLM_BF16),
             positions=tensor([5], RLM_I64), frequencies=tensor([32], RLM_F32),
             out_query=tensor([2, 5, 4, 64], RLM_BF16), out_key=tensor([2, 5, 2, 64], RLM_BF16))
    d.update(change)
    return call(lib, "rlm_rotary_positions",
                [d["query"], d["key"], d["positions"], d["frequencies"]], ctypes.c_int32(0),
                ctypes.c_double(1.0), d["out_query"], d["out_key"])


@pytest.mark.parametrize("change,words", [
    (dict(query=None), ["query"]),
    (dict(query=tensor([2, 5, 256], RLM_BF16)), ["query", "4-d"]),
    (dict(query=tensor([2, 5, 4, 64], RLM_I32)), ["query", "float32"]),
    (dict(query=tensor([2, 5, 4, 64], RLM_BF16, stride=[1280, 256, 1, 4])), ["query", "unit-stride"]),
    (dict(query=tensor([2, 5, 4, 64], RLM_BF16, data=0)), ["query", "null"]),
    (dict(key=tensor([2, 5, 2, 64], RLM_F16)), ["key", "dtype"]),
    (dict(key=tensor([2, 6, 2, 64], RLM_BF16)), ["key", "dim 1"]),
    (dict(key=tensor([2, 5, 2, 32], RLM_BF16)), ["key", "dim 3"]),
    (dict(frequencies=tensor([33], RLM_F32)), ["frequencies"]),
    (dict(frequencies=tensor([0], RLM_F32)), ["frequencies"]),
    (dict(frequencies=tensor([32], RLM_BF16)), ["frequencies", "float32"]),
    (dict(positions=tensor([5], RLM_F32)), ["positions", "int32/int64"]),
    (dict(positions=tensor([4], RLM_I64)), ["positions", "dim 0"]),
    (dict(positions=tensor([2, 4], RLM_I64)), ["positions", "dim 1"]),
    (dict(positions=tensor([5], RLM_I64, stride=[2])), ["positions", "contiguous"]),
    (dict(out_query=tensor([2, 5, 4, 32], RLM_BF16)), ["out_query"]),
    (dict(out_key=tensor([2, 5, 2, 64], RLM_BF16, stride=[1, 1, 1, 1])), ["out_key"]),
    (dict(query=tensor([2, 5, 4, 1032], RLM_BF16)), ["1024"]),
])
def test_rotary_positions_refuses(lib, change, words):
    refused(rotary(lib, **change), *words)


def to_caches(lib, ring=0, **change):
    d = dict(query=tensor([2, 5, 4, 64], RLM_BF16), key=tensor([2, 5, 2, 64], RLM_BF16),
             value=tensor([2, 5, 2, 64], RLM_BF16), position=tensor([], RLM_I64),
             frequencies=tensor([32], RLM_F32), key_cache=tensor([2, 16, 2, 64], RLM_BF16),
             value_cache=tensor([2, 16, 2, 64], RLM_BF16), lengths=None,
             out_query=tensor([2, 5, 4, 64], RLM_BF16))
    d.update(change)
    names = ("query", "key", "value", "position", "frequencies", "key_cache", "value_cache",
             "lengths")
    return call(lib, "rlm_rotary_to_caches", [d[n] for n in names], ctypes.c_int32(0),
                ctypes.c_double(1.0), ctypes.c_int32(ring), d["out_query"])


@pytest.mark.parametrize("change,words", [
    (dict(value=None), ["value"]),
    (dict(value=tensor([2, 5, 1, 64], RLM_BF16)), ["value", "dim 2"]),
    (dict(value=tensor([2, 5, 2, 64], RLM_F32)), ["value", "dtype"]),
    (dict(key_cache=tensor([2, 16, 1, 64], RLM_BF16)), ["key_cache", "dim 2"]),
    (dict(key_cache=tensor([2, 16, 2, 64], RLM_BF16, stride=[2048, 64, 64, 1])), ["key_cache", "overlap"]),
    (dict(key_cache=tensor([2, 16, 2, 64], RLM_BF16, stride=[0, 128, 64, 1])), ["key_cache", "overlap"]),
    (dict(value_cache=tensor([2, 15, 2, 64], RLM_BF16)), ["value_cache", "dim 1"]),
    (dict(value_cache=tensor([2, 16, 2, 64], RLM_F16)), ["value_cache", "dtype"]),
    (dict(position=tensor([3], RLM_I64)), ["position", "dim 0"]),
    (dict(position=tensor([2, 5], RLM_I64)), ["position"]),
    (dict(position=tensor([], RLM_F32)), ["position", "int32/int64"]),
    (dict(lengths=tensor([3], RLM_I64)), ["lengths", "dim 0"]),
    (dict(lengths=tensor([2], RLM_F32)), ["lengths"]),
    (dict(ring=1, key_cache=tensor([2, 12, 2, 64], RLM_BF16),
          value_cache=tensor([2, 12, 2, 64], RLM_BF16)), ["power-of-two"]),
    (dict(ring=1, key_cache=tensor([2, 4, 2, 64], RLM_BF16),
          value_cache=tensor([2, 4, 2, 64], RLM_BF16)), ["overwrite each other"]),
])
def test_rotary_to_caches_refuses(lib, change, words):
    refused(to_caches(lib, **change), *words)


# ---------------------------------------------------------------------------
# Block routing
# ---------------------------------------------------------------------------

def route(lib, block=32, window=64, top=4, strict=0, ring=0, **change):
    d = dict(query=tensor([2, 7, 1, 64], RLM_BF16), mean=tensor([2, 16, 4, 16], RLM_F32),
             std=tensor([2, 16, 4, 16], RLM_F32), gamma=tensor([4], RLM_F32),
             bias=tensor([4, 16], RLM_F32), positions=tensor([7], RLM_I64),
             blocks=tensor([2, 7, 1, 4], RLM_I32), scores=tensor([2, 7, 1, 4], RLM_F32))
    d.update(change)
    names = ("query", "mean", "std", "gamma", "bias", "positions")
    return call(lib, "rlm_block_route", [d[n] for n in names], i64(block), i64(window), i64(top),
                ctypes.c_int32(strict), ctypes.c_int32(ring), d["blocks"], d["scores"])


@pytest.mark.parametrize("change,words", [
    (dict(query=tensor([2, 7, 64], RLM_BF16)), ["router_query", "4-d"]),
    (dict(query=tensor([2, 7, 1, 32], RLM_BF16)), ["router_query", "dim 3"]),
    (dict(mean=tensor([2, 16, 4, 16], RLM_BF16)), ["block_mean", "float32"]),
    (dict(mean=tensor([1, 16, 4, 16], RLM_F32)), ["block_mean", "dim 0"]),
    (dict(std=tensor([2, 15, 4, 16], RLM_F32)), ["block_std", "dim 1"]),
    (dict(mean=tensor([2, 16, 4, 16], RLM_F32, data=0x1008)), ["16-byte"]),
    (dict(mean=tensor([2, 0, 4, 16], RLM_F32), std=tensor([2, 0, 4, 16], RLM_F32)), ["blocks"]),
    (dict(query=tensor([2, 7, 1, 24], RLM_BF16), mean=tensor([2, 16, 4, 6], RLM_F32),
          std=tensor([2, 16, 4, 6], RLM_F32)), ["multiple of 4"]),
    (dict(query=tensor([2, 7, 1, 2048], RLM_BF16), mean=tensor([2, 16, 4, 512], RLM_F32),
          std=tensor([2, 16, 4, 512], RLM_F32)), ["1024"]),
    (dict(gamma=tensor([3], RLM_F32)), ["gamma"]),
    (dict(bias=tensor([4, 0], RLM_F32)), ["bias"]),
    (dict(bias=tensor([4, 600], RLM_F32)), ["bias", "2048"]),
    (dict(block=0), ["block_size"]),
    (dict(window=-1), ["local_window"]),
    (dict(top=0), ["top_blocks"]),
    (dict(top=65), ["top_blocks"]),
    (dict(ring=1, block=24), ["power-of-two"]),
    (dict(ring=1, mean=tensor([2, 12, 4, 16], RLM_F32), std=tensor([2, 12, 4, 16], RLM_F32)),
     ["power-of-two"]),
    (dict(positions=tensor([7], RLM_F32)), ["positions"]),
    (dict(blocks=tensor([2, 7, 1, 5], RLM_I32)), ["out_blocks", "dim 3"]),
    (dict(blocks=tensor([2, 7, 1, 4], RLM_I64)), ["out_blocks"]),
    (dict(scores=tensor([2, 7, 2, 4], RLM_F32)), ["out_scores", "dim 2"]),
])
def test_block_route_refuses(lib, change, words):
    refused(route(lib, **change), *words)


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------

def attention(lib, block=32, window=64, ring=0, **change):
    d = dict(query=tensor([2, 7, 6, 64], RLM_BF16), key=tensor([2, 128, 3, 64], RLM_BF16),
             value=tensor([2, 128, 3, 64], RLM_BF16), blocks=tensor([2, 7, 4], RLM_I32),
             positions=tensor([2, 7], RLM_I64), out=tensor([2, 7, 6, 64], RLM_BF16),
             lse=tensor([2, 7, 6], RLM_F32))
    d.update(change)
    names = ("query", "key", "value", "blocks", "positions")
    return call(lib, "rlm_routed_attention", [d[n] for n in names], i64(block), i64(window),
                ctypes.c_double(0.125), ctypes.c_int32(ring), d["out"], d["lse"])


def with_dim(dim, dtype=RLM_BF16, data=0x1000):
    return dict(query=tensor([2, 7, 6, dim], dtype, data=data), key=tensor([2, 128, 3, dim], dtype),
                value=tensor([2, 128, 3, dim], dtype), out=tensor([2, 7, 6, dim], dtype))


@pytest.mark.parametrize("change,words", [
    (with_dim(60), ["head dim"]),
    (with_dim(264), ["head dim"]),
    (with_dim(0), ["head dim"]),
    (with_dim(64, data=0x1008), ["16-byte"]),
    (dict(query=tensor([2, 7, 7, 64], RLM_BF16)), ["multiple of the 3 key heads"]),
    (dict(key=tensor([2, 128, 0, 64], RLM_BF16)), ["key heads"]),
    (dict(key=tensor([2, 128, 3, 64], RLM_F32)), ["key_cache", "dtype"]),
    (dict(value=tensor([2, 127, 3, 64], RLM_BF16)), ["value_cache", "dim 1"]),
    (dict(value=tensor([2, 128, 3, 32], RLM_BF16)), ["value_cache", "dim 3"]),
    (dict(key=tensor([2, 128, 3, 64], RLM_BF16, stride=[24576, 196, 64, 1])), ["multiples of 8"]),
    (dict(key=tensor([2, 128, 3, 64], RLM_BF16, stride=[24576, 192, 1, 3])), ["unit-stride"]),
    (dict(blocks=tensor([2, 7, 4], RLM_I64)), ["blocks", "int32"]),
    (dict(blocks=tensor([7, 4], RLM_I32)), ["blocks"]),
    (dict(blocks=tensor([2, 6, 4], RLM_I32)), ["blocks", "dim 1"]),
    (dict(blocks=tensor([2, 7, 2, 4], RLM_I32)), ["blocks", "dim 2"]),
    (dict(blocks=tensor([2, 7, 65], RLM_I32)), ["64 picks"]),
    (dict(positions=tensor([2, 8], RLM_I64)), ["positions"]),
    (dict(positions=tensor([2, 7], RLM_F32)), ["positions"]),
    (dict(block=0), ["block_size"]),
    (dict(window=-1), ["local_window"]),
    (dict(ring=1, block=48), ["power-of-two"]),
    (dict(ring=1, key=tensor([2, 96, 3, 64], RLM_BF16), value=tensor([2, 96, 3, 64], RLM_BF16)),
     ["power-of-two"]),
    (dict(out=tensor([2, 7, 6, 64], RLM_F32)), ["out", "dtype"]),
    (dict(lse=tensor([2, 7, 5], RLM_F32)), ["out_lse", "dim 2"]),
    (dict(lse=tensor([2, 7, 6], RLM_BF16)), ["out_lse", "float32"]),
])
def test_routed_attention_refuses(lib, change, words):
    refused(attention(lib, **change), *words)


# ---------------------------------------------------------------------------
# Gated residual norm
# ---------------------------------------------------------------------------

def norm(lib, **change):
    d = dict(branch=tensor([9, 64], RLM_BF16), residual=tensor([9, 64], RLM_BF16),
             gate=tensor([], RLM_F32), weight=tensor([64], RLM_BF16), bias=None, post_weight=None,
             post_bias=None, hidden=tensor([9, 64], RLM_BF16), normalized=tensor([9, 64], RLM_BF16))
    d.update(change)
    return call(lib, "rlm_gated_residual_norm",
                [d["branch"], d["residual"], d["gate"], d["weight"], d["bias"]],
                ctypes.c_double(1e-5), d["post_weight"], d["post_bias"], ctypes.c_double(1e-5),
                ctypes.c_double(1.0), ctypes.c_int32(0), d["hidden"], d["normalized"])


@pytest.mark.parametrize("change,words", [
    (dict(branch=tensor([64], RLM_BF16)), ["branch", "2-d"]),
    (dict(branch=tensor([9, 64], RLM_I32)), ["branch"]),
    (dict(branch=tensor([9, 64], RLM_BF16, stride=[64, 2])), ["branch", "unit-stride"]),
    (dict(branch=tensor([9, 64], RLM_BF16, stride=[0, 1])), ["branch", "row stride"]),
    (dict(branch=tensor([9, 8200], RLM_BF16)), ["8192"]),
    (dict(residual=tensor([9, 64], RLM_F32)), ["residual", "dtype"]),
    (dict(residual=tensor([8, 64], RLM_BF16)), ["residual", "dim 0"]),
    (dict(gate=tensor([32], RLM_F32)), ["gate"]),
    (dict(gate=tensor([9, 64], RLM_F32)), ["gate", "dtype"]),
    (dict(gate=tensor([9, 1], RLM_BF16)), ["gate", "dim 1"]),
    (dict(gate=None), ["gate"]),
    (dict(gate=tensor([], RLM_I32)), ["gate"]),
    (dict(weight=tensor([32], RLM_BF16)), ["norm_weight"]),
    (dict(bias=tensor([64], RLM_I32)), ["norm_bias"]),
    (dict(post_bias=tensor([64], RLM_BF16)), ["post_weight"]),
    (dict(post_weight=tensor([63], RLM_BF16)), ["post_weight"]),
    (dict(hidden=tensor([9, 64], RLM_BF16, stride=[128, 1])), ["out_hidden", "contiguous"]),
    (dict(normalized=tensor([9, 64], RLM_F32)), ["out_normalized", "dtype"]),
])
def test_gated_residual_norm_refuses(lib, change, words):
    refused(norm(lib, **change), *words)


def test_calls_without_elements_return_at_once(lib):
    """No launch: these succeed on a machine without a GPU."""
    empty = dict(query=tensor([0, 5, 4, 64], RLM_BF16), key=tensor([0, 5, 2, 64], RLM_BF16),
                 out_query=tensor([0, 5, 4, 64], RLM_BF16), out_key=tensor([0, 5, 2, 64], RLM_BF16))
    assert rotary(lib, **empty)[0] == 0
    assert route(lib, query=tensor([2, 0, 1, 64], RLM_BF16), positions=tensor([0], RLM_I64),
                 blocks=tensor([2, 0, 1, 4], RLM_I32), scores=tensor([2, 0, 1, 4], RLM_F32))[0] == 0
    assert attention(lib, query=tensor([2, 0, 6, 64], RLM_BF16), blocks=tensor([2, 0, 4], RLM_I32),
                     positions=tensor([0], RLM_I64), out=tensor([2, 0, 6, 64], RLM_BF16),
                     lse=tensor([2, 0, 6], RLM_F32))[0] == 0
    none = tensor([0, 64], RLM_BF16)
    assert norm(lib, branch=none, residual=none, hidden=none, normalized=none)[0] == 0


def test_more_threads_than_one_launch_takes(lib):
    n = 1 << 29
    rows = dict(query=tensor([1, n, 1, 8], RLM_BF16), key=tensor([1, n, 1, 8], RLM_BF16),
                positions=tensor([n], RLM_I64), frequencies=tensor([4], RLM_F32),
                out_query=tensor([1, n, 1, 8], RLM_BF16), out_key=tensor([1, n, 1, 8], RLM_BF16))
    refused(rotary(lib, **rows), "rotary_positions", "too many rows")
    refused(route(lib, query=tensor([1, n, 1, 4], RLM_BF16), mean=tensor([1, 1, 1, 4], RLM_F32),
                  std=tensor([1, 1, 1, 4], RLM_F32), gamma=tensor([1], RLM_F32),
                  bias=tensor([1, 1], RLM_F32), positions=tensor([n], RLM_I64),
                  blocks=tensor([1, n, 1, 4], RLM_I32), scores=tensor([1, n, 1, 4], RLM_F32)),
            "block_route", "too many rows")
    one = dict(query=tensor([n, 1, 1, 8], RLM_BF16), key=tensor([n, 1, 1, 8], RLM_BF16),
               value=tensor([n, 1, 1, 8], RLM_BF16), blocks=tensor([n, 1, 1], RLM_I32),
               positions=tensor([n, 1], RLM_I64), out=tensor([n, 1, 1, 8], RLM_BF16),
               lse=tensor([n, 1, 1], RLM_F32))
    refused(attention(lib, **one), "routed_attention", "too many rows")
    wide = tensor([n, 8], RLM_BF16)
    refused(norm(lib, branch=wide, residual=wide, weight=tensor([8], RLM_BF16), hidden=wide,
                 normalized=wide), "gated_residual_norm", "too many rows")
