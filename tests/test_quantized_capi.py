"""Refusals of the entry points for 8-bit caches and 4-bit weights (no GPU needed): malformed
descriptors return hipErrorInvalidValue with a message before anything is launched."""
from __future__ import annotations

import ctypes

import pytest
import torch

from test_capi import RLM_BF16, RLM_F16, RLM_F32, RLM_I32, RLM_I64, lib, tensor  # noqa: F401
from test_routed_layer_capi import call, i64, refused

RLM_F8E4M3 = 5


def store(lib, ring=0, **change):
    d = dict(query=tensor([2, 5, 4, 64], RLM_BF16), key=tensor([2, 5, 2, 64], RLM_BF16),
             value=tensor([2, 5, 2, 64], RLM_BF16), position=tensor([], RLM_I64),
             frequencies=tensor([32], RLM_F32), key_cache=tensor([2, 16, 2, 64], RLM_F8E4M3),
             value_cache=tensor([2, 16, 2, 64], RLM_F8E4M3), key_scale=tensor([2, 16, 2], RLM_F32),
             value_scale=tensor([2, 16, 2], RLM_F32), lengths=None,
             out_query=tensor([2, 5, 4, 64], RLM_BF16))
    d.update(change)
    names = ("query", "key", "value", "position", "frequencies", "key_cache", "value_cache",
             "key_scale", "value_scale", "lengths")
    return call(lib, "rlm_rotary_to_quantized_caches", [d[n] for n in names], ctypes.c_int32(0),
                ctypes.c_double(1.0), ctypes.c_int32(ring), d["out_query"])


@pytest.mark.parametrize("change,words", [
    (dict(query=None), ["query"]),
    (dict(value=None), ["value"]),
    (dict(key_scale=None), ["key_scale", "missing"]),
    (dict(key_cache=tensor([2, 16, 2, 64], RLM_BF16)), ["key_cache", "float8_e4m3fn"]),
    (dict(value_cache=tensor([2, 16, 2, 32], RLM_F8E4M3)), ["value_cache", "dim 3"]),
    (dict(value_cache=tensor([2, 15, 2, 64], RLM_F8E4M3)), ["value_cache", "dim 1"]),
    (dict(key_cache=tensor([2, 16, 2, 64], RLM_F8E4M3, stride=[2048, 64, 0, 1])), ["overlap"]),
    (dict(key_scale=tensor([2, 16, 3], RLM_F32)), ["key_scale", "dim 2"]),
    (dict(value_scale=tensor([2, 15, 2], RLM_F32)), ["value_scale", "dim 1"]),
    (dict(value_scale=tensor([2, 16, 2], RLM_BF16)), ["value_scale", "float32"]),
    (dict(value_scale=tensor([2, 16, 2, 1], RLM_F32)), ["value_scale", "3-d"]),
    (dict(value_scale=tensor([2, 16, 2], RLM_F32, stride=[32, 2, 0])), ["value_scale", "overlap"]),
    (dict(value_scale=tensor([2, 16, 2], RLM_F32, data=0)), ["value_scale", "null"]),
    (dict(query=tensor([2, 5, 4, 264], RLM_BF16)), ["[1, 256]"]),
    (dict(frequencies=tensor([33], RLM_F32)), ["frequencies"]),
    (dict(position=tensor([3], RLM_I64)), ["position", "dim 0"]),
    (dict(lengths=tensor([2], RLM_F32)), ["lengths"]),
    (dict(ring=1, key_cache=tensor([2, 12, 2, 64], RLM_F8E4M3),
          value_cache=tensor([2, 12, 2, 64], RLM_F8E4M3), key_scale=tensor([2, 12, 2], RLM_F32),
          value_scale=tensor([2, 12, 2], RLM_F32)), ["power-of-two"]),
    (dict(out_query=tensor([2, 5, 4, 64], RLM_F32)), ["out_query"]),
])
def test_rotary_to_quantized_caches_refuses(lib, change, words):  # noqa: F811
    refused(store(lib, **change), *words)


def rows(lib, **change):
    d = dict(cache=tensor([2, 16, 2, 64], RLM_F8E4M3), scale=tensor([2, 16, 2], RLM_F32),
             rows=tensor([2, 9], RLM_I64), out=tensor([2, 9, 2, 64], RLM_BF16))
    d.update(change)
    return call(lib, "rlm_quantized_rows", [d["cache"], d["scale"], d["rows"], d["out"]])


@pytest.mark.parametrize("change,words", [
    (dict(cache=None), ["cache"]),
    (dict(cache=tensor([2, 16, 2, 64], RLM_BF16)), ["cache", "float8_e4m3fn"]),
    (dict(cache=tensor([2, 16, 128], RLM_F8E4M3)), ["cache", "4-d"]),
    (dict(scale=tensor([2, 16, 2], RLM_F16)), ["scale", "float32"]),
    (dict(scale=tensor([2, 17, 2], RLM_F32)), ["scale", "dim 1"]),
    (dict(rows=tensor([2, 9], RLM_F32)), ["rows", "int32/int64"]),
    (dict(rows=tensor([1, 9], RLM_I64)), ["rows", "dim 0"]),
    (dict(rows=tensor([9], RLM_I64)), ["rows", "2-d"]),
    (dict(out=tensor([2, 8, 2, 64], RLM_BF16)), ["out", "dim 1"]),
    (dict(out=tensor([2, 9, 2, 64], RLM_I32)), ["out", "float32"]),
    (dict(out=tensor([2, 9, 2, 64], RLM_BF16, stride=[2304, 256, 128, 2])), ["out", "contiguous"]),
    (dict(rows=None), ["out", "dim 1"]),
    (dict(cache=tensor([2, 1 << 30, 2, 64], RLM_F8E4M3), scale=tensor([2, 1 << 30, 2], RLM_F32),
          rows=None, out=tensor([2, 1 << 30, 2, 64], RLM_BF16)), ["too many"]),
])
def test_quantized_rows_refuses(lib, change, words):  # noqa: F811
    refused(rows(lib, **change), *words)


def attention(lib, block=32, window=64, ring=0, **change):
    d = dict(query=tensor([2, 7, 6, 64], RLM_BF16), key=tensor([2, 128, 3, 64], RLM_F8E4M3),
             value=tensor([2, 128, 3, 64], RLM_F8E4M3), key_scale=tensor([2, 128, 3], RLM_F32),
             value_scale=tensor([2, 128, 3], RLM_F32), blocks=tensor([2, 7, 4], RLM_I32),
             positions=tensor([2, 7], RLM_I64), out=tensor([2, 7, 6, 64], RLM_BF16),
             lse=tensor([2, 7, 6], RLM_F32))
    d.update(change)
    names = ("query", "key", "value", "key_scale", "value_scale", "blocks", "positions")
    return call(lib, "rlm_routed_attention_quantized", [d[n] for n in names], i64(block),
                i64(window), ctypes.c_double(0.125), ctypes.c_int32(ring), d["out"], d["lse"])


def with_dim(dim):
    return dict(query=tensor([2, 7, 6, dim], RLM_BF16), key=tensor([2, 128, 3, dim], RLM_F8E4M3),
                value=tensor([2, 128, 3, dim], RLM_F8E4M3), out=tensor([2, 7, 6, dim], RLM_BF16))


@pytest.mark.parametrize("change,words", [
    (with_dim(72), ["head dim", "multiple of 16"]),
    (with_dim(272), ["head dim"]),
    (with_dim(8), ["head dim"]),
    (dict(query=tensor([2, 7, 6, 64], RLM_F8E4M3)), ["query", "float32"]),
    (dict(key=tensor([2, 128, 3, 64], RLM_BF16)), ["key_cache", "float8_e4m3fn"]),
    (dict(value=tensor([2, 127, 3, 64], RLM_F8E4M3)), ["value_cache", "dim 1"]),
    (dict(key=tensor([2, 128, 3, 64], RLM_F8E4M3, stride=[24576, 200, 64, 1])), ["multiples of"]),
    (dict(value=tensor([2, 128, 3, 64], RLM_F8E4M3, data=0x1008)), ["16-byte"]),
    (dict(key_scale=None), ["key_scale", "missing"]),
    (dict(value_scale=tensor([2, 128, 3], RLM_F16)), ["value_scale", "float32"]),
    (dict(value_scale=tensor([2, 128, 2], RLM_F32)), ["value_scale", "dim 2"]),
    (dict(blocks=tensor([2, 7, 65], RLM_I32)), ["64 picks"]),
    (dict(block=0), ["block_size"]),
    (dict(ring=1, block=48), ["power-of-two"]),
    (dict(lse=tensor([2, 7, 6], RLM_BF16)), ["out_lse", "float32"]),
])
def test_routed_attention_quantized_refuses(lib, change, words):  # noqa: F811
    refused(attention(lib, **change), *words)


def linear(lib, group=64, **change):
    d = dict(input=tensor([5, 200], RLM_BF16), codes=tensor([3, 2, 64, 4], RLM_I32),
             scales=tensor([4, 40], RLM_BF16), zeros=None, bias=None,
             out=tensor([5, 40], RLM_BF16))
    d.update(change)
    return call(lib, "rlm_linear_4bit", [d["input"], d["codes"], d["scales"], d["zeros"]],
                i64(group), d["bias"], d["out"])


@pytest.mark.parametrize("change,words", [
    (dict(input=None), ["input"]),
    (dict(input=tensor([5, 200], RLM_I32)), ["input", "float32"]),
    (dict(input=tensor([5, 200], RLM_BF16, stride=[200, 2])), ["input", "unit-stride"]),
    (dict(input=tensor([5, 0], RLM_BF16)), ["width"]),
    (dict(input=tensor([1 << 22, 200], RLM_BF16)), ["2^22"]),
    (dict(codes=None), ["codes", "missing"]),
    (dict(codes=tensor([3, 2, 64], RLM_I32)), ["codes", "4-d"]),
    (dict(codes=tensor([3, 2, 64, 4], RLM_I64)), ["codes", "int32"]),
    (dict(codes=tensor([2, 2, 64, 4], RLM_I32)), ["codes", "dim 0"]),
    (dict(codes=tensor([3, 1, 64, 4], RLM_I32)), ["codes", "dim 1"]),
    (dict(codes=tensor([3, 2, 64, 4], RLM_I32, data=0x1004)), ["codes", "16-byte"]),
    (dict(scales=None), ["scales"]),
    (dict(scales=tensor([40], RLM_BF16)), ["scales"]),
    (dict(scales=tensor([3, 40], RLM_BF16)), ["scales", "dim 0"]),
    (dict(scales=tensor([4, 40], RLM_F16)), ["scales", "float32 or the input's"]),
    (dict(zeros=tensor([4, 39], RLM_BF16)), ["zeros", "dim 1"]),
    (dict(zeros=tensor([4, 40], RLM_F32)), ["zeros", "dtype"]),
    (dict(group=0), ["group_size"]),
    (dict(group=96), ["group_size"]),
    (dict(group=192), ["group_size"]),
    (dict(bias=tensor([39], RLM_BF16)), ["bias"]),
    (dict(bias=tensor([40], RLM_I32)), ["bias"]),
    (dict(out=tensor([5, 40], RLM_F32)), ["out", "dtype"]),
    (dict(out=tensor([5, 41], RLM_BF16)), ["out", "dim 1"]),
    (dict(out=tensor([5, 40], RLM_BF16, data=0x1008)), ["out", "16-byte"]),
])
def test_linear_4bit_refuses(lib, change, words):  # noqa: F811
    refused(linear(lib, **change), *words)


def gated(lib, activation=0, group=64, **change):
    d = dict(input=tensor([5, 200], RLM_BF16), out=tensor([5, 40], RLM_BF16))
    for side in ("gate", "up"):
        d.update({f"{side}_codes": tensor([3, 2, 64, 4], RLM_I32),
                  f"{side}_scales": tensor([4, 40], RLM_BF16), f"{side}_zeros": None})
    d.update(change)
    names = ("input", "gate_codes", "gate_scales", "gate_zeros", "up_codes", "up_scales",
             "up_zeros")
    return call(lib, "rlm_gated_linear_4bit", [d[n] for n in names], i64(group),
                ctypes.c_int32(activation), d["out"])


@pytest.mark.parametrize("change,words", [
    (dict(activation=2), ["activation"]),
    (dict(up_scales=None), ["up_scales"]),
    (dict(up_scales=tensor([4, 41], RLM_BF16)), ["up_scales", "dim 1"]),
    (dict(up_codes=tensor([4, 2, 64, 4], RLM_I32)), ["up_codes", "dim 0"]),
    (dict(up_scales=tensor([4, 40], RLM_F32)), ["up_scales", "dtype"]),
    (dict(gate_zeros=tensor([4, 40], RLM_BF16)), ["both or neither"]),
    (dict(up_zeros=tensor([4, 40], RLM_BF16)), ["both or neither"]),
    (dict(out=tensor([4, 40], RLM_BF16)), ["out", "dim 0"]),
])
def test_gated_linear_4bit_refuses(lib, change, words):  # noqa: F811
    refused(gated(lib, **change), *words)


def test_calls_without_elements_return_at_once(lib):  # noqa: F811
    """No launch: these succeed on a machine without a GPU."""
    assert store(lib, query=tensor([2, 0, 4, 64], RLM_BF16), key=tensor([2, 0, 2, 64], RLM_BF16),
                 value=tensor([2, 0, 2, 64], RLM_BF16),
                 out_query=tensor([2, 0, 4, 64], RLM_BF16))[0] == 0
    assert rows(lib, rows=tensor([2, 0], RLM_I64), out=tensor([2, 0, 2, 64], RLM_BF16))[0] == 0
    assert attention(lib, query=tensor([2, 0, 6, 64], RLM_BF16), blocks=tensor([2, 0, 4], RLM_I32),
                     positions=tensor([0], RLM_I64), out=tensor([2, 0, 6, 64], RLM_BF16),
                     lse=tensor([2, 0, 6], RLM_F32))[0] == 0
    none = dict(input=tensor([0, 200], RLM_BF16), out=tensor([0, 40], RLM_BF16))
    assert linear(lib, **none)[0] == 0
    assert gated(lib, **none)[0] == 0


def test_packing_on_the_cpu():
    """Codes come back from where the layout says they are; what is no code is refused."""
    from relation_lm.kernels.linear_4bit import pack_4bit, quantize_4bit
    g = torch.Generator().manual_seed(0)
    codes = torch.randint(0, 16, (37, 300), generator=g, dtype=torch.uint8)
    packed = pack_4bit(codes)
    assert packed.shape == (3, 3, 64, 4) and packed.dtype == torch.int32
    for n, k in [(0, 0), (36, 299), (17, 130), (5, 255), (31, 9)]:
        lane = 16 * (k % 32 // 8) + n % 16
        word = int(packed[n // 16, k // 128, lane, k % 128 // 32]) & 0xffffffff
        e = k % 8
        assert (word >> (4 * (e // 2) + 16 * (e % 2))) & 15 == int(codes[n, k])
    for bad in (codes.float(), codes[0], codes.int() - 9, codes + 1):
        with pytest.raises(ValueError, match="codes"):
            pack_4bit(bad)
    for bad in (torch.zeros(4), torch.zeros(4, 4, dtype=torch.int32)):
        with pytest.raises(ValueError, match="weight"):
            quantize_4bit(bad)
    with pytest.raises(ValueError, match="group_size"):
        quantize_4bit(torch.zeros(4, 64), 48)
    codes, scales, zeros = quantize_4bit(torch.zeros(4, 64), 32, symmetric=True)
    assert (codes == 8).all() and (scales == 1).all() and zeros is None
