"""CPU tests of the quantised serving operators: what they refuse, before anything reaches a GPU, and their form on the host."""
import ctypes

import numpy as np
import pytest
import torch

import quant_ref as qr
from irontensor_b200 import (Precision, QuantizedCache, QuantizedRows, Tensor, _lib, attention_decode_quantized, kv_cache_append,
                             kv_cache_read, linear_int8_forward, ops, quantize_rows, rope_positions)

FP32, BF16 = Precision.FP32, Precision.BF16


def tensor(*shape, precision=BF16):
    return Tensor(torch.zeros(shape, dtype=torch.float32 if precision is FP32 else torch.bfloat16), list(shape), precision)


def cache(B=2, max_len=8, Hkv=2, D=64):
    g = -(-D // 32)
    return QuantizedCache(torch.zeros((2, B, Hkv, max_len, 16 * g), dtype=torch.uint8), torch.zeros((2, B, Hkv, max_len, g), dtype=torch.bfloat16), D)


def ints(*values):
    return torch.tensor(values, dtype=torch.int32)


def test_cache_form_is_checked():
    c = cache(D=80)
    assert c.shape() == [2, 8, 2, 80] and c.codes.shape[-1] == 48 and c.byte_size() == 2 * 2 * 2 * 8 * (48 + 6)
    with pytest.raises(AssertionError, match="multiple of 8"):
        QuantizedCache(c.codes, c.scales, 84)
    with pytest.raises(AssertionError, match="codes must be"):
        QuantizedCache(c.codes, c.scales, 64)
    with pytest.raises(AssertionError, match="codes must be"):
        QuantizedCache(c.codes.to(torch.int8), c.scales, 80)
    with pytest.raises(AssertionError, match="scales must be"):
        QuantizedCache(c.codes, c.scales.float(), 80)
    with pytest.raises(AssertionError, match="scales must be"):
        QuantizedCache(c.codes, c.scales[:, :, :, 1:], 80)
    with pytest.raises(AssertionError, match="codes must be int8"):
        QuantizedRows(torch.zeros((4, 16), dtype=torch.uint8), torch.zeros(4))
    with pytest.raises(AssertionError, match="scales must be float32"):
        QuantizedRows(torch.zeros((4, 16), dtype=torch.int8), torch.zeros(3))


def test_attributes_set_anew_are_checked_when_they_are_used():
    c, r = cache(), QuantizedRows(torch.zeros((4, 16), dtype=torch.int8), torch.zeros(4))
    c.scales, r.scales = c.scales[:, :, :, 1:], torch.zeros(3)
    for call in (lambda: kv_cache_append(c, tensor(2, 1, 2, 64), tensor(2, 1, 2, 64), ints(0, 0)), lambda: kv_cache_read(c, 1),
                 lambda: attention_decode_quantized(tensor(2, 4, 64), c, ints(0, 0))):
        with pytest.raises(AssertionError, match="scales must be bfloat16"):
            call()
    good = QuantizedRows(torch.zeros((4, 16), dtype=torch.int8), torch.zeros(4))
    for x, w in ((r, good), (good, r)):
        with pytest.raises(AssertionError, match="scales must be float32"):
            linear_int8_forward(x, w)


@pytest.mark.parametrize("call,match", [
    (lambda: kv_cache_append(cache(), tensor(2, 1, 2, 64), tensor(2, 1, 2, 64, precision=FP32), ints(0, 0)), "same shape and precision"),
    (lambda: kv_cache_append(cache(), tensor(2, 1, 2, 32), tensor(2, 1, 2, 32), ints(0, 0)), "of the cache"),
    (lambda: kv_cache_append(cache(), tensor(2, 2, 64), tensor(2, 2, 64), ints(0, 0)), "of the cache"),
    (lambda: kv_cache_append(cache(), tensor(3, 1, 2, 64), tensor(3, 1, 2, 64), ints(0, 0, 0)), "of the cache"),
    (lambda: kv_cache_append(cache(), tensor(2, 1, 2, 64), tensor(2, 1, 2, 64), ints(0)), "lengths must have the shape"),
    (lambda: kv_cache_append(cache(), tensor(2, 1, 2, 64), tensor(2, 1, 2, 64), ints(0, 0).long()), "lengths must be .* int32"),
    (lambda: kv_cache_append(cache(), tensor(2, 1, 2, 64), tensor(2, 1, 2, 64), [0, 0]), "lengths must be .* int32"),
    (lambda: kv_cache_append(cache(), tensor(2, 1, 2, 64), tensor(2, 1, 2, 64), ints(0, 0), ints(1)), "counts must have the shape"),
    (lambda: kv_cache_read(cache(), -1), "negative"),
    (lambda: kv_cache_read(cache(), 1, ints(0)), "starts must have the shape"),
    (lambda: kv_cache_read(cache(), 1, None, ints(0)), "lengths must have the shape"),
    (lambda: attention_decode_quantized(tensor(2, 4, 32), cache(), ints(0, 0)), "of the cache"),
    (lambda: attention_decode_quantized(tensor(2, 1, 4, 64), cache(), ints(0, 0)), "of the cache"),
    (lambda: attention_decode_quantized(tensor(2, 3, 64), cache(), ints(0, 0)), "divisible"),
    (lambda: attention_decode_quantized(tensor(2, 4, 64), cache(), 5), "lengths must be .* int32"),
    (lambda: rope_positions(tensor(2, 3, 64), None, ints(0)), "4D"),
    (lambda: rope_positions(tensor(1, 2, 3, 7), None, ints(0, 1)[None]), "even"),
    (lambda: rope_positions(tensor(1, 2, 3, 64), tensor(1, 2, 3, 32), ints(0, 1)[None]), "k must be"),
    (lambda: rope_positions(tensor(1, 2, 3, 64), tensor(1, 2, 3, 64, precision=FP32), ints(0, 1)[None]), "precision of q"),
    (lambda: rope_positions(tensor(1, 2, 3, 64), None, ints(0, 1)), "positions must have the shape"),
    (lambda: rope_positions(tensor(1, 2, 3, 64), None, ints(0, 1)[None].float()), "int32"),
    (lambda: rope_positions(tensor(1, 2, 3, 64), None, ints(0, 1)[None, None].expand(3, 1, 2)), "sections"),
    (lambda: rope_positions(tensor(1, 2, 3, 64), None, ints(0, 1)[None, None].expand(3, 1, 2), sections=[10, 10, 10]), "add up"),
    (lambda: rope_positions(tensor(1, 2, 3, 64), None, ints(0, 1)[None, None].expand(3, 1, 2), sections=[40, -4, -4]), "add up"),
    (lambda: rope_positions(tensor(1, 2, 3, 64), None, ints(0, 1)[None, None].expand(5, 1, 2), sections=[8, 8, 8, 4, 4]), "1 to 4 axes"),
    (lambda: quantize_rows(tensor(2, 2, 16)), "rows, cols"),
    (lambda: linear_int8_forward(rows(3, 16), rows(8, 32)), "inner dimensions"),
    (lambda: linear_int8_forward(rows(3, 16), rows(24, 16), splits=[8, 8]), "splits"),
    (lambda: linear_int8_forward(rows(3, 16), rows(32, 16), splits=[8, 8, 8, 8]), "splits"),
    (lambda: linear_int8_forward(rows(3, 16), rows(24, 16), splits=[32, -8]), "splits"),
])
def test_arguments_that_do_not_fit_are_refused(call, match):
    with pytest.raises(AssertionError, match=match):
        call()


def rows(n, k):
    return QuantizedRows(torch.zeros((n, k), dtype=torch.int8), torch.zeros(n))


def test_tensors_on_the_host_are_refused():
    calls = (lambda: kv_cache_append(cache(), tensor(2, 1, 2, 64), tensor(2, 1, 2, 64), ints(0, 0)), lambda: kv_cache_read(cache(), 1),
             lambda: attention_decode_quantized(tensor(2, 4, 64), cache(), ints(0, 0)), lambda: quantize_rows(tensor(2, 16)),
             lambda: linear_int8_forward(rows(3, 16), rows(8, 16)), lambda: rope_positions(tensor(1, 2, 3, 64), None, ints(0, 1)[None]))
    for call in calls:
        with pytest.raises((AssertionError, RuntimeError), match="device"):
            call()


def test_c_entries_refuse_before_the_gpu():
    lib = _lib.load()
    n = ctypes.c_size_t()
    assert lib.it_attention_decode_q4_workspace_bytes(32, 32, 128, ctypes.byref(n)) == _lib.IT_OK and n.value > 32 * 32 * 130 * 4
    assert lib.it_attention_decode_q4_workspace_bytes(1, 1, 129, ctypes.byref(n)) == _lib.IT_ERR_UNSUPPORTED_SHAPE
    assert lib.it_attention_decode_q4_workspace_bytes(1, 1, 60, ctypes.byref(n)) == _lib.IT_ERR_UNSUPPORTED_SHAPE
    assert lib.it_attention_decode_q4_workspace_bytes(1, -1, 64, ctypes.byref(n)) == _lib.IT_ERR_INVALID_ARG
    assert lib.it_attention_decode_q4_workspace_bytes(1, 1, 64, None) == _lib.IT_ERR_INVALID_ARG
    none9, bad = [None] * 9, _lib.IT_ERR_INVALID_ARG
    assert lib.it_kv_cache_q4_append(None, None, _lib.IT_BF16, 1, 1, 1, 64, 8, *none9) == bad
    assert lib.it_kv_cache_q4_read(None, None, _lib.IT_BF16, 1, 1, 1, 64, 8, *none9[:8]) == bad
    assert lib.it_attention_decode_q4(None, None, _lib.IT_BF16, 1, 1, 1, 64, 8, *none9, 0) == bad
    assert lib.it_quantize_rows_i8(None, None, _lib.IT_BF16, 1, 16, None, None, None) == bad
    assert lib.it_linear_i8_fwd(None, None, _lib.IT_BF16, 1, 16, 8, None, None, None, None, 1, None, None) == bad
    assert lib.it_rope_positions(None, None, _lib.IT_F32, 1, 1, 1, 1, 8, 10000.0, 1, None, 0, 0, *none9[:5]) == bad
    assert b"null context" in lib.it_last_error()


def test_reference_bytes_hold_the_reference_values():
    """quant_ref.py packs rows, read back by the formula of the header."""
    x = np.random.default_rng(1).standard_normal((5, 80))
    c, s = qr.q4(x)
    b = qr.q4_bytes(c)
    words = b.view("<u4").reshape(5, 12)
    for d in range(80):
        j, t, e = d // 32, d % 32 // 8, d % 8
        u = (words[:, t * 3 + j] >> (4 * (e // 2) + 16 * (e % 2))) & 15
        assert np.array_equal(u.astype(int) - 8, c[:, d].astype(int))
    assert np.abs(c).max() == 7 and np.all(np.abs(qr.q4_values(x) - x) <= 0.5 * np.repeat(s, 32, -1)[:, :80] * 1.0000001)


# ------------------------------------------------------------------------------------------------ sizes of 2^31 and more
def shapeless(*shape, precision=BF16):
    """A tensor of this shape without memory."""
    return Tensor(torch.empty(shape, dtype=torch.float32 if precision is FP32 else torch.bfloat16, device="meta"), list(shape), precision)


def test_the_native_path_takes_sizes_below_2_31_only():
    for shape, ok in (((1, 2 ** 31 - 1, 1, 2), True), ((1, 2 ** 31, 1, 2), False), ((1, 2 ** 32 + 5, 1, 2), False), ((2 ** 32, 8), False), ((3, 0, 2 ** 40), False),
                      ((), True), ((0,), True)):
        assert ops._host_ops.fits(torch.empty(shape, dtype=torch.bfloat16, device="meta")) is ok, shape
    assert ops._host_ops.fits(None) is False


FAR = 2 ** 32 + 5


def with_lse(o, *shape):
    o.lse = shapeless(*shape, precision=FP32)
    return o


@pytest.mark.parametrize("call", [
    lambda: rope_positions(shapeless(1, FAR, 1, 2), None, torch.empty((1, FAR), dtype=torch.int32, device="meta")),
    lambda: rope_positions(shapeless(2 ** 32, 1, 1, 2), shapeless(2 ** 32, 1, 1, 2), torch.empty((2 ** 32, 1), dtype=torch.int32, device="meta")),
    lambda: ops.rope(shapeless(1, FAR, 1, 2)),
    lambda: ops.rope_qk(shapeless(1, FAR, 1, 2), shapeless(1, FAR, 1, 2)),
    lambda: ops.flash_attention(*[shapeless(1, 1, FAR, 1)] * 3, True),
    lambda: ops.attention(*[shapeless(1, FAR, 1, 1)] * 3, True),
    lambda: ops.attention(shapeless(1, 4, 1, 1), *[shapeless(1, FAR, 1, 1)] * 2, False),
    lambda: ops.attention_backward(*[shapeless(1, FAR, 1, 1)] * 4, with_lse(shapeless(1, FAR, 1, 1), 1, 1, FAR)),
    lambda: ops.attention_gqa(shapeless(FAR, 1, 2, 1), *[shapeless(FAR, 1, 1, 1)] * 2),
    lambda: ops.attention_gqa_backward(shapeless(FAR, 1, 2, 1), shapeless(FAR, 1, 2, 1), *[shapeless(FAR, 1, 1, 1)] * 2,
                                       with_lse(shapeless(FAR, 1, 2, 1), FAR, 2, 1)),
    lambda: ops.attention_backward_recompute(*[shapeless(1, 1, FAR, 1)] * 4),
    lambda: ops.attention_decode(shapeless(1, 1, 8), *[shapeless(1, FAR, 1, 8)] * 2, 5),
    lambda: ops.attention_packed(shapeless(1, FAR, 3), 1, 1, 1),
    lambda: ops.attention_packed_backward(shapeless(1, FAR, 1, 1), shapeless(1, FAR, 3), with_lse(shapeless(1, FAR, 1, 1), 1, 1, FAR), 1, 1, 1),
    lambda: ops.linear_forward(shapeless(FAR, 8), shapeless(8, 8)),
    lambda: ops.linear_backward(shapeless(FAR, 8), shapeless(FAR, 8), shapeless(8, 8)),
    lambda: ops.qkv_rope_forward(shapeless(1, FAR, 8), shapeless(6, 8), 1, 1, 2),
    lambda: quantize_rows(shapeless(FAR, 16)),
])
def test_sizes_that_32_bits_would_cut_off_are_refused(call):
    with pytest.raises(AssertionError, match="below 2\\^31"):
        call()


# ------------------------------------------------------------------------------------------------ bases below 1
@pytest.mark.parametrize("base,D,sections,per_axis,refused", [
    (1e-20, 128, [64], 0, True), (1e-3, 128, [64], 0, True), (5.5e-3, 4, [2], 0, False), (1e-7, 4, [2], 0, True), (1e-38, 2, [1], 0, False),
    (1e-3, 128, [32, 30, 2], 1, True), (1e-20, 12, [1, 5], 1, True), (1e-20, 6, [1, 1, 1], 1, False), (2e-3, 128, [64], 0, False), (0.0, 8, [4], 0, True),
])
def test_bases_whose_frequencies_leave_the_reduction_are_refused(base, D, sections, per_axis, refused):
    """By the entry itself, with a context that it must not look at (or, with nothing to rotate, need not)."""
    lib, nothing = _lib.load(), ctypes.create_string_buffer(4096)
    tokens = 1 if refused else 0
    rc = lib.it_rope_positions(nothing, nothing, _lib.IT_F32, tokens, 1, 1, 0, D, base, len(sections), (ctypes.c_int32 * len(sections))(*sections), per_axis, 0,
                               nothing, nothing, None, nothing, None)
    assert rc == (_lib.IT_ERR_INVALID_ARG if refused else _lib.IT_OK)
    if refused:
        assert b"base" in lib.it_last_error()
