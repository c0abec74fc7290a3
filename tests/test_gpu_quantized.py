"""GPU parity of the quantised serving operators against their definitions in 64 bits (quant_ref.py).

What is held in 4 or 8 bits is compared bit for bit.  Other results: a rounding to bf16 is off by at most 2^-8 of the value, to
fp32 by 2^-24."""
import math

import numpy as np
import pytest

import quant_ref as qr
from irontensor_b200 import (Precision, QuantizedCache, QuantizedRows, Tensor, _lib, attention_decode_quantized, attention_gqa, kv_cache_append,
                             kv_cache_read, linear_int8_forward, quantize_rows, rope_positions, synth)

pytestmark = pytest.mark.gpu
FP32, BF16 = Precision.FP32, Precision.BF16


def ints(a):
    import torch
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def to_tensor(a, precision):
    a = np.ascontiguousarray(a, np.float32)
    make = Tensor.from_f32_slice if precision is FP32 else Tensor.from_f32_as_bf16
    return make(a.reshape(-1), list(a.shape))


def values(rng, shape, precision, scale=1.0):
    x = (rng.standard_normal(shape) * scale).astype(np.float32)
    return x if precision is FP32 else synth.round_bf16(x).reshape(shape)


def cache_of(k, v, max_len, junk=True):
    """A QuantizedCache [B, max_len] of rows k, v [B, L, Hkv, D] laid out by quant_ref.py; positions behind L hold all bits and NaN."""
    import torch
    B, L, Hkv, D = k.shape
    g = -(-D // 32)
    codes = torch.full((2, B, Hkv, max_len, 16 * g), 0xFF if junk else 0x88, dtype=torch.uint8, device="cuda")
    scales = torch.full((2, B, Hkv, max_len, g), math.nan if junk else 0.0, dtype=torch.bfloat16, device="cuda")
    for i, x in enumerate((k, v)):
        c, s = qr.q4(x.transpose(0, 2, 1, 3))
        codes[i, :, :, :L], scales[i, :, :, :L] = torch.from_numpy(qr.q4_bytes(c)).cuda(), torch.from_numpy(s).cuda()
    return QuantizedCache(codes, scales, D)


def host(cache):
    return cache.codes.cpu().numpy(), cache.scales.double().cpu().numpy()


# ------------------------------------------------------------------------------------------------ writing
def hard_rows(rng, shape, precision):
    """Values with ties, zeros, subnormal, huge and non-finite groups among ordinary ones."""
    x = values(rng, shape, precision)
    flat = x.reshape(-1, shape[-1])
    for r in range(flat.shape[0]):
        kind = r % 12
        if kind == 1:
            flat[r] = 0.0
        elif kind == 2:      # 14 steps: every half of a step is hit
            flat[r] = rng.integers(-14, 15, shape[-1]) * 2.0 ** int(rng.integers(-20, 20))
        elif kind == 3:
            flat[r] *= 2.0 ** -101
        elif kind == 4:
            flat[r] = np.sign(flat[r]) * 3.0e38
        elif kind == 5:
            flat[r, 0] = np.nan
        elif kind == 6:
            flat[r, -1] = -np.inf
        elif kind == 7:      # one large value
            flat[r, 3] = 1000.0
        elif kind == 8:
            flat[r] = rng.integers(-7, 8, shape[-1]) * 0.5
        elif kind == 9:
            flat[r] *= 2.0 ** -90
    return x if precision is FP32 else synth.round_bf16(x).reshape(shape)


@pytest.mark.parametrize("precision", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("B,T,Hkv,D,starts,counts", [
    (1, 1, 1, 8, [0], None), (3, 1, 2, 64, [0, 5, 19], None), (2, 7, 3, 128, [4, 0], None), (2, 7, 3, 80, [4, 0], [0, 7]),
    (9, 13, 1, 96, [0, 1, 2, 3, 4, 5, 6, 7, 0], [13, 0, 1, 2, 3, 12, 13, 5, 6]), (2, 20, 4, 32, [0, 0], [20, 19]), (1, 9, 2, 40, [11], None),
])
def test_append_writes_the_documented_bytes_and_nothing_else(it_ctx, precision, B, T, Hkv, D, starts, counts):
    import torch
    rng = np.random.default_rng(B * 100 + T + D)
    k, v = hard_rows(rng, (B, T, Hkv, D), precision), hard_rows(rng, (B, T, Hkv, D), precision)
    max_len, g = 20, -(-D // 32)
    codes = rng.integers(0, 256, (2, B, Hkv, max_len, 16 * g)).astype(np.uint8)
    scales = rng.integers(1, 100, (2, B, Hkv, max_len, g)).astype(np.float64)
    cache = QuantizedCache(torch.from_numpy(codes.copy()).cuda(), torch.from_numpy(scales).to(torch.bfloat16).cuda(), D)
    new = kv_cache_append(cache, to_tensor(k, precision), to_tensor(v, precision), ints(starts), None if counts is None else ints(counts))
    assert it_ctx.poll_status() == 0
    n = [T] * B if counts is None else counts
    assert new.tolist() == [a + b for a, b in zip(starts, n)]
    for i, x in enumerate((k, v)):
        c, s = qr.q4(x)
        bytes_ = qr.q4_bytes(c)
        for b in range(B):
            for t in range(n[b]):
                codes[i, b, :, starts[b] + t], scales[i, b, :, starts[b] + t] = bytes_[b, t], s[b, t]
    got_codes, got_scales = host(cache)
    assert np.array_equal(got_scales, scales, equal_nan=True)
    assert np.array_equal(got_codes, codes)


@pytest.mark.parametrize("precision", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("B,T,Hkv,D", [(16, 1000, 8, 128), (2, 5000, 40, 24)])
def test_append_of_many_tokens_padded_to_one_length(it_ctx, precision, B, T, Hkv, D):
    """A CTA goes on to other tokens, of sequences of which each ends somewhere else."""
    rng = np.random.default_rng(55)
    k, v = hard_rows(rng, (B, T, Hkv, D), precision), hard_rows(rng, (B, T, Hkv, D), precision)
    counts = rng.integers(0, T + 1, B)
    counts[0], starts = T, rng.integers(0, 4, B)
    cache = QuantizedCache.zeros(B, T + 4, Hkv, D)
    new = kv_cache_append(cache, to_tensor(k, precision), to_tensor(v, precision), ints(starts), ints(counts))
    assert it_ctx.poll_status() == 0 and new.tolist() == (starts + counts).tolist()
    got_codes, got_scales = host(cache)
    for i, x in enumerate((k, v)):
        c, s = qr.q4(x)
        bytes_ = qr.q4_bytes(c)
        for b in range(B):
            there = slice(starts[b], starts[b] + counts[b])
            assert np.array_equal(got_scales[i, b, :, there], s[b, :counts[b]].swapaxes(0, 1), equal_nan=True)
            assert np.array_equal(got_codes[i, b, :, there], bytes_[b, :counts[b]].swapaxes(0, 1))
            got_codes[i, b, :, there], got_scales[i, b, :, there] = 0x88, 0
    assert np.all(got_codes == 0x88) and np.all(got_scales == 0)


def every_bf16_quotient(cols, exponents):
    """Rows of `cols` whose largest value goes through all 128 mantissas, each beside all mantissas of the given exponents below it."""
    x = np.concatenate([np.ldexp(np.arange(128, 256), e) for e in exponents])
    rows = []
    for largest in range(128, 256):
        below = x[x <= largest]
        below = np.concatenate([below, np.zeros(-len(below) % (cols - 1))]).reshape(-1, cols - 1)
        rows.append(np.concatenate([np.full((len(below), 1), largest), below], 1))
    x = np.concatenate(rows)
    x[:, 1::2] *= -1
    return x


def test_every_quotient_of_bf16_values(it_ctx):
    """Ties and all: what decides between two whole numbers is exact."""
    x = np.ldexp(every_bf16_quotient(32, range(-7, 1)), -7)
    L = len(x)
    t = to_tensor(x.reshape(1, L, 1, 32), BF16)
    cache = QuantizedCache.zeros(1, L, 1, 32)
    kv_cache_append(cache, t, t, ints([0]))
    rows = every_bf16_quotient(1168, range(-9, 1))
    got = quantize_rows(to_tensor(rows, BF16))
    assert it_ctx.poll_status() == 0
    c, s = qr.q4(x.reshape(1, L, 1, 32))
    codes, scales = host(cache)
    assert np.array_equal(scales[0, 0, 0], s[0, :, 0]) and np.array_equal(codes[0, 0, 0], qr.q4_bytes(c)[0, :, 0])
    c, s = qr.q8(rows)
    assert np.array_equal(got.scales.double().cpu().numpy(), s) and np.array_equal(got.codes.cpu().numpy(), c.astype(np.int8))


def test_append_beyond_the_cache_is_dropped_and_reported(it_ctx):
    """max_len 6: sequence 0 has room for one of two tokens, sequence 1 starts before the cache, sequence 2 behind it, 3 fits."""
    import torch
    rng = np.random.default_rng(5)
    k, v = values(rng, (4, 2, 1, 32), FP32), values(rng, (4, 2, 1, 32), FP32)
    cache = QuantizedCache.zeros(4, 6, 1, 32)
    new = kv_cache_append(cache, to_tensor(k, FP32), to_tensor(v, FP32), ints([5, -1, 9, 4]))
    torch.cuda.synchronize()
    with pytest.raises(_lib.ITError, match="length lay outside") as e:
        it_ctx.poll_status()
    assert e.value.status == _lib.IT_ERR_INVALID_ARG
    assert it_ctx.poll_status() == 0 and new.tolist() == [6, 1, 6, 6]
    _, scales = host(cache)
    written = scales[0, :, 0, :, 0] > 0
    assert written.tolist() == [[False] * 5 + [True], [True] + [False] * 5, [False] * 6, [False] * 4 + [True] * 2]
    # counts outside 0..tokens
    new = kv_cache_append(cache, to_tensor(k, FP32), to_tensor(v, FP32), ints([0, 0, 0, 0]), ints([-3, 5, 2, 0]))
    torch.cuda.synchronize()
    with pytest.raises(_lib.ITError, match="length lay outside"):
        it_ctx.poll_status()
    assert new.tolist() == [0, 2, 2, 0]


def test_a_full_cache_stops_nothing_else(it_ctx):
    """Launches between the one that found a sequence outside its cache and the report of it do their work: whole tiles of 8-bit
    products, attention, and the cache itself."""
    import torch
    from irontensor_b200 import attention
    rng = np.random.default_rng(51)
    x, w = (quantize_rows(to_tensor(values(rng, s, BF16), BF16)) for s in ((200, 256), (136, 256)))
    a = [to_tensor(values(rng, (1, 256, 2, 64), BF16), BF16) for _ in range(3)]
    q, k = to_tensor(values(rng, (2, 4, 64), BF16), BF16), to_tensor(values(rng, (2, 3, 2, 64), BF16), BF16)
    cache = QuantizedCache.zeros(2, 4, 2, 64)
    run = lambda n: [t.torch().clone() for t in (linear_int8_forward(x, w, FP32), attention(*a, True), attention_decode_quantized(q, cache, n))]
    kv_cache_append(cache, k, k, ints([0, 0]))
    want = run(ints([3, 3]))
    torch.cuda.synchronize()
    assert it_ctx.poll_status() == 0
    n = kv_cache_append(cache, k, k, ints([3, 4]), ints([0, 1]))     # sequence 1 is full
    got = run(torch.minimum(n, ints([3, 3])))
    torch.cuda.synchronize()
    with pytest.raises(_lib.ITError, match="length lay outside"):
        it_ctx.poll_status()
    assert it_ctx.poll_status() == 0 and n.tolist() == [3, 4]
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_a_full_cache_and_a_wait_that_ran_out_are_both_reported(it_ctx):
    """One poll each, the wait (20 ms on a barrier nothing arrives on) first; until then every synchronisation reports one of them."""
    import ctypes
    import torch
    from irontensor_b200 import CommandBatch
    k, cache = Tensor.zeros([1, 2, 1, 32], BF16), QuantizedCache.zeros(1, 3, 1, 32)
    assert kv_cache_append(cache, k, k, ints([2])).tolist() == [3]
    torch.cuda.synchronize()
    with pytest.raises(_lib.ITError, match="length lay outside") as e:    # of another stream
        with torch.cuda.stream(torch.cuda.Stream()):
            CommandBatch.sync()
    assert e.value.status == _lib.IT_ERR_INVALID_ARG
    _lib.check(it_ctx.lib.it_selftest_wait_timeout(it_ctx.handle, it_ctx.stream(), 20))
    with pytest.raises(_lib.ITError, match="ran out"):
        CommandBatch.sync()
    for text, word in (("ran out", 6), ("length lay outside", 7)):
        st = ctypes.c_int32()
        with pytest.raises(_lib.ITError, match=text):
            _lib.check(it_ctx.lib.it_attention_status_poll(it_ctx.handle, it_ctx.stream(), ctypes.byref(st)))
        assert st.value == word
    assert it_ctx.poll_status() == 0
    CommandBatch.sync()


@pytest.mark.parametrize("precision", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("B,L,Hkv,D,count,starts,lengths", [
    (1, 1, 1, 8, 1, None, None), (2, 9, 3, 64, 9, None, None), (3, 17, 2, 80, 5, [0, 12, 16], None), (2, 9, 1, 128, 12, [-2, 5], [9, 7]),
    (2, 11, 4, 96, 11, None, [0, 20]), (1, 40, 2, 40, 33, [3], [36]),
])
def test_read_gives_the_held_values_and_zeros_outside(it_ctx, precision, B, L, Hkv, D, count, starts, lengths):
    rng = np.random.default_rng(L + D)
    k, v = values(rng, (B, L, Hkv, D), FP32), values(rng, (B, L, Hkv, D), FP32)
    cache = cache_of(k, v, L, junk=False)
    got = kv_cache_read(cache, count, None if starts is None else ints(starts), None if lengths is None else ints(lengths), precision)
    assert it_ctx.poll_status() == 0
    for x, y in zip((k, v), got):
        held, want = qr.q4_values(x), np.zeros((B, count, Hkv, D))
        for b in range(B):
            for t in range(count):
                p = (starts[b] if starts else 0) + t
                if 0 <= p < min(L, lengths[b] if lengths else L):
                    want[b, t] = held[b, p]
        assert y.precision() is precision and np.array_equal(y.to_f32_host(), want)


@pytest.mark.parametrize("precision", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("B,T,Hkv", [(2, 1, 2), (3, 5, 2), (2, 9, 3), (7, 2, 5)])
@pytest.mark.parametrize("D", [8, 24, 40, 56, 72, 88, 104, 120, 16, 128])
def test_read_of_few_tokens_writes_every_value_of_every_head(it_ctx, precision, D, B, T, Hkv):
    """Several heads share a CTA, and with an odd number of 8 columns a head's last ones have no neighbour: by the C entry into memory
    that is NaN beforehand, with as much behind it that stays so."""
    import torch
    rng = np.random.default_rng(D + T)
    k, v = values(rng, (B, T, Hkv, D), FP32), values(rng, (B, T, Hkv, D), FP32)
    cache, n = cache_of(k, v, T + 3), B * T * Hkv * D
    out = torch.full((2, 2 * n), math.nan, dtype=torch.float32 if precision is FP32 else torch.bfloat16, device="cuda")
    _lib.check(it_ctx.lib.it_kv_cache_q4_read(it_ctx.handle, it_ctx.stream(), _lib.IT_F32 if precision is FP32 else _lib.IT_BF16, B, T, Hkv, D, T + 3,
                                              *cache._halves(), None, None, out[0].data_ptr(), out[1].data_ptr()))
    assert it_ctx.poll_status() == 0
    for x, y in zip((k, v), out.double().cpu().numpy()):
        assert np.array_equal(y[:n].reshape(B, T, Hkv, D), qr.q4_values(x)) and np.isnan(y[n:]).all()


# ------------------------------------------------------------------------------------------------ attention
def check_decode(it_ctx, precision, q, k, v, lengths, max_len, bound=1.0):
    """Error against 64 bits on the held values.  A score is a sum of D exact products in fp32, off by at most 2^-20 of the products'
    magnitudes (16 partial sums of at most 2^-23 each, with room for two); that, through exp, is a relative error of p.  P has 16
    bits (bf16 q) or 24.  With A = the largest |v|: 2 x 2^-20 x (sum of |q k| / sqrt(D), below 32 here) x A = 2^-14 A, plus 2^-16 A for P
    and less than 2^-16 A for sums of at most 40 terms a warp and the merges; and the rounding of the result."""
    cache = cache_of(k, v, max_len)
    o = attention_decode_quantized(to_tensor(q, precision), cache, ints(lengths))
    assert it_ctx.poll_status() == 0
    want, lse = qr.decode(q, qr.q4_values(k), qr.q4_values(v), lengths)
    got, got_lse = o.to_f32_host(), o.lse.to_f32_host()
    assert o.precision() is precision and np.isfinite(got).all()
    A = np.abs(qr.q4_values(v)).max()
    limit = (2.0 ** -14 + 2.0 ** -16) * A * bound + (2.0 ** -8 if precision is BF16 else 2.0 ** -24) * np.abs(want)
    assert np.all(np.abs(got - want) <= limit), np.abs(got - want).max()
    empty = np.asarray(lengths) == 0
    assert np.all(got[empty] == 0) and np.all(got_lse[empty] == -np.inf)
    assert np.all(np.abs(got_lse[~empty] - lse[~empty]) <= 2.0 ** -15 * bound + 2.0 ** -23 * np.abs(lse[~empty]))
    return o, cache


@pytest.mark.parametrize("precision", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("H,Hkv,D,lengths,max_len", [
    (1, 1, 8, [1], 1), (4, 4, 64, [100], 100), (4, 1, 128, [0, 1, 2, 31, 32, 33, 255, 256, 257], 300), (8, 1, 96, [40, 7], 64),
    (7, 7, 32, [5, 300], 301), (12, 4, 80, [600, 0, 64], 640), (16, 1, 64, [777], 1024), (24, 2, 128, [90, 1000], 1000), (2, 2, 120, [513], 700),
    (40, 2, 16, [129, 3], 130), (3, 1, 128, [4001], 8192), (6, 2, 56, [1500, 20, 700], 2048),
])
def test_decode_at_every_sequences_own_length(it_ctx, precision, H, Hkv, D, lengths, max_len):
    rng = np.random.default_rng(D + H + max_len)
    B, L = len(lengths), max(lengths)
    q = values(rng, (B, H, D), precision)
    k, v = values(rng, (B, L, Hkv, D), FP32), values(rng, (B, L, Hkv, D), FP32)
    check_decode(it_ctx, precision, q, k, v, lengths, max_len)


@pytest.mark.parametrize("precision", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("H,Hkv,D,max_len,lengths", [
    (8, 2, 128, 1 << 17, [3000, 1, 0, 900, 33]), (12, 1, 64, 1 << 18, [5000, 0, 31]), (4, 4, 32, 1 << 17, [2050, 700]), (6, 2, 96, 1 << 17, [0, 1500, 1]),
    (32, 2, 80, 1 << 17, [0, 2000]), (5, 1, 16, 1 << 19, [1025]), (2, 2, 48, 1 << 18, [0, 0]),
])
def test_decode_in_even_shares(it_ctx, precision, H, Hkv, D, max_len, lengths):
    """Room for long sequences: the persistent launch, whose CTAs share out what the lengths turn out to be."""
    rng = np.random.default_rng(D + H)
    B, L = len(lengths), max(max(lengths), 1)
    q = values(rng, (B, H, D), precision)
    k, v = values(rng, (B, L, Hkv, D), FP32), values(rng, (B, L, Hkv, D), FP32)
    check_decode(it_ctx, precision, q, k, v, lengths, max_len)


@pytest.mark.parametrize("precision", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("H,Hkv", [(3, 3), (4, 2), (3, 1), (8, 2), (5, 1), (12, 2), (8, 1), (9, 1), (32, 2), (17, 1)])
@pytest.mark.parametrize("D", [32, 64, 96, 128, 72])
def test_decode_of_groups_of_every_kind(it_ctx, precision, H, Hkv, D):
    """Up to four heads of a K/V head, up to eight, up to sixteen and more, for each number of groups of 32 columns; by a cluster and in
    even shares."""
    rng = np.random.default_rng(100 * D + H)
    lengths = [130, 0, 1, 700]
    q = values(rng, (4, H, D), precision)
    k, v = values(rng, (4, 700, Hkv, D), FP32), values(rng, (4, 700, Hkv, D), FP32)
    check_decode(it_ctx, precision, q, k, v, lengths, 700)
    check_decode(it_ctx, precision, q, k, v, lengths, 1 << 17)


def test_decode_of_the_most_rows(it_ctx):
    rng = np.random.default_rng(53)
    B, H, D = 4369, 15, 8
    q, k, v = values(rng, (B, H, D), BF16), values(rng, (B, 2, 1, D), FP32), values(rng, (B, 2, 1, D), FP32)
    check_decode(it_ctx, BF16, q, k, v, rng.integers(0, 3, B), 2)


def test_decode_by_two_graphs_at_once(it_ctx):
    """Captured on one stream, replayed on two: a graph's scratch memory is its own."""
    import torch
    rng = np.random.default_rng(54)
    cases = []
    for lengths in ([2900, 40], [1500, 2000]):
        q, k, v = values(rng, (2, 8, 64), BF16), values(rng, (2, 3000, 2, 64), FP32), values(rng, (2, 3000, 2, 64), FP32)
        want, cache = check_decode(it_ctx, BF16, q, k, v, lengths, 1 << 17)
        cases.append((want.torch().clone(), to_tensor(q, BF16), cache, ints(lengths)))
    side, graphs, outs = torch.cuda.Stream(), [], []
    torch.cuda.synchronize()
    for _, q, cache, n in cases:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=side):
            outs.append([attention_decode_quantized(q, cache, n) for _ in range(10)])
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert it_ctx.poll_status() == 0
    for (want, *_), got in zip(cases, outs):
        assert all(torch.equal(x.torch(), want) for x in got)
    del graphs, g


def test_decode_of_many_sequences_in_even_shares(it_ctx):
    """More sequences than a CTA has threads."""
    rng = np.random.default_rng(19)
    B, H, D = 700, 2, 64
    lengths = rng.integers(0, 70, B)
    lengths[[0, 255, 256, 699]] = [0, 69, 1, 40]
    q, k, v = values(rng, (B, H, D), BF16), values(rng, (B, 69, 1, D), FP32), values(rng, (B, 69, 1, D), FP32)
    check_decode(it_ctx, BF16, q, k, v, lengths, 2048)
    check_decode(it_ctx, BF16, q, k, v, np.zeros(B, int), 2048)


def launches_of(it_ctx, call):
    """2 for even shares (the attention and its merge), 1 for clusters."""
    before = it_ctx.launch_count()
    call()
    return it_ctx.launch_count() - before


@pytest.mark.parametrize("B", [127, 128, 129, 255, 256, 257, 600])
@pytest.mark.parametrize("precision,H,Hkv,D", [(BF16, 2, 1, 32), (BF16, 16, 2, 32), (BF16, 16, 1, 128), (FP32, 2, 1, 128), (FP32, 8, 1, 104)])
def test_even_shares_of_more_sequences_than_a_cta_has_threads(it_ctx, precision, H, Hkv, D, B):
    """The work in front of each sequence is added up 128 or 256 sequences at a time, in two passes: with empty sequences on both sides of
    every border, with only the last one not empty, and with nothing but empty ones."""
    rng = np.random.default_rng(B + D)
    lengths = rng.integers(0, 100, B)
    for border in (128, 256, 512):
        lengths[border - 2:border + 1] = 0
    lengths[[1, B - 1]] = [99, 33]
    q = values(rng, (B, H, D), precision)
    k, v = values(rng, (B, 99, Hkv, D), FP32), values(rng, (B, 99, Hkv, D), FP32)
    for n in (lengths, lengths * (np.arange(B) == B - 1), np.zeros(B, int)):
        assert launches_of(it_ctx, lambda: check_decode(it_ctx, precision, q, k, v, n, 1 << 15)) == 2


@pytest.mark.parametrize("precision", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("B,H,Hkv,D,max_len", [
    (5, 8, 2, 128, 1 << 17), (3, 12, 1, 64, 1 << 18), (2, 4, 4, 32, 1 << 17), (3, 6, 2, 96, 1 << 17), (2, 32, 2, 80, 1 << 17), (1, 5, 1, 16, 1 << 19),
    (2, 2, 2, 48, 1 << 18), (4, 3, 3, 32, 1 << 17), (4, 3, 1, 64, 1 << 17), (4, 8, 1, 72, 1 << 17), (4, 32, 2, 128, 1 << 17), (4, 17, 1, 96, 1 << 17),
    (2, 8, 2, 64, 1 << 17), (1, 6, 1, 128, 1 << 18), (4, 4, 4, 40, 1 << 18),
])
def test_caches_with_that_much_room_are_attended_to_in_even_shares(it_ctx, precision, B, H, Hkv, D, max_len):
    """The shapes by which the tests above and below mean to reach the persistent launch."""
    cache, q = QuantizedCache.zeros(B, max_len, Hkv, D), Tensor.zeros([B, H, D], precision)
    assert launches_of(it_ctx, lambda: attention_decode_quantized(q, cache, ints([1] * B))) == 2
    small = QuantizedCache.zeros(B, 256, Hkv, D)
    assert launches_of(it_ctx, lambda: attention_decode_quantized(q, small, ints([1] * B))) == 1
    assert it_ctx.poll_status() == 0


@pytest.mark.parametrize("precision", [BF16, FP32], ids=["bf16", "fp32"])
def test_decode_of_scales_far_apart(it_ctx, precision):
    """Values over many powers of two: a scale is taken as it is, and a group of zeros stays zero."""
    rng = np.random.default_rng(11)
    H, Hkv, D, lengths = 8, 2, 96, [200, 37]
    q = values(rng, (2, H, D), precision)
    k, v = values(rng, (2, 200, Hkv, D), FP32), values(rng, (2, 200, Hkv, D), FP32)
    k *= 2.0 ** rng.integers(-60, 1, (2, 200, Hkv, 1))
    v *= 2.0 ** rng.integers(-100, 1, (2, 200, Hkv, 1))
    k[:, 5], v[:, 6, :, 32:64] = 0.0, 0.0
    check_decode(it_ctx, precision, q, k, v, lengths, 256)
    v *= 2.0 ** 100
    check_decode(it_ctx, precision, q, k, v, lengths, 256)


@pytest.mark.parametrize("precision", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("H,Hkv,D,L,max_len", [(8, 2, 128, 300, 300), (8, 1, 64, 100, 128), (16, 1, 96, 77, 100), (4, 4, 40, 65, 1 << 18), (6, 1, 128, 200, 1 << 18)])
def test_decode_of_keys_with_one_large_channel(it_ctx, precision, H, Hkv, D, L, max_len):
    """Every group of 32 columns has one value some hundred times the others, whose codes are then 0, in a column where q is small; the
    rest of q is large and of one sign.  A score is as good as the few products that it is a sum of, whatever the sum of q: off by
    E = 2^-20 of the products' magnitudes at most (as check_decode has it), a p by 2 E of itself, and so the result by 2 E A
    beside what check_decode counts."""
    rng = np.random.default_rng(62)
    q = np.abs(values(rng, (1, H, D), precision)) + 1
    q[..., ::4] *= 2.0 ** -9
    q = q if precision is FP32 else synth.round_bf16(q.astype(np.float32)).reshape(q.shape)
    k, v = values(rng, (1, L, Hkv, D), FP32), values(rng, (1, L, Hkv, D), FP32)
    for j in range(0, D, 32):
        at = j + 4 * rng.integers(0, min(32, D - j) // 4, (L, Hkv))
        k[0, np.arange(L)[:, None], np.arange(Hkv), at] = 1000.0 + 10 * rng.standard_normal((L, Hkv))
    o = attention_decode_quantized(to_tensor(q, precision), cache_of(k, v, max_len), ints([L]))
    assert it_ctx.poll_status() == 0
    hk, hv = qr.q4_values(k), qr.q4_values(v)
    want, lse = qr.decode(q, hk, hv, [L])
    products = np.einsum("hd,lhd->hl", np.abs(q[0]).astype(np.float64), np.repeat(np.abs(hk[0]), H // Hkv, 1)).max(1) / math.sqrt(D)
    E, A = 2.0 ** -20 * products[None, :], np.abs(hv).max()
    assert np.all(np.abs(o.lse.to_f32_host() - lse) <= E + 2.0 ** -15 + 2.0 ** -23 * np.abs(lse)), np.abs(o.lse.to_f32_host() - lse).max()
    limit = (2 * E[..., None] + 2.0 ** -15) * A + (2.0 ** -8 if precision is BF16 else 2.0 ** -24) * np.abs(want)
    assert np.all(np.abs(o.to_f32_host() - want) <= limit)


def test_decode_with_one_overwhelming_key(it_ctx):
    """The maximum arrives late and dwarfs what was summed before it: the result is that key's value alone."""
    rng = np.random.default_rng(12)
    q, k, v = values(rng, (1, 4, 64), FP32), values(rng, (1, 900, 1, 64), FP32), values(rng, (1, 900, 1, 64), FP32)
    q[:] = np.abs(q[:, :1])
    k[:, 700] = 40.0 * np.sign(q[0, 0])
    o, _ = check_decode(it_ctx, FP32, q, k, v, [900], 900, bound=64.0)   # scores up to 64 times as large
    assert np.allclose(o.to_f32_host()[0], qr.q4_values(v)[0, 700, 0], rtol=1e-6, atol=1e-6)


def test_non_finite_keys_and_values_reach_their_sequence_only(it_ctx):
    import torch
    rng = np.random.default_rng(13)
    q, k, v = values(rng, (3, 4, 64), BF16), values(rng, (3, 50, 2, 64), BF16), values(rng, (3, 50, 2, 64), BF16)
    k[0, 10, 0, 3], v[1, 20, 1, 40] = np.nan, np.inf
    cache = QuantizedCache.zeros(3, 64, 2, 64)
    n = kv_cache_append(cache, to_tensor(k, BF16), to_tensor(v, BF16), torch.zeros(3, dtype=torch.int32, device="cuda"))
    o = attention_decode_quantized(to_tensor(q, BF16), cache, n).to_f32_host()
    assert it_ctx.poll_status() == 0
    assert np.isnan(o[0, :2]).all() and np.isfinite(o[0, 2:]).all()            # the heads that read K/V head 0
    assert np.isfinite(o[1, :2]).all() and np.isnan(o[1, 2:, 32:]).all() and np.isfinite(o[1, 2:, :32]).all()   # the group of 32
    assert np.isfinite(o[2]).all()


def test_decode_of_lengths_outside_the_cache(it_ctx):
    """Taken as the nearest length inside, and reported."""
    rng = np.random.default_rng(14)
    q, k, v = values(rng, (2, 2, 32), FP32), values(rng, (2, 70, 1, 32), FP32), values(rng, (2, 70, 1, 32), FP32)
    cache = cache_of(k, v, 70)
    import torch
    o = attention_decode_quantized(to_tensor(q, FP32), cache, ints([1000, -7]))
    got = o.torch().cpu().numpy()
    torch.cuda.synchronize()
    with pytest.raises(_lib.ITError, match="length lay outside"):
        it_ctx.poll_status()
    assert it_ctx.poll_status() == 0
    want, _ = qr.decode(q, qr.q4_values(k), qr.q4_values(v), [70, 0])
    assert np.abs(got - want).max() <= 2.0 ** -13 * np.abs(v).max() and np.all(got[1] == 0)


def test_decode_repeats_bit_for_bit_and_on_other_streams(it_ctx):
    import torch
    rng = np.random.default_rng(15)
    q, k, v = values(rng, (5, 16, 128), BF16), values(rng, (5, 3000, 2, 128), FP32), values(rng, (5, 3000, 2, 128), FP32)
    lengths = [3000, 1, 0, 2999, 1024]
    o, cache = check_decode(it_ctx, BF16, q, k, v, lengths, 4096)
    n, tq = ints(lengths), to_tensor(q, BF16)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(attention_decode_quantized(tq, cache, n))
    torch.cuda.synchronize()
    for x in outs:
        assert torch.equal(x.torch(), o.torch()) and torch.equal(x.lse.torch(), o.lse.torch())


def test_cache_offsets_beyond_32_bits(it_ctx):
    """140 million rows of 64 bytes: the last sequence's and head's rows lie past 2^32 bytes and 2^31 words."""
    import torch
    rng = np.random.default_rng(16)
    B, Hkv, max_len, D, T = 34, 64, 65536, 128, 5
    cache = QuantizedCache(torch.empty((2, B, Hkv, max_len, 64), dtype=torch.uint8, device="cuda"),
                           torch.empty((2, B, Hkv, max_len, 4), dtype=torch.bfloat16, device="cuda"), D)
    assert cache.codes.numel() // 8 > 2 ** 31
    k, v, q = values(rng, (B, T, Hkv, D), BF16), values(rng, (B, T, Hkv, D), BF16), values(rng, (B, Hkv, D), BF16)
    starts = torch.zeros(B, dtype=torch.int32, device="cuda")
    n = kv_cache_append(cache, to_tensor(k, BF16), to_tensor(v, BF16), starts)
    kr, vr = kv_cache_read(cache, T)
    o = attention_decode_quantized(to_tensor(q, BF16), cache, n).to_f32_host()
    far = kv_cache_append(cache, to_tensor(k, BF16), to_tensor(v, BF16), starts + (max_len - T))
    kf, _ = kv_cache_read(cache, T, starts + (max_len - T))
    assert it_ctx.poll_status() == 0 and far.tolist() == [max_len] * B
    hk, hv = qr.q4_values(k), qr.q4_values(v)
    assert np.array_equal(kr.to_f32_host(), hk) and np.array_equal(vr.to_f32_host(), hv) and np.array_equal(kf.to_f32_host(), hk)
    want, _ = qr.decode(q[-1:], hk[-1:], hv[-1:], [T])
    assert np.all(np.abs(o[-1:] - want) <= 2.0 ** -13 * np.abs(hv).max() + 2.0 ** -8 * np.abs(want))


# ------------------------------------------------------------------------------------------------ rotary embedding
@pytest.mark.parametrize("precision", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("B,S,H,Hkv,D,sections,per_axis,base", [
    (1, 1, 1, 0, 2, [1], False, 10000.0), (3, 5, 4, 2, 64, [32], False, 10000.0), (2, 33, 2, 1, 96, [20, 14, 14], False, 500000.0),
    (1, 70, 3, 3, 128, [0, 30, 34], True, 10000.0), (2, 7, 5, 1, 10, [2, 3], True, 100.0), (1, 300, 12, 4, 80, [10, 10, 10, 10], False, 10000.0),
    (40, 1, 32, 8, 128, [64], False, 10000.0),
])
def test_rope_at_given_positions(it_ctx, precision, B, S, H, Hkv, D, sections, per_axis, base):
    """A sine of an angle rounded to 32 bits after whole turns are taken off is off by 2^-23 (angle) and 2^-23 (the function), so a
    result by 2^-22 (|x0| + |x1|) and two roundings."""
    rng = np.random.default_rng(D + S)
    q, k = values(rng, (B, S, H, D), precision), values(rng, (B, S, max(Hkv, 1), D), precision)
    positions = rng.integers(-2 ** 31, 2 ** 31 - 1, (len(sections), B, S)) if S % 2 else rng.integers(0, 200000, (len(sections), B, S))
    tq, tk = to_tensor(q, precision), to_tensor(k, precision)
    at = ints(positions if len(sections) > 1 else positions[0])
    for inverse in (False, True):
        got = rope_positions(tq, tk if Hkv else None, at, base, sections, per_axis, inverse)
        assert it_ctx.poll_status() == 0
        for x, y in zip((q, k), got if Hkv else (got,)):
            want = qr.rope(x, positions, float(np.float32(base)), sections, per_axis, inverse)
            size = np.repeat(np.abs(x[..., 0::2]) + np.abs(x[..., 1::2]), 2, -1)
            limit = 2.0 ** -21 * size + (2.0 ** -8 if precision is BF16 else 2.0 ** -24) * np.abs(want)
            assert np.all(np.abs(y.to_f32_host() - want) <= limit)


@pytest.mark.parametrize("base,D,sections,per_axis", [(0.5, 64, [32], False), (0.25, 16, [3, 5], True), (2.0 ** -9, 20, [10], False)])
def test_rope_with_a_base_below_one(it_ctx, base, D, sections, per_axis):
    """Frequencies above 1, at positions near enough for both sides' angles: below 2^20 x 2^9, which 64 bits hold to 2^-24 (and the
    powers, off by 2^-52 of themselves on either side, to 2^-22), so a result is off by 2^-20 (|x0| + |x1|) and its roundings."""
    rng = np.random.default_rng(61)
    x, at = values(rng, (2, 50, 3, D), FP32), rng.integers(-2 ** 20, 2 ** 20, (len(sections), 2, 50))
    got = rope_positions(to_tensor(x, FP32), None, ints(at if len(sections) > 1 else at[0]), base, sections, per_axis)
    want = qr.rope(x, at, base, sections, per_axis)
    size = np.repeat(np.abs(x[..., 0::2]) + np.abs(x[..., 1::2]), 2, -1)
    assert it_ctx.poll_status() == 0 and np.all(np.abs(got.to_f32_host() - want) <= 2.0 ** -20 * size + 2.0 ** -24 * np.abs(want))
    with pytest.raises(_lib.ITError, match="frequencies above 512") as e:
        rope_positions(to_tensor(x, FP32), None, ints(at if len(sections) > 1 else at[0]), 1e-20, sections, per_axis)
    assert e.value.status == _lib.IT_ERR_INVALID_ARG


def test_rope_inverse_is_the_gradient(it_ctx):
    """Against differences: the rotation is linear, so with L = sum(g * rope(x)), dL/dx . d = L(x + d) - L(x) but for rounding."""
    rng = np.random.default_rng(21)
    x, g, d = (values(rng, (2, 9, 3, 64), FP32) for _ in range(3))
    at = ints(rng.integers(0, 5000, (2, 9)))
    turned = [rope_positions(to_tensor(t, FP32), None, at).to_f32_host().astype(np.float64) for t in (x + d, x)]
    grad = rope_positions(to_tensor(g, FP32), None, at, inverse=True).to_f32_host().astype(np.float64)
    diff = (g * (turned[0] - turned[1])).sum()
    assert abs((grad * d).sum() - diff) <= 2.0 ** -20 * (np.abs(g) * (np.abs(x) + np.abs(d)) * 4).sum()


def test_rope_of_odd_addresses(it_ctx):
    """Rows that start between 16-byte boundaries go in pairs."""
    import torch
    rng = np.random.default_rng(22)
    x = values(rng, (1, 6, 2, 64), BF16)
    flat = torch.zeros(x.size + 2, dtype=torch.bfloat16, device="cuda")
    flat[2:] = torch.from_numpy(x.reshape(-1)).to(torch.bfloat16).cuda()
    at = ints(np.arange(6)[None])
    a = rope_positions(Tensor(flat[2:], list(x.shape), BF16), None, at)
    b = rope_positions(to_tensor(x, BF16), None, at)
    assert it_ctx.poll_status() == 0 and torch.equal(a.torch(), b.torch())


@pytest.mark.parametrize("precision,D,offset", [(BF16, 64, 0), (FP32, 96, 0), (BF16, 20, 0), (BF16, 64, 2)])
def test_rope_in_place(it_ctx, precision, D, offset):
    """By the C entry, whose results may lie where q and k are."""
    import ctypes
    import torch
    rng = np.random.default_rng(52)
    q, k = to_tensor(values(rng, (2, 37, 5, D), precision), precision), to_tensor(values(rng, (2, 37, 3, D), precision), precision)
    at = ints(rng.integers(0, 5000, (2, 37)))
    want = [t.torch().flatten() for t in rope_positions(q, k, at)]
    def shifted(t):
        return torch.cat([torch.zeros(offset, dtype=t.dtype, device="cuda"), t.flatten()])[offset:]
    tq, tk = shifted(q.torch()), shifted(k.torch())
    _lib.check(it_ctx.lib.it_rope_positions(it_ctx.handle, it_ctx.stream(), _lib.IT_BF16 if precision is BF16 else _lib.IT_F32, 2, 37, 5, 3, D, 10000.0, 1,
                                            (ctypes.c_int32 * 1)(D // 2), 0, 0, at.data_ptr(), tq.data_ptr(), tk.data_ptr(), tq.data_ptr(), tk.data_ptr()))
    assert it_ctx.poll_status() == 0 and torch.equal(tq, want[0]) and torch.equal(tk, want[1])


def test_sizes_that_32_bits_would_cut_off_are_refused(it_ctx):
    """In front of any allocation of results: a prompt of 2^31 tokens in two columns."""
    import torch
    from irontensor_b200 import rope, rope_qk
    S = 2 ** 31
    x = Tensor(torch.empty((1, S, 1, 2), dtype=torch.bfloat16, device="cuda"), [1, S, 1, 2], BF16)
    at = torch.empty((1, S), dtype=torch.int32, device="cuda")
    before = it_ctx.launch_count()
    for call in (lambda: rope_positions(x, None, at), lambda: rope_positions(x, x, at), lambda: rope(x), lambda: rope_qk(x, x)):
        with pytest.raises(AssertionError, match="below 2\\^31"):
            call()
    assert it_ctx.launch_count() == before and it_ctx.poll_status() == 0
    del x, at
    torch.cuda.empty_cache()


# ------------------------------------------------------------------------------------------------ 8-bit projections
@pytest.mark.parametrize("precision", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("rows,cols", [(1, 16), (12, 48), (5, 2048), (3, 8192), (25, 8208), (2, 20000)])
def test_quantize_rows(it_ctx, precision, rows, cols):
    rng = np.random.default_rng(rows + cols)
    x = hard_rows(rng, (rows, cols), precision)
    if rows >= 12:   # ties of 127 steps
        x[2] = rng.integers(-254, 255, cols)
        x[2, 0] = 254
    got = quantize_rows(to_tensor(x, precision))
    assert it_ctx.poll_status() == 0
    c, s = qr.q8(x)
    assert np.array_equal(got.scales.double().cpu().numpy(), s, equal_nan=True)
    assert np.array_equal(got.codes.cpu().numpy(), c.astype(np.int8))


@pytest.mark.parametrize("precision", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("n,k,widths", [
    (1, 16, [8]), (3, 48, [24]), (8, 272, [120]), (9, 2048, [200]), (16, 80, [1000]), (17, 528, [16, 8, 16]), (31, 2048, [512, 64, 64]),
    (33, 144, [200]), (64, 4112, [520]), (130, 272, [9480]), (129, 128, [136, 128]), (700, 208, [4000, 0, 1000]), (2500, 144, [3080]), (300, 1040, [264]),
])
def test_linear_int8(it_ctx, precision, n, k, widths):
    """The integer sums are exact; they become fp32 (2^-24), are multiplied by the product of the scales (2^-24 and, with scales of
    more than 8 bits as here, 2^-24), and are stored."""
    import torch
    rng = np.random.default_rng(n + k)
    out = sum(widths)
    cx, cw = rng.integers(-127, 128, (n, k)).astype(np.int8), rng.integers(-127, 128, (out, k)).astype(np.int8)
    cx[0], cw[0] = 127, 127     # the largest sum
    sx, sw = rng.uniform(0.5, 2, n).astype(np.float32), rng.uniform(0.5, 2, out).astype(np.float32)
    x = QuantizedRows(torch.from_numpy(cx).cuda(), torch.from_numpy(sx).cuda())
    w = QuantizedRows(torch.from_numpy(cw).cuda(), torch.from_numpy(sw).cuda())
    got = linear_int8_forward(x, w, precision, widths if len(widths) > 1 else None)
    assert it_ctx.poll_status() == 0
    want = (cx.astype(np.float64) @ cw.T.astype(np.float64)) * sx[:, None].astype(np.float64) * sw.astype(np.float64)
    at = 0
    for width, y in zip(widths, got if len(widths) > 1 else (got,)):
        part = want[:, at:at + width]
        at += width
        assert y.precision() is precision and y.shape() == [n, width]
        assert np.all(np.abs(y.to_f32_host() - part) <= ((2.0 ** -8 if precision is BF16 else 2.0 ** -24) + 2.0 ** -22) * np.abs(part))


def test_linear_int8_of_the_longest_rows(it_ctx):
    """65536 products of 128 * 128 are 2^30: no sum leaves 32 bits."""
    import torch
    x = QuantizedRows(torch.full((2, 65536), -128, dtype=torch.int8, device="cuda"), torch.ones(2, device="cuda"))
    w = QuantizedRows(torch.full((8, 65536), -128, dtype=torch.int8, device="cuda"), torch.ones(8, device="cuda"))
    y = linear_int8_forward(x, w, FP32)
    assert it_ctx.poll_status() == 0 and np.all(y.to_f32_host() == 2.0 ** 30)
    big = QuantizedRows(torch.zeros((1, 65552), dtype=torch.int8, device="cuda"), torch.ones(1, device="cuda"))
    with pytest.raises(_lib.ITError, match="in_dim"):
        linear_int8_forward(big, big)


def test_refusals_on_the_device(it_ctx):
    import torch
    flat = torch.zeros(4 * 64 + 1, dtype=torch.bfloat16, device="cuda")
    cache = QuantizedCache.zeros(1, 8, 1, 64)
    with pytest.raises(_lib.ITError) as e:
        attention_decode_quantized(Tensor(flat[1:], [1, 4, 64], BF16), cache, ints([1]))
    assert e.value.status == _lib.IT_ERR_ALIGNMENT
    with pytest.raises(AssertionError, match="contiguous"):
        attention_decode_quantized(to_tensor(np.zeros((1, 4, 64)), BF16), QuantizedCache(torch.zeros((2, 1, 8, 2, 32), dtype=torch.uint8, device="cuda").transpose(2, 3),
                                   torch.zeros((2, 1, 8, 2, 2), dtype=torch.bfloat16, device="cuda").transpose(2, 3), 64), ints([1]))
    with pytest.raises(AssertionError, match="device"):
        attention_decode_quantized(to_tensor(np.zeros((1, 4, 64)), BF16), cache, torch.ones(1, dtype=torch.int32))
    with pytest.raises(_lib.ITError, match="16 columns"):
        quantize_rows(to_tensor(np.zeros((2, 24)), FP32))
    x = QuantizedRows(torch.zeros((2, 16), dtype=torch.int8, device="cuda"), torch.zeros(2, device="cuda"))
    w = QuantizedRows(torch.zeros((12, 16), dtype=torch.int8, device="cuda"), torch.zeros(12, device="cuda"))
    with pytest.raises(_lib.ITError, match="multiples of 8"):
        linear_int8_forward(x, w)
    with pytest.raises(_lib.ITError, match="base"):
        rope_positions(to_tensor(np.zeros((1, 1, 1, 8)), FP32), None, ints([[0]]), base=-1.0)


def test_scales_set_anew_have_one_dimension(it_ctx):
    x, w = (quantize_rows(to_tensor(np.ones((n, 16)), BF16)) for n in (2, 8))
    for rows in (x, w):
        good, rows.scales = rows.scales, rows.scales[:, None]
        with pytest.raises(AssertionError, match="scales must be float32"):
            linear_int8_forward(x, w)
        rows.scales = good
    y = linear_int8_forward(x, w, FP32).to_f32_host()
    assert np.all(y == np.float32(127 * 127 * 16 * float(x.scales[0]) * float(w.scales[0])))   # 18 and 16 bits: rounded once


def test_empty_calls(it_ctx):
    import torch
    z = lambda *s: Tensor.zeros(list(s), BF16)
    cache = QuantizedCache.zeros(2, 8, 1, 64)
    assert kv_cache_append(cache, z(2, 0, 1, 64), z(2, 0, 1, 64), ints([3, 5])).tolist() == [3, 5]
    assert kv_cache_read(cache, 0)[0].shape() == [2, 0, 1, 64]
    none = QuantizedCache.zeros(0, 8, 1, 64)
    assert attention_decode_quantized(z(0, 4, 64), none, ints([])).shape() == [0, 4, 64]
    assert attention_decode_quantized(z(2, 0, 64), cache, ints([0, 0])).shape() == [2, 0, 64]
    assert quantize_rows(z(0, 16)).shape() == [0, 16]
    e = QuantizedRows(torch.zeros((0, 16), dtype=torch.int8, device="cuda"), torch.zeros(0, device="cuda"))
    w = QuantizedRows(torch.zeros((8, 16), dtype=torch.int8, device="cuda"), torch.zeros(8, device="cuda"))
    assert linear_int8_forward(e, w).shape() == [0, 8] and linear_int8_forward(w, e).shape() == [8, 0]
    assert rope_positions(z(0, 3, 2, 64), None, torch.zeros((0, 3), dtype=torch.int32, device="cuda")).shape() == [0, 3, 2, 64]
    assert it_ctx.poll_status() == 0


# ------------------------------------------------------------------------------------------------ together
class Layer:
    """The attention layer of a model served in few bits, with the operators as a user calls them."""

    def __init__(self, rng, hidden, H, Hkv, D):
        self.H, self.Hkv, self.D, self.hidden = H, Hkv, D, hidden
        self.w_qkv = quantize_rows(to_tensor(rng.standard_normal(((H + 2 * Hkv) * D, hidden)) * hidden ** -0.5, BF16))
        self.w_o = quantize_rows(to_tensor(rng.standard_normal((hidden, H * D)) * (H * D) ** -0.5, BF16))

    def projected(self, x, positions):
        """x [batch, seq, hidden] -> rotated q, k and v."""
        B, S, _ = x.shape()
        H, Hkv, D = self.H, self.Hkv, self.D
        q, k, v = linear_int8_forward(quantize_rows(x.view([B * S, self.hidden])), self.w_qkv, BF16, [H * D, Hkv * D, Hkv * D])
        q, k = rope_positions(q.view([B, S, H, D]), k.view([B, S, Hkv, D]), positions)
        return q, k, v.view([B, S, Hkv, D])

    def prompt(self, x, cache, counts):
        import torch
        B, S, _ = x.shape()
        q, k, v = self.projected(x, torch.arange(S, dtype=torch.int32, device="cuda").expand(B, S).contiguous())
        lengths = kv_cache_append(cache, k, v, torch.zeros_like(counts), counts)
        return attention_gqa(q, k, v, True), lengths

    def step(self, x, cache, lengths):
        B = x.shape()[0]
        q, k, v = self.projected(x, lengths.view(B, 1))
        new = kv_cache_append(cache, k, v, lengths)
        o = attention_decode_quantized(q.view([B, self.H, self.D]), cache, new)
        return linear_int8_forward(quantize_rows(o.view([B, self.H * self.D])), self.w_o), new, (q, o)


def test_a_generation_step_of_a_ragged_batch(it_ctx):
    """Prompts of different lengths, then steps: attention over the cache against 64 bits on the values read back, the layer's output
    against the dequantised weights, and the rotated q against the reference's rotation at each sequence's own position."""
    import torch
    rng = np.random.default_rng(31)
    B, S, hidden, H, Hkv, D = 4, 70, 256, 8, 2, 64
    layer, cache, counts = Layer(rng, hidden, H, Hkv, D), QuantizedCache.zeros(B, 96, Hkv, D), [70, 1, 33, 64]
    x = to_tensor(rng.standard_normal((B, S, hidden)), BF16)
    _, lengths = layer.prompt(x, cache, ints(counts))
    assert lengths.tolist() == counts
    for step in range(3):
        x = to_tensor(rng.standard_normal((B, 1, hidden)), BF16)
        y, lengths, (q, o) = layer.step(x, cache, lengths)
        assert it_ctx.poll_status() == 0 and lengths.tolist() == [c + step + 1 for c in counts]
        n = max(lengths.tolist())
        k, v = (t.to_f32_host() for t in kv_cache_read(cache, n, None, lengths, FP32))
        want, _ = qr.decode(q.view([B, H, D]).to_f32_host(), k, v, lengths.tolist())
        assert np.all(np.abs(o.to_f32_host() - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -13 * np.abs(v).max())
        c, s = qr.q8(o.to_f32_host().reshape(B, H * D))
        full = (c * s[:, None]) @ layer.w_o.to_f32().to_f32_host().astype(np.float64).T
        # the dequantised weights are rounded to fp32 (2^-24): exact here, 7 + 8 bits
        assert np.all(np.abs(y.to_f32_host() - full) <= (2.0 ** -8 + 2.0 ** -22) * np.abs(full))


def test_a_captured_step_is_replayed_as_the_sequences_grow(it_ctx):
    """One graph of a step, replayed: lengths live on the device.  Equal, bit for bit, to the same steps called one by one."""
    import torch
    rng = np.random.default_rng(32)
    B, hidden, H, Hkv, D = 3, 128, 4, 2, 32
    layer = Layer(rng, hidden, H, Hkv, D)
    xs = [to_tensor(rng.standard_normal((B, 1, hidden)), BF16) for _ in range(5)]
    eager, lengths, ys = QuantizedCache.zeros(B, 64, Hkv, D), ints([0, 7, 30]), []
    for x in xs:
        y, lengths, _ = layer.step(x, eager, lengths)
        ys.append(y.torch().clone())
    cache, at = QuantizedCache.zeros(B, 64, Hkv, D), ints([0, 7, 30])
    x = Tensor(torch.zeros((B, 1, hidden), dtype=torch.bfloat16, device="cuda"), [B, 1, hidden], BF16)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        layer.step(x, QuantizedCache.zeros(B, 64, Hkv, D), at.clone())     # warm
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, new, _ = layer.step(x, cache, at)
        at.copy_(new)
    for i, xi in enumerate(xs):
        x.torch().copy_(xi.torch())
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y.torch(), ys[i]), i
    assert it_ctx.poll_status() == 0 and at.tolist() == lengths.tolist()
    assert torch.equal(cache.codes, eager.codes) and torch.equal(cache.scales, eager.scales)
    del graph
