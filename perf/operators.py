"""Serving from quantised weights and a quantised key/value cache, as timed cases.

A case is one pass of one operator (`op`) at one size:

  rope     rotary embedding of q and k at positions given per token, on one axis (sequences of a batch that stand at different
           lengths) or several (time, height, width of image and video tokens); "train" rotates gradients back as well
  append   new tokens' keys and values quantised to 4 bits into the cache behind each sequence's own length, and those rows read back
  read     a stretch of the cache read back as tensors
  decode   attention of one new token per sequence over the 4-bit cache, every sequence at its own length
  linear   a projection in 8-bit integers: tokens quantised row by row, times weights quantised channel by channel

Where `own` is false, run() computes the same in elementary torch operations.

Forms.  4 bits: 32 neighbouring columns of a head share a scale s, the largest magnitude / 7 rounded to 5 significant bits; a value
is s * c with a whole number c in -7..7.  A row (one position of one K/V head) is 4 * groups words of 32 bits; word t * groups + j
holds columns 32 j + 8 t + e, e = 0..7, as c + 8 in 4 bits at bit 4 * (e // 2) + 16 * (e % 2).  codes: uint8 [2, batch, kv_heads,
max_len, 16 * groups], keys first; scales: bf16 [2, batch, kv_heads, max_len, groups].  8 bits: a row's scale is its largest
magnitude / 127 rounded to 8 significant bits; a value is s * c with c in -127..127."""
import math

import torch

own = False

ROPE_BASE = 10000.0


# ------------------------------------------------------------------------------------------------ cases
def _rope(name, dtype, B, S, H, Hkv, D, axes, train):
    return _named(name, {"op": "rope", "dtype": dtype, "B": B, "S": S, "H": H, "Hkv": Hkv, "D": D, "axes": axes, "train": train})


def _append(name, dtype, B, T, Hkv, D, past, padded):
    return _named(name, {"op": "append", "dtype": dtype, "B": B, "T": T, "Hkv": Hkv, "D": D, "past": past, "padded": padded})


def _read(name, dtype, B, T, Hkv, D, past):
    return _named(name, {"op": "read", "dtype": dtype, "B": B, "T": T, "Hkv": Hkv, "D": D, "past": past})


def _decode(name, dtype, B, L, H, Hkv, D, ragged):
    return _named(name, {"op": "decode", "dtype": dtype, "B": B, "L": L, "H": H, "Hkv": Hkv, "D": D, "ragged": ragged})


def _linear(name, dtype, n, k, out, kv=0):
    """kv: width of the two last column ranges that come back as tensors of their own (0: one result)."""
    return _named(name, {"op": "linear", "dtype": dtype, "n": n, "in": k, "out": out, "kv": kv})


def _named(name, case):
    return dict(case, name=name) if name else case


def listed():
    return [
        # A generation step of a full batch: one token per sequence, every sequence at a far position of its own.
        _rope("rope_step", "bf16", 32, 1, 32, 8, 128, 1, False),
        # Training on video tokens: time, height and width positions, forward and backward, a head_dim that is no power of two.
        _rope("rope_video_train", "fp32", 2, 4093, 16, 4, 96, 3, True),
        # The new token of each sequence into the cache: latency.
        _append("append_step", "bf16", 32, 1, 8, 128, 4000, False),
        # Prompts of different lengths, padded to the longest, into an empty cache.
        _append("append_prompts", "bf16", 8, 2999, 8, 128, 0, True),
        # A conversation's history out of the cache again, for a pass that wants it whole, in fp32.
        _read("read_history", "fp32", 2, 8001, 4, 64, 50),
        # The tiny fp32 model that the framework's reference generates with.
        _decode("decode_fp32_tiny", "fp32", 1, 100, 4, 4, 64, False),
        # A handful of users of a hidden-2048 model.
        _decode("decode_few", "bf16", 4, 1000, 16, 4, 128, True),
        # One long document: few rows, so the long axis has to be split.
        _decode("decode_long", "bf16", 1, 131000, 16, 2, 128, False),
        # A full serving batch of ragged lengths, one of its slots empty: nothing but reading the cache counts.
        _decode("decode_batch", "bf16", 32, 8190, 32, 8, 128, True),
        # The q, k and v projections of one generation step: reading the weights.
        _linear("linear_step", "bf16", 4, 2048, 2560, 256),
        # A prompt of ragged length through a wide projection, fp32 activations.
        _linear("linear_prompt", "fp32", 2999, 2048, 6144),
        # Prompts of a whole batch at hidden 4096: the tensor cores' rate.
        _linear("linear_batch", "bf16", 8192, 4096, 12288),
    ]


def _log(rng, lo, hi):
    """A whole number in lo..hi, spread evenly over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_one(rng):
    op = rng.choice(("rope", "append", "read", "decode", "decode", "decode", "linear", "linear"))
    dtype = rng.choice(("bf16", "bf16", "fp32"))
    H = rng.choice((4, 8, 12, 16, 32))
    Hkv = H // rng.choice([g for g in (1, 2, 4, 8, 16) if H % g == 0])
    D = rng.choice((32, 64, 64, 80, 96, 128, 128))
    if op == "rope":
        return _rope(None, dtype, _log(rng, 1, 32), _log(rng, 1, 5000), H, Hkv, D, rng.choice((1, 2, 3)), rng.random() < 0.4)
    if op == "append":
        return _append(None, dtype, _log(rng, 1, 64), _log(rng, 1, 4000), Hkv, D, _log(rng, 1, 5000) - 1, rng.random() < 0.5)
    if op == "read":
        return _read(None, dtype, _log(rng, 1, 16), _log(rng, 1, 12000), Hkv, D, _log(rng, 1, 3000) - 1)
    if op == "decode":
        return _decode(None, dtype, _log(rng, 1, 64), _log(rng, 1, 140000), H, Hkv, D, rng.random() < 0.6)
    n, k, out = _log(rng, 1, 8192), 16 * _log(rng, 16, 256), 8 * _log(rng, 32, 1536)
    return _linear(None, dtype, n, k, out, 8 * (out // 64) if rng.random() < 0.4 else 0)


# What a drawn case may need at most (operations, bytes): no more than the largest listed case of its operator.
_MOST = {"rope": (1e12, 2.6e8), "append": (1e12, 1.3e8), "read": (1e12, 2.5e7), "decode": (1e12, 1.6e8), "linear": (8.3e11, 3.5e8)}


def draw(rng):
    while True:
        c = _draw_one(rng)
        w, (flops, nbytes) = work(c), _MOST[c["op"]]
        if w["flops"] <= flops and w["bytes"] <= nbytes and _cache_bytes(c) <= 4e8:
            return c


def _max_len(case):
    """Positions that the cache has room for: it grows in blocks of 256."""
    need = case["L"] if case["op"] == "decode" else case["past"] + case["T"]
    return (need + 255) // 256 * 256


def _cache_bytes(case):
    return 2 * case["B"] * case["Hkv"] * _max_len(case) * 18 * -(-case["D"] // 32) if "Hkv" in case and case["op"] != "rope" else 0


def _spread(n, most, uneven):
    """n lengths up to `most`: all alike, or evenly spread with an empty one where there are eight or more."""
    if not uneven or not most:
        return [most] * n
    lens = [max(1, most * (2 * i + 1) // (2 * n)) for i in range(n)]
    lens[-1] = most
    if n >= 8:
        lens[0] = 0
    return lens


# ------------------------------------------------------------------------------------------------ inputs
def _normal(gen, shape, dtype):
    t = torch.randn(shape, generator=gen, device="cuda")
    return t if dtype == "fp32" else t.to(torch.bfloat16)


def _shuffled(gen, values):
    t = torch.tensor(values, dtype=torch.int32, device="cuda")
    return t[torch.randperm(len(values), generator=gen, device="cuda")]


def _filled(gen, case, max_len):
    """A cache that holds normally distributed keys and values at every position.  Whole numbers of a normal distribution cut off
    at 7, with scales as groups of 32 such values have them: a cache need not be quantised to be read."""
    groups, shape = -(-case["D"] // 32), (2, case["B"], case["Hkv"], max_len)
    c = torch.randn(shape + (16 * groups, 2), generator=gen, device="cuda").mul_(3.2).round_().clamp_(-7, 7).to(torch.int8) + 8
    codes = (c[..., 0] + 16 * c[..., 1]).view(torch.uint8)
    s = (torch.rand(shape + (groups,), generator=gen, device="cuda") * 16).floor_() / 16 + 1.0    # 5 significant bits
    return codes, (s * 0.25).to(torch.bfloat16)


def prepare(case, seed):
    op, dt = case["op"], case["dtype"]
    gen = torch.Generator(device="cuda").manual_seed(seed)
    st = dict(case)
    if op == "rope":
        B, S, H, Hkv, D, axes = (case[k] for k in ("B", "S", "H", "Hkv", "D", "axes"))
        st["q"], st["k"] = _normal(gen, (B, S, H, D), dt), _normal(gen, (B, S, Hkv, D), dt)
        if case["train"]:
            st["d_q"], st["d_k"] = _normal(gen, (B, S, H, D), dt), _normal(gen, (B, S, Hkv, D), dt)
        at = torch.randint(0, 200000, (axes, B, 1), generator=gen, device="cuda", dtype=torch.int32)   # where a sequence stands
        step = torch.arange(S, dtype=torch.int32, device="cuda")
        side = max(1, math.isqrt(S))
        walk = [step, step // side % side, step % side] if axes > 1 else [step]                      # rows and columns of pictures
        st["positions"] = torch.stack([at[a] + walk[a] for a in range(axes)]).contiguous()
        st["sections"] = [D // 2] if axes == 1 else [D // 2 - (axes - 1) * (D // 6)] + [D // 6] * (axes - 1)
        return st
    if op == "linear":
        n, k, out = case["n"], case["in"], case["out"]
        x = torch.randn((n, k), generator=gen, device="cuda")
        x *= 1.0 + 8.0 * (torch.rand((1, k), generator=gen, device="cuda") < 0.01)     # a few large channels, as activations have
        st["x"] = x if dt == "fp32" else x.to(torch.bfloat16)
        c = (torch.randn((out, k), generator=gen, device="cuda") * 36.0).round_().clamp_(-127, 127).to(torch.int8)
        st["w_codes"] = c
        s = (torch.rand(out, generator=gen, device="cuda") + 1.0).to(torch.bfloat16)
        st["w_scales"] = s.float() / 2 ** round(math.log2(36.0 * k ** 0.5))
        st["splits"] = [out - 2 * case["kv"], case["kv"], case["kv"]] if case["kv"] else [out]
        return st
    B, Hkv, D, max_len = case["B"], case["Hkv"], case["D"], _max_len(case)
    if op == "decode":
        st["lengths"] = _shuffled(gen, _spread(B, case["L"], case["ragged"]))
        st["q"] = _normal(gen, (B, case["H"], D), dt)
        st["codes"], st["scales"] = _filled(gen, case, max_len)
        return st
    st["starts"] = _shuffled(gen, _spread(B, case["past"], True))
    if op == "read":
        st["codes"], st["scales"] = _filled(gen, case, max_len)
        return st
    st["counts"] = _shuffled(gen, _spread(B, case["T"], True)) if case["padded"] else None
    st["k"], st["v"] = _normal(gen, (B, case["T"], Hkv, D), dt), _normal(gen, (B, case["T"], Hkv, D), dt)
    groups = -(-D // 32)
    st["codes"] = torch.zeros((2, B, Hkv, max_len, 16 * groups), dtype=torch.uint8, device="cuda")
    st["scales"] = torch.zeros((2, B, Hkv, max_len, groups), dtype=torch.bfloat16, device="cuda")
    return st


# ------------------------------------------------------------------------------------------------ plain forms
def _keep_bits(t, bits):
    """Positive 64-bit numbers rounded to `bits` significant bits, ties to even."""
    drop = 53 - bits
    b = t.view(torch.int64)
    b = (b + ((1 << (drop - 1)) - 1) + ((b >> drop) & 1)) >> drop << drop
    return b.view(torch.float64)


def _quantise(x, most, bits):
    """(whole numbers, scales) of the last dimension of x: scale = largest magnitude / most, rounded to `bits` significant bits.
    In 64 bits: a value next to the middle of two whole numbers has to go to the right one."""
    x = x.double()
    s = _keep_bits(x.abs().amax(-1, keepdim=True) / most, bits)
    return torch.where(s > 0, torch.round(x / torch.where(s > 0, s, 1.0)), 0.0), s.squeeze(-1)


def _unpacked(codes, scales, D):
    """The values of cache rows, in 32 bits: codes [..., 16 * groups], scales [..., groups] -> [..., D]."""
    groups = scales.shape[-1]
    words = codes.view(torch.int32).unflatten(-1, (4, groups))                          # [..., t, j]
    e = torch.arange(8, dtype=torch.int32, device=codes.device)
    c = ((words.unsqueeze(-1) >> (4 * (e // 2) + 16 * (e % 2))) & 15) - 8                # [..., t, j, e]
    v = c.float() * scales.float().unsqueeze(-2).unsqueeze(-1)
    return v.transpose(-3, -2).flatten(-3)[..., :D]


def _packed(x, D):
    """Rows [..., D] as (codes, scales) of the cache."""
    groups = -(-D // 32)
    x = torch.nn.functional.pad(x, (0, 32 * groups - D)).unflatten(-1, (groups, 4, 8))
    c, s = _quantise(x.flatten(-2), 7, 5)
    u = (c + 8).to(torch.int64).unflatten(-1, (4, 8)).transpose(-3, -2)                 # [..., t, j, e]
    e = torch.arange(8, device=x.device)
    words = (u << (4 * (e // 2) + 16 * (e % 2))).sum(-1)
    words = torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)
    return words.flatten(-2).view(torch.uint8), s.to(torch.bfloat16)


def _rows(st, starts, count, lengths):
    """Positions starts[b] + t of the cache as [batch, count, kv_heads, head_dim] keys and values; zeros past a sequence's end."""
    at = starts.long()[:, None] + torch.arange(count, device=starts.device)             # [B, count]
    valid = at < lengths.long()[:, None]
    at, valid = at.clamp(max=st["codes"].shape[3] - 1)[None, :, None, :, None], valid[None, :, None, :, None]
    codes = torch.take_along_dim(st["codes"], at, 3)
    scales = torch.take_along_dim(st["scales"], at, 3)
    out = torch.where(valid, _unpacked(codes, scales, st["D"]), 0.0).transpose(2, 3)
    return out.contiguous().to(torch.float32 if st["dtype"] == "fp32" else torch.bfloat16)


def _rotated(x, c, s):
    a, b = x.float()[..., 0::2], x.float()[..., 1::2]
    return torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2).to(x.dtype)


def _plain_rope(st):
    D = st["D"]
    pair = torch.arange(D // 2, device="cuda")
    sections = torch.tensor(st["sections"], device="cuda")
    axis = (pair[:, None] >= sections.cumsum(0)).sum(1)
    angle = st["positions"].double()[axis].movedim(0, -1) * ROPE_BASE ** (-2.0 * pair.double() / D)     # [B, S, D/2], 64 bits
    c, s = angle.cos().float().unsqueeze(2), angle.sin().float().unsqueeze(2)
    out = (_rotated(st["q"], c, s), _rotated(st["k"], c, s))
    return out + (_rotated(st["d_q"], c, -s), _rotated(st["d_k"], c, -s)) if st["train"] else out


def _plain_append(st):
    T, max_len = st["T"], st["codes"].shape[3]
    counts = torch.full_like(st["starts"], T) if st["counts"] is None else st["counts"]
    new = st["starts"] + counts
    t = torch.arange(T, device="cuda")
    at = st["starts"].long()[:, None] + t                                               # [B, T]
    b, i = torch.nonzero((t < counts[:, None]) & (at < max_len), as_tuple=True)
    codes, scales = _packed(torch.stack((st["k"], st["v"])), st["D"])                   # [2, B, T, Hkv, ...]
    st["codes"][:, b, :, at[b, i]] = codes[:, b, i].transpose(0, 1)
    st["scales"][:, b, :, at[b, i]] = scales[:, b, i].transpose(0, 1)
    rows = _rows(st, st["starts"], T, new)
    return new, rows[0], rows[1]


def _plain_read(st):
    rows = _rows(st, st["starts"], st["T"], st["starts"] + st["T"])
    return rows[0], rows[1]


def _plain_decode(st):
    B, H, Hkv, D = (st[k] for k in ("B", "H", "Hkv", "D"))
    kv = _unpacked(st["codes"], st["scales"], D)                                        # [2, B, Hkv, max_len, D]
    q = st["q"].float().reshape(B, Hkv, H // Hkv, D)
    s = q @ kv[0].transpose(-1, -2) * D ** -0.5
    s = s.masked_fill(torch.arange(s.shape[-1], device="cuda") >= st["lengths"].long()[:, None, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    p = (s - m.clamp(min=-1e30)).exp()
    total = p.sum(-1, keepdim=True)
    o = p @ kv[1] / total.clamp(min=1e-30)
    return o.reshape(B, H, D).to(st["q"].dtype), (m + total.log()).reshape(B, H)


def _plain_linear(st):
    c, s = _quantise(st["x"], 127, 8)
    y = (c.float() @ st["w_codes"].float().T) * (s.float()[:, None] * st["w_scales"])
    return tuple(t.contiguous() for t in y.to(st["x"].dtype).split(st["splits"], -1))


# ------------------------------------------------------------------------------------------------ the framework's calls
def _tensor(t):
    from irontensor_b200 import Precision, Tensor
    return Tensor(t, t.shape, Precision.FP32 if t.dtype is torch.float32 else Precision.BF16)


def _own(st):
    import irontensor_b200 as it
    op = st["op"]
    precision = it.Precision.FP32 if st["dtype"] == "fp32" else it.Precision.BF16
    if op == "rope":
        q, k = it.rope_positions(_tensor(st["q"]), _tensor(st["k"]), st["positions"], ROPE_BASE, st["sections"])
        if not st["train"]:
            return q.torch(), k.torch()
        d_q, d_k = it.rope_positions(_tensor(st["d_q"]), _tensor(st["d_k"]), st["positions"], ROPE_BASE, st["sections"], inverse=True)
        return q.torch(), k.torch(), d_q.torch(), d_k.torch()
    if op == "linear":
        weight = it.QuantizedRows(st["w_codes"], st["w_scales"])
        y = it.linear_int8_forward(it.quantize_rows(_tensor(st["x"])), weight, precision, st["splits"])
        return tuple(t.torch() for t in y)
    cache = it.QuantizedCache(st["codes"], st["scales"], st["D"])
    if op == "decode":
        o = it.attention_decode_quantized(_tensor(st["q"]), cache, st["lengths"])
        return o.torch(), o.lse.torch()
    if op == "read":
        k, v = it.kv_cache_read(cache, st["T"], st["starts"], precision=precision)
        return k.torch(), v.torch()
    new = it.kv_cache_append(cache, _tensor(st["k"]), _tensor(st["v"]), st["starts"], st["counts"])
    k, v = it.kv_cache_read(cache, st["T"], st["starts"], new, precision)
    return new, k.torch(), v.torch()


def run(st):
    if own:
        return _own(st)
    return {"rope": _plain_rope, "append": _plain_append, "read": _plain_read, "decode": _plain_decode, "linear": _plain_linear}[st["op"]](st)


# ------------------------------------------------------------------------------------------------ what a pass needs
def work(case):
    op, e = case["op"], 4 if case["dtype"] == "fp32" else 2
    if op == "rope":
        B, S, n = case["B"], case["S"], (case["H"] + case["Hkv"]) * case["D"]
        passes = 2 if case["train"] else 1
        return {"bytes": passes * 2 * B * S * n * e + 4 * case["axes"] * B * S, "flops": passes * 3 * B * S * n}
    if op == "linear":
        n, k, out = case["n"], case["in"], case["out"]
        return {"bytes": n * k * e + out * k + 4 * out + n * out * e, "flops": 2 * n * k * out}
    B, Hkv, D = case["B"], case["Hkv"], case["D"]
    row = D / 2 + 2 * -(-D // 32)                 # a position of one head: codes and scales
    if op == "decode":
        tokens = sum(_spread(B, case["L"], case["ragged"]))
        return {"bytes": 2 * tokens * Hkv * row + B * case["H"] * (2 * D * e + 4) + 4 * B, "flops": 4 * tokens * case["H"] * D}
    if op == "read":
        return {"bytes": 2 * B * case["T"] * Hkv * (row + D * e) + 4 * B, "flops": 2 * B * case["T"] * Hkv * D}
    tokens = sum(_spread(B, case["T"], True)) if case["padded"] else B * case["T"]
    # read, quantise and write the new tokens; read their codes back and write the whole padded block
    return {"bytes": 2 * Hkv * (tokens * (D * e + 2 * row) + B * case["T"] * D * e) + 8 * B, "flops": 2 * tokens * Hkv * 4 * D}


# ------------------------------------------------------------------------------------------------ the definition, in 64 bits
def _nearest(x, most, bits):
    """The values that x [..., n] is held as: a scale and whole numbers per row of n."""
    x = x.to(torch.float64)
    m, power = torch.frexp(x.abs().max(-1, keepdim=True).values / most)
    s = torch.ldexp(torch.round(m * 2 ** bits), power - bits)
    return torch.where(s == 0, x * 0, torch.round(x / s.clamp(min=1e-300)) * s)


def _value_of(codes, scales, D):
    """Cache rows from their bytes: byte i of a row is in word i // 4 and holds two columns, 16 bits apart in the order of columns."""
    groups = scales.shape[-1]
    d = torch.arange(D, device=codes.device)
    j, t, e = d // 32, d % 32 // 8, d % 8
    byte = 4 * (t * groups + j) + 2 * (e % 2) + e // 4
    c = torch.where(e // 2 % 2 == 0, codes[..., byte] % 16, codes[..., byte] // 16).to(torch.float64) - 8
    return c * scales.to(torch.float64)[..., j]


def exact(case, seed):
    st, op = prepare(case, seed), case["op"]
    if op == "rope":
        D, start, angles = case["D"], 0, []
        for axis, n in enumerate(st["sections"]):
            i = torch.arange(start, start + n, device="cuda", dtype=torch.float64)
            angles.append(st["positions"][axis].to(torch.float64)[..., None] * torch.exp(-math.log(ROPE_BASE) * 2 * i / D))
            start += n
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), torch.cat(angles, -1))[:, :, None]
        names = ("q", "k", "d_q", "d_k") if case["train"] else ("q", "k")
        return tuple(torch.view_as_real(torch.view_as_complex(st[n].to(torch.float64).unflatten(-1, (D // 2, 2)).contiguous()) *
                                        (turn.conj() if n[0] == "d" else turn)).flatten(-2) for n in names)
    if op == "linear":
        y = _nearest(st["x"], 127, 8) @ (st["w_codes"].to(torch.float64) * st["w_scales"].to(torch.float64)[:, None]).T
        a, b = st["splits"][0], sum(st["splits"][:2])
        return (y[:, :a].contiguous(), y[:, a:b].contiguous(), y[:, b:].contiguous()) if case["kv"] else (y,)
    if op == "decode":
        B, H, Hkv, D = (case[k] for k in ("B", "H", "Hkv", "D"))
        o = torch.zeros((B, H, D), dtype=torch.float64, device="cuda")
        lse = torch.full((B, H), -math.inf, dtype=torch.float64, device="cuda")
        for b, n in enumerate(st["lengths"].tolist()):
            if n:
                k, v = _value_of(st["codes"][:, b, :, :n], st["scales"][:, b, :, :n], D)
                s = torch.einsum("hgd,hnd->hgn", st["q"][b].to(torch.float64).view(Hkv, H // Hkv, D), k) / math.sqrt(D)
                lse[b] = torch.logsumexp(s, -1).view(H)
                o[b] = torch.einsum("hgn,hnd->hgd", torch.softmax(s, -1), v).reshape(H, D)
        return o, lse
    B, T, starts = case["B"], case["T"], st["starts"].tolist()
    if op == "read":
        kv = _value_of(st["codes"], st["scales"], case["D"])
        return tuple(torch.stack([kv[i, b, :, s:s + T].transpose(0, 1) for b, s in enumerate(starts)]) for i in range(2))
    counts = [T] * B if st["counts"] is None else st["counts"].tolist()
    valid = torch.arange(T, device="cuda") < torch.tensor(counts, device="cuda")[:, None]
    out = []
    for x in (st["k"], st["v"]):
        parts = [_nearest(g, 7, 5) for g in x.split(32, -1)]
        out.append(torch.cat(parts, -1) * valid[:, :, None, None])
    return (torch.tensor([a + n for a, n in zip(starts, counts)], dtype=torch.int32, device="cuda"), out[0], out[1])
