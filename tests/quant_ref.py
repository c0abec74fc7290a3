"""The quantised operators in 64 bits on the host, from their definitions (test infrastructure)."""
import math

import numpy as np


def scale(most, steps, bits):
    """most / steps rounded to `bits` significant bits, ties to even; zero below 2^-100, NaN where a value is not finite."""
    most = np.asarray(most, np.float64)
    m, e = np.frexp(np.where(np.isfinite(most), most, 1.0) / steps)
    s = np.ldexp(np.rint(m * 2.0 ** bits), e - bits)
    return np.where(np.isfinite(most), np.where(most < 2.0 ** -100, 0.0, s), np.nan)


def whole(x, s, steps):
    """round(x / s), ties to even, within -steps..steps; 0 for s = 0 and NaN."""
    ok = s > 0
    with np.errstate(invalid="ignore"):
        c = np.rint(np.asarray(x, np.float64) / np.where(ok, s, 1.0))
    return np.where(ok, np.clip(np.nan_to_num(c), -steps, steps), 0.0)


def q4(x):
    """Rows [..., D] as (whole numbers [..., D], scales [..., groups])."""
    D = x.shape[-1]
    groups = -(-D // 32)
    parts = [x[..., 32 * j:32 * j + 32] for j in range(groups)]
    with np.errstate(invalid="ignore"):
        s = np.stack([np.minimum(scale(np.abs(np.where(np.isnan(p), np.inf, p)).max(-1), 7, 5), 2.0 ** 122) for p in parts], -1)
    return np.concatenate([whole(p, s[..., j:j + 1], 7) for j, p in enumerate(parts)], -1), s


def q4_values(x):
    c, s = q4(x)
    return c * np.repeat(s, 32, -1)[..., :x.shape[-1]]


def q4_bytes(c):
    """The documented bytes of rows of whole numbers [..., D] (columns past D are zeros: 8)."""
    D = c.shape[-1]
    groups = -(-D // 32)
    out = np.full(c.shape[:-1] + (16 * groups,), 0x88, np.uint8)
    for d in range(D):
        j, t, e = d // 32, d % 32 // 8, d % 8
        bit = 4 * (e // 2) + 16 * (e % 2)
        at = 4 * (t * groups + j) + bit // 8
        u = (c[..., d] + 8).astype(np.uint8)
        out[..., at] = (out[..., at] & (0x0F if bit % 8 else 0xF0)) | (u << (bit % 8))
    return out


def decode(q, k, v, lengths):
    """q [B, H, D], k and v [B, L, Hkv, D] -> o [B, H, D], lse [B, H]."""
    B, H, D = q.shape
    G = H // k.shape[2]
    o, lse = np.zeros((B, H, D)), np.full((B, H), -np.inf)
    for b in range(B):
        n = int(lengths[b])
        for h in range(H if n else 0):
            s = k[b, :n, h // G].astype(np.float64) @ q[b, h].astype(np.float64) / math.sqrt(D)
            m = s.max()
            p = np.exp(s - m)
            o[b, h] = p @ v[b, :n, h // G].astype(np.float64) / p.sum()
            lse[b, h] = m + np.log(p.sum())
    return o, lse


def rope(x, positions, base, sections, per_axis=False, inverse=False):
    """x [B, S, heads, D], positions [axes, B, S]."""
    D = x.shape[-1]
    angle, i = [], 0
    for a, n in enumerate(sections):
        f = [base ** (-j / n) if per_axis else base ** (-2.0 * (i + j) / D) for j in range(n)]
        angle.append(positions[a].astype(np.float64)[..., None] * np.array(f, np.float64).reshape(-1))
        i += n
    angle = np.concatenate(angle, -1)[:, :, None, :]
    c, s = np.cos(angle), np.sin(angle) * (-1 if inverse else 1)
    x0, x1 = x[..., 0::2].astype(np.float64), x[..., 1::2].astype(np.float64)
    return np.stack((x0 * c - x1 * s, x0 * s + x1 * c), -1).reshape(x.shape)


def q8(x):
    """Rows as (whole numbers, scales)."""
    with np.errstate(invalid="ignore"):
        s = scale(np.abs(np.where(np.isnan(x), np.inf, x)).max(-1), 127, 8)
    return whole(x, s[..., None], 127), s
