"""Plain forms, in 64 bits or in the formats' own roundings, of the paged cache, attention over it and four-bit weights."""
from __future__ import annotations

import numpy as np

SHIFT = np.array([0, 16, 4, 20, 8, 24, 12, 28], np.uint32)  # bit of value i of a word


def quantize(x16):
    """(codes, s, m) of groups of binary16 values [..., group]; a group with an infinity or NaN has a pair of NaN."""
    x = x16.astype(np.float32)
    bad = ~np.isfinite(x).all(-1, keepdims=True)
    x = np.where(bad, 0, x).astype(np.float32)
    lo, hi = x.min(-1, keepdims=True), x.max(-1, keepdims=True)
    s = ((hi - lo) / np.float32(15)).astype(np.float16).astype(np.float32)
    n = np.where(s > 0, np.rint((x - lo) / np.where(s > 0, s, 1).astype(np.float32)), 0).clip(0, 15).astype(np.uint32)
    s, lo = np.where(bad, np.nan, s), np.where(bad, np.nan, lo)
    return n, s[..., 0].astype(np.float16), lo[..., 0].astype(np.float16)


def words(codes):
    return np.bitwise_or.reduce(codes.astype(np.uint32).reshape(*codes.shape[:-1], -1, 8) << SHIFT, axis=-1)


def codes_of(w):
    return ((w[..., None] >> SHIFT) & 15).reshape(*w.shape[:-1], -1)


def values(codes, s, m):
    """What codes [..., group] of pairs s, m [...] stand for (products and sums of these are exact in 64 bits)."""
    with np.errstate(invalid="ignore", over="ignore"):
        return (s.astype(np.float64)[..., None] * codes + m.astype(np.float64)[..., None]).astype(np.float16)


def rows_of(x16, four_bit):
    """Cache rows of binary16 values [..., D]: themselves, or bytes."""
    if not four_bit:
        return x16
    D = x16.shape[-1]
    n, s, m = quantize(x16.reshape(*x16.shape[:-1], D // 32, 32))
    w = np.ascontiguousarray(words(n.reshape(x16.shape))).view(np.uint8)
    return np.concatenate([w, np.ascontiguousarray(np.stack([s, m], -1)).view(np.uint8).reshape(*x16.shape[:-1], D // 8)], -1)


def values_of(rows, four_bit):
    """The binary16 values [..., D] that cache rows stand for."""
    if not four_bit:
        return rows
    D = rows.shape[-1] * 8 // 5
    n = codes_of(np.ascontiguousarray(rows[..., :D // 2]).view(np.uint32)).reshape(*rows.shape[:-1], D // 32, 32)
    sm = np.ascontiguousarray(rows[..., D // 2:]).view(np.float16).reshape(*rows.shape[:-1], D // 32, 2)
    return values(n, sm[..., 0], sm[..., 1]).reshape(*rows.shape[:-1], D)


def rotate(x, pos, rope, interleaved):
    """[T, heads, D] turned, products and sums rounded to fp32, then binary16."""
    y = x.astype(np.float32)
    if rope is not None:
        rot = rope.shape[1]
        h = rot // 2
        cs = rope[np.minimum(pos, len(rope) - 1)][:, None]
        c, s = cs[..., :h], cs[..., h:]
        ia, ib = (np.arange(0, rot, 2), np.arange(1, rot, 2)) if interleaved else (np.arange(h), np.arange(h, rot))
        a, b = y[..., ia].copy(), y[..., ib].copy()
        y[..., ia] = a * c - b * s
        y[..., ib] = b * c + a * s
    with np.errstate(over="ignore"):
        return y.astype(np.float16)


def rope_table(positions, rot, base=10000.0):
    angle = np.arange(positions)[:, None] * base ** (-np.arange(0, rot, 2) / rot)
    return np.concatenate([np.cos(angle), np.sin(angle)], 1).astype(np.float32)


def sees(pos, t, causal, window, stride):
    """[rows, keys] of positions and keys."""
    p, t = np.asarray(pos)[:, None], np.asarray(t)[None]
    ok = t <= p if causal else np.ones((p.shape[0], t.shape[1]), bool)
    if window:
        near = t >= p - window
        ok &= (near | (t % stride == 0)) if stride else near
    return ok


def attention(q, k, v, pos, scale, causal=True, window=0, stride=0):
    """One sequence in 64 bits: q [n, Hq, D], k, v [L, H, D] -> (out, lse, tolerance), the tolerance for binary16 outputs.

    Off by at most: half a step of the output, 2^-11 |out|; half a step of each weight, 2^-11 sum w |v| (the sums divide the
    unrounded weights' total); and the fp32 scores, x in units of log2: D + 2 roundings of the sum of |q_i k_i| c, each 2^-24,
    which change a weight by ln 2 times that, once above and once below the division.  2^-20 covers the exponential, the
    sums' order (fewer than 16 roundings a level) and the division."""
    n, Hq, D = q.shape
    L, H, _ = k.shape
    ok = sees(pos, np.arange(L), causal, window, stride)
    out, lse, tol = np.zeros((n, Hq, D)), np.full((n, Hq), np.inf), np.zeros((n, Hq, D))
    for h in range(Hq):
        kk, vv = k[:, h // (Hq // H)].astype(np.float64), v[:, h // (Hq // H)].astype(np.float64)
        for i in range(n):
            s = ok[i]
            if not s.any():
                continue
            qi = q[i, h].astype(np.float64)
            x = kk[s] @ qi * scale
            M = x.max()
            w = np.exp(x - M)
            l = w.sum()
            out[i, h] = w @ vv[s] / l
            lse[i, h] = M + np.log(l)
            size = (np.abs(kk[s]) @ np.abs(qi)).max() * abs(scale)
            A = w @ np.abs(vv[s]) / l
            tol[i, h] = 2.0 ** -11 * np.abs(out[i, h]) + (2.0 ** -11 + 2 * (D + 2) * 2.0 ** -24 * size + 2.0 ** -20) * A + 2.0 ** -25
    return out, lse, tol
