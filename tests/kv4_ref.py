"""The 4-bit paged KV cache restated on the CPU: the byte layout from its
description in include/spec_b200.h, the append in separately rounded f32
operations (the stored bytes are to be equal), the attention in float64."""

import numpy as np

F32 = np.float32


def block_bytes(p, d):
    return p * d * 5 // 4


def code_address(p, d, j, ch, value):
    """Byte of channel ch of token j's codes; its nibble is ch % 2."""
    byte = ch // 2
    if not value:
        return j * (d // 2) + byte
    per = 256 // d
    quarter = ((j % per) * (d // 64) + byte // 32) ^ ((j // per) % (d // 32))
    return p * d // 2 + p * d // 8 + (j // per) * 128 + quarter * 32 + byte % 32


def scale_address(p, d, j, g, value):
    n = d // 32
    if not value:
        return p * d // 2 + (j * n + g) * 4
    return p * d + p * d // 8 + (j // 2) * n * 8 + g * 8 + (j % 2) * 4


def rotate(x, cos, sin, half):
    """x [heads, d] f32 with one position's table rows [d/2]; every operation rounded to f32."""
    y = np.empty_like(x)
    d = x.shape[-1]
    a, b = (x[:, :d // 2], x[:, d // 2:]) if half else (x[:, 0::2], x[:, 1::2])
    ya, yb = a * cos - b * sin, b * cos + a * sin
    if half:
        y[:, :d // 2], y[:, d // 2:] = ya, yb
    else:
        y[:, 0::2], y[:, 1::2] = ya, yb
    return y


def quantize(x):
    """x [d] f32 -> codes [d] uint8, scales [d/32, 2] f16, values [d] f32."""
    d = x.shape[0]
    if np.isnan(x).any():
        so = np.full((d // 32, 2), np.nan, np.float16)
        return np.zeros(d, np.uint8), so, np.full(d, np.nan, F32)
    g = np.clip(x, F32(-20000), F32(20000)).reshape(-1, 32)
    lo, hi = g.min(1, keepdims=True), g.max(1, keepdims=True)
    s = ((hi - lo) * F32(16.0 / 15.0)).astype(np.float16)
    o = (lo - s.astype(F32)).astype(np.float16)
    sf, of = s.astype(F32), o.astype(F32)
    with np.errstate(divide="ignore"):
        inv = np.where(sf > 0, F32(16) / sf, F32(0)).astype(F32)
    c = np.clip(np.rint((g - of) * inv - F32(16)), 0, 15)
    val = sf * (F32(1) + c.astype(F32) / F32(16)) + of
    return c.astype(np.uint8).reshape(-1), np.concatenate([s, o], 1), val.reshape(-1)


def store(block, p, d, j, codes, so, value):
    """Writes token j's codes and scales into a block (uint8 array)."""
    for ch in range(d):
        at = code_address(p, d, j, ch, value)
        keep = 0xF0 if ch % 2 == 0 else 0x0F
        block[at] = (int(block[at]) & keep) | (int(codes[ch]) << (4 * (ch % 2)))
    raw = np.ascontiguousarray(so).view(np.uint8)
    for g in range(d // 32):
        at = scale_address(p, d, j, g, value)
        block[at:at + 4] = raw[g]


def load(block, p, d, j, value):
    """Token j's values [d] in float64."""
    out = np.empty(d)
    for g in range(d // 32):
        at = scale_address(p, d, j, g, value)
        s, o = np.frombuffer(block[at:at + 4].tobytes(), np.float16).astype(np.float64)
        for ch in range(32 * g, 32 * g + 32):
            c = (int(block[code_address(p, d, j, ch, value)]) >> (4 * (ch % 2))) & 15
            out[ch] = s * (16 + c) / 16 + o
    return out


def sees(i, w, masks):
    """Whether row i of a sequence sees its step's row w (masks: of the sequence, or None)."""
    return bool((int(masks[i]) >> w) & 1) if masks is not None else w <= i


def attend(q, k, v, kv_len, masks, scale):
    """q [rows, heads, d], k / v [tokens, kv heads, d] float64 -> (out, bound).

    bound: how far an output may be from float64 when q.k and p.v take the
    stored values as f16 and sum in f32 (unit roundoff u = 2^-11 of f16).  A
    score is off by at most delta = |scale| sum |q||k| u (the rounding of k; q
    is exact up to 2^-24 of the row's largest entry) plus 2^-20 of it for the
    f32 sums; weights are then off by a factor within exp(+-2 delta), rounded
    to f16 once (u) on values rounded to f16 (u)."""
    rows, heads, d = q.shape
    g = heads // k.shape[1]
    out, bound = np.zeros_like(q), np.zeros_like(q)
    n = k.shape[0]
    see = np.array([[t < kv_len or sees(i, t - kv_len, masks) for t in range(n)] for i in range(rows)]).reshape(rows, n)
    u = 2.0 ** -11
    for i in range(rows):
        at = np.flatnonzero(see[i])
        if at.size == 0:
            continue
        for h in range(heads):
            kk, vv = k[at, h // g], v[at, h // g]
            s = kk @ q[i, h] * scale
            if np.isnan(s).any() or np.isnan(vv).any():
                out[i, h] = bound[i, h] = np.nan
                continue
            w = np.exp(s - s.max())
            w /= w.sum()
            mag = np.abs(kk) @ np.abs(q[i, h]) * abs(scale)
            delta = float(mag.max()) * (u + 2.0 ** -20) + \
                abs(scale) * float(np.abs(kk).sum(1).max()) * float(np.abs(q[i, h]).max()) * 2.0 ** -24
            out[i, h] = w @ vv
            bound[i, h] = (np.expm1(2 * delta) + 2.5 * u) * (w @ np.abs(vv)) + 1e-7
    return out, bound
