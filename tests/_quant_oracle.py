"""Plain numpy definitions, in 64 bits, of the quantised decode step: 4-bit weights, the 8-bit
cache and the draw of a token."""
from __future__ import annotations

import numpy as np

F8_TOP = {"e4m3": 8, "e5m2": 15}
F8_CODES = {"e4m3": 127, "e5m2": 124}  # finite non-negative codes


# ---------------------------------------------------------------- 4-bit weights
def w4_unpack(q, in_f):
    """Packed rows -> codes [out_f, in_f], from the layout's statement."""
    q = np.asarray(q, np.uint8)
    codes = np.zeros((q.shape[0], q.shape[1] * 2), np.uint8)
    for c in range(4):
        for i in range(4):
            for b in range(4):
                byte = q[:, 16 * c + 4 * i + b::64]
                codes[:, 32 * i + 8 * c + 2 * b::128] = byte & 15
                codes[:, 32 * i + 8 * c + 2 * b + 1::128] = byte >> 4
    return codes[:, :in_f]


def w4_pack(codes):
    out_f, in_f = codes.shape
    blocks = -(-in_f // 128)
    pad = np.zeros((out_f, blocks * 128), np.uint8)
    pad[:, :in_f] = codes
    q = np.zeros((out_f, blocks * 64), np.uint8)
    for c in range(4):
        for i in range(4):
            for b in range(4):
                q[:, 16 * c + 4 * i + b::64] = (pad[:, 32 * i + 8 * c + 2 * b::128]
                                                | pad[:, 32 * i + 8 * c + 2 * b + 1::128] << 4)
    return q


def w4_weights(codes, scale, zero, group):
    """f64 W [out_f, in_f]."""
    in_f = codes.shape[1]
    g = np.arange(in_f) // group
    z = 8.0 if zero is None else zero[g].T.astype(np.float64)
    return (codes.astype(np.float64) - z) * np.asarray(scale, np.float64)[g].T


# ---------------------------------------------------------------- 8-bit cache
def f8_values(f8):
    """Values of the non-negative finite codes, ascending with the code."""
    bits, bias = (3, 7) if f8 == "e4m3" else (2, 15)
    c = np.arange(F8_CODES[f8])
    e, m = c >> bits, c & ((1 << bits) - 1)
    return np.where(e == 0, m * 2.0 ** (1 - bias - bits),
                    (1 + m / 2.0 ** bits) * 2.0 ** (e - bias))


def f8_encode(x, f8):
    """Nearest code, ties to even, saturating; NaN -> 0x7f."""
    x = np.asarray(x, np.float64)
    v = f8_values(f8)
    mid = (v[1:] + v[:-1]) / 2
    a = np.abs(np.where(np.isnan(x), 0, x))
    k = np.searchsorted(mid, a, side="left")
    tie = (k < len(mid)) & (a == mid[np.minimum(k, len(mid) - 1)]) & (k % 2 == 1)
    code = (k + tie).astype(np.uint8)
    code = np.where(np.signbit(x), code | 0x80, code)
    return np.where(np.isnan(x), code & 0x80 | 0x7F, code).astype(np.uint8)


def f8_decode(c, f8):
    c = np.asarray(c, np.uint8)
    v = np.full(128, np.nan)
    v[:F8_CODES[f8]] = f8_values(f8)
    if f8 == "e5m2":
        v[124] = np.inf
    return np.where(c & 0x80, -1.0, 1.0) * v[c & 0x7F]


def f8_need_scale(amax, f8):
    """Smallest power of two (2^-64 at least) that holds amax."""
    top = 1.75 * 2.0 ** F8_TOP[f8]
    amax = np.asarray(amax, np.float64)
    e = np.where(amax > 0, np.ceil(np.log2(np.maximum(amax, 1e-300) / top)), -64)
    return 2.0 ** np.maximum(e, -64)


def f8_step(x, scale, f8):
    """Distance of neighbouring values of the type, times scale, at |x|."""
    bits, low = (3, -6) if f8 == "e4m3" else (2, -14)
    e = np.floor(np.log2(np.maximum(np.abs(x) / scale, 2.0 ** low)))
    return 2.0 ** (e - bits) * scale


def kv8_write(codes, scale, start, rows, block, f8):
    """Rows [n, heads, hd] (f64, prepared) into codes [max_seq, heads, hd] (uint8) and scale
    [blocks, heads] (f64), both changed in place."""
    n = rows.shape[0]
    r = start
    while r < start + n:
        j = r // block
        end = min((j + 1) * block, start + n)
        part = rows[r - start:end - start]
        fin = np.where(np.isfinite(part), np.abs(part), 0)
        new = f8_need_scale(fin.max(axis=(0, 2)), f8)
        if r % block:
            new = np.maximum(new, scale[j])
            old = f8_decode(codes[j * block:r], f8)
            grown = f8_encode(old * (scale[j] / new)[:, None], f8)
            codes[j * block:r] = np.where((new != scale[j])[:, None], grown, codes[j * block:r])
        scale[j] = new
        codes[r:end] = f8_encode(part / new[:, None], f8)
        r = end


def row_norm(x, w, eps):
    x = np.asarray(x, np.float64)
    return x if w is None else x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w


def row_rope(x, cos, sin):
    """x [..., hd] with one table row per leading index (broadcast over heads)."""
    if cos is None:
        return x
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    return np.concatenate((a * cos - b * sin, b * cos + a * sin), -1)


def attend(q, K, V, scale):
    """q [H, hd], K and V [rows, heads, hd] (f64) -> o [H, hd], and a bound of the error that f32
    arithmetic may make: scores off by (hd + 8) roundings of the sum of their products'
    magnitudes, sums over the rows and the values' products another rows + 8."""
    H, hd = q.shape
    rows, heads, _ = K.shape
    g = H // heads
    o, bound = np.empty((H, hd)), np.empty((H, hd))
    for h in range(H):
        k, v = K[:, h // g], V[:, h // g]
        s = k @ q[h] * scale
        p = np.exp(s - s.max())
        p /= p.sum()
        o[h] = p @ v
        ds = (hd + 8) * 2.0 ** -24 * (np.abs(k) @ np.abs(q[h])) * scale
        bound[h] = (2 * ds.max() + (rows + 8) * 2.0 ** -24) * (p @ np.abs(v))
    return o, bound


# ---------------------------------------------------------------- sampling
def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One row's token id by the definition."""
    l = np.asarray(logits, np.float64)
    l = np.where(np.isnan(l), -np.inf, l)
    top = l.max()
    if top == -np.inf:
        return -1
    if not temperature > 0:
        return int(np.argmax(l))
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.exp((l - top) / float(np.float32(temperature)))
    w = np.where(l == top, 1.0, np.where(l == -np.inf, 0.0, w))
    w[w < 2.0 ** -60] = 0
    order = np.lexsort((np.arange(len(l)), -l))
    if top_k >= 1:
        order = order[:top_k]
    ws = w[order]
    if top_p < 1:
        before = np.concatenate(([0.0], np.cumsum(ws)[:-1]))
        keep = before < float(np.float32(top_p)) * ws.sum()
        keep[0] = True
        order, ws = order[keep], ws[keep]
    if min_p > 0:
        keep = (ws >= float(np.float32(min_p))) | (ws == 1.0)
        order, ws = order[keep], ws[keep]
    order = np.sort(order)
    run = np.cumsum(w[order])
    u = float(np.float32(u))
    u = 0.0 if not u > 0 else min(u, 1 - 2.0 ** -24)
    return int(order[np.flatnonzero((run > u * run[-1]) & (w[order] > 0))[0]])
