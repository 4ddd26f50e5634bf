"""Plain 64-bit forms of the operators around an 8-bit paged cache, and the bounds their
kernels are held to (half a step per rounding, from the arithmetic each one does)."""
from __future__ import annotations

import numpy as np

from kvcache_amd import KVC_E4M3, KVC_F16, KVC_I8

TOP = {KVC_I8: 127.0, KVC_E4M3: 448.0}
NAME = {KVC_F16: "f16", KVC_I8: "i8", KVC_E4M3: "e4m3"}
H16 = 2.0 ** -11   # half a step of fp16, relative
E32 = 2.0 ** -24   # ... of fp32


def _e4m3_table():
    x = np.arange(256)
    e, f = (x >> 3) & 15, x & 7
    v = np.where(e == 0, f * 2.0 ** -9, (1 + f / 8) * 2.0 ** (e - 7.0))
    v = np.where((x & 127) == 127, np.nan, v)
    return np.where(x & 128, -v, v)


E4M3 = _e4m3_table()


def values(codes, kv_dtype):
    """The numbers that codes stand for, in 64 bits."""
    if kv_dtype == KVC_E4M3:
        return E4M3[codes.view(np.uint8)]
    return codes.astype(np.float64)


def code_dtype(kv_dtype):
    return {KVC_F16: np.float16, KVC_I8: np.int8, KVC_E4M3: np.uint8}[kv_dtype]


def round_e4m3(y):
    """Nearest e4m3 value, half to even, of |y| <= 448."""
    a = np.abs(y)
    e = np.maximum(np.floor(np.log2(np.maximum(a, 1e-30))), -6)
    step = 2.0 ** (e - 3)
    return np.rint(y / step) * step


def half_step(y, s, kv_dtype):
    """Half a step of the code that holds y under the scale s (broadcast over D)."""
    if kv_dtype == KVC_I8:
        return 0.5 * s + 0 * y
    with np.errstate(divide="ignore", invalid="ignore"):
        a = np.where(s > 0, np.abs(y) / np.where(s > 0, s, 1), 0)
    e = np.maximum(np.floor(np.log2(np.maximum(a, 1e-30))), -6)
    return 0.5 * 2.0 ** (e - 3) * s


def quantise(x, kv_dtype):
    """(codes as they lie in a pool, fp32 scales) of rows [..., D]: for making caches."""
    x = np.asarray(x, np.float64)
    s = (np.abs(x).max(-1) / TOP[kv_dtype]).astype(np.float32)
    y = x / np.where(s > 0, s, 1)[..., None]
    if kv_dtype == KVC_I8:
        return np.clip(np.rint(y), -127, 127).astype(np.int8), s
    v = round_e4m3(np.clip(y, -448, 448))
    order = np.argsort(E4M3[:127])
    mag = order[np.searchsorted(E4M3[:127][order], np.abs(v))]
    return (mag | np.where(np.signbit(v), 128, 0)).astype(np.uint8), s


def norm_rope(x, w, eps, pos, theta):
    """x [M, heads, D]: RMSNorm with weight w (None: none), rotary at pos [M]; 64 bits."""
    x = np.asarray(x, np.float64)
    d = x.shape[-1]
    if w is not None:
        x = x / np.sqrt((x ** 2).mean(-1, keepdims=True) + eps) * np.asarray(w, np.float64)
    ang = np.asarray(pos, np.float64)[:, None] * theta ** (-2.0 * np.arange(d // 2) / d)
    c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
    a, b = x[..., : d // 2], x[..., d // 2:]
    size = np.abs(a) + np.abs(b)
    return np.concatenate([a * c - b * s, b * c + a * s], -1), np.concatenate([size, size], -1)


def norm_rope_bound(size, d):
    """fp32 error of a normed and rotated value: the sum of squares adds d terms in d / 16 lanes
    (16 + 4 roundings), then a root, a quotient, two products (5), sine and cosine (an angle of a
    turn rounded once, 2 pi 2^-25, and 3 steps of their own), two products and a sum (3)."""
    return size * (20 + 5 + 8 + 6 + 3) * E32


def chunk_attention(q, k, v, n, window, cap, scale):
    """q [n, Hq, D] (the last n tokens), k, v [t, Hkv, D] of one sequence, 64 bits.  Returns
    out, sum_j p_j |v_j| and max_j of scale sum_d |q_d k_d| over the keys a row sees."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    t, hkv, d = k.shape
    hq = q.shape[1]
    out, mag, big = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape[:2])
    for i in range(n):
        p = t - n + i
        lo = max(0, p - window + 1) if window else 0
        for h in range(hq):
            kk, vv = k[lo:p + 1, h // (hq // hkv)], v[lo:p + 1, h // (hq // hkv)]
            z = kk @ q[i, h] * scale
            if cap:
                z = cap * np.tanh(z / cap)
            e = np.exp(z - z.max())
            e /= e.sum()
            out[i, h], mag[i, h] = e @ vv, e @ np.abs(vv)
            big[i, h] = (np.abs(kk) @ np.abs(q[i, h])).max() * abs(scale)
    return out, mag, big


def chunk_bound(out, mag, big, d, cap, *, p16=True, kv16=False):
    """p16: probabilities are rounded to fp16; kv16: dequantised K and V are.  A score off by e
    moves the result by at most 2 e sum p |v|: e is d roundings of the sum (fp32), one of K where
    it is rounded, and what the cap's quotient loses (2 cap 2^-21)."""
    e = big * (d * E32 + (H16 if kv16 else 0)) + 2.0 ** -20 + 2 * cap * 2.0 ** -21
    rel = (H16 if p16 else 0) + (H16 if kv16 else 0) + 2.0 ** -18
    return mag * (rel + 2 * e[..., None]) + np.abs(out) * H16 + 2.0 ** -24
