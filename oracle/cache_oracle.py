"""CPU oracle for the rotary tables, the paged cache and the decode over its
8-bit form: the definitions in numpy, fp64 (80-bit for angles).

TEST INFRASTRUCTURE ONLY, like ``attention_oracle``: the tests compare the
kernels with it, nothing in the library imports it.
"""
from __future__ import annotations

import math

import numpy as np

PI = np.longdouble("3.14159265358979323846264338327950288")


def e4m3_values():
    """The 256 values of e4m3 (sign, 4 exponent bits of bias 7, 3 mantissa bits; 0x7f and 0xff are NaN)."""
    c = np.arange(256)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e > 0, (1 + m / 8.0) * 2.0 ** (e - 7.0), m / 8.0 * 2.0 ** -6)
    v[(c & 127) == 127] = np.nan
    return np.where(c > 127, -v, v)


def to_e4m3(y):
    """Codes of the nearest e4m3 values, ties to even; |y| <= 448 or NaN."""
    y = np.asarray(y, np.float64)
    mag = np.abs(y)
    _, e = np.frexp(mag)
    q = 2.0 ** (np.maximum(e - 1, -6) - 3.0)
    near = np.rint(mag / q) * q
    table = e4m3_values()[:127]
    code = np.searchsorted(table, np.where(np.isnan(near), 0.0, near)).astype(np.uint8)
    code = np.where(np.isnan(y), 127, code).astype(np.uint8)
    return code | np.where(np.signbit(y) & ~np.isnan(y), 128, 0).astype(np.uint8)


def quantise_rows(x):
    """(codes, scale bytes) of rows x[..., D] (fp32 values): e the smallest integer
    with max|x| <= 448 * 2^e over the finite elements, in [-100, 120], 0 for zeros."""
    x = np.asarray(x, np.float64)
    top = np.where(np.isfinite(x), np.abs(x), 0.0).max(-1)
    m, e = np.frexp(top)                     # top = m 2^e, 448 = 0.875 * 2^9
    e = np.where(m > 0.875, e - 8, e - 9)
    e = np.where(top > 0, np.clip(e, -100, 120), 0)
    y = np.where(np.isfinite(x), x, np.nan) * 2.0 ** -e[..., None].astype(np.float64)
    return to_e4m3(y), (e + 127).astype(np.uint8)


def cache_values(codes, scale_bytes):
    """code * 2^(byte - 127), fp64; scale_bytes without the last axis of codes."""
    return e4m3_values()[codes] * 2.0 ** (scale_bytes.astype(np.float64) - 127)[..., None]


def frequencies(R, base, scaling="none", factor=1.0, original_length=0.0):
    """Radians per position of the R / 2 pairs (80-bit) and the factor on cos and sin."""
    L = np.longdouble
    i = np.arange(R // 2, dtype=L)
    b = L(base)
    if scaling == "ntk":
        b = b * L(factor) ** (L(R) / (R - 2))
    f = np.exp(-2 * i / R * np.log(b))
    if scaling == "linear":
        f = f / L(factor)
    elif scaling == "yarn":
        pair = [R * math.log(original_length / (2 * math.pi * n)) / (2 * math.log(base)) for n in (32.0, 1.0)]
        lo, hi = max(math.floor(pair[0]), 0), min(math.ceil(pair[1]), R - 1)
        r = np.clip((i - lo) / L(hi - lo if hi != lo else 0.001), 0, 1)
        return f / L(factor) * r + f * (1 - r), 0.1 * math.log(factor) + 1 if factor > 1 else 1.0
    elif scaling == "bands":
        r = np.clip((L(original_length) * f / (2 * PI) - 1) / 3, 0, 1)
        f = f / L(factor) * (1 - r) + f * r
    return f, 1.0


def table(first, length, R, base=10000.0, **scaling):
    """fp64 cos | sin table."""
    f, m = frequencies(R, base, **scaling)
    a = np.arange(first, first + length).astype(np.longdouble)[:, None] * f[None]
    return (np.concatenate([np.cos(a), np.sin(a)], 1) * m).astype(np.float64)


def rotate(x, pos, tab, interleaved, inverse=False, dtype=np.float64):
    """x [..., tokens, D] with pos [tokens] (or broadcastable over the leading axes), in `dtype` arithmetic."""
    x = np.asarray(x, dtype)
    R = tab.shape[1]
    inside = (pos >= 0) & (pos < tab.shape[0])
    row = tab[np.where(inside, pos, 0)].astype(dtype)
    c, s = row[..., :R // 2], row[..., R // 2:]
    s = -s if inverse else s
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if interleaved else (x[..., :R // 2], x[..., R // 2:R])
    y = x.copy()
    u, w = a * c - b * s, a * s + b * c
    if interleaved:
        y[..., 0:R:2], y[..., 1:R:2] = u, w
    else:
        y[..., :R // 2], y[..., R // 2:R] = u, w
    return np.where(inside[..., None], y, x)


def decode(q, k, v, scale):
    """One sequence: q [Hq, D], k, v [L, Hkv, D] fp64 -> O [Hq, D], LSE [Hq], and for
    the error bounds sum p|v| [Hq, D] and max_t scale * sum|q k| [Hq]."""
    Hq, D = q.shape
    L, Hkv, _ = k.shape
    G = Hq // Hkv
    if L == 0:
        return np.zeros((Hq, D)), np.full(Hq, -np.inf), np.zeros((Hq, D)), np.zeros(Hq)
    kk, vv = np.repeat(k, G, 1), np.repeat(v, G, 1)
    x = np.einsum("hd,lhd->hl", q, kk) * scale
    top = x.max(-1, keepdims=True)
    p = np.exp(x - top)
    tot = p.sum(-1, keepdims=True)
    p = p / tot
    size = np.einsum("hd,lhd->hl", np.abs(q), np.abs(kk)).max(-1) * scale
    return (np.einsum("hl,lhd->hd", p, vv), (top + np.log(tot))[:, 0], np.einsum("hl,lhd->hd", p, np.abs(vv)), size)
