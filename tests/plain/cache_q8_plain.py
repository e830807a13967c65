"""A key-value cache in 8 bits by its definition, in float64 NumPy.

Test-only oracle: codes and scales laid out value by value, rotation, reading back and attention of one token; nothing is
shared with the engine.
"""
from __future__ import annotations

import numpy as np

TOP = {0: 127.0, 1: 448.0}


def numbers(codes, form):
    """What 8-bit codes stand for: whole numbers (0), or 8-bit floats with 4 exponent and 3 mantissa bits, bias 7 (1)."""
    codes = np.asarray(codes, np.uint8)
    if form == 0:
        return codes.view(np.int8).astype(np.float64)
    e, m = (codes >> 3 & 15).astype(np.float64), (codes & 7).astype(np.float64)
    x = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10))
    x = np.where(codes & 127 == 127, np.nan, x)
    return np.where(codes & 128, -x, x)


def half_step(x, scale, form):
    """Half the distance of the numbers around x that codes of this scale stand for."""
    if form == 0:
        return np.broadcast_to(scale / 2, x.shape)
    return np.maximum(np.abs(x) * 2.0 ** -4, scale * 2.0 ** -10)


class Cache:
    def __init__(self, pages, nkv, hd, bs, form):
        self.pages, self.nkv, self.hd, self.bs, self.form, self.blocks = pages, nkv, hd, bs, form, -(-hd // 64)
        self.k = np.zeros((pages, nkv, bs // 16, self.blocks, 1024), np.uint8)
        self.v = np.zeros_like(self.k)
        self.scales = np.zeros((pages, nkv, 2, bs), np.float32)

    def places(self, off, values):
        """(block, byte of the block) of every channel of the token at ``off`` of a page's piece."""
        c, t = np.arange(self.hd), off % 16
        within = c % 64
        at = t // 4 * 256 + within % 16 * 16 + within // 16 * 4 + t % 4 if values else t * 64 + within
        return c // 64, at

    def codes_at(self, page, head, off, values):
        block, at = self.places(off, values)
        return (self.v if values else self.k)[page, head, off // 16, block, at]

    def put(self, page, head, off, values, codes, scale):
        block, at = self.places(off, values)
        (self.v if values else self.k)[page, head, off // 16, block, at] = codes
        self.scales[page, head, int(values), off] = scale

    def row(self, page, head, off, values):
        """The float64 numbers that a token's head stands for."""
        return numbers(self.codes_at(page, head, off, values), self.form) * np.float64(self.scales[page, head, int(values), off])

    def rows(self, table, begin, end, values):
        """[nkv, end - begin, hd] at the positions of a request's table; NaN where it names no page."""
        out = np.full((self.nkv, end - begin, self.hd), np.nan)
        for j in range(begin, end):
            page = table[j // self.bs]
            if 0 <= page < self.pages:
                for h in range(self.nkv):
                    out[h, j - begin] = self.row(page, h, j % self.bs, values)
        return out


def rotate(x, positions, inv_freq, rotary_dim):
    """[T, heads, hd]: pairs (i, i + rotary_dim / 2) turned by position times frequency."""
    half = rotary_dim // 2
    angle = np.asarray(positions, np.float64)[:, None] * np.asarray(inv_freq, np.float64)[None, :half]
    cos, sin = np.cos(angle)[:, None], np.sin(angle)[:, None]
    a, b = x[..., :half], x[..., half:rotary_dim]
    return np.concatenate([a * cos - b * sin, b * cos + a * sin, x[..., rotary_dim:]], axis=-1)


def attention(q, keys, values, scale, cap):
    """q [nh, hd] over keys and values [nkv, n, hd], rows that are NaN left out: (out, sum of p |v|, the scores, |q| . |k|)."""
    nh, nkv = q.shape[0], keys.shape[0]
    out, spread = np.zeros(q.shape), np.zeros(q.shape)
    most = 0.0
    for h in range(nh):
        k, v = keys[h // (nh // nkv)], values[h // (nh // nkv)]
        seen = ~np.isnan(k).any(axis=1)
        if not seen.any():
            continue
        k, v = k[seen], v[seen]
        z = k @ q[h] * scale
        most = max(most, float((np.abs(k) @ np.abs(q[h])).max()) * abs(scale))
        if cap:
            z = cap * np.tanh(z / cap)
        p = np.exp(z - z.max())
        p /= p.sum()
        out[h], spread[h] = p @ v, p @ np.abs(v)
    return out, spread, most
