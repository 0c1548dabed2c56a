"""The 8-bit key/value cache and its attention in plain numpy: what the kernels are held to."""
from __future__ import annotations

import numpy as np

BLOCK, TINY = 16, np.float32(2.0 ** -64)


def rotate(x, cos, sin, at, interleaved):
    """x [rows, heads, dim] fp32, at [rows, pairs] positions: every product and sum rounded to fp32."""
    y, pairs = x.astype(np.float32).copy(), cos.shape[1]
    pair = np.arange(pairs)
    ok = (at >= 0) & (at < cos.shape[0])
    safe = np.where(ok, at, 0)
    c, s = (np.where(ok, t[safe, pair], np.float32(np.nan))[:, None] for t in (cos, sin))
    u, w = (y[..., 0:2 * pairs:2], y[..., 1:2 * pairs:2]) if interleaved else (y[..., :pairs], y[..., pairs:2 * pairs])
    a, b = u * c - w * s, w * c + u * s
    u[...], w[...] = a, b
    return y


def tables(rows, pairs):
    angle = np.arange(rows)[:, None] * 10000.0 ** (-np.arange(pairs) / pairs)
    return np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)


def to_bf16(x):
    """fp32 as the bf16 bits of the nearest value, ties to even."""
    u = np.asarray(x, np.float32).view(np.uint32)
    return ((u + 0x7FFF + (u >> 16 & 1)) >> 16).astype(np.uint16)


def from_bf16(b):
    return (b.astype(np.uint32) << 16).view(np.float32)


class Held:
    """Codes [tokens, heads, dim] and scales [blocks, heads] of one sequence's keys or values in one layer."""

    def __init__(self, heads, dim):
        self.codes, self.scale = np.zeros((0, heads, dim), np.float32), np.zeros((0, heads), np.float32)

    def copy(self):
        h = Held(*self.codes.shape[1:])
        h.codes, h.scale = self.codes.copy(), self.scale.copy()
        return h

    def cut(self, n):
        self.codes, self.scale = self.codes[:n], self.scale[:-(-n // BLOCK)]

    def append(self, x):
        at, heads = self.codes.shape[0], x.shape[1]
        self.codes = np.concatenate([self.codes, np.zeros(x.shape, np.float32)])
        blocks = -(-self.codes.shape[0] // BLOCK)
        self.scale = np.concatenate([self.scale, np.zeros((blocks - self.scale.shape[0], heads), np.float32)])
        for b in range(at // BLOCK, blocks):
            lo, hi = max(at, b * BLOCK), min(self.codes.shape[0], (b + 1) * BLOCK)
            for h in range(heads):
                rows = x[lo - at:hi - at, h].astype(np.float32)
                if not np.isfinite(rows).all():
                    self.scale[b, h] = np.nan
                top = np.abs(rows).max()
                s = self.scale[b, h]
                if s != s:
                    self.codes[lo:hi, h] = 0
                    continue
                if lo == b * BLOCK or s <= TINY:
                    was, s = s, max(top / np.float32(127), TINY)
                    if lo > b * BLOCK:
                        self.codes[b * BLOCK:lo, h] = np.rint(self.codes[b * BLOCK:lo, h] * np.float32(was / s))
                else:
                    k = 0
                    while np.float32(top * np.float32(0.5) ** k) * (np.float32(1) / s) >= np.float32(127.5):
                        k += 1
                    f = np.float32(2.0 ** -k)
                    self.codes[b * BLOCK:lo, h] = np.rint(self.codes[b * BLOCK:lo, h] * f)
                    s = s / f
                self.scale[b, h] = s
                self.codes[lo:hi, h] = np.rint(rows * (np.float32(1) / s))

    def values(self, first=0, count=None):
        """fp32 [count, heads, dim]; zeros behind the end."""
        n = self.codes.shape[0]
        v = self.codes * np.repeat(self.scale, BLOCK, 0)[:n, :, None]
        count = n - first if count is None else count
        out = np.zeros((count, *v.shape[1:]), np.float32)
        part = v[first:first + count]
        out[:part.shape[0]] = part
        return out


def attend(q, k, v, first, window=0, sinks=0, scale=None):
    """Rows q [rows, heads, dim] at places first.. to k, v [tokens, kv heads, dim], in 64 bits: the result, the largest |score|
    (as a power of two), and the largest sum of |q k| (times the scale)."""
    q, k, v = (x.astype(np.float64) for x in (q, k, v))
    rows, heads, dim = q.shape
    g = heads // k.shape[1]
    out, top, total = np.zeros_like(q), 0.0, 0.0
    p, j = first + np.arange(rows)[:, None], np.arange(k.shape[0])[None]
    seen = j <= p
    if window:
        seen &= (j > p - window) | (j < sinks)
    for h in range(heads):
        a = scale or dim ** -0.5
        s = q[:, h] @ k[:, h // g].T * a
        with np.errstate(invalid="ignore", over="ignore"):
            s = np.where(seen, s, -np.inf)
            w = np.exp(s - np.where(np.isnan(s), -np.inf, s).max(1, keepdims=True))
            bad = np.isnan(s).any(1) | (seen & np.isnan(v[:, h // g]).any(1)).any(1)
            o = np.where(w[..., None] > 0, w[..., None] * np.where(seen[..., None], v[:, h // g], 0), 0).sum(1) / w.sum(1, keepdims=True)
        out[:, h] = np.where(bad[:, None], np.nan, o)
        top = max(top, float(np.abs(s[np.isfinite(s)]).max(initial=0)) / np.log(2))
        total = max(total, float(np.nanmax(np.abs(q[:, h]) @ np.abs(k[:, h // g]).T * a, initial=0)))
    return out, top, total
