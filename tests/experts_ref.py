"""Norms, routing and the experts' products in plain numpy and 64 bits, and how far the kernels may be off, from their arithmetic alone."""
from __future__ import annotations

import numpy as np

import oracle
from jax4j_amd import QuantType

STEP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8}  # half a step of a rounding, relative to the value


def to_bf16(x):
    u = np.asarray(x, np.float32).view(np.uint32)
    return ((u + 0x7FFF + (u >> 16 & 1)) >> 16).astype(np.uint16)


def from_bf16(b):
    return (np.asarray(b).astype(np.uint32) << 16).view(np.float32)


# ---- norms -----------------------------------------------------------------------------------


def _norm(x, ex, n):
    """A norm (kind, weight, bias, eps, add) of rows x that are known to within ex; and how far its 32-bit result may be off."""
    kind, weight, bias, eps, add = n
    w = np.ones(x.shape[1]) if weight is None else weight.astype(np.float64) + add
    b = np.zeros(x.shape[1]) if bias is None else bias.astype(np.float64)
    mean = x.mean(1, keepdims=True) if kind == "layer" else 0.0
    em = ex.mean(1, keepdims=True) if kind == "layer" else 0.0
    d = x - mean
    rms = np.sqrt((d * d).mean(1, keepdims=True) + eps)
    y = d / rms * w + b
    # the root of a mean of squares moves by no more than the root of the mean square of what moves the values
    er = np.sqrt(((ex + em) ** 2).mean(1, keepdims=True))
    off = np.abs(w) / rms * (ex + em + np.abs(d) / rms * er)
    # d, 1 / rms, their product, weight + add, the product with it, the sum with the bias: six roundings
    return y, off + 6 * STEP["f32"] * (np.abs(d / rms * w) + np.abs(b))


def norm(residual, block, gate, gate_every, scale, after, before):
    """(h, its error, before(h) or None, its error), before any rounding of the results."""
    rows, dim = (block if residual is None else residual).shape
    h, e = np.zeros((rows, dim)), np.zeros((rows, dim))
    if block is not None:
        h = block.astype(np.float64)
        if after is not None:
            h, e = _norm(h, e, after)
        if gate is not None:
            g = gate.astype(np.float64)[np.arange(rows) // gate_every if gate_every else np.zeros(rows, int)]
            h, e = h * g, e * np.abs(g)
        h, e = h * scale, (e + 2 * STEP["f32"] * np.abs(h)) * abs(scale)
    if residual is not None:
        r = residual.astype(np.float64)
        e = e + STEP["f32"] * (np.abs(h) + np.abs(r))
        h = h + r
    if before is None:
        return h, e, None, None
    return (h, e, *_norm(h, e, before))


# ---- routing ---------------------------------------------------------------------------------


def route(logits, k, score, bias=None, groups=1, top_groups=1, best=1, renormalize=False, scale=1.0):
    """ids and weights [rows, k], row by row."""
    rows, experts = logits.shape
    ids, weights = np.full((rows, k), -1, np.int32), np.zeros((rows, k))
    for r in range(rows):
        x = logits[r].astype(np.float64)
        live = ~np.isnan(x) & (x > -np.inf)
        s, log = np.zeros(experts), np.zeros(experts)
        if live.any():
            top = x[live].max()
            if score == "softmax":
                log[live] = np.where(x[live] == top, 0.0, x[live] - top) if np.isinf(top) else x[live] - top
                total = np.exp(log[live]).sum()
                s[live] = np.exp(log[live]) / total
            else:
                log[live] = -np.logaddexp(0.0, -x[live])
                s[live] = np.exp(log[live])
        key = x if bias is None else s + bias.astype(np.float64)
        with np.errstate(invalid="ignore"):
            live &= ~np.isnan(key) & (key > -np.inf)
        if groups > 1:
            size = experts // groups
            rank = []
            for g in range(groups):
                inside = np.sort(key[g * size:(g + 1) * size][live[g * size:(g + 1) * size]])[::-1][:best]
                rank.append(inside.sum() if inside.size else -np.inf)
            kept = sorted(range(groups), key=lambda g: (-rank[g], g))[:top_groups]
            live &= np.isin(np.arange(experts) // size, kept)
        at = np.where(live)[0]
        at = at[np.lexsort((at, -key[at]))][:k]
        ids[r, :at.size] = at
        if renormalize and at.size:
            w = np.exp(log[at] - log[at].max())
            weights[r, :at.size] = scale * w / w.sum()
        else:
            weights[r, :at.size] = scale * s[at]
    return ids, weights


# ---- the experts' products -------------------------------------------------------------------


def dequantize(blocks, qt: QuantType, rows, cols):
    """Weights [rows, cols], and what their sums are made of: with minima |scale code| + |minimum|, else |weight|."""
    w = oracle.dequant_matrix(qt.id, blocks, rows, cols).astype(np.float64)
    if qt is not QuantType.Q4_K:
        return w, np.abs(w)
    b = np.array(blocks, np.uint8).reshape(-1, 144)
    b[:, 2:4] = 0
    part = oracle.dequant_matrix(qt.id, b.reshape(-1), rows, cols).astype(np.float64)
    return w, np.abs(part) + np.abs(part - w)


def _activate(x, name):
    if name == "relu":
        return np.maximum(x, 0.0)
    if name == "gelu":
        return 0.5 * x * (1 + np.tanh(np.sqrt(2 / np.pi) * (x + 0.044715 * x ** 3)))
    return x / (1 + np.exp(-x))


def experts(x, ids, weights, gate, up, down, act, kind, exact_weights):
    """x [rows, dim]; of each matrix the weights and their parts, [experts, rows, cols] each; the results and how far the kernels may be off.

    Of a product over K: x as hi + lo has 22 bits (bf16 x is exact), below 2^-18 of the row's largest value an absolute error of
    2^-40 of it; weights are exact, or rounded to 11 bits; a sum of K products in 32 bits, a rounding for each, and for each block's scale, its
    minimum and what a wave or split adds: K + K / 8 + 40 of them at most. The inner activations have 22 or 11 bits, below the normal range
    2^-25 at a power that takes their bound |x|^2 G U to 2^14; the activation and the product with up: the slope of an activation is at
    most 1.13, its exponential is within 3 half steps, its reciprocal 2, and three roundings more. For results in bf16 a pair's share is rounded to 11 bits, below the normal range
    2^-25 at a power that takes its bound |x|^2 G U D sqrt(ffn), rounded up by 2^5 at most, to 2^14."""
    t, top = ids.shape
    half = kind == "bf16"
    y, off = np.zeros(x.shape), np.zeros(x.shape)
    few = lambda k: (k + k / 8 + 40) * STEP["f32"] + (0.0 if exact_weights else 2.0 ** (-11 if half else -21))  # noqa: E731
    for r in range(t):
        xr = x[r].astype(np.float64)
        ax, largest = np.abs(xr), np.abs(xr).max()
        ex = 0.0 if half else np.maximum(2.0 ** -22 * ax, 2.0 ** -40 * largest)
        for s in range(top):
            e = ids[r, s]
            if not 0 <= e < gate[0].shape[0]:
                continue
            ag, au, ad = gate[1][e], up[1][e], down[1][e]
            g, u = gate[0][e] @ xr, up[0][e] @ xr
            eg, eu = ag @ (few(xr.size) * ax + ex), au @ (few(xr.size) * ax + ex)
            a = _activate(g, act)
            h = a * u
            ea = 1.13 * eg + 8 * STEP["f32"] * (np.abs(a) + np.minimum(np.abs(g), 1.0) * (act != "relu"))
            bound = (xr @ xr) * np.sqrt((gate[0][e] ** 2).sum(1).max() * (up[0][e] ** 2).sum(1).max())
            eh = ea * (np.abs(u) + eu) + np.abs(a) * eu + 3 * STEP["f32"] * np.abs(h)
            eh = eh + np.maximum((2.0 ** -11 if half else 2.0 ** -22) * np.abs(h), 2.0 ** (-25 - 14 + 3) * bound)
            part, ep = down[0][e] @ h, ad @ (few(h.size) * np.abs(h) + eh)
            if half:
                ep = ep + np.maximum(2.0 ** -11 * np.abs(part), 2.0 ** (-25 - 14 + 5) * bound * np.sqrt(h.size * (down[0][e] ** 2).sum(1).max()))
            w = float(weights[r, s])
            y[r] += w * part
            off[r] += abs(w) * (ep + (top + 1) * STEP["f32"] * np.abs(part))
    return y, off
