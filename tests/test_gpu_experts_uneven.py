"""The experts' products (Experts.apply) over matrices with a few rows far larger than the others: what the others give keeps its digits.

Held is the 2-norm of the errors, of the results' columns but the large one, to what independent roundings come to at most, each taken as
large as it can be: half a step of every product's operands, of the activation and of a partial sum (sums of N terms: N roundings, each
of a sum that is in the root mean square no larger than the root of the terms' squares), carried on by the formula's derivatives.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

import experts_ref as ref
from jax4j_amd import Experts, QuantType
from jax4j_amd import synthetic as S
from test_gpu_experts import TYPES, apply

pytestmark = pytest.mark.gpu
SCALES = {"Q8_0": (34, (0,)), "Q4_0": (18, (0,)), "Q4_K": (144, (0, 2)), "Q6_K": (210, (208,))}  # a block's bytes, where its fp16 scales are
ROW, COLUMN = 37, 21  # the large row of gate and up, and of down


class Uneven:
    """Experts whose gate and up have one row `inner` times larger, and their down one `outer` times."""

    def __init__(self, backend, up, down, experts, dim, ffn, inner, outer, act="silu"):
        self.be, self.act, self.n, self.dim, self.ffn = backend, act, experts, dim, ffn
        self.kept, self.plain = [], []
        for i, (kind, rows, cols, at, factor) in enumerate(((up, ffn, dim, ROW, inner), (up, ffn, dim, ROW, inner), (down, dim, ffn, COLUMN, outer))):
            qt = QuantType[kind]
            size, places = SCALES[kind]
            blocks = np.array(S.quant_blocks(qt, 70 + i, experts * rows, cols), np.uint8).reshape(experts, rows, -1, size)
            for p in places:
                d = np.ascontiguousarray(blocks[:, at, :, p:p + 2]).view(np.float16)
                blocks[:, at, :, p:p + 2] = (d.astype(np.float32) * factor).astype(np.float16).view(np.uint8)
            blocks = blocks.reshape(-1)
            self.kept.append(backend.upload_quantized(blocks, qt, (experts * rows, cols)))
            self.plain.append(tuple(v.reshape(experts, rows, cols) for v in ref.dequantize(blocks, qt, experts * rows, cols)))
        self.experts = Experts(backend, *self.kept, experts=experts, activation=act)

    def close(self):
        self.experts.destroy()
        for w in self.kept:
            self.be.release(w)


@pytest.fixture(scope="module")
def layer(backend):
    made = {}

    def get(*key):
        if key not in made:
            made[key] = Uneven(backend, *key)
        return made[key]

    yield get
    for l in made.values():
        l.close()


def results(l, x, ids, kind):
    """Of rows with one expert each and weight 1: the results, their errors' size, and which rows have the large row's gate closed."""
    y, off, closed = np.zeros(x.shape), np.zeros(x.shape), np.zeros(len(x), bool)
    half = kind == "bf16"
    step = 2.0 ** -11 if half else 2.0 ** -22  # of x in fp32, the weights, the inner activations

    def product(w, part, v, ev):
        n = v.shape[1] * 9 / 8 + 40
        return v @ w.T, np.sqrt((v * v) @ (part * part).T * (2 * step ** 2 + n * 2.0 ** -48) + (ev * ev) @ (w * w).T)

    for e in range(l.n):
        at = np.where(ids[:, 0] == e)[0]
        xr = x[at].astype(np.float64)
        (gate, pg), (up, pu), (down, pd) = ((m[0][e], m[1][e]) for m in l.plain)
        g, eg = product(gate, pg, xr, np.zeros(xr.shape))
        u, eu = product(up, pu, xr, np.zeros(xr.shape))
        with np.errstate(over="ignore"):
            a = ref._activate(g, l.act)
        slope = np.minimum(1.13, 1.13 * np.exp(np.minimum(g + 2, 0)))  # of silu: at most 1.1, and below -2 at most e^g (1 - g) < e^(g + 2)
        ea = np.sqrt((slope * eg) ** 2 + (8 * 2.0 ** -24 * a) ** 2)
        h = a * u
        eh = np.sqrt((ea * u) ** 2 + (a * eu) ** 2 + (ea * eu) ** 2 + (step * h) ** 2)
        y[at], off[at] = product(down, pd, h, eh)
        closed[at] = g[:, ROW] < -30
    if half:
        off = np.hypot(off, 2.0 ** -11 * np.abs(y)) + ref.STEP["bf16"] * np.abs(y)
    return y, off, closed


@pytest.mark.parametrize("up,down", [("Q8_0", "Q8_0"), ("Q4_0", "Q4_0"), ("Q4_K", "Q6_K"), ("Q6_K", "Q4_K")])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("inner,outer", [(1, 1), (32, 32), (256, 1), (256, 256)])
def test_other_rows_keep_their_digits(layer, up, down, kind, inner, outer):
    l = layer(up, down, 2, 1024, 512, inner, outer)
    for rows in (1, 20, 120, 420):  # the kernels of one row, of few pairs and of many
        rng = np.random.default_rng(rows)
        x = torch.from_numpy(rng.standard_normal((rows, l.dim)).astype(np.float32)).to(TYPES[kind][1])
        ids = (np.arange(rows, dtype=np.int32) % 2)[:, None]
        got = apply(l, x, ids, np.ones((rows, 1), np.float32), kind)
        want, off, closed = results(l, x.float().numpy(), ids, kind)
        others = np.arange(l.dim) != COLUMN
        for some in (np.ones(rows, bool), closed) if inner > 1 else (np.ones(rows, bool),):
            at = np.ix_(some, others)
            error, bound = np.linalg.norm((got - want)[at]), np.linalg.norm(off[at])
            print(f"{rows} rows, {some.sum()} of them: {error / np.linalg.norm(want[at]):.2e}, bound {bound / np.linalg.norm(want[at]):.2e}")
            assert error <= bound or not some.any(), (rows, error, bound)
            own = np.abs(got - want)[some][:, COLUMN]
            assert np.linalg.norm(own) <= 4 * np.linalg.norm(off[some][:, COLUMN]), rows  # few values: four times the root mean square


@pytest.mark.parametrize("up,down", [("Q8_0", "Q8_0"), ("Q4_0", "Q4_0"), ("Q4_K", "Q6_K"), ("Q6_K", "Q4_K")])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("value", [np.inf, np.nan])
def test_a_row_of_down_that_is_not_finite_stays_alone(backend, up, down, kind, value):
    with np.errstate(invalid="ignore"):  # inf times 0
        l = Uneven(backend, up, down, 2, 256, 512, 1, value)
    try:
        others = np.arange(l.dim) != COLUMN
        l.plain[2] = tuple(np.where(others[None, :, None], v, 0.0) for v in l.plain[2])
        for rows in (1, 20, 120):
            rng = np.random.default_rng(rows)
            x = torch.from_numpy(rng.standard_normal((rows, l.dim)).astype(np.float32)).to(TYPES[kind][1])
            ids = (np.arange(rows, dtype=np.int32) % 2)[:, None]
            got = apply(l, x, ids, np.ones((rows, 1), np.float32), kind)
            assert not np.isfinite(got[:, COLUMN]).any()
            want, off, _ = results(l, x.float().numpy(), ids, kind)
            assert np.linalg.norm((got - want)[:, others]) <= np.linalg.norm(off[:, others]), rows
    finally:
        l.close()
