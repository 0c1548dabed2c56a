"""How near attention over the 8-bit cache comes to the formula in 64 bits, row by row, relative to the row's own size.

The bars of test_gpu_kv.py bound the worst case by the largest value of a sequence; a mean of thousands of values is far smaller
than that. Here an error is the 2-norm over a row's channels (or over some of them, with codes small beside the others')
of the difference, over that of the row.

A bf16 result is off by 2^-8 of each channel at most. Fp16 weights are off by 2^-11 of themselves at most, in any direction, so the
row by no more than that share of it (errors of one sign are a factor, others average as the values do). Queries are in bf16
here, which fp16 holds as they are; as whole numbers of 16 bits over the row's largest magnitude they are off by max|q| / 65200 in any
direction, at most, by 1/sqrt(3) of it in the mean square, so a score by d = scale |k| max|q| / 65200 / sqrt(3), and a row by as
much of its size; five times that covers the rows of a call.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

import kv_ref as R
from test_gpu_kv import KIND, dev_as, host, model  # noqa: F401

gpu = pytest.mark.gpu


def exact(q, k, v, first, window=0, sinks=0):
    """Rows q [rows, heads, dim] at places first.. to k, v [tokens, kv heads, dim], all finite, in 64 bits."""
    q, k, v = (x.astype(np.float64) for x in (q, k, v))
    rows, heads, dim = q.shape
    g, out = heads // k.shape[1], np.empty(q.shape)
    p, j = first + np.arange(rows)[:, None], np.arange(k.shape[0])[None]
    seen = j <= p
    if window:
        seen &= (j > p - window) | (j < sinks)
    for h in range(heads):
        s = np.where(seen, q[:, h] @ k[:, h // g].T * dim ** -0.5, -np.inf)
        w = np.exp(s - s.max(1, keepdims=True))
        out[:, h] = w @ v[:, h // g] / w.sum(1, keepdims=True)
    return out


def off(got, want, groups=None):
    """The largest error of a row and head, over each group of channels."""
    groups = [slice(None)] if groups is None else groups
    return max(float((np.linalg.norm((got - want)[..., g], axis=-1) / np.linalg.norm(want[..., g], axis=-1)).max()) for g in groups)


def bar(q, k):
    most = np.abs(q).max() / 65200 / 3 ** 0.5
    return 2.0 ** -8 + 2.0 ** -11 + 5 * most * np.linalg.norm(k, axis=-1).max() * q.shape[-1] ** -0.5


def attend(m, q, window=0, sinks=0):
    """The step's queries, into bf16."""
    rows, heads, dim = q.shape
    dq, _ = dev_as(q, "bf16")
    out = dev_as(np.zeros((rows, heads, dim)), "bf16")[0]
    torch.cuda.synchronize()
    m.kv.attend(0, dq.data_ptr(), out.data_ptr(), heads, q_type=KIND["bf16"], out_type=KIND["bf16"], window=window, sinks=sinks)
    return host(out, "bf16")


def bf16(x):
    return R.from_bf16(R.to_bf16(x))


# rows of a kv head of the kernels for some rows and for many (workgroups of 128 rows and of 256)
@gpu
@pytest.mark.parametrize("dim,heads,tokens", [(64, 4, 6), (96, 8, 4), (128, 4, 8), (128, 4, 20), (128, 4, 600), (256, 4, 20)])
@pytest.mark.parametrize("length,size", [(40, 4.0), (700, 1.0), (3500, 1.0)])
def test_channels_of_small_codes(model, dim, heads, tokens, length, size):  # noqa: F811
    """Channels whose values are a tenth and a thirtieth of the others': codes up to 13 and 4 beside 127. From weights on a few
    tokens to means of all."""
    m = model(kv_heads=1, head_dim=dim, pages=300, page_tokens=16, sequences=1, sequence_pages=300)
    rng = np.random.default_rng(dim + tokens + length)
    k, v = (rng.standard_normal((length + tokens, 1, dim)) for _ in range(2))
    part = np.arange(dim) % 3
    v *= np.array([1, 0.1, 1 / 30])[part]
    m.kv.extend([0], [length + tokens])
    m.write(0, [0], [length + tokens], k, v)
    m.kv.begin([0], [tokens])
    q = bf16(size * rng.standard_normal((tokens, heads, dim)))
    k, v = (h.values() for h in m.of(0, 0))
    want = exact(q, k, v, length)
    e = off(attend(m, q), want, [part == i for i in range(3)])
    assert e <= bar(q, k), f"off by {e:.3g} of a row, bar {bar(q, k):.3g}"


@gpu
@pytest.mark.parametrize("dim,heads,tokens", [(64, 4, 6), (96, 8, 4), (128, 4, 8), (128, 4, 20), (128, 4, 600), (256, 4, 20)])
@pytest.mark.parametrize("ahead", [0.2, 1.3, 4.5])
def test_equal_weights_behind_leading_tokens(model, dim, heads, tokens, ahead):  # noqa: F811
    """A token of every 64 ahead, the others of the same key, blocks of one scale: weights whose roundings are all the same, under
    values whose mean is small."""
    length = 6000
    m = model(kv_heads=1, head_dim=dim, pages=450, page_tokens=16, sequences=1, sequence_pages=450)
    rng = np.random.default_rng(dim + tokens)
    one = rng.standard_normal(dim)
    k = np.repeat(one[None, None], length + tokens, 0)
    q = bf16(one + 0.02 * rng.standard_normal((tokens, heads, dim)))
    k[::64, 0] += ahead * one / (one @ one) * dim ** 0.5
    v = rng.standard_normal((length + tokens, 1, dim))
    v[:, 0, 0] = 5 * rng.choice([-1, 1], length + tokens)  # the largest of every block
    v[::64] = 0
    m.kv.extend([0], [length + tokens])
    m.write(0, [0], [length + tokens], k, v)
    m.kv.begin([0], [tokens])
    k, v = (h.values() for h in m.of(0, 0))
    want = exact(q, k, v, length)
    e = off(attend(m, q), want)
    assert e <= bar(q, k), f"off by {e:.3g} of a row, bar {bar(q, k):.3g}"


@gpu
@pytest.mark.parametrize("group", [1, 3, 4, 8, 16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_weights_far_below_a_dominant_one(model, dim, group):  # noqa: F811
    """Up to 16 rows: a first token of nearly all the weight and no value, and thousands of a value of 1 at 2^-26 to 2^-20 of it.

    Weights are whole numbers of 2^-26 of the largest that their wave has seen. Rounded to the nearest, those of the wave with the
    first token (an eighth of them at least, a quarter at most) are each off by half a unit at most, evenly spread: sqrt(n / 12)
    units together, of which six times are allowed. Cut off they would be off by n / 2 units."""
    length, seqs = 8192, 32
    m = model(kv_heads=8, head_dim=dim, pages=128, page_tokens=64, sequences=seqs, sequence_pages=128)
    rng = np.random.default_rng(dim + group)
    u = rng.choice([-1.0, 1.0], dim) * dim ** -0.5
    x = rng.uniform(0, 6 * np.log(2), (length, 8, 1))
    x[0] = 26 * np.log(2)
    v = np.ones((length, 8, dim))
    v[0] = 0
    m.kv.extend([0], [length])
    m.write(0, [0], [length], x * u, v)
    m.kv.fork([0] * (seqs - 1), range(1, seqs))  # a workgroup each for all of a sequence and kv head
    m.kv.begin(range(seqs), [1] * seqs)
    q = (dim ** 0.5 * u * rng.uniform(0.98, 1.02, (seqs, 8 * group, 1))).astype(np.float32)
    dq, out = torch.from_numpy(q).cuda(), torch.zeros(q.shape, device="cuda")
    torch.cuda.synchronize()
    m.kv.attend(0, dq.data_ptr(), out.data_ptr(), 8 * group)
    k, v = (h.values() for h in m.of(0, 0))
    want = exact(q, k, v, length)  # the mean of the values is the share of the weight that the first token leaves
    units = want / (1 - want) * 2.0 ** 26
    logs = np.log2(127)
    e = np.abs(host(out) / want - 1)
    allowed = 6 * (length / 4 / 12) ** 0.5 / units + 2 * 2.0 ** -22 * (27 + logs + 8)
    assert (e <= allowed).all(), f"off by {e.max():.3g} of a row, bar {allowed.min():.3g}"


@gpu
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("dim,heads,tokens", [(64, 4, 6), (128, 4, 8), (128, 4, 20), (128, 4, 600), (256, 4, 20)])
def test_weights_of_more_rows_far_below_a_dominant_one(model, dim, heads, tokens, kind):  # noqa: F811
    """The same of 17 rows on: weights in fp16 (for fp32 a sum of two), whole numbers of 2^-32 of the largest down there."""
    length = 8192
    m = model(kv_heads=1, head_dim=dim, pages=150, page_tokens=64, sequences=1, sequence_pages=150)
    rng = np.random.default_rng(dim + tokens)
    u = rng.choice([-1.0, 1.0], dim) * dim ** -0.5
    x = rng.uniform(0, 6 * np.log(2), (length + tokens, 1, 1))
    x[0] = 26 * np.log(2)
    v = np.ones((length + tokens, 1, dim))
    v[0] = 0
    m.kv.extend([0], [length + tokens])
    m.write(0, [0], [length + tokens], x * u, v)
    m.kv.begin([0], [tokens])
    q = bf16(dim ** 0.5 * u * rng.uniform(0.98, 1.02, (tokens, heads, 1)))
    dq, _ = dev_as(q, kind)
    out = dev_as(np.zeros(q.shape), kind)[0]
    torch.cuda.synchronize()
    m.kv.attend(0, dq.data_ptr(), out.data_ptr(), heads, q_type=KIND[kind], out_type=KIND[kind])
    k, v = (h.values() for h in m.of(0, 0))
    want = exact(q, k, v, length)
    units = want / (1 - want) * 2.0 ** 32
    allowed = 6 * (length / 12) ** 0.5 / units + (bar(q, k) if kind == "bf16" else 4 * 2.0 ** -22 * (27 + np.log2(127) + 8))
    e = np.abs(host(out, kind) / want - 1)
    assert (e <= allowed).all(), f"off by {e.max():.3g} of a row, bar {allowed.min():.3g}"


# rows for some and for many, ranges of tokens in several workgroups, windows with first tokens
MASKED = [(128, 4, 8, 3500, 0, 0), (64, 4, 6, 6000, 1700, 4), (96, 8, 4, 3500, 130, 66), (128, 4, 40, 6000, 0, 0), (128, 4, 40, 6000, 1700, 4),
          (128, 4, 40, 6000, 3000, 500), (256, 4, 20, 3500, 50, 3), (128, 4, 600, 1500, 700, 5)]


def masked_inputs(dim, heads, tokens, length, window, sinks):
    rng = np.random.default_rng(dim + tokens + window)
    k, v = (rng.standard_normal((length + tokens, 1, dim)) for _ in range(2))
    return bf16(rng.standard_normal((tokens, heads, dim))), k, v


@gpu
@pytest.mark.parametrize("case", MASKED, ids=str)
def test_masks_of_long_contexts(model, case):  # noqa: F811
    dim, _, tokens, length, window, sinks = case
    m = model(kv_heads=1, head_dim=dim, pages=450, page_tokens=16, sequences=1, sequence_pages=450)
    q, k, v = masked_inputs(*case)
    m.kv.extend([0], [length + tokens])
    m.write(0, [0], [length + tokens], k, v)
    m.kv.begin([0], [tokens])
    k, v = (h.values() for h in m.of(0, 0))
    e = off(attend(m, q, window, sinks), exact(q, k, v, length, window, sinks))
    assert e <= bar(q, k), f"off by {e:.3g} of a row, bar {bar(q, k):.3g}"


@pytest.mark.parametrize("case", MASKED, ids=str)
def test_masks_off_by_one_token_fail(case):
    """What the bar above sees: the formula itself with a token too many or too few at either end (no GPU)."""
    _, _, tokens, length, window, sinks = case
    q, k, v = masked_inputs(*case)
    held = []
    for x in (k, v):
        held.append(R.Held(*x.shape[1:]))
        held[-1].append(x)
    k, v = (h.values() for h in held)
    want = exact(q, k, v, length, window, sinks)
    wrong = {"one back": (length - 1, window and window - 1, sinks), "one ahead": (length + 1, window and window + 1, sinks)}
    if window:
        wrong |= {"window less": (length, window - 1, sinks), "window more": (length, window + 1, sinks), "a first one more": (length, window, sinks + 1),
                  "a first one less": (length, window, sinks - 1)}
    for name, mask in wrong.items():
        rows = slice(None, -1) if name == "one ahead" else slice(None)  # behind the last token is none
        e = off(exact(q, k, v, *mask)[rows], want[rows])
        assert e > 2 * bar(q, k), f"{name}: {e:.3g}, bar {bar(q, k):.3g}"
