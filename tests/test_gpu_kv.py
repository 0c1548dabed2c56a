"""The 8-bit key/value cache on the GPU: rotary positions, append, read, attention, pages.

Bars. What the cache stores, and rotary positions in fp32, are the definition's bits (rounded to bf16 once where that is
the type). Attention is held to the 64-bit formula over the values the cache holds: a score in powers of two, t, is
rounded a handful of times near its own size and that of the value scale's logarithm, so weights are off by
d = 2^-22 (max |t| + max |log2 scale| + 8) at most, and a row, a mean of values under those weights, by 2 d max |v|.
A bf16 result adds half its last place, 2^-8 of it at most. Where rows are many and the result is bf16, q and the weights are
fp16 (half a last place, at most 2^-11 each, of the scaled products' sum and of the weight): d grows by 2^-11 (sum |q k| + 1).
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

import kv_ref as R
from jax4j_amd import DType, IllegalArgumentException, KvCache, Rope

pytestmark = pytest.mark.gpu
KIND = {"f32": DType.F32, "bf16": DType.BF16}


def dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def dev_as(x, kind):
    """(device tensor, the fp32 values in it)"""
    if kind == "f32":
        return dev(x.astype(np.float32)), x.astype(np.float32)
    b = R.to_bf16(x)
    return dev(b.view(np.int16)), R.from_bf16(b)


def host(t, kind="f32"):
    torch.cuda.synchronize()
    return t.cpu().numpy() if kind == "f32" else R.from_bf16(t.cpu().numpy().view(np.uint16))


class Model:
    """A cache and what it should hold."""

    def __init__(self, backend, **config):
        self.c = dict(dict(layers=1, kv_heads=2, head_dim=64, pages=64, page_tokens=16, sequences=4, sequence_pages=32), **config)
        self.kv = KvCache(backend, **self.c)
        self.held = {}

    def of(self, layer, seq):
        if (layer, seq) not in self.held:
            self.held[layer, seq] = [R.Held(self.c["kv_heads"], self.c["head_dim"]) for _ in range(2)]
        return self.held[layer, seq]

    def write(self, layer, seqs, tokens, k, v, kind="f32", **more):
        """Append to the current step and to what should be held."""
        (dk, k), (dv, v) = dev_as(k, kind), dev_as(v, kind)
        torch.cuda.synchronize()
        self.kv.append(layer, dk.data_ptr(), dv.data_ptr(), KIND[kind], **more)
        torch.cuda.synchronize()
        at = 0
        for s, t in zip(seqs, tokens):
            for h, x in zip(self.of(layer, s), (k, v)):
                h.append(x[at:at + t])
            at += t

    def grow(self, rng, seqs, tokens, size=1.0):
        self.kv.extend(seqs, tokens)
        shape = (sum(tokens), self.c["kv_heads"], self.c["head_dim"])
        for layer in range(self.c["layers"]):
            self.write(layer, seqs, tokens, size * rng.standard_normal(shape), size * rng.standard_normal(shape))

    def read(self, layer, seqs, first, count):
        shape = (len(seqs), count, self.c["kv_heads"], self.c["head_dim"])
        k, v = (torch.full(shape, 7.0, device="cuda") for _ in range(2))
        torch.cuda.synchronize()
        self.kv.read(layer, seqs, first, count, k.data_ptr(), v.data_ptr())
        return host(k), host(v)

    def check(self, seqs):
        for layer in range(self.c["layers"]):
            for s in seqs:
                n = self.kv.length(s)
                got = self.read(layer, [s], [0], n + 19)
                for x, h in zip(got, self.of(layer, s)):
                    assert h.codes.shape[0] == n
                    np.testing.assert_array_equal(x[0], h.values(0, n + 19), err_msg=f"layer {layer} sequence {s}")


@pytest.fixture
def model(backend):
    made = []

    def make(**config):
        made.append(Model(backend, **config))
        return made[-1]

    yield make
    for m in made:
        m.kv.destroy()


# ---- rotary positions ------------------------------------------------------------------------


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,heads,dim,rot,sections,interleaved", [
    (1, 1, 2, 2, None, False), (1, 40, 128, 128, None, True), (13, 3, 80, 80, (14, 13, 13), False), (7, 5, 96, 24, (4, 8), True),
    (5, 3, 70, 14, (3, 4), False), (300, 9, 64, 64, (16, 8, 8), False), (2049, 33, 128, 64, None, True), (3, 2, 258, 256, None, False), (2, 3, 2048, 256, None, True),
    (33, 1, 2046, 34, (17,), False), (70000, 1, 64, 64, None, False), (1, 700, 64, 32, None, True)])
def test_rope_into(backend, kind, rows, heads, dim, rot, sections, interleaved):
    rng = np.random.default_rng(rows)
    cos, sin = R.tables(501, rot // 2)
    sec = sections or (rot // 2,)
    pos = rng.integers(0, 501, (len(sec), rows)).astype(np.int32)
    if rows > 2:
        pos[0, 1], pos[-1, 2] = -1, 501  # no angle: NaN in the pairs of that axis
    pad = 8  # rows apart
    x, xv = dev_as(np.concatenate([rng.standard_normal((rows, heads * dim)), np.full((rows, pad), 9.0)], 1), kind)
    y, z = torch.zeros_like(x), x.clone()
    dc, ds, dp = dev(cos), dev(sin), dev(pos)
    rope = Rope(dc.data_ptr(), ds.data_ptr(), 501, rot, positions=dp.data_ptr(), sections=sections, interleaved=interleaved)
    torch.cuda.synchronize()
    backend.rope_into(x.data_ptr(), y.data_ptr(), rows, heads, dim, rope, KIND[kind], x_stride=heads * dim + pad, out_stride=heads * dim + pad)
    backend.rope_into(z.data_ptr(), z.data_ptr(), rows, heads, dim, rope, KIND[kind], x_stride=heads * dim + pad, out_stride=heads * dim + pad)
    axis = np.repeat(np.arange(len(sec)), sec)
    want = R.rotate(xv[:, :heads * dim].reshape(rows, heads, dim), cos, sin, pos[axis].T, interleaved).reshape(rows, -1)
    if kind == "bf16":
        want = np.where(np.isnan(want), np.nan, R.from_bf16(R.to_bf16(want)))
    for t, behind in ((y, 0.0), (z, 9.0)):
        got = host(t, kind)
        np.testing.assert_array_equal(got[:, :heads * dim], want)
        assert (got[:, heads * dim:] == behind).all()


# ---- append and read -------------------------------------------------------------------------


@pytest.mark.parametrize("dim,page,kind,interleaved,rot", [
    (64, 16, "f32", False, 0), (96, 32, "bf16", True, 96), (128, 16, "f32", True, 128), (128, 64, "f32", False, 64), (192, 32, "f32", False, 22),
    (256, 16, "bf16", False, 256)])
def test_append_and_read(model, dim, page, kind, interleaved, rot):
    m = model(layers=2, kv_heads=3, head_dim=dim, pages=40, page_tokens=page, sequences=3, sequence_pages=20)
    rng = np.random.default_rng(dim + page)
    cos, sin = R.tables(400, max(1, rot // 2))
    dc, ds = dev(cos), dev(sin)
    rope = Rope(dc.data_ptr(), ds.data_ptr(), 400, rot, interleaved=interleaved) if rot else None
    # steps of one token to many, of some of the sequences, of values that outgrow a block's scale or shrink
    steps = [([0, 1, 2], [5, 16, 1], 1.0), ([0], [1], 0.0), ([2, 0], [1, 1], 4.0), ([1], [1], 1e-3), ([1], [40], 1.0), ([0, 1, 2], [1, 3, 7], 30.0),
             ([2], [90], 2.0), ([0, 2], [9, 1], 300.0), ([0, 1, 2], [1, 1, 1], 1e-30), ([1], [1], 1e30)]
    for seqs, tokens, size in steps:
        m.kv.extend(seqs, tokens)
        rows = sum(tokens)
        place = np.concatenate([m.kv.length(s) - t + np.arange(t) for s, t in zip(seqs, tokens)])
        for layer in range(2):
            k, v = (size * rng.standard_normal((rows, 3, dim)) for _ in range(2))
            q = rng.standard_normal((rows, 6, dim))
            (dk, kv), (dv, vv), (dq, qv) = (dev_as(x, kind) for x in (k, v, q))
            dq0, out = dq.clone(), torch.zeros_like(dq)
            torch.cuda.synchronize()
            more = dict(rope=rope, heads=6)
            m.kv.append(layer, dk.data_ptr(), dv.data_ptr(), KIND[kind], q_ptr=dq.data_ptr(), q_out_ptr=out.data_ptr(), **more)
            m.kv.append(layer, dk.data_ptr(), dv.data_ptr(), KIND[kind], q_ptr=dq.data_ptr(), **more)  # again, and in place
            torch.cuda.synchronize()
            at = np.repeat(place[:, None], rot // 2, 1) if rot else None
            kr, qr = ((R.rotate(x, cos, sin, at, interleaved) for x in (kv, qv)) if rot else (kv, qv))
            want = qr if kind == "f32" else R.from_bf16(R.to_bf16(qr))
            np.testing.assert_array_equal(host(out, kind), want)
            np.testing.assert_array_equal(host(dq, kind), want)
            assert torch.equal(dk, dev_as(k, kind)[0]) and not torch.equal(dq0, dq) or not rot
            row = 0
            for s, t in zip(seqs, tokens):
                for h, x in zip(m.of(layer, s), (kr, vv)):
                    h.append(x[row:row + t])
                row += t
        m.check([0, 1, 2])
    got = m.read(1, [2, 0, 2], [3, 0, 200], 33)
    for x, which in zip(got, (0, 1)):
        for i, (s, f) in enumerate(((2, 3), (0, 0), (2, 200))):
            np.testing.assert_array_equal(x[i], m.of(1, s)[which].values(f, 33))


@pytest.mark.parametrize("tiny", [1e-18, 6e-18, 1e-19])
@pytest.mark.parametrize("size", [0.0, 1e-19, 7e-18, 2e-17, 1.0])
def test_block_of_tiny_values(model, tiny, size):
    """Codes of a block at the least scale stay what they stand for when another token sets the scale."""
    m = model(kv_heads=1, head_dim=64, pages=4, page_tokens=16, sequences=2, sequence_pages=2)
    rng = np.random.default_rng(5)
    for n, scale in ((5, tiny), (1, size), (2, tiny), (1, 4 * size)):
        k, v = scale * rng.uniform(-1, 1, (n, 1, 64)), scale * rng.uniform(-1, 1, (n, 1, 64))
        m.kv.extend([0], [n])
        m.write(0, [0], [n], k, v)
        m.check([0])
    assert np.abs(m.read(0, [0], [0], 5)[0]).max() < tiny + 2.0 ** -64 + 4 * size / 127  # one step of the scale in all


def test_append_of_rows_apart_and_of_uneven_steps(model):
    """k and v inside wider rows; one sequence of many tokens beside many of one."""
    m = model(kv_heads=2, head_dim=64, pages=200, page_tokens=16, sequences=40, sequence_pages=100)
    rng = np.random.default_rng(3)
    seqs, tokens = list(range(40)), [1] * 39 + [777]
    m.kv.extend(seqs, tokens)
    wide = rng.standard_normal((sum(tokens), 512 + 2 * 128 + 4)).astype(np.float32)
    d = dev(wide)
    torch.cuda.synchronize()
    m.kv.append(0, d.data_ptr() + 4 * 512, d.data_ptr() + 4 * 640, stride=wide.shape[1])
    row = 0
    for s, t in zip(seqs, tokens):
        for h, at in zip(m.of(0, s), (512, 640)):
            h.append(wide[row:row + t, at:at + 128].reshape(t, 2, 64))
        row += t
    m.check(seqs)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_values_that_are_not_finite(model, bad):
    m = model(kv_heads=2, head_dim=64)
    rng = np.random.default_rng(5)
    m.grow(rng, [0, 1], [20, 20])
    m.kv.extend([0, 1], [3, 20])
    k, v = rng.standard_normal((23, 2, 64)), rng.standard_normal((23, 2, 64))
    k[1, 0, 5] = v[22, 1, 63] = bad  # sequence 0's block 1, head 0; sequence 1's block 2, head 1
    m.write(0, [0, 1], [3, 20], k, v)
    m.grow(rng, [0], [30])
    m.check([0, 1])
    k0, v1 = m.of(0, 0)[0], m.of(0, 1)[1]
    assert np.isnan(k0.scale[1, 0]) and np.isnan(k0.scale).sum() == 1 and np.isnan(v1.scale[2, 1])
    for window in (0, 21, 18, 16):  # of the step of 30 tokens from place 23 on, those of later rows show nothing of block 1
        check_attend(m, rng, [0], [30], 4, window=window)
        check_attend(m, rng, [0], [30], 4, window=window, okind="bf16")
    m.kv.begin([1], [3])  # behind the block of the value that is not finite is none
    check_attend(m, rng, [1], [3], 4)


# ---- attention -------------------------------------------------------------------------------


def check_attend(m, rng, seqs, tokens, heads, window=0, sinks=0, scale=0.0, qkind="f32", okind="f32", size=1.0, layer=0, pad=0, begin=False, q=None):
    rows, dim = sum(tokens), m.c["head_dim"]
    if begin:
        m.kv.begin(seqs, tokens)
    x = np.full((rows, heads * dim + pad), 3.0)
    x[:, :heads * dim] = size * rng.standard_normal((rows, heads * dim)) if q is None else q
    dq, qv = dev_as(x, qkind)
    qv = qv[:, :heads * dim].reshape(rows, heads, dim)
    out = dev_as(np.full((rows, heads * dim + pad), 5.0), okind)[0]
    torch.cuda.synchronize()
    m.kv.attend(layer, dq.data_ptr(), out.data_ptr(), heads, q_type=KIND[qkind], out_type=KIND[okind], q_stride=heads * dim + pad,
                out_stride=heads * dim + pad, window=window, sinks=sinks, scale=scale)
    got = host(out, okind)
    assert (got[:, heads * dim:] == 5.0).all()
    got, row = got[:, :heads * dim].reshape(rows, heads, dim), 0
    worst = 0.0
    for s, t in zip(seqs, tokens):
        k, v = m.of(layer, s)
        n = k.codes.shape[0]
        want, top, products = R.attend(qv[row:row + t], k.values(), v.values(), n - t, window, sinks, scale)
        with np.errstate(invalid="ignore", divide="ignore"):
            logs = np.abs(np.log2(v.scale[np.isfinite(v.scale)])).max()
            d = 2.0 ** -22 * (top + logs + 8)
            if okind == "bf16" and max(tokens) * heads // m.c["kv_heads"] > 16:
                d += 2.0 ** -11 * (products + 1)
            bar = 2 * d * np.nanmax(np.abs(v.values()))
        part = got[row:row + t]
        assert np.array_equal(np.isnan(part), np.isnan(want)), f"sequence {s}"
        off = np.abs(part - want) - (2.0 ** -8 * np.abs(want) if okind == "bf16" else 0)
        off = np.where(np.isnan(want), 0, off)
        assert off.max() <= bar, f"sequence {s}: off by {off.max():.3g}, bar {bar:.3g}, at {np.unravel_index(off.argmax(), off.shape)}"
        worst = max(worst, off.max() / bar)
        row += t
    return worst


@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("group", [1, 4, 5, 8])
def test_attend_one_token(model, dim, group):
    """Sequences of one token up to several tiles, ends all over a tile, queries of both types."""
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 130, 300]
    m = model(kv_heads=2, head_dim=dim, pages=100, page_tokens=16, sequences=len(lens), sequence_pages=20)
    rng = np.random.default_rng(dim + group)
    seqs = list(range(len(lens)))
    m.grow(rng, seqs, lens)
    check_attend(m, rng, seqs, [1] * len(lens), 2 * group, begin=True)
    check_attend(m, rng, seqs[::-1], [1] * len(lens), 2 * group, begin=True, qkind="bf16", okind="bf16", pad=8)
    check_attend(m, rng, seqs, [1] * len(lens), 2 * group, window=20, sinks=3, begin=True)


@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (1, 1), (16, 4), (100, 0), (100, 64), (129, 70), (1000, 7), (300, 5000)])
def test_attend_windows(model, page, window, sinks):
    lens = [1, 40, 333, 700]
    m = model(kv_heads=2, head_dim=64, pages=150, page_tokens=page, sequences=4, sequence_pages=64)
    rng = np.random.default_rng(window + sinks)
    for part in ([1, 40, 300, 3], [33, 697]):  # pages lie between each other's
        m.grow(rng, [0, 1, 2, 3] if len(part) == 4 else [2, 3], part)
    for tokens, heads in ((1, 8), (1, 14), (2, 6), (3, 8)):
        who = [s for s in range(4) if lens[s] >= tokens]
        check_attend(m, rng, who, [tokens] * len(who), heads, window=window, sinks=sinks, begin=True)


@pytest.mark.parametrize("group,tokens", [(1, 3), (4, 1), (4, 2), (7, 1), (8, 2), (3, 5), (16, 1), (1, 17)])
def test_attend_few_rows_long(model, group, tokens):
    """Long enough that a sequence's tokens are several workgroups', short ones beside it."""
    m = model(kv_heads=1, head_dim=128, pages=400, page_tokens=32, sequences=3, sequence_pages=300)
    rng = np.random.default_rng(group)
    m.grow(rng, [0, 1, 2], [6000, tokens, 1500], 2.0)
    for window, sinks in ((0, 0), (1700, 4)):
        check_attend(m, rng, [0, 1, 2], [tokens] * 3, group, window=window, sinks=sinks, begin=True, size=2.0)


@pytest.mark.parametrize("okind", ["bf16", "f32"])
@pytest.mark.parametrize("dim,group,page", [(64, 1, 16), (96, 4, 32), (128, 4, 64), (128, 7, 16), (192, 2, 32), (256, 8, 16)])
def test_attend_many_rows(model, dim, group, page, okind):
    """Prompts whole and in chunks, rows that end all over a tile of them, sequences of uneven steps, windows."""
    m = model(kv_heads=2, head_dim=dim, pages=400, page_tokens=page, sequences=5, sequence_pages=100)
    rng = np.random.default_rng(dim + group)
    for seqs, tokens in (([0, 1, 2, 3, 4], [1, 17, 64, 129, 300]), ([0, 4, 2], [200, 33, 1]), ([3], [70])):
        m.grow(rng, seqs, tokens)
        check_attend(m, rng, seqs, tokens, 2 * group, okind=okind)
        check_attend(m, rng, seqs, tokens, 2 * group, okind=okind, window=50, sinks=3, qkind="bf16", pad=8, scale=0.3)
        check_attend(m, rng, seqs, tokens, 2 * group, okind=okind, window=1)
        check_attend(m, rng, seqs, tokens, 2 * group, okind=okind, window=130, sinks=66)


@pytest.mark.parametrize("okind", ["bf16", "f32"])
@pytest.mark.parametrize("dim,group,tokens,page", [(64, 8, 3, 16), (64, 32, 1, 64), (96, 4, 5, 32), (128, 4, 8, 64), (128, 7, 4, 32), (128, 1, 17, 16),
                                                   (128, 1, 32, 16), (128, 2, 9, 64), (192, 4, 6, 32), (256, 8, 4, 16)])
def test_attend_some_rows(model, dim, group, tokens, page, okind):
    """17 to 32 rows of a sequence (drafts that are verified): from the step alone to thousands of tokens in several ranges."""
    m = model(kv_heads=2, head_dim=dim, pages=600, page_tokens=page, sequences=5, sequence_pages=300)
    rng = np.random.default_rng(dim + group + tokens)
    seqs, lens = [4, 0, 2, 1, 3], [tokens, tokens + 1, 128, 700, 3500]
    m.grow(rng, seqs, lens, 2.0)
    for window, sinks, more in ((0, 0, {}), (50, 3, dict(qkind="bf16", pad=8, scale=0.3)), (1, 0, {}), (130, 66, {}), (1700, 4, {})):
        check_attend(m, rng, seqs, [tokens] * 5, 2 * group, window=window, sinks=sinks, okind=okind, begin=True, size=2.0, **more)


@pytest.mark.parametrize("okind", ["bf16", "f32"])
def test_attend_steps_of_every_kind(model, okind):
    """Few, some and many rows in one call, each long and short."""
    m = model(kv_heads=2, head_dim=128, pages=900, page_tokens=16, sequences=6, sequence_pages=400)
    rng = np.random.default_rng(37)
    seqs, tokens = [3, 0, 5, 1, 2, 4], [6, 1, 40, 4, 8, 100]
    m.grow(rng, seqs, [3000, 2500, 20, 700, 1, 1500])
    m.grow(rng, seqs, tokens)
    for window, sinks in ((0, 0), (500, 4)):
        check_attend(m, rng, seqs, tokens, 8, window=window, sinks=sinks, okind=okind)


@pytest.mark.parametrize("okind", ["bf16", "f32"])
def test_attend_some_rows_extremes(model, okind):
    """Tokens far ahead, blocks of zeros and of values far below others', keys and queries of all magnitudes, rows that are not finite."""
    m = model(kv_heads=1, head_dim=128, pages=160, page_tokens=16, sequences=3, sequence_pages=150)
    rng = np.random.default_rng(41)
    m.kv.extend([0, 1, 2], [400, 60, 1500])
    k, v = rng.standard_normal((1960, 1, 128)), rng.standard_normal((1960, 1, 128))
    k[100:104] *= 20
    v[:16] *= 1e-3
    v[200:240], k[300:320] = 0, 0
    v[400:460] *= 1e-12
    k[400:460] *= 1e12
    k[460:480] += 3  # first tokens that draw the weight and give little
    v[460:480] *= 1e-4
    m.write(0, [0, 1, 2], [400, 60, 1500], k, v)
    for size in (1e-20, 1.0, 3.0):
        check_attend(m, rng, [0, 2], [8, 8], 4, size=size, begin=True, okind=okind)
    check_attend(m, rng, [1], [7], 4, size=1e-12, begin=True, okind=okind)
    q = rng.standard_normal((8, 4 * 128))
    q[5, 130], q[2, 300] = np.nan, -np.inf
    dq = dev(q.astype(np.float32))
    out = dev_as(np.zeros((8, 512)), okind)[0]
    m.kv.begin([0], [8])
    torch.cuda.synchronize()
    m.kv.attend(0, dq.data_ptr(), out.data_ptr(), 4, out_type=KIND[okind])
    got = np.isnan(host(out, okind)).reshape(8, 4, 128)
    assert got[5, 1].all() and got[2, 2].all() and got.sum() == 2 * 128


@pytest.mark.parametrize("tokens", [6, 20])
def test_captured_steps_of_several_tokens(model, tokens):
    """The same of 24 and of 80 rows, while the sequence grows from one range of tokens to several."""
    m = model(kv_heads=2, head_dim=128, pages=400, page_tokens=16, sequences=2, sequence_pages=300)
    rng = np.random.default_rng(43)
    m.grow(rng, [0, 1], [300, 5])
    q, k, v = (torch.randn((2 * tokens, h, 128), device="cuda") for h in (8, 2, 2))
    out = torch.zeros_like(q)
    s = torch.cuda.Stream()
    m.kv.extend([0, 1], [tokens] * 2)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        m.kv.append(0, k.data_ptr(), v.data_ptr(), stream=s.cuda_stream)
        m.kv.attend(0, q.data_ptr(), out.data_ptr(), 8, stream=s.cuda_stream)
    for i in range(6):
        if i:
            m.kv.extend([0], [700])
            more = [torch.randn((700, 2, 128), device="cuda") for _ in range(2)]
            torch.cuda.synchronize()
            m.kv.append(0, more[0].data_ptr(), more[1].data_ptr())
            m.kv.extend([0, 1], [tokens] * 2)
        torch.cuda.synchronize()
        for x in (q, k, v):
            x.copy_(torch.randn_like(x))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        got = out.clone()
        m.kv.append(0, k.data_ptr(), v.data_ptr())
        m.kv.attend(0, q.data_ptr(), out.data_ptr(), 8)
        torch.cuda.synchronize()
        # other ranges of the tokens, so other roundings
        assert torch.allclose(got, out, rtol=0, atol=1e-5 * float(v.abs().max() + 4)), i


@pytest.mark.parametrize("okind", ["bf16", "f32"])
def test_attend_uneven_steps(model, okind):
    """A chunk of a prompt beside sequences of one token and of a few, short and long."""
    m = model(kv_heads=2, head_dim=128, pages=900, page_tokens=16, sequences=6, sequence_pages=400)
    rng = np.random.default_rng(31)
    seqs, tokens = [3, 0, 5, 1, 2, 4], [300, 1, 4, 5, 1, 17]
    m.grow(rng, seqs, [50, 4000, 20, 700, 1, 100])
    m.grow(rng, seqs, tokens)
    for window, sinks in ((0, 0), (500, 4)):
        check_attend(m, rng, seqs, tokens, 8, window=window, sinks=sinks, okind=okind)


@pytest.mark.parametrize("okind", ["bf16", "f32"])
def test_attend_many_rows_long(model, okind):
    """A chunk behind a long context: a row tile's tokens are several workgroups'."""
    m = model(kv_heads=1, head_dim=128, pages=400, page_tokens=32, sequences=2, sequence_pages=300)
    rng = np.random.default_rng(23)
    m.grow(rng, [0, 1], [6000, 100], 2.0)
    for window, sinks in ((0, 0), (1700, 4), (3000, 500)):
        check_attend(m, rng, [0, 1], [41, 30], 4, window=window, sinks=sinks, begin=True, okind=okind)


@pytest.mark.parametrize("okind", ["bf16", "f32"])
def test_attend_many_rows_extremes(model, okind):
    m = model(kv_heads=1, head_dim=128, pages=64, page_tokens=16, sequences=2, sequence_pages=40)
    rng = np.random.default_rng(29)
    m.kv.extend([0, 1], [400, 60])
    k, v = rng.standard_normal((460, 1, 128)), rng.standard_normal((460, 1, 128))
    k[100:104] *= 20
    v[:16] *= 1e-3
    v[200:240], k[300:320] = 0, 0
    v[400:] *= 1e-12
    k[400:] *= 1e12
    m.write(0, [0, 1], [400, 60], k, v)
    for size in (1e-20, 1.0, 3.0):
        check_attend(m, rng, [0], [390], 4, size=size, begin=True, okind=okind)
    check_attend(m, rng, [1], [50], 4, size=1e-12, begin=True, okind=okind)
    q = rng.standard_normal((390, 4 * 128))
    q[5, 130], q[100, 300] = np.nan, -np.inf
    dq = dev(q.astype(np.float32))
    out = dev_as(np.zeros((390, 512)), okind)[0]
    m.kv.begin([0], [390])
    torch.cuda.synchronize()
    m.kv.attend(0, dq.data_ptr(), out.data_ptr(), 4, out_type=KIND[okind])
    got = np.isnan(host(out, okind)).reshape(390, 4, 128)
    assert got[5, 1].all() and got[100, 2].all() and got.sum() == 2 * 128


@pytest.mark.parametrize("heads,tokens", [(4, 1), (6, 1), (10, 1), (6, 2), (6, 50)])
def test_attend_in_place(model, heads, tokens):
    """Out over q gives the bits that out apart from it gives, ranges of tokens and rows that do not fill a workgroup among them."""
    m = model(kv_heads=2, head_dim=128, pages=400, page_tokens=16, sequences=3, sequence_pages=200)
    rng = np.random.default_rng(heads)
    lens = [3000, 70, tokens]
    m.kv.extend([0, 1, 2], lens)
    m.write(0, [0, 1, 2], lens, rng.standard_normal((sum(lens), 2, 128)), rng.standard_normal((sum(lens), 2, 128)))
    m.kv.begin([0, 1, 2], [tokens] * 3)
    q = dev(rng.standard_normal((3 * tokens, heads * 128)).astype(np.float32))
    out = torch.zeros_like(q)
    torch.cuda.synchronize()
    m.kv.attend(0, q.data_ptr(), out.data_ptr(), heads)
    m.kv.attend(0, q.data_ptr(), q.data_ptr(), heads)
    torch.cuda.synchronize()
    assert torch.equal(q, out) and bool(torch.isfinite(out).all())


def test_attend_extremes(model):
    """Scores of hundreds, weights on one token, values and queries of all magnitudes, blocks of zeros, a scale of its own."""
    m = model(kv_heads=1, head_dim=128, pages=64, page_tokens=16, sequences=3, sequence_pages=40)
    rng = np.random.default_rng(9)
    m.kv.extend([0, 1, 2], [400, 200, 150])
    k, v = rng.standard_normal((750, 1, 128)), rng.standard_normal((750, 1, 128))
    k[100:116] *= 40  # some tokens far ahead
    v[:16] *= 1e-3    # first tokens that draw the weight and give little
    k[:4] += 3
    v[200:240], k[300:320] = 0, 0
    v[400:600] *= 1e-12
    k[400:600] *= 1e12
    v[600:] *= 1e15
    m.write(0, [0, 1, 2], [400, 200, 150], k, v)
    for size in (1e-20, 1.0, 5.0):
        check_attend(m, rng, [0], [2], 4, size=size, begin=True)
    check_attend(m, rng, [1], [1], 4, size=1e-12, begin=True)
    check_attend(m, rng, [2], [1], 4, size=3.0, begin=True, scale=0.5)
    q = rng.standard_normal((1, 4 * 128)) * 10.0 ** rng.integers(-9, 1, (1, 512))  # small channels beside large ones
    check_attend(m, rng, [0], [1], 4, q=q, begin=True)
    q[0, 130] = np.nan
    q[0, 300] = np.inf
    dq = dev(q.astype(np.float32))
    out = torch.zeros((1, 512), device="cuda")
    torch.cuda.synchronize()
    m.kv.attend(0, dq.data_ptr(), out.data_ptr(), 4)
    got = np.isnan(host(out)).reshape(4, 128)
    assert got[1:3].all() and not got[[0, 3]].any()


def test_attend_offsets_past_32_bits(model):
    """The last layer of a pool of over 4 GiB, pages at both of its ends."""
    m = model(layers=3, kv_heads=8, head_dim=256, pages=36000, page_tokens=16, sequences=3, sequence_pages=36000)
    assert 2 * 36000 * m.kv.info()["page_bytes"] > 2 ** 32
    rng = np.random.default_rng(11)
    m.kv.extend([0], [16 * 35990])  # takes the pool but for ten pages; its tokens are not written
    m.kv.extend([1], [150])
    m.kv.truncate([0], [0])
    m.kv.extend([2, 1], [100, 1])
    k, v = rng.standard_normal((101, 8, 256)), rng.standard_normal((101, 8, 256))
    m.write(2, [2, 1], [100, 1], k, v)
    m.held.clear()
    assert m.kv.tables([1])[0, 9] == 35999 and m.kv.tables([2])[0, 0] == 0
    m.kv.begin([1], [151])
    k1, v1 = rng.standard_normal((151, 8, 256)), rng.standard_normal((151, 8, 256))
    m.write(2, [1], [151], k1, v1)
    for h, x in zip(m.of(2, 2), (k, v)):
        h.append(x[:100])
    for s in (1, 2):
        got = m.read(2, [s], [0], m.kv.length(s))
        for x, h in zip(got, m.of(2, s)):
            np.testing.assert_array_equal(x[0], h.values())
    check_attend(m, rng, [2, 1], [1, 1], 16, layer=2, begin=True)


def test_attend_is_the_same_every_time(model):
    m = model(kv_heads=2, head_dim=128, pages=300, page_tokens=16, sequences=2, sequence_pages=300)
    rng = np.random.default_rng(13)
    m.grow(rng, [0, 1], [3000, 700])
    m.kv.begin([0, 1], [1, 1])
    q = torch.randn((2, 8, 128), device="cuda")
    outs = [torch.zeros_like(q) for _ in range(6)]
    torch.cuda.synchronize()
    for o in outs:
        m.kv.attend(0, q.data_ptr(), o.data_ptr(), 8)
    torch.cuda.synchronize()
    assert all(torch.equal(o, outs[0]) for o in outs[1:])


# ---- pages -----------------------------------------------------------------------------------


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("seed", [1, 2, 3])
def test_pages_hold_what_their_sequences_were_given(model, page, seed):
    """Extend, fork, copy, cut, evict, compact in random order: every sequence reads back what was appended to it."""
    m = model(layers=2, kv_heads=1, head_dim=64, pages=1280 // page, page_tokens=page, sequences=8, sequence_pages=640 // page)
    rng = np.random.default_rng(seed)
    gone = {}
    for _ in range(50):
        what = rng.choice(["extend", "extend", "fork", "copy", "cut", "free", "compact"])
        full = [s for s in range(8) if m.kv.length(s)]
        empty = [s for s in range(8) if not m.kv.length(s)]
        if what == "extend":
            seqs = [int(s) for s in rng.permutation(8)[:rng.integers(1, 4)]]
            tokens = [int(rng.choice([1, 2, rng.integers(1, 100)])) for _ in seqs]
            free = m.kv.info()["pages_free"]
            if sum(-(-t // page) + 1 for t in tokens) > free or any(m.kv.length(s) + t > 640 for s, t in zip(seqs, tokens)):
                continue
            m.grow(rng, seqs, tokens, 10.0 ** rng.integers(-2, 3))
        elif what in ("fork", "copy") and full and empty:
            src = [int(rng.choice(full)) for _ in empty[:2]]
            dst = empty[:len(src)]
            if what == "copy" and sum(-(-m.kv.length(s) // page) for s in src) > m.kv.info()["pages_free"]:
                continue
            m.kv.fork(src, dst, share=what == "fork")
            for a, b in zip(src, dst):
                for layer in range(2):
                    m.held[layer, b] = [h.copy() for h in m.of(layer, a)]
        elif what in ("cut", "free") and full:
            s = int(rng.choice(full))
            n = 0 if what == "free" else int(rng.integers(0, m.kv.length(s) + 1))
            m.kv.truncate([s], [n])
            for layer in range(2):
                for h in m.of(layer, s):
                    h.cut(n)
        elif what == "compact":
            m.kv.compact()
            used = m.kv.tables(range(8))
            assert used.max(initial=-1) < m.c["pages"] - m.kv.info()["pages_free"]
    m.check(range(8))


def test_evict(model):
    m = model(layers=1, kv_heads=2, head_dim=64, pages=40, page_tokens=16, sequences=2, sequence_pages=40)
    rng = np.random.default_rng(1)
    m.grow(rng, [0], [500])
    m.kv.evict([0], 100, 4)
    assert m.kv.info()["pages_free"] == 40 - 32 + (401 // 16 - 1) and (m.kv.tables([0])[0, 1:25] == -1).all()
    m.grow(rng, [1], [300], 1e4)  # into the freed pages
    m.grow(rng, [0], [1])
    check_attend(m, rng, [0], [1], 4, window=100, sinks=4)
    check_attend(m, rng, [0], [1], 4, window=60, sinks=4)
    for window, sinks in ((0, 0), (140, 4), (100, 17)):
        with pytest.raises(IllegalArgumentException, match="evicted"):
            check_attend(m, rng, [0], [1], 4, window=window, sinks=sinks)
    k, v = m.read(0, [0], [0], 501)
    want = m.of(0, 0)[0].values()
    want[16:400] = 0
    np.testing.assert_array_equal(k[0], want)
    m.kv.fork([0], [1]) if m.kv.length(1) == 0 else m.kv.truncate([1], [0])
    m.kv.fork([0], [1])
    m.held[0, 1] = [h.copy() for h in m.of(0, 0)]
    m.kv.compact()
    m.grow(rng, [1, 0], [1, 2])
    check_attend(m, rng, [1, 0], [1, 2], 4, window=98, sinks=4)


# ---- streams and graphs ----------------------------------------------------------------------


def test_calls_on_several_streams_run_in_order(model):
    m = model(layers=1, kv_heads=2, head_dim=128, pages=600, page_tokens=16, sequences=2, sequence_pages=300)
    rng = np.random.default_rng(17)
    m.grow(rng, [0], [4000])
    streams = [torch.cuda.Stream() for _ in range(3)]
    q = torch.randn((1, 8, 128), device="cuda")
    k, v = (torch.randn((1, 2, 128), device="cuda") for _ in range(2))
    outs = [torch.zeros_like(q) for _ in range(12)]
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        s = streams[i % 3].cuda_stream
        m.kv.extend([0], [1], stream=streams[(i + 1) % 3].cuda_stream)
        m.kv.append(0, k.data_ptr(), v.data_ptr(), stream=streams[(i + 2) % 3].cuda_stream)
        m.kv.attend(0, q.data_ptr(), o.data_ptr(), 8, stream=s)
    torch.cuda.synchronize()
    for i, o in enumerate(outs):  # the same on one stream
        m.kv.truncate([0], [4000 + i])
        want = torch.zeros_like(q)
        m.kv.extend([0], [1])
        m.kv.append(0, k.data_ptr(), v.data_ptr())
        m.kv.attend(0, q.data_ptr(), want.data_ptr(), 8)
        m.kv.truncate([0], [4000 + i + 1])
        torch.cuda.synchronize()
        assert torch.equal(o, want)
        m.kv.extend([0], [len(outs) - i]) if i + 1 < len(outs) else None


@pytest.mark.parametrize("start", [3, 700])
def test_captured_steps(model, start):
    """append and attend captured once; every replay serves the step that extend has set up by then."""
    m = model(layers=2, kv_heads=2, head_dim=128, pages=200, page_tokens=16, sequences=3, sequence_pages=100)
    rng = np.random.default_rng(19)
    m.grow(rng, [0, 1, 2], [start, 50, 1])
    q, k, v = (torch.randn((2, h, 128), device="cuda") for h in (8, 2, 2))
    out = [torch.zeros_like(q) for _ in range(2)]
    s = torch.cuda.Stream()
    m.kv.extend([0, 2], [1, 1])
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        for layer in range(2):
            m.kv.append(layer, k.data_ptr(), v.data_ptr(), stream=s.cuda_stream)
            m.kv.attend(layer, q.data_ptr(), out[layer].data_ptr(), 8, stream=s.cuda_stream)
        with pytest.raises(IllegalArgumentException, match="captured"):
            m.kv.extend([1], [1], stream=s.cuda_stream)
    for i, seqs in enumerate([None, [0, 2], [1, 0], [2, 1], [0, 1], [0, 2]] * 4):
        if seqs is not None:
            m.kv.extend(seqs, [1, 1])
        torch.cuda.synchronize()
        for x in (q, k, v):
            x.copy_(torch.randn_like(x))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in out]
        for layer in range(2):  # eager, the same step again
            m.kv.append(layer, k.data_ptr(), v.data_ptr())
            m.kv.attend(layer, q.data_ptr(), out[layer].data_ptr(), 8)
        torch.cuda.synchronize()
        for a, b in zip(got, out):
            # other ranges of the tokens, so other roundings
            assert torch.allclose(a, b, rtol=0, atol=1e-5 * float(v.abs().max() + 4)), i
