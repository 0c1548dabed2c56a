"""The experts' products (Experts.apply) against 64 bits on the oracle's dequantized weights."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import experts_ref as ref
from jax4j_amd import DType, Experts, IllegalArgumentException, QuantType
from jax4j_amd import synthetic as S

pytestmark = pytest.mark.gpu
TYPES = {"f32": (DType.F32, torch.float32), "bf16": (DType.BF16, torch.bfloat16)}
PAIRS = [("Q8_0", "Q8_0"), ("Q4_0", "Q4_0"), ("Q4_K", "Q6_K"), ("Q6_K", "Q4_K"), ("Q4_K", "Q8_0"), ("Q8_0", "Q4_0")]


class Layer:
    """Random experts on the GPU and their weights in 64 bits. The largest weights are about `size`."""

    def __init__(self, backend, up, down, experts, dim, ffn, act="silu", seed=1):
        self.be, self.act, self.up, self.down = backend, act, QuantType[up], QuantType[down]
        self.kept, self.plain = [], []
        for i, (qt, rows, cols) in enumerate(((self.up, ffn, dim), (self.up, ffn, dim), (self.down, dim, ffn))):
            blocks = S.quant_blocks(qt, 10 * seed + i, experts * rows, cols)
            self.kept.append(backend.upload_quantized(blocks, qt, (experts * rows, cols)))
            self.plain.append(tuple(v.reshape(experts, rows, cols) for v in ref.dequantize(blocks, qt, experts * rows, cols)))
        self.experts = Experts(backend, *self.kept, experts=experts, activation=act)
        self.n, self.dim, self.ffn = experts, dim, ffn

    def close(self):
        self.experts.destroy()
        for w in self.kept:
            self.be.release(w)


@pytest.fixture(scope="module")
def layer(backend):
    made = {}

    def get(*key):
        if key not in made:
            made[key] = Layer(backend, *key)
        return made[key]

    yield get
    for l in made.values():
        l.close()


def inputs(l, rows, top, kind, seed=0, scale=1.0):
    rng = np.random.default_rng(seed)
    x = torch.from_numpy((scale * rng.standard_normal((rows, l.dim))).astype(np.float32)).to(TYPES[kind][1])
    ids = np.argsort(rng.random((rows, l.n)), 1)[:, :top].astype(np.int32)
    w = rng.random((rows, top)).astype(np.float32)
    return x, ids, w


def apply(l, x, ids, w, kind, x_stride=0, out_stride=0, stream=0, workspace=False):
    rows, top = ids.shape
    if x_stride:
        wide = torch.full((rows, x_stride), 1e30, dtype=x.dtype)
        wide[:, :l.dim] = x
        x = wide
    x, out = x.cuda(), torch.full((rows + 1, out_stride or l.dim), 55.0, dtype=x.dtype, device="cuda")
    i, v = torch.from_numpy(np.ascontiguousarray(ids)).cuda(), torch.from_numpy(np.ascontiguousarray(w)).cuda()
    more = {}
    if workspace:
        n = l.experts.workspace(rows, top, TYPES[kind][0])
        space = torch.full((n,), 255, dtype=torch.uint8, device="cuda")  # NaN wherever nothing is written
        more = dict(workspace_ptr=space.data_ptr(), workspace_bytes=n)
    torch.cuda.synchronize()
    l.experts.apply(x.data_ptr(), i.data_ptr(), v.data_ptr(), out.data_ptr(), rows, top, TYPES[kind][0], x_stride=x_stride, out_stride=out_stride,
                    stream=stream, **more)
    torch.cuda.synchronize()
    assert (out[rows] == 55.0).all()
    if out_stride:
        assert (out[:rows, l.dim:] == 55.0).all()
    return out[:rows, :l.dim].float().cpu().numpy().astype(np.float64)


def check(l, x, ids, w, kind, got):
    want, off = ref.experts(x.float().numpy(), ids, w, *l.plain, l.act, kind, exact_weights=False)
    if kind == "bf16":
        off = off + ref.STEP["bf16"] * (np.abs(want) + off)
    off = off + 2.0 ** -126
    bad = ~(np.abs(got - want) <= off)
    assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], want[bad][:4], off[bad][:4])
    # the bound holds in the worst case; taken together, errors that are independent come to far less than a tenth of it
    norm = np.linalg.norm(got - want)
    if kind == "f32":
        assert norm <= 0.1 * np.linalg.norm(off), norm / np.linalg.norm(off)


@pytest.mark.parametrize("up,down", PAIRS)
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,top", [(1, 1), (1, 4), (2, 3), (7, 2), (40, 4), (150, 3)])
def test_types_and_rows(layer, up, down, kind, rows, top):
    l = layer(up, down, 6, 512, 256)
    x, ids, w = inputs(l, rows, top, kind, seed=rows)
    check(l, x, ids, w, kind, apply(l, x, ids, w, kind))


@pytest.mark.parametrize("up,down,dim,ffn", [("Q8_0", "Q8_0", 64, 64), ("Q8_0", "Q8_0", 192, 320), ("Q8_0", "Q8_0", 1088, 704), ("Q4_0", "Q4_0", 128, 128),
                                             ("Q4_0", "Q4_0", 384, 640), ("Q4_0", "Q8_0", 2176, 448), ("Q4_K", "Q6_K", 256, 256), ("Q6_K", "Q4_K", 2304, 512),
                                             ("Q4_K", "Q4_K", 768, 2304)])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_sizes(layer, up, down, dim, ffn, kind):
    l = layer(up, down, 3, dim, ffn)
    for rows in (1, 35):
        x, ids, w = inputs(l, rows, 2, kind, seed=dim)
        check(l, x, ids, w, kind, apply(l, x, ids, w, kind))


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_activations(layer, act, kind):
    l = layer("Q4_K", "Q6_K", 4, 256, 512, act)
    for scale in (0.01, 1.0, 30.0):
        x, ids, w = inputs(l, 9, 2, kind, scale=scale)
        check(l, x, ids, w, kind, apply(l, x, ids, w, kind))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [3, 90])
def test_choices(layer, kind, rows):
    """Slots without an expert, rows without any, one expert for all, the same expert twice, experts that no one chose."""
    l = layer("Q4_K", "Q6_K", 6, 512, 256)
    x, ids, w = inputs(l, rows, 4, kind)
    for change in range(5):
        i = ids.copy()
        if change == 0:
            i[::2, 1] = -1
            i[1::2, 2] = 6
            i[0] = -1
            i[-1] = 2 ** 31 - 1
        elif change == 1:
            i[:] = 5
        elif change == 2:
            i[:, 1] = i[:, 0]
        elif change == 3:
            i = np.where(i > 2, -2 ** 31, i).astype(np.int32)
        else:
            i[:] = -1
        got = apply(l, x, i, w, kind)
        check(l, x, i, w, kind, got) if change < 4 else None
        assert (got[((i < 0) | (i >= l.n)).all(1)] == 0).all()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e12, 1e17])
def test_scales(layer, kind, scale):
    """Activations far from 1, and rows of very different sizes in one tile."""
    l = layer("Q8_0", "Q8_0", 4, 256, 256)
    x, ids, w = inputs(l, 12, 2, kind)
    for r in range(0, 12, 3):
        x[r] *= scale
    x[1] = 0
    x[2, 1:] = 0
    check(l, x, ids, w, kind, apply(l, x, ids, w, kind))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [5, 100])
def test_values_that_are_not_finite(layer, kind, rows):
    l = layer("Q4_K", "Q6_K", 6, 512, 256)
    x, ids, w = inputs(l, rows, 2, kind)
    ids[:] = [[1, 3]]
    clean = apply(l, x, ids, w, kind)
    x[1, 7], x[3, 500] = float("nan"), float("-inf")
    w[4, 1] = np.nan
    got = apply(l, x, ids, w, kind)
    assert np.isnan(got[[1, 3, 4]]).all()
    rest = [r for r in range(rows) if r not in (1, 3, 4)]
    assert np.array_equal(got[rest], clean[rest])
    ids[[1, 3, 4]] = -1  # without an expert such a row is zeros
    assert (apply(l, x, ids, w, kind)[[1, 3, 4]] == 0).all()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_strides_workspaces_and_streams_give_the_same(layer, kind):
    l = layer("Q4_0", "Q4_0", 5, 384, 256)
    for rows in (2, 60):
        x, ids, w = inputs(l, rows, 3, kind)
        want = apply(l, x, ids, w, kind)
        check(l, x, ids, w, kind, want)
        stream = torch.cuda.Stream()
        for more in (dict(x_stride=400), dict(out_stride=392), dict(workspace=True), dict(stream=stream.cuda_stream), dict(stream=stream.cuda_stream, workspace=True)):
            assert np.array_equal(apply(l, x, ids, w, kind, **more), want), more


def test_a_row_does_not_depend_on_the_others(layer):
    """Bit for bit the same, whichever tile and place a row's pairs get, while the call's kernels are the same."""
    l = layer("Q4_K", "Q6_K", 6, 512, 256)
    x, ids, w = inputs(l, 64, 3, "f32")
    a = apply(l, x, ids, w, "f32")
    order = np.random.default_rng(3).permutation(64)
    b = apply(l, x[order], ids[order], w[order], "f32")
    assert np.array_equal(a[order], b)


@pytest.mark.parametrize("up,down", PAIRS)
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [50, 200, 410])
def test_pairs_enough_for_each_size_of_tile(layer, up, down, kind, rows):
    """25, 100 and 205 pairs an expert, on average, and one expert with a pair, one with 33, 65 and 97."""
    l = layer(up, down, 6, 256, 256)
    x, ids, w = inputs(l, rows, 3, kind, seed=rows)
    check(l, x, ids, w, kind, apply(l, x, ids, w, kind))
    if rows < 410:
        return
    for few in (1, 33, 65, 97):
        i = ids.copy()
        i[i == 2] = -1
        i[:few, 1] = 2
        check(l, x, i, w, kind, apply(l, x, i, w, kind))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_a_row_of_more_than_the_kernel_of_one_holds(layer, kind):
    l = layer("Q4_K", "Q6_K", 3, 8448, 256)
    x, ids, w = inputs(l, 1, 2, kind)
    check(l, x, ids, w, kind, apply(l, x, ids, w, kind))
    l = layer("Q8_0", "Q8_0", 6, 64, 8192)
    x, ids, w = inputs(l, 1, 6, kind)
    check(l, x, ids, w, kind, apply(l, x, ids, w, kind))


@pytest.mark.parametrize("up,down", PAIRS)
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_few_rows_of_many_experts(layer, up, down, kind):
    """Up to three rows with few pairs take the kernels of one row: as each row alone, bit for bit."""
    l = layer(up, down, 16, 512, 256)
    for rows, top in ((2, 4), (3, 2)):
        x, ids, w = inputs(l, rows, top, kind, seed=rows)
        ids[1] = ids[0]
        ids[-1, 0] = -1
        got = apply(l, x, ids, w, kind, x_stride=520, out_stride=528)
        check(l, x, ids, w, kind, got)
        for r in range(rows):
            assert np.array_equal(got[r:r + 1], apply(l, x[r:r + 1], ids[r:r + 1], w[r:r + 1], kind))


def some_rows(l, x, ids, w, kind, got, rows):
    check(l, x[rows].cpu(), ids[rows], w[rows], kind, got[rows])


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("workspace", [True, False])
def test_more_rows_than_a_range(layer, kind, workspace):
    """At most 2^17 pairs run together: three ranges, of 32834, 32833 and 32833 rows."""
    l = layer("Q8_0", "Q8_0", 6, 64, 64)
    x, ids, w = inputs(l, 98500, 3, kind)
    got = apply(l, x, ids, w, kind, workspace=workspace)
    some_rows(l, x, ids, w, kind, got, np.r_[0:9, 32830:32840, 65660:65672, 98490:98500])
    parts = [apply(l, x[a:b], ids[a:b], w[a:b], kind) for a, b in ((0, 32834), (32834, 65667), (65667, 98500))]
    assert np.array_equal(got, np.concatenate(parts))


@pytest.mark.parametrize("dim,ffn,rows", [(65536, 64, 8200), (64, 65536, 4110)])
def test_activations_of_more_than_2_31_bytes(layer, dim, ffn, rows):
    l = layer("Q8_0", "Q8_0", 2, dim, ffn)
    top = 1 if dim > ffn else 2
    gen = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(rows, dim, generator=gen, device="cuda")
    ids = np.arange(rows * top, dtype=np.int32).reshape(rows, top) % 2
    w = np.random.default_rng(1).random((rows, top)).astype(np.float32)
    got = apply(l, x, ids, w, "f32")
    some_rows(l, x, ids, w, "f32", got, np.r_[0:2, rows // 2 - 2:rows // 2 + 2, rows - 2:rows])


def test_two_streams_at_once(layer):
    l = layer("Q4_K", "Q6_K", 6, 512, 256)
    jobs = []
    for k in range(6):
        x, ids, w = inputs(l, 3 + 20 * k, 2, "f32", seed=k)
        want = apply(l, x, ids, w, "f32")
        jobs.append((x.cuda(), torch.from_numpy(ids).cuda(), torch.from_numpy(w).cuda(), torch.zeros(x.shape, device="cuda"), torch.cuda.Stream(), want))
    torch.cuda.synchronize()
    for _ in range(3):
        for x, ids, w, out, stream, _ in jobs:
            l.experts.apply(x.data_ptr(), ids.data_ptr(), w.data_ptr(), out.data_ptr(), *ids.shape, stream=stream.cuda_stream)
    torch.cuda.synchronize()
    for x, ids, w, out, stream, want in jobs:
        assert np.array_equal(out.cpu().numpy(), want)


@pytest.mark.parametrize("own", [True, False])
@pytest.mark.parametrize("rows", [1, 50])
def test_captured_and_replayed(layer, rows, own):
    """Two graphs, each with a workspace of its own, replayed in turn with other rows and other choices."""
    l = layer("Q4_K", "Q6_K", 6, 512, 256)
    graphs = []
    for k in range(2):
        x, ids, w = (torch.empty(s, device="cuda", dtype=t) for s, t in (((rows, 512), torch.float32), ((rows, 3), torch.int32), ((rows, 3), torch.float32)))
        out = torch.zeros(rows, 512, device="cuda")
        n = l.experts.workspace(rows, 3)
        space = torch.zeros(n, dtype=torch.uint8, device="cuda")
        ids.zero_(), w.zero_(), x.zero_()
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            more = dict(workspace_ptr=space.data_ptr(), workspace_bytes=n) if own else {}
            l.experts.apply(x.data_ptr(), ids.data_ptr(), w.data_ptr(), out.data_ptr(), rows, 3, stream=torch.cuda.current_stream().cuda_stream, **more)
        graphs.append((graph, x, ids, w, out, space))
    for turn in range(4):
        graph, x, ids, w, out, space = graphs[turn % 2]
        a, i, v = inputs(l, rows, 3, "f32", seed=turn)
        want = apply(l, a, i, v, "f32")
        x.copy_(a)
        ids.copy_(torch.from_numpy(i))
        w.copy_(torch.from_numpy(v))
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(out.cpu().numpy(), want), turn


def test_handles(backend):
    l = Layer(backend, "Q8_0", "Q8_0", 2, 64, 128)
    info = l.experts.info()
    assert (info["experts"], info["dim"], info["ffn"], info["weight_bytes"]) == (2, 64, 128, 3 * 2 * 64 * 128 // 32 * 34)
    with pytest.raises(IllegalArgumentException, match="live decode plan"):
        backend.release(l.kept[1])
    x = torch.zeros(1, 64, device="cuda")
    torch.cuda.synchronize()
    with pytest.raises(IllegalArgumentException, match="apart"):
        l.experts.apply(x.data_ptr(), x.data_ptr(), x.data_ptr(), x.data_ptr(), 1, 1)
    handle = l.experts.handle
    l.close()
    l.experts.handle = handle
    with pytest.raises(IllegalArgumentException, match="destroyed"):
        l.experts.apply(x.data_ptr(), x.data_ptr(), x.data_ptr(), x.data_ptr(), 1, 1)
