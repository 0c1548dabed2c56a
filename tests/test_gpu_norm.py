"""Norms before and after a block, its gate and the residual (Mi355xBackend.norm_into) against 64 bits."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import experts_ref as ref
from jax4j_amd import DType, IllegalArgumentException, Norm

pytestmark = pytest.mark.gpu
TYPES = {"f32": (DType.F32, torch.float32), "bf16": (DType.BF16, torch.bfloat16)}


def on_gpu(a, kind="f32", stride=0):
    """The values at the type's precision, on the GPU, rows `stride` values apart, and as numpy has them."""
    t = torch.from_numpy(np.ascontiguousarray(a, np.float32)).to(TYPES[kind][1])
    seen = t.float().numpy()
    if stride:
        wide = torch.full((*t.shape[:-1], stride), 77.0, dtype=t.dtype)
        wide[..., :t.shape[-1]] = t
        t = wide
    return t.cuda(), seen


def call(backend, case, seed=0, inplace=False):
    rng = np.random.default_rng(seed)
    rows, dim = case["rows"], case["dim"]
    kinds = {k: case.get(k, "f32") for k in ("residual", "block", "gate", "out")}
    pad = case.get("pad", 0)
    stride = dim + pad if pad else 0
    shape = (rows, dim)
    spread, shift = case.get("spread", 1.0), case.get("shift", 0.0)
    res, res_seen = on_gpu(spread * rng.standard_normal(shape) + shift, kinds["residual"], stride)
    blk, blk_seen = on_gpu(spread * rng.standard_normal(shape) + shift, kinds["block"], stride)
    every = case.get("every", 0)
    gates = -(-rows // every) if every else 1
    gate, gate_seen = on_gpu(rng.standard_normal((gates, dim)), kinds["gate"], stride)
    norms, plain = {}, {}
    keep = []
    for name in ("after", "before"):
        kind = case.get(name)
        if kind is None:
            norms[name] = plain[name] = None
            continue
        w, b = rng.standard_normal(dim).astype(np.float32), (rng.standard_normal(dim).astype(np.float32) if case.get("bias") else None)
        if case.get("no_weight"):
            w = None
        tw, tb = (None if v is None else torch.from_numpy(v).cuda() for v in (w, b))
        keep += [tw, tb]
        add = 1.0 if case.get("add") else 0.0
        norms[name] = Norm(tw.data_ptr() if w is not None else 0, kind, bias_ptr=tb.data_ptr() if b is not None else 0, eps=1e-5, weight_add=add)
        plain[name] = (kind, w, b, float(np.float32(1e-5)), add)
    has = case.get("has", ("residual", "block"))
    gated = case.get("gated", False)
    h = res if inplace else torch.full_like(res, 55.0)
    out = torch.full((rows, stride or dim), 55.0, dtype=TYPES[kinds["out"]][1], device="cuda")
    torch.cuda.synchronize()
    backend.norm_into(res.data_ptr() if "residual" in has else 0, out.data_ptr() if norms["before"] else 0, rows, dim, norms["before"],
                      residual_type=TYPES[kinds["residual"]][0], out_type=TYPES[kinds["out"]][0], block_ptr=blk.data_ptr() if "block" in has else 0,
                      block_type=TYPES[kinds["block"]][0], after=norms["after"], gate_ptr=gate.data_ptr() if gated else 0,
                      gate_type=TYPES[kinds["gate"]][0], gate_every=every, scale=case.get("scale", 1.0), residual_out_ptr=h.data_ptr(),
                      residual_stride=stride, block_stride=stride, gate_stride=stride, residual_out_stride=stride, out_stride=stride)
    backend.sync()
    eh, oh, ey, oy = ref.norm(res_seen if "residual" in has else None, blk_seen if "block" in has else None, gate_seen if gated else None, every,
                              float(np.float32(case.get("scale", 1.0))), plain["after"], plain["before"])
    for name, got, want, off, kind in (("h", h, eh, oh, kinds["residual"]), ("y", out, ey, oy, kinds["out"])):
        if want is None:
            continue
        g = got[:, :dim].float().cpu().numpy().astype(np.float64)
        off = off + (ref.STEP["bf16"] * (np.abs(want) + off) if kind == "bf16" else 0.0)
        bad = ~(np.abs(g - want) <= off)
        assert not bad.any(), (name, case, np.argwhere(bad)[:4], g[bad][:4], want[bad][:4], off[bad][:4])
        if stride:
            assert (got[:, dim:] == (77.0 if name == "h" and inplace else 55.0)).all()
    return h, out


@pytest.mark.parametrize("dim", [1, 7, 64, 65, 512, 520, 1000, 2048, 2052, 4096, 5001, 8192, 8200, 16384, 20000, 32768])
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_sizes(backend, dim, kind):
    call(backend, dict(rows=5, dim=dim, after=kind, before=kind, bias=kind == "layer", scale=0.25, out="bf16", block="bf16"))


@pytest.mark.parametrize("residual", ["f32", "bf16"])
@pytest.mark.parametrize("block", ["f32", "bf16"])
@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("gate", ["f32", "bf16"])
def test_types(backend, residual, block, out, gate):
    call(backend, dict(rows=9, dim=768, after="rms", before="rms", residual=residual, block=block, out=out, gate=gate, gated=True, every=4))


@pytest.mark.parametrize("case", [
    dict(rows=3, dim=640, before="rms", has=("residual",)),
    dict(rows=3, dim=640, before="rms", has=("block",), scale=-2.0),
    dict(rows=3, dim=640, has=("residual", "block"), gated=True),
    dict(rows=3, dim=640, has=("block",), after="layer", bias=True),
    dict(rows=3, dim=640, before="layer", no_weight=True),
    dict(rows=3, dim=640, before="rms", after="rms", add=True),
    dict(rows=67, dim=96, before="rms", after="layer", gated=True, every=13),
    dict(rows=6, dim=640, before="rms", after="rms", gated=True, pad=8, block="bf16"),
    dict(rows=6, dim=641, before="rms", after="rms", gated=True, pad=3, block="bf16", out="bf16"),
    # sums of squares above what 32 bits hold, and far below
    dict(rows=4, dim=1024, before="rms", spread=1e25),
    dict(rows=4, dim=1024, before="rms", spread=1e-25, has=("residual",)),
    # a mean far from the values' spread
    dict(rows=4, dim=4096, before="layer", shift=4096.0, has=("residual",)),
])
def test_parts(backend, case):
    call(backend, case)


@pytest.mark.parametrize("residual", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [768, 771])
def test_in_place_is_apart(backend, residual, dim):
    case = dict(rows=70, dim=dim, after="rms", before="layer", residual=residual, pad=5 if dim % 8 else 0)
    h0, y0 = call(backend, case)
    h1, y1 = call(backend, case, inplace=True)
    assert torch.equal(h0[:, :dim], h1[:, :dim]) and torch.equal(y0, y1)


def test_rows_are_independent_of_their_place(backend):
    """A row's result does not depend on the others: a row of NaN and infinities stays alone, and equal rows are equal."""
    x = torch.randn(300, 512, device="cuda")
    x[200] = x[3]
    x[7, 100], x[9, 5] = float("nan"), float("inf")
    y = torch.empty_like(x)
    torch.cuda.synchronize()
    backend.norm_into(x.data_ptr(), y.data_ptr(), 300, 512, Norm())
    backend.sync()
    assert torch.equal(y[200], y[3]) and y[7].isnan().all() and y[9].isnan().any()
    rest = [i for i in range(300) if i not in (7, 9)]
    assert y[rest].isfinite().all()


def test_many_rows_and_another_stream(backend):
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        x = torch.randn(70000, 64, device="cuda", dtype=torch.bfloat16)
        y = torch.empty_like(x)
        backend.norm_into(x.data_ptr(), y.data_ptr(), 70000, 64, Norm(), residual_type=DType.BF16, out_type=DType.BF16, stream=stream.cuda_stream)
        want = x.double() * torch.rsqrt(x.double().square().mean(-1, keepdim=True) + 1e-6)
        off = (y.double() - want).abs()
    stream.synchronize()
    assert bool((off <= want.abs() * (2.0 ** -8 + 8 * 2.0 ** -24)).all())


def test_captured_and_replayed(backend):
    x, w = torch.randn(33, 1024, device="cuda"), torch.randn(1024, device="cuda")
    h, y = torch.empty_like(x), torch.empty_like(x)
    norm = Norm(w.data_ptr())
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        backend.norm_into(x.data_ptr(), y.data_ptr(), 33, 1024, norm, residual_out_ptr=h.data_ptr(), stream=torch.cuda.current_stream().cuda_stream)
    for k in range(3):
        x.copy_(torch.randn(33, 1024, device="cuda") * (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        got = y.clone()
        y.zero_()
        torch.cuda.synchronize()
        backend.norm_into(x.data_ptr(), y.data_ptr(), 33, 1024, norm, residual_out_ptr=h.data_ptr())
        backend.sync()
        assert torch.equal(got, y)


def test_refusals_leave_memory_alone(backend):
    x = torch.zeros(8, 64, device="cuda")
    torch.cuda.synchronize()
    with pytest.raises(IllegalArgumentException, match="overlaps"):
        backend.norm_into(x.data_ptr(), x.data_ptr() + 64, 4, 64, Norm())
    with pytest.raises(IllegalArgumentException, match="together"):
        backend.norm_into(x.data_ptr(), x.data_ptr() + 1024, 4, 64)


@pytest.mark.parametrize("dim", [7, 48, 100, 1000, 1152, 3000, 5001])
def test_rows_of_equal_values(backend, dim):
    """Less their mean nothing is left, whatever dim is, with an eps far below what a mean off in its last bit would leave."""
    value = torch.tensor([[0.1], [1e6 / 3], [-7e-20], [3e30]], dtype=torch.float32)
    x = value.expand(4, dim).contiguous().cuda()
    out = torch.full((4, dim), 5.0, device="cuda")
    torch.cuda.synchronize()
    backend.norm_into(x.data_ptr(), out.data_ptr(), 4, dim, Norm(kind="layer", eps=1e-30))
    torch.cuda.synchronize()
    assert (out == 0).all()
