"""Norms of rows beyond 16384 values (Mi355xBackend.norm_into): wide and single loads, every part, in place, many rows."""
from __future__ import annotations

import pytest
import torch

from jax4j_amd import Norm
from test_gpu_norm import call

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [16385, 16392, 20000, 24001, 24576, 32767, 32768])
@pytest.mark.parametrize("after,before", [("rms", "layer"), ("layer", "rms"), (None, "rms"), ("layer", None)])
def test_parts_of_long_rows(backend, dim, after, before):
    case = dict(rows=7, dim=dim, bias=True, gated=True, every=3, scale=0.25, block="bf16", out="bf16")
    case.update({k: v for k, v in (("after", after), ("before", before)) if v})
    call(backend, case)
    call(backend, dict(case, residual="bf16", block="f32", gate="bf16", out="f32", pad=8))
    call(backend, dict(case, pad=3, has=("block",)))


@pytest.mark.parametrize("dim", [20000, 20003])
def test_long_rows_in_place(backend, dim):
    case = dict(rows=40, dim=dim, after="layer", before="rms", residual="bf16", pad=5 if dim % 8 else 0)
    h0, y0 = call(backend, case)
    h1, y1 = call(backend, case, inplace=True)
    assert torch.equal(h0[:, :dim], h1[:, :dim]) and torch.equal(y0, y1)


def test_long_rows_are_independent(backend):
    x = torch.randn(600, 16640, device="cuda")
    x[400] = x[3]
    x[7, 16600], x[9, 5] = float("nan"), float("inf")
    y = torch.empty_like(x)
    torch.cuda.synchronize()
    backend.norm_into(x.data_ptr(), y.data_ptr(), 600, 16640, Norm(kind="layer"))
    backend.sync()
    assert torch.equal(y[400], y[3]) and y[7].isnan().all()
    rest = [i for i in range(600) if i not in (7, 9)]
    assert y[rest].isfinite().all()
