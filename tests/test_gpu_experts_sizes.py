"""The experts' products (Experts.apply) on both sides of the sizes at which their kernels change, and over many experts."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from test_gpu_experts import apply, check, inputs, layer, some_rows  # noqa: F401

pytestmark = pytest.mark.gpu
KINDS = pytest.mark.parametrize("kind", ["f32", "bf16"])


@KINDS
@pytest.mark.parametrize("up,down", [("Q4_K", "Q6_K"), ("Q6_K", "Q4_K"), ("Q8_0", "Q8_0"), ("Q4_0", "Q4_0")])
@pytest.mark.parametrize("dim", [2048, 2304, 4096, 4352, 8192])
def test_a_row_of_each_width(layer, up, down, kind, dim):  # noqa: F811
    """x of up to 64, 128 and 256 blocks of 32 in LDS."""
    l = layer(up, down, 3, dim, 256)
    x, ids, w = inputs(l, 1, 2, kind, seed=dim)
    check(l, x, ids, w, kind, apply(l, x, ids, w, kind))


@KINDS
@pytest.mark.parametrize("up,down,experts,top,ffn", [
    # blocks of 32 in LDS: 480 (8 waves) and 496 (16), most with 64 KiB 481; 1196, most with a workgroup's LDS 1197; 1204 take other kernels
    ("Q4_K", "Q6_K", 32, 30, 512), ("Q4_K", "Q6_K", 32, 31, 512), ("Q6_K", "Q4_K", 32, 31, 512), ("Q8_0", "Q8_0", 48, 46, 832), ("Q8_0", "Q8_0", 48, 43, 896),
    ("Q4_0", "Q4_0", 4, 2, 16384), ("Q4_K", "Q6_K", 3, 2, 14336)])
def test_a_row_with_each_size_of_inner_activations(layer, up, down, kind, experts, top, ffn):  # noqa: F811
    l = layer(up, down, experts, 256 if up != "Q8_0" else 64, ffn)
    x, ids, w = inputs(l, 1, top, kind, seed=ffn)
    ids[0, -1] = -1 if top > 2 else ids[0, -1]
    check(l, x, ids, w, kind, apply(l, x, ids, w, kind))


@KINDS
@pytest.mark.parametrize("down", ["Q6_K", "Q4_K", "Q8_0", "Q4_0"])
@pytest.mark.parametrize("ffn", [2048, 2304, 3328, 5120])
def test_few_pairs_with_down_split(layer, down, kind, ffn):  # noqa: F811
    """Two to five ranges of down's K, the last one shorter."""
    l = layer("Q4_K" if down.endswith("K") else down, down, 2, 256, ffn)
    x, ids, w = inputs(l, 7, 1, kind, seed=ffn)
    check(l, x, ids, w, kind, apply(l, x, ids, w, kind))


@KINDS
@pytest.mark.parametrize("up,down,dim,ffn", [("Q4_K", "Q6_K", 1280, 1536), ("Q6_K", "Q4_K", 2048, 1024), ("Q6_K", "Q6_K", 768, 1280), ("Q4_K", "Q4_K", 1024, 768),
                                             ("Q8_0", "Q8_0", 448, 704), ("Q8_0", "Q8_0", 320, 1408), ("Q4_0", "Q4_0", 1408, 896), ("Q4_0", "Q8_0", 640, 960)])
def test_many_pairs_of_each_length(layer, up, down, kind, dim, ffn):  # noqa: F811
    """Whole turns of four stages of 64 columns and one, two or three stages more, in tiles of every size."""
    l = layer(up, down, 2, dim, ffn)
    for rows in (60, 150, 400):
        x, ids, w = inputs(l, rows, 1, kind, seed=rows)
        got = apply(l, x, ids, w, kind)
        some_rows(l, x, ids, w, kind, got, np.unique(np.r_[0:8, rows // 2:rows // 2 + 8, rows - 8:rows]))


@KINDS
@pytest.mark.parametrize("experts", [64, 128, 200, 256, 512, 1024])
def test_many_experts(layer, experts, kind):  # noqa: F811
    """From one row to some pairs an expert; then choices that crowd on a few experts, and most slots without one."""
    l = layer("Q8_0", "Q4_0", experts, 128, 128)
    for rows, top in ((1, 8), (2, 8), (3, 8), (5, 64), (33, 8), (600, 8), (30 * experts // 8, 8)):
        x, ids, w = inputs(l, rows, top, kind, seed=rows)
        at = np.unique(np.linspace(0, rows - 1, 24).astype(int))
        some_rows(l, x, ids, w, kind, apply(l, x, ids, w, kind), at)
        crowd = np.sort((np.random.default_rng(rows).random((rows, top)) ** 6 * experts).astype(np.int32), 1)
        crowd[:, 0] = experts - 1
        some_rows(l, x, crowd, w, kind, apply(l, x, crowd, w, kind), at)
        most = np.where(np.random.default_rng(rows + 1).random((rows, top)) < 0.95, -1, ids).astype(np.int32)
        got = apply(l, x, most, w, kind)
        some_rows(l, x, most, w, kind, got, at)
        assert (got[(most < 0).all(1)] == 0).all()


@KINDS
def test_many_experts_in_any_order_of_rows(layer, kind):  # noqa: F811
    """Bit for bit, whichever place a row's pairs get among those of their experts."""
    l = layer("Q8_0", "Q4_0", 256, 128, 128)
    x, ids, w = inputs(l, 3000, 8, kind)
    order = np.random.default_rng(3).permutation(3000)
    a, b = apply(l, x, ids, w, kind), apply(l, x[torch.from_numpy(order)], ids[order], w[order], kind)
    assert np.array_equal(a[order], b)
