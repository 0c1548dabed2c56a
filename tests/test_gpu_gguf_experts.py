"""A layer of experts out of a GGUF file's three-dimensional tensors (experts, rows, columns), as the products take it."""
from __future__ import annotations

from types import SimpleNamespace

import pytest

import experts_ref as ref
from gguf_fixtures import gguf_bytes
from jax4j_amd import Experts, QuantType
from jax4j_amd import synthetic as S
from jax4j_amd.gguf import GGUFFile
from test_gpu_experts import apply, check, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("up,down", [("Q4_K", "Q6_K"), ("Q8_0", "Q8_0")])
def test_three_dimensional_tensors(backend, tmp_path, up, down, kind):
    experts, dim, ffn = 5, 256, 512
    tensors, plain = [], []
    for i, (name, qt, rows, cols) in enumerate((("gate", QuantType[up], ffn, dim), ("up", QuantType[up], ffn, dim), ("down", QuantType[down], dim, ffn))):
        blocks = S.quant_blocks(qt, 30 + i, experts * rows, cols)
        tensors.append((f"blk.0.ffn_{name}_exps.weight", qt.id, [cols, rows, experts], blocks.tobytes()))
        plain.append(tuple(v.reshape(experts, rows, cols) for v in ref.dequantize(blocks, qt, experts * rows, cols)))
    path = tmp_path / "m.gguf"
    path.write_bytes(gguf_bytes([("general.architecture", 8, "llama")], tensors))
    with GGUFFile(path) as f:
        kept = [f.upload(backend, name) for name, *_ in tensors]
    assert [w.shape for w in kept] == [(experts * ffn, dim), (experts * ffn, dim), (experts * dim, ffn)]
    layer = SimpleNamespace(experts=Experts(backend, *kept, experts=experts), plain=plain, act="silu", n=experts, dim=dim)
    for rows in (1, 9, 100):
        x, ids, w = inputs(layer, rows, 2, kind, seed=rows)
        check(layer, x, ids, w, kind, apply(layer, x, ids, w, kind))
    layer.experts.destroy()
    for w in kept:
        backend.release(w)
