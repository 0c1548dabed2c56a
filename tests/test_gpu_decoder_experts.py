"""The example decoder with layers of experts, and such a layer's run of operators: norm, router, choice, experts, the next norm.

The decoder's bar is that of test_gpu_decoder_example.py, 5 % of the logits' 2-norm: every expert is chosen, so that no rounding decides a
choice, and the routing weights and the experts' products add errors of the sizes already there (activations in bf16 for prompts). In the
run each operator is held to its own bound, from what the one before it gave.
"""
from __future__ import annotations

import sys
from pathlib import Path
from types import SimpleNamespace

import numpy as np
import pytest
import torch

import experts_ref as ref
import kv_ref as R
from jax4j_amd import DType, Norm
from test_gpu_experts import Layer
from test_gpu_route import REL

pytestmark = pytest.mark.gpu
sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))


def plain(m, tokens):
    """Logits behind the last token."""
    def w(x):
        return torch.from_numpy(m.be.download(x_dev := m.be.dequantize(x)).reshape(x.shape)).cuda(), m.be.release(x_dev)

    h = m.embedding[torch.tensor(tokens, device="cuda")]
    n = len(tokens)
    cos, sin = m.cos.cpu().numpy(), m.sin.cpu().numpy()
    at = np.repeat(np.arange(n)[:, None], m.dim // 2, 1)
    for layer in m.weights:
        qkv = (m.norm(h) @ w(layer["qkv"])[0].t()).reshape(n, -1, m.dim).cpu().numpy()
        q, k, v = np.split(qkv, [m.heads, m.heads + m.kv_heads], 1)
        q, k = (R.rotate(x, cos, sin, at, True) for x in (q, k))
        o = R.attend(q, k, v, 0, m.window, m.sinks)[0].reshape(n, -1)
        h = torch.from_numpy(o).float().cuda() @ w(layer["o"])[0].t() + h
        x = m.norm(h)
        share = torch.softmax(x @ w(layer["router"])[0].t(), -1)
        gate, up, down = (w(layer[k])[0].reshape(m.experts, -1, w_cols) for k, w_cols in (("gate", m.d), ("up", m.d), ("down", layer["down"].shape[1])))
        for e in range(m.experts):
            h = h + share[:, e:e + 1] * ((torch.nn.functional.silu(x @ gate[e].t()) * (x @ up[e].t())) @ down[e].t())
    return m.norm(h[-1:]) @ w(m.head)[0].t()


def test_decoder_with_experts():
    from decoder import Decoder

    m = Decoder(layers=3, d=512, heads=4, kv_heads=2, head_dim=128, ffn=256, vocab=512, experts=4, top=4)
    try:
        rng = np.random.default_rng(3)
        text = {0: rng.integers(0, 512, 90).tolist(), 1: rng.integers(0, 512, 21).tolist()}
        logits = m.step([0, 1], [text[0], text[1]])
        for turn in range(4):
            if turn:
                new = {s: int(rng.integers(0, 512)) for s in text}
                logits = m.step(list(text), [[t] for t in new.values()])
                for s in text:
                    text[s].append(new[s])
            m.stream.synchronize()
            for i, s in enumerate(text):
                want = plain(m, text[s])
                assert float((logits[i:i + 1] - want).norm() / want.norm()) < 0.05
    finally:
        m.close()


def test_generate_with_experts(capsys):
    from decoder import Decoder, generate

    m = Decoder(layers=2, d=512, heads=4, kv_heads=2, head_dim=128, ffn=512, experts=8, top=2)
    try:
        with torch.cuda.stream(m.stream):
            generate(m, SimpleNamespace(prompt=40, tokens=3, beams=2))
        assert "3 sequences, 3 tokens each" in capsys.readouterr().out
    finally:
        m.close()


@pytest.mark.parametrize("kind,rows", [("f32", 1), ("f32", 13), ("bf16", 70)])
def test_a_layer_of_experts(backend, kind, rows):
    l = Layer(backend, "Q4_K", "Q6_K", 16, 512, 256)
    try:
        half = kind == "bf16"
        dt, torch_dt = (DType.BF16, torch.bfloat16) if half else (DType.F32, torch.float32)
        rng = np.random.default_rng(rows)
        h0, a0 = (torch.from_numpy(rng.standard_normal((rows, 512)).astype(np.float32)) for _ in range(2))
        wn = [(1 + 0.1 * rng.standard_normal(512)).astype(np.float32) for _ in range(2)]
        router = torch.from_numpy((rng.standard_normal((16, 512)) / 22).astype(np.float32)).cuda()
        h, a = h0.cuda(), a0.cuda()
        w1, w2 = (torch.from_numpy(w).cuda() for w in wn)
        x, y, z = (torch.empty(rows, 512, device="cuda", dtype=torch_dt) for _ in range(3))
        ids, weights = torch.empty(rows, 4, device="cuda", dtype=torch.int32), torch.empty(rows, 4, device="cuda")
        stream = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            s = stream.cuda_stream
            backend.norm_into(h.data_ptr(), x.data_ptr(), rows, 512, Norm(w1.data_ptr()), block_ptr=a.data_ptr(), residual_out_ptr=h.data_ptr(), out_type=dt, stream=s)
            h1 = h.clone()
            logits = x.float() @ router.t()
            backend.route_into(logits.data_ptr(), ids.data_ptr(), weights.data_ptr(), rows, 16, 4, renormalize=True, stream=s)
            l.experts.apply(x.data_ptr(), ids.data_ptr(), weights.data_ptr(), y.data_ptr(), rows, 4, dt, stream=s)
            backend.norm_into(h.data_ptr(), z.data_ptr(), rows, 512, Norm(w2.data_ptr()), block_ptr=y.data_ptr(), block_type=dt, residual_out_ptr=h.data_ptr(),
                              out_type=dt, stream=s)
        stream.synchronize()

        def near(got, want, off, step):
            got = got.double().cpu().numpy()
            assert (np.abs(got - want) <= off + step * (np.abs(want) + off) + 2.0 ** -126).all()

        n1, n2 = (("rms", w, None, 1e-6, 0.0) for w in wn)
        want_h, eh, want_x, ex = ref.norm(h0.numpy(), a0.numpy(), None, 0, 1.0, None, n1)
        near(h1, want_h, eh, ref.STEP["f32"])
        near(x, want_x, ex, ref.STEP[kind])
        want_ids, want_w = ref.route(logits.cpu().numpy(), 4, "softmax", renormalize=True)
        assert np.array_equal(ids.cpu().numpy(), want_ids)
        assert np.allclose(weights.cpu().numpy(), want_w, rtol=REL, atol=0)
        want_y, ey = ref.experts(x.float().cpu().numpy(), ids.cpu().numpy(), weights.cpu().numpy(), *l.plain, "silu", kind, exact_weights=False)
        near(y, want_y, ey, ref.STEP[kind])
        want_h, eh, want_z, ez = ref.norm(h1.cpu().numpy(), y.float().cpu().numpy(), None, 0, 1.0, None, n2)
        near(h, want_h, eh, ref.STEP["f32"])
        near(z, want_z, ez, ref.STEP[kind])
    finally:
        l.close()
