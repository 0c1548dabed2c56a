"""The example decoder against the same decoder in plain torch: fp32 throughout, keys and values as they are.

Bar: the cache's codes are off by half a step of 1/127 of their block's largest magnitude (about four standard deviations: 1.6 %
of one, evenly spread: 0.9 % in the mean), prefill rounds its activations to bf16 (0.2 %). Every layer adds such errors to the
residual, so the logits of a few layers stay well within 5 % of the plain ones in the 2-norm. A mask, a position or a page that
is wrong moves them by tens of percent.
"""
from __future__ import annotations

import sys
from pathlib import Path

import numpy as np
import pytest
import torch

import kv_ref as R

pytestmark = pytest.mark.gpu
sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))


@pytest.fixture(params=[0, 40], ids=["whole", "window"])
def model(request):
    from decoder import Decoder

    m = Decoder(layers=3, d=512, heads=4, kv_heads=2, head_dim=128, ffn=512, vocab=512, window=request.param)
    yield m
    m.close()


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
        gate, up = (m.norm(h) @ w(layer["gate_up"])[0].t()).chunk(2, -1)
        h = (torch.nn.functional.silu(gate) * up) @ w(layer["down"])[0].t() + h
    return m.norm(h[-1:]) @ w(m.head)[0].t()


def near(got, want):
    off = float((got - want).norm() / want.norm())
    assert off < 0.05, off


def test_prompt_tokens_beams_and_freed_pages(model):
    m = model
    rng = np.random.default_rng(3)
    text = {0: rng.integers(0, 512, 90).tolist(), 1: rng.integers(0, 512, 21).tolist()}
    logits = m.step([0, 1], [text[0], text[1]])
    m.stream.synchronize()
    for i in (0, 1):
        near(logits[i:i + 1], plain(m, text[i]))
    m.cache.fork([0, 0, 1], [2, 3, 4], stream=m.stream.cuda_stream)
    text |= {2: list(text[0]), 3: list(text[0]), 4: list(text[1])}
    for step in range(20):
        new = {s: int(rng.integers(0, 512)) for s in text}
        logits = m.step(list(text), [[t] for t in new.values()])
        for s in text:
            text[s].append(new[s])
    m.stream.synchronize()
    for i, s in enumerate(text):
        near(logits[i:i + 1], plain(m, text[s]))
    m.cache.truncate([0, 2], [0, 0])
    m.cache.compact(stream=m.stream.cuda_stream)
    more = rng.integers(0, 512, 33).tolist()  # a chunk behind what is there, and a new sequence in freed pages
    logits = m.step([3, 0], [more, text[1]])
    m.stream.synchronize()
    near(logits[:1], plain(m, text[3] + more))
    near(logits[1:], plain(m, text[1]))
