"""Attention captured behind a short context and run behind one so long that its ranges of tokens, as many as there is room for parts,
have to grow: what the same call gives in ranges of its own, up to the roundings of another order of sums (of means of the
values, which are about 4 at most: 1e-5 of that, as for captured steps elsewhere)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from test_gpu_kv import KIND, dev, model  # noqa: F401

pytestmark = pytest.mark.gpu


# rows of a kv head: few, some, many; room for 8, 5 and 16 ranges
@pytest.mark.parametrize("seqs,heads,tokens,short,long", [(64, 128, 1, 60, 20000), (64, 48, 4, 60, 20000), (1, 128, 32, 96, 6000)])
@pytest.mark.parametrize("window", [0, 5000])
def test_captured_behind_a_short_context(model, seqs, heads, tokens, short, long, window):  # noqa: F811
    m = model(kv_heads=8, head_dim=64, pages=long // 64 + 3 * seqs, page_tokens=64, sequences=seqs, sequence_pages=long // 64 + 3)
    rng = np.random.default_rng(tokens)

    def grow(s, n):
        k, v = (dev(rng.standard_normal((len(s) * n, 8, 64)).astype(np.float32)) for _ in range(2))
        m.kv.extend(s, [n] * len(s))
        torch.cuda.synchronize()
        m.kv.append(0, k.data_ptr(), v.data_ptr())
        torch.cuda.synchronize()

    def share():
        if seqs > 1:
            m.kv.fork([0] * (seqs - 1), range(1, seqs))
        grow(range(seqs), tokens)

    q = torch.randn((seqs * tokens, heads, 64), device="cuda")
    out = torch.zeros_like(q)
    call = lambda s: m.kv.attend(0, q.data_ptr(), out.data_ptr(), heads, q_type=KIND["f32"], window=window, stream=s)  # noqa: E731
    grow([0], short)
    share()
    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        call(s.cuda_stream)
    for length in (None, long // 3, long):
        if length:
            m.kv.truncate(range(seqs), [0] * seqs)
            grow([0], length)
            share()
        for _ in range(2):
            out.fill_(7.0)
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            got = out.clone()
            out.fill_(9.0)
            torch.cuda.synchronize()
            call(0)
            torch.cuda.synchronize()
            assert float((got - out).abs().max()) <= 4e-5, length
