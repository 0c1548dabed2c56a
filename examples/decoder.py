"""A small decoder on the engine: quantized projections, rotary positions, the 8-bit key/value cache and its attention.

Random weights (Q8_0) of a Llama-like shape; norms and the gate in torch. A prompt goes through the prefill GEMM and attention of
many rows, tokens through the batched GEMV and attention of few; sequences are forked into beams that share their pages, windowed
layers' old pages are freed, and the pool is compacted::

    python examples/decoder.py --layers 4 --prompt 300 --tokens 32 --beams 4
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import numpy as np
import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
from jax4j_amd import DType, KvCache, Mi355xBackend, QuantType, Rope  # noqa: E402


def q8_0(w: np.ndarray) -> np.ndarray:
    """GGUF Q8_0 blocks of a matrix."""
    b = w.reshape(-1, 32)
    d = (np.abs(b).max(1, keepdims=True) / 127).astype(np.float16)
    q = np.clip(np.rint(b / np.maximum(d.astype(np.float32), 1e-9)), -127, 127).astype(np.int8)
    return np.concatenate([d.view(np.uint8), q.view(np.uint8)], 1)


class Decoder:
    def __init__(self, layers=4, d=1024, heads=8, kv_heads=2, head_dim=128, ffn=2048, vocab=4096, pages=512, page_tokens=16, sequences=8,
                 sequence_pages=256, window=0, sinks=4, seed=0):
        self.be = Mi355xBackend()
        self.layers, self.d, self.heads, self.kv_heads, self.dim = layers, d, heads, kv_heads, head_dim
        self.window, self.sinks = window, sinks if window else 0
        rng = np.random.default_rng(seed)

        def matrix(rows, cols):
            w = q8_0((rng.standard_normal((rows, cols)) / np.sqrt(cols)).astype(np.float32))
            return self.be.upload_quantized(w, QuantType.Q8_0, (rows, cols))

        self.qkv_rows = (heads + 2 * kv_heads) * head_dim
        self.weights = [dict(qkv=matrix(self.qkv_rows, d), o=matrix(d, heads * head_dim), gate_up=matrix(2 * ffn, d), down=matrix(d, ffn))
                        for _ in range(layers)]
        self.embedding = torch.from_numpy(rng.standard_normal((vocab, d)).astype(np.float32)).cuda()
        self.head = matrix(vocab, d)
        self.cache = KvCache(self.be, layers=layers, kv_heads=kv_heads, head_dim=head_dim, pages=pages, page_tokens=page_tokens,
                             sequences=sequences, sequence_pages=sequence_pages)
        rows = page_tokens * sequence_pages
        angle = torch.arange(rows, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(head_dim // 2, dtype=torch.float64) * 2 / head_dim)
        self.cos, self.sin = angle.cos().float().cuda(), angle.sin().float().cuda()
        # a token's place in its sequence is its position
        self.rope = Rope(self.cos.data_ptr(), self.sin.data_ptr(), rows, head_dim, interleaved=True)
        self.stream = torch.cuda.Stream()  # torch's work and the engine's, in order
        torch.cuda.synchronize()

    def close(self):
        torch.cuda.synchronize()
        self.cache.destroy()
        for w in [m for layer in self.weights for m in layer.values()] + [self.head]:
            self.be.release(w)

    def product(self, w, x, add=None):
        """x [rows, cols] . w^T (+ add)."""
        s, rows = self.stream.cuda_stream, x.shape[0]
        y = torch.empty((rows, w.shape[0]), device="cuda")
        if rows <= 16:  # fp32 activations
            self.be.quant_matvec_into(w, x.contiguous().data_ptr(), 0 if add is None else add.data_ptr(), y.data_ptr(), rows, s)
            return y
        self.be.quant_matmul_into(w, x.to(torch.bfloat16).contiguous().data_ptr(), rows, "bf16", 0, 0, y.data_ptr(), s)
        return y if add is None else y + add

    @staticmethod
    def norm(x):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)

    def step(self, seqs, tokens):
        """Appends tokens[i] (a list) to sequence seqs[i]; logits [sequences, vocab] behind the last token of each, on the decoder's
        stream."""
        s, counts = self.stream.cuda_stream, [len(t) for t in tokens]
        with torch.cuda.stream(self.stream):
            h = self.embedding[torch.tensor([t for part in tokens for t in part], device="cuda")]
            rows = h.shape[0]
            few = rows <= 16
            self.cache.extend(seqs, counts, stream=s)
            out = torch.empty((rows, self.heads * self.dim), device="cuda", dtype=torch.float32 if few else torch.bfloat16)
            k_at, v_at = 4 * self.heads * self.dim, 4 * (self.heads + self.kv_heads) * self.dim
            for layer, w in enumerate(self.weights):
                qkv = self.product(w["qkv"], self.norm(h))
                p = qkv.data_ptr()
                # keys turned, quantized and stored, values stored, queries turned in place
                self.cache.append(layer, p + k_at, p + v_at, stride=self.qkv_rows, rope=self.rope, q_ptr=p, heads=self.heads,
                                  q_stride=self.qkv_rows, stream=s)
                self.cache.attend(layer, p, out.data_ptr(), self.heads, q_stride=self.qkv_rows, out_type=DType.F32 if few else DType.BF16,
                                  window=self.window, sinks=self.sinks, stream=s)
                h = self.product(w["o"], out, h)
                gate, up = self.product(w["gate_up"], self.norm(h)).chunk(2, -1)
                h = self.product(w["down"], torch.nn.functional.silu(gate) * up, h)
            last = torch.tensor(np.cumsum(counts) - 1, device="cuda")
            logits = self.product(self.head, self.norm(h[last]))
        if self.window:
            self.cache.evict(seqs, self.window, self.sinks, stream=s)
        return logits


def generate(m, a):
    rng = np.random.default_rng(1)
    prompts = [rng.integers(0, 4096, n).tolist() for n in (a.prompt, a.prompt // 3 + 1)]
    logits = m.step([0, 1], prompts)
    # the first prompt's likeliest tokens as beams beside it
    beams = list(range(2, 2 + a.beams - 1))
    if beams:
        m.cache.fork([0] * len(beams), beams, stream=m.stream.cuda_stream)
    top = torch.topk(logits[0], a.beams).indices.tolist()
    seqs, tokens = [0, *beams, 1], [*top, int(logits[1].argmax())]
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    start.record(m.stream)
    for _ in range(a.tokens):
        tokens = m.step(seqs, [[t] for t in tokens]).argmax(-1).tolist()
    end.record(m.stream)
    end.synchronize()
    info = m.cache.info()
    print(f"{len(seqs)} sequences, {a.tokens} tokens each in {start.elapsed_time(end):.1f} ms; {info['pages'] - info['pages_free']} pages in use")
    m.cache.truncate([0, 1], [0, 0])
    moved = m.cache.compact(stream=m.stream.cuda_stream)
    info = m.cache.info()
    print(f"two sequences freed, {moved} pages moved; {info['pages'] - info['pages_free']} pages in use")
    tokens = m.step(beams, [[t] for t in tokens[1:a.beams]]).argmax(-1).tolist() if beams else []
    print("next tokens of the beams left:", tokens)


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--prompt", type=int, default=300)
    ap.add_argument("--tokens", type=int, default=32)
    ap.add_argument("--beams", type=int, default=4)
    ap.add_argument("--window", type=int, default=0)
    a = ap.parse_args()
    m = Decoder(layers=a.layers, window=a.window)
    with torch.cuda.stream(m.stream):
        generate(m, a)
    m.close()


if __name__ == "__main__":
    main()
