"""Routing to experts (Mi355xBackend.route_into) against 64 bits: the choice exactly, the weights to their last bits."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import experts_ref as ref
from jax4j_amd import DType

pytestmark = pytest.mark.gpu
# The exponential is within 1 step of its value, of a difference that is rounded once (2^-24 of up to 90, as far as a score counts
# beside the largest: its weight moves by 90 2^-24 of itself); the sum of up to 1024 terms by lanes and exchanges within 26 steps; a
# quotient and a product a step each.
REL = (90 + 1 + 26 + 2 + 2) * 2.0 ** -24
TINY = 2.0 ** -126


def call(backend, logits, k, dtype="f32", bias=None, stride=0, **more):
    rows, experts = logits.shape
    t = torch.from_numpy(np.ascontiguousarray(logits, np.float32))
    if dtype == "bf16":
        t = t.bfloat16()
    seen = t.float().numpy()
    if stride:
        wide = torch.full((rows, stride), 1e9, dtype=t.dtype)
        wide[:, :experts] = t
        t = wide
    t = t.cuda()
    b = None if bias is None else torch.from_numpy(bias.astype(np.float32)).cuda()
    ids, weights = torch.full((rows + 1, k), 99, device="cuda", dtype=torch.int32), torch.full((rows + 1, k), 99.0, device="cuda")
    torch.cuda.synchronize()
    backend.route_into(t.data_ptr(), ids.data_ptr(), weights.data_ptr(), rows, experts, k, dtype=DType.BF16 if dtype == "bf16" else DType.F32,
                       stride=stride, bias_ptr=0 if b is None else b.data_ptr(), **more)
    backend.sync()
    assert (ids[rows] == 99).all() and (weights[rows] == 99.0).all()
    want_ids, want = ref.route(seen, k, more.get("score", "softmax"), None if bias is None else bias.astype(np.float32), more.get("groups", 1),
                               more.get("top_groups", 1), more.get("group_best", 1), more.get("renormalize", False), more.get("scale", 1.0))
    got_ids, got = ids[:rows].cpu().numpy(), weights[:rows].cpu().numpy().astype(np.float64)
    bad = np.argwhere(got_ids != want_ids)
    assert not bad.size, (bad[:4], got_ids[bad[0][0]], want_ids[bad[0][0]])
    assert (np.abs(got - want) <= REL * np.abs(want) + TINY * abs(more.get("scale", 1.0))).all(), np.abs(got - want).max()
    return got_ids, got


@pytest.mark.parametrize("experts", [1, 2, 7, 16, 32, 33, 60, 64, 100, 128, 129, 160, 256, 384, 512, 777, 1024])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
def test_sizes(backend, experts, score, biased):
    rng = np.random.default_rng(experts)
    for rows, k in ((1, 1), (1, min(8, experts)), (37, min(8, experts)), (5, min(33, experts)), (3, min(64, experts))):
        x = 3 * rng.standard_normal((rows, experts))
        bias = 0.3 * rng.standard_normal(experts) if biased else None
        call(backend, x, k, score=score, bias=bias, renormalize=k % 2 == 0, scale=2.5)


@pytest.mark.parametrize("groups,top_groups,best", [(2, 1, 1), (4, 2, 2), (8, 4, 2), (8, 8, 1), (16, 3, 2), (32, 5, 1), (64, 7, 1)])
@pytest.mark.parametrize("biased", [False, True])
def test_groups(backend, groups, top_groups, best, biased):
    rng = np.random.default_rng(groups)
    for experts in (64, 192, 256):
        x = 2 * rng.standard_normal((41, experts))
        x[rng.random(x.shape) < 0.1] = -np.inf
        x[3] = -np.inf
        x[4, 1:] = -np.inf
        k = min(6, experts // groups * top_groups)
        for score in ("softmax", "sigmoid"):
            call(backend, x, k, score=score, bias=0.2 * rng.standard_normal(experts) if biased else None, groups=groups, top_groups=top_groups,
                 group_best=best, renormalize=True)


@pytest.mark.parametrize("experts", [48, 300])
def test_ties_go_to_the_lowest_index(backend, experts):
    rng = np.random.default_rng(5)
    x = rng.integers(-2, 3, (50, experts)).astype(np.float32)
    x[0] = 0.0
    x[1] = np.where(np.arange(experts) % 2, 0.0, -0.0)  # equal zeros
    x[2] = 1e30
    bias = rng.integers(0, 2, experts) * 0.5
    for score in ("softmax", "sigmoid"):
        ids, _ = call(backend, x, 8, score=score)
        assert (ids[:3] == np.arange(8)).all()
        call(backend, x, 8, score=score, bias=bias, dtype="bf16")
        call(backend, x, 8, score=score, groups=4, top_groups=2, group_best=2)


@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("experts", [24, 200])
def test_what_may_not_be_chosen(backend, experts, biased):
    rng = np.random.default_rng(6)
    x = rng.standard_normal((30, experts)).astype(np.float32)
    x[0], x[1], x[2, 2:] = -np.inf, np.nan, -np.inf
    x[3, ::2] = np.nan
    x[4, 5] = np.inf
    x[5, [3, 9]] = np.inf
    x[6] = np.inf
    x[7] = np.finfo(np.float32).min
    x[8] = np.linspace(-1e38, 1e38, experts)
    bias = 0.1 * rng.standard_normal(experts).astype(np.float32) if biased else None
    if biased:
        bias[[1, 4]] = -np.inf, np.nan
    for score in ("softmax", "sigmoid"):
        for renormalize in (False, True):
            ids, w = call(backend, x, 5, score=score, bias=bias, renormalize=renormalize)
            assert (ids[:2] == -1).all() and (w[:2] == 0).all()


def test_sigmoid_shares_of_tiny_scores(backend):
    """Scores that 32 bits do not hold still share the weights."""
    x = np.full((3, 32), -300.0, np.float32)
    x[0, :4] = -200, -201, -202, -203
    x[1, :4] = -95, -96, -99, -105
    x[2, :4] = 40, 30, -200, -300
    call(backend, x, 4, score="sigmoid", renormalize=True)


def test_borders_that_32_bits_do_not_tell_apart(backend):
    """Sums of score and bias that differ by less than a step of 32 bits are put in their order."""
    rng = np.random.default_rng(7)
    x = rng.standard_normal((200, 64)).astype(np.float32)
    s = 1 / (1 + np.exp(-x[0].astype(np.float64)))
    bias = (1.0 - s).astype(np.float32)  # every sum of the first row within 2^-25 of 1
    x[1:] = x[0] + 1e-7 * rng.standard_normal((199, 64))
    call(backend, x, 8, score="sigmoid", bias=bias, renormalize=True)


def test_strides_types_and_many_rows(backend):
    rng = np.random.default_rng(8)
    call(backend, rng.standard_normal((11, 60)), 6, stride=67)
    call(backend, rng.standard_normal((11, 60)), 6, stride=61, dtype="bf16", score="sigmoid")
    call(backend, rng.standard_normal((5001, 96)), 7, dtype="bf16", renormalize=True)


def test_another_stream_and_a_graph(backend):
    x = torch.randn(77, 64, device="cuda")
    ids, w = torch.zeros(77, 8, device="cuda", dtype=torch.int32), torch.zeros(77, 8, device="cuda")
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        backend.route_into(x.data_ptr(), ids.data_ptr(), w.data_ptr(), 77, 64, 8, renormalize=True, stream=torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        x.copy_(torch.randn(77, 64, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        want, _ = ref.route(x.cpu().numpy(), 8, "softmax")
        assert (ids.cpu().numpy() == want).all()
        ids.zero_()
        torch.cuda.synchronize()
