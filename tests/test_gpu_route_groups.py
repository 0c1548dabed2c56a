"""Ranks of groups by the sum of their two best scores (Mi355xBackend.route_into) against 64 bits."""
from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def scores(x, score):
    """In 64 bits; of rows whose largest logit is finite."""
    with np.errstate(invalid="ignore", over="ignore"):
        if score == "sigmoid":
            return 1 / (1 + np.exp(-x))
        s = np.exp(x - x.max(1, keepdims=True))
    return s / s.sum(1, keepdims=True)


def call(backend, x, k, bias=None, **more):
    t = torch.from_numpy(x.astype(np.float32)).cuda()
    b = None if bias is None else torch.from_numpy(bias.astype(np.float32)).cuda()
    ids, weights = torch.full((len(x), k), 99, device="cuda", dtype=torch.int32), torch.full((len(x), k), 99.0, device="cuda")
    torch.cuda.synchronize()
    backend.route_into(t.data_ptr(), ids.data_ptr(), weights.data_ptr(), *x.shape, k, bias_ptr=0 if b is None else b.data_ptr(), **more)
    backend.sync()
    return ids.cpu().numpy(), weights.cpu().numpy().astype(np.float64)


def choice(x, k, score, groups, top_groups):
    """The k largest logits of the groups with the largest sums of two scores (of one where one is left)."""
    s = np.where(x > -np.inf, scores(x, score), -1.0).reshape(len(x), groups, -1)
    best = np.sort(s, -1)[..., ::-1][..., :2]
    rank = np.where(best[..., 0] < 0, -1.0, np.where(best < 0, 0.0, best).sum(-1))
    order = np.argsort(-rank, 1, kind="stable")[:, :top_groups]
    is_open = np.zeros(rank.shape, bool)
    np.put_along_axis(is_open, order, True, 1)
    key = np.where(np.repeat(is_open, x.shape[1] // groups, 1), x, -np.inf)
    ids = np.argsort(-key, 1, kind="stable")[:, :k]
    return np.where(np.take_along_axis(key, ids, 1) > -np.inf, ids, -1)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,groups,top_groups", [(16, 2, 1), (64, 4, 2), (192, 8, 3), (256, 16, 5), (1024, 64, 9)])
def test_two_best_are_summed_as_scores(backend, score, experts, groups, top_groups):
    rng = np.random.default_rng(experts)
    x = (3 * rng.standard_normal((60, experts))).astype(np.float32).astype(np.float64)
    x[rng.random(x.shape) < 0.3] = -np.inf
    x[5] = np.where(np.arange(experts) % (experts // groups) == 1, x[5], -np.inf)  # one of each group
    x[:, 0] = 0.0
    k = min(6, experts // groups * top_groups)
    ids, _ = call(backend, x, k, score=score, groups=groups, top_groups=top_groups, group_best=2)
    assert np.array_equal(ids, choice(x, k, score, groups, top_groups))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_the_row_s_best_expert_beside_a_weak_one(backend, score):
    """e^3 + e^-9 is more than 2 e, 3 - 9 less than 1 + 1; and a group of one live expert is held against sums of two (of sigmoids 0.95 and 1)."""
    x = np.array([[3.0, -9.0, 1.0, 1.0], [3.0, -np.inf, 0.0, 0.0], [0.0, 0.0, 3.0, -np.inf]])
    want = np.array([[0], [0], [2]]) if score == "softmax" else np.array([[2], [2], [0]])
    ids, _ = call(backend, x, 1, score=score, groups=2, top_groups=1, group_best=2)
    assert np.array_equal(ids, want)


def test_a_constant_added_to_a_row_changes_no_softmax(backend):
    """Logits of few bits, so that the sums with a constant are exact."""
    rng = np.random.default_rng(3)
    x = rng.integers(-64, 65, (50, 64)) / 16
    x[rng.random(x.shape) < 0.6] = -np.inf
    x[:, 9] = 0.0
    plain = call(backend, x, 4, groups=8, top_groups=3, group_best=2, renormalize=True)
    for shift in (-20.0, 20.0, 500.0):
        ids, weights = call(backend, x + shift, 4, groups=8, top_groups=3, group_best=2, renormalize=True)
        assert np.array_equal(ids, plain[0]) and np.array_equal(weights, plain[1]), shift


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("best", [1, 2])
def test_a_bias_of_zeros_is_no_bias(backend, score, best):
    rng = np.random.default_rng(best)
    x = 2 * rng.standard_normal((80, 96))
    x[rng.random(x.shape) < 0.2] = -np.inf
    more = dict(score=score, groups=8, top_groups=2, group_best=best, renormalize=True)
    plain, zeros = call(backend, x, 5, **more), call(backend, x, 5, bias=np.zeros(96), **more)
    assert np.array_equal(plain[0], zeros[0]) and np.array_equal(plain[1], zeros[1])
