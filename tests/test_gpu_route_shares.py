"""Weights of a softmax whose chosen scores lie far below the row's largest (Mi355xBackend.route_into)."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_route import REL
from test_gpu_route_groups import call

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("far", [80.0, 95.0, 104.0, 300.0, 5000.0])
@pytest.mark.parametrize("experts", [8, 200])
def test_softmax_shares_far_below_the_row_s_largest(backend, far, experts):
    """Renormalised weights are shares of what is chosen, whatever a bias or a group keeps out."""
    rng = np.random.default_rng(int(far))
    x = rng.standard_normal((20, experts)).astype(np.float32).astype(np.float64)
    x[:, 0] = far

    def near(got, ids):
        part = np.take_along_axis(x, ids, 1)
        part = np.exp(part - part.max(1, keepdims=True))
        want = part / part.sum(1, keepdims=True)
        assert (np.abs(got - want) <= REL * want).all(), (got[0], want[0])

    bias = np.zeros(experts)
    bias[0] = -np.inf
    ids, weights = call(backend, x, 3, bias=bias, renormalize=True)
    assert (ids > 0).all()
    near(weights, ids)
    ids, weights = call(backend, x, 3, bias=np.where(np.arange(experts) == 0, -2.0, 0.0), renormalize=True)
    assert (ids > 0).all()
    near(weights, ids)
