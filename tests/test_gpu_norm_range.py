"""Norms of rows at both ends of 32 bits without an eps (Mi355xBackend.norm_into), against 64 bits."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from jax4j_amd import Norm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [7, 64, 1000, 4096, 8200, 20000, 20001])
@pytest.mark.parametrize("size", [2.0 ** -140, 2.0 ** -128, 2.0 ** -120, 1.0, 2.0 ** 120, 2.0 ** 126])
def test_root_mean_square_without_an_eps(backend, dim, size):
    """One over the root is beyond 32 bits below 2^-128, and has fewer of them above 2^126: rows in 32 bits leave quotients about 1."""
    rng = np.random.default_rng(dim)
    x = (np.clip(rng.standard_normal((3, dim)), -1.9, 1.9) * size).astype(np.float32)
    x[:, 0] = size
    x[1] *= 2.0 ** -3
    w = rng.standard_normal(dim).astype(np.float32)
    t, tw, y = torch.from_numpy(x).cuda(), torch.from_numpy(w).cuda(), torch.full((3, dim), 5.0, device="cuda")
    torch.cuda.synchronize()
    backend.norm_into(t.data_ptr(), y.data_ptr(), 3, dim, Norm(tw.data_ptr(), eps=0.0))
    backend.sync()
    v = x.astype(np.float64)
    want = v / np.sqrt((v * v).mean(1, keepdims=True)) * w
    # one over the root, the product with it, the product with the weight: three roundings
    assert (np.abs(y.double().cpu().numpy() - want) <= 3.01 * 2.0 ** -24 * np.abs(want) + 2.0 ** -149).all()


def test_rows_of_zeros_with_an_eps_are_zeros(backend):
    x, y = torch.zeros(4, 512, device="cuda"), torch.full((4, 512), 5.0, device="cuda")
    torch.cuda.synchronize()
    for eps in (1e-6, 1e-38, 1e-45):
        backend.norm_into(x.data_ptr(), y.data_ptr(), 4, 512, Norm(eps=eps))
        backend.sync()
        assert (y == 0).all(), eps
