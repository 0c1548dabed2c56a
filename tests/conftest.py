"""Shared pytest setup: the `gpu` marker, repo-root imports and the engine fixtures."""
from __future__ import annotations

import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs an MI355X (gfx950) GPU; run with -m gpu")


@pytest.fixture(scope="session")
def backend():
    """The engine on cuda:0. GPU tests fail (not skip) when no gfx950 device is usable,
    like the reference's explicitly enabled GPU suites (CudaTensorTest.java:11-13)."""
    from jax4j_amd import Mi355xBackend

    be = Mi355xBackend()
    assert be.is_available(), "MI355X (gfx950) explicitly required for -m gpu tests"
    info = be.device_info()
    assert info["arch"].startswith("gfx950"), info
    return be


# Their reference ranks groups by sums of two logits. Those are not in the order of sums of scores, and change with a constant added to a
# row, which no softmax does: {3, -inf | 2, 2} gives 3 < 4, the same less 20 gives -17 > -36. test_gpu_route_groups.py holds the sums of scores.
SUMS_OF_LOGITS = [f"test_gpu_route.py::test_groups[False-{groups}]" for groups in ("4-2-2", "8-4-2", "16-3-2")]


def pytest_collection_modifyitems(items):
    for item in items:
        if item.nodeid.endswith(tuple(SUMS_OF_LOGITS)):
            item.add_marker(pytest.mark.xfail(reason="the reference ranks groups by sums of logits", strict=True))
