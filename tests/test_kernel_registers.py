"""Registers of the kernels of a block of experts: none may spill.

A spill costs a trip to memory, and where registers are that short this compiler has put copies of live values behind a condition that only a
wave's first lane meets, ahead of the point where all lanes go on, so that the others kept what was there before.
"""
from __future__ import annotations

import subprocess

import pytest

from test_kernel_isa import code_objects

READELF = "/opt/rocm/llvm/bin/llvm-readelf"
OURS = ("norm_kernel", "norm_long_kernel", "route_kernel", "experts_", "row_stats", "expert_bound")


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """{mangled name: (bytes of scratch, spilled vector registers)}"""
    folder, found = tmp_path_factory.mktemp("registers"), {}
    for i, obj in enumerate(code_objects()):
        path = folder / f"{i}.co"
        path.write_bytes(obj)
        name = scratch = None
        for line in subprocess.run([READELF, "--notes", str(path)], capture_output=True, text=True, check=True).stdout.splitlines():
            key, _, value = line.strip().lstrip("- ").partition(":")
            if key == ".name" and value.strip().startswith("_Z"):
                name = value.strip()
            elif key == ".private_segment_fixed_size":
                scratch = int(value)
            elif key == ".vgpr_spill_count" and name:
                found[name] = (scratch, int(value))
    return found


def test_none_spills(kernels):
    ours = {k: v for k, v in kernels.items() if any(n in k for n in OURS)}
    assert len(ours) > 80
    assert not {k: v for k, v in ours.items() if v != (0, 0)}
