"""Ranges that the attention kernels cut a row's tiles into (kv.h, compiled for the host): every tile is in one, and where a later
run of a captured call has more tiles than at the capture, no range has more than its share."""
from __future__ import annotations

import subprocess

import pytest

import fakehip
from jax4j_amd import build

SOURCE = r"""
#include <stdio.h>
#include <stdlib.h>

#include "kv.h"

using namespace j4q;

int main() {
    for (int splits = 2; splits <= kKvSplits; splits = splits < 20 ? splits + 1 : splits * 2)
        for (int split_tiles : {1, 2, 4, 5, 32, 100, 1000, 1 << 22})
            for (int tiles = 1; tiles <= 1 << 24; tiles = tiles < 300 ? tiles + 1 : tiles * 3 / 2) {
                KvAttend a;
                a.splits = splits;
                a.split_tiles = split_tiles;
                const int each = kv_range_tiles(tiles, a), ranges = kv_ranges(tiles, a);
                const long long share = ((long long)tiles + splits - 1) / splits;
                const long long last = tiles - (ranges - 1ll) * each;
                if (ranges < 1 || ranges > splits || each != (split_tiles > share ? split_tiles : share) || last < 1 || last > each) {
                    printf("%d tiles, %d splits of %d: %d ranges of %d\n", tiles, splits, split_tiles, ranges, each);
                    return 1;
                }
            }
    puts("even");
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    folder = tmp_path_factory.mktemp("ranges")
    (folder / "ranges.hip").write_text(SOURCE)
    subprocess.run([build.HIPCC, "--offload-host-only", "-std=c++17", "-O1", f"-I{build.CSRC}", f"-I{build.ROOT / 'include'}", "-o",
                    str(folder / "ranges"), str(folder / "ranges.hip")], check=True)
    return folder / "ranges"


def test_ranges_of_a_rows_tiles(program):
    p = subprocess.run([str(program)], capture_output=True, text=True)
    assert p.stdout == "even\n", p.stdout + p.stderr


def test_ranges_by_head_size_and_requests(tmp_path):
    """Ranges of a call (without a GPU): one up to as many tiles as were measured to be better off so, for each head size."""
    fakehip.run(fakehip.build_shim(tmp_path), """
        from jax4j_amd import KvCache
        a = address(1 << 20)
        for dim in (64, 96, 128, 192, 256):
            kv = KvCache(be, layers=1, kv_heads=8, head_dim=dim, pages=16 * 64, page_tokens=64, sequences=16, sequence_pages=64)
            one, half = (8, 24) if dim == 256 else (16, 32)
            for requests, tiles, ranges in ((1, one, 1), (1, one + 1, (one + 4) // 4), (16, half, 1), (16, half + 1, 2)):
                kv.truncate(range(16), [0] * 16)
                kv.extend(range(requests), [64 * tiles] * requests)
                kv.begin(range(requests), [1] * requests)
                log()
                kv.attend(0, a, a, 32)
                assert int(launches()[0][3]) == ranges, (dim, requests, tiles)
            kv.destroy()
    """)
